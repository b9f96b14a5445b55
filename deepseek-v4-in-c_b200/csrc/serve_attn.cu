// serve_attn.cu - entry points of the paged serving attention: packed prompts
// (dsv4cu_prompt_attn) and drafted trees over a paged cache
// (dsv4cu_tree_attn).
#include <math.h>

#include "serve_attn.cuh"
#include "serve_umma.cuh"

namespace dsv4cu {

struct Common {              // what both argument structs have
    void *o;
    const void *q, *k, *v;
    long ldo, ldq, ldk, ldv;
    int q_type, kv_type, n_req, nt, n_heads, n_kv, head_dim, window;
    float scale;
};

static int check_common(const char *what, const Common &c)
{
    if (c.n_req < 0 || c.nt < 0) return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: negative count", what);
    if (c.n_heads <= 0 || c.n_kv <= 0 || c.n_heads % c.n_kv)
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: %d query heads over %d key heads", what, c.n_heads, c.n_kv);
    if (c.window < 0) return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: window %d", what, c.window);
    if (!(c.scale > 0.0f) || isinf(c.scale * SA_LOG2E)) return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: scale must be positive and finite", what);
    if (!elem_known(c.q_type) || !elem_known(c.kv_type) || c.kv_type == DSV4CU_F32 ||
        (c.q_type != c.kv_type && !(c.q_type == DSV4CU_F32 && c.kv_type == DSV4CU_BF16)))
        return dsv4cu_set_error(DSV4CU_ERR_UNSUPPORTED, "%s: queries of type %d over keys of type %d", what, c.q_type,
                                c.kv_type);
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256 && c.head_dim != 512)
        return dsv4cu_set_error(DSV4CU_ERR_UNSUPPORTED, "%s: head_dim %d", what, c.head_dim);
    if ((int64_t)c.n_heads * c.head_dim > INT_MAX || c.n_kv > 65535 || (int64_t)c.nt * c.n_heads > INT_MAX)
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: too many heads or tokens", what);
    if (c.n_req == 0 || c.nt == 0) return DSV4CU_OK;
    if (!c.o || !c.q || !c.k) return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: NULL argument", what);
    if (c.o == c.q || c.o == c.k || c.o == c.v) return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: o may not lie over an input", what);
    const int qs = elem_bytes(c.q_type), ks = elem_bytes(c.kv_type);
    const int64_t qrow = (int64_t)c.n_heads * c.head_dim, krow = (int64_t)c.n_kv * c.head_dim;
    if (c.ldo < qrow || c.ldq < qrow || c.ldk < krow || (c.v && c.ldv < krow))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: a token's rows overlap the next one's", what);
    if (!aligned16(c.o) || !aligned16(c.q) || !aligned16(c.k) || !aligned16(c.v) || c.ldo * qs % 16 || c.ldq * qs % 16 ||
        c.ldk * ks % 16 || (c.v && c.ldv * ks % 16))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: rows must be 16-byte aligned", what);
    return DSV4CU_OK;
}

static SaArgs fill_common(const Common &c, const int *cu, const float *sink)
{
    SaArgs s = {};
    s.o = c.o;
    s.q = c.q;
    s.k = c.k;
    s.v = c.v;
    s.ldo = c.ldo;
    s.ldq = c.ldq;
    s.ldk = c.ldk;
    s.ldv = c.ldv;
    s.sink = sink;
    s.cu = cu;
    s.n_req = c.n_req;
    s.nt = c.nt;
    s.hq = c.n_heads;
    s.hkv = c.n_kv;
    sa_set_group(s, c.n_heads / c.n_kv);
    s.window = c.window ? c.window : INT_MAX;
    s.scale2 = c.scale * SA_LOG2E;
    s.splits = 1;
    return s;
}

// The tcgen05 kernel takes 16-bit operands at head dims 64 and 128 where TMA
// can copy the rows (strides below 2^40 bytes; cached pages of a power of two
// of at least 8 rows, the swizzle's period, in fewer than 2^31 slots).
static bool use_umma(const Common &c)
{
    return c.q_type != DSV4CU_F32 && c.head_dim <= 128 && c.ldk < (1l << 38) && (!c.v || c.ldv < (1l << 38));
}
static bool use_umma(const dsv4cu_tree_attn_args *a, const Common &c)
{
    return use_umma(c) && a->page_size >= 8 && (a->page_size & (a->page_size - 1)) == 0 &&
           (int64_t)a->n_pages * a->page_size <= INT_MAX;
}

static int serve_attn_run(const SaArgs &s, const Common &c, bool tree, bool umma, cudaStream_t st)
{
    if (umma)
        return c.q_type == DSV4CU_F16 ? serve_umma_f16(s, c.head_dim, tree, st) : serve_umma_bf16(s, c.head_dim, tree, st);
    if (c.q_type == DSV4CU_F32) return serve_attn_f32(s, c.head_dim, tree, st);
    return c.q_type == DSV4CU_F16 ? serve_attn_f16(s, c.head_dim, tree, st) : serve_attn_bf16(s, c.head_dim, tree, st);
}

static Common common_of(const dsv4cu_prompt_attn_args *a)
{
    return {a->o, a->q, a->k, a->v, a->ldo, a->ldq, a->ldk, a->ldv, a->q_type, a->kv_type, a->n_req, a->nt, a->n_heads,
            a->n_kv, a->head_dim, a->window, a->scale};
}
static Common common_of(const dsv4cu_tree_attn_args *a)
{
    return {a->o, a->q, a->k, a->v, a->ldo, a->ldq, a->ldk, a->ldv, a->q_type, a->kv_type, a->n_req, a->nt, a->n_heads,
            a->n_kv, a->head_dim, a->window, a->scale};
}

static int tree_check(const dsv4cu_tree_attn_args *a, const Common &c)
{
    int r = check_common("tree_attn", c);
    if (r) return r;
    if (a->page_size <= 0 || a->n_pages < 0 || a->max_pages < 0 || a->max_ctx < 0)
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "tree_attn: page_size %d, n_pages %d, max_pages %d, max_ctx %d",
                                a->page_size, a->n_pages, a->max_pages, a->max_ctx);
    if (a->max_nodes <= 0 || a->max_nodes > SA_MAX_NODES)
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "tree_attn: max_nodes %d not in 1 .. %d", a->max_nodes, SA_MAX_NODES);
    if (c.n_req > 65535) return dsv4cu_set_error(DSV4CU_ERR_ARG, "tree_attn: %d requests", c.n_req);
    if ((int64_t)a->max_nodes * c.n_heads > INT_MAX)      // row numbers of a request stay in 32 bits
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "tree_attn: %d nodes of %d heads", a->max_nodes, c.n_heads);
    if ((c.v == nullptr) != (a->v_cache == nullptr) && a->n_pages > 0)
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "tree_attn: v and v_cache go together");
    if (c.n_req == 0 || c.nt == 0) return DSV4CU_OK;
    if (!a->cu || !a->parent || !a->ctx_len || (a->max_pages > 0 && !a->table) || (a->n_pages > 0 && !a->k_cache))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "tree_attn: NULL array");
    if (!aligned16(a->k_cache) || !aligned16(a->v_cache))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "tree_attn: caches must be 16-byte aligned");
    return DSV4CU_OK;
}

// Row tiles, splits and blocks per split of a tree call. Splits only matter
// for speed: they come from the estimate max_ctx, and the kernel spreads the
// real blocks over them.
struct TreeShape {
    bool umma;
    int two, row_tiles, splits, chunk;
};
static TreeShape tree_shape(const dsv4cu_ctx *ctx, const dsv4cu_tree_attn_args *a, const Common &c)
{
    TreeShape s = {};
    s.umma = use_umma(a, c);
    const int64_t rows = (int64_t)a->max_nodes * (a->n_heads / a->n_kv);
    s.two = s.umma && rows > 128;
    const int BM = s.umma ? (s.two ? 256 : 128) : SA_BM, BN = s.umma ? a->head_dim : sa_block(a->head_dim, a->v == nullptr);
    s.row_tiles = (int)((rows + BM - 1) / BM);
    const int64_t ctas = (int64_t)s.row_tiles * a->n_kv * a->n_req;
    const int seen = a->window && a->window < a->max_ctx ? a->window : a->max_ctx;
    const int64_t blocks = (int64_t)seen / BN + 2;        // the cached ones and the nodes' own
    // about 4 CTAs per SM in all (8 where two run at a time): fewer leave SMs
    // idle at the end, more pay for set-up and partial rows - 4 (D + 2) bytes
    // each, written and read, which also sets the least blocks of a split
    const int64_t goal = (int64_t)ctx->sm_count * (s.umma && BN == 64 ? 8 : 4);
    int64_t least = min(rows, (int64_t)BM) * 16 / BN;
    if (least < 256 / BN) least = 256 / BN;
    int64_t chunk = (blocks * ctas + goal - 1) / goal;
    if (chunk < least) chunk = least;
    // the join keeps two numbers per split and row in 64 KB of shared memory
    const int64_t most = s.two ? 30 : 60;
    if (chunk < (blocks + most - 1) / most) chunk = (blocks + most - 1) / most;
    s.chunk = (int)chunk;
    s.splits = (int)((blocks + chunk - 1) / chunk);
    if (ctas > DSV4CU_MAX_COUNTERS) s.splits = 1;         // a counter per tile joins its splits
    return s;
}

static size_t tree_ws(const dsv4cu_tree_attn_args *a, int splits)
{
    if (splits <= 1) return 0;
    const size_t rows = (size_t)splits * a->nt * a->n_heads;
    return 2 * dsv4cu_align256(rows * 4) + dsv4cu_align256(rows * a->head_dim * 4);
}

}  // namespace dsv4cu

using namespace dsv4cu;

extern "C" int dsv4cu_prompt_attn(dsv4cu_ctx *ctx, const dsv4cu_prompt_attn_args *a, void *stream)
{
    if (!ctx || !a) return dsv4cu_set_error(DSV4CU_ERR_ARG, "prompt_attn: NULL argument");
    const Common c = common_of(a);
    int r = check_common("prompt_attn", c);
    if (r) return r;
    if (c.n_req == 0 || c.nt == 0) return DSV4CU_OK;
    if (!a->cu) return dsv4cu_set_error(DSV4CU_ERR_ARG, "prompt_attn: NULL cu");
    DeviceGuard guard;
    DSV4CU_CUDA_TRY(guard.enter(ctx->device));
    SaArgs s = fill_common(c, a->cu, a->sink);
    s.status = ctx->status;
    s.sms = ctx->sm_count;
    return serve_attn_run(s, c, false, use_umma(c), (cudaStream_t)stream);
}

extern "C" size_t dsv4cu_tree_attn_workspace(const dsv4cu_ctx *ctx, const dsv4cu_tree_attn_args *a)
{
    if (!ctx || !a || tree_check(a, common_of(a)) || a->n_req == 0 || a->nt == 0) return 0;
    return tree_ws(a, tree_shape(ctx, a, common_of(a)).splits);
}

extern "C" int dsv4cu_tree_attn(dsv4cu_ctx *ctx, const dsv4cu_tree_attn_args *a, void *stream)
{
    if (!ctx || !a) return dsv4cu_set_error(DSV4CU_ERR_ARG, "tree_attn: NULL argument");
    const Common c = common_of(a);
    int r = tree_check(a, c);
    if (r) return r;
    if (c.n_req == 0 || c.nt == 0) return DSV4CU_OK;
    DeviceGuard guard;
    DSV4CU_CUDA_TRY(guard.enter(ctx->device));
    SaArgs s = fill_common(c, a->cu, a->sink);
    s.kc = a->k_cache;
    s.vc = a->v_cache;
    s.table = a->table;
    s.ctx_len = a->ctx_len;
    s.parent = a->parent;
    s.page_size = a->page_size;
    s.page_log2 = -1;
    for (int i = 0; i < 31; i++)
        if (a->page_size == 1 << i) s.page_log2 = i;
    s.n_pages = a->n_pages;
    s.max_pages = a->max_pages;
    s.max_nodes = a->max_nodes;
    s.status = ctx->status;
    s.counters = ctx->counters;
    const TreeShape shape = tree_shape(ctx, a, c);
    s.two = shape.two;
    s.row_tiles = shape.row_tiles;
    s.splits = shape.splits;
    s.chunk = shape.chunk;
    if (s.splits > 1) {
        void *ws = nullptr;
        r = dsv4cu_ws_get(ctx, tree_ws(a, s.splits), &ws);
        if (r) return r;
        const size_t rows = dsv4cu_align256((size_t)s.splits * a->nt * a->n_heads * 4);
        s.pm = (float *)ws;
        s.pl = (float *)((char *)ws + rows);
        s.po = (float *)((char *)ws + 2 * rows);
    }
    return serve_attn_run(s, c, true, shape.umma, (cudaStream_t)stream);
}

// serve_attn.cuh - softmax attention of packed queries, for packed prompts and
// for trees of drafted tokens over a paged cache: what the two kernels share
// (masks, rows, splits and their join) and the mma.sync kernel, which covers
// every head dim, fp32 queries and any page size.
//
//   o_i = sum_{j in M(i)} e_ij v_j / (sum_{j in M(i)} e_ij + e^sink / e^m_i),
//   e_ij = exp(scale q_i.k_j - m_i), m_i the running maximum over M(i).
//
// A tile is 32 rows of one key head: row r is (token r / G, head r % G) of the
// G query heads that share it, so grouped heads read a key once. The keys come
// in blocks of BN, a bulk copy per row, into two stages of shared memory. The NW warps of a CTA each own D / NW of the head's
// dims for the whole pass - of the queries (mma fragments in registers), of
// the scores' contraction, and of the output's columns - so a head dim of 512
// needs no more than 255 registers a thread, and where the values are the key
// rows (this engine's latent cache) a warp reads the same slice of the same
// tile for both products. Per block: partial scores over the warp's dims to
// shared memory, their sum and the softmax by THREADS / 32 threads per row, the
// weights back through shared memory, then the output.
//
// fp32 queries (TERMS = 3) over a bf16 cache enter as three bf16 terms
// q = t0 + t1 + t2, which carry all 24 significand bits, and so do the
// weights: products are those of fp32. 16-bit queries use the weights rounded
// to the cache's type (up to 2^-8 of each weight in bf16, 2^-11 in f16: the size
// of the output's own rounding). The tensor core's own additions cut off low bits
// (toward zero, so they do not average out), therefore it only adds within a
// block; blocks are added in fp32 with rounding to nearest.
//
// Bound by mma.sync: 556 TFLOP/s at most on a B200, a third of tcgen05's, but
// 512 output columns and the scores do not fit TMEM together, and three terms
// of 128 query rows do not fit shared memory; 256 dims in 16 bits would fit
// tcgen05 and have no kernel there. Measured with 64 fp32 heads of
// 512 dims: 6 trees over up to 9000 tokens 201 us (51 GFLOP in three terms: 255
// TFLOP/s; of a block's time 0.30 in each product, 0.18 in the softmax); 301
// prompt tokens in a window of 128, 70 us (a third of it set-up and output of
// 602 tiles of two or three blocks). Copies of 16 bytes instead of whole rows
// cost 0.14 of a block's time.
//
// Masked entries: a masked score is -inf whatever its key holds. A masked
// value row is multiplied by a weight of exactly 0, which is only harmless
// when the value is finite: 0 x infinity and 0 x NaN are NaN. So a tile whose
// output is not finite looks (sa_suspect) for a non-finite value behind a mask
// - where a visible weight may also be 0 in 16 bits though it is not (the last
// of three terms, an f16 weight below 2^-25), also for a visible infinity, of
// keys too, whose queries have terms - and if there is one, serve_slow_rows
// computes the tile again from visible keys only. Rows outside a sequence and pages outside the pool are
// zeros in shared memory and are masked.
#pragma once

#include <limits.h>

#include "serve.h"
#include "tma_gemv.cuh"

namespace dsv4cu {

constexpr int SA_MAX_NODES = 128;
constexpr float SA_LOG2E = 1.4426950408889634f;
enum { SA_COPY = 77 };                // dsv4cu_ctx_status: a copy that did not arrive

struct SaArgs {
    const void *q, *k, *v;            // packed rows; v == NULL: the key rows are the values
    void *o;
    const float *sink;                // [hq] or NULL
    long ldq, ldk, ldv, ldo;          // elements between tokens
    const int *cu;                    // [n_req + 1]
    int n_req, nt, hq, hkv, G;
    unsigned g_mul, g_shift;          // x / G for 0 <= x < 2^31: sa_token
    int window;                       // keys a row may look back over, INT_MAX: all
    float scale2;                     // scale * log2 e
    // tree
    const void *kc, *vc;              // [n_pages][page_size][hkv][D]
    const int *table, *ctx_len, *parent;
    int page_size, page_log2, n_pages, max_pages;   // page_log2 < 0: not a power of two
    int max_nodes, row_tiles, splits;
    int chunk;                        // key blocks of a split, at least
    float *pm, *pl, *po;              // partials [splits][nt * hq](, D), splits > 1
    int *counters;                    // [n_req][hkv][row_tiles], zero between calls: splits done
    int *status;
    int sms, heads_first;             // prompts: SMs, order of the grid (sa_prompt_grid)
    int nst, two, box_log2;           // tcgen05 kernel: stages, two strips of rows per CTA, rows of a cached copy's box
};

// Token of a request's row: row / G, by a multiplication (Granlund and
// Montgomery 1994; m = g_mul below 2^32, rows below 2^31, so the sum fits).
static inline void sa_set_group(SaArgs &a, int G)
{
    a.G = G;
    a.g_shift = 0;
    while ((1ll << a.g_shift) < G) a.g_shift++;
    a.g_mul = (unsigned)((((1ull << a.g_shift) - (unsigned)G) << 32) / (unsigned)G + 1);
}
DSV4CU_DEV int sa_token(const SaArgs &a, int row) { return (int)((__umulhi((unsigned)row, a.g_mul) + (unsigned)row) >> a.g_shift); }

// The key blocks of request b of a tree call: blocks of BN cached keys from
// key0 on (no row looks further back than the shallowest one, at position
// ctx), then blocks of the request's own nodes; a split takes `per` of them
// and `used` splits have any.
struct SaSpan {
    int begin, len, ctx, kend, key0, nblk_c, nblk, per, used;   // kend: cached keys that the table can hold
};
DSV4CU_DEV SaSpan sa_span(const SaArgs &a, int b, int BN)
{
    SaSpan s;
    const int lo = __ldg(a.cu + b), hi = __ldg(a.cu + b + 1);
    s.begin = max(0, min(lo, a.nt));
    s.len = max(s.begin, min(hi, a.nt)) - s.begin;
    s.ctx = max(0, min(__ldg(a.ctx_len + b), INT_MAX - (1 << 20)));   // positions stay in 32 bits
    s.kend = (int)min((int64_t)s.ctx, (int64_t)a.max_pages * a.page_size);
    const int first = a.window > s.ctx ? 0 : s.ctx - a.window + 1;
    s.key0 = first / BN * BN;
    s.nblk_c = max(0, s.kend - s.key0 + BN - 1) / BN;
    s.nblk = s.nblk_c + (s.len + BN - 1) / BN;
    s.per = a.chunk;                                     // (nblk <= chunk * splits where max_ctx was right)
    if ((int64_t)a.chunk * a.splits < s.nblk) s.per = (s.nblk + a.splits - 1) / a.splits;
    s.used = (s.nblk + s.per - 1) / s.per;
    return s;
}

DSV4CU_DEV uint32_t sa_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// One contiguous copy, counted in bytes on `bar`; addresses and size multiples
// of 16.
DSV4CU_DEV void sa_bulk(void *dst, const void *src, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(sa_smem(dst)), "l"(src), "r"(bytes), "r"(sa_smem(bar)) : "memory");
}
DSV4CU_DEV void sa_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Bounded wait that polls: no suspend hint and no look at the clock on the
// way to a phase that completes in time.
DSV4CU_DEV bool sa_poll(uint64_t *bar, uint32_t parity, int *err, int code)
{
    const uint32_t a = sa_smem(bar);
    uint64_t t0 = 0;
    for (uint32_t i = 1;; i++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(a), "r"(parity) : "memory");
        if (ok) return true;
        if ((i & 1023u) == 0u) {
            const uint64_t now = globaltimer_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > MBAR_TIMEOUT_NS) break;
        }
    }
    atomicCAS(err, 0, code);
    return false;
}
DSV4CU_DEV void sa_ldsm4(uint32_t (&r)[4], const void *p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(sa_smem(p)) : "memory");
}
DSV4CU_DEV void sa_ldsm4_t(uint32_t (&r)[4], const void *p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(sa_smem(p)) : "memory");
}
template <bool F16>
DSV4CU_DEV void sa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                     "{%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                     "{%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
DSV4CU_DEV float sa_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool F16>
DSV4CU_DEV uint32_t sa_pack(float x, float y)
{
    if constexpr (F16) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
// Two values as TERMS packed words (bf16 terms). Every term but the last is
// what the ones before left over, cut to bf16's 8 significand bits: cutting
// cannot pass the largest bf16 as rounding up does for the largest floats, the
// subtractions are exact, and three terms of 8 bits hold all 24.
template <int TERMS, bool F16>
DSV4CU_DEV void sa_split(float x, float y, uint32_t (&w)[TERMS])
{
#pragma unroll
    for (int t = 0; t + 1 < TERMS; t++) {
        w[t] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
        x -= __uint_as_float(w[t] << 16);
        y -= __uint_as_float(w[t] & 0xFFFF0000u);
    }
    w[TERMS - 1] = sa_pack<F16>(x, y);
}
template <bool F16>
DSV4CU_DEV float sa_float(uint16_t b)
{
    if constexpr (F16) return __half2float(__ushort_as_half(b));
    else return __uint_as_float((uint32_t)b << 16);
}
template <bool F16>
DSV4CU_DEV bool sa_nonfinite(uint32_t w)
{
    constexpr uint32_t E = F16 ? 0x7C00u : 0x7F80u;
    return (w & E) == E || (w & (E << 16)) == (E << 16);
}
// The rows and keys of one CTA.
struct SaTile {
    int begin, len;       // token range of the request / sequence
    int r0, rows;         // first row of the tile, rows in it
    int kvh;
    int ctx, kend, key0;  // tree: cached tokens, those that the table holds; first key of the first (cached) block
    int nblk_c, blk0, blk1;   // cached blocks; this CTA's range of blocks (cached first, then nodes)
    int split, parts;     // tree: which split of how many
    const int *table;
};

// Sequence and tile of the prompt CTA number `id`. Sequence b has
// ceil(len * G / 2^LOG) tiles, and a later tile has more keys: CTAs start in the
// order of falling tile numbers over all sequences, so the short ones fill the
// end (29 prompts of 16001 tokens, 16 heads over 4, 64 dims: 75 us, sequence
// after sequence 91 us; 69 us since). For that a warp holds the tile counts of up to
// SA_SORTED sequences and searches for the tile number whose CTAs include `id`.
// More sequences come one after the other, in reverse, and so do tiles that a
// window of up to SA_EVEN keys makes nearly equal: there the search only costs
// (301 tokens of 64 heads of 512 dims, window 128: 77 against 70 us). All lanes
// of the warp return the same; begin < 0: no such tile.
constexpr int SA_SORTED = 128, SA_EVEN = 1024;
// Tiles of 2^log rows of n tokens; n * G fits 31 bits.
DSV4CU_DEV int sa_tiles(int n, int G, int log) { return (int)(((unsigned)(n * G) + (1u << log) - 1u) >> log); }
template <int R, int LOG>
DSV4CU_DEV void sa_find_sorted(const int *cu, int n_req, int nt, int G, int id, int &begin, int &len, int &tile)
{
    const int lane = threadIdx.x & 31;
    int lo[R], n[R], tiles[R], most = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int b = 32 * r + lane;
        lo[r] = n[r] = tiles[r] = 0;
        if (b < n_req) {
            lo[r] = max(0, min(__ldg(cu + b), nt));
            n[r] = max(lo[r], min(__ldg(cu + b + 1), nt)) - lo[r];
            tiles[r] = sa_tiles(n[r], G, LOG);
        }
        most = max(most, tiles[r]);
    }
    // the least x such that the tiles numbered x or higher are at most id
    int none = -1, x = __reduce_max_sync(0xFFFFFFFFu, most), before = 0;
    while (x - none > 1) {
        const int mid = (x + none) >> 1;
        int c = 0;
#pragma unroll
        for (int r = 0; r < R; r++) c += max(0, tiles[r] - mid);
        c = __reduce_add_sync(0xFFFFFFFFu, c);
        if (c <= id) {
            x = mid;
            before = c;
        } else {
            none = mid;
        }
    }
    tile = x - 1;
    int at = id - before;                            // among the sequences with a tile of this number
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool has = tile >= 0 && tiles[r] > tile;
        const unsigned m = __ballot_sync(0xFFFFFFFFu, has);
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, has && __popc(m & ((1u << lane) - 1u)) == at);
        if (hit && begin < 0) {
            begin = __shfl_sync(0xFFFFFFFFu, lo[r], __ffs(hit) - 1);
            len = __shfl_sync(0xFFFFFFFFu, n[r], __ffs(hit) - 1);
        }
        at -= __popc(m);
    }
}
template <int LOG>
DSV4CU_DEV void sa_find(const SaArgs &a, int &begin, int &len, int &tile)
{
    const int *cu = a.cu, n_req = a.n_req, nt = a.nt, G = a.G;
    int id = a.heads_first ? blockIdx.y : blockIdx.x;
    const int lane = threadIdx.x & 31;
    begin = -1;
    len = tile = 0;
    if (n_req <= SA_SORTED && a.window > SA_EVEN) {
        if (n_req <= 32) sa_find_sorted<1, LOG>(cu, n_req, nt, G, id, begin, len, tile);
        else sa_find_sorted<SA_SORTED / 32, LOG>(cu, n_req, nt, G, id, begin, len, tile);
        return;
    }
    id = (a.heads_first ? gridDim.y : gridDim.x) - 1 - id;
    int before = 0;
    for (int b0 = 0; b0 < n_req; b0 += 32) {
        const int b = b0 + lane;
        int lo = 0, n = 0;
        if (b < n_req) {
            lo = max(0, min(__ldg(cu + b), nt));
            n = max(lo, min(__ldg(cu + b + 1), nt)) - lo;
        }
        const int mine = sa_tiles(n, G, LOG);
        int pre = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xFFFFFFFFu, pre, o);
            if (lane >= o) pre += y;
        }
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, id < before + pre);
        if (hit) {
            const int l = __ffs(hit) - 1;
            begin = __shfl_sync(0xFFFFFFFFu, lo, l);
            len = __shfl_sync(0xFFFFFFFFu, n, l);
            tile = id - before - __shfl_sync(0xFFFFFFFFu, pre - mine, l);
            return;
        }
        before += __shfl_sync(0xFFFFFFFFu, pre, 31);
    }
}
// The grid of a prompt call of `tiles` tiles per key head: where they do not
// fill the GPU (`slots` CTAs) head by head, CTAs of all heads start in the same
// order (x the head); otherwise the heads come one after the other, whose keys
// then stay in L2 (32768 tokens of 64 heads over 8, 128 dims: 5 in 100 faster).
static inline dim3 sa_prompt_grid(SaArgs &a, int64_t tiles, int slots)
{
    a.heads_first = tiles < slots;
    return a.heads_first ? dim3(a.hkv, (unsigned)tiles) : dim3((unsigned)tiles, a.hkv);
}

// Row of cached key j, or NULL where its page is not in the pool.
DSV4CU_DEV const uint16_t *sa_cached(const SaArgs &a, const SaTile &t, const void *cache, int j, int D)
{
    const int pg = a.page_log2 >= 0 ? j >> a.page_log2 : j / a.page_size;
    if (pg >= a.max_pages) return nullptr;
    const int id = __ldg(t.table + pg);
    if (id < 0 || id >= a.n_pages) return nullptr;
    const size_t slot = (size_t)id * a.page_size + (j - pg * a.page_size);
    return reinterpret_cast<const uint16_t *>(cache) + (slot * a.hkv + t.kvh) * D;
}

template <bool F16, bool QF32>
DSV4CU_DEV float sa_load_q(const SaArgs &a, size_t at)
{
    if constexpr (QF32) return __ldg(reinterpret_cast<const float *>(a.q) + at);
    else return sa_float<F16>(__ldg(reinterpret_cast<const uint16_t *>(a.q) + at));
}
template <bool F16, bool OF32>
DSV4CU_DEV void sa_store_o(const SaArgs &a, size_t at, float x)
{
    if constexpr (OF32) reinterpret_cast<float *>(a.o)[at] = x;
    else reinterpret_cast<uint16_t *>(a.o)[at] = (uint16_t)(sa_pack<F16>(x, 0.0f) & 0xFFFFu);
}
// 1 / (l + sink term); a row without any visible key gives 0.
DSV4CU_DEV float sa_inv(float l, float m, const float *sink, int head)
{
    if (sink) l += sa_exp2(__ldg(sink + head) * SA_LOG2E - m);
    return l == 0.0f ? 0.0f : 1.0f / l;
}

// Whether a value of the tile's blocks could have made its output non-finite
// against the mask: a value that is not finite in a block that a mask crosses
// (full(block) false), or with ALL an infinite one anywhere, of the keys as
// well. This thread's share of the keys; rows are read from memory, D / 8
// pieces each.
template <int D, bool F16, bool ALL, class Full, class Row>
DSV4CU_DEV bool sa_suspect(const SaTile &t, int BN, int thread, int threads, Full full, Row row)
{
    constexpr uint32_t E = F16 ? 0x7C00u : 0x7F80u, M = F16 ? 0x03FFu : 0x007Fu;
    bool found = false;
    for (int blk = t.blk0; blk < t.blk1; blk++) {
        const bool masked = !full(blk);
        if (!masked && !ALL) continue;
        for (int x = thread; x < BN * (D / 8); x += threads) {
            const int j = x / (D / 8);
#pragma unroll
            for (int kv = ALL ? 0 : 1; kv < 2; kv++) {
                const uint16_t *v = row(blk, j, kv == 1);
                if (!v) continue;
                const uint4 w = __ldg(reinterpret_cast<const uint4 *>(v + (x - j * (D / 8)) * 8));
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (masked && kv == 1) found = found || sa_nonfinite<F16>(u[e]);
                    else found = found || (u[e] & (E | M)) == E || ((u[e] >> 16) & (E | M)) == E;
                }
            }
        }
    }
    return found;
}

// The tile's rows one by one, a warp per row and a lane per key, visible keys
// only, everything in fp32: the form that a tile falls back to when a value
// behind a mask is not finite. vis(token, block, key in block) and
// row(block, key in block, values) are the tile kernel's own mask and addresses.
template <int D, bool F16, bool QF32, class Vis, class Row>
__device__ __noinline__ void serve_slow_rows(const SaArgs &a, const SaTile &t, int BN, int warp, int warps, Vis vis,
                                             Row row)
{
    const int lane = threadIdx.x & 31;
    constexpr int E = D / 32;
    for (int r = warp; r < t.rows; r += warps) {
        const int tok = sa_token(a, t.r0 + r), head = t.kvh * a.G + t.r0 + r - tok * a.G;
        const size_t qat = (size_t)(t.begin + tok) * a.ldq + (size_t)head * D;
        float m = -INFINITY, l = 0.0f, o[E];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = 0.0f;
        for (int blk = t.blk0; blk < t.blk1; blk++)
            for (int j0 = 0; j0 < BN; j0 += 32) {
                const int j = j0 + lane;
                const bool see = j < BN && vis(tok, blk, j);
                float s = -INFINITY;
                if (see) {
                    const uint16_t *k = row(blk, j, false);
                    float dot = 0.0f;
                    for (int d = 0; d < D; d++) dot = fmaf(sa_load_q<F16, QF32>(a, qat + d), sa_float<F16>(__ldg(k + d)), dot);
                    s = dot * a.scale2;
                }
                float top = s;
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                const float nm = fmaxf(m, top), use = nm == -INFINITY ? 0.0f : nm;
                const float alpha = sa_exp2(m - use), p = see ? sa_exp2(s - use) : 0.0f;
                m = nm;
                float ps = p;
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) ps += __shfl_xor_sync(0xFFFFFFFFu, ps, x);
                l = l * alpha + ps;
#pragma unroll
                for (int e = 0; e < E; e++) o[e] *= alpha;
                unsigned todo = __ballot_sync(0xFFFFFFFFu, see);
                while (todo) {
                    const int jj = __ffs(todo) - 1;
                    todo &= todo - 1;
                    const float w = __shfl_sync(0xFFFFFFFFu, p, jj);
                    const uint16_t *v = row(blk, j0 + jj, true);
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] = fmaf(w, sa_float<F16>(__ldg(v + lane + 32 * e)), o[e]);
                }
            }
        if (t.parts > 1) {
            const size_t id = (size_t)t.split * a.nt * a.hq + (size_t)(t.begin + tok) * a.hq + head;
#pragma unroll
            for (int e = 0; e < E; e++) a.po[id * D + lane + 32 * e] = o[e];
            if (lane == 0) {
                a.pm[id] = m;
                a.pl[id] = l;
            }
        } else {
            const float inv = sa_inv(l, m, a.sink, head);
            const size_t at = (size_t)(t.begin + tok) * a.ldo + (size_t)head * D;
#pragma unroll
            for (int e = 0; e < E; e++) sa_store_o<F16, QF32>(a, at + lane + 32 * e, o[e] * inv);
        }
    }
}

// Joins the splits of a tile's rows: the partial outputs rescaled to the row's
// largest maximum and divided by the joint exp-sum (with the sink), in split
// order whichever split came last. No factor is below SA_LEAST, which adds nothing
// to a finite sum but keeps a visible infinity or NaN of a split that weighs next
// to nothing (a row of NaN scores alone has no maximum; a split without a visible
// key has sums of exactly 0). First the maxima and sums into sm (2 parts
// + 1 numbers a row), a row's factors by a thread; then the outputs, four
// columns per thread.
constexpr float SA_LEAST = 1.1754944e-38f;   // 2^-126
template <int D, bool F16, bool QF32, class Sync>
DSV4CU_DEV void sa_join(const SaArgs &a, const SaTile &t, float *sm, int tid, int threads, Sync sync)
{
    const size_t step = (size_t)a.nt * a.hq;
    const int rows = t.rows, parts = t.parts;
    float *inv = sm + parts * rows;
    float *ls = inv + rows;                              // [parts][rows]
    for (int x = tid; x < parts * rows; x += threads) {
        const int p = x / rows, r = x - p * rows, pr = t.r0 + r, tok = sa_token(a, pr), head = t.kvh * a.G + pr - tok * a.G;
        const size_t id = (size_t)(t.begin + tok) * a.hq + head + p * step;
        sm[x] = __ldcg(a.pm + id);
        ls[x] = __ldcg(a.pl + id);
    }
    sync();
    for (int r = tid; r < rows; r += threads) {
        float m = -INFINITY, l = 0.0f;
        for (int s = 0; s < parts; s++) {
            const float x = sm[s * rows + r];
            m = x > m || x != x ? x : m;                 // a NaN row stays one
        }
        const float use = m == -INFINITY ? 0.0f : m;
        for (int s = 0; s < parts; s++) {
            const float f = fmaxf(sa_exp2(sm[s * rows + r] - use), SA_LEAST);
            sm[s * rows + r] = f;
            l = fmaf(ls[s * rows + r], f, l);
        }
        inv[r] = sa_inv(l, m, a.sink, t.kvh * a.G + t.r0 + r - sa_token(a, t.r0 + r) * a.G);
    }
    sync();
    constexpr int B = 8;                                 // splits read at once, of two pieces each
    for (int x0 = tid; x0 < rows * (D / 4); x0 += 2 * threads) {
        float4 o[2];
        const float *src[2];
        int row[2];
        size_t at[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int x = min(x0 + u * threads, rows * (D / 4) - 1);   // the last piece twice where there is no second
            const int r = x / (D / 4), c = (x - r * (D / 4)) * 4, pr = t.r0 + r, tok = sa_token(a, pr),
                      head = t.kvh * a.G + pr - tok * a.G;
            o[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            row[u] = r;
            src[u] = a.po + ((size_t)(t.begin + tok) * a.hq + head) * D + c;
            at[u] = (size_t)(t.begin + tok) * a.ldo + (size_t)head * D + c;
        }
        for (int s0 = 0; s0 < parts; s0 += B) {
            float4 y[2][B];
#pragma unroll
            for (int s = 0; s < B; s++)
#pragma unroll
                for (int u = 0; u < 2; u++)
                    y[u][s] = s0 + s < parts ? __ldcg(reinterpret_cast<const float4 *>(src[u] + (s0 + s) * step * D))
                                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int s = 0; s < B; s++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float f = s0 + s < parts ? sm[(s0 + s) * rows + row[u]] : 0.0f;
                    o[u].x = fmaf(y[u][s].x, f, o[u].x);
                    o[u].y = fmaf(y[u][s].y, f, o[u].y);
                    o[u].z = fmaf(y[u][s].z, f, o[u].z);
                    o[u].w = fmaf(y[u][s].w, f, o[u].w);
                }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const float i = inv[row[u]];
            if constexpr (QF32)
                *reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.o) + at[u]) =
                    make_float4(o[u].x * i, o[u].y * i, o[u].z * i, o[u].w * i);
            else
                *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.o) + at[u]) =
                    make_uint2(sa_pack<F16>(o[u].x * i, o[u].y * i), sa_pack<F16>(o[u].z * i, o[u].w * i));
        }
    }
}

constexpr int SA_BM = 32;             // rows of a tile
constexpr int sa_warps(int D) { return D >= 128 ? 8 : 4; }

template <int D, int BN, int TERMS, bool F16, bool TREE>
__global__ void __launch_bounds__(32 * sa_warps(D), 1) serve_attn_kernel(const __grid_constant__ SaArgs a)
{
    constexpr int NW = sa_warps(D), THREADS = 32 * NW, BM = SA_BM;
    constexpr int RS = D + 8;                            // row stride of keys and values: 16 bytes over, so ldmatrix rows spread
    constexpr int DW = D / NW, KS = DW / 16, ON = DW / 8;   // dims of a warp, their k steps, their output n tiles
    constexpr int OG = ON < 4 ? ON : 4;                  // output n tiles accumulated at a time
    constexpr int SS = BN + 8, PS = BN + 8;              // row strides of partial scores and weights
    constexpr int TPR = THREADS / BM, CPT = BN / TPR;    // softmax: threads per row, columns per thread
    constexpr bool QF32 = TERMS > 1;
    static_assert(!(QF32 && F16), "three terms are bf16 terms");
    static_assert(KS >= 1 && ON % OG == 0 && OG % 2 == 0 && CPT % 4 == 0, "shape");
    extern __shared__ __align__(128) uint16_t sa_sm[];
    __shared__ int s_par[TREE ? SA_MAX_NODES : 1], s_depth[TREE ? SA_MAX_NODES : 1];
    __shared__ unsigned long long s_anc[TREE ? SA_MAX_NODES : 1][2];
    __shared__ __align__(8) uint64_t s_full[2];
    __shared__ uint8_t s_there[2][BN];                   // the key is there
    __shared__ int s_bad[2];                             // block with a missing row
    __shared__ float s_alpha[BM], s_m[BM], s_l[BM];
    const bool shared_v = a.v == nullptr;
    const int stage_el = (shared_v ? 1 : 2) * BN * RS;
    uint16_t *kvs = sa_sm;                               // [2][shared_v ? 1 : 2][BN][RS]
    float *part = reinterpret_cast<float *>(kvs + 2 * stage_el);       // [NW][BM][SS]
    uint16_t *ps = reinterpret_cast<uint16_t *>(part + NW * BM * SS);  // [TERMS][BM][PS]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;

    // ---- which rows and keys
    SaTile t;
    t.ctx = t.kend = t.key0 = t.nblk_c = t.split = 0;
    t.parts = 1;
    t.table = nullptr;
    t.kvh = !TREE && a.heads_first ? blockIdx.x : blockIdx.y;
    if constexpr (TREE) {
        const int b = blockIdx.z;
        const SaSpan sp = sa_span(a, b, BN);
        t.split = a.row_tiles == 1 ? blockIdx.x : blockIdx.x / a.row_tiles;
        t.begin = sp.begin;
        t.len = sp.len;
        if (t.len > a.max_nodes) {                       // refused whole: its rows are left as they were
            if (tid == 0) serve_refuse(a.status, DSV4CU_TREE_NODES);
            return;
        }
        if (t.split >= sp.used) return;
        t.parts = sp.used;
        t.r0 = (blockIdx.x - t.split * a.row_tiles) * BM;
        t.ctx = sp.ctx;
        t.kend = sp.kend;
        t.table = a.table + (size_t)b * a.max_pages;
        t.key0 = sp.key0;
        t.nblk_c = sp.nblk_c;
        t.blk0 = t.split * sp.per;
        t.blk1 = min(sp.nblk, t.blk0 + sp.per);
    } else {
        int tile;
        sa_find<5>(a, t.begin, t.len, tile);
        static_assert(BM == 32, "rows of a tile");
        if (t.begin < 0) return;
        t.r0 = tile * BM;
    }
    t.rows = min(BM, t.len * a.G - t.r0);
    if (t.rows <= 0) return;
    const int t_lo = sa_token(a, t.r0), t_hi = sa_token(a, t.r0 + t.rows - 1);
    if constexpr (!TREE) {
        t.key0 = a.window > t_lo ? 0 : t_lo - a.window + 1;   // blocks start at the first key of the window
        t.blk0 = 0;
        t.blk1 = (t_hi - t.key0) / BN + 1;
    }
    if constexpr (TREE) {
        // ancestors-or-self as bit sets, depths; a parent that does not come
        // before its child counts as none
        for (int i = tid; i < t.len; i += THREADS) s_par[i] = __ldg(a.parent + t.begin + i);
        __syncthreads();
        for (int i = tid; i < t.len; i += THREADS) {
            unsigned long long set[2] = {0, 0};
            int d = -1, x = i;
            for (;;) {
                set[x >> 6] |= 1ull << (x & 63);
                d++;
                const int p = s_par[x];
                if (p < 0 || p >= x) break;
                x = p;
            }
            s_anc[i][0] = set[0];
            s_anc[i][1] = set[1];
            s_depth[i] = d;
        }
    }
    // a key of block blk: its address, and whether token tok sees it (by
    // value: the fallback's call must not pin the tile to local memory)
    const SaArgs &a0 = a;
    auto row = [t, shared_v, ap = &a0](int blk, int j, bool values) -> const uint16_t * {
        const SaArgs &a = *ap;
        const bool vv = values && !shared_v;
        if (TREE && blk < t.nblk_c) {
            const int key = t.key0 + blk * BN + j;
            return key < t.kend ? sa_cached(a, t, vv ? a.vc : a.kc, key, D) : nullptr;
        }
        const int key = TREE ? (blk - t.nblk_c) * BN + j : t.key0 + blk * BN + j;
        if (key >= t.len) return nullptr;
        return reinterpret_cast<const uint16_t *>(vv ? a.v : a.k) + (size_t)(t.begin + key) * (vv ? a.ldv : a.ldk) +
               (size_t)t.kvh * D;
    };
    auto vis = [t, row, ap = &a0](int tok, int blk, int j) -> bool {
        const SaArgs &a = *ap;
        if constexpr (TREE) {
            if (blk < t.nblk_c) {
                const int key = t.key0 + blk * BN + j;
                return key < t.kend && t.ctx - key + s_depth[tok] < a.window && row(blk, j, false) != nullptr;
            }
            const int x = (blk - t.nblk_c) * BN + j;
            return x < t.len && (s_anc[tok][x >> 6] >> (x & 63) & 1) && s_depth[tok] - s_depth[x] < a.window;
        } else {
            const int key = t.key0 + blk * BN + j;
            return key <= tok && tok - key < a.window;
        }
    };
    // Thread j < BN brings row j of every block: a copy of the whole row, or
    // zeros where there is none. The row's address is looked up a block ahead.
    const uint16_t *next_k = nullptr, *next_v = nullptr;
    auto look_up = [&](int blk) {
        next_k = next_v = nullptr;
        if (tid < BN && blk < t.blk1) {
            next_k = row(blk, tid, false);
            if (!shared_v) next_v = row(blk, tid, true);
        }
    };
    auto issue = [&](int blk) {                          // the rows of the last look_up
        if (tid >= BN) return;
        const int st = (blk - t.blk0) & 1;
        uint16_t *dst = kvs + st * stage_el + tid * RS;
        s_there[st][tid] = next_k != nullptr;
        if (next_k) {
            mbar_arrive_expect_tx(&s_full[st], (shared_v ? 1 : 2) * D * 2);
            sa_bulk(dst, next_k, D * 2, &s_full[st]);
            if (!shared_v) sa_bulk(dst + BN * RS, next_v, D * 2, &s_full[st]);
        } else {
            s_bad[st] = blk;
            for (int c = 0; c < D; c += 8) {
                *reinterpret_cast<uint4 *>(dst + c) = make_uint4(0, 0, 0, 0);
                if (!shared_v) *reinterpret_cast<uint4 *>(dst + BN * RS + c) = make_uint4(0, 0, 0, 0);
            }
            sa_fence_async();                            // before a later copy into the same place
            mbar_arrive(&s_full[st]);
        }
    };
    if (tid < 2) {
        s_bad[tid] = -1;
        mbar_init(&s_full[tid], BN);
    }
    if (tid == 0) fence_mbar_init();
    if (tid < BM) {
        s_m[tid] = -INFINITY;
        s_l[tid] = 0.0f;
    }
    __syncthreads();
    look_up(t.blk0);
    issue(t.blk0);
    look_up(t.blk0 + 1);

    // ---- this warp's dims of the queries as mma fragments: rows g / g + 8 of
    // m tile mt, dims DW * warp + 16 kk + 2c.. / 2c + 8..
    uint32_t qa[2][KS][TERMS][4];
#pragma unroll
    for (int mt = 0; mt < 2; mt++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = 16 * mt + g + 8 * h, pr = t.r0 + min(r, t.rows - 1), tok = sa_token(a, pr), head = t.kvh * a.G + pr - tok * a.G;
            const size_t at = (size_t)(t.begin + tok) * a.ldq + (size_t)head * D + DW * warp + 2 * c;
#pragma unroll
            for (int kk = 0; kk < KS; kk++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    uint32_t w[TERMS];
                    if constexpr (QF32) {
                        const float2 x = __ldg(reinterpret_cast<const float2 *>(reinterpret_cast<const float *>(a.q) + at +
                                                                                16 * kk + 8 * e));
                        sa_split<TERMS, F16>(x.x, x.y, w);
                    } else {
                        w[0] = __ldg(reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint16_t *>(a.q) + at +
                                                                        16 * kk + 8 * e));
                    }
#pragma unroll
                    for (int x = 0; x < TERMS; x++) qa[mt][kk][x][2 * e + h] = w[x];
                }
        }

    const int arow = (lane & 7) + 8 * ((lane >> 3) & 1), acol = 8 * (lane >> 4);
    const int brow = (lane & 7) + 8 * (lane >> 4), bcol = 8 * ((lane >> 3) & 1);
    const int d0 = DW * warp;
    const bool second = t.rows > 16;                     // rows 16 .. 31 exist
    const int srow = tid / TPR, scol = (tid % TPR) * CPT, stok = sa_token(a, t.r0 + min(srow, t.rows - 1));
    float o[2][ON][4];
#pragma unroll
    for (int mt = 0; mt < 2; mt++)
#pragma unroll
        for (int n = 0; n < ON; n++) o[mt][n][0] = o[mt][n][1] = o[mt][n][2] = o[mt][n][3] = 0.0f;
    auto is_full = [t, t_lo, t_hi, ap = &a0](int blk) {   // no mask crosses the block (missing pages aside)
        if constexpr (TREE) {
            const int e = t.key0 + (blk + 1) * BN;
            return blk < t.nblk_c && e <= t.kend && t.ctx + t.len - (e - BN) <= ap->window;
        } else {
            const int base = t.key0 + blk * BN;
            return base + BN - 1 <= t_lo && t_hi - base < ap->window;
        }
    };

    bool arrives = true;
    for (int blk = t.blk0; blk < t.blk1; blk++) {
        const int st = (blk - t.blk0) & 1;
        if (blk + 1 < t.blk1) {
            issue(blk + 1);                              // into the stage that the block before this one left
            look_up(blk + 2);
        }
        // after a copy that does not arrive nothing is waited for any more
        if (arrives) arrives = sa_poll(&s_full[st], ((blk - t.blk0) >> 1) & 1, a.status, SA_COPY);
        uint16_t *kt = kvs + st * stage_el, *vt = shared_v ? kt : kt + BN * RS;
        const bool full = is_full(blk) && s_bad[st] != blk;
        // ---- partial scores over the warp's dims
#pragma unroll
        for (int n = 0; n < BN / 8; n += 4) {            // eight accumulators at a time cover the product's latency
            float s[2][4][4] = {};
#pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                uint32_t b[2][4];
#pragma unroll
                for (int u = 0; u < 2; u++) sa_ldsm4(b[u], kt + (8 * n + 16 * u + brow) * RS + d0 + 16 * kk + bcol);
#pragma unroll
                for (int x = TERMS - 1; x >= 0; x--)
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        sa_mma<F16>(s[0][u], qa[0][kk][x], b[u / 2][2 * (u & 1)], b[u / 2][2 * (u & 1) + 1]);
                        if (second) sa_mma<F16>(s[1][u], qa[1][kk][x], b[u / 2][2 * (u & 1)], b[u / 2][2 * (u & 1) + 1]);
                    }
            }
            float *dst = part + (warp * BM + g) * SS + 8 * n + 2 * c;
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
                if (mt == 0 || second)
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        *reinterpret_cast<float2 *>(dst + 16 * mt * SS + 8 * u) = make_float2(s[mt][u][0], s[mt][u][1]);
                        *reinterpret_cast<float2 *>(dst + (16 * mt + 8) * SS + 8 * u) = make_float2(s[mt][u][2], s[mt][u][3]);
                    }
        }
        __syncthreads();
        // ---- the row's scores (warp order), softmax
        {
            float x[CPT];
#pragma unroll
            for (int e = 0; e < CPT; e += 4) {
                float4 y = *reinterpret_cast<const float4 *>(part + srow * SS + scol + e);
#pragma unroll
                for (int w = 1; w < NW; w++) {
                    const float4 z = *reinterpret_cast<const float4 *>(part + (w * BM + srow) * SS + scol + e);
                    y.x += z.x;
                    y.y += z.y;
                    y.z += z.z;
                    y.w += z.w;
                }
                x[e] = y.x;
                x[e + 1] = y.y;
                x[e + 2] = y.z;
                x[e + 3] = y.w;
            }
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < CPT; e++) {
                x[e] *= a.scale2;
                if (!full) {
                    bool see;
                    if (TREE && blk < t.nblk_c)
                        see = s_there[st][scol + e] &&
                              t.ctx - (t.key0 + blk * BN + scol + e) + s_depth[stok] < a.window;
                    else
                        see = vis(stok, blk, scol + e);
                    if (!see) x[e] = -INFINITY;
                }
                top = fmaxf(top, x[e]);
            }
#pragma unroll
            for (int d = 1; d < TPR; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            const float old = s_m[srow], m = fmaxf(old, top), use = m == -INFINITY ? 0.0f : m;
            float sum = 0.0f;
            uint32_t w[TERMS][CPT / 2];
#pragma unroll
            for (int e = 0; e < CPT; e += 2) {
                const float y = sa_exp2(x[e] - use), z = sa_exp2(x[e + 1] - use);
                sum += y + z;
                uint32_t p[TERMS];
                sa_split<TERMS, F16>(y, z, p);
#pragma unroll
                for (int i = 0; i < TERMS; i++) w[i][e / 2] = p[i];
            }
#pragma unroll
            for (int i = 0; i < TERMS; i++)
#pragma unroll
                for (int e = 0; e < CPT / 2; e += 2)
                    *reinterpret_cast<uint2 *>(ps + (i * BM + srow) * PS + scol + 2 * e) = make_uint2(w[i][e], w[i][e + 1]);
#pragma unroll
            for (int d = 1; d < TPR; d <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
            if (tid % TPR == 0) {
                const float alpha = sa_exp2(old - use);
                s_alpha[srow] = alpha;
                s_m[srow] = m;
                s_l[srow] = s_l[srow] * alpha + sum;
            }
        }
        __syncthreads();
        // ---- output
        const float al[2][2] = {{s_alpha[g], s_alpha[g + 8]}, {s_alpha[g + 16], s_alpha[g + 24]}};
#pragma unroll
        for (int n0 = 0; n0 < ON; n0 += OG) {
            float acc[2][OG][4] = {};
#pragma unroll
            for (int kk = 0; kk < BN / 16; kk++) {
                uint32_t b[OG / 2][4];
#pragma unroll
                for (int n = 0; n < OG / 2; n++) {
                    sa_ldsm4_t(b[n], vt + (16 * kk + arow) * RS + d0 + 8 * n0 + 16 * n + acol);
                }
#pragma unroll
                for (int x = TERMS - 1; x >= 0; x--) {
                    uint32_t pa[2][4];
#pragma unroll
                    for (int mt = 0; mt < 2; mt++)
                        if (mt == 0 || second) sa_ldsm4(pa[mt], ps + (x * BM + 16 * mt + arow) * PS + 16 * kk + acol);
#pragma unroll
                    for (int n = 0; n < OG; n++) {
                        sa_mma<F16>(acc[0][n], pa[0], b[n / 2][2 * (n & 1)], b[n / 2][2 * (n & 1) + 1]);
                        if (second) sa_mma<F16>(acc[1][n], pa[1], b[n / 2][2 * (n & 1)], b[n / 2][2 * (n & 1) + 1]);
                    }
                }
            }
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int n = 0; n < OG; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[mt][n0 + n][e] = fmaf(o[mt][n0 + n][e], al[mt][e >> 1], acc[mt][n][e]);
        }
        __syncthreads();                                 // this stage, the weights and s_alpha are free
    }
    // no copy is on its way any more when the stages are written over
    for (int blk = max(t.blk0, t.blk1 - 2); !arrives && blk < t.blk1; blk++)
        sa_poll(&s_full[(blk - t.blk0) & 1], ((blk - t.blk0) >> 1) & 1, a.status, SA_COPY);
    bool done = false;
    {
        bool odd = false;
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int n = 0; n < ON; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) odd = odd || (16 * mt + g + 8 * (e >> 1) < t.rows && !isfinite(o[mt][n][e]));
        if (__syncthreads_or(odd) &&
            __syncthreads_or(sa_suspect<D, F16, (TERMS > 1 || F16)>(t, BN, tid, THREADS, is_full, row))) {
            serve_slow_rows<D, F16, QF32>(a, t, BN, warp, NW, vis, row);
            done = true;
        }
    }
    // rows through shared memory (every block is used up), so that whole lines
    // are stored
    constexpr int OS = D + 4;
    float *ob = reinterpret_cast<float *>(sa_sm);        // [BM][OS]
    const bool in_parts = t.parts > 1;
    if (!done) {
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int n = 0; n < ON; n++)
                    *reinterpret_cast<float2 *>(ob + (16 * mt + g + 8 * h) * OS + d0 + 8 * n + 2 * c) =
                        make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
        if (tid < t.rows) {
            const int tok = sa_token(a, t.r0 + tid), head = t.kvh * a.G + t.r0 + tid - tok * a.G;
            s_alpha[tid] = in_parts ? 1.0f : sa_inv(s_l[tid], s_m[tid], a.sink, head);
            if (in_parts) {
                const size_t id = (size_t)t.split * a.nt * a.hq + (size_t)(t.begin + tok) * a.hq + head;
                a.pm[id] = s_m[tid];
                a.pl[id] = s_l[tid];
            }
        }
    }
    __syncthreads();
    for (int x = tid; x < (done ? 0 : t.rows * (D / 8)); x += THREADS) {
        const int r = x / (D / 8), col = (x - r * (D / 8)) * 8, pr = t.r0 + r, tok = sa_token(a, pr),
                  head = t.kvh * a.G + pr - tok * a.G;
        const float f = s_alpha[r];
        float4 y = *reinterpret_cast<const float4 *>(ob + r * OS + col), z = *reinterpret_cast<const float4 *>(ob + r * OS + col + 4);
        y = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
        z = make_float4(z.x * f, z.y * f, z.z * f, z.w * f);
        const size_t at = (size_t)(t.begin + tok) * a.ldo + (size_t)head * D + col;
        if (in_parts || QF32) {
            float *dst = in_parts ? a.po + ((size_t)t.split * a.nt * a.hq + (size_t)(t.begin + tok) * a.hq + head) * D + col
                                  : reinterpret_cast<float *>(a.o) + at;
            *reinterpret_cast<float4 *>(dst) = y;
            *reinterpret_cast<float4 *>(dst + 4) = z;
        } else {
            *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(a.o) + at) =
                make_uint4(sa_pack<F16>(y.x, y.y), sa_pack<F16>(y.z, y.w), sa_pack<F16>(z.x, z.y), sa_pack<F16>(z.z, z.w));
        }
    }
    if (TREE && t.parts > 1) {
        // the tile's last split to finish joins them all
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            int *count = a.counters + ((size_t)blockIdx.z * a.hkv + t.kvh) * a.row_tiles + blockIdx.x % a.row_tiles;
            const bool last = atomicAdd(count, 1) == t.parts - 1;
            if (last) *count = 0;
            s_bad[0] = last;
        }
        __syncthreads();
        if (s_bad[0]) {
            __threadfence();
            sa_join<D, F16, QF32>(a, t, part, tid, THREADS, [] { __syncthreads(); });
        }
    }
}

constexpr int SA_SMEM_MAX = 220 * 1024;      // of 227 KB: the static arrays come on top
// Keys of a block: 64, or 32 where keys and values of 512 dims are apart (two
// stages of both then take the same 128 KB).
static inline int sa_block(int D, bool shared_v) { return D == 512 && !shared_v ? 32 : 64; }

template <int D, int BN, int TERMS, bool F16, bool TREE>
int serve_attn_launch(SaArgs a, cudaStream_t st)
{
    auto kern = serve_attn_kernel<D, BN, TERMS, F16, TREE>;
    constexpr int NW = sa_warps(D);
    static_assert((size_t)SA_BM * (D + 4) * 4 <= (size_t)2 * BN * (D + 8) * 2, "the output rows fit the stages");
    const size_t smem = (size_t)(a.v ? 4 : 2) * BN * (D + 8) * 2 + (size_t)NW * SA_BM * (BN + 8) * 4 +
                        (size_t)TERMS * SA_BM * (BN + 8) * 2;
    static_assert((size_t)(D == 512 && BN == 64 ? 2 : 4) * BN * (D + 8) * 2 + (size_t)NW * SA_BM * (BN + 8) * 4 +
                      (size_t)TERMS * SA_BM * (BN + 8) * 2 <= SA_SMEM_MAX, "shared memory");
    static SmemLimit lim;
    DSV4CU_CUDA_TRY(smem_limit(lim, (const void *)kern, (int)smem));
    dim3 grid;
    if (TREE) {
        grid = dim3(a.row_tiles * a.splits, a.hkv, a.n_req);
    } else {
        const int64_t tiles = (int64_t)a.nt * a.G / SA_BM + min(a.n_req, a.nt);
        if (tiles > INT_MAX) return dsv4cu_set_error(DSV4CU_ERR_ARG, "prompt_attn: %lld row tiles", (long long)tiles);
        grid = sa_prompt_grid(a, tiles, a.sms);
    }
    kern<<<grid, 32 * NW, smem, st>>>(a);
    DSV4CU_LAUNCH_CHECK();
    return DSV4CU_OK;
}

// One translation unit per operand kind.
int serve_attn_bf16(const SaArgs &a, int D, bool tree, cudaStream_t st);
int serve_attn_f16(const SaArgs &a, int D, bool tree, cudaStream_t st);
int serve_attn_f32(const SaArgs &a, int D, bool tree, cudaStream_t st);

template <int TERMS, bool F16, bool TREE>
int serve_attn_pick(const SaArgs &a, int D, cudaStream_t st)
{
    switch (D) {
    case 64: return serve_attn_launch<64, 64, TERMS, F16, TREE>(a, st);
    case 128: return serve_attn_launch<128, 64, TERMS, F16, TREE>(a, st);
    case 256: return serve_attn_launch<256, 64, TERMS, F16, TREE>(a, st);
    default:
        return a.v ? serve_attn_launch<512, 32, TERMS, F16, TREE>(a, st) : serve_attn_launch<512, 64, TERMS, F16, TREE>(a, st);
    }
}

}  // namespace dsv4cu

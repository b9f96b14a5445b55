// paged.cu - the paged cache's bookkeeping on the device: page plans (block
// tables, slot maps and the free-page ring from request lengths) and the
// write of key / value rows into their slots. No counterpart in the
// reference, whose cache is one request's host array.
#include <limits.h>

#include "serve.h"

namespace dsv4cu {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_ITEM_THREADS = 256;
constexpr int PLAN_SOLO_ITEMS = 4096;   // tokens one block handles by itself
constexpr int PLAN_SMEM_REQ = 2047;     // requests whose prefix sums fit the item kernel's shared copy

// Status words of dsv4cu_ctx_status.
enum { PLAN_NO_PAGES = 71, PLAN_TOKENS = 72, PLAN_TABLE = 73 };

struct PlanWs {           // what the scan leaves for the items, per request
    int *held;            // pages held before the call (clamped)
    int *seq;             // tokens before the call (clamped)
    int *first;           // [n_req + 1] pages granted to earlier requests
    int *back;            // [n_req + 1] pages released by earlier requests
    int *cu;              // [n_req + 1] tokens of earlier requests (clamped to INT_MAX)
    int64_t *ring_pos;    // [2] head and tail before the call
};

static size_t plan_ws_layout(int n_req, char *base, PlanWs *w)
{
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char *p = base + off;
        off += dsv4cu_align256(bytes);
        return p;
    };
    w->held = (int *)take((size_t)n_req * 4);
    w->seq = (int *)take((size_t)n_req * 4);
    w->first = (int *)take((size_t)(n_req + 1) * 4);
    w->back = (int *)take((size_t)(n_req + 1) * 4);
    w->cu = (int *)take((size_t)(n_req + 1) * 4);
    w->ring_pos = (int64_t *)take(16);
    return off;
}

DSV4CU_DEV void plan_status(int *status, int code) { atomicCAS(status, 0, code); }

// Inclusive sum of three values over the block's threads; total[] receives the
// block's sums.
DSV4CU_DEV void block_scan3(int64_t (&v)[3], int64_t (&total)[3], int64_t (*sm)[3])
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < 3; i++)
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xFFFFFFFFu, v[i], o);
            if (lane >= o) v[i] += x;
        }
    if (lane == 31)
#pragma unroll
        for (int i = 0; i < 3; i++) sm[warp][i] = v[i];
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int i = 0; i < 3; i++) {
            int64_t x = sm[lane][i];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
                if (lane >= o) x += y;
            }
            sm[lane][i] = x;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; i++) {
        if (warp) v[i] += sm[warp - 1][i];
        total[i] = sm[31][i];
    }
    __syncthreads();
}

// Largest b with a[b] <= x, a[0] = 0 <= x and a non-decreasing over n + 1
// entries; entries that do not grow (requests without items) are passed over.
DSV4CU_DEV int last_at_most(const int *a, int n, int x)
{
    int lo = 0, hi = n;                  // a[lo] <= x, and a[hi] > x or hi == n
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Everything that is not a running sum, one item per thread and independent of
// every other item: token t's position and slot, the i-th granted page's
// table entry, the i-th released page's ring entry. A token's page is read
// from the table where the request held it before the call and from the ring
// where it is granted now, so tokens do not wait for the table's new entries.
DSV4CU_DEV void plan_items(const dsv4cu_page_plan_args &a, const PlanWs &w, const int *cu, const int *first,
                           const int *back, int item0, int nitems)
{
    const int n = a.n_req;
    const int tokens = min(cu[n], a.nt_cap), granted = first[n], released = back[n];
    const int64_t head = w.ring_pos[0], tail = w.ring_pos[1];
    const unsigned np = (unsigned)a.n_pages;
    const unsigned head_m = (unsigned)((uint64_t)head % np), tail_m = (unsigned)((uint64_t)tail % np);
    for (int t = item0; t < a.nt_cap; t += nitems) {
        int req = -1, pos = -1, slot = -1;
        if (t < tokens) {
            req = last_at_most(cu, n, t);
            pos = (int)min((int64_t)w.seq[req] + (t - cu[req]), (int64_t)INT_MAX);
            const int pg = pos / a.page_size, held = w.held[req], grant = first[req + 1] - first[req];
            int entry = -1;
            if (pg < held) entry = a.table[(size_t)req * a.max_pages + pg];
            else if (pg - held < grant)
                entry = a.ring[(unsigned)(((uint64_t)head_m + (unsigned)(first[req] + pg - held)) % np)];
            if (entry >= 0 && entry < a.n_pages) slot = entry * a.page_size + (pos - pg * a.page_size);
        }
        a.slot[t] = slot;
        if (a.pos) a.pos[t] = pos;
        if (a.req) a.req[t] = req;
    }
    for (int i = item0; i < granted; i += nitems) {
        const int r = last_at_most(first, n, i);
        a.table[(size_t)r * a.max_pages + w.held[r] + (i - first[r])] =
            a.ring[(unsigned)(((uint64_t)head_m + (unsigned)i) % np)];
    }
    for (int i = item0; i < released; i += nitems) {
        const int r = last_at_most(back, n, i);
        a.ring[(unsigned)(((uint64_t)tail_m + (unsigned)i) % np)] = a.table[(size_t)r * a.max_pages + (i - back[r])];
    }
}

// The running sums over the requests (tokens, pages granted, pages released),
// one block; with solo set the block does the items as well.
__global__ void __launch_bounds__(PLAN_THREADS) plan_scan_kernel(const dsv4cu_page_plan_args a, const PlanWs w,
                                                                 int solo, int *status)
{
    __shared__ int64_t sm[32][3];
    pdl_trigger();
    const int tid = threadIdx.x;
    const int64_t head = a.ring_pos[0], tail = a.ring_pos[1];
    const int64_t avail = max((int64_t)0, min(tail - head, (int64_t)a.n_pages));
    int64_t carry[3] = {0, 0, 0};
    bool no_pages = false, narrow = false;
    for (int b0 = 0; b0 < a.n_req; b0 += PLAN_THREADS) {
        const int b = b0 + tid;
        int seq = 0, held = 0;
        int64_t v[3] = {0, 0, 0}, total[3];
        if (b < a.n_req) {
            const int nl = a.new_len[b];
            seq = max(0, a.seq_len[b]);
            held = max(0, min(a.held[b], a.max_pages));
            if (nl < 0) {
                v[2] = held;
            } else {
                const int64_t want = ((int64_t)seq + nl + a.page_size - 1) / a.page_size;
                narrow = narrow || want > a.max_pages;
                v[0] = nl;
                v[1] = max((int64_t)0, min(want, (int64_t)a.max_pages) - held);
            }
        }
        const int64_t own1 = v[1], own2 = v[2];
        block_scan3(v, total, sm);
        if (b < a.n_req) {
            const int64_t end = carry[1] + v[1];      // pages wanted up to and including this request
            if (b == 0) w.cu[0] = a.cu[0] = w.first[0] = w.back[0] = 0;
            w.seq[b] = seq;
            w.held[b] = held;
            w.cu[b + 1] = a.cu[b + 1] = (int)min(carry[0] + v[0], (int64_t)INT_MAX);
            w.first[b + 1] = (int)min(end, avail);
            w.back[b + 1] = (int)min(carry[2] + v[2], (int64_t)INT_MAX);
            no_pages = no_pages || (own1 > 0 && end > avail);
            const int64_t grant = min(end, avail) - min(end - own1, avail);
            a.held_out[b] = own2 > 0 || a.new_len[b] < 0 ? 0 : held + (int)grant;
        }
        for (int i = 0; i < 3; i++) carry[i] += total[i];
    }
    if (tid == 0) {
        w.ring_pos[0] = head;
        w.ring_pos[1] = tail;
        a.ring_pos_out[0] = head + min(carry[1], avail);
        a.ring_pos_out[1] = tail + carry[2];
        if (carry[0] > a.nt_cap) plan_status(status, PLAN_TOKENS);
    }
    if (no_pages) plan_status(status, PLAN_NO_PAGES);
    if (narrow) plan_status(status, PLAN_TABLE);
    if (solo) {
        __syncthreads();
        plan_items(a, w, w.cu, w.first, w.back, tid, PLAN_THREADS);
    }
}

__global__ void __launch_bounds__(PLAN_ITEM_THREADS) plan_item_kernel(const dsv4cu_page_plan_args a, const PlanWs w)
{
    __shared__ int sm[3][PLAN_SMEM_REQ + 1];
    pdl_wait();
    const int *cu = w.cu, *first = w.first, *back = w.back;
    if (a.n_req <= PLAN_SMEM_REQ) {
        for (int i = threadIdx.x; i <= a.n_req; i += PLAN_ITEM_THREADS) {
            sm[0][i] = cu[i];
            sm[1][i] = first[i];
            sm[2][i] = back[i];
        }
        __syncthreads();
        cu = sm[0];
        first = sm[1];
        back = sm[2];
    }
    plan_items(a, w, cu, first, back, blockIdx.x * PLAN_ITEM_THREADS + threadIdx.x, gridDim.x * PLAN_ITEM_THREADS);
}

// ---------------------------------------------------------------- writes
// cache[slot[t]] = rows[t], rounded to the cache's type, eight elements per
// thread; blockIdx.y 0 the keys, 1 the values. Bound by memory: every row is
// read once and written once.
struct WriteArgs {
    const void *src[2];
    void *dst[2];
    long ld[2];
    const int *slot;
    int nt, vecs, n_slots;   // vecs: 8-element pieces of a row
};

template <bool SRC32, bool F16>
DSV4CU_DEV uint4 write_load8(const void *src, size_t at)
{
    if constexpr (!SRC32) {
        return *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(src) + at);
    } else {
        const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(src) + at);
        const float4 x = p[0], y = p[1];
        uint4 r;
        if constexpr (F16) {
            const __half2 h[4] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w), __floats2half2_rn(y.x, y.y),
                                  __floats2half2_rn(y.z, y.w)};
            r = *reinterpret_cast<const uint4 *>(h);
        } else {
            const __nv_bfloat162 h[4] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w),
                                         __floats2bfloat162_rn(y.x, y.y), __floats2bfloat162_rn(y.z, y.w)};
            r = *reinterpret_cast<const uint4 *>(h);
        }
        return r;
    }
}

template <bool SRC32, bool F16>
__global__ void __launch_bounds__(256) paged_write_kernel(const WriteArgs a)
{
    const int which = blockIdx.y;
    const int64_t n = (int64_t)a.nt * a.vecs;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int t = (int)(i / a.vecs), c = (int)(i - (int64_t)t * a.vecs);
        const int slot = __ldg(a.slot + t);
        if (slot < 0 || slot >= a.n_slots) continue;
        const uint4 v = write_load8<SRC32, F16>(a.src[which], (size_t)t * a.ld[which] + (size_t)c * 8);
        reinterpret_cast<uint4 *>(a.dst[which])[(size_t)slot * a.vecs + c] = v;
    }
}

}  // namespace dsv4cu

using namespace dsv4cu;

extern "C" size_t dsv4cu_page_plan_workspace(int n_req)
{
    PlanWs w;
    return n_req > 0 ? plan_ws_layout(n_req, nullptr, &w) : 0;
}

extern "C" int dsv4cu_page_plan(dsv4cu_ctx *ctx, const dsv4cu_page_plan_args *a, void *stream)
{
    if (!ctx || !a) return dsv4cu_set_error(DSV4CU_ERR_ARG, "page_plan: NULL argument");
    if (a->n_req < 0 || a->nt_cap < 0) return dsv4cu_set_error(DSV4CU_ERR_ARG, "page_plan: negative count");
    if (a->page_size <= 0 || a->n_pages <= 0 || a->max_pages <= 0)
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "page_plan: page_size %d, n_pages %d, max_pages %d", a->page_size,
                                a->n_pages, a->max_pages);
    if ((int64_t)a->n_pages * a->page_size > INT_MAX)
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "page_plan: %d pages of %d: slots pass 32 bits", a->n_pages,
                                a->page_size);
    if (!a->cu || !a->ring || !a->ring_pos || !a->ring_pos_out ||
        (a->n_req > 0 && (!a->seq_len || !a->new_len || !a->held || !a->held_out || !a->table)) ||
        (a->nt_cap > 0 && !a->slot))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "page_plan: NULL array");
    DeviceGuard guard;
    DSV4CU_CUDA_TRY(guard.enter(ctx->device));
    cudaStream_t st = (cudaStream_t)stream;
    if (a->n_req == 0) {
        // no request: an empty prefix, an unchanged ring, every token row empty
        DSV4CU_CUDA_TRY(cudaMemsetAsync(a->cu, 0, sizeof(int), st));
        if (a->ring_pos_out != a->ring_pos)
            DSV4CU_CUDA_TRY(cudaMemcpyAsync(a->ring_pos_out, a->ring_pos, 16, cudaMemcpyDeviceToDevice, st));
        for (int *p : {a->slot, a->pos, a->req})
            if (p && a->nt_cap) DSV4CU_CUDA_TRY(cudaMemsetAsync(p, 0xFF, (size_t)a->nt_cap * 4, st));
        return DSV4CU_OK;
    }
    void *ws = nullptr;
    int r = dsv4cu_ws_get(ctx, dsv4cu_page_plan_workspace(a->n_req), &ws);
    if (r) return r;
    PlanWs w;
    plan_ws_layout(a->n_req, (char *)ws, &w);
    const bool solo = a->nt_cap <= PLAN_SOLO_ITEMS;
    plan_scan_kernel<<<1, PLAN_THREADS, 0, st>>>(*a, w, solo ? 1 : 0, ctx->status);
    DSV4CU_LAUNCH_CHECK();
    if (!solo) {
        const int blocks = min((a->nt_cap + PLAN_ITEM_THREADS - 1) / PLAN_ITEM_THREADS, ctx->sm_count * 8);
        DSV4CU_CUDA_TRY(launch_pdl(plan_item_kernel, dim3(blocks), dim3(PLAN_ITEM_THREADS), 0, st, *a, w));
    }
    return DSV4CU_OK;
}

extern "C" int dsv4cu_paged_write(dsv4cu_ctx *ctx, void *k_cache, void *v_cache, int cache_type, const void *k,
                                  const void *v, int src_type, long ldk, long ldv, const int *slot, int nt,
                                  int n_slots, int n_kv, int head_dim, void *stream)
{
    if (!ctx) return dsv4cu_set_error(DSV4CU_ERR_ARG, "paged_write: NULL context");
    if (nt < 0 || n_slots <= 0 || n_kv <= 0 || head_dim <= 0)
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "paged_write: nt %d, n_slots %d, n_kv %d, head_dim %d", nt, n_slots,
                                n_kv, head_dim);
    if (!elem_known(cache_type) || cache_type == DSV4CU_F32 || !elem_known(src_type) ||
        (src_type != DSV4CU_F32 && src_type != cache_type))
        return dsv4cu_set_error(DSV4CU_ERR_UNSUPPORTED, "paged_write: rows of type %d into a cache of type %d", src_type,
                                cache_type);
    if (head_dim % 8) return dsv4cu_set_error(DSV4CU_ERR_UNSUPPORTED, "paged_write: head_dim %d not a multiple of 8", head_dim);
    if ((v_cache == nullptr) != (v == nullptr))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "paged_write: values need both v and v_cache");
    if (nt == 0) return DSV4CU_OK;
    if (!k_cache || !k || !slot) return dsv4cu_set_error(DSV4CU_ERR_ARG, "paged_write: NULL array");
    const int64_t row = (int64_t)n_kv * head_dim;
    if (row > INT_MAX) return dsv4cu_set_error(DSV4CU_ERR_ARG, "paged_write: row of %lld elements", (long long)row);
    const int es = elem_bytes(src_type);
    if (!aligned16(k_cache) || !aligned16(k) || ldk < row || ldk * es % 16 ||
        (v && (!aligned16(v_cache) || !aligned16(v) || ldv < row || ldv * es % 16)))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "paged_write: rows must be 16-byte aligned and at least a row apart");
    DeviceGuard guard;
    DSV4CU_CUDA_TRY(guard.enter(ctx->device));
    WriteArgs w = {{k, v}, {k_cache, v_cache}, {ldk, ldv}, slot, nt, (int)(row / 8), n_slots};
    const int64_t n = (int64_t)nt * w.vecs;
    const dim3 grid((unsigned)min((n + 255) / 256, (int64_t)ctx->sm_count * 16), v ? 2 : 1);
    cudaStream_t st = (cudaStream_t)stream;
    if (src_type != DSV4CU_F32) paged_write_kernel<false, false><<<grid, 256, 0, st>>>(w);
    else if (cache_type == DSV4CU_F16) paged_write_kernel<true, true><<<grid, 256, 0, st>>>(w);
    else paged_write_kernel<true, false><<<grid, 256, 0, st>>>(w);
    DSV4CU_LAUNCH_CHECK();
    return DSV4CU_OK;
}

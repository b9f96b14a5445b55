// paged.cu - the paged cache's bookkeeping on the device: page plans (block
// tables, slot maps and the free-page ring from request lengths) and the
// write of key / value rows into their slots. No counterpart in the
// reference, whose cache is one request's host array.
#include <limits.h>

#include "serve.h"

namespace dsv4cu {

constexpr int PLAN_THREADS = 1024;       // of the block that scans alone
constexpr int PLAN_ITEM_THREADS = 256;
constexpr int PLAN_SOLO_ITEMS = 4096;    // tokens one block handles by itself
constexpr int PLAN_FUSED_REQ = 1024;     // requests whose sums every block keeps in shared memory

struct PlanWs {           // what the scan leaves for the items, per request; in the workspace or in shared memory
    int *held;            // pages held before the call (clamped)
    int *seq;             // tokens before the call (clamped)
    int *first;           // [n_req + 1] pages granted to earlier requests
    int *back;            // [n_req + 1] pages released by earlier requests
    int *cu;              // [n_req + 1] tokens of earlier requests (clamped to INT_MAX)
    int *ring_at;         // [2] head and tail before the call, as places of the ring
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
    w->ring_at = (int *)take(8);
    return off;
}

// Inclusive sum of three values over the block's threads; total[] receives the
// block's sums.
template <int WARPS>
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
#pragma unroll
    for (int i = 0; i < 3; i++) {
        int64_t before = 0, all = 0;
        if constexpr (WARPS == 32) {                     // the warps' sums by a lane each
            int64_t x = sm[lane][i];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
                if (lane >= o) x += y;
            }
            all = __shfl_sync(0xFFFFFFFFu, x, 31);
            before = __shfl_sync(0xFFFFFFFFu, x, warp > 0 ? warp - 1 : 0);
            if (warp == 0) before = 0;
        } else {
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                if (w < warp) before += sm[w][i];
                all += sm[w][i];
            }
        }
        v[i] += before;
        total[i] = all;
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

// Everything that is not a running sum, every item independent of the others:
// token t's position and slot, the i-th granted page's
// table entry, the i-th released page's ring entry. A token's page is read
// from the table where the request held it before the call and from the ring
// where it is granted now, so tokens do not wait for the table's new entries.
template <int V>
DSV4CU_DEV void plan_items(const dsv4cu_page_plan_args &a, const PlanWs &w, const int *cu, const int *first,
                           const int *back, int item0, int nitems)
{
    const int n = a.n_req;
    const int tokens = min(cu[n], a.nt_cap), granted = first[n], released = back[n];
    const unsigned np = (unsigned)a.n_pages, head = (unsigned)w.ring_at[0], tail = (unsigned)w.ring_at[1];
    auto popped = [&](int i) {                           // ring place of the i-th granted page, i < n_pages
        const unsigned at = head + (unsigned)i;
        return at >= np ? at - np : at;
    };
    // V tokens in a row per thread: one search, a page's entry once, whole stores
    const bool whole = V == 4 && (((uintptr_t)a.slot | (uintptr_t)a.pos | (uintptr_t)a.req) & 15u) == 0;
    for (int64_t t0 = V * (int64_t)item0; t0 < a.nt_cap; t0 += V * (int64_t)nitems) {
        int req[V], pos[V], slot[V], b = -1, page = -1, entry = -1;
#pragma unroll
        for (int e = 0; e < V; e++) {
            const int t = (int)min(t0 + e, (int64_t)a.nt_cap);
            req[e] = pos[e] = slot[e] = -1;
            if (t >= tokens) continue;
            if (b < 0) b = last_at_most(cu, n, t);
            else if (t >= cu[b + 1]) {
                while (t >= cu[b + 1]) b++;
                page = -1;
            }
            req[e] = b;
            pos[e] = (int)min((int64_t)w.seq[b] + (t - cu[b]), (int64_t)INT_MAX);
            const int pg = pos[e] / a.page_size;
            if (pg != page) {
                const int held = w.held[b], grant = first[b + 1] - first[b];
                page = pg;
                entry = -1;
                if (pg < held) entry = a.table[(size_t)b * a.max_pages + pg];
                else if (pg - held < grant)
                    entry = a.ring[popped(first[b] + pg - held)];
            }
            if (entry >= 0 && entry < a.n_pages) slot[e] = entry * a.page_size + (pos[e] - pg * a.page_size);
        }
        if (whole && t0 + V <= a.nt_cap) {
            auto put = [&](int *dst, const int (&x)[V]) {
                if (dst) *reinterpret_cast<int4 *>(dst + t0) = make_int4(x[0], x[1 % V], x[2 % V], x[3 % V]);
            };
            put(a.slot, slot);
            put(a.pos, pos);
            put(a.req, req);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) {
                if (t0 + e >= a.nt_cap) break;
                a.slot[t0 + e] = slot[e];
                if (a.pos) a.pos[t0 + e] = pos[e];
                if (a.req) a.req[t0 + e] = req[e];
            }
        }
    }
    for (int i = item0; i < granted; i += nitems) {
        const int r = last_at_most(first, n, i);
        a.table[(size_t)r * a.max_pages + w.held[r] + (i - first[r])] =
            a.ring[popped(i)];
    }
    for (int i = item0; i < released; i += nitems) {
        const int r = last_at_most(back, n, i);
        a.ring[((uint64_t)tail + (unsigned)i) % np] = a.table[(size_t)r * a.max_pages + (i - back[r])];
    }
}

// The running sums over the requests (tokens, pages granted, pages released)
// into w; `speak`: this block also writes the call's own outputs.
template <int THREADS>
DSV4CU_DEV void plan_scan(const dsv4cu_page_plan_args &a, const PlanWs &w, bool speak, int *status)
{
    __shared__ int64_t sm[THREADS / 32][3];
    const int tid = threadIdx.x;
    const int64_t head = a.ring_pos[0], tail = a.ring_pos[1];
    const int64_t avail = max((int64_t)0, min(tail - head, (int64_t)a.n_pages));
    int64_t carry[3] = {0, 0, 0};
    bool no_pages = false, narrow = false;
    for (int b0 = 0; b0 < a.n_req; b0 += THREADS) {
        const int b = b0 + tid;
        int seq = 0, held = 0, nl = 0;
        int64_t v[3] = {0, 0, 0}, total[3];
        if (b < a.n_req) {
            nl = a.new_len[b];
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
        const int64_t own = v[1];
        block_scan3<THREADS / 32>(v, total, sm);
        if (b < a.n_req) {
            const int64_t end = carry[1] + v[1];      // pages wanted up to and including this request
            const int cu = (int)min(carry[0] + v[0], (int64_t)INT_MAX);
            if (b == 0) w.cu[0] = w.first[0] = w.back[0] = 0;
            w.seq[b] = seq;
            w.held[b] = held;
            w.cu[b + 1] = cu;
            w.first[b + 1] = (int)min(end, avail);
            w.back[b + 1] = (int)min(carry[2] + v[2], (int64_t)INT_MAX);
            no_pages = no_pages || (own > 0 && end > avail);
            if (speak) {
                if (b == 0) a.cu[0] = 0;
                a.cu[b + 1] = cu;
                a.held_out[b] = nl < 0 ? 0 : held + (int)(min(end, avail) - min(end - own, avail));
            }
        }
        for (int i = 0; i < 3; i++) carry[i] += total[i];
    }
    if (tid < 2) w.ring_at[tid] = (int)((uint64_t)(tid ? tail : head) % (unsigned)a.n_pages);
    if (speak) {
        if (tid == 0) {
            a.ring_pos_out[0] = head + min(carry[1], avail);
            a.ring_pos_out[1] = tail + carry[2];
            if (carry[0] > a.nt_cap) serve_refuse(status, DSV4CU_NO_ROWS);
        }
        if (no_pages) serve_refuse(status, DSV4CU_NO_PAGES);
        if (narrow) serve_refuse(status, DSV4CU_NO_ENTRIES);
    }
}

// One launch: every block sums the requests up for itself in shared memory and
// does its share of the items. The table and ring entries that the items write
// are never ones that they or the sums read, so blocks need no order - unless
// the outputs lie over the inputs, which takes a single block.
__global__ void __launch_bounds__(PLAN_ITEM_THREADS) plan_fused_kernel(const dsv4cu_page_plan_args a, int *status)
{
    __shared__ int sm[5][PLAN_FUSED_REQ + 1];
    __shared__ int at[2];
    const PlanWs w = {sm[0], sm[1], sm[2], sm[3], sm[4], at};
    plan_scan<PLAN_ITEM_THREADS>(a, w, blockIdx.x == 0, status);
    __syncthreads();
    const int item = blockIdx.x * PLAN_ITEM_THREADS + threadIdx.x, items = gridDim.x * PLAN_ITEM_THREADS;
    if (a.nt_cap <= 2 * items) plan_items<1>(a, w, w.cu, w.first, w.back, item, items);
    else plan_items<4>(a, w, w.cu, w.first, w.back, item, items);
}

// Two launches: the sums by one block into the workspace (with solo set it
// does the items as well), then the items.
__global__ void __launch_bounds__(PLAN_THREADS) plan_scan_kernel(const dsv4cu_page_plan_args a, const PlanWs w,
                                                                 int solo, int *status)
{
    pdl_trigger();
    plan_scan<PLAN_THREADS>(a, w, true, status);
    if (solo) {
        __syncthreads();
        plan_items<4>(a, w, w.cu, w.first, w.back, threadIdx.x, PLAN_THREADS);
    }
}

__global__ void __launch_bounds__(PLAN_ITEM_THREADS) plan_item_kernel(const dsv4cu_page_plan_args a, const PlanWs w)
{
    pdl_wait();
    plan_items<4>(a, w, w.cu, w.first, w.back, blockIdx.x * PLAN_ITEM_THREADS + threadIdx.x, gridDim.x * PLAN_ITEM_THREADS);
}

// ---------------------------------------------------------------- writes
// cache[slot[t]] = rows[t], rounded to the cache's type, eight elements per
// thread; blockIdx.y 0 the keys, 1 the values. Bound by memory: every row with a
// slot is read once and written once, a row without one is not read (65111 fp32
// rows of 512 into bf16: 38.6 us, 5.2 TB/s, 0.79 of the measured copy rate; one in
// nine skipped 35.2 us, 5.1 TB/s; 48 rows of 8 x 128: 2.0 us).
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
    // One launch up to 1024 requests: as many blocks as the tokens take, one
    // where the outputs lie over the inputs. 24 requests of 8 tokens: 3.6 us
    // against 4.5 us by one block of 1024 threads (in place, by one block of 256:
    // 5.5 us); 300 prompts of 195,000 tokens: 7.1 us against 7.9 us in two launches
    // (in place: 10.5 us).
    const bool solo = a->nt_cap <= PLAN_SOLO_ITEMS, over = a->held_out == a->held || a->ring_pos_out == a->ring_pos;
    const int blocks = max(1, min((a->nt_cap + PLAN_ITEM_THREADS - 1) / PLAN_ITEM_THREADS, ctx->sm_count * 2));
    if (a->n_req <= PLAN_FUSED_REQ && (solo || !over)) {
        plan_fused_kernel<<<over ? 1 : blocks, PLAN_ITEM_THREADS, 0, st>>>(*a, ctx->status);
        DSV4CU_LAUNCH_CHECK();
        return DSV4CU_OK;
    }
    void *ws = nullptr;
    int r = dsv4cu_ws_get(ctx, dsv4cu_page_plan_workspace(a->n_req), &ws);
    if (r) return r;
    PlanWs w;
    plan_ws_layout(a->n_req, (char *)ws, &w);
    plan_scan_kernel<<<1, PLAN_THREADS, 0, st>>>(*a, w, solo ? 1 : 0, ctx->status);
    DSV4CU_LAUNCH_CHECK();
    if (!solo) DSV4CU_CUDA_TRY(launch_pdl(plan_item_kernel, dim3(blocks), dim3(PLAN_ITEM_THREADS), 0, st, *a, w));
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

// verify.cu - verification of drafted token trees against the target model.
// No counterpart in the reference, which decodes one greedy token at a time.
//
// A request's nodes are its tree in an order where parents come before their
// children; node 0 is the last committed token. A node i > 0 is tested when its
// parent is the current node, and becomes the current node when it is
// accepted, so one pass over the indexes walks the tree.
//
// Sampled: rest = p[cur], mass = 1 at every new current node; node i with
// token x is accepted when u_i * mass * q(x) < rest(x), q = draft[cur], and
// otherwise rest = max(rest - mass q, 0), mass = sum rest. Without draft
// probabilities q(x) = 1 and a refused token leaves: mass -= rest(x),
// rest(x) = 0. Accepting with min(1, rest(x) / (mass q(x))) and continuing
// with the normalised remainder keeps the target's distribution. The next
// token is the first x whose running sum of rest passes u_0 * sum(rest). All
// of it in doubles, products and differences rounded one by one; only the
// order of the sums is the kernel's own, and it is fixed.
//
// One cluster per request, CTA r on the r-th slice of the vocabulary. Every
// CTA walks the tree by itself: the probabilities of every node's token in its
// parent's rows are gathered up front by a thread each, so the walk waits for
// no memory. What needs the whole row is a sum that each CTA takes over its
// slice and stores into the others' shared memory (one cluster barrier per
// sum; two sets of slots, so the next sum does not disturb readers). A row
// comes from memory once; later sums and the rescan of the one segment that
// holds the token find it in L2.
//
// Bound by latency: a request's sums come one after the other (1.6 on average
// over sampled trees of 8, up to 4), each a few batches of loads, a conversion
// of every element to double (16 a clock and SM) and a cluster barrier. 64
// trees over 129280 tokens: 30 us, where the bytes of one row of p and one of
// draft each take 10 us; one chain of 5 over 32000: 8.3 us. Four CTAs of 256
// threads per SM keep all 64 clusters resident; asking for a row's slice in L2
// ahead of its loads changed nothing (31.7 us).
#include <math.h>

#include <cooperative_groups.h>

#include "serve.h"

namespace dsv4cu {
namespace cg = cooperative_groups;

constexpr int VER_MAX_NODES = 128;
constexpr int VER_MAX_VOCAB = 1 << 30; // indexes a step past the row's end stay in 32 bits
constexpr int VER_THREADS = 256;
constexpr int VER_BATCH = 32;         // elements a lane has in flight, of one row or of both
constexpr int VER_WARPS = VER_THREADS / 32;
constexpr int VER_CL = 8;             // CTAs per request: the largest portable cluster

struct VerifyArgs {
    int *accepted, *next, *path, *slot_out;
    const int *tokens, *parent, *cu, *slot, *best;
    const float *p, *draft, *u;
    long ldp, ldd;
    int n_req, nt, vocab;
    int *status;
};

// Request b's node range within [0, nt]; false where it has no node (or more
// than the operator covers).
DSV4CU_DEV bool ver_range(const VerifyArgs &a, int b, int &begin, int &n)
{
    const int lo = __ldg(a.cu + b), hi = __ldg(a.cu + b + 1);
    begin = max(0, min(lo, a.nt));
    n = max(begin, min(hi, a.nt)) - begin;
    return n > 0 && n <= VER_MAX_NODES;
}

DSV4CU_DEV void ver_refuse(const VerifyArgs &a, int b, int begin, int n)
{
    a.accepted[b] = 0;
    a.next[b] = -1;
    for (int i = 0; i < n; i++) {
        a.path[begin + i] = -1;
        if (a.slot_out) a.slot_out[begin + i] = -1;
    }
    if (n > VER_MAX_NODES) serve_refuse(a.status, DSV4CU_VERIFY_NODES);
}

// Writes path and slot_out of one request from the accepted line (line[0] = 0).
DSV4CU_DEV void ver_write(const VerifyArgs &a, int b, int begin, int n, const int *line, int accepted, int tid, int step)
{
    for (int i = tid; i < n; i += step) {
        a.path[begin + i] = i <= accepted ? line[i] : -1;
        if (a.slot_out) {
            int d = -1;
            for (int k = 0; k <= accepted; k++)
                if (line[k] == i) d = k;
            a.slot_out[begin + i] = d < 0 ? -1 : __ldg(a.slot + begin + d);
        }
    }
}

// Greedy: a node is accepted when its token is the target's pick at the
// current node. One warp per request: the warp loads its nodes into shared
// memory, lane 0 walks them there.
__global__ void __launch_bounds__(128) verify_greedy_kernel(const VerifyArgs a)
{
    __shared__ int s_par[4][VER_MAX_NODES], s_tok[4][VER_MAX_NODES], s_best[4][VER_MAX_NODES];
    __shared__ int line[4][VER_MAX_NODES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.x * 4 + warp;
    if (b >= a.n_req) return;
    int begin, n;
    if (!ver_range(a, b, begin, n)) {
        if (lane == 0) ver_refuse(a, b, begin, n);
        return;
    }
    for (int i = lane; i < n; i += 32) {
        s_par[warp][i] = __ldg(a.parent + begin + i);
        s_tok[warp][i] = __ldg(a.tokens + begin + i);
        s_best[warp][i] = __ldg(a.best + begin + i);
    }
    __syncwarp();
    int cur = 0, acc = 0;
    if (lane == 0) {
        line[warp][0] = 0;
        for (int i = 1; i < n; i++)
            if (s_par[warp][i] == cur && s_tok[warp][i] == s_best[warp][cur]) {
                cur = i;
                line[warp][++acc] = i;
            }
        a.accepted[b] = acc;
        a.next[b] = s_best[warp][cur];
    }
    acc = __shfl_sync(0xFFFFFFFFu, acc, 0);
    __syncwarp();
    ver_write(a, b, begin, n, line[warp], acc, lane, 32);
}

DSV4CU_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
DSV4CU_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The remainder of the current row after the refusals so far. With draft
// probabilities the refusals' masses add up: max(max(p - c0 q, 0) - c1 q, 0) =
// max(p - (c0 + c1) q, 0) for q >= 0.
struct Rest {
    const float *p, *q;       // rows of the current node; q NULL without draft probabilities
    double c;                 // sum of the masses refused at (with q)
    const int *gone;          // refused tokens (without q)
    int k;                    // refusals
};

DSV4CU_DEV double ver_less(float pv, float qv, double c)
{
    return fmax(__dsub_rn((double)pv, __dmul_rn(c, (double)qv)), 0.0);
}
DSV4CU_DEV double ver_rest(const Rest &r, float pv, float qv, int x)
{
    if (r.q) return r.k ? ver_less(pv, qv, r.c) : (double)pv;
    for (int i = 0; i < r.k; i++)
        if (r.gone[i] == x) return 0.0;
    return (double)pv;
}

// Sum of the remainder over elements [lo, hi) by one warp; every lane returns
// the sum. LESS: with a draft row to take off.
template <bool LESS>
DSV4CU_DEV double ver_segment(const Rest &r, int lo, int hi, int lane)
{
    constexpr int B = LESS ? VER_BATCH / 2 : VER_BATCH;
    double s[2] = {0.0, 0.0};
    int x0 = lo;
    bool plain = true;                           // no refused token lies in this segment
    if (!LESS)
        for (int i = 0; i < r.k; i++) plain = plain && (r.gone[i] < lo || r.gone[i] >= hi);
    if (plain && (((uintptr_t)(r.p + lo) | (LESS ? (uintptr_t)(r.q + lo) : 0)) & 15u) == 0) {
        const float4 *p = reinterpret_cast<const float4 *>(r.p + lo) + lane;
        const float4 *q = reinterpret_cast<const float4 *>(r.q + lo) + lane;
        for (; x0 + 32 * B <= hi; x0 += 32 * B, p += 8 * B, q += 8 * B) {
            float4 pv[B / 4], qv[B / 4];
#pragma unroll
            for (int j = 0; j < B / 4; j++) {
                pv[j] = __ldg(p + 32 * j);
                if (LESS) qv[j] = __ldg(q + 32 * j);
            }
#pragma unroll
            for (int j = 0; j < B / 4; j++) {
                s[0] += LESS ? ver_less(pv[j].x, qv[j].x, r.c) : (double)pv[j].x;
                s[1] += LESS ? ver_less(pv[j].y, qv[j].y, r.c) : (double)pv[j].y;
                s[0] += LESS ? ver_less(pv[j].z, qv[j].z, r.c) : (double)pv[j].z;
                s[1] += LESS ? ver_less(pv[j].w, qv[j].w, r.c) : (double)pv[j].w;
            }
        }
    } else if (plain) {
        const float *p = r.p + lo + lane, *q = r.q + lo + lane;
        for (; x0 + 32 * B <= hi; x0 += 32 * B, p += 32 * B, q += 32 * B) {
            float pv[B], qv[B];
#pragma unroll
            for (int j = 0; j < B; j++) {
                pv[j] = __ldg(p + 32 * j);
                if (LESS) qv[j] = __ldg(q + 32 * j);
            }
#pragma unroll
            for (int j = 0; j < B; j++) s[j & 1] += LESS ? ver_less(pv[j], qv[j], r.c) : (double)pv[j];
        }
    }
    for (; x0 < hi; x0 += 128) {                 // the rest (or a segment with a refused token), four at a time
        float pv[4], qv[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int x = x0 + 32 * j + lane;
            pv[j] = x < hi ? __ldg(r.p + x) : 0.0f;
            qv[j] = LESS && x < hi ? __ldg(r.q + x) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) s[j & 1] += plain ? (LESS ? ver_less(pv[j], qv[j], r.c) : (double)pv[j])
                                                      : ver_rest(r, pv[j], 0.0f, x0 + 32 * j + lane);
    }
    double t = s[0] + s[1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    return t;
}

__global__ void __cluster_dims__(VER_CL, 1, 1) __launch_bounds__(VER_THREADS, 4) verify_sample_kernel(const VerifyArgs a)
{
    __shared__ double part[VER_WARPS];
    __shared__ double slots[2][VER_CL];
    __shared__ float s_p[VER_MAX_NODES], s_q[VER_MAX_NODES];
    __shared__ int s_par[VER_MAX_NODES], s_tok[VER_MAX_NODES], line[VER_MAX_NODES], gone[VER_MAX_NODES];
    __shared__ float s_u[VER_MAX_NODES];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), b = blockIdx.x / VER_CL;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int begin, n;
    if (!ver_range(a, b, begin, n)) {           // the whole cluster leaves together
        if (rank == 0 && tid == 0) ver_refuse(a, b, begin, n);
        return;
    }
    cluster_arrive();
    for (int i = tid; i < n; i += VER_THREADS) {
        const int par = __ldg(a.parent + begin + i), x = __ldg(a.tokens + begin + i);
        s_u[i] = __ldg(a.u + begin + i);
        s_par[i] = par;
        s_tok[i] = x;
        const bool in = i > 0 && par >= 0 && par < i && x >= 0 && x < a.vocab;
        s_p[i] = in ? __ldg(a.p + (size_t)(begin + par) * a.ldp + x) : 0.0f;
        s_q[i] = in && a.draft ? __ldg(a.draft + (size_t)(begin + par) * a.ldd + x) : 0.0f;
    }
    if (tid == 0) line[0] = 0;
    __syncthreads();
    // no CTA stores into another's shared memory before that one has started:
    // each has said so above, while its loads were on their way
    cluster_wait();
    // this CTA's slice and this warp's segment of it, multiples of 32 elements
    const int per = ((a.vocab + VER_CL - 1) / VER_CL + 31) & ~31;
    const int lo = min(a.vocab, rank * per), hi = min(a.vocab, lo + per);
    const int seg = ((per + VER_WARPS - 1) / VER_WARPS + 31) & ~31;
    const int wlo = min(hi, lo + warp * seg), whi = min(hi, wlo + seg);

    Rest r = {a.p + (size_t)begin * a.ldp, a.draft ? a.draft + (size_t)begin * a.ldd : nullptr, 0.0, gone, 0};
    double mass = 1.0;
    // Sum of the remainder over the row, the same bits in every thread of the
    // cluster: warps in order inside a slice, slices in order.
    int set = 0;
    auto row_sum = [&]() -> double {
        const double s = r.q && r.k ? ver_segment<true>(r, wlo, whi, lane) : ver_segment<false>(r, wlo, whi, lane);
        set ^= 1;
        if (lane == 0) part[warp] = s;
        __syncthreads();
        if (tid < VER_CL) {
            double t = 0.0;
#pragma unroll
            for (int w = 0; w < VER_WARPS; w++) t += part[w];
            *cluster.map_shared_rank(&slots[set][rank], tid) = t;
        }
        cluster.sync();
        double t = 0.0;
#pragma unroll
        for (int c = 0; c < VER_CL; c++) t += slots[set][c];
        return t;
    };
    int cur = 0, acc = 0;
    double total = 0.0;
    bool have_total = false;                     // `total` is the sum of the present remainder
    for (int i = 1; i < n; i++) {                // uniform over the cluster: all threads read the same values
        if (s_par[i] != cur) continue;
        const int x = s_tok[i];
        const bool in = x >= 0 && x < a.vocab;
        const float pv = s_p[i], qv = s_q[i];
        const double left = ver_rest(r, pv, qv, x);
        double bar = __dmul_rn((double)s_u[i], mass);
        if (r.q) bar = __dmul_rn(bar, (double)qv);
        if (in && bar < left) {
            cur = i;
            acc++;
            if (tid == 0) line[acc] = i;
            r.p = a.p + (size_t)(begin + i) * a.ldp;
            if (a.draft) r.q = a.draft + (size_t)(begin + i) * a.ldd;
            r.k = 0;
            r.c = 0.0;
            mass = 1.0;
            have_total = false;
            continue;
        }
        r.c += mass;
        if (!r.q) {
            __syncthreads();                     // the last node's list is read
            if (tid == 0) gone[r.k] = x;
            __syncthreads();
        }
        r.k++;
        if (r.q) {
            mass = total = row_sum();
            have_total = true;
        } else {
            mass = fmax(__dsub_rn(mass, left), 0.0);
            have_total = false;
        }
    }
    if (!have_total) total = row_sum();
    auto draws = [](double t) { return t > 0.0 && t < (double)INFINITY; };   // a sum that a token can be drawn from
    if (!draws(total)) {                         // nothing left, or no number: the target's row itself
        r.k = 0;
        total = row_sum();
    }
    // the slice whose running sum passes the threshold, then the warp, then the element
    const double want = __dmul_rn((double)s_u[0], total);
    const double *sums = slots[set];
    int owner = -1;
    double before = 0.0;
    if (draws(total)) {
        int last = -1;
        double run = 0.0, last_before = 0.0;
        for (int c = 0; c < VER_CL && owner < 0; c++) {
            if (sums[c] > 0.0) {
                last = c;
                last_before = run;
            }
            if (run + sums[c] > want) {
                owner = c;
                before = run;
            }
            run += sums[c];
        }
        if (owner < 0) {                         // u not below 1: the last slice with anything in it
            owner = last;
            before = last_before;
        }
    }
    if (rank == 0) {
        if (tid == 0) {
            a.accepted[b] = acc;
            if (owner < 0) a.next[b] = -1;
        }
        __syncthreads();                         // line is complete
        ver_write(a, b, begin, n, line, acc, tid, VER_THREADS);
    }
    if (owner != rank) return;                   // no remote shared memory is read from here on
    int wsel = -1, wlast = -1;
    double wbefore = 0.0, run = before, lbefore = 0.0;
    for (int w = 0; w < VER_WARPS && wsel < 0; w++) {
        if (part[w] > 0.0) {
            wlast = w;
            lbefore = run;
        }
        if (run + part[w] > want) {
            wsel = w;
            wbefore = run;
        }
        run += part[w];
    }
    if (wsel < 0) {
        wsel = wlast;
        wbefore = lbefore;
    }
    // that warp's segment once more, cut over all warps; the one that holds the
    // threshold looks at its elements in order
    const int slo = min(hi, lo + wsel * seg), shi = min(hi, slo + seg);
    const int sub = ((seg + VER_WARPS - 1) / VER_WARPS + 31) & ~31;
    const int blo = min(shi, slo + warp * sub), bhi = min(shi, blo + sub);
    const double mine = r.q && r.k ? ver_segment<true>(r, blo, bhi, lane) : ver_segment<false>(r, blo, bhi, lane);
    __syncthreads();                             // part is read
    if (lane == 0) part[warp] = mine;
    __syncthreads();
    int sel = -1, last = -1;
    double base = 0.0, lastbase = 0.0;
    run = wbefore;
    for (int w = 0; w < VER_WARPS && sel < 0; w++) {
        if (part[w] > 0.0) {
            last = w;
            lastbase = run;
        }
        if (run + part[w] > want) {
            sel = w;
            base = run;
        }
        run += part[w];
    }
    if (sel < 0) {                               // rounding of the segment's sum: the last piece with mass
        sel = last;
        base = lastbase;
    }
    if (sel < 0) sel = 0;
    if (warp != sel) return;
    int found = -1, lastpos = -1;
    for (int x1 = blo; x1 < bhi && found < 0; x1 += 256) {
        float pw[8], qw[8];                      // eight steps' loads at once
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int x = x1 + 32 * j + lane;
            pw[j] = x < bhi ? __ldg(r.p + x) : 0.0f;
            qw[j] = x < bhi && r.q && r.k ? __ldg(r.q + x) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int x0 = x1 + 32 * j;
            if (x0 >= bhi || found >= 0) break;
            const double v = ver_rest(r, pw[j], qw[j], x0 + lane);
            double c = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xFFFFFFFFu, c, o);
                if (lane >= o) c += y;
            }
            const unsigned pos = __ballot_sync(0xFFFFFFFFu, v > 0.0);
            const unsigned hit = __ballot_sync(0xFFFFFFFFu, v > 0.0 && base + c > want);
            if (hit) found = x0 + __ffs(hit) - 1;
            if (pos) lastpos = x0 + 31 - __clz(pos);
            base += __shfl_sync(0xFFFFFFFFu, c, 31);
        }
    }
    if (found < 0) found = lastpos;              // the piece's last token with mass
    if (lane == 0) a.next[b] = found;
}

}  // namespace dsv4cu

using namespace dsv4cu;

static int verify_check(dsv4cu_ctx *ctx, const char *what, int *accepted, int *next, int *path, const int *tokens,
                        const int *parent, const int *cu, const int *slot, int *slot_out, int n_req, int nt)
{
    if (!ctx) return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: NULL context", what);
    if (n_req < 0 || nt < 0) return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: negative count", what);
    if (n_req == 0) return DSV4CU_OK;
    if (!accepted || !next || !cu || (nt > 0 && (!path || !tokens || !parent)))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: NULL array", what);
    if ((slot == nullptr) != (slot_out == nullptr))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: slot and slot_out go together", what);
    if (slot && slot == slot_out) return dsv4cu_set_error(DSV4CU_ERR_ARG, "%s: slot_out may not alias slot", what);
    return DSV4CU_OK;
}

extern "C" int dsv4cu_verify_greedy(dsv4cu_ctx *ctx, int *accepted, int *next, int *path, const int *tokens,
                                    const int *parent, const int *cu, const int *best, const int *slot,
                                    int *slot_out, int n_req, int nt, void *stream)
{
    int r = verify_check(ctx, "verify_greedy", accepted, next, path, tokens, parent, cu, slot, slot_out, n_req, nt);
    if (r || n_req == 0) return r;
    if (nt > 0 && !best) return dsv4cu_set_error(DSV4CU_ERR_ARG, "verify_greedy: NULL best");
    DeviceGuard guard;
    DSV4CU_CUDA_TRY(guard.enter(ctx->device));
    VerifyArgs a = {accepted, next, path, slot_out, tokens, parent, cu, slot, best, nullptr, nullptr, nullptr, 0, 0,
                    n_req, nt, 0, ctx->status};
    verify_greedy_kernel<<<(n_req + 3) / 4, 128, 0, (cudaStream_t)stream>>>(a);
    DSV4CU_LAUNCH_CHECK();
    return DSV4CU_OK;
}

extern "C" int dsv4cu_verify_sample(dsv4cu_ctx *ctx, int *accepted, int *next, int *path, const int *tokens,
                                    const int *parent, const int *cu, const float *p, long ldp, const float *draft,
                                    long ldd, const float *u, int vocab, const int *slot, int *slot_out, int n_req,
                                    int nt, void *stream)
{
    int r = verify_check(ctx, "verify_sample", accepted, next, path, tokens, parent, cu, slot, slot_out, n_req, nt);
    if (r || n_req == 0) return r;
    if (vocab <= 0 || vocab > VER_MAX_VOCAB || ldp < vocab || (draft && ldd < vocab))
        return dsv4cu_set_error(DSV4CU_ERR_ARG, "verify_sample: vocab %d, row strides %ld and %ld", vocab, ldp, ldd);
    if (n_req > 0x7FFFFFFF / VER_CL) return dsv4cu_set_error(DSV4CU_ERR_ARG, "verify_sample: %d requests", n_req);
    if (nt > 0 && (!p || !u)) return dsv4cu_set_error(DSV4CU_ERR_ARG, "verify_sample: NULL probabilities");
    DeviceGuard guard;
    DSV4CU_CUDA_TRY(guard.enter(ctx->device));
    VerifyArgs a = {accepted, next, path, slot_out, tokens, parent, cu, slot, nullptr, p, draft, u, ldp, ldd,
                    n_req, nt, vocab, ctx->status};
    verify_sample_kernel<<<n_req * VER_CL, VER_THREADS, 0, (cudaStream_t)stream>>>(a);
    DSV4CU_LAUNCH_CHECK();
    return DSV4CU_OK;
}

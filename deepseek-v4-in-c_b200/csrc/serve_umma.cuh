// serve_umma.cuh - softmax attention of packed queries on tcgen05, for head
// dims 64 and 128 in 16 bits: packed prompts, and drafted trees over a paged
// cache whose pages TMA can copy. The mathematics, the packing of grouped
// heads into rows and the masks are those of serve_attn.cuh.
//
// A CTA works on two strips of 128 rows with their scores S (BN fp32 columns)
// and outputs O (D columns) in TMEM; keys come in blocks of BN.
//   warp 0       TMA of key and value blocks, two rings of stages
//   warp 1       TMEM and the single MMA thread: S = Q K^T, then O += P V with
//                P read from TMEM and V as it lies (its rows are the
//                contraction: a transposed operand, nothing is moved)
//   warps 4-7    the first strip's softmax, a thread per row: no shuffles, the
//   warps 8-11   second strip's. A thread reads its row of S, writes it back as
//                16-bit weights over S, and holds the running maximum and sum.
// The two strips take turns: while one is in its softmax the tensor core runs
// the other's products, so neither waits for the other for long.
//
// What a strip is: with more than 128 rows, rows 0-127 and 128-255 over the
// same key blocks (a block is read once for both); with fewer, the same rows
// twice, even blocks and odd blocks, joined at the end - so a single strip
// (decoding) also overlaps its products with its softmax.
//
// The running maximum moves only when a row's new one is more than 8 (in
// log2) above it: weights stay below 2^8, sums and products are exact to the
// same relative rounding, and the outputs in TMEM are seldom rescaled.
//
// Bound by: per block and strip at head dim 128, 1024 clocks of products
// against 1024 of exponentials (16 a clock and SM for 128 x 128 scores), which
// the turns overlap; at head dim 64 the exponentials; for trees of few rows the
// cache's bytes. Measured on one B200:
//   32768 causal tokens, 64 heads over 8, 128 dims: 13.6 ms in a short run
//   (1290 TFLOP/s, 0.77 of the measured bf16 rate), 15.5 to 16.2 ms repeated at
//   the power limit; products and copies alone take 11.8 ms.
//   29 prompts, 16001 tokens, 16 heads over 4, 64 dims: 69 us. (Before tiles
//   started longest first: 92 us, 107 us with one CTA of 128-key blocks per SM.)
//   A strip's block takes 2700 clocks, 2050 of them at the exponential unit's
//   rate for the four strips of an SM; a polynomial for a quarter to a half of
//   the exponentials: 73 to 77 us.
//   32 trees of 8 to 16 nodes over up to 32000 tokens, 64 heads over 8: 511 us
//   (5.7 TB/s, 0.87 of the measured copy rate), 590 us with other work between the
//   calls; with two stages instead of three a fifth more.
#pragma once

#include <cuda.h>

#include "serve_attn.cuh"
#include "tmap.h"
#include "umma.cuh"

namespace dsv4cu {

constexpr int SU_THREADS = 384;
// Keys per block, CTAs per SM and registers a thread (copy and product warps,
// softmax warps). Head dim 128 takes the SM's whole TMEM and its registers for
// 128-key blocks. Head dim 64 has half the products per score, so its softmax
// and the fixed parts of a CTA weigh more: 64-key blocks fit twice, and one
// CTA's set-up and output run beside the other's blocks.
template <int D>
struct SuShape {
    static constexpr int BN = D, CTAS = D == 64 ? 2 : 1, FEW = D == 64 ? 48 : 72, MANY = D == 64 ? 96 : 216;
};
constexpr int SU_SUB = 128 * 128;         // bytes of 128 rows x 64 columns of the queries
constexpr int SU_MAX_STAGES = 4;
constexpr float SU_LAZY = 8.0f;           // log2 units the running maximum may fall behind
enum { SUE_KEMPTY = 81, SUE_VEMPTY, SUE_KFULL, SUE_VFULL, SUE_S, SUE_P, SUE_O, SUE_Q, SUE_DRAIN, SUE_ALIGN };

// Instruction descriptor of kind::f16: fp32 accumulator, both operands of one
// 16-bit type (0 f16, 1 bf16), N >> 3 in bits 17-22, M >> 4 in bits 24-28; bit
// 16 = B with its rows as the contraction.
__host__ __device__ constexpr uint32_t su_idesc(bool f16, int N, bool bt)
{
    return (1u << 4) | ((f16 ? 0u : 1u) << 7) | ((f16 ? 0u : 1u) << 10) | ((bt ? 1u : 0u) << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// The value tile [keys][64 columns] x D / 64 read with keys as the contraction:
// 8-key groups 1024 bytes apart (stride byte offset), 64-column groups `sub`
// bytes apart (leading byte offset).
DSV4CU_DEV uint64_t su_desc_v(const void *p, uint32_t sub)
{
    const uint64_t a = umma::saddr(p);
    return ((a >> 4) & 0x3FFFull) | ((uint64_t)(sub >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
DSV4CU_DEV void su_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// The same with A in TMEM: lane = row, 16-bit pairs per column.
DSV4CU_DEV void su_mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 consecutive columns of this thread's lane.
DSV4CU_DEV void su_ld32(uint32_t taddr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(taddr) : "memory");
}
// 16 columns, arrived.
DSV4CU_DEV void su_ld16(uint32_t taddr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
DSV4CU_DEV void su_st16(uint32_t taddr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
DSV4CU_DEV void su_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Behind su_wait_ld: values of a load that arithmetic may only use from here
// on (nothing else ties the use of a loaded register to the wait).
DSV4CU_DEV void su_loaded32(uint32_t *r)
{
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
DSV4CU_DEV void su_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
DSV4CU_DEV void su_bar(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory"); }
template <int N>
DSV4CU_DEV void su_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(N) : "memory"); }
// The same with an OR over the threads.
template <int N>
DSV4CU_DEV int su_bar_or(int id, int x)
{
    int r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(x), "r"(id), "n"(N) : "memory");
    return r;
}
template <int R>
DSV4CU_DEV void su_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
DSV4CU_DEV void su_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }

// True in one lane of the (converged) warp.
DSV4CU_DEV bool su_elect()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Pairs of floats for the packed fp32 instructions.
DSV4CU_DEV uint64_t su_f2(float x, float y)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
DSV4CU_DEV uint64_t su_u2(uint32_t x, uint32_t y)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
    return r;
}
DSV4CU_DEV void su_unf2(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
DSV4CU_DEV uint64_t su_fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
DSV4CU_DEV uint64_t su_add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Largest of three, NaN if any is.
DSV4CU_DEV float su_max3(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Box of a [row][head][column] map; x = column (a multiple of 64).
DSV4CU_DEV void su_tma(void *dst, const CUtensorMap *map, int x, int head, int row, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(umma::saddr(dst)), "l"(map), "r"(x), "r"(head), "r"(row), "r"(umma::saddr(bar)) : "memory");
}
// Bits lo .. hi of 128 as four words (empty where lo > hi).
DSV4CU_DEV uint32_t su_range(int lo, int hi, int word)
{
    const int l = max(0, lo - 32 * word), h = min(31, hi - 32 * word);
    return l > h ? 0u : (0xFFFFFFFFu << l) & (0xFFFFFFFFu >> (31 - h));
}

// What a CTA shares besides the operand tiles, in front of them. Three stages
// of 128-key blocks and a strip's queries then fill the 227 KB exactly.
struct SuShared {
    uint64_t kfull[SU_MAX_STAGES], kempty[SU_MAX_STAGES], vfull[SU_MAX_STAGES], vempty[SU_MAX_STAGES];
    uint64_t sfull[2], pfull[2], ofull[2], qfull, drain;
    SaTile t;                                            // for what is seldom looked at
    uint32_t anc[SA_MAX_NODES][4];                       // tree: ancestors-or-self
    uint32_t tmem;
    int odd[2];
    int16_t par[SA_MAX_NODES];
    uint8_t depth[SA_MAX_NODES];
};
constexpr int SU_SHARED = 3 * 1024;
static_assert(sizeof(SuShared) <= SU_SHARED, "the tiles start on the swizzle's period");

template <int D, bool F16, bool TREE>
__global__ void __launch_bounds__(SU_THREADS, SuShape<D>::CTAS) serve_umma_kernel(const __grid_constant__ CUtensorMap mk,
                                                                   const __grid_constant__ CUtensorMap mv,
                                                                   const __grid_constant__ CUtensorMap mkc,
                                                                   const __grid_constant__ CUtensorMap mvc,
                                                                   const __grid_constant__ SaArgs a)
{
    constexpr int BN = SuShape<D>::BN, DC = D / 64;      // keys of a block, 64-column tiles of a row
    constexpr int KSUB = BN * 128, QB = DC * SU_SUB, KVB = DC * KSUB;   // bytes: block's tile, strip's queries, block
    constexpr int TM_COLS = 2 * BN + 2 * D;
    extern __shared__ __align__(1024) uint8_t smem[];
    SuShared &sh = *reinterpret_cast<SuShared *>(smem);
    uint8_t *qs = smem + SU_SHARED, *ks = qs + (a.two ? 2 : 1) * QB, *vs = ks + a.nst * KVB;
    uint64_t *kfull = sh.kfull, *kempty = sh.kempty, *vfull = sh.vfull, *vempty = sh.vempty, *sfull = sh.sfull,
             *pfull = sh.pfull, *ofull = sh.ofull;
    uint64_t &qfull = sh.qfull, &drain = sh.drain;
    uint8_t *s_depth = sh.depth;
    uint32_t (*s_anc)[4] = sh.anc;
    int *s_odd = sh.odd;
    if (umma::saddr(smem) & 1023u) {                     // the swizzle's period; never so without static shared memory
        if (threadIdx.x == 0) atomicCAS(a.status, 0, SUE_ALIGN);
        return;
    }
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    const int rows_cta = a.two ? 256 : 128;

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
        if (t.len > a.max_nodes) {
            if (threadIdx.x == 0) serve_refuse(a.status, DSV4CU_TREE_NODES);
            return;
        }
        if (t.split >= sp.used) return;
        t.parts = sp.used;
        t.r0 = (blockIdx.x - t.split * a.row_tiles) * rows_cta;
        t.ctx = sp.ctx;
        t.kend = sp.kend;
        t.table = a.table + (size_t)b * a.max_pages;
        t.key0 = sp.key0;
        t.nblk_c = sp.nblk_c;
        t.blk0 = t.split * sp.per;
        t.blk1 = min(sp.nblk, t.blk0 + sp.per);
    } else {
        int tile;
        sa_find<8>(a, t.begin, t.len, tile);             // prompts always have two strips
        if (t.begin < 0) return;
        t.r0 = tile * rows_cta;
    }
    t.rows = min(rows_cta, t.len * a.G - t.r0);
    if (t.rows <= 0) return;
    const int tok_end = sa_token(a, t.r0 + t.rows - 1);       // the CTA's last token
    const bool alt = t.rows <= 128;                      // one strip: even and odd blocks
    if constexpr (!TREE) {                               // blocks start at the first key of the window
        const int tok = sa_token(a, t.r0);
        t.key0 = a.window > tok ? 0 : tok - a.window + 1;
    }
    // strip s: rows [row0, row0 + n), key blocks from `first` to `end` by `step`
    auto strip_first = [&](int s) {
        if constexpr (TREE) return t.blk0 + (alt ? s : 0);
        const int tok = sa_token(a, t.r0 + (alt ? 0 : 128 * s)), lo = a.window > tok ? 0 : tok - a.window + 1;
        return (lo - t.key0) / BN + (alt ? s : 0);
    };
    auto strip_end = [&](int s) {
        if constexpr (TREE) return t.blk1;
        return ((alt || s ? tok_end : sa_token(a, t.r0 + 127)) - t.key0) / BN + 1;
    };
    const int f0 = strip_first(0), f1 = strip_first(1), e0 = strip_end(0), e1 = strip_end(1), step = alt ? 2 : 1;
    if constexpr (!TREE) {
        t.blk0 = f0;
        t.blk1 = e1;
    }
    const int c0 = f0, c1 = e1;                          // all blocks of the CTA: the second strip ends last

    if (warp == 0) {
        // the copies start as soon as their barriers are set up
        if (lane == 0) {
            sh.t = t;
            for (int s = 0; s < SU_MAX_STAGES; s++) {
                mbar_init(&kfull[s], 1);
                mbar_init(&kempty[s], 1);
                mbar_init(&vfull[s], 1);
                mbar_init(&vempty[s], 1);
            }
            for (int s = 0; s < 2; s++) {
                mbar_init(&sfull[s], 1);
                mbar_init(&pfull[s], 4);
                mbar_init(&ofull[s], 1);
                s_odd[s] = 0;
            }
            mbar_init(&qfull, 8);
            mbar_init(&drain, 1);
            fence_mbar_init();
        }
        __syncwarp();
        su_arrive<SU_THREADS>(4);
        su_regs_dec<SuShape<D>::FEW>();
        // ------------------------------------------------ copies
        const int boxes = TREE ? BN >> a.box_log2 : 1;
        bool ok = true;
        int n = 0;
        for (int b = c0; b < c1 && ok; b++, n++) {
            const int st = n % a.nst, u = n / a.nst;
            const bool cached = TREE && b < t.nblk_c;
            int row = 0;
            bool mine = lane == 0;
            if (cached) {
                const int key = t.key0 + b * BN + (lane << a.box_log2);
                mine = lane < boxes && key < t.kend;
                if (mine) {
                    const int pg = key >> a.page_log2, id = __ldg(t.table + pg);
                    mine = id >= 0 && id < a.n_pages;
                    row = id * a.page_size + (key - (pg << a.page_log2));
                }
            } else {
                row = t.begin + (TREE ? (b - t.nblk_c) * BN : t.key0 + b * BN);
            }
            const unsigned go = __ballot_sync(0xFFFFFFFFu, mine);
            const uint32_t off = cached ? (uint32_t)lane << (a.box_log2 + 7) : 0u;   // this box's first row
            const uint32_t bytes = cached ? (uint32_t)__popc(go) * DC << (a.box_log2 + 7) : (uint32_t)KVB;
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                uint64_t *full = kv ? &vfull[st] : &kfull[st], *empty = kv ? &vempty[st] : &kempty[st];
                if (lane == 0 && u > 0) ok = sa_poll(empty, (u - 1) & 1, a.status, kv ? SUE_VEMPTY : SUE_KEMPTY);
                ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(full, bytes);
                __syncwarp();
                uint8_t *dst = (kv ? vs : ks) + st * KVB + off;
                const CUtensorMap *map = cached ? (kv ? &mvc : &mkc) : (kv ? &mv : &mk);
                if (mine)
#pragma unroll
                    for (int c = 0; c < DC; c++) su_tma(dst + c * KSUB, map, 64 * c, t.kvh, row, full);
            }
        }
        // every issued copy lands before the CTA can exit
        if (lane == 0)
            for (int j = max(0, n - a.nst); j < n; j++) {
                mbar_wait(&kfull[j % a.nst], (j / a.nst) & 1, nullptr, 0);
                mbar_wait(&vfull[j % a.nst], (j / a.nst) & 1, nullptr, 0);
            }
    } else {
        // The softmax warps' queries are on their way while the rest is set up:
        // strip s by its own warps, a single strip by all.
        constexpr int QN = D / 8;                            // 16-byte pieces of a thread
        uint4 qw[QN];
        const int q_s = alt ? 0 : (warp - 4) >> 2, q_n = alt ? 256 : 128, q_i = (threadIdx.x - 128) & (q_n - 1);
        if (warp >= 4) {
            const int n = min(128, t.rows - 128 * q_s);
#pragma unroll
            for (int e = 0; e < QN; e++) {
                const int x = q_i + e * q_n, r = x / (D / 8), ch = x - r * (D / 8);
                qw[e] = make_uint4(0, 0, 0, 0);
                if (r < n) {
                    const int pr = t.r0 + 128 * q_s + r, tok = sa_token(a, pr), head = t.kvh * a.G + pr - tok * a.G;
                    qw[e] = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(a.q) +
                                                                  (size_t)(t.begin + tok) * a.ldq + (size_t)head * D + 8 * ch));
                }
            }
        }
        if (warp == 1) {
            umma::tmem_alloc(&sh.tmem, TM_COLS);
            umma::tmem_relinquish();
        }
        int lost = 0;                                        // a page of these blocks is not in the pool
        if constexpr (TREE) {
            const int k_lo = t.key0 + t.blk0 * BN, k_hi = min(t.kend, t.key0 + min(t.blk1, t.nblk_c) * BN);
            if (k_lo < k_hi)
                for (int pg = (k_lo >> a.page_log2) + threadIdx.x - 32; pg <= (k_hi - 1) >> a.page_log2; pg += SU_THREADS - 32) {
                    const int id = __ldg(t.table + pg);
                    lost |= id < 0 || id >= a.n_pages;
                }
            for (int i = threadIdx.x - 32; i < t.len; i += SU_THREADS - 32) sh.par[i] = (int16_t)max(-1, min(__ldg(a.parent + t.begin + i), SA_MAX_NODES));
        }
        umma::fence_before();
        su_bar<SU_THREADS>(4);                          // the barriers are set up, TMEM is there
        if constexpr (TREE) lost = su_bar_or<SU_THREADS - 32>(5, lost);
        umma::fence_after();
        if constexpr (TREE) {
            for (int i = threadIdx.x - 32; i < t.len; i += SU_THREADS - 32) {
                uint32_t set[4] = {0, 0, 0, 0};
                int d = -1, x = i;
                for (;;) {
#pragma unroll
                    for (int w = 0; w < 4; w++) set[w] |= (x >> 5) == w ? 1u << (x & 31) : 0u;
                    d++;
                    const int p = sh.par[x];
                    if (p < 0 || p >= x) break;
                    x = p;
                }
#pragma unroll
                for (int w = 0; w < 4; w++) s_anc[i][w] = set[w];
                s_depth[i] = (uint8_t)d;
            }
            su_bar<SU_THREADS - 32>(5);
        }
        const uint32_t tmem = sh.tmem;
        const uint32_t tm_s = tmem, tm_o = tmem + 2 * BN;    // strip s: S at + BN s, O at + D s

        if (warp < 4) {
            su_regs_dec<SuShape<D>::FEW>();
            if (warp == 1) {
                // ------------------------------------------------ products
                // The whole warp walks the blocks and one elected lane issues: what
                // the instructions take comes from warp-uniform values (broadcast
                // once), so descriptors stay in uniform registers. Issued by a lone
                // lane, moving them there took longer than the products.
                constexpr uint32_t id_s = su_idesc(F16, BN, false), id_o = su_idesc(F16, D, true);
                auto same = [](int x) { return __shfl_sync(0xFFFFFFFFu, x, 0); };
                const bool one = su_elect();
                const int u0 = same(c0), u1 = same(c1), g0 = same(f0), g1 = same(f1), h0 = same(e0), h1 = same(e1);
                const int nst = a.nst;
                const bool ualt = same(alt) != 0;
                const int ustep = ualt ? 2 : 1;
                const uint32_t ts = (uint32_t)same((int)tm_s), to = (uint32_t)same((int)tm_o);
                // operand descriptors: the address field counts 16 bytes, and shared
                // memory ends before it overflows
                const uint64_t dq = umma::desc_sw128(qs), dk = umma::desc_sw128(ks), dv = su_desc_v(vs, KSUB);
                uint32_t once = 0;                           // blocks that one of their two strips has scored
                bool ok = sa_poll(&qfull, 0, a.status, SUE_Q);
                umma::fence_after();
                // scores of strip s against block b: its key stage and phase
                auto scores = [&](int s, int b) {
                    const int n = b - u0, use = n / nst, st = n - use * nst;
                    ok = ok && sa_poll(&kfull[st], use & 1, a.status, SUE_KFULL);
                    if (!ok) return;
                    umma::fence_after();
                    const uint64_t q = dq + (uint32_t)((ualt ? 0 : s) * (QB >> 4)), k = dk + (uint32_t)(st * (KVB >> 4));
                    const uint32_t bit = 1u << (b & 31);
                    const bool both = !ualt && b >= g1 && b < h0;    // two strips read this block
                    const bool last = !both || (once & bit);
                    once = both && !last ? once | bit : once & ~bit;
                    if (one) {
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++) {
                            su_mma(ts + BN * s, q + (((kk >> 2) * SU_SUB + 32 * (kk & 3)) >> 4),
                                   k + (((kk >> 2) * KSUB + 32 * (kk & 3)) >> 4), id_s, kk > 0);
                        }
                        umma::commit(&sfull[s]);
                        if (last) umma::commit(&kempty[st]);
                    }
                    __syncwarp();
                };
                if (g0 < h0) scores(0, g0);
                if (g1 < h1) scores(1, g1);
                uint32_t turn[2] = {0, 0};
                int st = 0, phase = 0;
                for (int b = u0; b < u1 && ok; b++) {
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        if (ualt ? ((b - u0) & 1) != s : s ? b < g1 : b >= h0) continue;   // strip 0 ends first, strip 1 starts last
                        ok = ok && sa_poll(&pfull[s], turn[s] & 1, a.status, SUE_P) &&
                             sa_poll(&vfull[st], phase, a.status, SUE_VFULL);
                        ok = __all_sync(0xFFFFFFFFu, ok);
                        if (!ok) break;
                        umma::fence_after();
                        const uint64_t v = dv + (uint32_t)(st * (KVB >> 4));
                        const uint32_t more = turn[s] > 0;
                        const bool last = s == 1 || ualt || b < g1;  // strip 1 comes second
                        if (one) {
#pragma unroll
                            for (int kk = 0; kk < BN / 16; kk++)
                                su_mma_ta(to + D * s, ts + BN * s + 8 * kk, v + (2048 >> 4) * kk, id_o, kk > 0 ? 1u : more);
                            if (last) umma::commit(&vempty[st]);
                        }
                        __syncwarp();
                        turn[s]++;
                        if (b + ustep < (s ? h1 : h0)) scores(s, b + ustep);
                        else if (one) umma::commit(&ofull[s]);
                    }
                    if (++st == nst) {
                        st = 0;
                        phase ^= 1;
                    }
                }
                // the products in flight complete before TMEM is released
                if (one) {
                    umma::commit(&drain);
                    mbar_wait(&drain, 0, a.status, SUE_DRAIN);
                }
                __syncwarp();
            }
        } else {
            su_regs_inc<SuShape<D>::MANY>();
            // ------------------------------------------------ softmax
            const int s = (warp - 4) >> 2, i = (threadIdx.x - 128) & 127;    // strip; row, and key in prepared values
            const int row0 = alt ? 0 : 128 * s, rows = min(128, t.rows - row0);
            {
                uint8_t *q = qs + (alt ? 0 : s) * QB;
#pragma unroll
                for (int e = 0; e < QN; e++) {
                    const int x = q_i + e * q_n, r = x / (D / 8), ch = x - r * (D / 8);
                    if (r < 128) *reinterpret_cast<uint4 *>(q + (ch >> 3) * SU_SUB + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = qw[e];
                }
                sa_fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&qfull);
            }
            const int first = s ? f1 : f0, end = s ? e1 : e0;
            const bool live = 32 * (warp & 3) < rows;        // this warp has rows
            const int tok = sa_token(a, t.r0 + row0 + min(i, max(0, rows - 1)));
            const int tok_lo = sa_token(a, t.r0 + row0), tok_hi = sa_token(a, t.r0 + row0 + rows - 1);
            const int depth = TREE ? s_depth[tok] : 0;
            const uint32_t quarter = (uint32_t)(32 * (warp & 3)) << 16;
            const uint32_t sp_s = tm_s + BN * s + quarter, sp_o = tm_o + D * s + quarter;
            float m = -INFINITY, l = 0.0f;
            uint32_t turn = 0;
            bool ok = true;
            // blocks full_lo .. full_hi - 1 are crossed by no mask (missing pages aside)
            int full_lo, full_hi;
            if constexpr (TREE) {
                const int back = t.ctx + t.len - a.window;   // no key below this is in every row's window
                full_lo = back <= t.key0 ? 0 : (back - t.key0 + BN - 1) / BN;
                full_hi = (t.kend - t.key0) / BN;         // at least 0 where there are cached blocks
            } else {
                const int back = tok_hi - a.window + 1 - t.key0;
                full_lo = back <= 0 ? 0 : (back + BN - 1) / BN;
                full_hi = (tok_lo + 1 - t.key0) / BN;
            }
            auto is_full = [full_lo, full_hi](int b) { return b >= full_lo && b < full_hi; };
            const SaTile *tp = &sh.t;
            auto in_pool = [&](int key) {
                if (key >= tp->kend) return false;
                const int id = __ldg(tp->table + (key >> a.page_log2));
                return id >= 0 && id < a.n_pages;
            };
            for (int b = first; b < end; b += step, turn++) {
                // ---- the mask
                const bool masked = !is_full(b) || (TREE && lost);
                constexpr int W = BN / 32;                   // mask words of a block
                uint32_t vis[W];
                ok = __all_sync(0xFFFFFFFFu, sa_poll(&sfull[s], turn & 1, a.status, SUE_S));
                if (!ok) break;
                const bool cached = TREE && b < tp->nblk_c;
                const int base = TREE && !cached ? (b - tp->nblk_c) * BN : tp->key0 + b * BN;
                // keys that are not there: behind the sequence, the nodes or the
                // cache, or on a missing page
                if (masked && (cached ? lost || base + BN > tp->kend : base + BN > tp->len)) {
                    // values of absent keys become zeros (what the copies left, or
                    // brought from the next sequence, may be no number). Behind
                    // this block's scores lie the products of every block before
                    // it, so the stage's last use is over and its barrier is at
                    // most one phase away: the parity below means this block.
                    const int n = b - c0, st = n % a.nst;
                    ok = __all_sync(0xFFFFFFFFu, sa_poll(&vfull[st], (n / a.nst) & 1, a.status, SUE_VFULL));
                    if (!ok) break;
                    if (i < BN && !(cached ? in_pool(base + i) : base + i < tp->len)) {
                        uint8_t *v = vs + st * KVB + i * 128;
#pragma unroll
                        for (int c = 0; c < DC; c++)
#pragma unroll
                            for (int x = 0; x < 8; x++) *reinterpret_cast<uint4 *>(v + c * KSUB + 16 * x) = make_uint4(0, 0, 0, 0);
                    }
                    sa_fence_async();
                }
                if (masked) {
                    if (cached) {
                        const int pos = tp->ctx + depth, lo = a.window > pos ? 0 : pos - a.window + 1 - base;
#pragma unroll
                        for (int w = 0; w < W; w++) {
                            vis[w] = su_range(lo, tp->kend - 1 - base, w);
                            if (lost) vis[w] &= __ballot_sync(0xFFFFFFFFu, in_pool(base + 32 * w + lane));
                        }
                    } else if (TREE) {
#pragma unroll
                        for (int w = 0; w < W; w++) vis[w] = s_anc[tok][base / 32 + w];
                        if (depth >= a.window)
                            for (int x = base; x < min(tp->len, base + BN); x++)
                                if (depth - s_depth[x] >= a.window) {
#pragma unroll
                                    for (int w = 0; w < W; w++) vis[w] &= (x - base) >> 5 == w ? ~(1u << (x & 31)) : ~0u;
                                }
                    } else {
                        const int lo = a.window > tok ? 0 : tok - a.window + 1 - base;
#pragma unroll
                        for (int w = 0; w < W; w++) vis[w] = su_range(lo, tok - base, w);
                    }
                }
                if (live) {
                    umma::fence_after();
                    uint32_t x[BN];
#pragma unroll
                    for (int c = 0; c < BN / 32; c++) su_ld32(sp_s + 32 * c, x + 32 * c);
                    su_wait_ld();
#pragma unroll
                    for (int c = 0; c < BN / 32; c++) su_loaded32(x + 32 * c);
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < BN; k++)
                            if (!((vis[k >> 5] >> (k & 31)) & 1u)) x[k] = 0xFF800000u;
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < BN; k += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            top[e] = su_max3(top[e], __uint_as_float(x[k + 2 * e]), __uint_as_float(x[k + 2 * e + 1]));
                    float mrow = su_max3(su_max3(top[0], top[1], top[2]), top[3], top[3]) * a.scale2;
                    if (mrow == INFINITY) mrow = __uint_as_float(0x7FC00000u);   // inf - inf: the row is NaN, as NaN scores make it
                    const bool move = !(mrow <= m + SU_LAZY);
                    if (__any_sync(0xFFFFFFFFu, move)) {
                        const float to = move ? mrow : m, alpha = move ? sa_exp2(m - to) : 1.0f;
                        m = to;
                        l *= alpha;
                        if (turn > 0) {                      // the products so far are complete: S came behind them
#pragma unroll 2
                            for (int c = 0; c < D; c += 16) {    // few columns at a time: the scores stay in registers
                                uint32_t o[16];
                                su_ld16(sp_o + c, o);
#pragma unroll
                                for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                                su_st16(sp_o + c, o);
                            }
                        }
                    }
                    const float use = m == -INFINITY ? 0.0f : m;
                    const uint64_t scale2 = su_f2(a.scale2, a.scale2), shift2 = su_f2(-use, -use);
                    uint64_t sum[2] = {su_f2(l, 0.0f), su_f2(0.0f, 0.0f)};
#pragma unroll
                    for (int c = 0; c < BN / 32; c++) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            float p, q;
                            su_unf2(su_fma2(su_u2(x[32 * c + 2 * k], x[32 * c + 2 * k + 1]), scale2, shift2), p, q);
                            p = sa_exp2(p);
                            q = sa_exp2(q);
                            sum[k & 1] = su_add2(sum[k & 1], su_f2(p, q));
                            w[k] = sa_pack<F16>(p, q);
                        }
                        su_st16(sp_s + 16 * c, w);
                    }
                    float s0, s1;
                    su_unf2(su_add2(sum[0], sum[1]), s0, s1);
                    l = s0 + s1;
                    su_wait_st();
                    umma::fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[s]);
            }
            // ---- outputs
            // At head dim 128 a prompt's loop needs every register: its tile is
            // read back (32768 causal tokens 16.1 -> 15.8 ms); elsewhere holding
            // it is faster (64 dims 69 us, read back 71 us).
            const SaTile &u = D == 128 && !TREE ? sh.t : t;
            const bool any = first < end;
            if (any) ok = ok && __all_sync(0xFFFFFFFFu, sa_poll(&ofull[s], 0, a.status, SUE_O));
            umma::fence_after();
            const SaArgs &a0 = a;
            auto row_of = [tp, ap = &a0](int blk, int j, bool values) -> const uint16_t * {
                const SaArgs &a = *ap;
                const SaTile &t = *tp;
                const bool vv = values && a.v != nullptr;
                if (TREE && blk < t.nblk_c) {
                    const int key = t.key0 + blk * BN + j;
                    return key < t.kend ? sa_cached(a, t, vv ? a.vc : a.kc, key, D) : nullptr;
                }
                const int key = TREE ? (blk - t.nblk_c) * BN + j : t.key0 + blk * BN + j;
                if (key >= t.len) return nullptr;
                return reinterpret_cast<const uint16_t *>(vv ? a.v : a.k) + (size_t)(t.begin + key) * (vv ? a.ldv : a.ldk) +
                       (size_t)t.kvh * D;
            };
            auto sees = [tp, row_of, ap = &a0, dp = s_depth, an = s_anc](int tok, int blk, int j) -> bool {
                const SaArgs &a = *ap;
                const SaTile &t = *tp;
                if constexpr (TREE) {
                    if (blk < t.nblk_c) {
                        const int key = t.key0 + blk * BN + j;
                        return key < t.kend && t.ctx - key + dp[tok] < a.window && row_of(blk, j, false) != nullptr;
                    }
                    const int x = (blk - t.nblk_c) * BN + j;
                    return x < t.len && (an[tok][x >> 5] >> (x & 31) & 1) && dp[tok] - dp[x] < a.window;
                } else {
                    const int key = t.key0 + blk * BN + j;
                    return key <= tok && tok - key < a.window;
                }
            };
            // A warp's rows go out through its own part of the shared memory that
            // the products are done with, so that stores cover whole rows. With two
            // strips that is the strip's queries; a single strip first adds its
            // even and odd blocks: each half of the columns is finished by one
            // strip's warps, which get the other strip's share of it through xch.
            constexpr int PN = D == 128 ? 16 : 8;            // 16-byte pieces of a row per pass
            constexpr int XN = D / 8;                        // 16-byte pieces of half a row of floats
            constexpr int XH = 128 * XN * 16;                // bytes of one strip's share
            static_assert(2 * XH + 8 * PN * 512 <= 2 * 2 * KVB || 2 * XH + 8 * PN * 512 <= 2 * SU_MAX_STAGES * KVB, "stages");
            uint8_t *out = alt ? ks + 2 * XH + (warp - 4) * (PN * 512) : qs + s * QB + (warp & 3) * (PN * 512);
            float f_own = 1.0f;
            const int col0 = alt ? s * (D / 2) : 0, ncol = alt ? D / 2 : D;
            if (alt) {
                float2 *ml = reinterpret_cast<float2 *>(ks + 2 * XH);
                su_bar<256>(1);                              // both strips' products are complete: the stages are free
                ml[128 * s + i] = make_float2(m, l);
                su_bar<256>(1);
                const float2 other = ml[128 * (s ^ 1) + i];
                const float top = m != m || other.x != other.x ? m + other.x : fmaxf(m, other.x);
                const float use = top == -INFINITY ? 0.0f : top;
                f_own = sa_exp2(m - use);
                l = l * f_own + other.y * sa_exp2(other.x - use);
                m = top;
                if (live) {
                    uint8_t *x = ks + (s ^ 1) * XH + i * (XN * 16);
                    for (int c = 0; c < D / 2; c += 16) {
                        uint32_t o[16];
                        if (any) su_ld16(sp_o + (s ^ 1) * (D / 2) + c, o);
#pragma unroll
                        for (int k = 0; k < 16; k += 4) {
                            float y[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) y[e] = any ? __uint_as_float(o[k + e]) * f_own : 0.0f;
                            *reinterpret_cast<float4 *>(x + ((((c + k) >> 2) ^ (i & 7)) << 4)) = make_float4(y[0], y[1], y[2], y[3]);
                        }
                    }
                }
                su_bar<256>(1);
            }
            bool odd = false;
            if (live) {
                const int head = u.kvh * a.G + u.r0 + row0 + min(i, max(0, rows - 1)) - tok * a.G;
                const bool part = TREE && u.parts > 1;
                const float inv = part ? 1.0f : sa_inv(l, m, a.sink, head);
                const size_t row_id = (size_t)(u.begin + tok) * a.hq + head;
                const size_t id = (size_t)u.split * a.nt * a.hq + row_id;
                if (part && i < rows && (!alt || s == 0)) {
                    a.pm[id] = m;
                    a.pl[id] = l;
                }
                char *dst = part ? reinterpret_cast<char *>(a.po + id * D + col0)
                                 : reinterpret_cast<char *>(reinterpret_cast<uint16_t *>(a.o) + (size_t)(u.begin + tok) * a.ldo +
                                                            (size_t)head * D + col0);
                const uint8_t *x = ks + s * XH + i * (XN * 16);
                const int mine = min(32, rows - 32 * (warp & 3));    // rows of this warp
                int piece = 0;                               // of the pass
                for (int c = 0; c < ncol; c += 16) {         // a loop: its code is cold at every launch
                    uint32_t o[16];
                    if (any) su_ld16(sp_o + col0 + c, o);
                    float y[16];
#pragma unroll
                    for (int k = 0; k < 16; k++) y[k] = any ? __uint_as_float(o[k]) * f_own : 0.0f;
                    if (alt)
#pragma unroll
                        for (int k = 0; k < 16; k += 4) {
                            const float4 z = *reinterpret_cast<const float4 *>(x + ((((c + k) >> 2) ^ (i & 7)) << 4));
                            y[k] += z.x;
                            y[k + 1] += z.y;
                            y[k + 2] += z.z;
                            y[k + 3] += z.w;
                        }
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        odd = odd || !isfinite(y[k]);
                        y[k] *= inv;
                    }
                    uint8_t *w = out + lane * (PN * 16);
                    if (part) {
#pragma unroll
                        for (int k = 0; k < 16; k += 4)
                            *reinterpret_cast<float4 *>(w + (((piece + k / 4) ^ (lane & 7)) << 4)) =
                                make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]);
                        piece += 4;
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; k += 8)
                            *reinterpret_cast<uint4 *>(w + (((piece + k / 8) ^ (lane & 7)) << 4)) =
                                make_uint4(sa_pack<F16>(y[k], y[k + 1]), sa_pack<F16>(y[k + 2], y[k + 3]),
                                           sa_pack<F16>(y[k + 4], y[k + 5]), sa_pack<F16>(y[k + 6], y[k + 7]));
                        piece += 2;
                    }
                    if (piece == PN || c + 16 >= ncol) {     // the pass is full: 2^b pieces per row
                        const int b = 31 - __clz(piece);
                        __syncwarp();
#pragma unroll 4
                        for (int e = 0; e < (mine << b); e += 32) {
                            const int r = (e + lane) >> b, pc = (e + lane) & (piece - 1);
                            char *d = reinterpret_cast<char *>(__shfl_sync(0xFFFFFFFFu, (unsigned long long)dst, r & 31));
                            if (r < mine)
                                *reinterpret_cast<uint4 *>(d + 16 * pc) =
                                    *reinterpret_cast<const uint4 *>(out + r * (PN * 16) + ((pc ^ (r & 7)) << 4));
                        }
                        __syncwarp();
                        dst += 16 * piece;
                        piece = 0;
                    }
                }
                odd = odd && i < rows;
            }
            // a row that is not finite: was it a value behind the mask?
            const int who = alt ? 0 : s;
            if (odd) s_odd[who] = 1;
            alt ? su_bar<256>(1) : su_bar<128>(2 + s);
            if (s_odd[who]) {
                SaTile ts = u;
                ts.r0 = u.r0 + row0;
                ts.rows = rows;
                if (!alt) {
                    ts.blk0 = first;
                    ts.blk1 = end;
                }
                const int threads = alt ? 256 : 128, thread = alt ? threadIdx.x - 128 : i;
                if (sa_suspect<D, F16, F16>(ts, BN, thread, threads, is_full, row_of)) s_odd[who] = 2;
                alt ? su_bar<256>(1) : su_bar<128>(2 + s);
                if (s_odd[who] == 2) serve_slow_rows<D, F16, false>(a, ts, BN, thread >> 5, threads >> 5, sees, row_of);
            }
            if (TREE && u.parts > 1) {
                // the tile's last split to finish joins them all
                __threadfence();
                su_bar<256>(1);
                if (threadIdx.x == 128) {
                    int *count = a.counters + ((size_t)blockIdx.z * a.hkv + u.kvh) * a.row_tiles + blockIdx.x % a.row_tiles;
                    const bool last = atomicAdd(count, 1) == u.parts - 1;
                    if (last) *count = 0;
                    s_odd[0] = last;
                }
                su_bar<256>(1);
                if (s_odd[0]) {
                    __threadfence();
                    sa_join<D, F16, false>(a, u, reinterpret_cast<float *>(ks), threadIdx.x - 128, 256, [] { su_bar<256>(1); });
                }
            }
        }
    }
    umma::fence_before();
    __syncthreads();
    if (warp == 1) {
        umma::fence_after();
        umma::tmem_dealloc(sh.tmem, TM_COLS);
    }
}

// Map of a [rows][heads][D] 16-bit tensor, boxes of 64 columns x 1 head x box_rows rows.
static inline int su_map(CUtensorMap *map, const void *base, int D, int heads, int64_t rows, long ld, int box_rows,
                         bool f16)
{
    return tmap_encode_rows(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, D, heads,
                            rows, (uint64_t)D * 2, (uint64_t)ld * 2, 64, box_rows);
}

template <int D, bool F16>
int serve_umma_launch(SaArgs a, bool tree, cudaStream_t st)
{
    using S = SuShape<D>;
    constexpr int QB = D / 64 * SU_SUB, KVB = D / 64 * S::BN * 128;
    int r;
    CUtensorMap mk, mv, mkc, mvc;
    if ((r = su_map(&mk, a.k, D, a.hkv, a.nt, a.ldk, S::BN, F16))) return r;
    if ((r = su_map(&mv, a.v ? a.v : a.k, D, a.hkv, a.nt, a.v ? a.ldv : a.ldk, S::BN, F16))) return r;
    mkc = mk;
    mvc = mv;
    dim3 grid;
    if (tree) {
        const int bn_log2 = S::BN == 64 ? 6 : 7;
        a.box_log2 = a.page_log2 < bn_log2 ? a.page_log2 : bn_log2;
        if (a.n_pages > 0) {
            const int64_t slots = (int64_t)a.n_pages * a.page_size;
            const long row = (long)a.hkv * D;
            if ((r = su_map(&mkc, a.kc, D, a.hkv, slots, row, 1 << a.box_log2, F16))) return r;
            if ((r = su_map(&mvc, a.vc ? a.vc : a.kc, D, a.hkv, slots, row, 1 << a.box_log2, F16))) return r;
        }
        grid = dim3(a.row_tiles * a.splits, a.hkv, a.n_req);
    } else {
        a.two = 1;
        const int64_t tiles = (int64_t)a.nt * a.G / 256 + min(a.n_req, a.nt);
        if (tiles > INT_MAX) return dsv4cu_set_error(DSV4CU_ERR_ARG, "prompt_attn: %lld row tiles", (long long)tiles);
        grid = sa_prompt_grid(a, tiles, a.sms * S::CTAS);
    }
    // as many stages as fit: 227 KB for one CTA; half of the SM's 228 KB less
    // the 1 KB that each CTA costs for two
    constexpr int LIMIT = S::CTAS == 2 ? 113 * 1024 : 227 * 1024;
    const int fixed = (a.two ? 2 : 1) * QB + SU_SHARED;
    a.nst = min(SU_MAX_STAGES, (LIMIT - fixed) / (2 * KVB));
    const size_t smem = fixed + (size_t)2 * a.nst * KVB;
    auto kern = tree ? serve_umma_kernel<D, F16, true> : serve_umma_kernel<D, F16, false>;
    static SmemLimit lim[2];
    DSV4CU_CUDA_TRY(smem_limit(lim[tree], (const void *)kern, (int)smem));
    // the warps' register shares are taken from what the block is launched with
    static int regs[2];
    if (!regs[tree]) {
        cudaFuncAttributes f;
        DSV4CU_CUDA_TRY(cudaFuncGetAttributes(&f, (const void *)kern));
        regs[tree] = f.numRegs;
    }
    if (regs[tree] * SU_THREADS < S::FEW * 128 + S::MANY * 256)
        return dsv4cu_set_error(DSV4CU_ERR_UNSUPPORTED, "serving attention: launched with %d registers a thread", regs[tree]);
    kern<<<grid, SU_THREADS, smem, st>>>(mk, mv, mkc, mvc, a);
    DSV4CU_LAUNCH_CHECK();
    return DSV4CU_OK;
}

int serve_umma_bf16(const SaArgs &a, int D, bool tree, cudaStream_t st);
int serve_umma_f16(const SaArgs &a, int D, bool tree, cudaStream_t st);

}  // namespace dsv4cu

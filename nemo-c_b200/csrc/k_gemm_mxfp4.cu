// GEMM of MXFP4 rows: C[m][n] (=, +=) alpha * act(sum_k A[m][k] W[n][k] + bias[n]), both operands
// as 4-bit codes with a power-of-two scale per 32 columns. tcgen05.mma (kind::mxf4, block-scaled)
// multiplies the codes as they are: every product of two codes and two scales is exact, the sums
// are fp32 in tensor memory, and nothing is rounded before the epilogue.
//
// Orientation: weight rows are the MMA's 128-row side (tensor-memory lanes), activation rows its
// columns, so that one kernel serves one row and thousands: a warp's 32 lanes hold 32 neighbouring
// output columns of an output row, and each store of the epilogue is one contiguous run.
//
// A unit of work is one weight tile of 128 rows (GLU: two, value rows n and gate rows n + N/2) by one
// tile of BN activation rows. One stage holds 256 columns of k: the weight and activation codes, brought
// in by TMA with the 128-byte swizzle, and their scale tiles, one bulk copy each. The MMA thread copies the
// scales from shared to tensor memory (tcgen05.cp; each stage has tensor-memory columns of its own,
// so a later stage's copy never meets an MMA that still reads them) and issues four MMAs of 64 columns per
// weight tile.
//
// Few units: a cluster of 2, 4 or 8 CTAs splits k; the partial tiles meet in shared memory across
// the cluster and are added in the order of their ranks, so results do not depend on scheduling.
// Otherwise persistent CTAs walk the units, the epilogue of one running beside the MMAs of the
// next. Warp roles: warp 0 loads, warp 1 owns tensor memory and issues the MMAs, the others run
// the epilogue. Every wait on a barrier is bounded: on a timeout the CTA records an
// error, takes part in the remaining cluster barriers and unwinds.
//
// Measured (tensor products alone): 14322 x 1024 x 4096 to fp32 38.8 to 41.7 us (2.9 PFLOP/s or more, 1.8 times the
// measured bf16 rate), accumulating 67 us; 8192 cubed 248 us (4.4 PFLOP/s); 1792 x 4096 x 1024 to bf16 with SiLU 12.2 us,
// with GLU 10.1 us; one row by 1024 x 4096 5.0 us. What held it back, in the order found: the issuing thread (descriptors computed for each
// MMA in divergent code: 82 us for the first shape; constant words and an unrolled stage 59 us; uniform control
// flow, so that operands come from uniform registers, 50 us; the same for the loading warp 40 us); then, where k is
// short, the epilogue: accumulators released as soon as they are in registers, two groups of epilogue
// warps in turn (14322 x 4096 x 1024 with SiLU: 83 us, 62 us). What is left there is the special-function
// units' two operations per output (32 % busy at 1792 rows) behind 3.03 units per SM in 4 turns.
#include <cuda.h>
#include <cstring>
#include <type_traits>
#include <atomic>
#include "cluster.cuh"
#include "elt.cuh"
#include "mxfp4.cuh"
#include "sm100.cuh"

extern "C" int *nb_tc_error_ptr(void);

namespace {

constexpr int BM = 128;   // weight rows per tile
constexpr int BKB = 128;  // code bytes per row and stage: 256 columns of k, one swizzle span
constexpr int ATOM = 512; // bytes of one scale tile (128 rows x 128 columns of k)
constexpr int ERR = 11;   // codes of waits that gave up: a free stage, a free accumulator, a stage's data, a unit's products

struct MxArgs {
    const uint8_t *as, *ws;  // scales
    const float *bias;
    void *C;
    int64_t ldc;
    int M, N, K, kblocks, katoms, splits, kb_per_split, n_wtiles, n_mtiles, units, act, accumulate, vec;
    float alpha;
    int *err;
};

template <int BN, int WT>
struct Cfg {
    // Epilogue groups of 8 warps, which take units in turn: two where units are large and many, so that one
    // group's activations run beside the other's loads and stores (the registers of GLU allow one)
    static constexpr int GROUPS = BN == 128 && WT == 1 ? 2 : 1, THREADS = 64 + 256 * GROUPS;
    // k split over a cluster: not with tiles of 128 rows, which are only taken where tiles of 64 would outnumber the SMs
    static constexpr bool SPLIT = BN < 128;
    static constexpr int W_BYTES = BM * BKB, A_BYTES = BN * BKB;
    static constexpr int WS_OFF = WT * W_BYTES + A_BYTES;      // scales: 2 atoms per weight tile, 2 for the activations
    static constexpr int STAGE = WS_OFF + (WT + 1) * 2 * ATOM;
    static constexpr int STAGES = WT == 2 ? 4 : BN == 128 ? 5 : BN == 64 ? 7 : 8;
    static constexpr int SLOTS = WT == 1 ? 2 : BN == 128 ? 3 : 4;  // accumulators of BN columns
    static constexpr int SC_COLS = (WT + 1) * 8;                 // scale columns per stage
    static constexpr int COLS = SLOTS * BN + STAGES * SC_COLS;
    static constexpr int TMEM_COLS = COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    // 16-bit outputs pass through shared memory: per epilogue warp 32 rows of 32 columns, 80 bytes apart
    static constexpr int OUT = BN >= 64 ? GROUPS * 8 * 32 * 80 : 0;
    static constexpr int SMEM = 1024 + STAGES * STAGE + OUT + 256;
    static_assert(SMEM <= 232448, "shared memory");
    static_assert(COLS <= 512, "tensor memory");
    static_assert(STAGE % 1024 == 0, "swizzled tiles start on 1 KB");
    static_assert(!SPLIT || WT * BN * BM * 4 <= STAGES * STAGE, "partial tiles reuse the stages");
};

__device__ __forceinline__ void bulk_g2s(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(bytes),
                 "r"(sm100::smem_u32(bar))
                 : "memory");
}

// Shared-memory descriptors, low word: address / 16 (and a leading offset of 16 bytes, unused, for the
// operands); the high words are constants, so one thread can issue an MMA every few instructions.
// Operand tiles: K-major, 128-byte swizzle, groups of 8 rows 1024 bytes apart; 32 bytes of k further on
// is an address 32 bytes on. Scale tiles: 32 rows of 16 bytes, contiguous, no swizzle (core matrices of
// 8 rows x 16 bytes are 128 bytes apart).
constexpr uint32_t OPERAND_HI = (1024 >> 4) | 1u << 14 | 2u << 29, SCALE_HI = (128 >> 4) | 1u << 14;
__device__ __forceinline__ uint64_t desc64(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ uint64_t desc_operand(uint32_t smem_addr) { return desc64(smem_addr >> 4 | 1u << 16, OPERAND_HI); }
__device__ __forceinline__ uint64_t desc_scale(uint32_t smem_addr) { return desc64(smem_addr >> 4, SCALE_HI); }
// 32 lanes x 16 bytes, written to all four 32-lane quarters of tensor memory.
__device__ __forceinline__ void cp_scale(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Instruction descriptor, kind::mxf4: e2m1 x e2m1 with ue8m0 scales, both operands K-major. An
// MMA takes two scales per row out of a word of four: half 0 or half 1 of it.
__host__ __device__ constexpr uint32_t idesc_mxf4(int N, int half) {
    return ((uint32_t)(half * 2) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(BM >> 7) << 27) |
           ((uint32_t)(half * 2) << 29);
}
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    // (accumulate: constant but for the first MMA of a unit)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}

// 32 lanes x 16 consecutive columns; the values are there after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
          "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
}
// Waits for this warp's loads; naming the loaded values keeps their uses behind the wait.
template <int CN>
__device__ __forceinline__ void tmem_wait_ld(float (&v)[CN]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < CN; ++j) asm volatile("" : "+f"(v[j]));
}

// 16 lanes x 32 columns in the layout of a matrix fragment: v[4 k + 2 h + e] is lane 8 h + t / 4, column
// 8 k + 2 (t % 4) + e.
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
          "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
}
// Four 8 x 8 matrices of 16-bit elements, transposed: thread t names row t % 8 of matrix t / 8.
__device__ __forceinline__ void store_frag_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *(const uint32_t *)&h;
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *(const uint32_t *)&h;
    }
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sm100::smem_u32(bar)) : "memory");
}
// bias -> act -> alpha -> store or accumulate, one output element.
template <typename T>
__device__ __forceinline__ void finish(const MxArgs &p, int m, int n, float va, float vb, float ba, float bb) {
    float v = va + ba;
    if (p.act == NEMO_ACT_GLU)
        v *= nb::sigmoid_fast(vb + bb);
    else if (p.act == NEMO_ACT_SILU)
        v *= nb::sigmoid_fast(v);
    else if (p.act == NEMO_ACT_RELU)
        v = v < 0.0f ? 0.0f : v;  // a NaN stays one
    v *= p.alpha;
    T *c = (T *)p.C + (int64_t)m * p.ldc + n;
    if (p.accumulate) v += nb::to_f32(*c);
    *c = nb::from_f32<T>(v);
}
// Two rows of one output column; g: GLU's gates.
template <int ACT>
__device__ __forceinline__ void activate(float &v0, float &v1, float g0, float g1, float ba, float bb, float alpha) {
    nb::f2 x = nb::add2(nb::pack2(v0, v1), nb::dup2(ba));
    if (ACT == NEMO_ACT_SILU) x = nb::mul2(x, nb::sigmoid2(x));
    if (ACT == NEMO_ACT_GLU) x = nb::mul2(x, nb::sigmoid2(nb::add2(nb::pack2(g0, g1), nb::dup2(bb))));
    if (ACT == NEMO_ACT_RELU) {
        float a, b;
        nb::unpack2(x, a, b);
        x = nb::pack2(a < 0.0f ? 0.0f : a, b < 0.0f ? 0.0f : b);
    }
    nb::unpack2(nb::mul2(x, nb::dup2(alpha)), v0, v1);
}
// CN rows of one output column.
template <int ACT, int CN>
__device__ __forceinline__ void activate_rows(float (&v)[CN], const float (&g)[CN], float ba, float bb, float alpha) {
#pragma unroll
    for (int j = 0; j < CN; j += 2) activate<ACT>(v[j], v[j + 1], g[j], g[j + 1], ba, bb, alpha);
}
// A fragment (tmem_ld_frag): ba, bb hold the biases of its two lanes.
template <int ACT>
__device__ __forceinline__ void activate_frag(float (&v)[16], const float (&g)[16], const float *ba, const float *bb, float alpha) {
#pragma unroll
    for (int k = 0; k < 8; ++k) activate<ACT>(v[2 * k], v[2 * k + 1], g[2 * k], g[2 * k + 1], ba[k & 1], bb[k & 1], alpha);
}
#define MX_ACT_SWITCH(act, CALL)                     \
    switch (act) {                                   \
        case NEMO_ACT_SILU: CALL(NEMO_ACT_SILU); break; \
        case NEMO_ACT_RELU: CALL(NEMO_ACT_RELU); break; \
        case NEMO_ACT_GLU: CALL(NEMO_ACT_GLU); break;   \
        default: CALL(NEMO_ACT_NONE); break;          \
    }
template <typename T, int CN>
__device__ __forceinline__ void finish_rows(const MxArgs &p, int m, int n, int count, float (&v)[CN], const float (&g)[CN], float ba, float bb) {
#define CALL(A) activate_rows<A, CN>(v, g, ba, bb, p.alpha)
    MX_ACT_SWITCH(p.act, CALL)
#undef CALL
    T *c = (T *)p.C + (int64_t)m * p.ldc + n;
    if (p.accumulate) {
#pragma unroll
        for (int j = 0; j < CN; ++j)
            if (j < count) v[j] += nb::to_f32(c[j * p.ldc]);
    }
    if (count >= CN) {
#pragma unroll
        for (int j = 0; j < CN; ++j, c += p.ldc) *c = nb::from_f32<T>(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < CN; ++j, c += p.ldc)
            if (j < count) *c = nb::from_f32<T>(v[j]);
    }
}

template <typename T, int BN, int WT>
__global__ void __launch_bounds__(Cfg<BN, WT>::THREADS, 1)
    gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, const __grid_constant__ MxArgs p) {
    using C = Cfg<BN, WT>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *stages = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *outs = stages + C::STAGES * C::STAGE;
    uint64_t *full = (uint64_t *)(outs + C::OUT);
    uint64_t *empty = full + C::STAGES;
    uint64_t *acc_full = empty + C::STAGES;     // [SLOTS] MMA -> epilogue
    uint64_t *acc_empty = acc_full + C::SLOTS;  // [SLOTS] epilogue -> MMA
    uint32_t *tmem_holder = (uint32_t *)(acc_empty + C::SLOTS);
    volatile int *flags = (volatile int *)(tmem_holder + 1);  // [0] a wait gave up, [1 + group] an epilogue group's own

    // the same in every lane, and known to be: what the issuing warp computes then stays in uniform registers,
    // which is where the tensor instructions take their operands from
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { sm100::mbar_init(&full[s], 1); sm100::mbar_init(&empty[s], 1); }
        for (int s = 0; s < C::SLOTS; ++s) { sm100::mbar_init(&acc_full[s], 1); sm100::mbar_init(&acc_empty[s], 1); }
        flags[0] = flags[1] = flags[2] = 0;
        sm100::fence_mbar_init();
        sm100::tma_prefetch_desc(&tmW);
        sm100::tma_prefetch_desc(&tmA);
    }
    if (warp == 1) {
        sm100::tmem_alloc(tmem_holder, C::TMEM_COLS);
        sm100::tmem_relinquish();
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_holder, 0);
    nb::pdl_wait();

    constexpr bool glu = WT == 2;
    const bool split = C::SPLIT && p.splits > 1;
    const int rank = split ? (int)nb::cluster_rank() : 0;
    const int u0 = split ? blockIdx.x / p.splits : blockIdx.x, ustep = split ? p.units : gridDim.x;
    const int kb0 = rank * p.kb_per_split, kb1 = min(p.kblocks, kb0 + p.kb_per_split);
    // first weight row of tile i of unit u
    auto wrow = [&](int wt, int i) { return wt * BM + (i ? p.N / 2 : 0); };

    if (warp == 0) {
        const bool leader = elect_one();
        int it = 0;
        for (int u = u0; u < p.units; u += ustep) {
            const int mt = u % p.n_mtiles, wt = u / p.n_mtiles;
            const int r0 = wrow(wt, 0), r1 = wrow(wt, 1);
            const uint8_t *ws0 = p.ws + (int64_t)(r0 / BM) * p.katoms * ATOM, *ws1 = p.ws + (int64_t)(r1 / BM) * p.katoms * ATOM;
            const uint8_t *as = p.as + (int64_t)(mt * BN / 128) * p.katoms * ATOM;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % C::STAGES;
                ok = __all_sync(0xffffffffu, !flags[0] && (it < C::STAGES || sm100::mbar_wait(&empty[s], ((it / C::STAGES) - 1) & 1)));
                if (!ok) break;
                if (leader) {
                    uint8_t *st = stages + s * C::STAGE;
                    const uint32_t sb = (uint32_t)min(2, p.katoms - kb * 2) * ATOM;  // scale tiles of these columns
                    const int64_t at = (int64_t)kb * (2 * ATOM);  // 2 GB of scales a row of tiles at K = 2^29
                    sm100::mbar_arrive_expect_tx(&full[s], WT * (C::W_BYTES + sb) + C::A_BYTES + sb);
                    sm100::tma_load_2d(st, &tmW, &full[s], kb * BKB, r0);
                    bulk_g2s(st + C::WS_OFF, ws0 + at, sb, &full[s]);
                    if (glu) {
                        sm100::tma_load_2d(st + C::W_BYTES, &tmW, &full[s], kb * BKB, r1);
                        bulk_g2s(st + C::WS_OFF + 2 * ATOM, ws1 + at, sb, &full[s]);
                    }
                    sm100::tma_load_2d(st + WT * C::W_BYTES, &tmA, &full[s], kb * BKB, mt * BN);
                    bulk_g2s(st + C::WS_OFF + WT * 2 * ATOM, as + at, sb, &full[s]);
                }
                __syncwarp();
            }
            if (!ok) {
                if (!flags[0]) { flags[0] = 1; atomicExch(p.err, ERR + 0); }
                break;
            }
        }
        // a launch that gave up waits for its own copies before its shared memory goes away
        if (__any_sync(0xffffffffu, flags[0]))
            for (int j = max(0, it - C::STAGES); j < it; ++j) sm100::mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, 100000000LL);
    } else if (warp == 1) {
        const bool leader = elect_one();
        int it = 0, t = 0;
        for (int u = u0; u < p.units; u += ustep, ++t) {
            if (__any_sync(0xffffffffu, flags[0])) break;
            bool ok = true;
#pragma unroll
            for (int i = 0; i < WT; ++i) {
                const int q = t * WT + i;
                if (q >= C::SLOTS && !sm100::mbar_wait(&acc_empty[q % C::SLOTS], ((q / C::SLOTS) - 1) & 1)) ok = false;
            }
            if (!__all_sync(0xffffffffu, ok)) { flags[0] = 1; atomicExch(p.err, ERR + 1); break; }
            sm100::tc_fence_after();
            // activation tiles of 64 rows: the second one of a scale tile (128 rows) finds its scales two columns on
            const int sb_at = WT * 8 + (BN == 64 ? u % p.n_mtiles % 2 * 2 : 0);
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % C::STAGES;
                if (!__all_sync(0xffffffffu, sm100::mbar_wait(&full[s], (it / C::STAGES) & 1))) { flags[0] = 1; atomicExch(p.err, ERR + 2); break; }
                sm100::tc_fence_after();
                const uint32_t st = sm100::smem_u32(stages + s * C::STAGE);
                const uint32_t sc = tmem + C::SLOTS * BN + s * C::SC_COLS;
                auto stage = [&](int atoms, int steps) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i <= WT; ++i) {  // weight tiles, then the activations
#pragma unroll
                        for (int a = 0; a < 2; ++a)
                            if (a < atoms) cp_scale(sc + i * 8 + a * 4, desc_scale(st + C::WS_OFF + (i * 2 + a) * ATOM));
                    }
#pragma unroll
                    for (int i = 0; i < WT; ++i) {
                        const uint32_t d = tmem + ((t * WT + i) % C::SLOTS) * BN;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            if (kk < steps)
                                mma_mxf4(d, desc_operand(st + i * C::W_BYTES + kk * 32), desc_operand(st + WT * C::W_BYTES + kk * 32), idesc_mxf4(BN, kk & 1),
                                         sc + i * 8 + (kk >> 1) * 4, sc + sb_at + (kk >> 1) * 4, kb != kb0 || kk != 0);
                    }
                };
                const int left = p.K - kb * 256;
                if (leader) {
                    if (left >= 256) stage(2, 4);
                    else stage(left > 128 ? 2 : 1, min(4, (left + 63) / 64));
                    sm100::mma_commit(&empty[s]);
                }
                __syncwarp();
            }
            if (leader)
#pragma unroll
                for (int i = 0; i < WT; ++i) sm100::mma_commit(&acc_full[(t * WT + i) % C::SLOTS]);
            __syncwarp();
        }
    } else if (warp >= 2) {
        const int group = (warp - 2) >> 3, q = warp & 3, half = ((warp - 2) >> 2) & 1;  // the 32 lanes and the half of the columns of this warp
        const int row = q * 32 + lane, etid = (threadIdx.x - 64) & 255;
        constexpr int HALF = BN >= 32 ? BN / 2 : BN;
        const int jbeg = half * HALF, jend = jbeg < BN ? jbeg + HALF : jbeg;
        const int nout = glu ? p.N / 2 : p.N;
        int t = group;
        for (int u = u0 + group * ustep; u < p.units; u += C::GROUPS * ustep, t += C::GROUPS) {
            const int mt = u % p.n_mtiles, wt = u / p.n_mtiles, m0 = mt * BN, mcount = min(BN, p.M - m0);
            // biases first: they arrive while the unit's products are formed. One per lane, or (FRAG) those of
            // the fragments' lanes 8 h + lane / 4.
            const bool frag = C::OUT && sizeof(T) == 2 && p.vec;
            float ba[WT][4], bb[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
#pragma unroll
                for (int i = 0; i < WT; ++i) {
                    const int n = wrow(wt, i) + q * 32 + (frag ? h * 8 + lane / 4 : lane);
                    ba[i][h] = p.bias && n < p.N && (frag || h == 0) ? p.bias[n] : 0.0f;
                }
                bb[h] = glu ? ba[WT - 1][h] : 0.0f;  // of the gates
            }
            bool good = true;
#pragma unroll
            for (int i = 0; i < WT; ++i)
                if (!sm100::mbar_wait(&acc_full[(t * WT + i) % C::SLOTS], ((t * WT + i) / C::SLOTS) & 1)) good = false;
            if (!good) { flags[1 + group] = 1; flags[0] = 1; atomicExch(p.err, ERR + 3); }
            // the group's flag is written only by its threads before this barrier: all of them decide alike
            sm100::named_barrier(1 + group, 256);
            if (flags[1 + group]) break;
            sm100::tc_fence_after();
            const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
            if (split) {  // partial tiles to shared memory: [tile][column][lane]
                float *part = (float *)stages;
#pragma unroll
                for (int i = 0; i < WT; ++i)
                    for (int j0 = jbeg; j0 < jend && j0 < mcount; j0 += 16) {
                        float v[16];
                        sm100::tmem_ld16(lanes + ((t * WT + i) % C::SLOTS) * BN + j0, v);
#pragma unroll
                        for (int jj = 0; jj < 16; ++jj) part[(i * BN + j0 + jj) * BM + row] = v[jj];
                    }
            } else {
                // The warp's whole share to registers at once; then the accumulator (GLU: and its gates') is free for the
                // MMAs of a later unit, before anything is computed or stored.
                constexpr int CH = HALF / 16;
                float v[CH][16], g[CH][16];
                const uint32_t acc = lanes + (t * WT % C::SLOTS) * BN + jbeg, gate = lanes + ((t * WT + 1) % C::SLOTS) * BN + jbeg;
                const bool mine = jbeg < BN;
                if (mine) {
#pragma unroll
                    for (int k = 0; k < CH; ++k) {
                        // fragments: columns 32 (k / 2), lanes 16 (k & 1); rows: columns 16 k
                        if (frag) tmem_ld_frag(acc + (k >> 1) * 32 + ((k & 1) << 20), v[k]);
                        else tmem_ld(acc + k * 16, v[k]);
                        if (glu) {
                            if (frag) tmem_ld_frag(gate + (k >> 1) * 32 + ((k & 1) << 20), g[k]);
                            else tmem_ld(gate + k * 16, g[k]);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < CH; ++k) {
                        tmem_wait_ld(v[k]);
                        if (glu) tmem_wait_ld(g[k]);
                    }
                }
                sm100::tc_fence_before();
                sm100::named_barrier(1 + group, 256);
                if (etid < WT) mbar_arrive(&acc_empty[(t * WT + etid) % C::SLOTS]);
                if (!mine) continue;
                const int n1 = wt * BM;
                if (frag) {
                    // transposed through shared memory into runs of eight columns: one 16-byte store where
                    // single elements take eight
                    uint8_t *buf = outs + (warp - 2) * 32 * 80;
                    const int nq = n1 + q * 32;
                    // where this thread's matrix row goes (matrix = lane / 8: columns 8 (m & 1), rows 8 (m / 2))
                    const uint32_t to = sm100::smem_u32(buf) + (8 * (lane >> 4) + (lane & 7)) * 80 + ((lane >> 3) & 1) * 16;
#pragma unroll
                    for (int c0 = 0; c0 < CH; c0 += 2) {
                        if (jbeg + c0 * 16 >= mcount) break;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float(&vv)[16] = v[c0 + h];
#define CALL(A) activate_frag<A>(vv, g[c0 + h], &ba[0][2 * h], &bb[2 * h], p.alpha)
                            MX_ACT_SWITCH(p.act, CALL)
#undef CALL
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                store_frag_t(to + k * 16 * 80 + h * 32, pack16<T>(vv[8 * k], vv[8 * k + 1]), pack16<T>(vv[8 * k + 2], vv[8 * k + 3]),
                                             pack16<T>(vv[8 * k + 4], vv[8 * k + 5]), pack16<T>(vv[8 * k + 6], vv[8 * k + 7]));
                        }
                        __syncwarp();
                        const int n = nq + (lane & 3) * 8, j0 = jbeg + c0 * 16;
                        T *c = (T *)p.C + (int64_t)(m0 + j0 + lane / 4) * p.ldc + n;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint4 o = *(const uint4 *)(buf + (k * 8 + lane / 4) * 80 + (lane & 3) * 16);
                            if (n < nout && j0 + k * 8 + lane / 4 < mcount) *(uint4 *)(c + k * 8 * p.ldc) = o;
                        }
                        __syncwarp();
                    }
                } else if (n1 + row < nout) {
#pragma unroll
                    for (int k = 0; k < CH; ++k)
                        if (jbeg + k * 16 < mcount) finish_rows<T, 16>(p, m0 + jbeg + k * 16, n1 + row, mcount - jbeg - k * 16, v[k], g[k], ba[0][0], bb[0]);
                }
            }
        }
    }
    __syncwarp();
    if (split) {
        // one unit per cluster: each rank adds and finishes its share of the columns
        __syncthreads();
        nb::cluster_sync();
        const int mt = u0 % p.n_mtiles, wt = u0 / p.n_mtiles, m0 = mt * BN, mcount = min(BN, p.M - m0);
        // a warp takes a column at a time, four neighbouring lanes of the tile per thread, the ranks' partials in order
        const int nout = glu ? p.N / 2 : p.N, per = (mcount + p.splits - 1) / p.splits;
        const int j1 = min(mcount, (rank + 1) * per), n = wt * BM + lane * 4;
        float base[4], bgate[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            base[k] = p.bias && n + k < nout ? p.bias[n + k] : 0.0f;
            bgate[k] = glu && p.bias && n + k < nout ? p.bias[n + k + p.N / 2] : 0.0f;
        }
        const uint32_t part = sm100::smem_u32(stages) + lane * 16;
        if (!flags[0] && n < nout)
            for (int j = rank * per + warp; j < j1; j += C::THREADS / 32) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f), g = v;
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < p.splits) {
                        const float4 a = nb::ld_cluster4(part + j * BM * 4, r);
                        v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
                        if (glu) {
                            const float4 b = nb::ld_cluster4(part + (BN + j) * BM * 4, r);
                            g.x += b.x; g.y += b.y; g.z += b.z; g.w += b.w;
                        }
                    }
                const float vv[4] = { v.x, v.y, v.z, v.w }, gg[4] = { g.x, g.y, g.z, g.w };
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n + k < nout) finish<T>(p, m0 + j, n + k, vv[k], gg[k], base[k], bgate[k]);
            }
        nb::cluster_sync();  // no CTA leaves while another reads its shared memory
    }
    sm100::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        sm100::tc_fence_after();
        sm100::tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static std::atomic<EncodeTiled> fn{nullptr};
    EncodeTiled f = fn.load();
    if (!f) {
        void *q = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) != cudaSuccess || !q) return nullptr;
        fn.store(f = (EncodeTiled)q);
    }
    return f;
}

// Codes as bytes: [rows][K / 2], boxes of 128 bytes by box_rows; columns past K / 2 read as zero.
int code_map(CUtensorMap *m, const uint8_t *base, int64_t K, int64_t rows, int64_t ld, int box_rows) {
    EncodeTiled f = encoder();
    if (!f) return nb_set_error("nemo_gemm_mxfp4: cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[2] = { (cuuint64_t)(K / 2), (cuuint64_t)rows };
    cuuint64_t strides[1] = { (cuuint64_t)ld };
    cuuint32_t box[2] = { (cuuint32_t)BKB, (cuuint32_t)box_rows };
    cuuint32_t es[2] = { 1, 1 };
    CUresult r = f(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return nb_set_error("nemo_gemm_mxfp4: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return 0;
}

template <typename T, int BN, int WT>
int run(const nemo_gemm_mxfp4_args_t *a, cudaStream_t st) {
    using C = Cfg<BN, WT>;
    constexpr bool glu = WT == 2;
    CUtensorMap mw, ma;
    if (code_map(&mw, a->W, a->K, a->N, a->ldw, BM) || code_map(&ma, a->A, a->K, a->M, a->lda, BN)) return -1;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return nb_set_error("nemo_gemm_mxfp4: no CUDA device");
    MxArgs p;
    memset(&p, 0, sizeof p);
    p.as = a->a_scales; p.ws = a->w_scales; p.bias = a->bias; p.C = a->C; p.ldc = a->ldc;
    p.M = a->M; p.N = a->N; p.K = a->K; p.act = a->act; p.accumulate = a->accumulate; p.alpha = a->alpha;
    p.vec = sizeof(T) == 2 && ((uintptr_t)a->C & 15) == 0 && a->ldc % 8 == 0 && (glu ? a->N / 2 : a->N) % 8 == 0;
    p.kblocks = (a->K + 255) / 256;
    p.katoms = (a->K + 127) / 128;
    p.n_wtiles = ((glu ? a->N / 2 : a->N) + BM - 1) / BM;
    p.n_mtiles = (a->M + BN - 1) / BN;
    const int64_t units = (int64_t)p.n_wtiles * p.n_mtiles;
    if (units > 0x3fffffff) return nb_set_error("nemo_gemm_mxfp4: too many tiles");
    p.units = (int)units;
    // k is split over a cluster while the CTAs fit the SMs and the k-blocks saved (0.16 us each) pay for
    // joining the partial tiles (about 1 us + 7 ns per column and rank). M = 1, N = 1024, K = 4096: 5.9 us whole, 5.0 us
    // in the 4 parts that this takes, 4.6 us in 8; M = 1, N = 256, K = 8192: 8.9 us whole, 4.7 us in 8. Against: M = 7,
    // N = 2048, K = 1024 3.5 us whole, 4.5 us in 2 or 4; M = 256, N = 1024, K = 4096 6.5 us whole, 7.7 and 6.9 us.
    int splits = 1;
    float best = 0.16f * p.kblocks;
    for (int s = 2; C::SPLIT && s <= 8 && p.units * s <= sms && s <= p.kblocks; s *= 2) {
        const int per = (p.kblocks + s - 1) / s;
        const float cost = 0.16f * per + 1.0f + 0.007f * BN * s;
        if (cost < best && (s - 1) * per < p.kblocks) {  // every rank has k-blocks
            best = cost;
            splits = s;
        }
    }
    p.kb_per_split = (p.kblocks + splits - 1) / splits;
    p.splits = splits;
    p.err = nb_tc_error_ptr();
    if (!p.err) return nb_set_error("nemo_gemm_mxfp4: device error word unavailable");
    auto kernel = gemm_mxfp4_kernel<T, BN, WT>;
    if (nb_smem_attr((const void *)kernel, C::SMEM)) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits > 1 ? p.units * splits : p.units < sms ? p.units : sms);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (nb_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = splits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaLaunchKernelEx(&cfg, kernel, mw, ma, p);
    return nb_check_launch("gemm_mxfp4_kernel");
}

template <typename T>
int by_rows(const nemo_gemm_mxfp4_args_t *a, cudaStream_t st) {
    const bool glu = a->act == NEMO_ACT_GLU;
    if (a->M <= 16) return glu ? run<T, 16, 2>(a, st) : run<T, 16, 1>(a, st);
    // 64 rows a tile where all tiles then still run at once, on more SMs with less to finish for each (256 x 4096 x
    // 1024: 6.4 us with 128 rows, 5.0 us with 64; 1792 x 1024 x 4096, two turns with 64: 9.3 and 11.3 us)
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return nb_set_error("nemo_gemm_mxfp4: no CUDA device");
    const int64_t tiles = (int64_t)(((glu ? a->N / 2 : a->N) + BM - 1) / BM) * ((a->M + 63) / 64);
    if (a->M <= 64 || tiles <= sms) return glu ? run<T, 64, 2>(a, st) : run<T, 64, 1>(a, st);
    return glu ? run<T, 128, 2>(a, st) : run<T, 128, 1>(a, st);
}

}  // namespace

extern "C" int nemo_gemm_mxfp4(const nemo_gemm_mxfp4_args_t *a, void *stream) {
    if (!a) return nb_set_error("nemo_gemm_mxfp4: null arguments");
    if (a->M < 0 || a->M > (1 << 30) || a->N < 0 || a->N > (1 << 30) || a->K < 0 || a->K > (1 << 30)) return nb_set_error("nemo_gemm_mxfp4: bad shape M=%d N=%d K=%d", a->M, a->N, a->K);
    if (a->act < NEMO_ACT_NONE || a->act > NEMO_ACT_GLU) return nb_set_error("nemo_gemm_mxfp4: unknown activation %d", a->act);
    if (!nb::elt_ok(a->c_elt)) return nb_set_error("nemo_gemm_mxfp4: unknown element type %d", a->c_elt);
    if (a->K == 0 || a->K % 32) return nb_set_error("nemo_gemm_mxfp4: K=%d must be a positive multiple of 32", a->K);
    if (a->act == NEMO_ACT_GLU && a->N % 256) return nb_set_error("nemo_gemm_mxfp4: GLU needs N=%d to be a multiple of 256 (whole scale tiles in each half)", a->N);
    if (a->accumulate && a->c_elt != NEMO_ELT_F32) return nb_set_error("nemo_gemm_mxfp4: accumulate needs an fp32 output");
    if (a->M == 0 || a->N == 0) return 0;
    if (!a->A || !a->a_scales || !a->W || !a->w_scales || !a->C) return nb_set_error("nemo_gemm_mxfp4: null pointer");
    if (((uintptr_t)a->A | (uintptr_t)a->W | (uintptr_t)a->a_scales | (uintptr_t)a->w_scales) & 15 || a->lda % 16 || a->ldw % 16)
        return nb_set_error("nemo_gemm_mxfp4: codes, scales and code row pitches must be 16-byte aligned");
    if (a->lda < a->K / 2 || a->ldw < a->K / 2) return nb_set_error("nemo_gemm_mxfp4: code row pitches below K / 2 bytes");
    if (a->M > 1 && a->ldc < (a->act == NEMO_ACT_GLU ? a->N / 2 : a->N)) return nb_set_error("nemo_gemm_mxfp4: ldc below the output columns");
    if ((uintptr_t)a->C % nb::elt_size(a->c_elt) || (uintptr_t)a->bias % 4) return nb_set_error("nemo_gemm_mxfp4: C and bias must be aligned to their type");
    int rc = 0;
    NB_ELT_SWITCH(a->c_elt, T, rc = by_rows<T>(a, (cudaStream_t)stream));
    return rc;
}

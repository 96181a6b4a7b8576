// Selective state-space scan with carried state, for prompts, chunks and single rows.
//
//   h[d][n] = exp(step A[d][n]) h[d][n] + step x[d] B[n],   y[d] = (sum_n h[d][n] C[n] + skip[d] x[d]) silu(z[d])
//
// The state is held in fp32 registers. What belongs to a (row, channel) and not to a state (the step with
// its softplus, the gate, the output) is computed once. Where LPC lanes share a channel, rows (or
// streams) are dealt out among them for that, and the sums over the states of several rows are folded
// together: V values over LPC lanes take about V shuffles, and each sum ends in the lane that writes it.
//
// Two kernels: single rows, bound by the state's bytes, and runs of rows, bound by the exponentials
// (one per row, channel and state on the special-function units, 16 a clock an SM).
#include <type_traits>
#include "elt.cuh"
#include "cluster.cuh"

namespace {

using namespace nb;

struct ScanArgs {
    const void *x, *dt, *z, *B, *C;
    int64_t x_ld, x_ss, dt_ld, dt_ss, z_ld, z_ss, bc_ld, bc_ss;
    const float *A, *skip, *dt_bias, *state_in;
    float *state_out;
    void *y;
    int64_t y_ld, y_ss;
    const int *lens;
    int streams, c, D, N, per_group, softplus;
    int tiles, units;  // a warp's worth of channels: of a group, of a stream
    int64_t items;     // single rows: warps; runs: channel tiles of all streams
    int lw, tw, ranks; // runs: warps in a block, chunks of time in it, blocks of a cluster
};

// The special-function units' 2^x makes decays e^-v too small on average: by 5.1e-9 to 8.4e-9 of the value for v from
// 1e-5 to 3e-3, 2.4e-8 to 2.5e-8 from 3e-3 to 0.03, 1.6e-8 to 0.3, 2.5e-8 to 3 (a million values each; single values
// are within 1.5e-7 up to 1). That is less than a step of fp32, but the same way in every row of a long memory.
// With 2^-26 in the exponent, 1.03e-8 of the value, they are too large by 1.9e-9 to 5.3e-9 up to 3e-3, and too
// small by 1.5e-8 to 0.03, 6e-9 to 0.3 and 1.5e-8 to 3. It is too little to turn a decay of 1 into anything else.
// (Chunks are folded without it: two decays each, against one a row.)
constexpr float EVEN = 0x1p-26f;

// log(1 + e^v) = max(v, 0) + log1p(e), e = exp(-|v|) <= 1, and log1p(e) = 2 artanh(e / (2 + e)): the
// argument is at most 1/3, so seven terms of the series leave 1.4e-8 of it. No cancellation at either end.
__device__ __forceinline__ float softplus_f(float v) {
    const float e = ex2(-fabsf(v) * LOG2E);
    const float s = __fdividef(e, 2.0f + e), q = s * s;
    float p = 1.0f / 13.0f;
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    p = fmaf(p * q, s, s);
    return fmaf(2.0f, p, fmaxf(v, 0.0f));
}

// An element as it is loaded, and its value: kept apart, so that nothing waits for a load until its
// value is used
__device__ __forceinline__ uint32_t raw(const float *p) { return __float_as_uint(*p); }
__device__ __forceinline__ uint32_t raw(const __nv_bfloat16 *p) { return *(const unsigned short *)p; }
__device__ __forceinline__ uint32_t raw(const __half *p) { return *(const unsigned short *)p; }
template <typename T>
__device__ __forceinline__ float cooked(uint32_t v) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(v);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(v << 16);
    else return __half2float(__ushort_as_half((unsigned short)v));
}

// ---- single rows -----------------------------------------------------------------------------
// One row per stream: bound by HBM (8 N bytes of state per channel). A warp owns 32 / LPC channels of
// SB streams: the streams' rows are taken together, so that SB states are in flight per lane and A is
// read once for them. What is left above HBM's time is the time between a warp's loads and its stores,
// so instructions count: 1024 streams of 2048 channels, 16 states, bf16: 59 us (4.8 TB/s, 0.74 of the measured
// copy rate) where the same plan with 566 instructions a warp, predicated loads and a shuffle per stream's
// liveness took 78 us; N = 64, 1024 channels: 121 us, was 184 us.
constexpr int STEP_NT = 128, STEP_SB = 4;

template <typename T, int LPC, bool V4>
__global__ void __launch_bounds__(STEP_NT, 6) scan_step_kernel(const __grid_constant__ ScanArgs a) {
    constexpr int CPW = 32 / LPC, SB = LPC < STEP_SB ? LPC : STEP_SB, REP = LPC / SB;
    nb::pdl_wait();
    const uint32_t w = blockIdx.x * (STEP_NT / 32) + (threadIdx.x >> 5);  // (a 64-bit division is a hundred instructions)
    if (w >= (uint32_t)a.items) return;
    const int lane = threadIdx.x & 31, sub = lane % LPC, n0 = sub * 4, v = sub / REP;  // this lane's states, and its stream of SB
    const uint32_t sblk = w / (uint32_t)a.units;
    const int64_t s0 = (int64_t)sblk * SB;
    const int unit = (int)(w - sblk * a.units), grp = (uint32_t)unit / (uint32_t)a.tiles;
    const int dg = (unit - grp * a.tiles) * CPW + lane / LPC;
    const bool on = dg < a.per_group, st4 = n0 < a.N;
    const int d = grp * a.per_group + (on ? dg : a.per_group - 1);

    // four states of a lane, as they are loaded (those past N: zeros)
    auto load4 = [&](const auto *p, auto &o) __attribute__((always_inline)) {
        typedef typename std::remove_reference<decltype(o)>::type Vec4;
        if (V4 && st4) {
            o = *(const Vec4 *)p;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (V4 || n0 + j >= a.N) o.v[j] = 0.0f;
                else o.v[j] = p[j];
        }
    };
    // everything is asked for before anything is used; streams past the last one read the last one's
    Vec<float, 4> h[SB], A4;
    Vec<T, 4> b[SB], c[SB];
    const int left = (int)min((int64_t)SB, a.streams - s0);  // streams that exist
    const int64_t per_stream = (int64_t)a.D * a.N, lane_at = (int64_t)d * a.N + n0;
    const int64_t s = s0 + v;  // this lane's stream: it computes the stream's step and writes its output
    const int64_t sr = s0 + min(v, left - 1);
    const float *sp = a.state_in + s0 * per_stream + lane_at;
    const T *bp = (const T *)a.B + s0 * a.bc_ss + (int64_t)grp * a.N + n0, *cp = (const T *)a.C + (bp - (const T *)a.B);
#pragma unroll
    for (int r = 0; r < SB; ++r) {
        if (a.state_in) load4(sp, h[r]);
        else h[r].v[0] = h[r].v[1] = h[r].v[2] = h[r].v[3] = 0.0f;
        load4(bp, b[r]);
        load4(cp, c[r]);
        const bool more = r + 1 < left;
        sp += more ? per_stream : 0;
        bp += more ? a.bc_ss : 0;
        cp += more ? a.bc_ss : 0;
    }
    const bool live = v < left && (!a.lens || a.lens[s] > 0);
    const uint32_t rx = raw((const T *)a.x + sr * a.x_ss + d), rd = raw((const T *)a.dt + sr * a.dt_ss + d);
    const uint32_t rz = a.z ? raw((const T *)a.z + sr * a.z_ss + d) : 0;
    load4(a.A + lane_at, A4);
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, skip = a.skip ? a.skip[d] : 0.0f;

    const float xv = cooked<T>(rx);
    float step = cooked<T>(rd) + bias, gate = cooked<T>(rz);
    if (a.softplus) step = softplus_f(step);
    gate = a.z ? gate * nb::sigmoid_fast(gate) : 1.0f;
    const float sx = step * xv;
    step *= LOG2E;
    const uint32_t alive = __ballot_sync(0xffffffffu, live);  // bit r * REP: stream r has a row, for all channels alike
    const f2 A2[2] = { pack2(A4.v[0], A4.v[1]), pack2(A4.v[2], A4.v[3]) };
    float sum[SB];
#pragma unroll
    for (int r = 0; r < SB; ++r) {
        const f2 st2 = dup2(__shfl_sync(0xffffffffu, step, r * REP, LPC)), in2 = dup2(__shfl_sync(0xffffffffu, sx, r * REP, LPC));
        sum[r] = 0.0f;
        if (alive >> (r * REP) & 1) {  // without a row the state stays
            f2 acc = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float e0, e1;
                unpack2(fma2(st2, A2[j], dup2(EVEN)), e0, e1);
                f2 hh = fma2(pack2(ex2(e0), ex2(e1)), pack2(h[r].v[2 * j], h[r].v[2 * j + 1]),
                             mul2(in2, pack2(to_f32(b[r].v[2 * j]), to_f32(b[r].v[2 * j + 1]))));
                if (!V4) {  // states past N stay zeros (an infinite input times zero is a NaN)
                    unpack2(hh, e0, e1);
                    hh = pack2(n0 + 2 * j < a.N ? e0 : 0.0f, n0 + 2 * j + 1 < a.N ? e1 : 0.0f);
                }
                const f2 cc = pack2(to_f32(c[r].v[2 * j]), to_f32(c[r].v[2 * j + 1]));
                acc = j ? fma2(hh, cc, acc) : mul2(hh, cc);
                unpack2(hh, h[r].v[2 * j], h[r].v[2 * j + 1]);
            }
            float lo, hi;
            unpack2(acc, lo, hi);
            sum[r] = lo + hi;
        }
    }
    if (V4 && !st4) {  // a lane of states past N
#pragma unroll
        for (int r = 0; r < SB; ++r) sum[r] = 0.0f;
    }
    nb::WarpFold<SB, LPC / 2>::run(sum, lane);
    if (live && on && sub % REP == 0) ((T *)a.y)[s * a.y_ss + d] = nb::from_f32<T>(fmaf(skip, xv, sum[0]) * gate);
    if (a.state_out && on) {
        float *p = a.state_out + s0 * per_stream + lane_at;
#pragma unroll
        for (int r = 0; r < SB; ++r, p += per_stream)
            if (r < left) {
                if (V4) {
                    if (st4) *(Vec<float, 4> *)p = h[r];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (n0 + j < a.N) p[j] = h[r].v[j];
                }
            }
    }
}

template <typename T, int LPC, bool V4>
int run_step(ScanArgs a, cudaStream_t st) {
    constexpr int CPW = 32 / LPC, SB = LPC < STEP_SB ? LPC : STEP_SB;
    a.tiles = (a.per_group + CPW - 1) / CPW;
    a.units = a.D / a.per_group * a.tiles;
    a.items = (a.streams + SB - 1) / SB * (int64_t)a.units;
    const int64_t blocks = (a.items * 32 + STEP_NT - 1) / STEP_NT;
    if (a.items > 0x7fffffff) return nb_set_error("nemo_selective_scan: too many streams");
    nb::launch(scan_step_kernel<T, LPC, V4>, dim3((unsigned)blocks), STEP_NT, 0, st, a);
    return nb_check_launch("scan_step_kernel");
}

// ---- runs of rows ----------------------------------------------------------------------------

// softplus_f of two values
__device__ __forceinline__ f2 softplus2(f2 v) {
    float a, b;
    unpack2(v, a, b);
    const f2 e = pack2(ex2(-fabsf(a) * LOG2E), ex2(-fabsf(b) * LOG2E));
    float u, w;
    unpack2(add2(e, dup2(2.0f)), u, w);
    const f2 s = mul2(e, pack2(rcp(u), rcp(w))), q = mul2(s, s);
    f2 p = dup2(1.0f / 13.0f);
    p = fma2(p, q, dup2(1.0f / 11.0f));
    p = fma2(p, q, dup2(1.0f / 9.0f));
    p = fma2(p, q, dup2(1.0f / 7.0f));
    p = fma2(p, q, dup2(1.0f / 5.0f));
    p = fma2(p, q, dup2(1.0f / 3.0f));
    p = fma2(mul2(p, q), s, s);
    return fma2(dup2(2.0f), p, pack2(fmaxf(a, 0.0f), fmaxf(b, 0.0f)));
}

// A lane owns a channel's whole state where N <= 16 (else LPC lanes, 16 states each, with the rows'
// steps and outputs dealt out among them), so steps, gates and sums never leave its registers; only B
// and C, shared by the warp's channels, pass through shared memory. A warp runs one chunk of rows of its
// channels. Where the channels alone do not fill the GPU, time is cut as well: TW warps of a block
// and R blocks of a cluster hold chunks of the same channels. Each chunk but the last finds the state
// it ends in when started from zero (the first one from the true state), and the sum of its steps, all
// at once. A chunk's true first state is then folded from those before it, h <- exp(A sum of steps) h + end,
// and all chunks run again, from their true first states, writing y. Nothing
// but shared memory is needed for that, and the order of the sums is fixed.
//
// Measured: 64 streams x 200 rows x 2048 channels, 16 states, bf16: 163 us, of which the special-function units
// are busy 69 % (their 17 exponentials and more per row and channel) and instructions issue 51 %, 118 a row
// for 32 channels; 16384 rows of one stream, two passes: 468 us (70 % and 46 %). Four lanes a
// channel with rows prepared by other warps in shared memory: 500 us for the latter in one pass, bound by
// shared memory's 128 bytes a clock (steps, B, C and sums pass through it for every lane).
constexpr int LW_MAX = 8;  // warps per block: 4 or 8
template <int BYTES>
__device__ __forceinline__ void cp_async(void *dst, const void *src, bool is) {  // is false: zeros
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "n"(BYTES), "r"(is ? BYTES : 0)
                 : "memory");
}


// A raw tile in shared memory: U rows of the warp's x, dt and z, then of B and C, in chunks of CB bytes.
template <typename T, int LPC, int NS, int U>
struct LongTile {
    static constexpr int CPW = 32 / LPC, NP = LPC * NS, ES = sizeof(T);
    static constexpr int CB = CPW * ES < 16 ? CPW * ES : 16;
    static constexpr int XC = CPW * ES / CB, BC = NP * ES / CB > 0 ? NP * ES / CB : 1;  // chunks in a row
    static constexpr int XB = U * XC * CB, BB = U * BC * CB;
    static constexpr int TILE = 3 * XB + 2 * BB;
    // tiles in the ring: four, or two of the large ones, so that 16 warps still fit an SM (16384 fp32 rows: 621 us with
    // four tiles of 4 KB a warp, 478 us with two)
    static constexpr int Q = TILE < 4096 ? 4 : 2;
};

// What a lane of the kernel for runs works on: its channel, and its warp's chunk of the stream's rows.
template <int LPC, int NS, int U>
struct Place {
    int rank, chunk, chunks, unit, grp, tb, te;
    bool on;
    int64_t s, d;
    __device__ __forceinline__ Place(const ScanArgs &a, uint32_t block, uint32_t thread) {
        constexpr int CPW = 32 / LPC;
        const int warp = thread >> 5, lane = thread & 31;
        rank = a.ranks > 1 ? block % a.ranks : 0;
        const uint32_t item = (block / (uint32_t)a.ranks) * ((uint32_t)a.lw / (uint32_t)a.tw) + (uint32_t)warp / (uint32_t)a.tw;  // (stream, channel tile)
        const bool real = item < (uint32_t)a.items;
        const uint32_t su = real ? item / (uint32_t)a.units : 0;
        s = su;
        unit = real ? (int)(item - su * a.units) : 0;
        grp = (uint32_t)unit / (uint32_t)a.tiles;
        const int dg = (unit - grp * a.tiles) * CPW + lane / LPC;
        on = real && dg < a.per_group;
        d = grp * a.per_group + min(dg, a.per_group - 1);
        const int len = !real ? 0 : a.lens ? max(0, min(a.lens[s], a.c)) : a.c;
        chunks = a.tw * a.ranks;
        chunk = rank * a.tw + warp % a.tw;
        const int rows = (len + chunks * U - 1) / (chunks * U) * U;  // rows per chunk, whole tiles
        tb = min(len, chunk * rows);
        te = min(len, tb + rows);
    }
};

// States past N fill up a lane with zeros. Times an infinite input or step that is a NaN, which stays, in all of them
// alike, and goes into the outputs. Channels that were left with one (or whose infinite state cannot be folded over
// chunks), those of the lanes in `hit`, run once more, row by row from the stream's first one and with their own
// states alone, writing the chunk's outputs. 64 streams x 200 rows, 1024 channels: states past N kept out of every
// row's sum by a condition cost 4 to 12 %, a test in every tile 1 to 6 %, this nothing where no channel needs it, and 1.0
// to 1.5 us a row where one does. Its addresses are formed anew: kept in registers while the kernel's own passes
// run, which have none left, they cost up to 16 %.
template <typename T, int LPC, int NS, int U>
__device__ __forceinline__ void run_again(const ScanArgs &a, uint32_t hit, f2 (&h)[NS / 2]) {
    uint32_t block, thread;
    asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(block));
    asm volatile("mov.u32 %0, %%tid.x;" : "=r"(thread));
    const Place<LPC, NS, U> p(a, block, thread);
    const int lane = thread & 31, sub = lane % LPC, count = min(NS, a.N - sub * NS);  // this lane's states
    const bool again = (hit >> (lane - sub) & (2u << (LPC - 1)) - 1) != 0;            // the same in all lanes of a channel
    const int64_t at = (p.s * a.D + p.d) * a.N + sub * NS, bc = p.s * a.bc_ss + (int64_t)p.grp * a.N + sub * NS;
    const float *A = a.A + p.d * a.N + sub * NS;
    const T *X = (const T *)a.x + p.s * a.x_ss + p.d, *DT = (const T *)a.dt + p.s * a.dt_ss + p.d;
    if (again) {
#pragma unroll
        for (int j = 0; j < NS; j += 2)
            h[j / 2] = pack2(a.state_in && j < count ? a.state_in[at + j] : 0.0f, a.state_in && j + 1 < count ? a.state_in[at + j + 1] : 0.0f);
    }
    for (int t = 0; t < p.te; ++t) {
        float sum = 0.0f;
        const float x = to_f32(X[(int64_t)t * a.x_ld]);
        if (again) {
            float step = to_f32(DT[(int64_t)t * a.dt_ld]) + (a.dt_bias ? a.dt_bias[p.d] : 0.0f);
            if (a.softplus) step = softplus_f(step);
            const T *B = (const T *)a.B + bc + (int64_t)t * a.bc_ld, *C = (const T *)a.C + bc + (int64_t)t * a.bc_ld;
#pragma unroll
            for (int j = 0; j < NS; j += 2) {
                float v[2];
                unpack2(h[j / 2], v[0], v[1]);
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (j + k < count) {
                        v[k] = fmaf(ex2(fmaf(step * LOG2E, A[j + k], EVEN)), v[k], step * x * to_f32(B[j + k]));
                        sum = fmaf(v[k], to_f32(C[j + k]), sum);
                    }
                h[j / 2] = pack2(v[0], v[1]);
            }
        }
#pragma unroll
        for (int o = 1; o < LPC; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (again && p.on && sub == 0 && t >= p.tb) {
            float v = fmaf(a.skip ? a.skip[p.d] : 0.0f, x, sum);
            if (a.z) {
                const float z = to_f32(((const T *)a.z)[p.s * a.z_ss + p.d + (int64_t)t * a.z_ld]);
                v *= z * nb::sigmoid_fast(z);
            }
            ((T *)a.y)[p.s * a.y_ss + p.d + (int64_t)t * a.y_ld] = nb::from_f32<T>(v);
        }
    }
}

template <typename T, int LPC, int NS, int U, bool V4, bool ASYNC>
__global__ void __launch_bounds__(32 * LW_MAX, 2) scan_long_kernel(const __grid_constant__ ScanArgs a) {
    constexpr int CPW = 32 / LPC, NP = LPC * NS, RP = U / LPC;  // channels per warp, padded states, rows per lane and tile
    constexpr int QUADS = U * NP / 4, QL = (QUADS + 31) / 32;   // groups of four states in a tile, per lane
    using K = LongTile<T, LPC, NS, U>;
    const int LW = a.lw;
    extern __shared__ __align__(16) float smem[];  // [LW][2][U][NP]: the warps' tiles of B and C; ASYNC: [LW][Q] raw tiles
    float *ends = smem + LW * 2 * U * NP + (ASYNC ? LW * K::Q * K::TILE / 4 : 0);  // [LW + 1][NS + 1][32]: end states and sums of steps of the warps' chunks, of the whole block
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPC, n0 = sub * NS;
    nb::pdl_wait();
    const Place<LPC, NS, U> here(a, blockIdx.x, threadIdx.x);
    const int rank = here.rank, chunk = here.chunk, chunks = here.chunks, unit = here.unit, grp = here.grp, tb = here.tb, te = here.te;
    const bool on = here.on;
    const int64_t s = here.s, d = here.d;
    const int nch = min(CPW, a.per_group - (unit - grp * a.tiles) * CPW);  // this warp's channels

    f2 A2[NS / 2], h[NS / 2];
    const int64_t at = (s * a.D + d) * a.N + n0;
    auto load_states = [&](const float *p, f2 (&o)[NS / 2]) {
#pragma unroll
        for (int j = 0; j < NS / 2; j += 2) {
            float f[4];
            if (V4 && n0 + 2 * j < a.N) {
                const float4 v = *(const float4 *)(p + 2 * j);
                f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) f[k] = !V4 && n0 + 2 * j + k < a.N ? p[2 * j + k] : 0.0f;
            }
            o[j] = pack2(f[0], f[1]);
            o[j + 1] = pack2(f[2], f[3]);
        }
    };
    load_states(a.A + d * a.N + n0, A2);
#pragma unroll
    for (int j = 0; j < NS / 2; ++j) h[j] = 0;
    if (chunk == 0 && a.state_in) load_states(a.state_in + at, h);
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, skip = a.skip ? a.skip[d] : 0.0f;
    const T *X = (const T *)a.x + s * a.x_ss + d, *DT = (const T *)a.dt + s * a.dt_ss + d;
    const T *Z = a.z ? (const T *)a.z + s * a.z_ss + d : nullptr;
    T *Y = (T *)a.y + s * a.y_ss + d;
    const T *B = (const T *)a.B + s * a.bc_ss + (int64_t)grp * a.N, *C = (const T *)a.C + s * a.bc_ss + (int64_t)grp * a.N;
    typedef float Tile[U][NP];
    Tile &sb = ((Tile *)smem)[2 * warp], &sc = ((Tile *)smem)[2 * warp + 1];

    // The chunk's rows: WRITE with the outputs, otherwise the end state and the sum of the steps alone.
    auto pass = [&](auto write) __attribute__((always_inline)) {
        constexpr bool WRITE = decltype(write)::value;
        float total = 0.0f;
        uint32_t rx[RP], rd[RP], rz[RP];
        nb::Vec<T, 4> rb[QL], rc[QL];
        // ASYNC: tiles of the warp's rows on their way to shared memory, Q - 1 of them; rows that do not exist
        // are filled with zeros
        const int64_t first = grp * a.per_group + (unit - grp * a.tiles) * CPW - d;  // the warp's first channel, from this lane's
        uint8_t *ring = (uint8_t *)(smem + LW * 2 * U * NP) + warp * K::Q * K::TILE;
        auto copy_rows = [&](const T *base, int64_t ld, int t0, int row_bytes, int off, auto chunks) __attribute__((always_inline)) {
            constexpr int XC = decltype(chunks)::value;  // at most so many chunks of CB bytes in a row
#pragma unroll
            for (int k = 0; k < (U * XC + 31) / 32; ++k) {
                const int e = lane + k * 32, row = e / XC, at = e % XC * K::CB;
                if (e < U * XC && at < row_bytes) {
                    const bool is = t0 + row < te;
                    cp_async<K::CB>(ring + off + row * XC * K::CB + at, (const uint8_t *)(base + (int64_t)(is ? t0 + row : tb) * ld) + at, is);
                }
            }
        };
        auto issue = [&](int t0, int slot) __attribute__((always_inline)) {
            if (t0 < te) {
                const int s0 = slot * K::TILE, mine_bytes = nch * (int)sizeof(T), bc_bytes = a.N * (int)sizeof(T);
                copy_rows(X + first, a.x_ld, t0, mine_bytes, s0, std::integral_constant<int, K::XC>{});
                copy_rows(DT + first, a.dt_ld, t0, mine_bytes, s0 + K::XB, std::integral_constant<int, K::XC>{});
                if (WRITE && Z) copy_rows(Z + first, a.z_ld, t0, mine_bytes, s0 + 2 * K::XB, std::integral_constant<int, K::XC>{});
                copy_rows(B, a.bc_ld, t0, bc_bytes, s0 + 3 * K::XB, std::integral_constant<int, K::BC>{});
                if (WRITE) copy_rows(C, a.bc_ld, t0, bc_bytes, s0 + 3 * K::XB + K::BB, std::integral_constant<int, K::BC>{});
            }
            asm volatile("cp.async.commit_group;" ::: "memory");  // an empty one too: the count tells which tile has landed
        };
        // this lane's next rows of x, dt, z and its groups of B and C
        const T *px = X + (int64_t)(tb + sub * RP) * a.x_ld, *pd = DT + (int64_t)(tb + sub * RP) * a.dt_ld;
        const T *pz = WRITE && Z ? Z + (int64_t)(tb + sub * RP) * a.z_ld : nullptr;
        T *py = Y + (int64_t)(tb + sub * RP) * a.y_ld;
        const int64_t bc0 = (int64_t)(tb + lane / (NP / 4)) * a.bc_ld + lane % (NP / 4) * 4;
        const T *pb = B + bc0, *pc = C + bc0;
        auto fetch = [&](int left) __attribute__((always_inline)) {  // left: rows of the chunk from this tile on
            const bool all = left >= U;
#pragma unroll
            for (int r = 0; r < RP; ++r) {
                const int k = all ? r : min(sub * RP + r, left - 1) - sub * RP;  // a row that does not exist: the last one
                rx[r] = raw(px + k * a.x_ld);
                rd[r] = raw(pd + k * a.dt_ld);
                if (WRITE && Z) rz[r] = raw(pz + k * a.z_ld);
            }
            px += U * a.x_ld;
            pd += U * a.dt_ld;
            if (WRITE && Z) pz += U * a.z_ld;
#pragma unroll
            for (int k = 0; k < QL; ++k) {
                // group e = lane + 32 k of the tile: row e / (NP / 4) of it, state e % (NP / 4) * 4
                constexpr int QR = NP / 4;
                const int e = lane + k * 32, row = e / QR, n = e % QR * 4;
                const bool is = e < QUADS && (all || row < left);
                const int64_t off = QR >= 32 ? (int64_t)(row - lane / QR) * a.bc_ld + (n - lane % QR * 4) : (int64_t)(k * 32 / QR) * a.bc_ld;
#pragma unroll
                for (int j = 0; j < 4; ++j) rb[k].v[j] = rc[k].v[j] = nb::from_f32<T>(0.0f);
                if (V4) {
                    if (is && n < a.N) {
                        rb[k] = *(const nb::Vec<T, 4> *)(pb + off);
                        if (WRITE) rc[k] = *(const nb::Vec<T, 4> *)(pc + off);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (is && n + j < a.N) {
                            rb[k].v[j] = pb[off + j];
                            if (WRITE) rc[k].v[j] = pc[off + j];
                        }
                }
            }
            pb += U * a.bc_ld;
            pc += U * a.bc_ld;
        };
        int slot = 0;  // of the tile at t0
        if (ASYNC) {
#pragma unroll
            for (int q = 0; q < K::Q - 1; ++q) issue(tb + q * U, q);
        } else if (tb < te) {
            fetch(te - tb);
        }
        for (int t0 = tb; t0 < te; t0 += U) {
            if (ASYNC) {
                asm volatile("cp.async.wait_group %0;" ::"n"(K::Q - 2) : "memory");
                __syncwarp();
                const uint8_t *raw_tile = ring + slot * K::TILE;
#pragma unroll
                for (int r = 0; r < RP; ++r) {
                    const T *q = (const T *)(raw_tile + (sub * RP + r) * K::XC * K::CB) + lane / LPC;
                    rx[r] = raw(q);
                    rd[r] = raw((const T *)((const uint8_t *)q + K::XB));
                    if (WRITE && Z) rz[r] = raw((const T *)((const uint8_t *)q + 2 * K::XB));
                }
#pragma unroll
                for (int k = 0; k < QL; ++k) {
                    const int e = lane + k * 32, row = e / (NP / 4), n = e % (NP / 4) * 4;
                    if (e < QUADS && n < a.N) {
                        const T *q = (const T *)(raw_tile + 3 * K::XB + row * K::BC * K::CB) + n;
                        rb[k] = *(const nb::Vec<T, 4> *)q;
                        if (WRITE) rc[k] = *(const nb::Vec<T, 4> *)((const uint8_t *)q + K::BB);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) rb[k].v[j] = rc[k].v[j] = nb::from_f32<T>(0.0f);
                    }
                }
                issue(t0 + (K::Q - 1) * U, slot == 0 ? K::Q - 1 : slot - 1);  // into the slot of the tile before
                slot = slot + 1 == K::Q ? 0 : slot + 1;
            } else {
                __syncwarp();
            }
#pragma unroll
            for (int k = 0; k < QL; ++k) {
                const int e = lane + k * 32;
                if (e < QUADS) {
                    const int r = e / (NP / 4), n = e % (NP / 4) * 4;
                    *(float4 *)&sb[r][n] = make_float4(nb::to_f32(rb[k].v[0]), nb::to_f32(rb[k].v[1]), nb::to_f32(rb[k].v[2]), nb::to_f32(rb[k].v[3]));
                    if (WRITE)
                        *(float4 *)&sc[r][n] = make_float4(nb::to_f32(rc[k].v[0]), nb::to_f32(rc[k].v[1]), nb::to_f32(rc[k].v[2]), nb::to_f32(rc[k].v[3]));
                }
            }
            float xv[RP], step[RP], sx[RP], gate[RP];
#pragma unroll
            for (int r = 0; r < RP; ++r) {
                xv[r] = cooked<T>(rx[r]);
                step[r] = cooked<T>(rd[r]) + bias;
                if (WRITE && Z) gate[r] = cooked<T>(rz[r]);
            }
            const int live = te - t0;  // rows of this tile that exist
            if (!ASYNC && live > U) fetch(live - U);
            if (a.softplus) {
#pragma unroll
                for (int r = 0; r + 1 < RP; r += 2) unpack2(softplus2(pack2(step[r], step[r + 1])), step[r], step[r + 1]);
                if (RP == 1) step[0] = softplus_f(step[0]);
            }
#pragma unroll
            for (int r = 0; r < RP; ++r) {
                const bool is = sub * RP + r < live;  // a row behind the last one keeps the state: a step and an input of 0
                sx[r] = is ? step[r] * xv[r] : 0.0f;
                step[r] = is ? step[r] * LOG2E : 0.0f;
                if (WRITE && Z) gate[r] *= nb::sigmoid_fast(gate[r]);
            }
            __syncwarp();
            float sum[U];
            auto advance = [&](int r) __attribute__((always_inline)) {
                const float st = LPC == 1 ? step[r % RP] : __shfl_sync(0xffffffffu, step[r % RP], r / RP, LPC);
                const float in = LPC == 1 ? sx[r % RP] : __shfl_sync(0xffffffffu, sx[r % RP], r / RP, LPC);
                const f2 st2 = dup2(st), in2 = dup2(in);
                asm volatile("" ::: "memory");  // one row's B and C in registers at a time
                if (!WRITE) total += st;
                f2 acc = 0;
#pragma unroll
                for (int q = 0; q < NS / 4; ++q) {
                    const float4 bv = *(const float4 *)&sb[r][n0 + 4 * q];
                    float4 cv;
                    if (WRITE) cv = *(const float4 *)&sc[r][n0 + 4 * q];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        f2 &hh = h[2 * q + j];
                        float e0, e1;
                        unpack2(fma2(st2, A2[2 * q + j], dup2(EVEN)), e0, e1);
                        hh = fma2(pack2(ex2(e0), ex2(e1)), hh, mul2(in2, j ? pack2(bv.z, bv.w) : pack2(bv.x, bv.y)));
                        if (WRITE) {
                            const f2 cc = j ? pack2(cv.z, cv.w) : pack2(cv.x, cv.y);
                            acc = q + j ? fma2(hh, cc, acc) : mul2(hh, cc);
                        }
                    }
                }
                float lo, hi;
                unpack2(acc, lo, hi);
                sum[r] = lo + hi;
            };
            if (live >= U) {
#pragma unroll
                for (int r = 0; r < U; ++r) advance(r);
            } else {  // (rows that do not exist keep the state, so leaving them out only saves their time)
#pragma unroll
                for (int r = 0; r < U; ++r) {
                    sum[r] = 0.0f;
                    if (r < live) advance(r);
                }
            }
            if (WRITE) {
                nb::WarpFold<U, LPC / 2>::run(sum, lane);  // lane sub: rows sub * RP ..
#pragma unroll
                for (int r = 0; r < RP; ++r) {
                    if (on && sub * RP + r < live) {
                        float v = fmaf(skip, xv[r], sum[r]);
                        if (Z) v *= gate[r];
                        py[r * a.y_ld] = nb::from_f32<T>(v);
                    }
                }
                py += U * a.y_ld;
            }
        }
        return total;
    };

    float *mine = ends + warp * (NS + 1) * 32 + lane, *block = ends + LW * (NS + 1) * 32 + lane;
    // h <- exp(A sum) h + end of a chunk (or of a block's chunks), given how to read it. The decay is applied
    // as two halves, and not to a state of zero: step by step a growing channel overflows when its
    // state does, not when its growth over a chunk would.
    // An infinite state stays so row by row, but times a chunk's decay of zero it is a NaN; and infinite steps leave no
    // sum. Such a channel is `odd`; whether it is, is looked at (CHECK) only where a state that is not finite came out.
    bool odd = false;
    __shared__ uint8_t odds[32 * LW_MAX];  // kept there while the rows run
    auto fold = [&](auto get, auto check) __attribute__((always_inline)) {
        constexpr bool CHECK = decltype(check)::value;
        const float sum = get(NS);
        const f2 half = dup2(0.5f * sum);
        if (CHECK) odd |= fabsf(sum) == INFINITY;
#pragma unroll
        for (int j = 0; j < NS / 2; ++j) {
            float e0, e1, h0, h1;
            unpack2(mul2(half, A2[j]), e0, e1);
            unpack2(h[j], h0, h1);
            if (CHECK) odd |= fabsf(h0) == INFINITY || fabsf(h1) == INFINITY;
            e0 = ex2(e0);
            e1 = ex2(e1);
            h[j] = add2(pack2(h0 == 0.0f ? 0.0f : h0 * e0 * e0, h1 == 0.0f ? 0.0f : h1 * e1 * e1), pack2(get(2 * j), get(2 * j + 1)));
        }
    };
    // from a state of zero over the blocks before `r` and the chunks w0 .. w1 - 1 of this one; the sum of the latter
    auto fold_all = [&](int r, int w0, int w1, auto check) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NS / 2; ++j) h[j] = 0;
        const uint32_t b = (uint32_t)__cvta_generic_to_shared(block);
        for (int q = 0; q < r; ++q) fold([&](int k) { return nb::ld_cluster(b + k * 128, q); }, check);
        float total = 0.0f;
        for (int w = w0; w < w1; ++w) {
            const float *e = ends + w * (NS + 1) * 32 + lane;
            fold([&](int k) { return e[k * 32]; }, check);
            total += e[NS * 32];
        }
        return total;
    };
    auto fold_odd = [&](int r, int w0, int w1) __attribute__((always_inline)) {
        const float total = fold_all(r, w0, w1, std::false_type{});
        f2 wild = 0;
#pragma unroll
        for (int j = 0; j < NS / 2; ++j) wild = fma2(h[j], dup2(0.0f), wild);
        float lo, hi;
        unpack2(wild, lo, hi);
        odd = false;
        if (lo + hi != 0.0f) fold_all(r, w0, w1, std::true_type{});  // the same states again
        return total;
    };
    if (chunks > 1) {
        auto put = [&](float *to, float total) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NS / 2; ++j) {
                float lo, hi;
                unpack2(h[j], lo, hi);
                to[2 * j * 32] = lo;
                to[(2 * j + 1) * 32] = hi;
            }
            to[NS * 32] = total;
        };
        put(mine, chunk < chunks - 1 ? pass(std::false_type{}) : 0.0f);
        __syncthreads();
        if (a.ranks > 1) {  // one channel tile per block
            if (warp == LW - 1 && rank < a.ranks - 1) {
                const float total = fold_odd(0, 0, LW);
                put(block, odd ? INFINITY : total);
            }
            nb::cluster_sync();
        }
        fold_odd(rank, warp - warp % a.tw, warp);  // the state before the chunk
        odds[threadIdx.x] = odd;
        if (chunk == 0 && a.state_in) load_states(a.state_in + at, h);
        pass(std::true_type{});
    } else {
        pass(std::true_type{});
    }

    {
        float lo, hi;
        unpack2(h[NS / 2 - 1], lo, hi);
        const uint32_t hit = __ballot_sync(0xffffffffu, on && ((chunks > 1 && odds[threadIdx.x]) || (n0 + NS > a.N && !(hi == 0.0f))));
        if (hit) run_again<T, LPC, NS, U>(a, hit, h);
    }
    if (chunks > 1) {
        // no block leaves while another reads its shared memory; and no chunk writes a state that is to replace
        // the one before it while the first chunk may still read that
        if (a.ranks > 1) nb::cluster_sync();
        else __syncthreads();
    }
    if (a.state_out && on && chunk == chunks - 1) {
#pragma unroll
        for (int j = 0; j < NS / 2; j += 2) {
            float f[4];
            unpack2(h[j], f[0], f[1]);
            unpack2(h[j + 1], f[2], f[3]);
            float *p = a.state_out + at + 2 * j;
            if (V4) {
                if (n0 + 2 * j < a.N) *(float4 *)p = make_float4(f[0], f[1], f[2], f[3]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n0 + 2 * j + k < a.N) p[k] = f[k];
            }
        }
    }
}

template <typename T, int LPC, int NS, int U, bool V4, bool ASYNC>
int launch_long(ScanArgs a, cudaStream_t st) {
    constexpr int CPW = 32 / LPC;
    a.tiles = (a.per_group + CPW - 1) / CPW;
    a.units = a.D / a.per_group * a.tiles;
    a.items = (int64_t)a.streams * a.units;
    // Time is cut where the channels give less than five warps an SM: a chunk costs its rows twice, less
    // the outputs (16384 rows of 2048 channels: 10.6 ms whole, 0.50 ms in 64 chunks; 24 streams of 600 rows
    // of 1024 channels, 5.2 warps an SM: 0.22 ms whole, 0.21 to 0.25 ms in 2 to 8). Then until there are
    // 32 warps an SM (8 streams of up to 2500 rows of 2048 channels: 0.62 ms with 8, 0.40 ms with 16, 0.35 ms with
    // 32), at 32 rows a chunk at least.
    int chunks = 1;
    if (a.items < 148 * 5)
        while (chunks < 64 && a.items * chunks < 148 * 32 && chunks * 2 * 32 <= a.c) chunks *= 2;
    // blocks of four warps spread better where one block need not hold several chunks (64 streams of 200 rows, in
    // tiles of four: 170 us, 192 us with eight)
    const int LW = a.lw = chunks == 1 ? 4 : 8;
    a.tw = chunks < LW ? chunks : LW;
    a.ranks = chunks / a.tw;
    const int per_block = LW / a.tw;
    const int64_t blocks = (a.items + per_block - 1) / per_block * a.ranks;
    if (a.items > 0x7fffffff || blocks > 0x7fffffff) return nb_set_error("nemo_selective_scan: too many streams");
    using K = LongTile<T, LPC, NS, U>;
    const size_t smem = (LW * 2 * U * LPC * NS + (chunks > 1 ? (LW + 1) * (NS + 1) * 32 : 0)) * sizeof(float) + (ASYNC ? LW * K::Q * K::TILE : 0);
    auto kernel = scan_long_kernel<T, LPC, NS, U, V4, ASYNC>;
    if (nb_smem_attr((const void *)kernel, smem)) return -1;
    if (a.ranks == 1) {
        nb::launch(kernel, dim3((unsigned)blocks), 32 * LW, smem, st, a);
    } else {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)blocks);
        cfg.blockDim = dim3(32 * LW);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = a.ranks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = nb_pdl_enabled() ? 2 : 1;
        cudaLaunchKernelEx(&cfg, kernel, a);
    }
    return nb_check_launch("scan_long_kernel");
}

template <typename T, int LPC, int NS, bool V4>
int run_long(const ScanArgs &a, cudaStream_t st) {
    // asynchronous copies of 16 bytes (8 where a warp has four 16-bit channels) where all rows allow it (in tiles of four rows, recording of
    // 16384 rows: 495 us without, 485 us with; prompts 347 and 319 us)
    constexpr int E = 16 / sizeof(T);
    const uintptr_t ptrs = (uintptr_t)a.x | (uintptr_t)a.dt | (uintptr_t)a.z | (uintptr_t)a.B | (uintptr_t)a.C;
    const int64_t strides = a.x_ld | a.x_ss | a.dt_ld | a.dt_ss | (a.z ? a.z_ld | a.z_ss : 0) | a.bc_ld | a.bc_ss;
    constexpr int U = LPC < 4 ? 4 : LPC;  // rows a tile: at least one per lane of a channel
    if constexpr (V4)
        if (ptrs % 16 == 0 && strides % E == 0 && a.per_group % E == 0 && a.N % E == 0) {
            // eight rows a tile where a lane holds a channel and runs are long (recording 490 us with four, 466 us with
            // eight; chunks of 7 fp32 rows 33 and 42 us)
            if constexpr (LPC == 1)
                if (a.c >= 32) return launch_long<T, LPC, NS, 8, true, true>(a, st);
            return launch_long<T, LPC, NS, U, true, true>(a, st);
        }
    return launch_long<T, LPC, NS, U, V4, false>(a, st);
}

template <typename T, bool V4>
int by_size(const ScanArgs &a, cudaStream_t st) {
    // (runs of 2 rows for 256 streams of 2048 channels: 30 us with the kernel for runs, 61 us row by row)
    if (a.c == 1) {
        if (a.N <= 4) return run_step<T, 1, V4>(a, st);
        if (a.N <= 8) return run_step<T, 2, V4>(a, st);
        if (a.N <= 16) return run_step<T, 4, V4>(a, st);
        if (a.N <= 32) return run_step<T, 8, V4>(a, st);
        if (a.N <= 64) return run_step<T, 16, V4>(a, st);
        return run_step<T, 32, V4>(a, st);
    }
    if (a.N <= 4) return run_long<T, 1, 4, V4>(a, st);
    if (a.N <= 8) return run_long<T, 1, 8, V4>(a, st);
    if (a.N <= 16) return run_long<T, 1, 16, V4>(a, st);
    if (a.N <= 32) return run_long<T, 2, 16, V4>(a, st);
    if (a.N <= 64) return run_long<T, 4, 16, V4>(a, st);
    return run_long<T, 8, 16, V4>(a, st);
}

}  // namespace

extern "C" int nemo_selective_scan(const nemo_selective_scan_args_t *p, void *stream) {
    if (!p) return nb_set_error("nemo_selective_scan: null arguments");
    if (p->streams < 0 || p->c < 0 || p->c > (1 << 30) || p->D < 0 || p->D > (1 << 24))
        return nb_set_error("nemo_selective_scan: bad shape streams=%d c=%d D=%d", p->streams, p->c, p->D);
    if (p->N < 1 || p->N > 128) return nb_set_error("nemo_selective_scan: N=%d outside 1..128", p->N);
    if (p->groups < 1 || p->D % p->groups) return nb_set_error("nemo_selective_scan: D=%d is not a multiple of groups=%d", p->D, p->groups);
    if (!nb::elt_ok(p->elt)) return nb_set_error("nemo_selective_scan: unknown element type %d", p->elt);
    if (p->streams == 0 || p->D == 0 || (p->c == 0 && !p->state_out)) return 0;
    if (!p->A || (p->c > 0 && (!p->x || !p->dt || !p->B || !p->C || !p->y))) return nb_set_error("nemo_selective_scan: null pointer");
    if (p->c > 1 && (p->x_ld < p->D || p->dt_ld < p->D || p->y_ld < p->D || (p->z && p->z_ld < p->D) || p->bc_ld < (int64_t)p->groups * p->N))
        return nb_set_error("nemo_selective_scan: row pitches below the row's elements");
    // (with lens the rows written are known on the device alone: one row a stream is looked at, then)
    if (nb_rows_overlap(p->streams, p->y_sstride, p->lens && p->c > 1 ? 1 : p->c, p->y_ld, p->D))
        return nb_set_error("nemo_selective_scan: rows of y overlap (y_sstride=%lld)", (long long)p->y_sstride);
    const int es = nb::elt_size(p->elt);
    if (((uintptr_t)p->x | (uintptr_t)p->dt | (uintptr_t)p->z | (uintptr_t)p->B | (uintptr_t)p->C | (uintptr_t)p->y) % es ||
        ((uintptr_t)p->A | (uintptr_t)p->skip | (uintptr_t)p->dt_bias | (uintptr_t)p->state_in | (uintptr_t)p->state_out) % 4)
        return nb_set_error("nemo_selective_scan: buffers must be aligned to their type");
    ScanArgs a = {};
    a.x = p->x; a.dt = p->dt; a.z = p->z; a.B = p->B; a.C = p->C;
    a.x_ld = p->x_ld; a.x_ss = p->x_sstride; a.dt_ld = p->dt_ld; a.dt_ss = p->dt_sstride;
    a.z_ld = p->z_ld; a.z_ss = p->z_sstride; a.bc_ld = p->bc_ld; a.bc_ss = p->bc_sstride;
    a.A = p->A; a.skip = p->skip; a.dt_bias = p->dt_bias; a.state_in = p->state_in; a.state_out = p->state_out;
    a.y = p->y; a.y_ld = p->y_ld; a.y_ss = p->y_sstride; a.lens = p->lens;
    a.streams = p->streams; a.c = p->c; a.D = p->D; a.N = p->N; a.per_group = p->D / p->groups; a.softplus = p->dt_softplus;
    // four states at a time where every row of A, the states, B and C allows it
    const bool v4 = p->N % 4 == 0 && (((uintptr_t)p->A | (uintptr_t)p->state_in | (uintptr_t)p->state_out) & 15) == 0 &&
                    (((uintptr_t)p->B | (uintptr_t)p->C) % (4 * es)) == 0 && ((p->bc_ld | p->bc_sstride) & 3) == 0;
    int rc = 0;
    cudaStream_t st = (cudaStream_t)stream;
    NB_ELT_SWITCH(p->elt, T, rc = v4 ? by_size<T, true>(a, st) : by_size<T, false>(a, st));
    return rc;
}

// Selective state-space scan with carried state, for prompts, chunks and single rows.
//
//   h[d][n] = exp(step A[d][n]) h[d][n] + step x[d] B[n],   y[d] = (sum_n h[d][n] C[n] + skip[d] x[d]) silu(z[d])
//
// The state is held in fp32 registers: LPC lanes share a channel, four states each, so that a
// warp reads the state of its channels as one contiguous run and a row's sum over the states is a few
// shuffles.
#include "elt.cuh"

namespace {

constexpr int NT = 128;
constexpr float LOG2E = 1.4426950408889634f;

struct ScanArgs {
    const void *x, *dt, *z, *B, *C;
    int64_t x_ld, x_ss, dt_ld, dt_ss, z_ld, z_ss, bc_ld, bc_ss;
    const float *A, *skip, *dt_bias, *state_in;
    float *state_out;
    void *y;
    int64_t y_ld, y_ss;
    const int *lens;
    int streams, c, D, N, per_group, softplus, wps;  // channels per group, warps per stream
    int64_t warps;
};

// log(1 + e^v); for v > 20 that is v to fp32
__device__ __forceinline__ float softplus_f(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

template <typename T, int LPC, bool V4>
__global__ void __launch_bounds__(NT) selective_scan_kernel(const __grid_constant__ ScanArgs a) {
    constexpr int CPW = 32 / LPC;  // channels per warp
    nb::pdl_wait();
    const int64_t w = ((int64_t)blockIdx.x * NT + threadIdx.x) >> 5;
    if (w >= a.warps) return;
    const int lane = threadIdx.x & 31, n0 = (lane % LPC) * 4;
    const int64_t s = w / a.wps;
    const int d = (int)(w - s * a.wps) * CPW + lane / LPC;
    const bool on = d < a.D;
    const int dd = on ? d : a.D - 1;
    const int len = a.lens ? max(0, min(a.lens[s], a.c)) : a.c;
    float A2[4], h[4];
    const int64_t sat = (s * a.D + dd) * (int64_t)a.N + n0;
#pragma unroll
    for (int j = 0; j < 4; ++j) A2[j] = h[j] = 0.0f;
    if (V4) {
        if (n0 < a.N) {
            const float4 t = *(const float4 *)(a.A + (int64_t)dd * a.N + n0);
            A2[0] = t.x; A2[1] = t.y; A2[2] = t.z; A2[3] = t.w;
            if (a.state_in) {
                const float4 u = *(const float4 *)(a.state_in + sat);
                h[0] = u.x; h[1] = u.y; h[2] = u.z; h[3] = u.w;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < a.N) {
                A2[j] = a.A[(int64_t)dd * a.N + n0 + j];
                if (a.state_in) h[j] = a.state_in[sat + j];
            }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) A2[j] *= LOG2E;
    const float bias = a.dt_bias ? a.dt_bias[dd] : 0.0f, skip = a.skip ? a.skip[dd] : 0.0f;
    const T *x = (const T *)a.x + s * a.x_ss + dd, *dt = (const T *)a.dt + s * a.dt_ss + dd;
    const T *z = a.z ? (const T *)a.z + s * a.z_ss + dd : nullptr;
    const int64_t bc = s * a.bc_ss + (int64_t)(dd / a.per_group) * a.N + n0;
    const T *B = (const T *)a.B + bc, *C = (const T *)a.C + bc;
    T *y = (T *)a.y + s * a.y_ss + dd;
    for (int t = 0; t < len; ++t) {
        float b[4], c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = c[j] = 0.0f;
        if (V4) {
            if (n0 < a.N) {
                const nb::Vec<T, 4> tb = *(const nb::Vec<T, 4> *)(B + (int64_t)t * a.bc_ld), tc = *(const nb::Vec<T, 4> *)(C + (int64_t)t * a.bc_ld);
#pragma unroll
                for (int j = 0; j < 4; ++j) { b[j] = nb::to_f32(tb.v[j]); c[j] = nb::to_f32(tc.v[j]); }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < a.N) { b[j] = nb::to_f32(B[(int64_t)t * a.bc_ld + j]); c[j] = nb::to_f32(C[(int64_t)t * a.bc_ld + j]); }
        }
        const float xv = nb::to_f32(x[(int64_t)t * a.x_ld]);
        float step = nb::to_f32(dt[(int64_t)t * a.dt_ld]) + bias;
        if (a.softplus) step = softplus_f(step);
        const float sx = step * xv;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = fmaf(exp2f(step * A2[j]), h[j], sx * b[j]);
            sum = fmaf(h[j], c[j], sum);
        }
#pragma unroll
        for (int o = LPC / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (on && lane % LPC == 0) {
            float v = fmaf(skip, xv, sum);
            if (z) {
                const float zv = nb::to_f32(z[(int64_t)t * a.z_ld]);
                v *= zv * nb::sigmoid_fast(zv);
            }
            y[(int64_t)t * a.y_ld] = nb::from_f32<T>(v);
        }
    }
    if (a.state_out && on) {
        if (V4) {
            if (n0 < a.N) *(float4 *)(a.state_out + sat) = make_float4(h[0], h[1], h[2], h[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < a.N) a.state_out[sat + j] = h[j];
        }
    }
}

template <typename T, int LPC, bool V4>
int run(ScanArgs a, cudaStream_t st) {
    a.wps = (a.D * LPC + 31) / 32;
    a.warps = (int64_t)a.streams * a.wps;
    const int64_t blocks = (a.warps * 32 + NT - 1) / NT;
    if (blocks > 0x7fffffff) return nb_set_error("nemo_selective_scan: too many streams");
    nb::launch(selective_scan_kernel<T, LPC, V4>, dim3((unsigned)blocks), NT, 0, st, a);
    return nb_check_launch("selective_scan_kernel");
}

template <typename T, bool V4>
int by_states(const ScanArgs &a, cudaStream_t st) {
    if (a.N <= 4) return run<T, 1, V4>(a, st);
    if (a.N <= 8) return run<T, 2, V4>(a, st);
    if (a.N <= 16) return run<T, 4, V4>(a, st);
    if (a.N <= 32) return run<T, 8, V4>(a, st);
    if (a.N <= 64) return run<T, 16, V4>(a, st);
    return run<T, 32, V4>(a, st);
}

}  // namespace

extern "C" int nemo_selective_scan(const nemo_selective_scan_args_t *p, void *stream) {
    if (!p) return nb_set_error("nemo_selective_scan: null arguments");
    if (p->streams < 0 || p->c < 0 || p->D < 0 || p->D > (1 << 24))
        return nb_set_error("nemo_selective_scan: bad shape streams=%d c=%d D=%d", p->streams, p->c, p->D);
    if (p->N < 1 || p->N > 128) return nb_set_error("nemo_selective_scan: N=%d outside 1..128", p->N);
    if (p->groups < 1 || p->D % p->groups) return nb_set_error("nemo_selective_scan: D=%d is not a multiple of groups=%d", p->D, p->groups);
    if (!nb::elt_ok(p->elt)) return nb_set_error("nemo_selective_scan: unknown element type %d", p->elt);
    if (p->streams == 0 || p->D == 0 || (p->c == 0 && !p->state_out)) return 0;
    if (!p->A || (p->c > 0 && (!p->x || !p->dt || !p->B || !p->C || !p->y))) return nb_set_error("nemo_selective_scan: null pointer");
    if (p->c > 1 && (p->x_ld < p->D || p->dt_ld < p->D || p->y_ld < p->D || (p->z && p->z_ld < p->D) || p->bc_ld < (int64_t)p->groups * p->N))
        return nb_set_error("nemo_selective_scan: row pitches below the row's elements");
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
    NB_ELT_SWITCH(p->elt, T, rc = v4 ? by_states<T, true>(a, st) : by_states<T, false>(a, st));
    return rc;
}

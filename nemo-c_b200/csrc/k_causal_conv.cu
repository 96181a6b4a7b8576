// Causal depthwise convolution with carried history, for prompts, chunks and single rows.
//
// y[t][d] = act(bias[d] + sum_j w[d][j] u[t + j]) over u = (taps - 1 history rows, x rows). Bound by
// HBM: each element is read and written once (2 taps + 4 operations on it). A thread owns four
// neighbouring channels for a run of rows and slides a window of taps rows through registers, so a row
// is loaded once per run; the taps - 1 rows before the run come from the history or from the rows that
// the run before it owns (L1/L2). The rows of a stream are cut into runs until the threads fill the GPU.
//
// 32767 x 2048 bf16 rows, 4 taps: 48.6 us (5.5 TB/s, 0.84 of the measured copy rate). What it took: eight
// channels a thread 110 us (134 registers, 12 warps an SM), four 84 us; the weights as vectors 78 us;
// rows on their way in shared memory 48.6 us (3 or 6 groups of them: 55 us).
#include "elt.cuh"

namespace {

constexpr int NT = 128;
constexpr int R = 4, Q = 4;  // rows per group, groups of rows in the ring

struct ConvArgs {
    const void *x;
    int64_t x_ld, x_ss;
    const float *w, *bias;
    const void *hist_in;
    void *hist_out, *y;
    int64_t y_ld, y_ss;
    const int *lens;
    int64_t items;  // (stream, run, channel group), the last fastest
    int c, D, groups, runs, run_rows, act;
};

// V channels of a row: as they are loaded, and as pairs of fp32 (V = 1: a pair with an idle half)
template <typename T, int V>
__device__ __forceinline__ void widen(const nb::Vec<T, V> &t, nb::f2 (&o)[(V + 1) / 2]) {
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) o[i] = nb::pack2(nb::to_f32(t.v[2 * i]), 2 * i + 1 < V ? nb::to_f32(t.v[2 * i + 1 < V ? 2 * i + 1 : 0]) : 0.0f);
}

template <int BYTES>
__device__ __forceinline__ void cp_async(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "n"(BYTES) : "memory");
}

template <typename T, int V, int TAPS>
__global__ void __launch_bounds__(NT) causal_conv_kernel(const __grid_constant__ ConvArgs a) {
    constexpr int P = (V + 1) / 2;
    typedef nb::Vec<T, V> Row;
    constexpr bool AHEAD = V == 4;  // (single elements are too small for asynchronous copies)
    __shared__ Row ring[AHEAD ? Q * R : 1][NT];
    nb::pdl_wait();
    const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
    if (i >= a.items) return;
    int64_t s;
    int run, g;
    if (a.items <= 0xffffffffLL) {  // (a 64-bit division is a hundred instructions)
        const uint32_t sr = (uint32_t)i / (uint32_t)a.groups, su = sr / (uint32_t)a.runs;
        g = (int)((uint32_t)i - sr * a.groups);
        run = (int)(sr - su * a.runs);
        s = su;
    } else {
        const int64_t sr = i / a.groups;
        g = (int)(i - sr * a.groups);
        s = sr / a.runs;
        run = (int)(sr - s * a.runs);
    }
    const int d = g * V;
    const int len = a.lens ? max(0, min(a.lens[s], a.c)) : a.c;
    const int t0 = run * a.run_rows, t1 = min(len, t0 + a.run_rows);
    if (t0 >= t1 && run) return;
    const T *x = (const T *)a.x + s * a.x_ss + d;
    const int64_t hs = s * (TAPS - 1) * (int64_t)a.D + d;
    const T *hist = a.hist_in ? (const T *)a.hist_in + hs : nullptr;
    // row t of u without the offset: a history row for t < 0
    auto row = [&](int t) __attribute__((always_inline)) {
        Row o;
        if (t >= 0) {
            o = *(const Row *)(x + (int64_t)t * a.x_ld);
        } else if (hist) {
            o = *(const Row *)(hist + (int64_t)(t + TAPS - 1) * a.D);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) o.v[k] = nb::from_f32<T>(0.0f);
        }
        return o;
    };
    if (t0 < t1) {
        // Rows on their way wait in shared memory, in slots of the thread that asked for them (no barrier):
        // Q - 1 groups of R rows. In registers four rows a thread were the most, and HBM half idle.
        const T *px = x + (int64_t)t0 * a.x_ld;
        const int whole = AHEAD ? (t1 - t0) / R : 0;  // groups of R rows
        auto fetch = [&](int f) __attribute__((always_inline)) {
            if constexpr (AHEAD) if (f < whole) {
                const T *q = px + (int64_t)f * R * a.x_ld;
#pragma unroll
                for (int r = 0; r < R; ++r) cp_async<sizeof(Row)>(&ring[(f % Q) * R + r][threadIdx.x], q + r * a.x_ld);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");  // an empty one too: the count tells which group has landed
        };
        if (AHEAD)
#pragma unroll
            for (int f = 0; f < Q - 1; ++f) fetch(f);
        nb::f2 win[TAPS][P], w[TAPS][P], b[P];  // the last TAPS rows, oldest first
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) widen<T, V>(row(t0 - (TAPS - 1) + j), win[j + 1]);
        // the weights of V channels lie together: TAPS vectors of four where a thread owns four channels
        // (loaded one by one they cost a warp 16 times the transactions)
        float wf[V * TAPS], bf[V];
        const float *wp = a.w + (int64_t)d * TAPS;
        if (V == 4) {
#pragma unroll
            for (int j = 0; j < TAPS; ++j) {
                const float4 q = ((const float4 *)wp)[j];
                wf[4 * j] = q.x; wf[4 * j + 1] = q.y; wf[4 * j + 2] = q.z; wf[4 * j + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V * TAPS; ++j) wf[j] = wp[j];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) bf[k] = a.bias ? a.bias[d + k] : 0.0f;
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const int k1 = 2 * k + 1 < V ? 2 * k + 1 : 2 * k;
            b[k] = nb::pack2(bf[2 * k], bf[k1]);
#pragma unroll
            for (int j = 0; j < TAPS; ++j) w[j][k] = nb::pack2(wf[2 * k * TAPS + j], wf[k1 * TAPS + j]);
        }
        T *y = (T *)a.y + s * a.y_ss + d + (int64_t)t0 * a.y_ld;
        auto put = [&](const Row &u) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < TAPS - 1; ++j)
#pragma unroll
                for (int k = 0; k < P; ++k) win[j][k] = win[j + 1][k];
            widen<T, V>(u, win[TAPS - 1]);
            Row o;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                nb::f2 v = b[k];
#pragma unroll
                for (int j = 0; j < TAPS; ++j) v = nb::fma2(w[j][k], win[j][k], v);
                if (a.act == NEMO_ACT_SILU) v = nb::mul2(v, nb::sigmoid2(v));
                float lo, hi;
                nb::unpack2(v, lo, hi);
                o.v[2 * k] = nb::from_f32<T>(lo);
                if (2 * k + 1 < V) o.v[2 * k + 1 < V ? 2 * k + 1 : 0] = nb::from_f32<T>(hi);
            }
            *(Row *)y = o;
            y += a.y_ld;
        };
        for (int f = 0; f < whole; ++f) {
            asm volatile("cp.async.wait_group %0;" ::"n"(Q - 2) : "memory");
            Row cur[R];
#pragma unroll
            for (int r = 0; r < R; ++r) cur[r] = ring[(f % Q) * R + r][threadIdx.x];
            fetch(f + Q - 1);  // into the slots of group f - 1
#pragma unroll
            for (int r = 0; r < R; ++r) put(cur[r]);
        }
        px += (int64_t)whole * R * a.x_ld;
        for (int t = t0 + whole * R; t < t1; ++t, px += a.x_ld) put(*(const Row *)px);
    }
    // The thread that reads these channels' history rows replaces them, so both may be one buffer.
    if (TAPS > 1 && a.hist_out && run == 0) {
        T *h = (T *)a.hist_out + hs;
        Row last[TAPS > 1 ? TAPS - 1 : 1];
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) last[j] = row(len - (TAPS - 1) + j);
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) *(Row *)(h + (int64_t)j * a.D) = last[j];
    }
}

template <typename T, int V, int TAPS>
int run(ConvArgs a, const nemo_causal_conv_args_t *p, cudaStream_t st) {
    a.groups = p->D / V;
    // runs of at least 8 rows (the window's taps - 1 rows are read again for each), and no more of
    // them than fill the GPU's 148 x 2048 threads
    const int64_t base = (int64_t)p->streams * a.groups;
    int64_t runs = (148 * 2048 + base - 1) / base;
    runs = runs < 1 ? 1 : runs;
    int64_t rows = (p->c + runs - 1) / runs;
    rows = rows < 8 ? 8 : rows;
    a.run_rows = (int)rows;
    a.runs = p->c > 0 ? (int)((p->c + rows - 1) / rows) : 1;  // without rows only the history moves
    a.items = base * a.runs;
    const int64_t blocks = (a.items + NT - 1) / NT;
    if (blocks > 0x7fffffff) return nb_set_error("nemo_causal_conv: too many rows");
    nb::launch(causal_conv_kernel<T, V, TAPS>, dim3((unsigned)blocks), NT, 0, st, a);
    return nb_check_launch("causal_conv_kernel");
}

template <typename T, int V>
int by_taps(const ConvArgs &a, const nemo_causal_conv_args_t *p, cudaStream_t st) {
    switch (p->taps) {
        case 1: return run<T, V, 1>(a, p, st);
        case 2: return run<T, V, 2>(a, p, st);
        case 3: return run<T, V, 3>(a, p, st);
        case 4: return run<T, V, 4>(a, p, st);
        case 5: return run<T, V, 5>(a, p, st);
        case 6: return run<T, V, 6>(a, p, st);
        case 7: return run<T, V, 7>(a, p, st);
        default: return run<T, V, 8>(a, p, st);
    }
}

}  // namespace

extern "C" int nemo_causal_conv(const nemo_causal_conv_args_t *p, void *stream) {
    if (!p) return nb_set_error("nemo_causal_conv: null arguments");
    if (p->streams < 0 || p->c < 0 || p->c > (1 << 30) || p->D < 0) return nb_set_error("nemo_causal_conv: bad shape streams=%d c=%d D=%d", p->streams, p->c, p->D);
    if (p->taps < 1 || p->taps > 8) return nb_set_error("nemo_causal_conv: taps=%d outside 1..8", p->taps);
    if (!nb::elt_ok(p->elt)) return nb_set_error("nemo_causal_conv: unknown element type %d", p->elt);
    if (p->act != NEMO_ACT_NONE && p->act != NEMO_ACT_SILU) return nb_set_error("nemo_causal_conv: activation %d is neither none nor silu", p->act);
    if (p->streams == 0 || p->D == 0) return 0;
    if (!p->w || (p->c > 0 && (!p->x || !p->y))) return nb_set_error("nemo_causal_conv: null pointer");
    if (p->c > 1 && (p->x_ld < p->D || p->y_ld < p->D)) return nb_set_error("nemo_causal_conv: row pitches below D=%d", p->D);
    // (with lens the rows written are known on the device alone: one row a stream is looked at, then)
    if (nb_rows_overlap(p->streams, p->y_sstride, p->lens && p->c > 1 ? 1 : p->c, p->y_ld, p->D))
        return nb_set_error("nemo_causal_conv: rows of y overlap (y_sstride=%lld)", (long long)p->y_sstride);
    const int es = nb::elt_size(p->elt);
    const uintptr_t ptrs = (uintptr_t)p->x | (uintptr_t)p->y | (uintptr_t)p->hist_in | (uintptr_t)p->hist_out;
    if (ptrs % es || ((uintptr_t)p->w | (uintptr_t)p->bias) % 4) return nb_set_error("nemo_causal_conv: buffers must be aligned to their type");
    if (p->c == 0 && !p->hist_out) return 0;
    ConvArgs a = {};
    a.x = p->x; a.x_ld = p->x_ld; a.x_ss = p->x_sstride;
    a.w = p->w; a.bias = p->bias;
    a.hist_in = p->hist_in; a.hist_out = p->hist_out;
    a.y = p->y; a.y_ld = p->y_ld; a.y_ss = p->y_sstride;
    a.lens = p->lens; a.c = p->c; a.D = p->D; a.act = p->act;
    const int V = 4;
    const bool vec = p->D % V == 0 && ptrs % (V * es) == 0 && (uintptr_t)p->w % 16 == 0 && ((p->x_ld | p->y_ld | (p->streams > 1 ? p->x_sstride | p->y_sstride : 0)) % V) == 0;
    int rc = 0;
    cudaStream_t st = (cudaStream_t)stream;
    NB_ELT_SWITCH(p->elt, T, rc = vec ? by_taps<T, 4>(a, p, st) : by_taps<T, 1>(a, p, st));
    return rc;
}

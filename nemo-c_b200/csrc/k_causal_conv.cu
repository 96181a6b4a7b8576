// Causal depthwise convolution with carried history, for prompts, chunks and single rows.
//
// y[t][d] = act(bias[d] + sum_j w[d][j] u[t + j]) over u = (taps - 1 history rows, x rows). Bound by
// HBM: each element is read and written once (2 taps + 4 operations on it). A thread owns V
// neighbouring channels (16 bytes of a row) for a run of rows and slides a window of taps rows through
// registers, so a row is loaded once per run; the taps - 1 rows before the run come from the history
// or from the rows that the run before it owns (L1/L2). The rows of a stream are cut into runs until
// the threads fill the GPU.
#include "elt.cuh"

namespace {

constexpr int NT = 128;

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

template <typename T, int V>
__device__ __forceinline__ void load(float (&o)[V], const T *p) {
    const nb::Vec<T, V> t = *(const nb::Vec<T, V> *)p;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = nb::to_f32(t.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store(T *p, const float (&v)[V]) {
    nb::Vec<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) t.v[i] = nb::from_f32<T>(v[i]);
    *(nb::Vec<T, V> *)p = t;
}

template <typename T, int V, int TAPS>
__global__ void __launch_bounds__(NT) causal_conv_kernel(const __grid_constant__ ConvArgs a) {
    nb::pdl_wait();
    const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
    if (i >= a.items) return;
    const int64_t sr = i / a.groups;
    const int g = (int)(i - sr * a.groups);
    const int64_t s = sr / a.runs;
    const int run = (int)(sr - s * a.runs), d = g * V;
    const int len = a.lens ? max(0, min(a.lens[s], a.c)) : a.c;
    const int t0 = run * a.run_rows, t1 = min(len, t0 + a.run_rows);
    if (t0 >= t1 && run) return;
    const T *x = (const T *)a.x + s * a.x_ss + d;
    const int64_t hs = s * (TAPS - 1) * (int64_t)a.D + d;
    const T *hist = a.hist_in ? (const T *)a.hist_in + hs : nullptr;
    // row t of u without the offset: a history row for t < 0
    auto row = [&](int t, float (&o)[V]) {
        if (t >= 0)
            load<T, V>(o, x + (int64_t)t * a.x_ld);
        else if (hist)
            load<T, V>(o, hist + (int64_t)(t + TAPS - 1) * a.D);
        else
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = 0.0f;
    };
    float win[TAPS][V];  // the last TAPS rows, oldest first
#pragma unroll
    for (int j = 0; j < TAPS - 1; ++j) row(t0 - (TAPS - 1) + j, win[j + 1]);
    if (t0 < t1) {
        float w[TAPS][V], b[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            b[k] = a.bias ? a.bias[d + k] : 0.0f;
#pragma unroll
            for (int j = 0; j < TAPS; ++j) w[j][k] = a.w[(int64_t)(d + k) * TAPS + j];
        }
        T *y = (T *)a.y + s * a.y_ss + d;
        for (int t = t0; t < t1; ++t) {
            float o[V];
#pragma unroll
            for (int j = 0; j < TAPS - 1; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) win[j][k] = win[j + 1][k];
            load<T, V>(win[TAPS - 1], x + (int64_t)t * a.x_ld);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float v = b[k];
#pragma unroll
                for (int j = 0; j < TAPS; ++j) v = fmaf(w[j][k], win[j][k], v);
                o[k] = a.act == NEMO_ACT_SILU ? v * nb::sigmoid_fast(v) : v;
            }
            store<T, V>(y + (int64_t)t * a.y_ld, o);
        }
    }
    // The thread that reads these channels' history rows replaces them, so both may be one buffer.
    if (TAPS > 1 && a.hist_out && run == 0) {
        T *h = (T *)a.hist_out + hs;
        float last[TAPS > 1 ? TAPS - 1 : 1][V];
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) row(len - (TAPS - 1) + j, last[j]);
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) store<T, V>(h + (int64_t)j * a.D, last[j]);
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
    if (p->streams < 0 || p->c < 0 || p->D < 0) return nb_set_error("nemo_causal_conv: bad shape streams=%d c=%d D=%d", p->streams, p->c, p->D);
    if (p->taps < 1 || p->taps > 8) return nb_set_error("nemo_causal_conv: taps=%d outside 1..8", p->taps);
    if (!nb::elt_ok(p->elt)) return nb_set_error("nemo_causal_conv: unknown element type %d", p->elt);
    if (p->act != NEMO_ACT_NONE && p->act != NEMO_ACT_SILU) return nb_set_error("nemo_causal_conv: activation %d is neither none nor silu", p->act);
    if (p->streams == 0 || p->D == 0) return 0;
    if (!p->w || (p->c > 0 && (!p->x || !p->y))) return nb_set_error("nemo_causal_conv: null pointer");
    if (p->c > 1 && (p->x_ld < p->D || p->y_ld < p->D)) return nb_set_error("nemo_causal_conv: row pitches below D=%d", p->D);
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
    const int V = 16 / es;
    const bool vec = p->D % V == 0 && (ptrs & 15) == 0 && ((p->x_ld | p->y_ld | p->x_sstride | p->y_sstride) % V) == 0;
    int rc = 0;
    cudaStream_t st = (cudaStream_t)stream;
    NB_ELT_SWITCH(p->elt, T, rc = vec ? by_taps<T, 16 / sizeof(T)>(a, p, st) : by_taps<T, 1>(a, p, st));
    return rc;
}

/* nemo_gpu: C-ABI of the B200 kernels (sm_100a). Plain pointers and sizes; device pointers
   unless stated; `stream` is a cudaStream_t (NULL = legacy default stream). Every entry point
   returns 0 on success or -1 after recording a message retrievable with nemo_gpu_last_error().

   These replace the reference's string-keyed Metal dispatch (src/gpu.h:20-41, src/gpu.m) and the
   kernel launchers of src/model.h:71-76 plus the direct dispatches in src/encoder.c and
   src/decoder.c. The math of each entry point is that of the Metal kernel it cites.

   Devices: a process drives one GPU through these entry points (nemo_gemm's split-K workspace is
   allocated once, on the device current at its first call). Per-kernel shared-memory limits are
   kept per device, and nemo_gemm_noalloc keeps its set-up per device. */
#ifndef NEMO_GPU_H
#define NEMO_GPU_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { NEMO_ACT_NONE = 0, NEMO_ACT_SILU = 1, NEMO_ACT_RELU = 2, NEMO_ACT_GLU = 3 };
enum { NEMO_FMT_F32 = 0, NEMO_FMT_BF16X2 = 1 };

/* C[row(m)][n] (= or +=) alpha * act(sum_k A[m][k] * W[n][k] + bias[g][n]).
   Replaces k_gemm (src/model.h:71, src/model.c:70-99) and its kernels gemm_bf16 / gemm_spec /
   gemm_mma (src/kernels.metal:12-208); like k_gemm it picks the kernel by row count:
   M <= 16 streams the weights through CUDA cores; larger M runs tcgen05 tensor-core tiles.
   Row mapping (new: lets one launch cover many streams and write into per-stream caches):
   m -> group g = m / rpg, r = m % rpg; C element at C + g*gstride + (rowoff + r)*ldc + n,
   bias at bias + g*bias_gstride + n. rowoff is read from device memory (NULL = 0).
   A formats: NEMO_FMT_F32 (fp32 [M][lda]) or NEMO_FMT_BF16X2 (two bf16 planes, hi at A and
   lo = A - hi at A + a_plane elements; hi + lo carries 16 mantissa bits). The C output may
   also be written as NEMO_FMT_BF16X2 planes (c_plane apart) for a following tensor-core GEMM. */
typedef struct {
    const void *A;
    int64_t lda, a_plane;
    int a_fmt;
    const uint16_t *W;
    int64_t ldw;
    const float *bias;
    int64_t bias_gstride;
    void *C;
    int64_t ldc, c_plane;
    int c_fmt;
    int rpg;
    int64_t gstride;
    const int *rowoff;
    const int *dynM; /* if non-NULL: rows actually processed = min(M, *dynM), read on the device */
    int M, N, K;
    int act, accumulate;
    float alpha;
    float *c32;      /* optional: also write the fp32 value at c32[m * ldc32 + n] (dense rows) */
    int64_t ldc32;
} nemo_gemm_args_t;
int nemo_gemm(const nemo_gemm_args_t *a, void *stream);
/* Force a kernel family for tests and the kernel sweep: 0 = by row count (default),
   1 = CUDA-core weight streaming, 2 = tcgen05 tensor cores (tile layout by row count),
   3 = CUDA-core tiled, 4 = tensor cores with weight-major tiles (weights on the MMA's 128-row
   side), 5 = tensor cores with activation-major tiles (128 activation rows x 128/256 weights),
   6 = activation-major tiles scheduled stream-K (every CTA an equal share of the k-blocks of all
   tiles; kind 5's plan when the row count is dynamic). */
int nemo_gemm_forced(const nemo_gemm_args_t *a, int kind, void *stream);
/* Allocation-free tensor-core GEMM (no counterpart in the reference, whose Metal GEMMs need no
   split-K scratch). Same arguments and results as nemo_gemm for NEMO_FMT_BF16X2 activations of
   1..32 rows; its split-K scratch is a fixed 5 MiB array inside the library, so it never
   allocates device memory. For hosts that cannot allocate once running: a real-time audio
   callback driving one stream (cudaMalloc may synchronize the device) and servers that reserve
   their device memory up front. It makes nemo_gemm's checks (null pointers, shape, GLU with an
   odd N, accumulate into a non-fp32 output; M = 0 does nothing) and returns -1 with
   nemo_gpu_last_error() set for more rows, other activation formats, or a plan that would exceed
   the scratch. The first call on each device (that device current) does the set-up, including a
   blocking clear of the split-K arrival counters; make it before any stream capture. Later calls
   clear nothing (the kernel leaves the counters at zero) unless nemo_gpu_check_device_errors has
   reported a failed device wait since, in which case the next call clears them again, blocking.
   Calls on one device share the scratch: calls that overlap in time race and must be serialized
   on one stream. */
int nemo_gemm_noalloc(const nemo_gemm_args_t *a, void *stream);

/* Row LayerNorm. Replaces k_layernorm (src/model.h:73; kernel src/kernels.metal:258-288).
   Y may be written as NEMO_FMT_BF16X2 planes (y_plane apart) for a tensor-core consumer. */
int nemo_layernorm(const float *X, const float *g, const float *b, void *Y, int y_fmt, int64_t y_plane,
                   int M, int D, float eps, void *stream);
/* Y1 = LN(X; g1, b1), Y2 = LN(Y1; g2, b2). Replaces k_layernorm2 (src/model.h:72; kernel
   src/kernels.metal:212-255). Y1 is fp32; Y2 may be BF16X2 planes. */
int nemo_layernorm2(const float *X, const float *g1, const float *b1, const float *g2, const float *b2,
                    float *Y1, void *Y2, int y2_fmt, int64_t y2_plane, int M, int D, float eps, void *stream);

/* Relative-position attention over a K/V cache window for `streams` independent streams.
   Replaces the attention_rel dispatch (src/encoder.c:161-165; kernel src/kernels.metal:293-348).
   Per stream s: queries are rows [*pos, *pos + c) of Q + s*q_sstride ([.][ldq]); keys/values
   rows [*pos - *cache_len, *pos + c) of K + s*kv_sstride / V + s*kv_sstride ([.][ldk]), so
   L = *cache_len + c (<= Lmax); pos and cache_len are read from device ints. P: [2*Lmax-1][D] position table. Output
   O + s*o_sstride ([c][D]) as fp32 or BF16X2 planes (o_plane apart). Limits: head dim 128, c <= 16,
   Lmax <= 96; Q, K, V, P, bias_u and bias_v 16-byte aligned; ldq, ldk, q_sstride, kv_sstride and D
   multiples of 4 floats (an error otherwise). */
int nemo_attention_rel(const float *Q, int64_t ldq, int64_t q_sstride, const float *K, const float *V, int64_t ldk,
                       int64_t kv_sstride, const int *pos, const int *cache_len, const float *P, const float *bias_u,
                       const float *bias_v, void *O, int o_fmt, int64_t o_plane, int64_t o_sstride,
                       int streams, int c, int Lmax, int H, int dh, int D, float scale, void *stream);

/* Causal depthwise conv (taps rows, history in place) + LayerNorm + SiLU, `streams` streams.
   Replaces the dwconv_ln_silu dispatch (src/encoder.c:172-174; kernel src/kernels.metal:361-409).
   din rows for stream s start at din + s*din_sstride + (*pos - (taps-1))*D. */
int nemo_dwconv_ln_silu(const float *din, int64_t din_sstride, const int *pos, const float *W, const float *g,
                        const float *b, void *Y, int y_fmt, int64_t y_plane, int streams, int c, int D, int taps,
                        float eps, void *stream);

/* 1 -> C channel 3x3 stride-2 conv + ReLU, causal padding, `streams` windows of [T][F] each
   (x_sstride apart). Replaces conv2d_c1_s2_relu (src/kernels.metal:413-432). Y: [s][T1][F1][C]. */
int nemo_conv2d_c1_s2_relu(const float *X, int64_t x_sstride, const float *W, const float *bias, float *Y,
                           int streams, int T, int F, int T1, int F1, int C, void *stream);
/* The first two subsampling stages in one pass: conv2d_c1_s2_relu followed by dwconv2d_s2
   (src/encoder.c:125-130), without the intermediate [T1][F1][C] map. X: `streams` windows of
   [T][F] (x_sstride apart); Y: [s][T2][F2][C] as fp32 or bf16 planes (y_plane apart). */
int nemo_subsample_front(const float *X, int64_t x_sstride, const float *W0, const float *b0, const float *W2, const float *b2, void *Y,
                         int y_fmt, int64_t y_plane, int streams, int T, int F, int C, void *stream);
/* Depthwise 3x3 stride-2 conv. Replaces dwconv2d_s2 (src/kernels.metal:435-454). X [s][T][F][C]. */
int nemo_dwconv2d_s2(const float *X, const float *W, const float *bias, float *Y, int streams, int T, int F,
                     int T1, int F1, int C, void *stream);
/* Gather rows [*lo, *lo + c) of each stream's [T][F][C] map and flatten them channel-major into
   [s*c][C*F] fp32 (flatten_cf, src/kernels.metal:457-462, restricted to the rows the chunk keeps
   at src/encoder.c:258). */
int nemo_flatten_rows(const float *X, float *Y, const int *lo, int streams, int T, int F, int C, int c, void *stream);

/* Log-mel frames (the transform of src/mel.c:115-173: Hann(400) centred in 512 points,
   double-precision FFT, power, 128 Slaney filters, log(x + 2^-24)) of `streams` sample spans:
   frame f of stream s reads span[s * span_stride + f * 160 .. + 512) (pre-emphasised samples,
   already reflected at the stream edges) and goes to out[s * out_stride + f * 128 ..]. */
int nemo_logmel_frames(const float *span, int64_t span_stride, int streams, int nframes, float *out, int64_t out_stride, void *stream);

/* Sample-rate conversion of `streams` streams at once: outputs [out0, out0 + count) of the
   windowed-sinc resampler of src/resample.c:34-82 (the sums of produce(), src/resample.c:52-71;
   the host keeps the FIFO bookkeeping). Output j is sum_k h(k - j r) x[k] / sum_k h(k - j r),
   r = in_rate / out_rate, over ceil(j r - half) <= k <= floor(j r + half), with x zero outside
   [0, nin). Row s of `in` (in_ld apart) holds input samples [in_start, in_start + in_len) of
   stream s, which must include every k in [0, nin) the outputs reach; output j of stream s goes
   to out[s * out_ld + j - out0]. Rates up to about 20x the output rate (shared-memory bound). */
int nemo_resample(const float *in, int64_t in_ld, int64_t in_start, int64_t in_len, int64_t nin, int64_t out0, int count, int in_rate,
                  int out_rate, float *out, int64_t out_ld, int streams, void *stream);

/* LSTM cell on gates [rows][4H] (i, f, g, o). Replaces lstm_cell (src/kernels.metal:475-486). */
int nemo_lstm_cell(const float *gates, const float *c_in, float *c_out, float *h_out, int rows, int H, void *stream);
/* Joint + argmax per row: logits = W . relu(enc[r] + pred[r]) + b (W bf16 [V][H]); ties ->
   lowest index. out_idx[r], out_val[r]. Replaces joint_partial + argmax_reduce
   (src/kernels.metal:490-550, dispatched at src/decoder.c:81-90). enc row r at enc + r*enc_ld,
   pred row r at pred + r*pred_ld (pred_ld 0 = one shared prediction vector). */
int nemo_joint_argmax(const float *enc, int64_t enc_ld, const float *pred, int64_t pred_ld, const uint16_t *W,
                      const float *bias, int V, int H, int rows, int *out_idx, float *out_val, void *stream);

/* ---- operators of streaming state-space layers -------------------------------------------------
   The reference has none of these: they serve layers, built by the caller, whose projections are held
   in 4 bits and whose sequence mixer carries a fixed state (causal convolution + selective scan)
   instead of a K/V window; nemoasr_open reads no such checkpoints. Activations may be fp32, bf16 or
   fp16 (NEMO_ELT_*); sums and states are fp32 and a value is rounded once, to nearest even, where it
   is stored. Values, small tensors and states need the alignment of their type; rows whose base and
   pitch are 16-byte aligned are moved 16 bytes at a time. Buffers that are written must not overlap
   others unless stated. Nothing is allocated and nothing synchronises; calls may be captured into graphs and may run on several streams at once. */
enum { NEMO_ELT_F32 = 0, NEMO_ELT_BF16 = 1, NEMO_ELT_F16 = 2 };

/* MXFP4 rows. A block is 32 consecutive columns of a row; its scale is 2^e with e = floor(log2 of
   its largest magnitude) - 2, not below 2^-127, held as the byte e + 127; a value is its e2m1 code
   (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times the scale, rounded to nearest, ties to the
   even code, beyond 6 to 6. A block that holds an infinity or a NaN gets the byte 255 (NaN) and zero
   codes. Codes: two a byte, the even column in the low nibble, rows ldq bytes apart. Scales: tiles
   of 128 rows x 4 blocks, byte (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4 of tile
   (r / 128) * ceil(K / 128) + b / 4 for row r and block b; nemo_mxfp4_scale_bytes(rows, K) bytes.
   The quantiser writes the bytes of its rows (those of a last, partly filled tile of columns as 0)
   and leaves the bytes of rows past the last one alone. K: a multiple of 32. */
int64_t nemo_mxfp4_scale_bytes(int64_t rows, int64_t K);
int nemo_mxfp4_quantize(const void *X, int x_elt, int64_t ldx, int64_t rows, int64_t K, uint8_t *codes, int64_t ldq, uint8_t *scales, void *stream);
/* The values that codes and scales stand for (rounded to y_elt; a NaN scale gives NaN). */
int nemo_mxfp4_dequantize(const uint8_t *codes, int64_t ldq, const uint8_t *scales, int64_t rows, int64_t K, void *Y, int y_elt, int64_t ldy, void *stream);

/* C[m][n] (= or +=) alpha * act(sum_k A[m][k] W[n][k] + bias[n]) for MXFP4 rows A [M][K] and W [N][K]
   on the block-scaled tensor cores: products are exact, sums fp32. The epilogue is nemo_gemm's: bias
   -> act -> alpha -> store or accumulate (fp32 C only); NEMO_ACT_GLU pairs columns n and n + N/2 into
   N/2 outputs, a * sigmoid(b), and needs N to be a multiple of 256. K: a positive multiple of 32; M, N and
   K up to 2^30. Codes, scales and code pitches 16-byte aligned. Scale bytes of the columns past K must not be 255 (the
   quantiser writes 0); those of the rows past M or N may hold anything. */
typedef struct {
    const uint8_t *A;
    int64_t lda;              /* bytes */
    const uint8_t *a_scales;
    const uint8_t *W;
    int64_t ldw;              /* bytes */
    const uint8_t *w_scales;
    const float *bias;        /* [N] or NULL */
    void *C;
    int64_t ldc;              /* elements */
    int c_elt;
    int M, N, K;
    int act, accumulate;
    float alpha;
} nemo_gemm_mxfp4_args_t;
int nemo_gemm_mxfp4(const nemo_gemm_mxfp4_args_t *a, void *stream);

/* Causal depthwise convolution over the rows of `streams` independent streams, with carried history:
   y[t][d] = act(bias[d] + sum_j w[d][j] * u[t + j]), u = the taps - 1 history rows, then the x rows.
   Stream s has lens[s] rows (device ints, taken into 0..c; NULL: c each); rows of y behind its last
   one are left as they were. hist_in [streams][taps-1][D] (NULL: zeros) holds the rows before this
   call's, hist_out the last taps - 1 rows of u after it (NULL: not kept); they may be the same
   buffer. Rows of y must not overlap (refused where it shows: c rows a stream, or with lens one).
   taps 1..8, c up to 2^30; act NEMO_ACT_NONE or NEMO_ACT_SILU. One row per stream is the single-token form. */
typedef struct {
    const void *x;
    int64_t x_ld, x_sstride;
    const float *w;           /* [D][taps] */
    const float *bias;        /* [D] or NULL */
    const void *hist_in;
    void *hist_out;
    void *y;
    int64_t y_ld, y_sstride;
    const int *lens;
    int streams, c, D, taps;
    int elt;                  /* of x, y and the history */
    int act;
} nemo_causal_conv_args_t;
int nemo_causal_conv(const nemo_causal_conv_args_t *a, void *stream);

/* Selective state-space scan over the rows of `streams` independent streams, with carried state.
   With step = dt[t][d] + dt_bias[d] (softplus of it where dt_softplus) and group g = d / (D / groups):
     h[d][n] = exp(step * A[d][n]) * h[d][n] + step * x[t][d] * B[t][g][n]
     y[t][d] = (sum_n h[d][n] * C[t][g][n] + skip[d] * x[t][d]) * silu(z[t][d])
   z, skip and dt_bias may be NULL (no gate, 0, 0). Rows of B and C hold groups * N elements. Stream s
   has lens[s] rows (device ints, taken into 0..c; NULL: c each); rows of y behind its last one are
   left as they were. state_in [streams][D][N] (NULL: zeros), state_out the state after the last row
   (of no rows: the state before; NULL: not kept); they may be the same buffer. Rows of y must not
   overlap (refused where it shows: c rows a stream, or with lens one). N 1..128, D up to
   2^24 and a multiple of groups, c up to 2^30. x, dt, z, B and C rows behind a stream's last one are
   not used, but may be read. One row per stream is the single-token form. */
typedef struct {
    const void *x;
    int64_t x_ld, x_sstride;
    const void *dt;
    int64_t dt_ld, dt_sstride;
    const void *z;
    int64_t z_ld, z_sstride;
    const void *B;
    const void *C;
    int64_t bc_ld, bc_sstride;
    const float *A;           /* [D][N] */
    const float *skip;
    const float *dt_bias;
    int dt_softplus;
    const float *state_in;
    float *state_out;
    void *y;
    int64_t y_ld, y_sstride;
    const int *lens;
    int streams, c, D, N, groups;
    int elt;                  /* of x, dt, z, B, C and y */
} nemo_selective_scan_args_t;
int nemo_selective_scan(const nemo_selective_scan_args_t *a, void *stream);

const char *nemo_gpu_last_error(void);
/* 0 if no kernel has reported a device-side failure (a bounded wait that gave up instead of
   hanging); otherwise -1 with the message in nemo_gpu_last_error(). Synchronous (reads a flag);
   each failure is reported once. */
int nemo_gpu_check_device_errors(void);
/* Diagnostic: launch a wait that nothing completes, bounded by limit_cycles clock cycles, to show
   that a device wait which runs out returns an error status instead of hanging or trapping.
   kind 0 = the tensor-core kernels' mbarrier wait, kind 1 = the persistent kernels' grid barrier.
   The next nemo_gpu_check_device_errors (and the next nemoasr_feed / batch step, through err)
   reports it, once. The reference surfaces Metal command-buffer errors the same way through
   err/errlen (src/gpu.m:131-134); it has no such self-test. */
int nemo_gpu_wait_selftest(int kind, long long limit_cycles, void *stream);
/* Number of CUDA kernels this library has launched (directly or by graph launch) since load. */
uint64_t nemo_gpu_launch_count(void);

#ifdef __cplusplus
}
#endif
#endif

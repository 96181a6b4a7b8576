// Microscaled 4-bit rows (MXFP4): quantisation and its inverse.
//
// A block is 32 consecutive columns of a row. With m the block's largest magnitude the scale is
// the power of two 2^e, e = floor(log2 m) - 2 (two is the exponent of the format's largest value,
// 6 = 1.5 * 2^2), held as the byte e + 127 and not below 2^-127; each value is x / 2^e rounded to
// the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, larger magnitudes to 6) with
// its sign. x / 2^e is a multiplication by a power of two, exact wherever the code is not zero, so the
// codes are rounded once.
// A block that holds an infinity or a NaN has no such scale: its byte is 255 (the format's NaN)
// and its codes are zero, so every value of it reads back as NaN.
//
// Both kernels are bound by HBM (2.5 to 4.5 bytes moved per element, no reuse).
// 16384 x 4096 bf16: quantised in 33 us (5.1 TB/s, 0.78 of the measured copy rate; 40 us with eight columns a
// thread and single scale bytes), there and back in 65 us. A thread keeps 32 or 64 bytes on their way: 2048
// threads an SM cover HBM's latency.
#include "elt.cuh"
#include "mxfp4.cuh"

namespace {

constexpr int NT = 256;

// Eight values to eight codes, two a byte, the even column in the low nibble.
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// (row, column group) of group i of a row-major sequence with `per` groups a row
__device__ __forceinline__ void place(int64_t i, int64_t total, int per, int64_t &row, int &g) {
    if (total <= 0xffffffffLL) {
        const uint32_t r = (uint32_t)i / (uint32_t)per;
        row = r;
        g = (int)((uint32_t)i - r * (uint32_t)per);
    } else {
        row = i / per;
        g = (int)(i - row * per);
    }
}

// Two neighbouring lanes share a block, 16 columns each (32 or 64 bytes in flight a lane). TILES: K is a
// multiple of 128, so eight lanes always hold a row's four blocks of one scale tile, whose bytes are
// stored as one word. Lanes past the last group still take part in the exchange.
template <typename T, bool VEC, bool TILES>
__global__ void __launch_bounds__(NT) mxfp4_quantize_kernel(const T *X, int64_t ldx, int64_t groups, int gpr, uint8_t *Q, int64_t ldq, uint8_t *S) {
    nb::pdl_wait();
    const int kt = (gpr + 7) / 8;  // scale tiles along a row
    const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
    const bool live = i < groups;
    int64_t row;
    int g;
    place(live ? i : groups - 1, groups, gpr, row, g);
    const T *x = X + row * ldx + (int64_t)g * 16;
    float v[16];
    if (VEC) {
        constexpr int E = 16 / sizeof(T);
        nb::Vec<T, E> t[16 / E];
#pragma unroll
        for (int j = 0; j < 16 / E; ++j) t[j] = ((const nb::Vec<T, E> *)x)[j];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = nb::to_f32(t[j / E].v[j % E]);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = nb::to_f32(x[j]);
    }
    uint32_t top = 0;  // magnitudes compare as their bits; infinities and NaN are the largest
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const int ex = (int)(top >> 23);
    const bool bad = ex == 255;
    const int byte = bad ? 255 : max(ex - 2, 0);
    const float inv = bad ? 0.0f : __uint_as_float((uint32_t)(254 - byte) << 23);  // 2^(127 - byte), byte <= 252
    uint32_t codes[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = v[8 * k + j] * inv;
        codes[k] = bad ? 0u : pack8(w);
    }
    uint32_t word = (uint32_t)byte;
    if (TILES) {  // lane 8 m gathers the bytes of its own, the next, .. of four blocks
        word |= __shfl_down_sync(0xffffffffu, word, 2) << 8;
        word |= __shfl_down_sync(0xffffffffu, word, 4) << 16;
    }
    if (!live) return;
    uint8_t *q = Q + row * ldq + (int64_t)g * 8;
    if (VEC) {
        *(uint2 *)q = make_uint2(codes[0], codes[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = (uint8_t)(codes[j >> 2] >> (8 * (j & 3)));
    }
    if (TILES) {
        if ((g & 7) == 0) *(uint32_t *)(S + mxfp4::scale_at(row, g >> 1, kt)) = word;
    } else if ((g & 1) == 0) {
        uint8_t *s = S + mxfp4::scale_at(row, g >> 1, kt);
        *s = (uint8_t)byte;
        if (g + 2 == gpr)  // the row's last block: the rest of its tile reads as 2^-127
            for (int p = (g >> 1) % 4 + 1, o = 1; p < 4; ++p, ++o) s[o] = 0;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(NT) mxfp4_dequantize_kernel(const uint8_t *Q, int64_t ldq, const uint8_t *S, int64_t groups, int gpr, T *Y, int64_t ldy) {
    nb::pdl_wait();
    const int kt = (gpr + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
    if (i >= groups) return;
    int64_t row;
    int g;
    place(i, groups, gpr, row, g);
    const uint8_t *q = Q + row * ldq + (int64_t)g * 8;
    uint32_t codes[2];
    if (VEC) {
        const uint2 t = *(const uint2 *)q;
        codes[0] = t.x;
        codes[1] = t.y;
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) codes[k] = q[4 * k] | (uint32_t)q[4 * k + 1] << 8 | (uint32_t)q[4 * k + 2] << 16 | (uint32_t)q[4 * k + 3] << 24;
    }
    const float scale = mxfp4::scale_value(S[mxfp4::scale_at(row, g >> 1, kt)]);
    T *y = Y + row * ldy + (int64_t)g * 16;
    constexpr int E = 16 / sizeof(T);
    nb::Vec<T, E> o[16 / E];
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j / E].v[j % E] = nb::from_f32<T>(mxfp4::code_value(codes[j >> 3] >> (4 * (j & 7))) * scale);
    if (VEC) {
#pragma unroll
        for (int j = 0; j < 16 / E; ++j) ((nb::Vec<T, E> *)y)[j] = o[j];
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = o[j / E].v[j % E];
    }
}

int check(const char *what, const void *a, int elt, int64_t ld, int64_t rows, int64_t K, const void *q, int64_t ldq, const void *s) {
    if (rows < 0 || K < 0 || K > (1LL << 31) - 32) return nb_set_error("%s: bad shape rows=%lld K=%lld", what, (long long)rows, (long long)K);
    if (K % 32) return nb_set_error("%s: K=%lld must be a multiple of 32 (one scale per 32 columns)", what, (long long)K);
    if (!nb::elt_ok(elt)) return nb_set_error("%s: unknown element type %d", what, elt);
    if (rows == 0 || K == 0) return 0;
    if (!a || !q || !s) return nb_set_error("%s: null pointer", what);
    if (rows > 1 && (ld < K || ldq < K / 2)) return nb_set_error("%s: row pitches %lld and %lld are below %lld columns", what, (long long)ld, (long long)ldq, (long long)K);
    if ((uintptr_t)a % nb::elt_size(elt)) return nb_set_error("%s: values must be aligned to their type", what);
    return 0;
}

}  // namespace

extern "C" int64_t nemo_mxfp4_scale_bytes(int64_t rows, int64_t K) {
    return rows <= 0 || K <= 0 ? 0 : ((rows + 127) / 128) * ((K + 127) / 128) * 512;
}

extern "C" int nemo_mxfp4_quantize(const void *X, int x_elt, int64_t ldx, int64_t rows, int64_t K, uint8_t *codes, int64_t ldq, uint8_t *scales, void *stream) {
    if (check("nemo_mxfp4_quantize", X, x_elt, ldx, rows, K, codes, ldq, scales)) return -1;
    if (rows == 0 || K == 0) return 0;
    const int64_t groups = rows * (K / 16), blocks = (groups + NT - 1) / NT;
    if (blocks > 0x7fffffff) return nb_set_error("nemo_mxfp4_quantize: too many values");
    const bool vec = ((uintptr_t)X & 15) == 0 && (ldx * nb::elt_size(x_elt)) % 16 == 0 && ((uintptr_t)codes & 7) == 0 && ldq % 8 == 0;
    const bool tiles = K % 128 == 0 && ((uintptr_t)scales & 3) == 0;
    cudaStream_t st = (cudaStream_t)stream;
    NB_ELT_SWITCH(x_elt, T, {
        auto kernel = vec ? (tiles ? mxfp4_quantize_kernel<T, true, true> : mxfp4_quantize_kernel<T, true, false>)
                          : (tiles ? mxfp4_quantize_kernel<T, false, true> : mxfp4_quantize_kernel<T, false, false>);
        nb::launch(kernel, dim3((unsigned)blocks), NT, 0, st, (const T *)X, ldx, groups, (int)(K / 16), codes, ldq, scales);
    });
    return nb_check_launch("mxfp4_quantize_kernel");
}

extern "C" int nemo_mxfp4_dequantize(const uint8_t *codes, int64_t ldq, const uint8_t *scales, int64_t rows, int64_t K, void *Y, int y_elt, int64_t ldy,
                                     void *stream) {
    if (check("nemo_mxfp4_dequantize", Y, y_elt, ldy, rows, K, codes, ldq, scales)) return -1;
    if (rows == 0 || K == 0) return 0;
    const int64_t groups = rows * (K / 16), blocks = (groups + NT - 1) / NT;
    if (blocks > 0x7fffffff) return nb_set_error("nemo_mxfp4_dequantize: too many values");
    const bool vec = ((uintptr_t)Y & 15) == 0 && (ldy * nb::elt_size(y_elt)) % 16 == 0 && ((uintptr_t)codes & 7) == 0 && ldq % 8 == 0;
    cudaStream_t st = (cudaStream_t)stream;
    NB_ELT_SWITCH(y_elt, T, nb::launch(vec ? mxfp4_dequantize_kernel<T, true> : mxfp4_dequantize_kernel<T, false>, dim3((unsigned)blocks), NT, 0, st, codes, ldq,
                                       scales, groups, (int)(K / 16), (T *)Y, ldy));
    return nb_check_launch("mxfp4_dequantize_kernel");
}

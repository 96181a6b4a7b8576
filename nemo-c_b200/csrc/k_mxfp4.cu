// Microscaled 4-bit rows (MXFP4): quantisation and its inverse.
//
// A block is 32 consecutive columns of a row. With m the block's largest magnitude the scale is
// the power of two 2^e, e = floor(log2 m) - 2 (two is the exponent of the format's largest value,
// 6 = 1.5 * 2^2), held as the byte e + 127 and not below 2^-127; each value is x / 2^e rounded to
// the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, larger magnitudes to 6) with
// its sign. x / 2^e is an exact multiplication by a power of two, so the codes are rounded once.
// A block that holds an infinity or a NaN has no such scale: its byte is 255 (the format's NaN)
// and its codes are zero, so every value of it reads back as NaN.
//
// Both kernels are bound by HBM (2.03 to 6.03 bytes moved per element and no reuse).
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

// Four neighbouring lanes share a block, eight columns each. Lanes of a warp past the last column
// group still take part in the exchange.
template <typename T, bool VEC>
__global__ void __launch_bounds__(NT) mxfp4_quantize_kernel(const T *X, int64_t ldx, int64_t groups, int gpr, uint8_t *Q, int64_t ldq, uint8_t *S) {
    nb::pdl_wait();
    const int kt = (gpr + 15) / 16;  // scale tiles along a row
    const int64_t step = (int64_t)gridDim.x * NT;
    for (int64_t i0 = (int64_t)blockIdx.x * NT; i0 < groups; i0 += step) {
        const int64_t i = i0 + threadIdx.x;
        const bool live = i < groups;
        const int64_t ii = live ? i : groups - 1;
        int64_t row;
        int g;
        if (groups <= 0xffffffffLL) {
            const uint32_t r32 = (uint32_t)ii / (uint32_t)gpr;
            row = r32;
            g = (int)((uint32_t)ii - r32 * (uint32_t)gpr);
        } else {
            row = ii / gpr;
            g = (int)(ii - row * gpr);
        }
        const T *x = X + row * ldx + (int64_t)g * 8;
        float v[8];
        if (VEC) {
            constexpr int E = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 8 / E; ++j) {
                const nb::Vec<T, E> t = *(const nb::Vec<T, E> *)(x + j * E);
#pragma unroll
                for (int e = 0; e < E; ++e) v[j * E + e] = nb::to_f32(t.v[e]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = nb::to_f32(x[j]);
        }
        uint32_t top = 0;  // magnitudes compare as their bits; infinities and NaN are the largest
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = (int)(top >> 23);
        const bool bad = ex == 255;
        const int byte = bad ? 255 : max(ex - 2, 0);
        const float inv = bad ? 0.0f : __uint_as_float((uint32_t)(254 - byte) << 23);  // 2^(127 - byte), byte <= 252
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= inv;
        uint32_t codes = pack8(v);
        if (bad) codes = 0;
        if (live) {
            uint8_t *q = Q + row * ldq + (int64_t)g * 4;
            if (VEC) {
                *(uint32_t *)q = codes;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = (uint8_t)(codes >> (8 * j));
            }
            if ((g & 3) == 0) {
                uint8_t *s = S + mxfp4::scale_at(row, g >> 2, kt);
                *s = (uint8_t)byte;
                if (g + 4 == gpr)  // the row's last block: the rest of its tile reads as 2^-127
                    for (int p = (g >> 2) % 4 + 1, o = 1; p < 4; ++p, ++o) s[o] = 0;
            }
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(NT) mxfp4_dequantize_kernel(const uint8_t *Q, int64_t ldq, const uint8_t *S, int64_t groups, int gpr, T *Y, int64_t ldy) {
    nb::pdl_wait();
    const int kt = (gpr + 15) / 16;
    const int64_t step = (int64_t)gridDim.x * NT;
    for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < groups; i += step) {
        int64_t row;
        int g;
        if (groups <= 0xffffffffLL) {
            const uint32_t r32 = (uint32_t)i / (uint32_t)gpr;
            row = r32;
            g = (int)((uint32_t)i - r32 * (uint32_t)gpr);
        } else {
            row = i / gpr;
            g = (int)(i - row * gpr);
        }
        const uint8_t *q = Q + row * ldq + (int64_t)g * 4;
        uint32_t codes;
        if (VEC)
            codes = *(const uint32_t *)q;
        else
            codes = q[0] | (uint32_t)q[1] << 8 | (uint32_t)q[2] << 16 | (uint32_t)q[3] << 24;
        const float scale = mxfp4::scale_value(S[mxfp4::scale_at(row, g >> 2, kt)]);
        T *y = Y + row * ldy + (int64_t)g * 8;
        T o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = nb::from_f32<T>(mxfp4::code_value(codes >> (4 * j)) * scale);
        if (VEC) {
            constexpr int E = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 8 / E; ++j) *(nb::Vec<T, E> *)(y + j * E) = *(const nb::Vec<T, E> *)(o + j * E);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = o[j];
        }
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
    const int64_t groups = rows * (K / 8);
    const int64_t blocks = (groups + NT - 1) / NT;
    const int grid = (int)(blocks < 148 * 64 ? blocks : 148 * 64);
    const bool vec = ((uintptr_t)X & 15) == 0 && (ldx * nb::elt_size(x_elt)) % 16 == 0 && ((uintptr_t)codes & 3) == 0 && ldq % 4 == 0;
    cudaStream_t st = (cudaStream_t)stream;
    NB_ELT_SWITCH(x_elt, T, nb::launch(vec ? mxfp4_quantize_kernel<T, true> : mxfp4_quantize_kernel<T, false>, grid, NT, 0, st, (const T *)X, ldx, groups,
                                       (int)(K / 8), codes, ldq, scales));
    return nb_check_launch("mxfp4_quantize_kernel");
}

extern "C" int nemo_mxfp4_dequantize(const uint8_t *codes, int64_t ldq, const uint8_t *scales, int64_t rows, int64_t K, void *Y, int y_elt, int64_t ldy,
                                     void *stream) {
    if (check("nemo_mxfp4_dequantize", Y, y_elt, ldy, rows, K, codes, ldq, scales)) return -1;
    if (rows == 0 || K == 0) return 0;
    const int64_t groups = rows * (K / 8);
    const int64_t blocks = (groups + NT - 1) / NT;
    const int grid = (int)(blocks < 148 * 64 ? blocks : 148 * 64);
    const bool vec = ((uintptr_t)Y & 15) == 0 && (ldy * nb::elt_size(y_elt)) % 16 == 0 && ((uintptr_t)codes & 3) == 0 && ldq % 4 == 0;
    cudaStream_t st = (cudaStream_t)stream;
    NB_ELT_SWITCH(y_elt, T, nb::launch(vec ? mxfp4_dequantize_kernel<T, true> : mxfp4_dequantize_kernel<T, false>, grid, NT, 0, st, codes, ldq, scales, groups,
                                       (int)(K / 8), (T *)Y, ldy));
    return nb_check_launch("mxfp4_dequantize_kernel");
}

// The storage of MXFP4 rows, shared by the kernels that write and read it.
#pragma once
#include <stdint.h>

namespace mxfp4 {

// Scale bytes lie in tiles of 128 rows x 4 blocks (512 bytes), the tiles of 128 rows one after the
// other along the row (kt of them): inside a tile, byte (row % 32) * 16 + (row % 128 / 32) * 4 +
// block % 4. That is the order in which a tile goes to tensor memory (32 lanes of 16 bytes).
__host__ __device__ __forceinline__ int64_t scale_at(int64_t row, int block, int kt) {
    return ((row >> 7) * kt + (block >> 2)) * 512 + (int64_t)((row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3));
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
    return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fffffffu : byte << 23);
}

// The value of the code in the low four bits of c: sign, two exponent bits and one mantissa bit,
// moved to the top of an fp32 number of exponent field 0..3; 2^126 takes the difference of the
// exponent biases back (the subnormal codes 0 and 0.5 included).
__device__ __forceinline__ float code_value(uint32_t c) {
    return __uint_as_float((c & 7) << 22 | (c & 8) << 28) * 0x1p126f;
}

}  // namespace mxfp4

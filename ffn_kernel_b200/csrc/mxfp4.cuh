// MXFP4 on the device: blocks of 32 values along the contraction share one power of two 2^E, held as the
// byte E + 127 (255: the block holds an infinity or a NaN); a value is four bits, sign, two exponent bits
// and one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6.
//
//   E = clamp(floor(log2(max |x|)) - 2, -127, 127)     (the largest value lands in [4, 8))
//   q = x / 2^E rounded to the nearest of the eight magnitudes, ties to even, at most 6
//
// floor(log2) is the exponent field of the fp32 number and 1 / 2^E a power of two, so both steps are exact in
// fp32 and the only rounding is the one to four bits: any two implementations agree bit for bit.
//
// Storage of a [rows, cols] matrix: codes uint8 [rows, ld], two values a byte, the lower column in the low half,
// ld = 16 * ceil(cols / 32) bytes; scales uint8 in atoms of 128 rows x 4 blocks (512 bytes), the order in which
// tcgen05.cp moves them into tensor memory: atom [row / 128][block / 4], inside it byte
// (row % 32) * 16 + (row % 128 / 32) * 4 + block % 4.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace ffnk {

constexpr int kMxAtomBytes = 512;   // scales of 128 rows x 4 blocks

__host__ __device__ constexpr int64_t mx_code_ld(int64_t cols) { return (cols + 31) / 32 * 16; }
__host__ __device__ constexpr int64_t mx_k_atoms(int64_t cols) { return (cols + 127) / 128; }
__host__ __device__ constexpr int64_t mx_row_atoms(int64_t rows) { return (rows + 127) / 128; }

// byte offset of the four scales of (row, blocks 4 * k_atom ...)
__device__ __forceinline__ int64_t mx_scale_word(int64_t row, int64_t k_atom, int64_t k_atoms) {
  return ((row >> 7) * k_atoms + k_atom) * kMxAtomBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// bits of max |x| over a block (an integer maximum: a NaN is above infinity) -> scale byte
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t absmax_bits) {
  const int e = static_cast<int>(absmax_bits >> 23);       // E + 127 = e - 2, not below 0 (subnormal and zero blocks: 0)
  return e == 255 ? 255u : (e > 2 ? static_cast<uint32_t>(e - 2) : 0u);
}
// 1 / 2^E as a float; a block that is not finite gets 0 (its codes are 0)
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) {
  return byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23);
}
// 2^E as a float, byte 0 is the subnormal 2^-127
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(byte == 0u ? 0x00400000u : byte << 23);
}
// products that keep subnormal operands and results (this library is compiled with flush-to-zero fast math)
__device__ __forceinline__ float mul_keep_subnormals(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// max(|a|, |b|, |c|), a NaN if one of them is
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// eight scaled values -> eight codes, the first in the lowest four bits
__device__ __forceinline__ uint32_t mx_pack8(const float (&v)[8]) {
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
// eight values of a block -> eight codes: the one place where values are rounded to four bits.  inv: mx_inverse_scale(byte).
__device__ __forceinline__ uint32_t mx_round8(const float (&x)[8], uint32_t byte, float inv) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = mul_keep_subnormals(x[i], inv);
  return byte == 255u ? 0u : mx_pack8(v);
}
// eight codes -> eight values (exact in fp16)
__device__ __forceinline__ void mx_unpack8(uint32_t c, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(c));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// A lane holds 32 bytes of a row, one 256-bit load: 16 values of a 16-bit type (two lanes a block) or 8 of fp32 (four).
template <typename T> struct MxLane {
  static constexpr int values = 32 / sizeof(T);
  static constexpr int chunk = 32 * values;          // columns of one warp step
  static constexpr int lanes_per_block = 32 / values;
};
struct MxRaw {
  uint32_t w[8];
};

// Values c ... of a row; beyond `cols` zeros.  align: bytes the rows are aligned to (32, 16, or less).
template <typename T>
__device__ __forceinline__ MxRaw load_lane(const T* row, int c, int cols, int align) {
  MxRaw r;
  if (align >= 16 && c + MxLane<T>::values <= cols) {
    if (align >= 32) {
      asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
                   : "l"(row + c));
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + c)), b = __ldg(reinterpret_cast<const uint4*>(row + c) + 1);
      r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
      r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 2) {
        const int k = c + 2 * i;
        const uint32_t lo = k < cols ? reinterpret_cast<const unsigned short*>(row)[k] : 0u;
        const uint32_t hi = k + 1 < cols ? reinterpret_cast<const unsigned short*>(row)[k + 1] : 0u;
        r.w[i] = lo | hi << 16;
      } else {
        r.w[i] = c + i < cols ? reinterpret_cast<const uint32_t*>(row)[c + i] : 0u;
      }
    }
  }
  return r;
}

// bits of the lane's max |x| as fp32 (16-bit types: packed integer maxima of two values at a time, converted once)
template <typename T>
__device__ __forceinline__ uint32_t absmax_bits(const MxRaw& r) {
  constexpr uint32_t mask = sizeof(T) == 2 ? 0x7FFF7FFFu : 0x7FFFFFFFu;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 2) m = __vmaxu2(m, r.w[i] & mask);
    else m = max(m, r.w[i] & mask);
  }
  if constexpr (sizeof(T) == 2) m = max(m & 0xFFFFu, m >> 16);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
  else if constexpr (sizeof(T) == 2) return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
  else return m;
}

template <typename T>
__device__ __forceinline__ float raw_value(const MxRaw& r, int i) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? r.w[i >> 1] & 0xFFFF0000u : r.w[i >> 1] << 16);
  else if constexpr (sizeof(T) == 2) return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? r.w[i >> 1] >> 16 : r.w[i >> 1])));
  else return __uint_as_float(r.w[i]);
}

}  // namespace ffnk

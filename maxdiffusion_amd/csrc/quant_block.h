// e4m3 with one power-of-two scale per block of 128: what the quantiser and the norm with a quantised output share.
#pragma once
#include "mdattn_common.h"

namespace mdattn {

// Rows of channels are walked in chunks of 8; nothing but an element's alignment is asked of their addresses (the loads are
// 16 bytes wide all the same: this card takes them at any address).
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

__device__ __forceinline__ unsigned row16_umax(unsigned x) {
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0u, x, 0xB1, 0xF, 0xF, true));
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0u, x, 0x4E, 0xF, 0xF, true));
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0u, x, 0x141, 0xF, 0xF, true));
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0u, x, 0x140, 0xF, 0xF, true));
  return x;
}

// The scale byte of a block whose largest magnitude has these bits (the maximum of magnitudes is taken on their bits, where a NaN
// is larger than an infinity and that larger than any number).  448 = 1.75 * 2^8: the exponent less 8, one more where the
// mantissa is above 1.75; a zero or anything below 2^-118 gets the smallest scale, 2^-127.
__device__ __forceinline__ unsigned scale_byte(unsigned absmax_bits) {
  const int e = (int)(absmax_bits >> 23);
  const int byte = e - 8 + ((absmax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e == 255 ? 255u : (unsigned)max(byte, 0);
}
// 2^-(byte - 127): at most 2^127, and above the smallest normal number for every byte that a finite block has
__device__ __forceinline__ float scale_inverse(unsigned byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }

// eight scaled values to e4m3 (round to nearest even; none is above 448).  A block that is not finite holds NaNs.
__device__ __forceinline__ u32x2 to_e4m3x8(const float* f, float inv, unsigned byte) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv, f[1] * inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * inv, f[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * inv, f[5] * inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * inv, f[7] * inv, hi, true);
  const bool nan = byte == 255u;
  return u32x2{nan ? 0x7F7F7F7Fu : (unsigned)lo, nan ? 0x7F7F7F7Fu : (unsigned)hi};
}

// eight channels of a row as they are loaded
template <typename T>
struct Chunk;
template <>
struct Chunk<__bf16> {
  u32x4 u;
  __device__ __forceinline__ void load(const __bf16* p) { u = *reinterpret_cast<const u32x4_any*>(p); }
  __device__ __forceinline__ void load_some(const __bf16* p, int n) {
    unsigned short e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < n ? reinterpret_cast<const unsigned short*>(p)[i] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = e[2 * i] | (unsigned)e[2 * i + 1] << 16;
  }
  __device__ __forceinline__ void zero() { u = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Chunk<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const f32x4_any*>(p);
    b = *reinterpret_cast<const f32x4_any*>(p + 4);
  }
  __device__ __forceinline__ void load_some(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = i < n ? p[i] : 0.f;
      b[i] = i + 4 < n ? p[i + 4] : 0.f;
    }
  }
  __device__ __forceinline__ void zero() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[i + 4] = b[i]; }
  }
};

inline int64_t ceil_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
// bytes between the scale rows of `cols` columns: whole words, which the product loads
inline int64_t scale_stride(int64_t cols) { return ceil_to((cols + 127) / 128, 4); }

}  // namespace mdattn

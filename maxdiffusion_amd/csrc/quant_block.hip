// Quantisation to e4m3 with one power-of-two scale per block of 128 channels of a row, or per 128 x 128, of the matrix, of its
// transpose, or of both from one read.
//
// A power of two: x * 2^-e is exact, so that the stored value is the one nearest to x in its block's grid however it is computed, and the
// scale is an operand of the matrix cores' scaled product.  It costs at most one binary place at the bottom of e4m3's range, none of
// its precision.
#include "mdattn_common.h"
#include "mdlayers.h"
#include "quant_block.h"

namespace mdattn {
namespace {

// eight channels from c on; zeros past C
template <typename T>
__device__ __forceinline__ void load8(Chunk<T>& x, const T* row, int64_t c, int64_t C) {
  if (c + 8 <= C) x.load(row + c);
  else if (c < C) x.load_some(row + c, (int)(C - c));
  else x.zero();
}
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

struct QuantArgs {
  const void* x;
  uint8_t *q, *s, *qt, *st;
  float* colsum;
  int64_t R, C, x_stride;
  int64_t ldq, lds, ldt, ldst;  // bytes of a row of q, scales, qt, scales_t
  int blocks;                   // blocks of 128 columns
  int64_t units;
};

// Rows alone, blocks of 1 x 128: 16 lanes to a block, four blocks per thread in flight.  Bound by memory: 75,600 x 5,120 in bf16 194 to 216 us,
// 5.4 to 6.0 TB/s read and written.
constexpr int kUnits = 4;
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs a) {
  const int l16 = threadIdx.x & 15;
  // one division of 64 bits, of the workgroup's first block, and small ones from there: 1 x 5,120, one workgroup, 2.6 and 2.3 us
  const int64_t first = (int64_t)blockIdx.x * (16 * kUnits), row0 = first / a.blocks;
  const unsigned block0 = (unsigned)(first - row0 * a.blocks) + (threadIdx.x >> 4);
  const int64_t left = a.units - first - (threadIdx.x >> 4);
  Chunk<T> x[kUnits];
  int64_t row[kUnits];
  unsigned block[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const unsigned at = block0 + 16 * i, down = at / (unsigned)a.blocks;
    row[i] = row0 + down;
    block[i] = at - down * a.blocks;
    if (16 * i < left) load8(x[i], static_cast<const T*>(a.x) + row[i] * a.x_stride, block[i] * 128 + l16 * 8, a.C);
    else x[i].zero();
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    if (16 * i >= left) break;
    float f[8];
    x[i].get(f);
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, magnitude(f[e]));
    const unsigned byte = scale_byte(row16_umax(m));
    *reinterpret_cast<u32x2*>(a.q + row[i] * a.ldq + block[i] * 128 + l16 * 8) = to_e4m3x8(f, scale_inverse(byte), byte);
    if (l16 == 0) a.s[row[i] * a.lds + block[i]] = (uint8_t)byte;
  }
}

// A tile of 128 x 128 per workgroup.  A thread holds 8 rows x 8 columns: the 16 lanes of a row group cover a row's 128 columns, the 16
// row groups the 128 rows.  The transposed bytes go through LDS, 8 rows of a column in one word, so that whole 128-byte rows of qt
// are stored; word g of column c sits at g ^ (c / 8), without which the 16 lanes that write 8 columns apart would meet in one bank.
// Bound by memory: both ways in blocks of 128 x 128, 15,360 x 5,120 in bf16, 55 us, 5.7 TB/s; of 1 x 128, 18,900 x 5,120, 77 to 83 us, 4.7 to
// 5.0 TB/s, of which the transposed scales' bytes, each a store to a line of its own, cost a tenth.
template <typename T, int BLOCK_ROWS>
__global__ __launch_bounds__(256) void quant_tile_kernel(QuantArgs a) {
  __shared__ u32x2 tile[128][16];
  __shared__ unsigned col_max[4][128];
  __shared__ float col_sum[4][128];
  const int tid = threadIdx.x, l16 = tid & 15, g = tid >> 4, wave = tid >> 6;
  const int64_t rb = blockIdx.x / a.blocks, cb = blockIdx.x - rb * a.blocks;
  const int64_t r0 = rb * 128 + g * 8, c0 = cb * 128 + l16 * 8;
  Chunk<T> x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (r0 + i < a.R) load8(x[i], static_cast<const T*>(a.x) + (r0 + i) * a.x_stride, c0, a.C);
    else x[i].zero();
  }
  unsigned cm[8] = {};
  float cs[8] = {};
  unsigned block_byte = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float f[8];
    x[i].get(f);
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cm[e] = max(cm[e], magnitude(f[e]));
      cs[e] += f[e];
      m = max(m, magnitude(f[e]));
    }
    if (BLOCK_ROWS == 1 && a.q) {
      const unsigned byte = scale_byte(row16_umax(m));
      if (r0 + i < a.R) {
        *reinterpret_cast<u32x2*>(a.q + (r0 + i) * a.ldq + c0) = to_e4m3x8(f, scale_inverse(byte), byte);
        if (l16 == 0) a.s[(r0 + i) * a.lds + cb] = (uint8_t)byte;
      }
    }
  }
  // over the four row groups of a wave, then over the four waves
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const u32x2 p = __builtin_amdgcn_permlane16_swap(cm[e], cm[e], false, false);
    const unsigned m = max(p[0], p[1]);
    const u32x2 h = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    if ((tid & 48) == 0) col_max[wave][l16 * 8 + e] = max(h[0], h[1]);
  }
  if (a.colsum) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const u32x2 p = __builtin_amdgcn_permlane16_swap(__float_as_uint(cs[e]), __float_as_uint(cs[e]), false, false);
      const float s = xhalf_sum(__uint_as_float(p[0]) + __uint_as_float(p[1]));
      if ((tid & 48) == 0) col_sum[wave][l16 * 8 + e] = s;
    }
  }
  __syncthreads();
  if (a.colsum && tid < 128 && cb * 128 + tid < a.C)
    a.colsum[rb * a.C + cb * 128 + tid] = (col_sum[0][tid] + col_sum[1][tid]) + (col_sum[2][tid] + col_sum[3][tid]);
  if constexpr (BLOCK_ROWS == 128) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = l16 * 8 + e;
      m = max(m, max(max(col_max[0][c], col_max[1][c]), max(col_max[2][c], col_max[3][c])));
    }
    block_byte = scale_byte(row16_umax(m));
    if (tid == 0) {
      if (a.s) a.s[rb * a.lds + cb] = (uint8_t)block_byte;
      if (a.st) a.st[cb * a.ldst + rb] = (uint8_t)block_byte;
    }
    if (a.q) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f[8];
        x[i].get(f);
        if (r0 + i < a.R) *reinterpret_cast<u32x2*>(a.q + (r0 + i) * a.ldq + c0) = to_e4m3x8(f, scale_inverse(block_byte), block_byte);
      }
    }
  }
  if (!a.qt) return;
  float inv[8];
  unsigned bytes[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = l16 * 8 + e;
    bytes[e] = BLOCK_ROWS == 128 ? block_byte : scale_byte(max(max(col_max[0][c], col_max[1][c]), max(col_max[2][c], col_max[3][c])));
    inv[e] = scale_inverse(bytes[e]);
    if (BLOCK_ROWS == 1 && g == 0 && cb * 128 + c < a.C) a.st[(cb * 128 + c) * a.ldst + rb] = (uint8_t)bytes[e];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // four rows of all eight columns, into half a word each
    unsigned w[8];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      float f0[8], f1[8];
      x[4 * h + i].get(f0);
      x[4 * h + i + 1].get(f1);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (i == 0) w[e] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f0[e] * inv[e], f1[e] * inv[e], 0, false);
        else w[e] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f0[e] * inv[e], f1[e] * inv[e], (int)w[e], true);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[l16 * 8 + e][g ^ l16][h] = bytes[e] == 255u ? 0x7F7F7F7Fu : w[e];
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int c = it * 32 + (tid >> 3), at = tid & 7, y = c >> 3;
    if (cb * 128 + c >= a.C) continue;
    const u32x2 lo = tile[c][(2 * at) ^ y], hi = tile[c][(2 * at + 1) ^ y];
    *reinterpret_cast<u32x4*>(a.qt + (cb * 128 + c) * a.ldt + rb * 128 + at * 16) = u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
}

}  // namespace
}  // namespace mdattn

using namespace mdattn;

extern "C" int mdattn_quant_block_e4m3(void* stream, const void* x, int x_is_f32, int64_t R, int64_t C, int64_t x_stride, int block_rows, void* q,
                                       void* scales, void* qt, void* scales_t, float* colsum) {
  if (!x || R <= 0 || C <= 0 || !q != !scales || !qt != !scales_t || (!q && !qt)) return MDATTN_E_BADARG;
  if (block_rows != 1 && block_rows != 128) return MDATTN_E_UNSUPPORTED;
  const uintptr_t words = reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(scales_t) | reinterpret_cast<uintptr_t>(colsum);
  if ((reinterpret_cast<uintptr_t>(x) & (x_is_f32 ? 3u : 1u)) || !aligned16(q) || !aligned16(qt) || (words & 3u)) return MDATTN_E_ALIGN;
  if (R > ((int64_t)1 << 40) / C || C > 0x7FFFFFFF - 128) return MDATTN_E_UNSUPPORTED;
  QuantArgs a{};
  a.x = x; a.q = (uint8_t*)q; a.s = (uint8_t*)scales; a.qt = (uint8_t*)qt; a.st = (uint8_t*)scales_t; a.colsum = colsum;
  a.R = R; a.C = C; a.x_stride = x_stride;
  a.ldq = ceil_to(C, 128); a.lds = scale_stride(C); a.ldt = ceil_to(R, 128); a.ldst = scale_stride(R);
  a.blocks = (int)((C + 127) / 128);
  hipStream_t st = (hipStream_t)stream;
  a.units = R * a.blocks;
  const int64_t rows_grid = (a.units + 16 * kUnits - 1) / (16 * kUnits);
  if (block_rows == 1 && !qt && !colsum && grid_fits(rows_grid, 256)) {  // (past 1.07e9 blocks by tiles, of which there are half as many)
    if (x_is_f32) MDATTN_LAUNCH((quant_rows_kernel<float>), dim3((unsigned)rows_grid), dim3(256), 0, st, a);
    else MDATTN_LAUNCH((quant_rows_kernel<__bf16>), dim3((unsigned)rows_grid), dim3(256), 0, st, a);
    return launch_status();
  }
  const int64_t grid = (R + 127) / 128 * a.blocks;
  if (!grid_fits(grid, 256)) return MDATTN_E_UNSUPPORTED;
#define MDATTN_QUANT(T, BR) MDATTN_LAUNCH((quant_tile_kernel<T, BR>), dim3((unsigned)grid), dim3(256), 0, st, a)
  if (x_is_f32) { if (block_rows == 1) MDATTN_QUANT(float, 1); else MDATTN_QUANT(float, 128); }
  else { if (block_rows == 1) MDATTN_QUANT(__bf16, 1); else MDATTN_QUANT(__bf16, 128); }
#undef MDATTN_QUANT
  return launch_status();
}

// Layer norm (plain, affine, modulated per batch element) with its backward pass, and with its output quantised to e4m3.
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  r = (var + eps)^-1/2,  h = (x - mean) r,  y = h (o + w) + b
//   a = g (o + w),  dx = r (a - mean a - h mean(a h)),  dw = sum over rows g h,  db = sum over rows g
//
// One pass over the data: a team of threads owns whole rows, a thread the same few chunks of 8 channels in each of its rows, so that w, b and
// the sums of dw and db stay in its registers while the rows pass by, the next row already on its way.  All teams together walk a window of
// neighbouring rows (75,600 x 5,120 with a stretch of rows each: 8 % slower).  A wave makes the mean of
// its own part and the squares around that mean; the parts join as  M2 = sum M2_w + n_w (mean_w - mean)^2  (Chan et al., Updating
// formulae and a pairwise algorithm for computing sample variances, 1979), which loses nothing where the mean is large against the
// deviation, and takes one exchange through LDS, and one barrier, per row.
// Bound by memory.  bf16 rows, read and written: 75,600 x 5,120 forward 283 us and backward 426 us, both 5.4 TB/s; 32,760 x 1,536 32 to 35 us;
// with a quantised output 30 us, 5.0 TB/s (75,600 x 5,120 252 us, 4.6: the scale bytes are scattered stores).  f32 rows of 600 MB: forward 4.1
// to 5.6 TB/s, backward 4.4 to 5.2.  Backward above 12,288 channels, where 1,024 threads leave each 128 registers and 7 to 113 are spilled:
// bf16 2.8 to 3.4 TB/s (5.3 at 12,288), f32 2.5 to 2.9.  Short calls are bound by the way of a row through memory and its reductions: 4,112 x
// 1,280 forward 7 us, backward 11 and 4 for the sums.
#include "norm_rows.h"

namespace mdattn {
namespace {

struct NormArgs {
  const void* x;
  void* y;
  const void *w, *b;
  uint8_t* scales;
  int64_t rows, wb_stride;                // rows of a group
  int64_t x_sg, x_sr, y_sg, y_sr;
  int64_t scale_stride;
  int C, wb_f32, blocks;                  // workgroups of a group
  float eps, offset;                      // offset: 0 where there is no w
};

enum { kToBf16 = 0, kToF32 = 1, kToE4m3 = 2 };

template <typename T, int OUT, int NV, int MAXT, bool TAIL>
__global__ __launch_bounds__(MAXT) void layer_norm_kernel(NormArgs a) {
  __shared__ float2 part[2][kMaxWaves];
  const int group = blockIdx.x / a.blocks, block = blockIdx.x - group * a.blocks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const Deal<NV, TAIL> deal(a.C, threadIdx.x, blockDim.x);
  const T* x = static_cast<const T*>(a.x) + group * a.x_sg;
  Chunk<T> now[NV], next[NV];
  deal.load(next, x + block * a.x_sr);
  float w[NV][8], b[NV][8];
  deal.vector(w, a.w, a.wb_f32, group * a.wb_stride, 1.f);
  deal.vector(b, a.b, a.wb_f32, group * a.wb_stride, 0.f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) w[j][e] += a.offset;
  const float inv_c = 1.f / a.C, n_wave = deal.count(wave);
  const float inv_n = n_wave > 0.f ? 1.f / n_wave : 0.f;

  int odd = 0;
  for (int64_t row = block; row < a.rows; row += a.blocks, odd ^= 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) now[j] = next[j];
    if (row + a.blocks < a.rows) deal.load(next, x + (row + a.blocks) * a.x_sr);
    float f[NV][8], sum = 0.f, sq = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      now[j].get(f[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += f[j][e];
    }
    float mean = wave_sum(sum) * inv_n;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = deal.has(j, e) ? f[j][e] - mean : 0.f;
        sq += d * d;
      }
    float m2 = wave_sum(sq);
    if (waves > 1) {
      float2* slot = part[odd];  // the other one is read until the next barrier
      if ((threadIdx.x & 63) == 0) slot[wave] = make_float2(mean, m2);
      __syncthreads();
      float all = 0.f;
      for (int i = 0; i < waves; ++i) all += slot[i].x * deal.count(i);
      all *= inv_c;
      m2 = 0.f;
      for (int i = 0; i < waves; ++i) {
        const float d = slot[i].x - all;
        m2 += slot[i].y + deal.count(i) * d * d;
      }
      mean = all;
    }
    const float r = rsqrtf(m2 * inv_c + a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[j][e] = (f[j][e] - mean) * r * w[j][e] + b[j][e];
      if constexpr (OUT == kToE4m3) {
        unsigned m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (!deal.has(j, e)) f[j][e] = 0.f;
          m = max(m, __float_as_uint(f[j][e]) & 0x7FFFFFFFu);
        }
        const unsigned byte = scale_byte(row16_umax(m));  // 16 lanes hold a block of 128
        const int64_t at = group * a.rows + row, ld = (a.C + 127) / 128 * 128;
        if (deal.c[j] < ld) {
          *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(a.y) + at * ld + deal.c[j]) = to_e4m3x8(f[j], scale_inverse(byte), byte);
          if ((threadIdx.x & 15) == 0) a.scales[at * a.scale_stride + deal.c[j] / 128] = (uint8_t)byte;
        }
      } else if constexpr (OUT == kToF32) {
        deal.store(j, static_cast<float*>(a.y) + group * a.y_sg + row * a.y_sr, f[j]);
      } else {
        deal.store(j, static_cast<__bf16*>(a.y) + group * a.y_sg + row * a.y_sr, f[j]);
      }
    }
  }
}

struct NormBwdArgs {
  const void *x, *g, *w;
  void* dx;
  float* part;  // [workgroup][2][C]: its rows' dw and db; null: neither is wanted
  int64_t rows, wb_stride;
  int64_t x_sg, x_sr, g_sg, g_sr, d_sg, d_sr;
  int C, wb_f32, blocks, team;  // workgroups of a group; threads of a team
  float eps, offset;
};

// A workgroup is one team or several, which walk a row each and add up their dw and db at the end, in their order: the sums of all
// workgroups are written and read once more.  (Team after team, each adding to the one before, 4,112 x 1,280 took 14.9 us, by all threads
// at once 10.7.)
template <typename T, int NV, int MAXT, bool TAIL>
__global__ __launch_bounds__(MAXT) void layer_norm_bwd_kernel(NormBwdArgs a) {
  __shared__ float4 part[2][kMaxWaves];
  extern __shared__ __align__(16) float sums[];  // of several teams: [team][2][C rounded up to 8]
  const int group = blockIdx.x / a.blocks, block = blockIdx.x - group * a.blocks;
  const int teams = blockDim.x / a.team, waves = a.team >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = wave / waves, first_wave = mine * waves;
  const Deal<NV, TAIL> deal(a.C, threadIdx.x - first_wave * 64, a.team);
  const T* x = static_cast<const T*>(a.x) + group * a.x_sg;
  const T* g = static_cast<const T*>(a.g) + group * a.g_sg;
  T* dx = static_cast<T*>(a.dx) + group * a.d_sg;
  const int64_t step = (int64_t)a.blocks * teams;
  int64_t row = (int64_t)block * teams + mine;
  Chunk<T> xn[NV], gn[NV];
  {
    const int64_t at = min(row, a.rows - 1);
    deal.load(xn, x + at * a.x_sr);
    deal.load(gn, g + at * a.g_sr);
  }
  float w[NV][8], dw[NV][8], db[NV][8];
  deal.vector(w, a.w, a.wb_f32, group * a.wb_stride, 1.f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[j][e] += a.offset;
      dw[j][e] = db[j][e] = 0.f;
    }
  const float inv_c = 1.f / a.C, n_wave = deal.count(wave - first_wave);
  const float inv_n = n_wave > 0.f ? 1.f / n_wave : 0.f;

  int odd = 0;
  for (int64_t row0 = (int64_t)block * teams; row0 < a.rows; row0 += step, row += step, odd ^= 1) {  // all teams as often: they share the barrier
    float f[NV][8], q[NV][8], sum = 0.f, sq = 0.f, sa = 0.f, sad = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      xn[j].get(f[j]);
      gn[j].get(q[j]);
    }
    if (row + step < a.rows) {
      deal.load(xn, x + (row + step) * a.x_sr);
      deal.load(gn, g + (row + step) * a.g_sr);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum += f[j][e];
        sa += q[j][e] * w[j][e];  // (g is 0 where there is no channel)
      }
    float mean = wave_sum(sum) * inv_n;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = deal.has(j, e) ? f[j][e] - mean : 0.f;
        sq += d * d;
        sad += q[j][e] * w[j][e] * d;
      }
    float m2 = wave_sum(sq);
    sa = wave_sum(sa);
    sad = wave_sum(sad);
    if (waves > 1) {
      float4* slot = part[odd];
      if ((threadIdx.x & 63) == 0) slot[wave] = make_float4(mean, m2, sa, sad);
      __syncthreads();
      float all = 0.f;
      for (int i = 0; i < waves; ++i) all += slot[first_wave + i].x * deal.count(i);
      all *= inv_c;
      m2 = sa = sad = 0.f;
      for (int i = 0; i < waves; ++i) {
        const float4 p = slot[first_wave + i];
        const float d = p.x - all;
        m2 += p.y + deal.count(i) * d * d;
        sa += p.z;
        sad += p.w + p.z * d;  // the sum of a (x - mean) around the common mean
      }
      mean = all;
    }
    if (row >= a.rows) continue;
    const float r = rsqrtf(m2 * inv_c + a.eps);
    const float c1 = sa * inv_c, c2 = sad * inv_c * r;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float h = (f[j][e] - mean) * r;
        dw[j][e] += q[j][e] * h;
        db[j][e] += q[j][e];
        o[e] = r * (q[j][e] * w[j][e] - c1 - h * c2);
      }
      deal.store(j, dx + row * a.d_sr, o);
    }
  }
  if (a.part == nullptr) return;
  float* p = a.part + (int64_t)blockIdx.x * 2 * a.C;
  if (teams > 1) {  // each team's row of sums to LDS, then every thread adds up a few columns of all teams, in their order
    const int ld = (a.C + 7) / 8 * 8;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (deal.c[j] >= a.C) continue;
      f32x4* at = reinterpret_cast<f32x4*>(sums + mine * 2 * ld + deal.c[j]);
      at[0] = f32x4{dw[j][0], dw[j][1], dw[j][2], dw[j][3]};
      at[1] = f32x4{dw[j][4], dw[j][5], dw[j][6], dw[j][7]};
      at += ld / 4;
      at[0] = f32x4{db[j][0], db[j][1], db[j][2], db[j][3]};
      at[1] = f32x4{db[j][4], db[j][5], db[j][6], db[j][7]};
    }
    __syncthreads();
    for (int i = threadIdx.x * 4; i < 2 * ld; i += blockDim.x * 4) {
      f32x4 s = *reinterpret_cast<const f32x4*>(sums + i);
      for (int t = 1; t < teams; ++t) s += *reinterpret_cast<const f32x4*>(sums + t * 2 * ld + i);
      const int plane = i >= ld, c = i - plane * ld;
      float* out = p + plane * a.C + c;
      if (!TAIL || c + 4 <= a.C) {
        *reinterpret_cast<f32x4_any*>(out) = s;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < a.C) out[e] = s[e];
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    deal.keep(j, p, dw[j]);
    deal.keep(j, p + a.C, db[j]);
  }
}

// 64 columns of a group per workgroup, 16 partial sums each.
__global__ __launch_bounds__(1024) void sum_rows_kernel(SumArgs a) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, i0 = threadIdx.x >> 6;
  const int64_t cols = (a.C + 63) / 64, group = blockIdx.x / cols, c = (blockIdx.x - group * cols) * 64 + lane;
  void* out = blockIdx.y ? a.out1 : a.out0;
  if (out == nullptr) return;
  const float* p = a.part + group * a.n * a.row_stride + blockIdx.y * a.plane_stride + (c < a.C ? c : a.C - 1);
  float s = 0.f;
  int64_t i = i0;
  for (; i + 112 < a.n; i += 128) {  // eight loads on their way
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[(i + 16 * j) * a.row_stride];
#pragma unroll
    for (int j = 0; j < 8; ++j) s += v[j];
  }
  for (; i < a.n; i += 16) s += p[i * a.row_stride];
  part[i0][lane] = s;
  __syncthreads();
  if (i0 == 0 && c < a.C) {
    s = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s += part[j][lane];
    const int64_t at = group * a.C + c;
    if (a.f32) static_cast<float*>(out)[at] = s;
    else static_cast<__bf16*>(out)[at] = (__bf16)s;
  }
}

// Rows in flight on a CU, by their bytes: enough to keep the memory busy, and no more, which would make the rows' pages compete.  18 KB of
// rows forward, in bf16 the best number or near it at all but one of the widths measured (512 channels: eighteen rows 6.05 TB/s, six 3.7; 1,536: six
// 5.9, three 4.9, twelve 5.5; 2,560: four 5.6, three 4.8; 5,120: two 5.5, four 5.2; 8,192: one 6.2, two 5.5; but 2,048: five 5.6, four 5.9), 36 with a quantised output, whose arithmetic needs
// more waves (5,120: two 3.4, four 4.5), 32 of x and g backward (2,048: four 4.9, twelve 3.8; 5,120: two 5.2, four 4.4).
struct BwdShape {
  Shape s;
  int teams, blocks;
};
// Several teams to a workgroup of up to 256 threads: their dw and db leave it as one row of sums.
BwdShape bwd_shape(int64_t groups, int64_t rows, int C, int x_is_f32) {
  BwdShape b{shape_of(C), 1, 0};
  if (b.s.threads < 256) b.teams = 256 / b.s.threads;
  const int per_cu = rows_per_cu((int64_t)C * (x_is_f32 ? 8 : 4), 32768, 1);
  b.blocks = blocks_of(groups, (rows + b.teams - 1) / b.teams, 256 * (int64_t)((per_cu + b.teams - 1) / b.teams));
  return b;
}

template <typename T, int OUT>
int launch_norm(hipStream_t st, const NormArgs& a, const Shape& s, unsigned grid) {
#define MDATTN_NORM(NV, MAXT)                                                                                              \
  if (s.nv == NV && (s.threads <= 256 ? 256 : s.threads) == MAXT) {                                                              \
    if (a.C % 8) MDATTN_LAUNCH((layer_norm_kernel<T, OUT, NV, MAXT, true>), dim3(grid), dim3(s.threads), 0, st, a);      \
    else MDATTN_LAUNCH((layer_norm_kernel<T, OUT, NV, MAXT, false>), dim3(grid), dim3(s.threads), 0, st, a);             \
  }
  MDATTN_NORM(1, 256) MDATTN_NORM(2, 256) MDATTN_NORM(3, 256) MDATTN_NORM(2, 512) MDATTN_NORM(3, 512) MDATTN_NORM(2, 1024)
#undef MDATTN_NORM
  return launch_status();
}

int norm(hipStream_t st, NormArgs& a, int x_is_f32, int out, int64_t groups) {
  if (out == kToE4m3) merge_groups(groups, a.rows, a.wb_stride, {{&a.x_sg, &a.x_sr}});
  else merge_groups(groups, a.rows, a.wb_stride, {{&a.x_sg, &a.x_sr}, {&a.y_sg, &a.y_sr}});
  const Shape s = shape_of(a.C);
  const int64_t row_bytes = (int64_t)a.C * (x_is_f32 ? 4 : 2);
  const int64_t target = 256 * (int64_t)(out == kToE4m3 ? rows_per_cu(row_bytes, 36864, 2) : rows_per_cu(row_bytes, 18432, 1));
  // a few rows per workgroup: one each, whose latencies then overlap (2,674 x 1,001 in f32 8.1 and 6.7 us, 4,680 x 1,536 7.8 and 6.8)
  a.blocks = groups * a.rows <= 4 * target ? (int)a.rows : blocks_of(groups, a.rows, target);
  const int64_t grid = groups * a.blocks;
  if (!grid_fits(grid, s.threads)) return MDATTN_E_UNSUPPORTED;
  if (x_is_f32) {
    if (out == kToE4m3) return launch_norm<float, kToE4m3>(st, a, s, (unsigned)grid);
    return out == kToF32 ? launch_norm<float, kToF32>(st, a, s, (unsigned)grid) : launch_norm<float, kToBf16>(st, a, s, (unsigned)grid);
  }
  if (out == kToE4m3) return launch_norm<__bf16, kToE4m3>(st, a, s, (unsigned)grid);
  return out == kToF32 ? launch_norm<__bf16, kToF32>(st, a, s, (unsigned)grid) : launch_norm<__bf16, kToBf16>(st, a, s, (unsigned)grid);
}

}  // namespace

int sum_rows_launch(hipStream_t st, const SumArgs& a, int64_t groups, int planes) {
  MDATTN_LAUNCH(sum_rows_kernel, dim3((unsigned)sum_rows_grid(groups, a.C), (unsigned)planes), dim3(1024), 0, st, a);
  return launch_status();
}
}  // namespace mdattn

using namespace mdattn;

extern "C" int mdattn_layer_norm(void* stream, const void* x, int x_is_f32, void* y, int y_is_f32, const void* w, const void* b, int wb_is_f32,
                                 int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row, int64_t y_stride_group,
                                 int64_t y_stride_row, int64_t wb_stride, float eps, float w_offset) {
  if (!x || !y || !sizes_ok(groups, rows, C) || !(eps >= 0.f) || !(w_offset == w_offset)) return MDATTN_E_BADARG;
  if (C > kMaxC) return MDATTN_E_UNSUPPORTED;
  if (!elem_aligned(x, x_is_f32) || !elem_aligned(y, y_is_f32) || !elem_aligned(w, wb_is_f32) || !elem_aligned(b, wb_is_f32)) return MDATTN_E_ALIGN;
  NormArgs a{};
  a.x = x; a.y = y; a.w = w; a.b = b;
  a.rows = rows; a.wb_stride = wb_stride; a.C = C; a.wb_f32 = wb_is_f32; a.eps = eps; a.offset = w ? w_offset : 0.f;
  a.x_sg = x_stride_group; a.x_sr = x_stride_row; a.y_sg = y_stride_group; a.y_sr = y_stride_row;
  return norm((hipStream_t)stream, a, x_is_f32, y_is_f32 ? kToF32 : kToBf16, groups);
}

extern "C" int mdattn_layer_norm_e4m3(void* stream, const void* x, int x_is_f32, void* q, void* scales, const void* w, const void* b, int wb_is_f32,
                                      int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row, int64_t wb_stride,
                                      float eps, float w_offset) {
  if (!x || !q || !scales || !sizes_ok(groups, rows, C) || !(eps >= 0.f) || !(w_offset == w_offset)) return MDATTN_E_BADARG;
  if (C > kMaxC) return MDATTN_E_UNSUPPORTED;
  if (!elem_aligned(x, x_is_f32) || !aligned16(q) || !elem_aligned(w, wb_is_f32) || !elem_aligned(b, wb_is_f32)) return MDATTN_E_ALIGN;
  NormArgs a{};
  a.x = x; a.y = q; a.scales = static_cast<uint8_t*>(scales); a.w = w; a.b = b;
  a.rows = rows; a.wb_stride = wb_stride; a.C = C; a.wb_f32 = wb_is_f32; a.eps = eps; a.offset = w ? w_offset : 0.f;
  a.x_sg = x_stride_group; a.x_sr = x_stride_row; a.scale_stride = scale_stride(C);
  return norm((hipStream_t)stream, a, x_is_f32, kToE4m3, groups);
}

extern "C" int64_t mdattn_layer_norm_bwd_workspace_floats(int64_t groups, int64_t rows, int C) {
  if (!sizes_ok(groups, rows, C) || C > kMaxC) return 0;
  // (bf16 rows: as many workgroups as f32 ones, or more; and for groups that are merged, or not)
  const int64_t apart = groups * bwd_shape(groups, rows, C, 0).blocks, merged = bwd_shape(1, groups * rows, C, 0).blocks;
  return (apart > merged ? apart : merged) * 2 * C;
}

extern "C" int mdattn_layer_norm_bwd(void* stream, const void* x, int x_is_f32, const void* g, void* dx, const void* w, void* dw, void* db,
                                     int wb_is_f32, int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row,
                                     int64_t g_stride_group, int64_t g_stride_row, int64_t dx_stride_group, int64_t dx_stride_row,
                                     int64_t wb_stride, float eps, float w_offset, float* workspace, int64_t workspace_floats) {
  if (!x || !g || !dx || !sizes_ok(groups, rows, C) || !(eps >= 0.f) || !(w_offset == w_offset) || (dw && !w)) return MDATTN_E_BADARG;
  if (C > kMaxC) return MDATTN_E_UNSUPPORTED;
  const bool sums = dw || db;
  if (sums && (!workspace || workspace_floats < mdattn_layer_norm_bwd_workspace_floats(groups, rows, C))) return MDATTN_E_BADARG;
  if (!elem_aligned(x, x_is_f32) || !elem_aligned(g, x_is_f32) || !elem_aligned(dx, x_is_f32) || !elem_aligned(w, wb_is_f32) ||
      !elem_aligned(dw, wb_is_f32) || !elem_aligned(db, wb_is_f32) || !elem_aligned(workspace, 1))
    return MDATTN_E_ALIGN;
  NormBwdArgs a{};
  a.x = x; a.g = g; a.w = w; a.dx = dx; a.part = sums ? workspace : nullptr;
  a.rows = rows; a.wb_stride = wb_stride; a.C = C; a.wb_f32 = wb_is_f32; a.eps = eps; a.offset = w ? w_offset : 0.f;
  a.x_sg = x_stride_group; a.x_sr = x_stride_row; a.g_sg = g_stride_group; a.g_sr = g_stride_row; a.d_sg = dx_stride_group; a.d_sr = dx_stride_row;
  merge_groups(groups, a.rows, wb_stride, {{&a.x_sg, &a.x_sr}, {&a.g_sg, &a.g_sr}, {&a.d_sg, &a.d_sr}});
  const BwdShape b = bwd_shape(groups, a.rows, C, x_is_f32);
  a.blocks = b.blocks;
  a.team = b.s.threads;
  const int64_t grid = groups * a.blocks, sum_grid = sum_rows_grid(wb_stride ? groups : 1, C);
  if (!grid_fits(grid, b.s.threads * b.teams) || (sums && !grid_fits(sum_grid, 1024))) return MDATTN_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const unsigned threads = (unsigned)(b.s.threads * b.teams), lds = b.teams > 1 ? b.teams * 8u * (unsigned)ceil_to(C, 8) : 0u;
#define MDATTN_NORM(T, NV, MAXT)                                                                                                      \
  if (b.s.nv == NV && (threads <= 256 ? 256 : threads) == MAXT) {                                                                         \
    if (C % 8) MDATTN_LAUNCH((layer_norm_bwd_kernel<T, NV, MAXT, true>), dim3((unsigned)grid), dim3(threads), lds, st, a);          \
    else MDATTN_LAUNCH((layer_norm_bwd_kernel<T, NV, MAXT, false>), dim3((unsigned)grid), dim3(threads), lds, st, a);               \
  }
#define MDATTN_NORMS(T) MDATTN_NORM(T, 1, 256) MDATTN_NORM(T, 2, 256) MDATTN_NORM(T, 3, 256) MDATTN_NORM(T, 2, 512) MDATTN_NORM(T, 3, 512) MDATTN_NORM(T, 2, 1024)
  if (x_is_f32) { MDATTN_NORMS(float) }
  else { MDATTN_NORMS(__bf16) }
#undef MDATTN_NORMS
#undef MDATTN_NORM
  const int rc = launch_status();
  if (rc != MDATTN_OK || !sums) return rc;
  // shared w and b: one sum over the workgroups of all groups
  const SumArgs r{workspace, dw, db, wb_stride ? a.blocks : grid, 2 * (int64_t)C, C, C, wb_is_f32};
  return sum_rows_launch(st, r, wb_stride ? groups : 1, 2);
}

extern "C" int mdattn_sum_rows(void* stream, const float* rows, int64_t n, int64_t C, void* out, int out_is_f32) {
  if (!rows || !out || n <= 0 || C <= 0) return MDATTN_E_BADARG;
  if (!grid_fits((C + 63) / 64, 1024)) return MDATTN_E_UNSUPPORTED;
  if (!elem_aligned(rows, 1) || !elem_aligned(out, out_is_f32)) return MDATTN_E_ALIGN;
  const SumArgs r{rows, out, nullptr, n, C, 0, C, out_is_f32};
  return sum_rows_launch((hipStream_t)stream, r, 1, 1);
}

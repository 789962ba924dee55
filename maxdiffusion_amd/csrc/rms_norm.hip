// RMS norm with the residual's addition in front of it, with its backward pass, and with its output quantised to e4m3.
//
//   s = x + residual,  r = (sum s^2 / C + eps)^-1/2,  h = s r,  y = h (o + w) + b
//   a = g (o + w),  ds = r (a - h mean(a h)) + gs,  dw = sum over rows g h,  db = sum over rows g
//
// As the layer norm: a team of threads owns whole rows, a thread the same few chunks of 8 channels in each of its rows; w, b and the sums of dw
// and db stay in its registers while the rows pass by, the next row already on its way.  A row's one sum (two backward) takes one exchange
// through LDS and one barrier.  h is formed from the f32 sum that s is rounded from.  The backward pass has the rounded one, whose roundings (2^-9 of an
// element on average) change a gradient in bf16 by less than its own; where w, and with it dw, is f32 beside an s in bf16, x and the residual
// take its place, one more read of a row.
// Bound by memory where rows are many: 75,600 rows of 5,120 in bf16, with a residual, scale and shift, 540 us (3.1 GB at 5.7 TB/s, above a copy's
// 4.9: streaming stores); into e4m3, 4,096 x 4,096, 22 us (5.4 TB/s).  Few or odd rows wait for a row's way through memory and its sum: one row
// 3.1 us, 2,674 of 1,001 with an f32 residual 8.9 us (3.6 TB/s), their backward pass 14.6 us (2.9 TB/s) and 3.9 for the sums of dw and db.
// Backward in bf16: 75,600 rows of 5,120 551 us (5.6 TB/s), from x and the residual 654 (5.9); 4,096 x 4,096 27 and 30 us (5.0, 5.6), the sums 4.
// Above 12,288 channels 1,024 threads have 128 registers each, and 50 to 328 values of theirs are spilled (124 to 320 bytes of scratch a lane; f32 rows of
// 8,193 to 12,288 spill 8 to 24 bytes): 4,096 x 16,384 in bf16 196 us (2.7 TB/s; 12,288 5.3), from x and the residual 262, in f32 426 (2.5; 12,288 4.7).
#include "norm_rows.h"

namespace mdattn {
namespace {

struct RmsArgs {
  const void *x, *res;
  void *y, *s;
  const void *w, *b;
  uint8_t* scales;
  int64_t rows, wb_stride;  // rows of a group
  int64_t x_sg, x_sr, r_sg, r_sr, y_sg, y_sr, s_sg, s_sr;
  int64_t scale_stride;
  int C, wb_f32, blocks;  // workgroups of a group
  float eps, offset;      // offset: 0 where there is no w
};

// T: of x and y; R: of the residual and s; QUANT: y in blocks of e4m3
template <typename T, typename R, bool QUANT, int NV, int MAXT, bool TAIL>
__global__ __launch_bounds__(MAXT) void rms_norm_kernel(RmsArgs a) {
  __shared__ float part[2][kMaxWaves];
  const int group = blockIdx.x / a.blocks, block = blockIdx.x - group * a.blocks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const Deal<NV, TAIL> deal(a.C, threadIdx.x, blockDim.x);
  const T* x = static_cast<const T*>(a.x) + group * a.x_sg;
  const R* res = a.res ? static_cast<const R*>(a.res) + group * a.r_sg : nullptr;
  Chunk<T> xn[NV];
  Chunk<R> rn[NV];
  deal.load(xn, x + block * a.x_sr);
  if (res) deal.load(rn, res + block * a.r_sr);
  float w[NV][8], b[NV][8];
  deal.vector(w, a.w, a.wb_f32, group * a.wb_stride, 1.f);
  deal.vector(b, a.b, a.wb_f32, group * a.wb_stride, 0.f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) w[j][e] += a.offset;
  const float inv_c = 1.f / a.C;

  int odd = 0;
  for (int64_t row = block; row < a.rows; row += a.blocks, odd ^= 1) {
    float f[NV][8], sq = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      xn[j].get(f[j]);
      if (res) {
        float q[8];
        rn[j].get(q);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[j][e] += q[e];
      }
    }
    if (row + a.blocks < a.rows) {
      deal.load(xn, x + (row + a.blocks) * a.x_sr);
      if (res) deal.load(rn, res + (row + a.blocks) * a.r_sr);
    }
    if (res) {
      R* s = static_cast<R*>(a.s) + group * a.s_sg + row * a.s_sr;
#pragma unroll
      for (int j = 0; j < NV; ++j) deal.store(j, s, f[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += f[j][e] * f[j][e];  // (0 where there is no channel)
    sq = wave_sum(sq);
    if (waves > 1) {
      float* slot = part[odd];  // the other one is read until the next barrier
      if ((threadIdx.x & 63) == 0) slot[wave] = sq;
      __syncthreads();
      sq = 0.f;
      for (int i = 0; i < waves; ++i) sq += slot[i];
    }
    const float r = rsqrtf(sq * inv_c + a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[j][e] = f[j][e] * r * w[j][e] + b[j][e];
      if constexpr (QUANT) {
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
      } else {
        deal.store(j, static_cast<T*>(a.y) + group * a.y_sg + row * a.y_sr, f[j]);
      }
    }
  }
}

struct RmsBwdArgs {
  const void *s, *res, *g, *gs, *w;  // res: added to s, of its type (bf16)
  void *ds, *dx;
  float* part;  // [workgroup][2][C]: its rows' dw and db; null: neither is wanted
  int64_t rows, wb_stride;
  int64_t s_sg, s_sr, r_sg, r_sr, g_sg, g_sr, gs_sg, gs_sr;
  int C, wb_f32, blocks, team;  // workgroups of a group; threads of a team
  float eps, offset;
};

// R: of s, gs and ds; T: of g and dx.  A workgroup is one team or several, which walk a row each and add up their dw and db at the end, in their
// order: the sums of all workgroups are written and read once more.
template <typename R, typename T, int NV, int MAXT, bool TAIL>
__global__ __launch_bounds__(MAXT) void rms_norm_bwd_kernel(RmsBwdArgs a) {
  __shared__ float2 part[2][kMaxWaves];
  extern __shared__ __align__(16) float sums[];  // of several teams: [team][2][C rounded up to 8]
  const int group = blockIdx.x / a.blocks, block = blockIdx.x - group * a.blocks;
  const int teams = blockDim.x / a.team, waves = a.team >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = wave / waves, first_wave = mine * waves;
  const Deal<NV, TAIL> deal(a.C, threadIdx.x - first_wave * 64, a.team);
  const R* s = static_cast<const R*>(a.s) + group * a.s_sg;
  [[maybe_unused]] const R* res = a.res ? static_cast<const R*>(a.res) + group * a.r_sg : nullptr;
  const T* g = static_cast<const T*>(a.g) + group * a.g_sg;
  const R* gs = a.gs ? static_cast<const R*>(a.gs) + group * a.gs_sg : nullptr;
  const int64_t out = (int64_t)group * a.rows * a.C;
  const int64_t step = (int64_t)a.blocks * teams;
  int64_t row = (int64_t)block * teams + mine;
  constexpr bool Narrow = sizeof(R) == 2;
  Chunk<R> sn[NV], un[NV];
  [[maybe_unused]] Chunk<R> rn[NV];
  Chunk<T> gn[NV];
  auto load = [&](int64_t at) __attribute__((always_inline)) {
    deal.load(sn, s + at * a.s_sr);
    if constexpr (Narrow) {
      if (res) deal.load(rn, res + at * a.r_sr);
    }
    deal.load(gn, g + at * a.g_sr);
    if (gs) deal.load(un, gs + at * a.gs_sr);
  };
  load(min(row, a.rows - 1));
  float w[NV][8], dw[NV][8], db[NV][8];
  deal.vector(w, a.w, a.wb_f32, group * a.wb_stride, 1.f);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[j][e] += a.offset;
      dw[j][e] = db[j][e] = 0.f;
    }
  const float inv_c = 1.f / a.C;

  int odd = 0;
  for (int64_t row0 = (int64_t)block * teams; row0 < a.rows; row0 += step, row += step, odd ^= 1) {  // all teams as often: they share the barrier
    float f[NV][8], q[NV][8], u[NV][8], sq = 0.f, sa = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      sn[j].get(f[j]);
      if constexpr (Narrow) {
        if (res) {
          float r[8];
          rn[j].get(r);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[j][e] += r[e];
        }
      }
      gn[j].get(q[j]);
      if (gs) {
        un[j].get(u[j]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[j][e] = 0.f;
      }
    }
    if (row + step < a.rows) load(row + step);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sq += f[j][e] * f[j][e];
        sa += q[j][e] * w[j][e] * f[j][e];
      }
    sq = wave_sum(sq);
    sa = wave_sum(sa);
    if (waves > 1) {
      float2* slot = part[odd];
      if ((threadIdx.x & 63) == 0) slot[wave] = make_float2(sq, sa);
      __syncthreads();
      sq = sa = 0.f;
      for (int i = 0; i < waves; ++i) {
        sq += slot[first_wave + i].x;
        sa += slot[first_wave + i].y;
      }
    }
    if (row >= a.rows) continue;
    const float r = rsqrtf(sq * inv_c + a.eps), c = sa * inv_c * r;  // c: mean(a h)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float h = f[j][e] * r;
        dw[j][e] += q[j][e] * h;
        db[j][e] += q[j][e];
        o[e] = r * (q[j][e] * w[j][e] - h * c) + u[j][e];
      }
      deal.store(j, static_cast<R*>(a.ds) + out + row * a.C, o);
      if (a.dx) deal.store(j, static_cast<T*>(a.dx) + out + row * a.C, o);
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
      f32x4 v = *reinterpret_cast<const f32x4*>(sums + i);
      for (int t = 1; t < teams; ++t) v += *reinterpret_cast<const f32x4*>(sums + t * 2 * ld + i);
      const int plane = i >= ld, c = i - plane * ld;
      float* at = p + plane * a.C + c;
      if (!TAIL || c + 4 <= a.C) {
        *reinterpret_cast<f32x4_any*>(at) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < a.C) at[e] = v[e];
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

// Several teams to a workgroup of up to 256 threads: their dw and db leave it as one row of sums.
struct BwdShape {
  Shape s;
  int teams, blocks;
};
BwdShape bwd_shape(int64_t groups, int64_t rows, int C, int64_t row_bytes) {
  BwdShape b{shape_of(C), 1, 0};
  if (b.s.threads < 256) b.teams = 256 / b.s.threads;
  const int per_cu = rows_per_cu(row_bytes, 32768, 1);
  b.blocks = blocks_of(groups, (rows + b.teams - 1) / b.teams, 256 * (int64_t)((per_cu + b.teams - 1) / b.teams));
  return b;
}

template <typename T, typename R, bool QUANT>
int launch_rms(hipStream_t st, const RmsArgs& a, const Shape& s, unsigned grid) {
#define MDATTN_NORM(NV, MAXT)                                                                                                  \
  if (s.nv == NV && (s.threads <= 256 ? 256 : s.threads) == MAXT) {                                                            \
    if (a.C % 8) MDATTN_LAUNCH((rms_norm_kernel<T, R, QUANT, NV, MAXT, true>), dim3(grid), dim3(s.threads), 0, st, a);         \
    else MDATTN_LAUNCH((rms_norm_kernel<T, R, QUANT, NV, MAXT, false>), dim3(grid), dim3(s.threads), 0, st, a);                \
  }
  MDATTN_NORM(1, 256) MDATTN_NORM(2, 256) MDATTN_NORM(3, 256) MDATTN_NORM(2, 512) MDATTN_NORM(3, 512) MDATTN_NORM(2, 1024)
#undef MDATTN_NORM
  return launch_status();
}

template <bool QUANT>
int rms(hipStream_t st, RmsArgs& a, int x_is_f32, int r_is_f32, int64_t groups) {
  int64_t none_g = a.x_sg, none_r = a.x_sr;  // of a tensor that is not there
  const Strides xs{&a.x_sg, &a.x_sr}, rs = a.res ? Strides{&a.r_sg, &a.r_sr} : Strides{&none_g, &none_r}, ss = a.res ? Strides{&a.s_sg, &a.s_sr} : rs;
  if (QUANT) merge_groups(groups, a.rows, a.wb_stride, {xs, rs, ss});
  else merge_groups(groups, a.rows, a.wb_stride, {xs, rs, ss, {&a.y_sg, &a.y_sr}});
  const Shape s = shape_of(a.C);
  const int64_t row_bytes = (int64_t)a.C * ((x_is_f32 ? 4 : 2) + (a.res ? (r_is_f32 ? 4 : 2) : 0));
  const int64_t target = 256 * (int64_t)(QUANT ? rows_per_cu(row_bytes, 36864, 2) : rows_per_cu(row_bytes, 18432, 1));
  a.blocks = groups * a.rows <= 4 * target ? (int)a.rows : blocks_of(groups, a.rows, target);
  const int64_t grid = groups * a.blocks;
  if (!grid_fits(grid, s.threads)) return MDATTN_E_UNSUPPORTED;
  if (x_is_f32) return launch_rms<float, float, QUANT>(st, a, s, (unsigned)grid);
  return a.res && r_is_f32 ? launch_rms<__bf16, float, QUANT>(st, a, s, (unsigned)grid) : launch_rms<__bf16, __bf16, QUANT>(st, a, s, (unsigned)grid);
}

int rms_checks(const void* x, int x_is_f32, const void* res, int r_is_f32, const void* y, const void* s, const void* w, const void* b, int wb_is_f32,
               int64_t groups, int64_t rows, int C, float eps, float w_offset) {
  if (!x || !y || (res == nullptr) != (s == nullptr) || !sizes_ok(groups, rows, C) || !(eps >= 0.f) || !(w_offset == w_offset)) return MDATTN_E_BADARG;
  if (C > kMaxC || (res && x_is_f32 && !r_is_f32)) return MDATTN_E_UNSUPPORTED;
  if (!elem_aligned(x, x_is_f32) || !elem_aligned(res, r_is_f32) || !elem_aligned(s, r_is_f32) || !elem_aligned(w, wb_is_f32) || !elem_aligned(b, wb_is_f32))
    return MDATTN_E_ALIGN;
  return MDATTN_OK;
}

}  // namespace
}  // namespace mdattn

using namespace mdattn;

extern "C" int mdattn_rms_norm(void* stream, const void* x, int x_is_f32, const void* residual, int r_is_f32, void* y, void* s, const void* w,
                               const void* b, int wb_is_f32, int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row,
                               int64_t r_stride_group, int64_t r_stride_row, int64_t y_stride_group, int64_t y_stride_row, int64_t s_stride_group,
                               int64_t s_stride_row, int64_t wb_stride, float eps, float w_offset) {
  const int rc = rms_checks(x, x_is_f32, residual, r_is_f32, y, s, w, b, wb_is_f32, groups, rows, C, eps, w_offset);
  if (rc != MDATTN_OK) return rc;
  if (!elem_aligned(y, x_is_f32)) return MDATTN_E_ALIGN;
  RmsArgs a{};
  a.x = x; a.res = residual; a.y = y; a.s = s; a.w = w; a.b = b;
  a.rows = rows; a.wb_stride = wb_stride; a.C = C; a.wb_f32 = wb_is_f32; a.eps = eps; a.offset = w ? w_offset : 0.f;
  a.x_sg = x_stride_group; a.x_sr = x_stride_row; a.r_sg = r_stride_group; a.r_sr = r_stride_row;
  a.y_sg = y_stride_group; a.y_sr = y_stride_row; a.s_sg = s_stride_group; a.s_sr = s_stride_row;
  return rms<false>((hipStream_t)stream, a, x_is_f32, r_is_f32, groups);
}

extern "C" int mdattn_rms_norm_e4m3(void* stream, const void* x, int x_is_f32, const void* residual, int r_is_f32, void* q, void* scales, void* s,
                                    const void* w, const void* b, int wb_is_f32, int64_t groups, int64_t rows, int C, int64_t x_stride_group,
                                    int64_t x_stride_row, int64_t r_stride_group, int64_t r_stride_row, int64_t s_stride_group, int64_t s_stride_row,
                                    int64_t wb_stride, float eps, float w_offset) {
  const int rc = rms_checks(x, x_is_f32, residual, r_is_f32, q, s, w, b, wb_is_f32, groups, rows, C, eps, w_offset);
  if (rc != MDATTN_OK) return rc;
  if (!scales) return MDATTN_E_BADARG;
  if (!aligned16(q)) return MDATTN_E_ALIGN;
  RmsArgs a{};
  a.x = x; a.res = residual; a.y = q; a.scales = static_cast<uint8_t*>(scales); a.s = s; a.w = w; a.b = b;
  a.rows = rows; a.wb_stride = wb_stride; a.C = C; a.wb_f32 = wb_is_f32; a.eps = eps; a.offset = w ? w_offset : 0.f;
  a.x_sg = x_stride_group; a.x_sr = x_stride_row; a.r_sg = r_stride_group; a.r_sr = r_stride_row;
  a.s_sg = s_stride_group; a.s_sr = s_stride_row; a.scale_stride = scale_stride(C);
  return rms<true>((hipStream_t)stream, a, x_is_f32, r_is_f32, groups);
}

extern "C" int64_t mdattn_rms_norm_bwd_workspace_floats(int64_t groups, int64_t rows, int C) {
  if (!sizes_ok(groups, rows, C) || C > kMaxC) return 0;
  // (the smallest rows: as many workgroups as any others, or more; and for groups that are merged, or not)
  const int64_t apart = groups * bwd_shape(groups, rows, C, 4 * (int64_t)C).blocks, merged = bwd_shape(1, groups * rows, C, 4 * (int64_t)C).blocks;
  return (apart > merged ? apart : merged) * 2 * C;
}

extern "C" int mdattn_rms_norm_bwd(void* stream, const void* s, int s_is_f32, const void* residual, const void* g, int g_is_f32, const void* gs,
                                   void* ds, void* dx, const void* w, void* dw, void* db, int wb_is_f32, int64_t groups, int64_t rows, int C,
                                   int64_t s_stride_group, int64_t s_stride_row, int64_t r_stride_group, int64_t r_stride_row,
                                   int64_t g_stride_group, int64_t g_stride_row, int64_t gs_stride_group, int64_t gs_stride_row, int64_t wb_stride,
                                   float eps, float w_offset, float* workspace, int64_t workspace_floats) {
  if (!s || !g || !ds || !sizes_ok(groups, rows, C) || !(eps >= 0.f) || !(w_offset == w_offset) || (dw && !w)) return MDATTN_E_BADARG;
  if (C > kMaxC || (g_is_f32 && !s_is_f32) || (dx && g_is_f32) || (residual && s_is_f32)) return MDATTN_E_UNSUPPORTED;
  const bool sums = dw || db;
  if (sums && (!workspace || workspace_floats < mdattn_rms_norm_bwd_workspace_floats(groups, rows, C))) return MDATTN_E_BADARG;
  if (!elem_aligned(s, s_is_f32) || !elem_aligned(residual, 0) || !elem_aligned(gs, s_is_f32) || !elem_aligned(ds, s_is_f32) || !elem_aligned(g, g_is_f32) || !elem_aligned(dx, 0) ||
      !elem_aligned(w, wb_is_f32) || !elem_aligned(dw, wb_is_f32) || !elem_aligned(db, wb_is_f32) || !elem_aligned(workspace, 1))
    return MDATTN_E_ALIGN;
  RmsBwdArgs a{};
  a.s = s; a.res = residual; a.g = g; a.gs = gs; a.w = w; a.ds = ds; a.dx = dx; a.part = sums ? workspace : nullptr;
  a.rows = rows; a.wb_stride = wb_stride; a.C = C; a.wb_f32 = wb_is_f32; a.eps = eps; a.offset = w ? w_offset : 0.f;
  a.s_sg = s_stride_group; a.s_sr = s_stride_row; a.r_sg = r_stride_group; a.r_sr = r_stride_row; a.g_sg = g_stride_group; a.g_sr = g_stride_row; a.gs_sg = gs_stride_group; a.gs_sr = gs_stride_row;
  int64_t none_g = a.s_sg, none_r = a.s_sr;
  int64_t no_res_g = a.s_sg, no_res_r = a.s_sr;
  const Strides us = gs ? Strides{&a.gs_sg, &a.gs_sr} : Strides{&none_g, &none_r}, rs = residual ? Strides{&a.r_sg, &a.r_sr} : Strides{&no_res_g, &no_res_r};
  merge_groups(groups, a.rows, wb_stride, {{&a.s_sg, &a.s_sr}, {&a.g_sg, &a.g_sr}, us, rs});
  const BwdShape b = bwd_shape(groups, a.rows, C, (int64_t)C * ((s_is_f32 ? 4 : 2) * (1 + (gs != nullptr) + (residual != nullptr)) + (g_is_f32 ? 4 : 2)));
  a.blocks = b.blocks;
  a.team = b.s.threads;
  const int64_t grid = groups * a.blocks, sum_groups = wb_stride ? groups : 1;
  if (!grid_fits(grid, b.s.threads * b.teams) || (sums && !grid_fits(sum_rows_grid(sum_groups, C), 1024))) return MDATTN_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const unsigned threads = (unsigned)(b.s.threads * b.teams), lds = b.teams > 1 ? b.teams * 8u * (unsigned)ceil_to(C, 8) : 0u;
#define MDATTN_NORM(R, T, NV, MAXT)                                                                                                         \
  if (b.s.nv == NV && (threads <= 256 ? 256 : threads) == MAXT) {                                                                           \
    if (C % 8) MDATTN_LAUNCH((rms_norm_bwd_kernel<R, T, NV, MAXT, true>), dim3((unsigned)grid), dim3(threads), lds, st, a);                 \
    else MDATTN_LAUNCH((rms_norm_bwd_kernel<R, T, NV, MAXT, false>), dim3((unsigned)grid), dim3(threads), lds, st, a);                      \
  }
#define MDATTN_NORMS(R, T) \
  MDATTN_NORM(R, T, 1, 256) MDATTN_NORM(R, T, 2, 256) MDATTN_NORM(R, T, 3, 256) MDATTN_NORM(R, T, 2, 512) MDATTN_NORM(R, T, 3, 512) MDATTN_NORM(R, T, 2, 1024)
  if (!s_is_f32) { MDATTN_NORMS(__bf16, __bf16) }
  else if (g_is_f32) { MDATTN_NORMS(float, float) }
  else { MDATTN_NORMS(float, __bf16) }
#undef MDATTN_NORMS
#undef MDATTN_NORM
  const int rc = launch_status();
  if (rc != MDATTN_OK || !sums) return rc;
  // shared w and b: one sum over the workgroups of all groups
  return sum_rows_launch(st, {workspace, dw, db, wb_stride ? a.blocks : grid, 2 * (int64_t)C, C, C, wb_is_f32}, sum_groups, 2);
}

// Rows of channels dealt to teams of threads: what the norms over the last axis share.
#pragma once
#include "mdlayers.h"
#include "quant_block.h"

namespace mdattn {

constexpr int kMaxWaves = 16;

__device__ __forceinline__ float wave_sum(float x) {
  x = row16_sum(x);
  const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xhalf_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

__device__ __forceinline__ void store8(__bf16* p, const float* f) {
  const uint4 u = pack8(f);
  __builtin_nontemporal_store(u32x4{u.x, u.y, u.z, u.w}, reinterpret_cast<u32x4_any*>(p));
}
__device__ __forceinline__ void store8(float* p, const float* f) {
  __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4_any*>(p));
  __builtin_nontemporal_store(f32x4{f[4], f[5], f[6], f[7]}, reinterpret_cast<f32x4_any*>(p + 4));
}

// A row of C channels dealt to a team of threads: slot j of a thread is chunk j * team + tid.  TAIL: C is not a multiple of 8, and the
// last chunk is walked by elements.
template <int NV, bool TAIL>
struct Deal {
  int c[NV];  // first channel of each slot
  int C, team;
  __device__ __forceinline__ Deal(int C_, int tid, int team_) : C(C_), team(team_) {
#pragma unroll
    for (int j = 0; j < NV; ++j) c[j] = (j * team + tid) * 8;
  }
  __device__ __forceinline__ bool has(int j, int e) const { return TAIL ? c[j] + e < C : c[j] < C; }
  template <typename T>
  __device__ __forceinline__ void load(Chunk<T> (&x)[NV], const T* row) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (TAIL ? c[j] + 8 <= C : c[j] < C) x[j].load(row + c[j]);
      else if (TAIL && c[j] < C) x[j].load_some(row + c[j], C - c[j]);
      else x[j].zero();
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(int j, T* row, const float* f) const {
    if (TAIL ? c[j] + 8 <= C : c[j] < C) {
      store8(row + c[j], f);
    } else if (TAIL && c[j] < C) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c[j] + e < C) row[c[j] + e] = (T)f[e];
    }
  }
  // f32 that is read again soon
  __device__ __forceinline__ void keep(int j, float* row, const float* f) const {
    if (TAIL ? c[j] + 8 <= C : c[j] < C) {
      *reinterpret_cast<f32x4_any*>(row + c[j]) = f32x4{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<f32x4_any*>(row + c[j] + 4) = f32x4{f[4], f[5], f[6], f[7]};
    } else if (TAIL && c[j] < C) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c[j] + e < C) row[c[j] + e] = f[e];
    }
  }
  // w or b of one group as f32; `none` where there is none, zeros where there is no channel
  __device__ __forceinline__ void vector(float (&v)[NV][8], const void* p, int is_f32, int64_t at, float none) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = none;
      if (p == nullptr) continue;
      if (is_f32) {
        Chunk<float> x[NV];
        load(x, static_cast<const float*>(p) + at);
        x[j].get(v[j]);
      } else {
        Chunk<__bf16> x[NV];
        load(x, static_cast<const __bf16*>(p) + at);
        x[j].get(v[j]);
      }
    }
  }
  // channels that the slots of the team's wave `w` hold
  __device__ __forceinline__ float count(int w) const {
    int n = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) n += min(max(C - (j * team + w * 64) * 8, 0), 512);
    return (float)n;
  }
};

// out[g][c] = sum over i < n of part[g * n + i][plane][c], plane 0 to out0, 1 to out1 (null: left out).
struct SumArgs {
  const float* part;
  void *out0, *out1;
  int64_t n, row_stride, plane_stride;
  int64_t C;
  int f32;
};
inline int64_t sum_rows_grid(int64_t groups, int64_t C) { return groups * ((C + 63) / 64); }  // workgroups of 1,024 threads
int sum_rows_launch(hipStream_t st, const SumArgs& a, int64_t groups, int planes);

constexpr int kMaxC = 16384;
// How a row is dealt: chunks per thread and threads of a team.  The fewest places that hold a row, with a power of two of threads: teams of
// five or six waves sit unevenly on the four SIMDs of a CU (quantised rows of 5,120: 320 threads 2.6 TB/s, 256 with a sixth of the places
// empty 4.5).
struct Shape {
  int nv, threads;
};
inline Shape shape_of(int C) {
  const int chunks = (C + 7) / 8;
  Shape best{0, 0};
  for (int t = 64; t <= 1024; t *= 2)
    for (int nv = 1; nv <= 3; ++nv)
      if (nv * t >= chunks && (best.nv == 0 || nv * t < best.nv * best.threads || (nv * t == best.nv * best.threads && nv > best.nv))) best = {nv, t};
  return best;
}
inline int rows_per_cu(int64_t row_bytes, int64_t in_flight, int least) { return (int)((in_flight + row_bytes / 2) / row_bytes < least ? least : (in_flight + row_bytes / 2) / row_bytes); }
// Workgroups of one group of so many rows, of all groups' `target`, and no more than go through them in as many rounds
inline int blocks_of(int64_t groups, int64_t rows, int64_t target) {
  const int64_t n = (target + groups - 1) / groups, rounds = (rows + n - 1) / n;
  return (int)((rows + rounds - 1) / rounds);
}
// A tensor's strides of a group and of a row.  Groups that share w and b, and follow one another as rows do, are one group of all rows.
struct Strides {
  int64_t *group, *row;
};
template <int N>
void merge_groups(int64_t& groups, int64_t& rows, int64_t wb_stride, const Strides (&all)[N]) {
  if (groups == 1 || wb_stride != 0) return;
  for (const Strides& s : all) {
    if (rows > 1 && *s.group != rows * *s.row) return;
  }
  if (rows == 1) {
    for (const Strides& s : all) *s.row = *s.group;
  }
  rows *= groups;
  groups = 1;
}

inline bool sizes_ok(int64_t groups, int64_t rows, int C) {
  return groups > 0 && rows > 0 && C > 0 && rows < ((int64_t)1 << 40) / groups;
}
inline bool elem_aligned(const void* p, int is_f32) { return (reinterpret_cast<uintptr_t>(p) & (is_f32 ? 3u : 1u)) == 0; }

}  // namespace mdattn

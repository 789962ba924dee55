// c [M, N] = a b^T + bias over e4m3 operands with one power-of-two scale per block of 128 along K:
//   c[m, n] = sum over k-blocks 2^(ea[m, kb] + eb[n, kb]) sum over k in kb qa[m, k] qb[n, k]
// The scales are operands of the matrix cores' scaled product (32 x 32 x 64): a block costs no instruction but the read of its byte.
#include "mdattn_common.h"
#include "mdlayers.h"
#include "quant_block.h"

namespace mdattn {
namespace {

struct MatmulArgs {
  const uint8_t *a, *b, *sa, *sb;
  const void* bias;
  __bf16* c;
  float* part;       // split over K: f32 sums [piece][M][N]
  int64_t c_stride, M, N;
  int64_t ld, ls;    // bytes of an operand's row, and of a row of scales
  int b_shift, bias_f32;
  int kb, kb_piece;  // k-blocks, and those of a piece (a multiple of 4)
  int mt, nt, total, chunk;
};

__device__ __forceinline__ float bias_at(const void* p, int f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const __bf16*>(p)[i];
}

// One workgroup, four waves in 2 x 2, computes BM x BN.  A stage of LDS holds 128 bytes of each row of both tiles, written by
// direct loads; 16-byte chunk c of row r sits at c ^ ((r >> 1) & 7), which spreads 16 rows' reads of one chunk over all banks.  While a stage is
// multiplied the next one is on its way: one barrier per 128 of K, behind which the first half of the next stage's fragments are read
// under the second half's products.
template <int BM, int BN>
__global__ __launch_bounds__(256) void matmul_fp8_kernel(MatmulArgs p) {
  constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 32, TN = WN / 32;
  constexpr int kStage = (BM + BN) * 128, kScales = (BM + BN) * 4;
  constexpr int kLoads = (BM + BN) / 32;  // direct loads of a stage by one wave: 8 rows each
  constexpr int kScaleLoads = (BM + BN) / 256;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hh = lane >> 5, wm = wave & 1, wn = wave >> 1;

  // neighbouring workgroups sit on different dies: each die takes a contiguous piece of the tiles, in groups of 8 rows of them
  int id = (blockIdx.x & 7) * p.chunk + (blockIdx.x >> 3);
  if (id >= p.total) return;
  const int piece = id / (p.mt * p.nt);
  id -= piece * p.mt * p.nt;
  const int band = id / (8 * p.nt), rows = min(p.mt - band * 8, 8), in = id - band * 8 * p.nt;
  const int64_t m0 = (int64_t)(band * 8 + in % rows) * BM, n0 = (int64_t)(in / rows) * BN;
  const int kb0 = piece * p.kb_piece, nk = min(p.kb_piece, p.kb - kb0);

  // what this lane loads: byte offsets from the tile's first row (rows past the end read the last one; they are not stored)
  const uint8_t* a_at = p.a + m0 * p.ld + (int64_t)kb0 * 128;
  const uint8_t* b_at = p.b + n0 * p.ld + (int64_t)kb0 * 128;
  unsigned from[kLoads], from_s[kScaleLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = (wave + 4 * i) * 8 + (lane >> 3);  // row of the stage: a's, then b's
    const int64_t left = r < BM ? p.M - 1 - m0 : p.N - 1 - n0;
    const int64_t row = min((int64_t)(r < BM ? r : r - BM), left);
    from[i] = (unsigned)(row * p.ld + ((lane & 7) ^ ((r >> 1) & 7)) * 16);
  }
  const uint8_t* sa_at = p.sa + m0 * p.ls + kb0;
  const uint8_t* sb_at = p.sb + (n0 >> p.b_shift) * p.ls + kb0;
#pragma unroll
  for (int i = 0; i < kScaleLoads; ++i) {
    const int r = (wave + 4 * i) * 64 + lane;
    if (r < BM) from_s[i] = (unsigned)(min((int64_t)r, p.M - 1 - m0) * p.ls);
    else from_s[i] = (unsigned)(((min(n0 + r - BM, p.N - 1) >> p.b_shift) - (n0 >> p.b_shift)) * p.ls);
  }
  const unsigned lds = lds_addr_of(smem);
  auto request = [&](int k) {  // stage k, and the scales of the four stages that begin with it
    const unsigned to = lds + (k & 1) * kStage + wave * 1024;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) lds_dma16((wave + 4 * i) * 8 < BM ? a_at : b_at, from[i], to + i * 4096);
    a_at += 128;
    b_at += 128;
    if ((k & 3) == 0) {
      const unsigned to_s = lds + 2 * kStage + ((k >> 2) & 1) * kScales + wave * 256;
#pragma unroll
      for (int i = 0; i < kScaleLoads; ++i) lds_dma4((wave + 4 * i) * 64 < BM ? sa_at : sb_at, from_s[i], to_s + i * 1024);
      sa_at += 4;
      sb_at += 4;
    }
  };

  f32x16 acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.f;
  i32x8 fa[2][TM], fb[2][TN];
  int sa[TM], sb[TN], sa_next[TM], sb_next[TN];
  const char* ra = smem + (wm * WM + l32) * 128;
  const char* rb = smem + (BM + wn * WN + l32) * 128;
  const int swz = (l32 >> 1) & 7;
  auto fragment = [&](const char* at, int j) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(at + (((4 * j + 2 * hh) ^ swz) * 16));
    const u32x4 hi = *reinterpret_cast<const u32x4*>(at + (((4 * j + 2 * hh + 1) ^ swz) * 16));
    return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  auto read_half = [&](int k, int j) {
    const int s = (k & 1) * kStage;
#pragma unroll
    for (int m = 0; m < TM; ++m) fa[j][m] = fragment(ra + s + m * 4096, j);
#pragma unroll
    for (int n = 0; n < TN; ++n) fb[j][n] = fragment(rb + s + n * 4096, j);
  };
  auto read_scales = [&](int k) {
    const char* s = smem + 2 * kStage + ((k >> 2) & 1) * kScales + (k & 3);
#pragma unroll
    for (int m = 0; m < TM; ++m) sa_next[m] = *reinterpret_cast<const uint8_t*>(s + (wm * WM + m * 32 + l32) * 4);
#pragma unroll
    for (int n = 0; n < TN; ++n) sb_next[n] = *reinterpret_cast<const uint8_t*>(s + (BM + wn * WN + n * 32 + l32) * 4);
  };
  auto multiply = [&](int j) {
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int m = 0; m < TM; ++m)
        acc[n][m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[j][n], fa[j][m], acc[n][m], 0, 0, 0, sb[n], 0, sa[m]);
  };
  auto everyone_has_it = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  request(0);
  everyone_has_it();
  if (nk > 1) request(1);
  read_scales(0);
  read_half(0, 0);
  for (int k = 0; k < nk; ++k) {
#pragma unroll
    for (int m = 0; m < TM; ++m) sa[m] = sa_next[m];
#pragma unroll
    for (int n = 0; n < TN; ++n) sb[n] = sb_next[n];
    read_half(k, 1);
    multiply(0);
    everyone_has_it();  // stage k is read, stage k + 1 has landed
    if (k + 2 < nk) request(k + 2);
    if (k + 1 < nk) {
      read_scales(k + 1);
      read_half(k + 1, 0);
    }
    multiply(1);
  }

  // lane l32 holds output row m0 + .. + l32; register i of it column (i & 3) + 8 (i >> 2) + 4 hh of 32
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int64_t row = m0 + wm * WM + m * 32 + l32;
    if (row >= p.M) continue;
#pragma unroll
    for (int n = 0; n < TN; ++n) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t col = n0 + wn * WN + n * 32 + 8 * q + 4 * hh;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = acc[n][m][4 * q + e];
          if (p.bias && !p.part && col + e < p.N) v[e] += bias_at(p.bias, p.bias_f32, col + e);
        }
        if (p.part) {
          float* o = p.part + ((int64_t)piece * p.M + row) * p.N + col;
          if (col + 4 <= p.N) *reinterpret_cast<f32x4_any*>(o) = f32x4{v[0], v[1], v[2], v[3]};
          else
            for (int e = 0; e < 4; ++e)
              if (col + e < p.N) o[e] = v[e];
        } else {
          __bf16* o = p.c + row * p.c_stride + col;
          typedef u32x2 u32x2_half __attribute__((aligned(2)));
          if (col + 4 <= p.N) *reinterpret_cast<u32x2_half*>(o) = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
          else
            for (int e = 0; e < 4; ++e)
              if (col + e < p.N) o[e] = (__bf16)v[e];
        }
      }
    }
  }
}

// the pieces of a product that was split over K, in their order, then the bias
__global__ __launch_bounds__(256) void join_pieces_kernel(const float* part, int pieces, const void* bias, int bias_f32, __bf16* c, int64_t c_stride,
                                                          int64_t M, int64_t N) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < M * N; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / N, col = i - row * N;
    float s = 0.f;
    for (int j = 0; j < pieces; ++j) s += part[j * M * N + i];
    if (bias) s += bias_at(bias, bias_f32, col);
    c[row * c_stride + col] = (__bf16)s;
  }
}

struct Plan {
  int tile, pieces, kb_piece;
};
Plan plan_of(int64_t M, int64_t N, int64_t K) {
  const int kb = (int)((K + 127) / 128);
  return {128, 1, (kb + 3) / 4 * 4};
}
int64_t floats_of(const Plan& p, int64_t M, int64_t N) { return p.pieces > 1 ? p.pieces * M * N : 0; }

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M > 0 && N > 0 && K > 0 && M < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && K <= (1 << 23) && (M + 127) / 128 * ((N + 127) / 128) < (1 << 27);
}

template <int BM, int BN>
int launch(hipStream_t st, MatmulArgs& a, int pieces) {
  constexpr int kBytes = 2 * ((BM + BN) * 128 + (BM + BN) * 4);
  static LdsOptIn flag;
  const int rc = lds_opt_in(flag, reinterpret_cast<const void*>(&matmul_fp8_kernel<BM, BN>), kBytes);
  if (rc != MDATTN_OK) return rc;
  a.mt = (int)((a.M + BM - 1) / BM);
  a.nt = (int)((a.N + BN - 1) / BN);
  a.total = a.mt * a.nt * pieces;
  a.chunk = (a.total + 7) / 8;
  MDATTN_LAUNCH((matmul_fp8_kernel<BM, BN>), dim3((unsigned)(a.chunk * 8)), dim3(256), kBytes, st, a);
  return launch_status();
}

}  // namespace
}  // namespace mdattn

using namespace mdattn;

extern "C" int64_t mdattn_matmul_fp8_block_workspace_floats(int64_t M, int64_t N, int64_t K) {
  return sizes_ok(M, N, K) ? floats_of(plan_of(M, N, K), M, N) : 0;
}

extern "C" int mdattn_matmul_fp8_block(void* stream, const void* a, const void* a_scales, const void* b, const void* b_scales, int b_block_rows,
                                       const void* bias, int bias_is_f32, void* c, int64_t c_stride, int64_t M, int64_t N, int64_t K,
                                       float* workspace, int64_t workspace_floats) {
  if (!a || !a_scales || !b || !b_scales || !c || M <= 0 || N <= 0 || K <= 0 || c_stride < N) return MDATTN_E_BADARG;
  if ((b_block_rows != 1 && b_block_rows != 128) || !sizes_ok(M, N, K)) return MDATTN_E_UNSUPPORTED;
  const uintptr_t words = reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b_scales);
  if (!aligned16(a) || !aligned16(b) || (words & 3u) || (reinterpret_cast<uintptr_t>(c) & 1u) ||
      (reinterpret_cast<uintptr_t>(bias) & (bias_is_f32 ? 3u : 1u)) || !aligned16(workspace))
    return MDATTN_E_ALIGN;
  Plan plan = plan_of(M, N, K);
  MatmulArgs p{};
  p.a = (const uint8_t*)a; p.b = (const uint8_t*)b; p.sa = (const uint8_t*)a_scales; p.sb = (const uint8_t*)b_scales;
  p.bias = bias; p.bias_f32 = bias_is_f32; p.c = (__bf16*)c; p.c_stride = c_stride; p.M = M; p.N = N;
  p.ld = ceil_to(K, 128); p.ls = scale_stride(K); p.b_shift = b_block_rows == 128 ? 7 : 0;
  p.kb = (int)(p.ld / 128);
  if (plan.pieces > 1 && (!workspace || workspace_floats < floats_of(plan, M, N))) plan.pieces = 1, plan.kb_piece = (p.kb + 3) / 4 * 4;
  p.kb_piece = plan.kb_piece;
  p.part = plan.pieces > 1 ? workspace : nullptr;
  hipStream_t st = (hipStream_t)stream;
  const int rc = launch<128, 128>(st, p, plan.pieces);
  if (rc != MDATTN_OK || plan.pieces == 1) return rc;
  const int64_t groups = (M * N + 255) / 256;
  MDATTN_LAUNCH(join_pieces_kernel, dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(256), 0, st, workspace, plan.pieces, bias, bias_is_f32,
                (__bf16*)c, c_stride, M, N);
  return launch_status();
}

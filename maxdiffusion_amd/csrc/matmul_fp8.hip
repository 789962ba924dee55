// c [M, N] = a b^T + bias over e4m3 operands with one power-of-two scale per block of 128 along K:
//   c[m, n] = sum over k-blocks 2^(ea[m, kb] + eb[n, kb]) sum over k in kb qa[m, k] qb[n, k]
// The scales are operands of the matrix cores' scaled product (32 x 32 x 64): a block costs no instruction but the read of its byte.
#include <type_traits>

#include "mdattn_common.h"
#include "mdlayers.h"
#include "quant_block.h"

namespace mdattn {
namespace {

// acc += a b^T of 32 x 32 x 64, scaled by byte PH of sa and of sb.  As one statement with the accumulator in the accumulation registers, where
// the 256 of a wave's 128 x 128 just fit: the compiler's own form moved them about, and spilled.  The statement hides what
// it is from the compiler, so that the waits are here: two cycles between the vector ALU's write of an operand and its read (they cost
// nothing, the pipe being busy with the product before), and the ones after the last product.
template <int PH>
__device__ __forceinline__ void mfma(f32x16& acc, const i32x8& a, const i32x8& b, int sa, int sb) {
#define MDATTN_MFMA(SEL) \
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 " SEL : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb))
  if constexpr (PH == 0) MDATTN_MFMA("op_sel_hi:[0,0,0]");
  if constexpr (PH == 1) MDATTN_MFMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  if constexpr (PH == 2) MDATTN_MFMA("op_sel_hi:[1,1,0]");
  if constexpr (PH == 3) MDATTN_MFMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef MDATTN_MFMA
}

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

// a pointer that is the same in all lanes, in scalar registers whatever the compiler makes of the branches around it
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
  return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float bias_at(const void* p, int f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const __bf16*>(p)[i];
}

// One workgroup, four waves in 2 x 2, computes BM x BN.  A stage of LDS holds 128 bytes of each row of both tiles, written by
// direct loads; 16-byte chunk c of row r sits at c ^ ((r >> 1) & 7), which spreads 16 rows' reads of one chunk over all banks.  A step
// multiplies a stage in two halves of K: under the products of the first half the second half's fragments are read; then the one barrier
// of the step, by which the next stage has landed and this one has been read; under the products of the second half the next stage's first
// fragments are read and the stage after it is requested into the place of this one.  A matrix instruction keeps its pipe busy for 64
// cycles, in which the wave issues the reads and requests that stand behind it: their order is the program's (sched_barrier).
template <int BM, int BN>
__global__ __launch_bounds__(256) void matmul_fp8_kernel(MatmulArgs p) {
  constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 32, TN = WN / 32, kProducts = TM * TN;
  constexpr int kStage = (BM + BN) * 128, kScales = (BM + BN) * 4;
  constexpr int kLoads = (BM + BN) / 32;  // direct loads of a stage by one wave: 8 rows each
  constexpr int kScaleLoads = (BM + BN) / 256;
  constexpr int kLoadsPer = kLoads / kProducts;
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
  const uint8_t* a_at = uniform(p.a + m0 * p.ld + (int64_t)kb0 * 128);
  const uint8_t* b_at = uniform(p.b + n0 * p.ld + (int64_t)kb0 * 128);
  unsigned from[kLoads], from_s[kScaleLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {  // the first half of them are a's rows
    const int r = (wave + 4 * i) * 8 + (lane >> 3);
    const int64_t row = i < kLoads * BM / (BM + BN) ? min((int64_t)r, p.M - 1 - m0) : min((int64_t)r - BM, p.N - 1 - n0);
    from[i] = (unsigned)(row * p.ld + ((lane & 7) ^ ((r >> 1) & 7)) * 16);
  }
  const uint8_t* sa_at = uniform(p.sa + m0 * p.ls + kb0);
  const uint8_t* sb_at = uniform(p.sb + (n0 >> p.b_shift) * p.ls + kb0);
#pragma unroll
  for (int i = 0; i < kScaleLoads; ++i) {
    const int r = (wave + 4 * i) * 64 + lane;
    if (r < BM) from_s[i] = (unsigned)(min((int64_t)r, p.M - 1 - m0) * p.ls);
    else from_s[i] = (unsigned)(((min(n0 + r - BM, p.N - 1) >> p.b_shift) - (n0 >> p.b_shift)) * p.ls);
  }
  const unsigned lds = lds_addr_of(smem);
  auto request = [&](int stage, int i) {  // the i-th load of the next stage
    lds_dma16(i < kLoads * BM / (BM + BN) ? a_at : b_at, from[i], lds + stage * kStage + wave * 1024 + i * 4096);
  };
  int ahead = nk - 1;  // stages that are not requested yet; past the last one it is requested again, and not read
  auto requested = [&] {
    const int by = ahead > 0 ? 128 : 0;
    a_at = uniform(a_at + by);
    b_at = uniform(b_at + by);
    --ahead;
  };
  int scale_slot = 0;
  auto request_scales = [&] {  // of the next four stages, or the last ones again
    const unsigned to = __builtin_amdgcn_readfirstlane(lds + 2 * kStage + scale_slot * kScales + wave * 256);
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) lds_dma4((wave + 4 * i) * 64 < BM ? sa_at : sb_at, from_s[i], to + i * 1024);
    const int by = ahead > 3 ? 4 : 0;
    sa_at = uniform(sa_at + by);
    sb_at = uniform(sb_at + by);
    scale_slot ^= 1;
  };

  f32x16 acc[TN][TM];  // zeros, made where they stay: from the vector registers they would be copied in every pass of the loop
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m)
      asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_fp8_fp8 %0, %1, %1, 0" : "=a"(acc[n][m]) : "v"(0l));
  i32x8 fa[2][TM], fb[2][TN];
  int sa[TM], sb[TN];  // four stages' scale bytes
  // where this lane's 16-byte chunks of a fragment begin, by stage and half: the rest of an address is a constant of the instruction
  typedef const char __attribute__((address_space(3))) * Lds;
  Lds ra[2][2][2], rb[2][2][2];
#pragma unroll
  for (int stage = 0; stage < 2; ++stage)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int chunk = ((4 * j + 2 * hh + q) ^ ((l32 >> 1) & 7)) * 16 + stage * kStage;
        ra[stage][j][q] = (Lds)smem + (wm * WM + l32) * 128 + chunk;
        rb[stage][j][q] = (Lds)smem + (BM + wn * WN + l32) * 128 + chunk;
        asm volatile("" : "+v"(ra[stage][j][q]), "+v"(rb[stage][j][q]));
      }
  auto fragment = [&](const Lds (&at)[2], int off) {
    typedef const u32x4 __attribute__((address_space(3))) * Chunk;
    const u32x4 lo = *(Chunk)(at[0] + off), hi = *(Chunk)(at[1] + off);
    return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  // the i-th fragment of half j, in the order in which the products want them
  auto read = [&](int stage, int j, int i) {
    if (i == 0) fb[j][0] = fragment(rb[stage][j], 0);
    else if (i <= TM) fa[j][i - 1] = fragment(ra[stage][j], (i - 1) * 4096);
    else fb[j][i - TM] = fragment(rb[stage][j], (i - TM) * 4096);
  };
  auto read_scales = [&](int slot) {
    const char* s = smem + 2 * kStage + slot * kScales;
#pragma unroll
    for (int m = 0; m < TM; ++m) sa[m] = *reinterpret_cast<const int*>(s + (wm * WM + m * 32 + l32) * 4);
#pragma unroll
    for (int n = 0; n < TN; ++n) sb[n] = *reinterpret_cast<const int*>(s + (BM + wn * WN + n * 32 + l32) * 4);
  };
  auto everyone_has_it = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  // step k, PH = k & 3
  auto step = [&](auto ph) __attribute__((always_inline)) {
    constexpr int PH = decltype(ph)::value, kNow = PH & 1;
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      const int n = i / TM, m = i % TM;
      mfma<PH>(acc[n][m], fb[0][n], fa[0][m], sb[n], sa[m]);
      if (i < TM + TN) read(kNow, 1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    everyone_has_it();
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      const int n = i / TM, m = i % TM;
      mfma<PH>(acc[n][m], fb[1][n], fa[1][m], sb[n], sa[m]);
      if (i < TM + TN) read(kNow ^ 1, 0, i);
#pragma unroll
      for (int l = 0; l < kLoadsPer; ++l) request(kNow, i * kLoadsPer + l);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (PH == 2) request_scales();
    requested();
    if (PH == 3) read_scales(scale_slot ^ 1);
  };

#pragma unroll
  for (int i = 0; i < kLoads; ++i) request(0, i);
  request_scales();
  float* bias = reinterpret_cast<float*>(smem + 2 * (kStage + kScales));  // of the tile's columns, for the end
  if ((int)threadIdx.x < BN) bias[threadIdx.x] = p.bias && n0 + threadIdx.x < p.N ? bias_at(p.bias, p.bias_f32, n0 + threadIdx.x) : 0.f;
  requested();
  everyone_has_it();
#pragma unroll
  for (int i = 0; i < kLoads; ++i) request(1, i);
  requested();
  read_scales(0);
#pragma unroll
  for (int i = 0; i < TM + TN; ++i) read(0, 0, i);
  for (int left = nk;; left -= 4) {
    step(std::integral_constant<int, 0>{});
    if (left == 1) break;
    step(std::integral_constant<int, 1>{});
    if (left == 2) break;
    step(std::integral_constant<int, 2>{});
    if (left == 3) break;
    step(std::integral_constant<int, 3>{});
    if (left == 4) break;
  }
  asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");  // (the last product's result: 16 passes and a few)
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m) asm volatile("" : "+a"(acc[n][m]));  // nothing reads it above this

  // lane l32 holds output row m0 + .. + l32; register i of it column (i & 3) + 8 (i >> 2) + 4 hh of 32
  if (p.part) {
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const int64_t row = m0 + wm * WM + m * 32 + l32;
      if (row >= p.M) continue;
      float* o = p.part + ((int64_t)piece * p.M + row) * p.N;
#pragma unroll
      for (int n = 0; n < TN; ++n) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t col = n0 + wn * WN + n * 32 + 8 * q + 4 * hh;
          if (col + 4 <= p.N) {
            *reinterpret_cast<f32x4_any*>(o + col) = f32x4{acc[n][m][4 * q], acc[n][m][4 * q + 1], acc[n][m][4 * q + 2], acc[n][m][4 * q + 3]};
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < p.N) o[col + e] = acc[n][m][4 * q + e];
          }
        }
      }
    }
    return;
  }
  // The outputs by whole rows, through LDS: 32 rows of the wave at a time in a place of its own, the 16-byte chunk c of row r at
  // c ^ (r & (kChunks - 1)).  (Stored from the registers, 16 bytes of a row at a time, they took as long as 20 steps.)
  constexpr int kChunks = WN / 8;
  __syncthreads();
  char* mine = smem + wave * (32 * WN * 2);
  const bool wide = p.c_stride % 8 == 0 && p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.c) & 15) == 0;
#pragma unroll
  for (int m = 0; m < TM; ++m) {
#pragma unroll
    for (int n = 0; n < TN; ++n) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 b = *reinterpret_cast<const float4*>(bias + wn * WN + n * 32 + 8 * q + 4 * hh);
        const u32x2 v{pack2(acc[n][m][4 * q] + b.x, acc[n][m][4 * q + 1] + b.y), pack2(acc[n][m][4 * q + 2] + b.z, acc[n][m][4 * q + 3] + b.w)};
        *reinterpret_cast<u32x2*>(mine + l32 * (WN * 2) + (((n * 4 + q) ^ (l32 & (kChunks - 1))) * 16) + hh * 8) = v;
      }
    }
#pragma unroll
    for (int i = 0; i < kChunks / 2; ++i) {
      const int r = i * (64 / kChunks) + lane / kChunks, c = lane % kChunks;
      const u32x4 v = *reinterpret_cast<const u32x4*>(mine + r * (WN * 2) + ((c ^ (r & (kChunks - 1))) * 16));
      const int64_t row = m0 + wm * WM + m * 32 + r, col = n0 + wn * WN + c * 8;
      if (row >= p.M) continue;
      __bf16* o = p.c + row * p.c_stride + col;
      if (wide) {
        if (col < p.N) *reinterpret_cast<u32x4*>(o) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < p.N) reinterpret_cast<unsigned short*>(o)[e] = (unsigned short)(v[e / 2] >> (16 * (e & 1)));
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
  const int64_t big = (M + 255) / 256 * ((N + 255) / 256);
  return {big >= 192 ? 256 : 128, 1, (kb + 3) / 4 * 4};
}
int64_t floats_of(const Plan& p, int64_t M, int64_t N) { return p.pieces > 1 ? p.pieces * M * N : 0; }

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M > 0 && N > 0 && K > 0 && M < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && K <= (1 << 23) && (M + 127) / 128 * ((N + 127) / 128) < (1 << 27);
}

template <int BM, int BN>
int launch(hipStream_t st, MatmulArgs& a, int pieces) {
  constexpr int kBytes = 2 * ((BM + BN) * 128 + (BM + BN) * 4) + BN * 4;
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
  const int rc = plan.tile == 256 ? launch<256, 256>(st, p, plan.pieces) : launch<128, 128>(st, p, plan.pieces);
  if (rc != MDATTN_OK || plan.pieces == 1) return rc;
  const int64_t groups = (M * N + 255) / 256;
  MDATTN_LAUNCH(join_pieces_kernel, dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(256), 0, st, workspace, plan.pieces, bias, bias_is_f32,
                (__bf16*)c, c_stride, M, N);
  return launch_status();
}

// c [M, N] = a b^T + bias over e4m3 operands with one power-of-two scale per block of 128 along K:
//   c[m, n] = sum over k-blocks 2^(ea[m, kb] + eb[n, kb]) sum over k in kb qa[m, k] qb[n, k]
// The scales are operands of the matrix cores' scaled product (16 x 16 x 128, a block of K): a block costs no instruction but the read of its
// scales' word and a shift.
// Sums are f32, but for what the instruction does in each step: it aligns eight neighbouring products to the largest of them and cuts 14 bits
// below it, in every 8-bit form.  That is 1.6e-5 of a result, a 100th of what rounding it to bf16 loses; one result in 400 so rounds to the other side
// of where an f32 sum would, which makes 2.3e-4 of the outputs' length, and their distance from 64 bits, 1.7e-3, is that of the rounded f32 sums.
#include <type_traits>

#include "mdattn_common.h"
#include "mdlayers.h"
#include "quant_block.h"

namespace mdattn {
namespace {

// acc += a b^T of 16 x 16 x 128, scaled by the low bytes of sa and of sb.  As one statement with the accumulator in the accumulation registers,
// where the 256 of a wave's 128 x 128 just fit: the compiler's own form moved them about, and spilled.  The statement hides what it is from
// the compiler, so that the waits are here: two cycles between the vector ALU's write of an operand and its read (they cost nothing, the
// pipe being busy with the product before), and the ones after the last product.  (32 x 32 x 64 draws 5 % more power, which is what bounds a
// large product: 4.15 against 4.37 PFLOP/s from registers.)
__device__ __forceinline__ void mfma(f32x4& acc, const i32x8& a, const i32x8& b, int sa, int sb) {
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb));
}
// nothing reads a sum above this, not even to move it to a vector register
__device__ __forceinline__ void pin(f32x4& acc) { asm volatile("" : "+a"(acc)); }
__device__ __forceinline__ void mfma_zero(f32x4& acc) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_fp8_fp8 %0, %1, %1, 0" : "=a"(acc) : "v"(0l));
}

struct MatmulArgs {
  const uint8_t *a, *b, *sa, *sb;
  const void* bias;
  __bf16* c;
  float* part;       // split over K: each piece's f32 sums
  int64_t c_stride, M, N;
  int64_t ld, ls;    // bytes of an operand's row, and of a row of scales
  int b_shift, bias_f32;
  int kb, kb_piece;  // k-blocks, and those of a piece (a multiple of 4)
  int mt, nt, total;  // tiles: down, across, and with the pieces
  int wide;          // 16-byte stores of c
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

// What a workgroup keeps in LDS: two stages, sets of scale words (a set serves four stages, or a tile's last ones: as many sets as stages can be
// under way, and the one that is read), each wave's bias values and a place to turn its outputs.  Stages and sets follow one another in rings
// whose sizes are powers of two.
constexpr int kStages = 2;
template <int BM, int BN>
struct Layout {
  static constexpr int kStage = (BM + BN) * 128, kScales = (BM + BN) * 4, kSets = 4;
  static constexpr int kRing = kStages * kStage, kSetRing = kSets * kScales;
  static constexpr int kScaleAt = kRing;
  static constexpr int kBiasAt = kScaleAt + kSetRing;
  static constexpr int kCols = BN >= 256 ? 64 : 32;  // columns that are turned at a time
  static constexpr int kTurnAt = kBiasAt + 4 * (BN / 2) * 4;
  static constexpr int kBytes = kTurnAt + 4 * 32 * kCols * 2;
  static constexpr int kResident = 256 * (160 * 1024 / kBytes), kDieTiles = kResident / 8;
};

// The order of a product's tiles: down, then across, in bands of kBand rows of them.  A round of the resident workgroups so covers 16 rows and 16
// columns of tiles of 256, of which each die takes 8 and 4: the dies share what they read through the memory's own cache, and a round's part
// of both operands (32 x 256 rows of K bytes) stays in it up to a K of 30,000.  (Each die on a stretch of the order of its own, which reads
// the same through its L2, needs 8 such stretches' rows: 18,900 x 5,120 x 15,360 1,160 us against 1,067, 75,600 x 5,120 x 13,824 4,155
// against 3,763, 18,900 x 5,120 x 10,240 692 and 693.)
constexpr int kBand = 16, kDieRows = 8, kDiesDown = kBand / kDieRows;
struct TileAt {
  int m, n;
};
__device__ __forceinline__ TileAt tile_of(int id, int mt, int nt) {
  const int band = id / (kBand * nt), rows = min(mt - band * kBand, kBand), in = id - band * kBand * nt;
  return {band * kBand + in % rows, in / rows};
}

// A wave's sums to memory: of each 16 x 16, lane l holds row l % 16 and columns 4 (l / 16) to + 3.  By whole rows, through LDS: 32 rows x kCols
// columns at a time, 16-byte chunk c of row r at c ^ ((r >> 1) & (chunks - 1)).  (Stored from the registers, 16 bytes of a row at a time, they
// took as long as 20 steps.)  Rows whose 16-byte chunks are not aligned (N or c_stride no multiple of 8) go two bytes at a time: 2,674 x 5,121 x
// 2,048 53 us, 5,120 columns 31; 18,900 x 5,121 x 5,120 477 and 353.
template <int BM, int BN, int TM, int TN>
__device__ __forceinline__ void store_rows(const MatmulArgs& p, f32x4 (&acc)[TN][TM], char* smem, int64_t m0, int64_t n0, int lane, int wave) {
  using L = Layout<BM, BN>;
  constexpr int WM = BM / 2, WN = BN / 2;
  const int l16 = lane & 15, h = lane >> 4;
  m0 += (wave & 1) * WM;
  n0 += (wave >> 1) * WN;
  // LDS serves a wave's requests in order: a block's writes, its reads and the next block's writes follow one another unwaited, and a
  // block is stored while the next is turned.
  constexpr int kChunks = L::kCols / 8, kPasses = 32 * kChunks / 64, kRows = 64 / kChunks, kPart = L::kCols / 16, kDown = TM / 2, kBlocks = kDown * TN / kPart;
  float* bias = reinterpret_cast<float*>(smem + L::kBiasAt) + wave * WN;
#pragma unroll
  for (int i = 0; i < WN; i += 64) bias[i + lane] = p.bias && n0 + i + lane < p.N ? bias_at(p.bias, p.bias_f32, n0 + i + lane) : 0.f;
  char* mine = smem + L::kTurnAt + wave * (32 * L::kCols * 2);
  char* put = mine + l16 * (L::kCols * 2) + (h & 1) * 8;
  const int r0 = lane / kChunks, c0 = lane % kChunks, swap = (l16 >> 1) & (kChunks - 1);
  const char* get = mine + r0 * (L::kCols * 2);
  const int rows = (int)min(p.M - m0, (int64_t)WM), cols = (int)min(p.N - n0, (int64_t)WN);
  __bf16* out = p.c + (m0 + r0) * p.c_stride + n0 + c0 * 8;
  u32x4 v[2][kPasses];
  auto store = [&](int block) __attribute__((always_inline)) {
    const int m = block % kDown, col = block / kDown * L::kCols;
    const int left = c0 * 8 + col < cols ? rows - r0 - m * 32 : 0;  // rows of this lane's columns from here on
    __bf16* o = out + m * 32 * p.c_stride + col;
    if (p.wide) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        if (i * kRows < left) __builtin_nontemporal_store(v[block & 1][i], reinterpret_cast<u32x4*>(o + i * kRows * p.c_stride));
    } else {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const u32x4 x = v[block & 1][i];
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const unsigned word = e < 4 ? (e < 2 ? x[0] : x[1]) : (e < 6 ? x[2] : x[3]);
          if (i * kRows < left && c0 * 8 + col + e < cols)
            reinterpret_cast<unsigned short*>(o + i * kRows * p.c_stride)[e] = (unsigned short)(word >> (16 * (e & 1)));
        }
      }
    }
  };
  float4 b[kPart];
#pragma unroll
  for (int block = 0; block < kBlocks; ++block) {
    const int m0s = block % kDown * 2, n1 = block / kDown * kPart;
    if (m0s == 0) {
#pragma unroll
      for (int n = 0; n < kPart; ++n) b[n] = *reinterpret_cast<const float4*>(bias + (n1 + n) * 16 + 4 * h);
    }
#pragma unroll
    for (int n = 0; n < kPart; ++n)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        f32x4& f = acc[n1 + n][m0s + m];
        pin(f);
        *reinterpret_cast<u32x2*>(put + m * (16 * L::kCols * 2) + ((n * 2 + (h >> 1)) ^ swap) * 16) =
            u32x2{pack2(f[0] + b[n].x, f[1] + b[n].y), pack2(f[2] + b[n].z, f[3] + b[n].w)};
      }
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
      v[block & 1][i] = *reinterpret_cast<const u32x4*>(get + i * (kRows * L::kCols * 2) + ((c0 ^ (((i * kRows + r0) >> 1) & (kChunks - 1))) * 16));
    if (block) store(block - 1);
    __builtin_amdgcn_sched_barrier(0);
  }
  store(kBlocks - 1);
}

// A piece's sums in the order of the registers, whole and in f32: [piece][tile][wave][n][m][lane], four columns each (join_pieces_kernel)
template <int BM, int BN, int TM, int TN>
__device__ __forceinline__ void store_piece(const MatmulArgs& p, f32x4 (&acc)[TN][TM], int tile, int piece, int lane, int wave) {
  f32x4* o = reinterpret_cast<f32x4*>(p.part) + ((int64_t)piece * (p.mt * p.nt) + tile) * (BM * BN / 4) + wave * (BM * BN / 16) + lane;
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      pin(acc[n][m]);
      o[(n * TM + m) * 64] = acc[n][m];
    }
}

// A workgroup of four waves in 2 x 2 computes BM x BN at a time, and as many such tiles as it takes for the resident workgroups to get through
// all of them.  A stage of LDS holds 128 bytes of each row of both operands, written by direct loads; 16-byte chunk c of row r sits at
// c ^ ((r >> 1) & 7), which spreads 16 rows' reads of one chunk over all banks.  A step multiplies all of a wave's rows of a with the
// first half of its rows of b, then with the second.  Under the products of the first half the stage's second fragments are read (the lower half
// of a wave's rows has the first ones), and the lower halves of the stage two further on are requested into the place of this one's, which
// all waves have read; under the products of the second half the next stage's first fragments are read, each into the registers of one that
// has been used up, and the upper halves are requested.  A barrier ends each half.  So the requests are spread evenly (a CU takes 64 bytes a
// cycle, half of a step's cycles for its 64 KB: all of them under one half stood in each other's way and the products'), and each has a
// whole step to land: 75,600 x 5,120 x 5,120 on zeros, where power is no limit, 1,320 us with one barrier a step and the requests in its
// second half, 1,191 so; on normal numbers 1,525 and 1,481.
// Bound by the matrix cores under the chip's power limit: 75,600 x 5,120 x 5,120 at 2.7 PFLOP/s, on zeros at 3.4.  Of what is left on zeros,
// the barriers cost 4 %, the requests 2 to 11 % (the longer K, the more comes from beyond L2), the stores of the outputs 1 to 6 %, turning
// them 2.5 us a tile; the waits for what was requested nothing.
// A matrix instruction keeps its pipe busy for 32 cycles, in which the wave issues the reads and requests that stand behind it: their order is
// the program's (sched_barrier).  The stages are one stream over a workgroup's tiles: while the outputs of one tile are stored, the first
// stages of the next are on their way.
template <int BM, int BN, bool PIECES>
__global__ __launch_bounds__(256) void matmul_fp8_kernel(MatmulArgs p) {
  using L = Layout<BM, BN>;
  constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16, HM = TM / 2, HN = TN / 2, kProducts = TM * HN;
  constexpr int kLoads = (BM + BN) / 32;  // direct loads of a stage by one wave: 8 rows each; the first of them a's rows
  constexpr int kLoadsA = BM / 32;
  constexpr int kScaleLoads = (BM + BN) / 256;
  constexpr int kReads = HM + HN;         // fragments that are read under half a step's products
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, h = lane >> 4, wm = wave & 1, wn = wave >> 1;

  // Round by round, as many tiles as there are resident workgroups, in the order of tile_of; of a last, smaller round each die takes a
  // contiguous eighth.
  struct Tile {
    int64_t m0, n0;
    int tile, piece, kb0, nk;
  };
  constexpr int kResident = L::kResident, kWide = L::kDieTiles / kDieRows;
  const int die = blockIdx.x & 7, slot = blockIdx.x >> 3;  // neighbouring workgroups sit on different dies
  const int full = p.total / kResident, rest = p.total % kResident, rest_die = (rest + 7) / 8;
  const int in_full = ((die / kDiesDown) * kWide + slot / kDieRows) * kBand + (die % kDiesDown) * kDieRows + slot % kDieRows;
  const int in_rest = die * rest_die + slot;
  const int last = full + (slot < rest_die && in_rest < rest);  // rounds of this workgroup
  auto tile_at = [&](int round) {
    int id = round * kResident + (round < full ? in_full : in_rest);
    Tile t;
    t.piece = id / (p.mt * p.nt);
    id -= t.piece * p.mt * p.nt;
    t.tile = id;
    const TileAt at = tile_of(id, p.mt, p.nt);
    t.m0 = (int64_t)at.m * BM;
    t.n0 = (int64_t)at.n * BN;
    t.kb0 = t.piece * p.kb_piece;
    t.nk = min(p.kb_piece, p.kb - t.kb0);
    return t;
  };
  int round = 0;
  if (last == 0) return;

  // what this lane loads: byte offsets from the tile's first row (rows past the end read the last one; they are not stored)
  unsigned from[kLoads], from_s[kScaleLoads];
  const uint8_t *a_at, *b_at, *sa_at, *sb_at;
  int to_request, requested_of_tile;
  auto aim = [&](const Tile& t) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (wave + 4 * i) * 8 + (lane >> 3);
      const int row = i < kLoadsA ? min(r, (int)min(p.M - 1 - t.m0, (int64_t)BM)) : min(r - BM, (int)min(p.N - 1 - t.n0, (int64_t)BN));
      from[i] = (unsigned)row * (unsigned)p.ld + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
      const int r = (wave + 4 * i) * 64 + lane;
      const int row = r < BM ? min(r, (int)min(p.M - 1 - t.m0, (int64_t)BM))
                             : (min(r - BM, (int)min(p.N - 1 - t.n0, (int64_t)BN)) + (int)(t.n0 & ((1 << p.b_shift) - 1))) >> p.b_shift;
      from_s[i] = (unsigned)row * (unsigned)p.ls;
    }
    a_at = uniform(p.a + t.m0 * p.ld + (int64_t)t.kb0 * 128);
    b_at = uniform(p.b + t.n0 * p.ld + (int64_t)t.kb0 * 128);
    sa_at = uniform(p.sa + t.m0 * p.ls + t.kb0);
    sb_at = uniform(p.sb + (t.n0 >> p.b_shift) * p.ls + t.kb0);
    to_request = t.nk;
    requested_of_tile = 0;
  };
  const unsigned lds = lds_addr_of(smem);  // (0: a kernel's only LDS)
  unsigned place = lds + wave * 1024;      // of the stage that is requested next
  auto request = [&](int i) {  // its i-th load
    lds_dma16(i < kLoadsA ? a_at : b_at, from[i], (unsigned)__builtin_amdgcn_readfirstlane(place + i * 4096));
  };
  // the order of a stage's loads: first the rows that a wave's first fragments are in, the lower half of its rows of a and of b
  auto load_of = [](int l) {
    constexpr int kRun = BM / 128;  // loads of half a wave's rows
    const int in = l % (kLoads / 2);
    return in / kRun * 2 * kRun + l / (kLoads / 2) * kRun + in % kRun;
  };
  unsigned scale_place = wave * 256;
  int aimed = 0;  // the round whose tile's stages are being requested; past the last one, that one again
  auto request_scales = [&] {  // of four stages, with the first of them
    if ((requested_of_tile & 3) == 0) {
#pragma unroll
      for (int i = 0; i < kScaleLoads; ++i)
        lds_dma4((wave + 4 * i) * 64 < BM ? sa_at : sb_at, from_s[i], (unsigned)__builtin_amdgcn_readfirstlane(lds + L::kScaleAt + scale_place + i * 1024));
      sa_at = uniform(sa_at + 4);
      sb_at = uniform(sb_at + 4);
      scale_place = (scale_place + L::kScales) & (L::kSetRing - 1);
    }
  };
  auto advance = [&] {
    a_at = uniform(a_at + 128);
    b_at = uniform(b_at + 128);
    place = (place + L::kStage) & (L::kRing - 1);
  };
  auto count = [&] {
    ++requested_of_tile;
    if (--to_request == 0) {
      ++aimed;
      aim(tile_at(min(aimed, last - 1)));
    }
  };

  f32x4 acc[TN][TM];
  i32x8 fa[TM], fb[TN];
  int sa[TM], sb[TN];
  // where this lane's two 16-byte chunks of a fragment, and its scale, are in the stage that is read: the rest of an address is a constant of
  // the instruction.  (Chunks h and h + 4: which bytes of a block meet in which lane is free where it is the same for a and b.  The read
  // serves lanes of different h together: with chunks 2 h and 2 h + 1 they met in their banks, 8.1 cycles a read against 4.3.)
  typedef const char __attribute__((address_space(3))) * Lds;
  typedef const u32x4 __attribute__((address_space(3))) * Quad;
  typedef const int __attribute__((address_space(3))) * Word;
  unsigned ra[2], rb[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int chunk = ((h + 4 * q) ^ ((l16 >> 1) & 7)) * 16;
    ra[q] = lds + (wm * WM + l16) * 128 + chunk;
    rb[q] = lds + (BM + wn * WN + l16) * 128 + chunk;
  }
  const unsigned rsa = lds + L::kScaleAt + (wm * WM + l16) * 4, rsb = lds + L::kScaleAt + (BM + wn * WN + l16) * 4;
  unsigned set = 0;  // of scales, the one that is read
  auto read_a = [&](int m) {
    const u32x4 lo = *(Quad)((Lds)(uintptr_t)ra[0] + m * 2048), hi = *(Quad)((Lds)(uintptr_t)ra[1] + m * 2048);
    fa[m] = i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  auto read_b = [&](int n) {
    const u32x4 lo = *(Quad)((Lds)(uintptr_t)rb[0] + n * 2048), hi = *(Quad)((Lds)(uintptr_t)rb[1] + n * 2048);
    fb[n] = i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  // the scales of the first fragments (half 0) or of the second: words of four steps, shifted where they are used
  auto read_scales = [&](int half) {
#pragma unroll
    for (int m = 0; m < HM; ++m) sa[half * HM + m] = *((Word)(uintptr_t)(rsa + set) + (half * HM + m) * 16);
#pragma unroll
    for (int n = 0; n < HN; ++n) sb[half * HN + n] = *((Word)(uintptr_t)(rsb + set) + (half * HN + n) * 16);
  };
  // the half of the next stage that is read next has landed (behind its loads there are at least those of a stage), and this wave has
  // what it read: in all waves
  auto everyone_has_it = [] { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((kStages - 1) * kLoads) : "memory"); };

  Tile t = tile_at(0);
  aim(t);
#pragma unroll
  for (int s = 0; s < kStages; ++s) {
    request_scales();
#pragma unroll
    for (int l = 0; l < kLoads; ++l) request(load_of(l));
    advance();
    count();
  }
  everyone_has_it();
#pragma unroll
  for (int m = 0; m < HM; ++m) read_a(m);
#pragma unroll
  for (int n = 0; n < HN; ++n) read_b(n);
  read_scales(0);
  everyone_has_it();
  for (;;) {
    // zeros, made where they stay: from the vector registers they would be copied in every pass of the loop
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int m = 0; m < TM; ++m) mfma_zero(acc[n][m]);
#pragma unroll 1
    for (int k = 0; k < t.nk; ++k) {
      const int shift = 8 * (k & 3);
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        const int m = i / HN, n = i % HN;
        mfma(acc[n][m], fb[n], fa[m], sb[n] >> shift, sa[m] >> shift);
        if (i == 0) {
          if (shift == 0) read_scales(1);
          request_scales();
        }
#pragma unroll
        for (int r = 0; r < kReads; ++r)  // a's first: their products come in this half.  Done by three quarters: the barrier waits for them
          if (r * 3 * kProducts / 4 / kReads == i) {
            if (r < HM) read_a(HM + r);
            else read_b(HN + r - HM);
          }
#pragma unroll
        for (int l = 0; l < kLoads / 2; ++l)
          if ((2 * l + 1) * kProducts / kLoads == i) request(load_of(l));
        __builtin_amdgcn_sched_barrier(0);
      }
      everyone_has_it();
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        const int m = i / HN, n = HN + i % HN;
        mfma(acc[n][m], fb[n], fa[m], sb[n] >> shift, sa[m] >> shift);
        if (i == 0) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            ra[q] ^= L::kStage;
            rb[q] ^= L::kStage;
          }
        }
#pragma unroll
        for (int r = 0; r < kReads; ++r)  // b's and a's in turn, a's behind the products that use up what was there
          if (r * 3 * kProducts / 4 / kReads == i) {
            if (r % 2 == 0) read_b(r / 2);
            else read_a(r / 2);
          }
        if (i == 3 * kProducts / 4 && (k + 1 == t.nk || shift == 24)) {
          set = (set + L::kScales) & (L::kSetRing - 1);
          read_scales(0);
        }
#pragma unroll
        for (int l = 0; l < kLoads / 2; ++l)
          if (2 * l * kProducts / kLoads == i) request(load_of(kLoads / 2 + l));
        if (i == kProducts - 2) advance();
        if (i == kProducts - 1) count();
        __builtin_amdgcn_sched_barrier(0);
      }
      everyone_has_it();
    }
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // (the last product's result: 16 passes and a few)
    if constexpr (PIECES) {
      store_piece<BM, BN>(p, acc, t.tile, t.piece, lane, wave);
    } else {
      store_rows<BM, BN>(p, acc, smem, t.m0, t.n0, lane, wave);
    }
    if (++round >= last) break;
    t = tile_at(round);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was requested past the end
}

// the pieces of a product that was split over K, in their order, then the bias.  A thread takes four columns of a row in each piece, 16
// bytes where store_piece left them.
template <int BM, int BN>
__global__ __launch_bounds__(256) void join_pieces_kernel(MatmulArgs p, int pieces) {
  constexpr int TM = BM / 32, TN = BN / 32;
  const int tile = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
  const int lane = i & 63, m = (i >> 6) % TM, n = (i >> 6) / TM % TN, wave = i / (BM * BN / 16);
  const TileAt t = tile_of(tile, p.mt, p.nt);
  const int64_t row = (int64_t)t.m * BM + (wave & 1) * (BM / 2) + m * 16 + (lane & 15);
  const int64_t col = (int64_t)t.n * BN + (wave >> 1) * (BN / 2) + n * 16 + 4 * (lane >> 4);
  if (row >= p.M || col >= p.N) return;
  const f32x4* at = reinterpret_cast<const f32x4*>(p.part) + (int64_t)tile * (BM * BN / 4) + i;
  const int64_t step = (int64_t)p.mt * p.nt * (BM * BN / 4);
  f32x4 s = at[0];
  for (int j = 1; j < pieces; ++j) s += at[j * step];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (p.bias && col + e < p.N) s[e] += bias_at(p.bias, p.bias_f32, col + e);
  __bf16* o = p.c + row * p.c_stride + col;
  if (p.wide) {
    *reinterpret_cast<u32x2*>(o) = u32x2{pack2(s[0], s[1]), pack2(s[2], s[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < p.N) o[e] = (__bf16)s[e];
  }
}

// Few rows of a: bound by b's bytes, which pass straight from memory to the registers of the one wave that multiplies them (16 x 16 x 128: a
// load covers 64 bytes of each of 16 rows; of 32 rows, 32 bytes, it was 20 % slower): 1 x 5,120 by 30,720 rows, 157 MB, 27 us, 5.8 TB/s.  A workgroup takes 16 rows of b and all of a's, 16 TM
// at most; its waves share K out in groups of four blocks, a scale word's, and their sums meet in LDS in a fixed order.
template <int TM, int W>
__global__ __launch_bounds__(64 * W) void matmul_fp8_rows_kernel(MatmulArgs p) {
  __shared__ f32x4 part[W][TM][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, h = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t brow = min(n0 + l16, p.N - 1);
  const uint8_t* b = p.b + brow * p.ld + h * 16;
  const uint8_t* sb = p.sb + (brow >> p.b_shift) * p.ls;
  const uint8_t* a[TM];
  const uint8_t* sa[TM];
  f32x4 acc[TM];
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int64_t row = min((int64_t)(m * 16 + l16), p.M - 1);
    a[m] = p.a + row * p.ld + h * 16;
    sa[m] = p.sa + row * p.ls;
    acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // this lane's 32 bytes of a block (which of a block's bytes meet in which lane is the same for a and b)
  auto operand = [](const uint8_t* at) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(at), hi = *reinterpret_cast<const u32x4*>(at + 64);
    return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  for (int g = wave; g * 4 < p.kb; g += W) {
    const int sbw = *reinterpret_cast<const int*>(sb + g * 4);
    int saw[TM];
#pragma unroll
    for (int m = 0; m < TM; ++m) saw[m] = *reinterpret_cast<const int*>(sa[m] + g * 4);
    auto block = [&](auto i) __attribute__((always_inline)) {
      constexpr int I = decltype(i)::value;
      const int64_t at = (int64_t)(g * 4 + I) * 128;
      const i32x8 fb = operand(b + at);
#pragma unroll
      for (int m = 0; m < TM; ++m) acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, operand(a[m] + at), acc[m], 0, 0, I, sbw, I, saw[m]);
    };
    using std::integral_constant;
    if (g * 4 + 4 <= p.kb) {
      block(integral_constant<int, 0>{});
      block(integral_constant<int, 1>{});
      block(integral_constant<int, 2>{});
      block(integral_constant<int, 3>{});
    } else {
      block(integral_constant<int, 0>{});
      if (g * 4 + 1 < p.kb) block(integral_constant<int, 1>{});
      if (g * 4 + 2 < p.kb) block(integral_constant<int, 2>{});
    }
  }
#pragma unroll
  for (int m = 0; m < TM; ++m) part[wave][m][lane] = acc[m];
  __syncthreads();
  if (threadIdx.x >= TM * 64) return;
  const int64_t row = wave * 16 + l16, col = n0 + 4 * h;  // (wave: the 16 rows that it sums)
  if (row >= p.M || col >= p.N) return;
  f32x4 s = part[0][wave][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) s += part[w][wave][lane];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (p.bias && col + e < p.N) s[e] += bias_at(p.bias, p.bias_f32, col + e);
  __bf16* o = p.c + row * p.c_stride + col;
  if (p.wide) {
    *reinterpret_cast<u32x2*>(o) = u32x2{pack2(s[0], s[1]), pack2(s[2], s[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < p.N) o[e] = (__bf16)s[e];
  }
}

// How a product is run: tiles of so many rows and columns (0: matmul_fp8_rows_kernel), pieces of K, and k-blocks of a piece.
struct Plan {
  int tile, pieces, kb_piece;
  double us;
};
constexpr int kFewRows = 32;
constexpr int kAlone = 256;  // tiles of 128 by whose number each has its CU to itself
// The fastest by a model of steps of 128 of K, of a tile's time beside them, and of the pieces' sums.  Its constants (a step 1.42 us in a tile of
// 256, 0.57 in one of 128 that has its CU to itself, 1.0 where two share it; 8 and 4 us beside the steps; the sums at 1.4 TB/s) compare the
// forms; as times they are upper bounds, by up to 45 %.  Measured now: a step 1.35 us in a tile of 256 (1.0 while most CUs are idle, and the
// clock is higher), 0.42 and 0.85 in one of 128; beside the steps 5 us and 3 more for the first tile of 256, 4.4 and 3.6; the sums 3.2 TB/s.  Each of 26
// products from 64 x 5,120 x 5,120 to 32,760 x 4,608 x 1,536 was forced through both tiles in 1 to 8 pieces: what is chosen here was the fastest or within
// 5 % of it.  (4,096^3: tiles of 256 52 us, of 128 61; 4,680 x 4,608 x 1,536 40 and 38; 1,000 x 1,000 x 16,384: 64 tiles of 128 whole 56, in
// four pieces 25.)
Plan plan_of(int64_t M, int64_t N, int64_t K) {
  const int kb = (int)((K + 127) / 128);
  if (M <= kFewRows && grid_fits((N + 15) / 16, 512)) return {0, 1, kb, 4.0 + (double)N * K / 3e6};
  Plan best{128, 1, (kb + 3) / 4 * 4, 1e30};
  for (int tile = 128; tile <= 256; tile += 128) {
    const int64_t tiles = (M + tile - 1) / tile * ((N + tile - 1) / tile);
    for (int pieces = 1; pieces <= 64 && pieces * 4 < kb + 4; ++pieces) {
      const int per = ((kb + pieces - 1) / pieces + 3) / 4 * 4, made = (kb + per - 1) / per;
      if (made != pieces) continue;
      if (pieces > 1 && tiles * pieces > 1024) break;
      const int64_t all = tiles * pieces, resident = tile == 256 ? 256 : 512;
      const double step = tile == 256 ? 1.42 : all <= kAlone ? 0.57 : 1.0;
      double us = (double)((all + resident - 1) / resident) * ((tile == 256 ? 8.0 : 4.0) + step * (pieces == 1 ? kb : per));
      if (pieces > 1) us += 2.0 + (double)all * tile * tile * 4 / 1.4e6;
      if (us < best.us) best = {tile, pieces, per, us};
    }
  }
  return best;
}
// Rows of c that go first, in tiles of 256 and whole rounds of them, where what remains is faster by a plan of its own than as one more round
// that leaves most of the chip idle; 0: all go together.  (75,600 x 5,120 x 5,120, 23.1 rounds: 1,395 us and 1,386;
// 4,200 x 5,120 x 13,824, 1.3 rounds: 262 and 236; 4,160 x 4,160 x 5,120 104 and 79.)
int64_t rows_first(const Plan& all, int64_t M, int64_t N, int64_t K) {
  const int64_t nt = (N + 255) / 256, tiles = (M + 255) / 256 * nt;
  if (all.tile != 256 || all.pieces != 1 || tiles <= 256) return 0;
  const int64_t first = tiles / 256 * 256 / nt * 256;
  if (first == 0 || first >= M) return 0;
  const double us = 2.0 + plan_of(first, N, K).us + plan_of(M - first, N, K).us;
  return us < all.us ? first : 0;
}
int64_t floats_of(const Plan& p, int64_t M, int64_t N) { return p.pieces > 1 ? p.pieces * ceil_to(M, p.tile) * ceil_to(N, p.tile) : 0; }

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M > 0 && N > 0 && K > 0 && M < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && K <= (1 << 23) && (M + 127) / 128 * ((N + 127) / 128) < (1 << 27);
}

template <int BM, int BN, bool PIECES>
int launch(hipStream_t st, const MatmulArgs& a) {
  using L = Layout<BM, BN>;
  constexpr int kBytes = L::kBytes;
  static LdsOptIn flag;
  const int rc = lds_opt_in(flag, reinterpret_cast<const void*>(&matmul_fp8_kernel<BM, BN, PIECES>), kBytes);
  if (rc != MDATTN_OK) return rc;
  const int grid = a.total < L::kResident ? (a.total + 7) / 8 * 8 : L::kResident;
  MDATTN_LAUNCH((matmul_fp8_kernel<BM, BN, PIECES>), dim3((unsigned)grid), dim3(256), kBytes, st, a);
  return launch_status();
}
template <int BM, int BN>
int launch_tiles(hipStream_t st, MatmulArgs& a, int pieces) {
  a.mt = (int)((a.M + BM - 1) / BM);
  a.nt = (int)((a.N + BN - 1) / BN);
  a.total = a.mt * a.nt * pieces;
  if (pieces == 1) return launch<BM, BN, false>(st, a);
  if (a.mt * a.nt > 65535) return MDATTN_E_UNSUPPORTED;  // (only few tiles are split)
  const int rc = launch<BM, BN, true>(st, a);
  if (rc != MDATTN_OK) return rc;
  MDATTN_LAUNCH((join_pieces_kernel<BM, BN>), dim3(BM * BN / 1024, (unsigned)(a.mt * a.nt)), dim3(256), 0, st, a, pieces);
  return launch_status();
}

int run(hipStream_t st, MatmulArgs p, Plan plan, int64_t workspace_floats, float* workspace) {
  if (plan.pieces > 1 && (!workspace || workspace_floats < floats_of(plan, p.M, p.N))) plan.pieces = 1, plan.kb_piece = (p.kb + 3) / 4 * 4;
  p.kb_piece = plan.kb_piece;
  p.part = plan.pieces > 1 ? workspace : nullptr;
  if (plan.tile == 0) {
    const dim3 grid((unsigned)((p.N + 15) / 16));
    if (p.M <= 16) MDATTN_LAUNCH((matmul_fp8_rows_kernel<1, 8>), grid, dim3(512), 0, st, p);
    else MDATTN_LAUNCH((matmul_fp8_rows_kernel<2, 8>), grid, dim3(512), 0, st, p);
    return launch_status();
  }
  return plan.tile == 256 ? launch_tiles<256, 256>(st, p, plan.pieces) : launch_tiles<128, 128>(st, p, plan.pieces);
}

}  // namespace
}  // namespace mdattn

using namespace mdattn;

extern "C" int64_t mdattn_matmul_fp8_block_workspace_floats(int64_t M, int64_t N, int64_t K) {
  if (!sizes_ok(M, N, K)) return 0;
  const Plan all = plan_of(M, N, K);
  const int64_t first = rows_first(all, M, N, K);
  return first ? floats_of(plan_of(M - first, N, K), M - first, N) : floats_of(all, M, N);
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
  MatmulArgs p{};
  p.a = (const uint8_t*)a; p.b = (const uint8_t*)b; p.sa = (const uint8_t*)a_scales; p.sb = (const uint8_t*)b_scales;
  p.bias = bias; p.bias_f32 = bias_is_f32; p.c = (__bf16*)c; p.c_stride = c_stride; p.M = M; p.N = N;
  p.ld = ceil_to(K, 128); p.ls = scale_stride(K); p.b_shift = b_block_rows == 128 ? 7 : 0;
  p.kb = (int)(p.ld / 128);
  p.wide = c_stride % 8 == 0 && N % 8 == 0 && aligned16(c);
  hipStream_t st = (hipStream_t)stream;
  const Plan all = plan_of(M, N, K);
  const int64_t first = rows_first(all, M, N, K);
  if (!first) return run(st, p, all, workspace_floats, workspace);
  p.M = first;
  const int rc = run(st, p, {256, 1, (p.kb + 3) / 4 * 4, 0}, 0, nullptr);
  if (rc != MDATTN_OK) return rc;
  p.a += first * p.ld;
  p.sa += first * p.ls;
  p.c += first * c_stride;
  p.M = M - first;
  return run(st, p, plan_of(p.M, N, K), workspace_floats, workspace);
}

// Backward pass of attention over packed sequences (attn_packed.hip) for gfx950 (MI355X), bf16 MFMA.  With s = scale q.k, p = exp(s - lse),
// dp = dout.v, delta = rowsum(dout out):
//   dv = p^T dout,   ds = p (dp - delta),   dq = scale ds k,   dk = scale ds^T q,   dk and dv over all heads of a group.
//
// Two passes, no atomics: every gradient is accumulated by the waves that own its rows.
//   dq pass       a wave owns 32 rows of a group (head r % G of token r / G), their q and dout in registers, and walks the keys they see.
//                 It leaves -lse / scale and -delta of its rows, which start the MFMA chains that they are subtracted from.
//   dk / dv pass  a wave owns 32 keys, their k and v in registers, and walks the tokens that see them, head after head of the group: the sum over
//                 the heads is the same accumulator.  S and dP are formed in both passes: seven matrix products where five are necessary.
// Tiles of 32 rows pass through a ring of two slots in LDS, filled by direct global -> LDS loads.  Per tile, with the forward's fragments:
// S^T or S and dP by row reads, then the accumulation by transposing reads; W = P or dS is packed to bf16 as the B operand it already is.
// Blocks that no row of a wave sees, or no key of it is seen by, are not computed.
// The dk / dv pass has a workgroup per 128 keys and head of k and v, of which the first ones of a causal sequence walk all of its tokens in every
// head: these walks are cut into pieces, whose f32 sums a third kernel adds up in their order.
// Roundings.  P and dS go into their products in bf16.  delta takes out and what its rounding left (rest): dS = p (dp - delta) is small beside both
// where a key has most of a row's weight, and with the rounded out alone dq of sequences of 3, 8, 64 and 600 tokens, causal, with a direction that all
// logits share, is off by 8.1, 6.3, 3.9 and 2.8e-3 of its size, with rest by 2.5, 2.5, 2.4 and 2.4 (its own rounding 1.7).  dS in two parts would
// bring that to 1.7, for a third more matrix products.
// Bound.  A tile costs LDS as many cycles as the matrix pipes: 1 KB of fragments read per product of 32 cycles and wave, 128 bytes a cycle with
// four waves.  100 to 4,096 tokens x 8 sequences, 32 heads on 8, causal: dq 229 us (1.01 PFLOP/s, pipes busy 50 % of the cycles), dk / dv 358 us
// (0.86, 41 %), the pieces' sums 32 us; 8,192 tokens at head dim 64 385, 594 and 34 us (1.07 and 0.93 PFLOP/s).
#include <algorithm>
#include <cmath>

#include "attn_packed.h"
#include "mdattn_host.h"

namespace mdattn {
namespace {

struct PackedBwdArgs {
  const __bf16 *q, *k, *v, *out, *rest, *dout;
  const float* lse;
  __bf16 *dq, *dk, *dv;
  float* aux;  // [2][heads][q_rows]: -lse / scale, -delta
  PackedSeqs seqs;
  Divisor group;
  int kv_heads, D, causal;
  RowStrides qs, ks, vs, os, dqs, dks, dvs;
  float c, scale;
  int pieces, piece_tiles;  // of the dk / dv pass, tiles of 32 tokens
  float* part;             // [piece][2][kv_heads][k_rows][D]
};

template <int HD>
constexpr int bwd_slot(bool aux) { return 2 * PackedBlock<HD>::Bytes + (aux ? 256 : 0); }

// A wave's 32 rows of a gradient, 64 columns at a time through `stage`: as the accumulators lie, a store would touch 16 bytes of each of 32
// rows.  at(row) is the address of a row's first element.
constexpr int kStageRow = 64 * 2 + 16, kStageRows = 32 * kStageRow;
template <int ND, bool PADDED, class At>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[ND], float mul, int row0, int rows, int D, int lane, char* stage, At at) {
  const int l32 = lane & 31, hh = lane >> 5, rr = lane >> 3, cc = lane & 7;
#pragma unroll
  for (int d0 = 0; d0 < ND; d0 += 2) {
    // LDS accesses of one wave execute in order: the reads see the writes above them, and the next round's writes follow
#pragma unroll
    for (int db = d0; db < (d0 + 2 < ND ? d0 + 2 : ND); ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint2 u;
        u.x = pack2(acc[db][4 * g] * mul, acc[db][4 * g + 1] * mul);
        u.y = pack2(acc[db][4 * g + 2] * mul, acc[db][4 * g + 3] * mul);
        *reinterpret_cast<uint2*>(stage + l32 * kStageRow + ((db - d0) * 32 + 8 * g + 4 * hh) * 2) = u;
      }
    const int col = d0 * 32 + cc * 8;
    if (col >= (PADDED ? D : ND * 32)) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + 8 * j + rr;
      const uint4 u = *reinterpret_cast<const uint4*>(stage + (8 * j + rr) * kStageRow + cc * 16);
      if (row < rows) *reinterpret_cast<uint4*>(at(row) + col) = u;
    }
  }
}
// The same for f32 partial sums [rows][D], 32 columns at a time.
template <int ND, bool PADDED>
__device__ __forceinline__ void store_partial(const f32x16 (&acc)[ND], float mul, float* base, int row0, int rows, int D, int lane, char* stage) {
  const int l32 = lane & 31, hh = lane >> 5, rr = lane >> 3, cc = lane & 7;
#pragma unroll
  for (int db = 0; db < ND; ++db) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(stage + l32 * kStageRow + (8 * g + 4 * hh) * 4) =
          f32x4{acc[db][4 * g] * mul, acc[db][4 * g + 1] * mul, acc[db][4 * g + 2] * mul, acc[db][4 * g + 3] * mul};
    const int col = db * 32 + cc * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + 8 * j + rr;
      const f32x4 u = *reinterpret_cast<const f32x4*>(stage + (8 * j + rr) * kStageRow + cc * 16);
      if (row < rows && (!PADDED || col < D)) *reinterpret_cast<f32x4*>(base + (int64_t)row * D + col) = u;
    }
  }
}

template <bool PADDED>
__device__ __forceinline__ bf16x8 load_frag(const __bf16* p, int col, int D) {
  return !PADDED || col < D ? *reinterpret_cast<const bf16x8*>(p + col) : __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
}

// A wave in its products goes before the other in its softmax (one sequence of 4,096 to 8,192 tokens 1 to 2.5 % faster; at head dim 64, where three share
// the pipes, short calls 5 % slower: left out).
template <int HD>
__device__ __forceinline__ void priority(int high) {
  if constexpr (HD == 128) {
    if (high) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
  }
}

// ---------------------------------------------------------------------------------------------------------------------- dq
template <int HD, int DC, bool PADDED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 3 : 2, HD == 64 ? 3 : 2))) void packed_dq_kernel(PackedBwdArgs a) {
  using T = PackedBlock<HD>;
  constexpr int NJ = DC / 16, ND = (DC + 31) / 32, kSlot = bwd_slot<HD>(false), GPW = 32 / T::RPI / 4, BM = 128;
  constexpr int LA = HD == 128 ? 4 : 2;  // fragments read ahead of the MFMAs
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rank = blockIdx.x / a.kv_heads, head = blockIdx.x - rank * a.kv_heads, G = a.group.d;
  const SeqTile s = find_tile<BM, false>(a.seqs, G, rank, lane);
  if (s.none) return;
  const int tile = s.tile, rows = s.m * G, r0 = tile * BM + wave * 32;
  auto token_of = [&](int r) __attribute__((always_inline)) { return (int)div_by((unsigned)r, a.group); };
  auto row_of = [&](__bf16* p, const RowStrides& st, int r) __attribute__((always_inline)) {
    const int t = token_of(r);
    return p + (int64_t)(s.q0 + t) * st.row + (int64_t)(head * G + r - t * G) * st.head;
  };
  if (s.gap) {
    for (int i = tid; i < BM * (HD / 8); i += 256) {
      const int r = tile * BM + i / (HD / 8), col = i % (HD / 8) * 8;
      if (r < rows && col < a.D) *reinterpret_cast<uint4*>(row_of(a.dq, a.dqs, r) + col) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  const int r = min(r0 + l32, rows - 1), token = token_of(r);  // (rows past the end repeat the last one and are not stored)
  auto sees = [&](int t) __attribute__((always_inline)) { return a.causal ? min(max(t + 1 + s.n - s.m, 0), s.n) : s.n; };
  const int lim = sees(token);
  const int all = __builtin_amdgcn_readlane(lim, 0), some = __builtin_amdgcn_readlane(lim, 31);
  const int nt = (sees(token_of(min(tile * BM + BM, rows) - 1)) + 31) / 32;

  const __bf16* kp = a.k + (int64_t)s.k0 * a.ks.row + head * a.ks.head;
  const __bf16* vp = a.v + (int64_t)s.k0 * a.vs.row + head * a.vs.head;
  const unsigned smem_addr = lds_addr_of(smem);
  const int grow = T::row(lane), col0 = T::chunk(lane, wave) * 8, col = !PADDED || col0 < a.D ? col0 : 0;
  [[maybe_unused]] const uint64_t mask = __builtin_amdgcn_ballot_w64(!PADDED || col0 < a.D);
  const unsigned kofs = (unsigned)(grow * (int)a.ks.row + col) * 2u, vofs = (unsigned)(grow * (int)a.vs.row + col) * 2u;
  auto load = [&](auto... at) __attribute__((always_inline)) {
    if constexpr (PADDED) lds_dma16(at..., mask);
    else lds_dma16(at...);
  };
  auto request = [&](int slot, int t) __attribute__((always_inline)) {
    const unsigned Ks = smem_addr + (unsigned)(slot * kSlot), Vs = Ks + T::Bytes;
#pragma unroll
    for (int i = 0; i < GPW; ++i) {
      const int g = wave + 4 * i;
      if (t * 32 + 32 <= s.n) {
        const int64_t row = t * 32 + T::RPI * g;
        load(kp + row * a.ks.row, kofs, Ks + (unsigned)g * 1024u);
        load(vp + row * a.vs.row, vofs, Vs + (unsigned)g * 1024u);
      } else {  // rows past the sequence's end repeat its last one
        const int64_t row = min(t * 32 + T::RPI * g + grow, s.n - 1);
        load(kp + row * a.ks.row + col, Ks + (unsigned)g * 1024u);
        load(vp + row * a.vs.row + col, Vs + (unsigned)g * 1024u);
      }
    }
  };
  if constexpr (PADDED) {  // chunks past the head dim: zeros that no load touches
    for (int i = tid * 16; i < 2 * kSlot; i += 4096) *reinterpret_cast<uint4*>(smem + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
  }
  if (nt > 0) request(0, 0);

  bf16x8 qf[NJ], gf[NJ];
  float ndelta = 0.f;
  {
    const int64_t row = s.q0 + token, h = head * G + r - token * G;
    const __bf16 *pq = a.q + row * a.qs.row + h * a.qs.head, *pg = a.dout + row * a.os.row + h * a.os.head, *po = a.out + row * a.os.row + h * a.os.head;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      qf[j] = load_frag<PADDED>(pq, j * 16 + hh * 8, a.D);
      gf[j] = load_frag<PADDED>(pg, j * 16 + hh * 8, a.D);
      const bf16x8 of = load_frag<PADDED>(po, j * 16 + hh * 8, a.D);
#pragma unroll
      for (int e = 0; e < 8; ++e) ndelta = __builtin_fmaf(-(float)of[e], (float)gf[j][e], ndelta);
    }
    if (a.rest) {
      const __bf16* pr = a.rest + row * a.os.row + h * a.os.head;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const bf16x8 rf = load_frag<PADDED>(pr, j * 16 + hh * 8, a.D);
#pragma unroll
        for (int e = 0; e < 8; ++e) ndelta = __builtin_fmaf(-(float)rf[e], (float)gf[j][e], ndelta);
      }
    }
  }
  ndelta = xhalf_sum(ndelta);
  const float lse = a.lse[(int64_t)(head * G + r - token * G) * a.seqs.q_rows + s.q0 + token];
  // in front of the factor of the logits; rows that see no key: p = 0
  const float nlse = lse == -INFINITY ? -INFINITY : -lse / a.scale;
  if (hh == 0 && r0 + l32 < rows) {
    float* to = a.aux + (int64_t)(head * G + r - token * G) * a.seqs.q_rows + s.q0 + token;
    to[0] = nlse;
    to[(int64_t)a.kv_heads * G * a.seqs.q_rows] = ndelta;
  }

  f32x16 acc[ND];
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
  const float c = a.c;
  const unsigned row_at = T::row_at(lane), trans_at = T::trans_at(lane);
  auto block = [&](unsigned at, int k0) __attribute__((always_inline)) {
    auto frag = [&](int n) __attribute__((always_inline)) {
      if (n < NJ) return read_row_frag((at + row_at) ^ (unsigned)(32 * n));
      if (n < 2 * NJ) return read_row_frag(((at + row_at) ^ (unsigned)(32 * (n - NJ))) + T::Bytes);
      const int sg = (n - 2 * NJ) % ND, half = (n - 2 * NJ) / ND;
      const unsigned x = (at + trans_at) ^ (unsigned)(64 * sg);
      return read_trans_frag(x + (unsigned)(half * 16 * T::Row), (x ^ 32u) + (unsigned)((8 + half * 16) * T::Row));
    };
    f32x16 S, dP;
#pragma unroll
    for (int i = 0; i < 16; ++i) { S[i] = nlse; dP[i] = ndelta; }
    bf16x8 win[LA];
#pragma unroll
    for (int n = 0; n < LA; ++n) win[n] = frag(n);
    priority<HD>(1);
#pragma unroll
    for (int n = 0; n < 2 * NJ; ++n) {
      if (n < NJ) S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[n % LA], qf[n % NJ], S, 0, 0, 0);
      else dP = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[n % LA], gf[n % NJ], dP, 0, 0, 0);
      win[n % LA] = frag(n + LA);
      __builtin_amdgcn_sched_barrier(0);
    }
    priority<HD>(0);
    if (k0 + 32 > all) {
      asm volatile("" ::: "memory");  // keeps the branch
      const int at0 = k0 + 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (at0 + 8 * (i >> 2) + (i & 3) >= lim) S[i] = -INFINITY;
    }
    bf16x8 W[2];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      unsigned pk[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(S[8 * hb + e] * c), p1 = __builtin_amdgcn_exp2f(S[8 * hb + e + 1] * c);
        pk[e >> 1] = pack2(p0 * dP[8 * hb + e], p1 * dP[8 * hb + e + 1]);  // (the factor `scale` is applied once, to the accumulators)
      }
      W[hb] = __builtin_bit_cast(bf16x8, u32x4{pk[0], pk[1], pk[2], pk[3]});
    }
    priority<HD>(1);
#pragma unroll
    for (int jv = 0; jv < 2 * ND; ++jv) {
      acc[jv % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[(2 * NJ + jv) % LA], W[jv / ND], acc[jv % ND], 0, 0, 0);
      if (jv + LA < 2 * ND) win[(2 * NJ + jv) % LA] = frag(2 * NJ + jv + LA);
      __builtin_amdgcn_sched_barrier(0);
    }
    priority<HD>(0);
  };
  for (int t = 0; t < nt; ++t) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's share of tile t has landed
    __syncthreads();                     // ... and everyone's; the other slot is free
    if (t + 1 < nt) request((t + 1) & 1, t + 1);
    const unsigned at = smem_addr + (unsigned)((t & 1) * kSlot);
    if (t * 32 < some) block(at, t * 32);
  }
  __syncthreads();  // every wave has finished reading the ring, and no load into it is in flight: it now stages the output
  store_rows<ND, PADDED>(acc, a.scale, r0, rows, a.D, lane, smem + wave * kStageRows,
                         [&](int row) __attribute__((always_inline)) { return row_of(a.dq, a.dqs, row); });
}

// ---------------------------------------------------------------------------------------------------------------------- dk, dv
// What a tile of 128 keys meets: the tokens from `first` on, `tiles` tiles of 32 of them in each head; the walk over all heads in `pieces` pieces of
// `each` tiles.
struct KeyWalk {
  int first, tiles, pieces, each;
};
__device__ __forceinline__ KeyWalk key_walk(const SeqTile& s, int key0, int G, int causal, int piece_tiles, int pieces) {
  KeyWalk k;
  k.first = causal ? max(key0 - s.n + s.m, 0) & ~31 : 0;
  k.tiles = (s.m - k.first + 31) >> 5;  // (none: no token)
  const int walk = k.tiles * G;
  k.pieces = min(max((walk + piece_tiles - 1) / piece_tiles, 1), pieces);
  k.each = (walk + k.pieces - 1) / k.pieces;
  return k;
}

template <int HD, int DC, bool PADDED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 3 : 2, HD == 64 ? 3 : 2))) void packed_dkv_kernel(PackedBwdArgs a) {
  using T = PackedBlock<HD>;
  constexpr int NJ = DC / 16, ND = (DC + 31) / 32, kSlot = bwd_slot<HD>(true), kAux = 2 * T::Bytes, GPW = 32 / T::RPI / 4, BM = 128;
  constexpr int LA1 = HD == 128 ? 2 : 0, LA3 = HD == 128 ? 6 : 0;  // fragments read ahead in the chains and in the accumulations
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rank = blockIdx.x / a.kv_heads, head = blockIdx.x - rank * a.kv_heads, G = a.group.d;
  const SeqTile s = find_tile<BM, true>(a.seqs, G, rank, lane);
  if (s.none) return;
  const int key0 = (s.tiles - 1 - s.tile) * BM, w0 = key0 + wave * 32;  // (causal: the first keys meet the most tokens)
  const int piece = gridDim.y - 1 - blockIdx.y;  // (the long walks' last pieces first, the short walks' only ones in the end)
  if (s.gap) {
    if (piece) return;
    for (int i = tid; i < BM * (HD / 8); i += 256) {
      const int64_t r = key0 + i / (HD / 8);
      const int col = i % (HD / 8) * 8;
      if (r >= s.n || col >= a.D) continue;
      *reinterpret_cast<uint4*>(a.dk + (s.k0 + r) * a.dks.row + head * a.dks.head + col) = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(a.dv + (s.k0 + r) * a.dvs.row + head * a.dvs.head + col) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  const KeyWalk kw = key_walk(s, key0, G, a.causal, a.piece_tiles, a.pieces);
  if (piece >= kw.pieces) return;
  const int begin = piece * kw.each, nt = min(kw.each, kw.tiles * G - begin);  // (no token: none; the last piece may be empty)
  // the first token that sees a lane's key
  const int from = a.causal ? max(min(w0 + l32, s.n - 1) - s.n + s.m, 0) : 0;
  const int none_below = __builtin_amdgcn_readlane(from, 0), all_from = __builtin_amdgcn_readlane(from, 31);
  const bool idle = w0 >= s.n;  // a wave without keys brings its share of the tiles

  const unsigned smem_addr = lds_addr_of(smem);
  const int64_t aux_delta = (int64_t)a.kv_heads * G * a.seqs.q_rows;
  [[maybe_unused]] const uint64_t mask = __builtin_amdgcn_ballot_w64(!PADDED || T::chunk(lane, wave) * 8 < a.D);
  auto load = [&](auto... at) __attribute__((always_inline)) {
    if constexpr (PADDED) lds_dma16(at..., mask);
    else lds_dma16(at...);
  };
  // the walk: head g of the group, tokens from token0 on
  struct At {
    int g, token0;
  };
  auto next = [&](At& at) __attribute__((always_inline)) {
    at.token0 += 32;
    if (at.token0 >= s.m) {
      at.token0 = kw.first;
      ++at.g;
    }
  };
  auto request = [&](int slot, const At& at) __attribute__((always_inline)) {
    const unsigned Qs = smem_addr + (unsigned)(slot * kSlot), Gs = Qs + T::Bytes;
    int ln = lane;
    asm volatile("" : "+v"(ln));  // opaque: what follows from the lane is formed again for every tile, the accumulators need the registers
    const int64_t h = head * G + at.g, t0 = s.q0 + at.token0;
    const int left = s.m - at.token0;  // tokens; those past the end repeat the last one
    // wave 0: -lse / scale of the 32 tokens, then their -delta, 64 floats behind the tiles
    if (wave == 0) {
      const float* p = a.aux + h * a.seqs.q_rows + t0 + min(ln & 31, left - 1);
      lds_dma4(ln < 32 ? p : p + aux_delta, Qs + kAux);
    }
    const int c0 = T::chunk(ln, wave) * 8, col = !PADDED || c0 < a.D ? c0 : 0;
    const __bf16 *qt = a.q + t0 * a.qs.row + h * a.qs.head, *gt = a.dout + t0 * a.os.row + h * a.os.head;
#pragma unroll
    for (int i = 0; i < GPW; ++i) {
      const int g = wave + 4 * i;
      if (left >= 32) {
        load(qt + (int64_t)(T::RPI * g) * a.qs.row, (unsigned)(T::row(ln) * (int)a.qs.row + col) * 2u, Qs + (unsigned)g * 1024u);
        load(gt + (int64_t)(T::RPI * g) * a.os.row, (unsigned)(T::row(ln) * (int)a.os.row + col) * 2u, Gs + (unsigned)g * 1024u);
      } else {
        const int r = min(T::RPI * g + T::row(ln), left - 1);
        load(qt, (unsigned)(r * (int)a.qs.row + col) * 2u, Qs + (unsigned)g * 1024u);
        load(gt, (unsigned)(r * (int)a.os.row + col) * 2u, Gs + (unsigned)g * 1024u);
      }
    }
  };
  if constexpr (PADDED) {  // chunks past the head dim: zeros that no load touches
    for (int i = tid * 16; i < 2 * kSlot; i += 4096) *reinterpret_cast<uint4*>(smem + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
  }
  At ahead{0, kw.first};
  if (nt > 0) {
    ahead.g = begin / kw.tiles;
    ahead.token0 = kw.first + (begin - ahead.g * kw.tiles) * 32;
    request(0, ahead);
  }
  bf16x8 kf[NJ], vf[NJ];
  {
    const int64_t row = s.k0 + min(w0 + l32, s.n - 1);
    const __bf16 *pk = a.k + row * a.ks.row + head * a.ks.head, *pv = a.v + row * a.vs.row + head * a.vs.head;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      kf[j] = load_frag<PADDED>(pk, j * 16 + hh * 8, a.D);
      vf[j] = load_frag<PADDED>(pv, j * 16 + hh * 8, a.D);
    }
  }
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[db][i] = dv[db][i] = 0.f;
  const float c = a.c;
  const unsigned row_at = T::row_at(lane), trans_at = T::trans_at(lane);

  auto block = [&](unsigned at, int token0) __attribute__((always_inline)) {
    auto aux4 = [&](int i) __attribute__((always_inline)) { return *(lds_f32x4_at)(at + (unsigned)(kAux + 4 * i)); };
    auto frag = [&](int n) __attribute__((always_inline)) {
      return n < NJ ? read_row_frag((at + row_at) ^ (unsigned)(32 * n)) : read_row_frag(((at + row_at) ^ (unsigned)(32 * (n - NJ))) + T::Bytes);
    };
    auto frag3 = [&](int n) __attribute__((always_inline)) {  // of q and of dout in turn
      const int jv = n >> 1, second = n & 1, sg = jv % ND, half = jv / ND;
      const unsigned x = (at + trans_at) ^ (unsigned)(64 * sg);
      return read_trans_frag(x + (unsigned)(half * 16 * T::Row + second * T::Bytes), (x ^ 32u) + (unsigned)((8 + half * 16) * T::Row + second * T::Bytes));
    };
    f32x16 S, dP;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 u0 = aux4(8 * g + 4 * hh), u1 = aux4(32 + 8 * g + 4 * hh);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        S[4 * g + e] = u0[e];
        dP[4 * g + e] = u1[e];
      }
    }
    priority<HD>(1);
    if constexpr (LA1 > 0) {
      bf16x8 win[LA1];
#pragma unroll
      for (int n = 0; n < LA1; ++n) win[n] = frag(n);
#pragma unroll
      for (int n = 0; n < 2 * NJ; ++n) {
        if (n < NJ) S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[n % LA1], kf[n % NJ], S, 0, 0, 0);
        else dP = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[n % LA1], vf[n % NJ], dP, 0, 0, 0);
        if (n + LA1 < 2 * NJ) win[n % LA1] = frag(n + LA1);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag(j), kf[j], S, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < NJ; ++j) dP = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag(NJ + j), vf[j], dP, 0, 0, 0);
    }
    priority<HD>(0);
    if (token0 < all_from || token0 + 32 > s.m) {  // tokens that do not see the key, and what is behind the last
      asm volatile("" ::: "memory");  // keeps the branch
      const int at0 = token0 + 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int tk = at0 + 8 * (i >> 2) + (i & 3);
        if (tk < from || tk >= s.m) { S[i] = -INFINITY; dP[i] = 0.f; }
      }
    }
    bf16x8 W[2], P[2];
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      unsigned wpk[4], ppk[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(S[8 * hb + e] * c), p1 = __builtin_amdgcn_exp2f(S[8 * hb + e + 1] * c);
        wpk[e >> 1] = pack2(p0 * dP[8 * hb + e], p1 * dP[8 * hb + e + 1]);
        ppk[e >> 1] = pack2(p0, p1);
      }
      W[hb] = __builtin_bit_cast(bf16x8, u32x4{wpk[0], wpk[1], wpk[2], wpk[3]});
      P[hb] = __builtin_bit_cast(bf16x8, u32x4{ppk[0], ppk[1], ppk[2], ppk[3]});
    }
    priority<HD>(1);
    if constexpr (LA3 > 0) {
      bf16x8 win[LA3];
#pragma unroll
      for (int n = 0; n < LA3; ++n) win[n] = frag3(n);
#pragma unroll
      for (int n = 0; n < 4 * ND; ++n) {
        const int jv = n >> 1;
        if (n & 1) dv[jv % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[n % LA3], P[jv / ND], dv[jv % ND], 0, 0, 0);
        else dk[jv % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[n % LA3], W[jv / ND], dk[jv % ND], 0, 0, 0);
        if (n + LA3 < 4 * ND) win[n % LA3] = frag3(n + LA3);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int jv = 0; jv < 2 * ND; ++jv) {
        dk[jv % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag3(2 * jv), W[jv / ND], dk[jv % ND], 0, 0, 0);
        dv[jv % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag3(2 * jv + 1), P[jv / ND], dv[jv % ND], 0, 0, 0);
      }
    }
    priority<HD>(0);
  };
  for (int t = 0; t < nt; ++t) {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    const int token0 = ahead.token0;
    if (t + 1 < nt) {
      next(ahead);
      request((t + 1) & 1, ahead);
    }
    if (!idle && token0 + 32 > none_below) block(smem_addr + (unsigned)((t & 1) * kSlot), token0);
  }
  __syncthreads();
  // the lane number once more: the loop has no register for it
  const int ln = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  char* stage = smem + wave * kStageRows;
  if (kw.pieces > 1) {
    const int64_t tensor = (int64_t)a.kv_heads * a.seqs.k_rows * a.D, at = (int64_t)piece * 2 * tensor + ((int64_t)head * a.seqs.k_rows + s.k0) * a.D;
    store_partial<ND, PADDED>(dk, a.scale, a.part + at, w0, s.n, a.D, ln, stage);
    store_partial<ND, PADDED>(dv, 1.0f, a.part + at + tensor, w0, s.n, a.D, ln, stage);
    return;
  }
  store_rows<ND, PADDED>(dk, a.scale, w0, s.n, a.D, ln, stage, [&](int row) __attribute__((always_inline)) {
    return a.dk + (int64_t)(s.k0 + row) * a.dks.row + head * a.dks.head;
  });
  store_rows<ND, PADDED>(dv, 1.0f, w0, s.n, a.D, ln, stage, [&](int row) __attribute__((always_inline)) {
    return a.dv + (int64_t)(s.k0 + row) * a.dvs.row + head * a.dvs.head;
  });
}

// The pieces' sums of dk (blockIdx.y 0) and dv (1), added in their order, for the tiles of 128 keys whose rows were cut; a tile's elements to
// gridDim.z workgroups where there are few.
__global__ __launch_bounds__(256) void packed_reduce_kernel(PackedBwdArgs a) {
  const int lane = threadIdx.x & 63, rank = blockIdx.x / a.kv_heads, head = blockIdx.x - rank * a.kv_heads, G = a.group.d;
  const SeqTile s = find_tile<128, true>(a.seqs, G, rank, lane);
  if (s.none || s.gap) return;
  const int key0 = s.tile * 128, cpr = a.D / 8;
  const KeyWalk kw = key_walk(s, key0, G, a.causal, a.piece_tiles, a.pieces);
  if (kw.pieces == 1) return;
  const int64_t tensor = (int64_t)a.kv_heads * a.seqs.k_rows * a.D;
  const float* part = a.part + blockIdx.y * tensor + ((int64_t)head * a.seqs.k_rows + s.k0 + key0) * a.D;
  const RowStrides st = blockIdx.y ? a.dvs : a.dks;
  __bf16* out = (blockIdx.y ? a.dv : a.dk) + (int64_t)(s.k0 + key0) * st.row + head * st.head;
  const int n = min(128, s.n - key0) * cpr;
  for (int i = blockIdx.z * 256 + threadIdx.x; i < n; i += 256 * gridDim.z) {
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const f32x4* p = reinterpret_cast<const f32x4*>(part) + 2 * i;
#pragma unroll 4
    for (int k = 0; k < kw.pieces; ++k, p += tensor / 2) {
      const f32x4 u = p[0], v = p[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) { f[e] += u[e]; f[4 + e] += v[e]; }
    }
    const int row = i / cpr;
    *reinterpret_cast<uint4*>(out + (int64_t)row * st.row + (i - row * cpr) * 8) = pack8(f);
  }
}

// How the dk / dv pass is cut, and the workspace: the rows' two numbers, then the pieces' sums.
struct BwdPlan {
  int pieces, piece_tiles;
  int64_t aux_floats, floats, tiles;  // tiles: of 128 keys, of all heads
};
BwdPlan bwd_plan(const mdattn_packed* p) {
  const int64_t group = p->heads / p->kv_heads;
  const int64_t max_q = p->max_q > 0 && p->max_q < p->q_rows ? p->max_q : p->q_rows, max_k = p->max_k > 0 && p->max_k < p->k_rows ? p->max_k : p->k_rows;
  BwdPlan b{1, 1 << 30, 0, 0, 0};
  b.aux_floats = ((int64_t)p->q_rows * p->heads * 2 + 3) & ~(int64_t)3;
  const int64_t tiles = (max_k + 127) / 128 * p->sequences, most = p->k_rows / 128 + p->sequences, walk = (max_q + 31) / 32 * group;
  b.tiles = (tiles < most ? tiles : most) * p->kv_heads;
  // The walks whole, long ones first, or in n parts, by what the last place on the chip (two workgroups per CU, three at head dims up to 64) then
  // ends at, in tiles.  `place`: what each has to walk; of lengths that differ, known by their mean and their largest, some two thirds of what
  // tiles that all met the longest would have.  A part costs its sums' way to memory and back, 130 KB in each of the places, as much as 15 tiles, parts
  // at all another 25; with a part to each place (less a few: they do not fill evenly) the longest is waited for, with more (causal, or lengths that
  // differ) half of one, else whole rounds.  us whole / in parts: 4 x 4,096 tokens, causal, 32 heads on 8 of 128, 1,782 / 1,792 in 2; 8 x 1,024
  // 290 / 322 in 3; 8 from 100 to 4,096 1,179 / 1,106 in 4; one of 8,192 1,996 / 1,767 in 7; that, 8 on 1, 2,384 / 525 in 12; one of 2,048, no
  // mask, 32 on 8, 378 / 235 in 4, 252 in 3, 248 in 6.
  const int places = p->head_dim > 64 ? 512 : 768;
  const double even = std::min(1.0, (double)p->k_rows / std::max(1.0, (double)max_k * p->sequences));
  const double place = (double)b.tiles * walk / (p->causal ? 2 : 1) / places * (1 + even) / 2;
  const int64_t sums = 2 * std::max<int64_t>((int64_t)p->k_rows * p->kv_heads * p->head_dim, 1);
  const int64_t most_parts = std::min({(int64_t)64, walk / 16, (int64_t)((1 << 28) / sums)});  // (a GiB of sums at most, whatever the hints are)
  double best = 1.05 * std::max((double)walk, place);
  for (int n = 2; n <= most_parts; ++n) {
    const double part = (double)walk / n, parts = b.tiles * (p->causal ? 0.5 * (n + 1) : n);
    const double end = 25 + (parts <= 0.95 * places || (!p->causal && parts <= places) ? part + 15
                             : p->causal || even < 0.95                               ? place + 15 * parts / places + 0.5 * part
                                                                                      : std::ceil(parts / places) * (part + 15));
    if (end < best) {
      best = end;
      b.pieces = n;
    }
  }
  if (b.pieces > 1) b.piece_tiles = (int)((walk + b.pieces - 1) / b.pieces);
  b.floats = b.aux_floats + (b.pieces > 1 ? b.pieces * sums : 0);
  return b;
}

template <int HD, int DC, bool PADDED>
int launch(hipStream_t st, const PackedBwdArgs& a, int64_t dq_grid, int64_t dkv_grid) {
  constexpr int ring = 2 * bwd_slot<HD>(true), stage = 4 * kStageRows, bytes = ring > stage ? ring : stage;
  if (dq_grid) {
    MDATTN_LAUNCH((packed_dq_kernel<HD, DC, PADDED>), dim3((unsigned)dq_grid), dim3(256), bytes, st, a);
    const int rc = launch_status();
    if (rc != MDATTN_OK) return rc;
  }
  if (!dkv_grid) return MDATTN_OK;
  MDATTN_LAUNCH((packed_dkv_kernel<HD, DC, PADDED>), dim3((unsigned)dkv_grid, (unsigned)a.pieces), dim3(256), bytes, st, a);
  const int rc = launch_status();
  if (rc != MDATTN_OK || a.pieces == 1) return rc;
  const unsigned share = dkv_grid < 32 ? 8 : dkv_grid < 256 ? (unsigned)(256 / dkv_grid) : 1;
  MDATTN_LAUNCH(packed_reduce_kernel, dim3((unsigned)dkv_grid, 2, share), dim3(256), 0, st, a);
  return launch_status();
}

}  // namespace
}  // namespace mdattn

using namespace mdattn;

extern "C" int64_t mdattn_bwd_bf16_packed_workspace_floats(const mdattn_packed* p) {
  return packed_sizes(p) == MDATTN_OK ? bwd_plan(p).floats : 0;
}

extern "C" int mdattn_host_packed_bwd_plan(const mdattn_packed* p, mdattn_host_packed_plan* plan) {
  const int rc = packed_sizes(p);
  if (rc != MDATTN_OK) return rc;
  const BwdPlan b = bwd_plan(p);
  *plan = {1, packed_order(p, b.tiles), b.pieces, b.piece_tiles, packed_tiles(p->k_rows, p->sequences, 128) * b.pieces * p->kv_heads};
  return MDATTN_OK;
}

extern "C" int mdattn_bwd_bf16_packed(void* stream, const mdattn_packed* p, const void* q, const void* k, const void* v, const void* out,
                                      const void* rest, const void* dout, const float* lse, void* dq, void* dk, void* dv, const mdattn_strides* q_strides,
                                      const mdattn_strides* k_strides, const mdattn_strides* v_strides, const mdattn_strides* o_strides,
                                      const mdattn_strides* dq_strides, const mdattn_strides* dk_strides, const mdattn_strides* dv_strides,
                                      float scale, float* workspace, int64_t workspace_floats) {
  const int rc = packed_sizes(p);
  if (rc != MDATTN_OK) return rc;
  if (!(scale > 0.f) || !(scale < INFINITY) || p->k_lengths) return MDATTN_E_BADARG;
  if (scale < 1e-30f) return MDATTN_E_UNSUPPORTED;  // (lse / scale has to be a number)
  for (const mdattn_strides* s : {q_strides, k_strides, v_strides, o_strides, dq_strides, dk_strides, dv_strides}) {
    if (!s) return MDATTN_E_BADARG;
    if (!packed_strides_ok(s, s == q_strides || s == o_strides ? p->heads / p->kv_heads : 0)) return MDATTN_E_ALIGN;
  }
  if ((p->q_rows && (!q || !out || !dout || !lse || !dq)) || (p->k_rows && (!k || !v || !dk || !dv))) return MDATTN_E_BADARG;
  for (const void* t : {q, k, v, out, rest, dout, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)workspace})
    if (!aligned16(t)) return MDATTN_E_ALIGN;
  if (!packed_aligned(p) || (reinterpret_cast<uintptr_t>(lse) & 3)) return MDATTN_E_ALIGN;
  if (p->q_rows == 0 && p->k_rows == 0) return MDATTN_OK;
  const BwdPlan b = bwd_plan(p);
  if (!workspace || workspace_floats < b.floats) return MDATTN_E_BADARG;
  PackedBwdArgs a{};
  a.q = static_cast<const __bf16*>(q); a.k = static_cast<const __bf16*>(k); a.v = static_cast<const __bf16*>(v);
  a.out = static_cast<const __bf16*>(out); a.rest = static_cast<const __bf16*>(rest); a.dout = static_cast<const __bf16*>(dout); a.lse = lse;
  a.dq = static_cast<__bf16*>(dq); a.dk = static_cast<__bf16*>(dk); a.dv = static_cast<__bf16*>(dv);
  a.aux = workspace;
  a.part = workspace + b.aux_floats;
  a.seqs = {p->q_offsets, p->k_offsets, nullptr, p->sequences, p->q_rows, p->k_rows, packed_order(p, b.tiles), 256 / p->kv_heads};
  a.group = divisor((unsigned)(p->heads / p->kv_heads));
  a.kv_heads = p->kv_heads; a.D = p->head_dim; a.causal = p->causal;
  auto strides = [](const mdattn_strides* s) { return RowStrides{s->seq, s->head}; };
  a.qs = strides(q_strides); a.ks = strides(k_strides); a.vs = strides(v_strides); a.os = strides(o_strides);
  a.dqs = strides(dq_strides); a.dks = strides(dk_strides); a.dvs = strides(dv_strides);
  a.c = scale * kLog2e; a.scale = scale;
  a.pieces = b.pieces; a.piece_tiles = b.piece_tiles;
  const int64_t dq_grid = p->q_rows ? packed_tiles((int64_t)p->q_rows * a.group.d, p->sequences, 128) * p->kv_heads : 0;
  const int64_t dkv_grid = p->k_rows ? packed_tiles(p->k_rows, p->sequences, 128) * p->kv_heads : 0;
  if (!grid_fits(dq_grid, 256) || !grid_fits(dkv_grid, 256)) return MDATTN_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  if (a.D == 64) return launch<64, 64, false>(st, a, dq_grid, dkv_grid);
  if (a.D < 64) return launch<64, 64, true>(st, a, dq_grid, dkv_grid);
  if (a.D <= 80) return launch<128, 80, true>(st, a, dq_grid, dkv_grid);
  if (a.D <= 96) return launch<128, 96, true>(st, a, dq_grid, dkv_grid);
  if (a.D < 128) return launch<128, 128, true>(st, a, dq_grid, dkv_grid);
  return launch<128, 128, false>(st, a, dq_grid, dkv_grid);
}

// Attention over packed sequences for gfx950 (MI355X), bf16 MFMA: causal or not, the heads of q in groups that share a head of k and v.
//
//   s = scale q.k over the keys that the row sees,  p = exp(s - lse),  out = p v,  lse = log sum exp s
//
// Rows.  A tile's rows are a group's: row r of a sequence is head r % G of token r / G.  One read of a tile of keys then serves all heads of
// the group, a causal tile spans 1 / G of the tokens (and of the keys that only some of its rows see), and one token of a group of
// four already fills four rows.
// Work.  A wave owns 32 rows and walks keys in blocks of 32 through a ring in LDS, filled by direct global -> LDS loads: S^T = K Q^T, so that
// a lane holds 16 keys of one row and the accumulators are, packed to bf16, the B operand of O^T += V^T P^T.  The softmax keeps no running
// maximum but a reference point per row, moved (in a rarely taken branch) when a sum of P leaves its range.  Keys that a row does not see get
// s = -inf, in the blocks that hold such keys; blocks that no row of a wave sees are not computed.
// Few rows (one or a few tokens) have a kernel of their own, bound by the keys' way from memory.
// With few tiles the keys are cut into pieces besides; each leaves un-normalised f32 rows, joined by a third kernel in a fixed order.
#include <algorithm>
#include <type_traits>

#include "attn_packed.h"

namespace mdattn {
namespace {

constexpr float kRange = 16777216.f;  // a partial sum of P above 2^24 moves the row's reference point

struct PackedArgs {
  const __bf16 *q, *k, *v;
  __bf16* out;
  float* lse;
  PackedSeqs seqs;
  Divisor group;
  int kv_heads, D, causal;
  RowStrides qs, ks, vs, os;
  float c;  // scale * log2(e)
  int pieces, piece_keys;
  float* part;  // [piece][kv_heads][q_rows * group][D]
  float2* ml;   // [piece][kv_heads][q_rows * group]: reference point (log2 units) and sum of P
};

template <int HD>
struct FwdShape {
  static constexpr int NB = HD == 64 ? 2 : 1;      // blocks of 32 keys of a slot
  static constexpr int SLOTS = HD == 64 ? 2 : 3;
  static constexpr int Keys = 32 * NB, Half = NB * PackedBlock<HD>::Bytes, Slot = 2 * Half;
  static constexpr int BM = 128;
};

// rows of no sequence: tile `tile` of them
template <int BM, int HD>
__device__ __forceinline__ void fill_gap(const PackedArgs& a, const SeqTile& s, int head, int tid) {
  const int G = a.group.d, rows = s.m * G;
  for (int i = tid; i < BM * (HD / 8); i += 256) {
    const int r = s.tile * BM + i / (HD / 8), col = i % (HD / 8) * 8;
    if (r >= rows) continue;
    const int t = (int)div_by((unsigned)r, a.group), h = head * G + r - t * G;
    if (col < a.D) *reinterpret_cast<uint4*>(a.out + (int64_t)(s.q0 + t) * a.os.row + (int64_t)h * a.os.head + col) = make_uint4(0u, 0u, 0u, 0u);
    if (col == 0 && a.lse) a.lse[(int64_t)h * a.seqs.q_rows + s.q0 + t] = -INFINITY;
  }
}

// The softmax of a row's running sums: P = exp2(c s - mc) of 16 keys per lane and their sum against the row's reference point m (mc = m c), which
// moves, with O and l, when a sum leaves its range.  Rows that have seen no key yet have m = -1e30, from which any logit is out of range.
struct RowState {
  float m, mc, l;
};
template <int ND>
__device__ __forceinline__ void soft_block(const f32x16& S, float c, RowState& st, f32x16 (&O)[ND], bf16x8 (&P)[2]) {
  auto soft = [&]() __attribute__((always_inline)) {
    float sum = 0.f;
#pragma unroll
    for (int hb = 0; hb < 2; ++hb) {
      unsigned pk[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[8 * hb + e], c, -st.mc));
        const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[8 * hb + e + 1], c, -st.mc));
        sum = (hb == 0 && e == 0) ? x0 : sum + x0;
        sum += x1;
        pk[e >> 1] = pack2(x0, x1);
        asm volatile("" : "+v"(pk[e >> 1]), "+v"(sum));  // packed as soon as they exist
      }
      P[hb] = __builtin_bit_cast(bf16x8, u32x4{pk[0], pk[1], pk[2], pk[3]});
    }
    return sum;
  };
  float sum = soft();
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum <= kRange)) != 0, 0)) {
    float top = S[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, S[i]);
    const float mnew = fmaxf(st.m, xhalf_max(top));
    float alpha = __builtin_amdgcn_exp2f((st.m - mnew) * c);
    st.m = mnew;
    st.mc = st.m * c;
    asm volatile("" : "+v"(alpha));  // keeps the rescale inside this rarely taken branch
    st.l *= alpha;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) O[db][i] *= alpha;
    sum = soft();
  }
  st.l += sum;
}

// A row's fragments straight from memory, waited for here, with what is on its way into LDS: in the loop behind, the compiler would wait for them in
// every block of keys, and with that for the keys requested since (16,384 tokens x 32 heads 1,895 -> @@ us).
template <int NJ, bool PADDED>
__device__ __forceinline__ void load_row(bf16x8 (&f)[NJ], const __bf16* p, int hh, int D) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) f[j] = !PADDED || j * 16 + hh * 8 < D ? *reinterpret_cast<const bf16x8*>(p + j * 16) : __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
#pragma unroll
  for (int j = 0; j < NJ; ++j) asm volatile("" : "+v"(f[j]));
}

// A wave's 32 rows from row r0 of the sequence on, normalised, rounded and stored as whole rows through `stage` (32 rows of kOutRow bytes that
// nobody else touches any more): as the accumulators lie, a store would touch 16 bytes of each of 32 rows.
template <int ND>
constexpr int kOutRow = ND * 64 + 16;
template <int ND, int DC, bool PADDED>
__device__ __forceinline__ void store_out(const PackedArgs& a, const SeqTile& s, const f32x16 (&O)[ND], float l, float mc, int head, int r0, int lane,
                                          char* stage) {
  constexpr int RowB = kOutRow<ND>, LPR = ND == 3 ? 16 : ND * 4, RPI = 64 / LPR;  // lanes per row, rows per store
  const int l32 = lane & 31, hh = lane >> 5, G = a.group.d, rows = s.m * G;
  // rows that see no key give 0 and -inf; a sum that is not a number stays one
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  if (a.lse && hh == 0 && r0 + l32 < rows) {
    const int t = (int)div_by((unsigned)(r0 + l32), a.group);
    a.lse[(int64_t)(head * G + r0 + l32 - t * G) * a.seqs.q_rows + s.q0 + t] = l == 0.f ? -INFINITY : (mc + __log2f(l)) * kLn2;
  }
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint2 u;
      u.x = pack2(O[db][4 * g] * inv, O[db][4 * g + 1] * inv);
      u.y = pack2(O[db][4 * g + 2] * inv, O[db][4 * g + 3] * inv);
      *reinterpret_cast<uint2*>(stage + l32 * RowB + hh * 8 + (db * 32 + g * 8) * 2) = u;
    }
  // LDS accesses of one wave execute in order: the reads below see the writes above
  const int rr = lane / LPR, cc = lane % LPR;
  if (cc * 8 >= (PADDED ? a.D : DC)) return;
#pragma unroll
  for (int j = 0; j < 32 / RPI; ++j) {
    const int row = r0 + j * RPI + rr;
    if (row >= rows) break;
    const int t = (int)div_by((unsigned)row, a.group);
    st_nt(reinterpret_cast<uint4*>(a.out + (int64_t)(s.q0 + t) * a.os.row + (int64_t)(head * G + row - t * G) * a.os.head + cc * 8),
          *reinterpret_cast<const uint4*>(stage + (j * RPI + rr) * RowB + cc * 16));
  }
}

template <int HD, int DC, bool PADDED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 4 : 3, HD == 64 ? 4 : 3))) void packed_fwd_kernel(PackedArgs a) {
  using T = PackedBlock<HD>;
  using F = FwdShape<HD>;
  constexpr int NJ = DC / 16, ND = (DC + 31) / 32, NB = F::NB, SLOTS = F::SLOTS;
  constexpr int GPW = F::Keys / T::RPI / 4;  // row groups per wave, slot and tensor
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // (fragment addresses are formed by xor)
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // neighbouring workgroups, which go to different dies, take different heads: with eight heads of k and v each die's L2 holds one of them
  const int rank = blockIdx.x / a.kv_heads, head = blockIdx.x - rank * a.kv_heads, G = a.group.d;
  const SeqTile s = find_tile<F::BM, false>(a.seqs, G, rank, lane);
  if (s.none) return;
  const int64_t group_rows = (int64_t)a.seqs.q_rows * G;
  const int tile = s.tile, rows = s.m * G, r0 = tile * F::BM + wave * 32;
  const bool split = a.part != nullptr;
  auto token_of = [&](int r) __attribute__((always_inline)) { return (int)div_by((unsigned)r, a.group); };
  if (s.gap) {
    if (blockIdx.y == 0) fill_gap<F::BM, HD>(a, s, head, tid);
    return;
  }

  // keys that a row sees, of those of this piece
  const int r = min(r0 + l32, rows - 1);  // (rows past the end repeat the last one and are not stored)
  const int token = token_of(r);
  const int piece = blockIdx.y, kb = piece * a.piece_keys;
  const int ke = piece == a.pieces - 1 ? s.n : min(s.n, kb + a.piece_keys);
  auto sees = [&](int t) __attribute__((always_inline)) { return min(ke, a.causal ? max(t + 1 + s.n - s.m, 0) : s.n) - kb; };
  const int lim = sees(token);                                       // (may be negative)
  const int all = __builtin_amdgcn_readlane(lim, 0), some = __builtin_amdgcn_readlane(lim, 31);  // keys that all, some rows of the wave see
  const int end = sees(token_of(min(tile * F::BM + F::BM, rows) - 1));  // some row of the workgroup
  const int nt = (end + F::Keys - 1) / F::Keys;                        // slots visited; zero or less: none

  const __bf16* kp = a.k + (int64_t)(s.k0 + kb) * a.ks.row + head * a.ks.head;
  const __bf16* vp = a.v + (int64_t)(s.k0 + kb) * a.vs.row + head * a.vs.head;
  const unsigned smem_addr = lds_addr_of(smem);
  const int grow = T::row(lane), col0 = T::chunk(lane, wave) * 8;  // (groups wave, wave + 4, ...: the swizzle sees the same)
  const int col = !PADDED || col0 < a.D ? col0 : 0;
  [[maybe_unused]] const uint64_t mask = __builtin_amdgcn_ballot_w64(!PADDED || col0 < a.D);
  const unsigned kofs = (unsigned)(grow * (int)a.ks.row + col) * 2u, vofs = (unsigned)(grow * (int)a.vs.row + col) * 2u;
  auto load = [&](auto... at) __attribute__((always_inline)) {
    if constexpr (PADDED) lds_dma16(at..., mask);
    else lds_dma16(at...);
  };
  const int n = s.n - kb;  // rows of k and v from kp on
  auto request = [&](int slot, int t) __attribute__((always_inline)) {
    const unsigned Ks = smem_addr + (unsigned)(slot * F::Slot), Vs = Ks + F::Half;
    if (t * F::Keys + F::Keys <= n) {
#pragma unroll
      for (int i = 0; i < GPW; ++i) {
        const int g = wave + 4 * i;
        const int64_t row = t * F::Keys + T::RPI * g;
        load(kp + row * a.ks.row, kofs, Ks + (unsigned)g * 1024u);
        load(vp + row * a.vs.row, vofs, Vs + (unsigned)g * 1024u);
      }
    } else {  // rows past the sequence's end repeat its last one
#pragma unroll
      for (int i = 0; i < GPW; ++i) {
        const int g = wave + 4 * i;
        const int64_t row = min(t * F::Keys + T::RPI * g + grow, n - 1);
        load(kp + row * a.ks.row + col, Ks + (unsigned)g * 1024u);
        load(vp + row * a.vs.row + col, Vs + (unsigned)g * 1024u);
      }
    }
  };

  if constexpr (PADDED) {  // chunks past the head dim: zeros that no load touches
    for (int i = tid * 16; i < SLOTS * F::Slot; i += 4096) *reinterpret_cast<uint4*>(smem + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < SLOTS - 1; ++t)
    if (t < nt) request(t, t);
  bf16x8 qf[NJ];
  load_row<NJ, PADDED>(qf, a.q + (int64_t)(s.q0 + token) * a.qs.row + (int64_t)(head * G + r - token * G) * a.qs.head + hh * 8, hh, a.D);
  f32x16 O[ND];
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[db][i] = 0.f;
  const float c = a.c;
  RowState st{-1e30f, -1e30f * c, 0.f};
  const unsigned row_at = T::row_at(lane), trans_at = T::trans_at(lane);

  // a block of 32 keys, the first of them key `k0` of the piece, at `at` (its V a half slot on)
  auto block = [&](unsigned at, int k0) __attribute__((always_inline)) {
    constexpr int FPB = NJ + 2 * ND;
    auto frag = [&](int i) __attribute__((always_inline)) {
      if (i < NJ) return read_row_frag((at + row_at) ^ (unsigned)(32 * i));
      const int sg = (i - NJ) % ND, half = (i - NJ) / ND;
      const unsigned v = (at + F::Half + trans_at) ^ (unsigned)(64 * sg);
      return read_trans_frag(v + (unsigned)(half * 16 * T::Row), (v ^ 32u) + (unsigned)((8 + half * 16) * T::Row));
    };
    constexpr int LA = HD == 128 ? 2 : 0;  // fragments read ahead of the MFMAs
    [[maybe_unused]] bf16x8 win[LA > 0 ? LA : 1];
    if constexpr (LA > 0) {
#pragma unroll
      for (int i = 0; i < LA; ++i) win[i] = frag(i);
    }
    __builtin_amdgcn_s_setprio(1);
    f32x16 S;
#pragma unroll
    for (int i = 0; i < 16; ++i) S[i] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if constexpr (LA > 0) {
        S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[j % LA], qf[j], S, 0, 0, 0);
        if (j + LA < FPB) win[j % LA] = frag(j + LA);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag(j), qf[j], S, 0, 0, 0);
      }
    }
    if (k0 + 32 > all) {
      asm volatile("" ::: "memory");  // keeps the branch
      const int at0 = k0 + 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (at0 + 8 * (i >> 2) + (i & 3) >= lim) S[i] = -INFINITY;
    }
    __builtin_amdgcn_s_setprio(0);
    bf16x8 P[2];
    soft_block<ND>(S, c, st, O, P);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int jv = 0; jv < 2 * ND; ++jv) {
      if constexpr (LA > 0) {
        const int i = NJ + jv;
        O[jv % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(win[i % LA], P[jv / ND], O[jv % ND], 0, 0, 0);
        if (i + LA < FPB) win[i % LA] = frag(i + LA);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        O[jv % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag(NJ + jv), P[jv / ND], O[jv % ND], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };

  int slot = 0, fill = SLOTS - 1;
  for (int t = 0; t < nt; ++t) {
    // this wave's share of slot t has landed (the SLOTS - 2 slots requested after it may be on their way), and everyone's; the slot
    // read last is free
    if (SLOTS > 2 && t + 1 < nt) __builtin_amdgcn_s_waitcnt(0x0F70 | ((SLOTS - 2) * 2 * GPW));
    else __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    if (t + SLOTS - 1 < nt) request(fill, t + SLOTS - 1);
    const unsigned at = smem_addr + (unsigned)(slot * F::Slot);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int k0 = t * F::Keys + 32 * b;
      if (k0 < some) block(at + (unsigned)(b * T::Bytes), k0);
    }
    slot = slot == SLOTS - 1 ? 0 : slot + 1;
    fill = fill == SLOTS - 1 ? 0 : fill + 1;
  }
  __syncthreads();  // every wave has finished reading the ring, and no load into it is in flight: it now stages the output
  const float l = xhalf_sum(st.l), mc = st.mc;

  if (split) {
    if (r0 + l32 >= rows) return;
    const int64_t at = ((int64_t)piece * a.kv_heads + head) * group_rows + (int64_t)s.q0 * G + r0 + l32;
    if (hh == 0) a.ml[at] = make_float2(mc, l);
    if (nt <= 0) return;
    float* p = a.part + at * a.D + 4 * hh;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (!PADDED || db * 32 + 8 * g < a.D)
          *reinterpret_cast<f32x4*>(p + db * 32 + 8 * g) = f32x4{O[db][4 * g], O[db][4 * g + 1], O[db][4 * g + 2], O[db][4 * g + 3]};
    return;
  }
  static_assert(4 * 32 * kOutRow<ND> <= SLOTS * F::Slot, "the staged rows fit the ring");
  store_out<ND, DC, PADDED>(a, s, O, l, mc, head, r0, lane, smem + wave * 32 * kOutRow<ND>);
}

// ---------------------------------------------------------------------------------------------------------------------- pipelined
// The same for head dim 128, software-pipelined inside the wave: one instruction stream holds the eight PV products of key block b - 1, the eight
// score products of block b + 1 and the softmax of block b, with a share of the softmax behind each product and the LDS read of a
// fragment one product of its kind ahead of its use.  64 keys per slot, K(t) beside V(t - 1), in a ring of four slots (128 KB, a
// workgroup per CU), whose loads are two slots ahead of their use; one barrier per 64 keys.  Blocks in front of the first and behind the last are
// masked whole (P = 0) and walked like the others.
constexpr int kPipeSlot = 4 * PackedBlock<128>::Bytes, kPipeHalf = 2 * PackedBlock<128>::Bytes, kPipeBytes = 4 * kPipeSlot;

__device__ const u32x4 kZeros = {0u, 0u, 0u, 0u};

template <int NW>
__global__ __launch_bounds__(NW * 64) void packed_pipe_kernel(PackedArgs a) {
  using T = PackedBlock<128>;
  constexpr int BM = NW * 32, GPW = 16 / NW;  // row groups per wave, slot and tensor
  constexpr int kFirst = 2;                   // the product behind which the softmax starts: the scores' last one has left the pipe
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rank = blockIdx.x / a.kv_heads, head = blockIdx.x - rank * a.kv_heads, G = a.group.d;
  const SeqTile s = find_tile<BM, false>(a.seqs, G, rank, lane);
  if (s.none) return;
  if (s.gap) {
    if (tid < 256) fill_gap<BM, 128>(a, s, head, tid);
    return;
  }
  const int rows = s.m * G, r0 = s.tile * BM + wave * 32;
  auto token_of = [&](int r) __attribute__((always_inline)) { return (int)div_by((unsigned)r, a.group); };
  const int r = min(r0 + l32, rows - 1), token = token_of(r);  // (rows past the end repeat the last one and are not stored)
  auto sees = [&](int t) __attribute__((always_inline)) { return a.causal ? min(max(t + 1 + s.n - s.m, 0), s.n) : s.n; };
  const int lim = sees(token), all = __builtin_amdgcn_readlane(lim, 0), some = __builtin_amdgcn_readlane(lim, 31);
  const int nt = (sees(token_of(min(s.tile * BM + BM, rows) - 1)) + 63) / 64;  // slots that hold a key that some row of the workgroup sees

  bf16x8 qf[8];
  {
    const __bf16* p = a.q + (int64_t)(s.q0 + token) * a.qs.row + (int64_t)(head * G + r - token * G) * a.qs.head + hh * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) qf[j] = *reinterpret_cast<const bf16x8*>(p + j * 16);
  }
  const __bf16* kp = a.k + (int64_t)s.k0 * a.ks.row + head * a.ks.head;
  const __bf16* vp = a.v + (int64_t)s.k0 * a.vs.row + head * a.vs.head;
  const unsigned smem_addr = lds_addr_of(smem);
  const int grow = T::row(lane), col = T::chunk(lane, wave) * 8;  // (groups wave, wave + 4, ...: the swizzle sees the same)
  const unsigned kofs = (unsigned)(grow * (int)a.ks.row + col) * 2u, vofs = (unsigned)(grow * (int)a.vs.row + col) * 2u;
  auto request = [&](int slot, int t) __attribute__((always_inline)) {
    const unsigned Ks = smem_addr + (unsigned)(slot * kPipeSlot), Vs = Ks + kPipeHalf;
    if (t >= 1 && t * 64 + 64 <= s.n) {
#pragma unroll
      for (int i = 0; i < GPW; ++i) {
        const int g = wave + NW * i;
        lds_dma16(kp + (int64_t)(t * 64 + 4 * g) * a.ks.row, kofs, Ks + (unsigned)g * 1024u);
        lds_dma16(vp + (int64_t)(t * 64 - 64 + 4 * g) * a.vs.row, vofs, Vs + (unsigned)g * 1024u);
      }
    } else {  // keys past the sequence's end repeat its last one and meet masked logits; V's rows outside it are zeros, which P = 0 meets
#pragma unroll
      for (int i = 0; i < GPW; ++i) {
        const int g = wave + NW * i, row = t * 64 + 4 * g + grow;
        const __bf16* v = (unsigned)(row - 64) < (unsigned)s.n ? vp + (int64_t)(row - 64) * a.vs.row + col : reinterpret_cast<const __bf16*>(&kZeros);
        lds_dma16(kp + (int64_t)min(row, s.n - 1) * a.ks.row + col, Ks + (unsigned)g * 1024u);
        lds_dma16(v, Vs + (unsigned)g * 1024u);
      }
    }
  };
  if (nt > 0) {
    request(0, 0);
    request(1, 1);
    request(2, 2);
  }
  f32x16 O[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[db][i] = 0.f;
  const float c = a.c;
  RowState st{-1e30f, -1e30f * c, 0.f};
  f32x16 Sa, Sb;        // logits of odd, even blocks
  u32x4 Pa[2], Pb[2];   // probabilities of odd, even blocks as the PV product's operand
  bf16x8 kf[2], vf[2];  // fragments read ahead
#pragma unroll
  for (int i = 0; i < 16; ++i) { Sa[i] = -INFINITY; Sb[i] = 0.f; }  // block -1
#pragma unroll
  for (int i = 0; i < 2; ++i) Pa[i] = Pb[i] = u32x4{0u, 0u, 0u, 0u};

  const unsigned row_at = smem_addr + T::row_at(lane), trans_at = smem_addr + T::trans_at(lane);
  // fragment j of K's block at byte `at` of the ring, jv of V's
  auto k_frag = [&](int at, int j) __attribute__((always_inline)) { return read_row_frag((row_at ^ (unsigned)(32 * j)) + (unsigned)at); };
  auto v_frag = [&](int at, int jv) __attribute__((always_inline)) {
    const unsigned x = trans_at ^ (unsigned)(64 * (jv & 3));
    return read_trans_frag(x + (unsigned)(at + (jv >> 2) * 16 * T::Row), (x ^ 32u) + (unsigned)(at + (8 + (jv >> 2) * 16) * T::Row));
  };
  // One block: the softmax of SC (block blk) into PC, the product of PP (blk - 1) with V at vc, the scores SN (blk + 1) from K at kc; kn, vn: the
  // places of the next ones.
  auto iter = [&](f32x16& SC, f32x16& SN, u32x4 (&PC)[2], u32x4 (&PP)[2], int kc, int kn, int vc, int vn, int blk) __attribute__((always_inline)) {
    if (blk * 32 + 32 > all) {
      asm volatile("" ::: "memory");  // keeps the branch
      const int at0 = blk * 32 + 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (at0 + 8 * (i >> 2) + (i & 3) >= lim) SC[i] = -INFINITY;
    }
    float sum = 0.f, even = 0.f;
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      const int j = n >> 1;
      if ((n & 1) == 0) {
        O[j & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[j & 1], __builtin_bit_cast(bf16x8, PP[j >> 2]), O[j & 3], 0, 0, 0);
        vf[(j + 1) & 1] = j < 7 ? v_frag(vc, j + 1) : v_frag(vn, 0);
      } else {
        if (j == 0) {
          f32x16 z;
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = 0.f;
          SN = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[0], qf[0], z, 0, 0, 0);
        } else {
          SN = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[j & 1], qf[j], SN, 0, 0, 0);
        }
        kf[(j + 1) & 1] = j < 7 ? k_frag(kc, j + 1) : k_frag(kn, 0);
      }
      const int e0 = n < kFirst ? 0 : (n - kFirst) * 16 / (16 - kFirst), e1 = n < kFirst ? 0 : (n + 1 - kFirst) * 16 / (16 - kFirst);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (e < e0 || e >= e1) continue;
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(SC[e], c, -st.mc));
        if ((e & 1) == 0) {
          even = x;
          asm volatile("" : "+v"(even));  // pins the work behind its product
        } else {
          unsigned pk = pack2(even, x);
          sum = e == 1 ? even + x : sum + (even + x);
          asm volatile("" : "+v"(pk), "+v"(sum));
          PC[e >> 3][(e >> 1) & 3] = pk;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum <= kRange)) != 0, 0)) {  // (no product with V is on its way here)
      bf16x8 P[2];
      soft_block<4>(SC, c, st, O, P);
#pragma unroll
      for (int i = 0; i < 2; ++i) PC[i] = __builtin_bit_cast(u32x4, P[i]);
      sum = 0.f;
    }
    st.l += sum;
  };

  const int last = (some + 31) / 32;  // the block behind this wave's last: its iteration holds that one's product with V
  auto period = [&](int t, auto slot) __attribute__((always_inline)) {
    constexpr int cur = decltype(slot)::value * kPipeSlot, nxt = ((decltype(slot)::value + 1) & 3) * kPipeSlot, B = T::Bytes, H = kPipeHalf;
    // slot t + 1 has landed, this wave's share and everyone's (the one requested after it may be on its way); slot t - 1 has been read
    if (t + 2 <= nt) __builtin_amdgcn_s_waitcnt(0x0F70 | (2 * GPW));
    else __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    if (2 * t - 1 <= last) iter(Sa, Sb, Pa, Pb, cur, cur + B, cur + H, cur + H + B, 2 * t - 1);
    // in the middle of the period, where not all waves queue for it
    if (t + 3 <= nt) request((decltype(slot)::value + 3) & 3, t + 3);
    if (2 * t <= last) iter(Sb, Sa, Pb, Pa, cur + B, nxt, cur + H + B, nxt + H, 2 * t);
  };
  if (nt > 0) {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    kf[0] = k_frag(0, 0);
    vf[0] = v_frag(kPipeHalf, 0);
    for (int t = 0; t <= nt; t += 4) {
      period(t, std::integral_constant<int, 0>{});
      if (t + 1 > nt) break;
      period(t + 1, std::integral_constant<int, 1>{});
      if (t + 2 > nt) break;
      period(t + 2, std::integral_constant<int, 2>{});
      if (t + 3 > nt) break;
      period(t + 3, std::integral_constant<int, 3>{});
    }
  }
  __syncthreads();  // every wave has finished reading the ring, and no load into it is in flight: it now stages the output
  store_out<4, 128, false>(a, s, O, xhalf_sum(st.l), st.mc, head, r0, lane, smem + wave * 32 * kOutRow<4>);
}

// ---------------------------------------------------------------------------------------------------------------------- few rows
// 32 rows of a group (four tokens of eight heads, say) per workgroup, all four waves the same ones.  The keys go by pieces of piece_keys, one to a
// workgroup at a time; in a piece the waves take blocks of 32 keys in turn, each through buffers of its own in LDS, one for K and one for V, so that no
// wave waits for another: the next K is requested once the scores of this one are formed, the next V once its product is.  Four waves and
// two workgroups per CU keep some 64 to 128 KB of keys on their way, what 256 CUs need at 8 TB/s.  The waves' sums are joined through LDS,
// the pieces' by packed_combine_kernel.  The workgroups walk the list of pieces, whose length is known on the device only.
template <int HD>
constexpr int few_bytes() {
  constexpr int ring = 8 * PackedBlock<HD>::Bytes, stage = (4 * 32 * 68 + 4 * 32 * 2) * 4;
  return ring > stage ? ring : stage;
}
template <int HD, int DC, bool PADDED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 3 : 2, HD == 64 ? 3 : 2))) void packed_few_kernel(PackedArgs a) {
  using T = PackedBlock<HD>;
  constexpr int NJ = DC / 16, ND = (DC + 31) / 32, LPB = 32 / T::RPI;  // loads per block and tensor
  constexpr int NV = HD == 128 ? 4 : 2;                                 // row groups that the swizzle tells apart
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.group.d;
  const int64_t group_rows = (int64_t)a.seqs.q_rows * G;
  auto token_of = [&](int r) __attribute__((always_inline)) { return (int)div_by((unsigned)r, a.group); };
  const unsigned mine = lds_addr_of(smem) + (unsigned)(wave * 2 * T::Bytes), row_at = T::row_at(lane), trans_at = T::trans_at(lane);
  const int grow = T::row(lane);
  int col[NV];
  [[maybe_unused]] uint64_t mask[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = T::chunk(lane, i) * 8;
    mask[i] = __builtin_amdgcn_ballot_w64(col[i] < a.D);
    if (PADDED && col[i] >= a.D) col[i] = 0;
  }
  const float c = a.c;

  for (int item = blockIdx.x;; item += gridDim.x) {
    const int rank = item / a.kv_heads, head = item - rank * a.kv_heads;
    int piece;
    const SeqTile s = find_piece(a.seqs, G, rank, lane, a.piece_keys, a.pieces, piece);
    if (s.none) return;
    if (s.gap) {
      fill_gap<32, HD>(a, s, head, tid);
      continue;
    }
    const int rows = s.m * G, r0 = s.tile * 32, kb = piece * a.piece_keys;
    const int ke = piece == a.pieces - 1 ? s.n : min(s.n, kb + a.piece_keys);
    const int r = min(r0 + l32, rows - 1), token = token_of(r);  // (rows past the end repeat the last one and are not stored)
    auto sees = [&](int t) __attribute__((always_inline)) { return min(ke, a.causal ? max(t + 1 + s.n - s.m, 0) : s.n) - kb; };
    const int lim = sees(token), all = __builtin_amdgcn_readlane(lim, 0), some = __builtin_amdgcn_readlane(lim, 31);
    const int nt = (some - 32 * wave + 127) / 128;  // this wave's blocks: 128 t + 32 wave; zero or less: none

    const __bf16* kp = a.k + (int64_t)(s.k0 + kb) * a.ks.row + head * a.ks.head;
    const __bf16* vp = a.v + (int64_t)(s.k0 + kb) * a.vs.row + head * a.vs.head;
    auto request = [&](const __bf16* p, const RowStrides& st, unsigned to, int t) __attribute__((always_inline)) {
      const int k0 = t * 128 + 32 * wave;
#pragma unroll
      for (int i = 0; i < LPB; ++i) {
        // rows past the sequence's end repeat its last one
        const __bf16* at = p + (int64_t)min(k0 + T::RPI * i + grow, s.n - kb - 1) * st.row + col[i % NV];
        if constexpr (PADDED) lds_dma16(at, to + (unsigned)i * 1024u, mask[i % NV]);
        else lds_dma16(at, to + (unsigned)i * 1024u);
      }
    };
    if constexpr (PADDED) {  // chunks past the head dim: zeros that no load touches
      for (int i = lane * 16; i < 2 * T::Bytes; i += 1024) *reinterpret_cast<uint4*>(smem + wave * 2 * T::Bytes + i) = make_uint4(0u, 0u, 0u, 0u);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (nt > 0) {
      request(kp, a.ks, mine, 0);
      request(vp, a.vs, mine + T::Bytes, 0);
    }
    bf16x8 qf[NJ];
    load_row<NJ, PADDED>(qf, a.q + (int64_t)(s.q0 + token) * a.qs.row + (int64_t)(head * G + r - token * G) * a.qs.head + hh * 8, hh, a.D);
    f32x16 O[ND];
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) O[db][i] = 0.f;
    RowState st{-1e30f, -1e30f * c, 0.f};
    for (int t = 0; t < nt; ++t) {
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LPB) : "memory");  // K has landed, V may be on its way
      f32x16 S;
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_row_frag((mine + row_at) ^ (unsigned)(32 * j)), qf[j], S, 0, 0, 0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K's buffer has been read
      if (t + 1 < nt) request(kp, a.ks, mine, t + 1);
      const int k0 = t * 128 + 32 * wave;
      if (k0 + 32 > all) {
        asm volatile("" ::: "memory");  // keeps the branch
        const int at0 = k0 + 4 * hh;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (at0 + 8 * (i >> 2) + (i & 3) >= lim) S[i] = -INFINITY;
      }
      bf16x8 P[2];
      soft_block<ND>(S, c, st, O, P);
      if (t + 1 < nt) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LPB) : "memory");  // V has landed, the next K may be on its way
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int jv = 0; jv < 2 * ND; ++jv) {
        const unsigned v = (mine + T::Bytes + trans_at) ^ (unsigned)(64 * (jv % ND));
        constexpr int Up = T::Row;
        O[jv % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            read_trans_frag(v + (unsigned)(jv / ND * 16 * Up), (v ^ 32u) + (unsigned)((8 + jv / ND * 16) * Up)), P[jv / ND], O[jv % ND], 0, 0, 0);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V's buffer has been read
      if (t + 1 < nt) request(vp, a.vs, mine + T::Bytes, t + 1);
    }
    st.l = xhalf_sum(st.l);

    // the four waves' shares brought to one reference point, 64 columns of a head at a time
    constexpr int Ld = 64 + 4;  // floats of a staged row
    static_assert((4 * 32 * Ld + 4 * 32 * 2) * 4 <= few_bytes<HD>(), "the staged rows fit");
    float* stage = reinterpret_cast<float*>(smem);
    float2* ml = reinterpret_cast<float2*>(stage + 4 * 32 * Ld);
    const int64_t part_row = ((int64_t)piece * a.kv_heads + head) * group_rows + (int64_t)s.q0 * G;  // of the sequence's first row
#pragma unroll
    for (int d0 = 0; d0 < ND; d0 += 2) {
      __syncthreads();  // the buffers, or the columns before, have been read
#pragma unroll
      for (int db = d0; db < (d0 + 2 < ND ? d0 + 2 : ND); ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(stage + (wave * 32 + l32) * Ld + (db - d0) * 32 + 8 * g + 4 * hh) =
              f32x4{O[db][4 * g], O[db][4 * g + 1], O[db][4 * g + 2], O[db][4 * g + 3]};
      if (hh == 0) ml[wave * 32 + l32] = make_float2(st.mc, st.l);
      __syncthreads();
      const int lr = tid >> 3, cc = (tid & 7) * 8, row = r0 + lr, at = d0 * 32 + cc;
      if (row >= rows || at >= (PADDED ? a.D : DC)) continue;
      float top = -INFINITY, sum = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (ml[w * 32 + lr].y != 0.f) top = fmaxf(top, ml[w * 32 + lr].x);  // (a share without weight carries no reference point)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 u = ml[w * 32 + lr];
        const float x = u.y != 0.f ? __builtin_amdgcn_exp2f(u.x - top) : 0.f;
        const float* o = stage + (w * 32 + lr) * Ld + cc;
        sum += x * u.y;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += x * o[e];
      }
      if (a.part) {
        if (at == 0) {
          a.ml[part_row + row] = make_float2(top, sum);
          // the first piece says of the pieces that the sequence does not have that they have no weight
          if (piece == 0)
            for (int p = max(1, (s.n + a.piece_keys - 1) / a.piece_keys); p < a.pieces; ++p) a.ml[p * group_rows * a.kv_heads + part_row + row] = make_float2(0.f, 0.f);
        }
        f32x4* p = reinterpret_cast<f32x4*>(a.part + (part_row + row) * a.D + at);
        p[0] = f32x4{f[0], f[1], f[2], f[3]};
        p[1] = f32x4{f[4], f[5], f[6], f[7]};
        continue;
      }
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= inv;
      const int t = token_of(row), h = head * G + row - t * G;
      *reinterpret_cast<uint4*>(a.out + (int64_t)(s.q0 + t) * a.os.row + (int64_t)h * a.os.head + at) = pack8(f);
      if (at == 0 && a.lse) a.lse[(int64_t)h * a.seqs.q_rows + s.q0 + t] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
    }
    __syncthreads();  // the next piece's keys go where the rows were staged
  }
}

// The pieces of the keys joined, in their order: a workgroup per row, lane p of each wave with the weight of piece p, each wave the sums of every
// fourth piece.  All loads go out at once, those of pieces without weight among them, whose rows are not used: 64 pieces of 32 rows 8.7 -> @@ us.
constexpr int kMaxPieces = 64;
__global__ __launch_bounds__(256) void packed_combine_kernel(PackedArgs a) {
  __shared__ float part[3][128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x, group_rows = (int64_t)a.seqs.q_rows * a.group.d, rows = group_rows * a.kv_heads;
  const int head = (int)(row / group_rows), c = 2 * lane;
  const unsigned rg = (unsigned)(row - head * group_rows), t = div_by(rg, a.group), h = head * a.group.d + rg - t * a.group.d;
  const int first = a.seqs.q_off[0], last = a.seqs.q_off[a.seqs.count];
  const float2 u = a.ml[min(lane, a.pieces - 1) * rows + row];
  const float* p = a.part + row * a.D + (c < a.D ? c : 0);
  float2 o[kMaxPieces / 4];
#pragma unroll
  for (int i = 0; i < kMaxPieces / 4; ++i)
    if (4 * i + wave < a.pieces) o[i] = *reinterpret_cast<const float2*>(p + (4 * i + wave) * rows * a.D);
  if ((int)t < first || (int)t >= last) return;  // rows of no sequence: zeros already
  const bool has = lane < a.pieces && u.y != 0.f;
  float top = has ? u.x : -INFINITY;  // (a piece without weight carries no reference point)
#pragma unroll
  for (int i = 1; i < 64; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
  const float x = has ? __builtin_amdgcn_exp2f(u.x - top) : 0.f;
  float sum = has ? x * u.y : 0.f;
#pragma unroll
  for (int i = 1; i < 64; i *= 2) sum += __shfl_xor(sum, i);
  float f0 = 0.f, f1 = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxPieces / 4; ++i) {
    if (4 * i + wave >= a.pieces) break;
    const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 4 * i + wave));
    if (w == 0.f) continue;  // (nothing may stand there; a weight that is not a number stays one)
    f0 += w * o[i].x;
    f1 += w * o[i].y;
  }
  if (wave) {
    part[wave - 1][c] = f0;
    part[wave - 1][c + 1] = f1;
  }
  __syncthreads();
  if (wave || c >= a.D) return;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    f0 += part[w][c];
    f1 += part[w][c + 1];
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  *reinterpret_cast<unsigned*>(a.out + (int64_t)t * a.os.row + (int64_t)h * a.os.head + c) = pack2(f0 * inv, f1 * inv);
  if (c == 0 && a.lse) a.lse[(int64_t)h * a.seqs.q_rows + t] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
}

// How a call is launched.
struct FwdPlan {
  int kind, pieces, piece_keys;
  int64_t floats, tiles;  // tiles: of 128 rows (few rows: 32), of all heads
  void cut(const mdattn_packed* p, int64_t max_k, int64_t keys) {
    keys = (std::max(keys, (max_k + kMaxPieces - 1) / kMaxPieces) + 127) / 128 * 128;
    const int64_t n = (max_k + keys - 1) / keys;
    if (n < 2) return;
    pieces = (int)n;
    piece_keys = (int)keys;
    floats = n * p->q_rows * p->heads * (p->head_dim + 2);
  }
};
enum { kFew, kFlat, kPipe4, kPipe8 };
FwdPlan fwd_plan(const mdattn_packed* p) {
  const int64_t group = p->heads / p->kv_heads;
  const int64_t max_q = p->max_q > 0 && p->max_q < p->q_rows ? p->max_q : p->q_rows, max_k = p->max_k > 0 && p->max_k < p->k_rows ? p->max_k : p->k_rows;
  FwdPlan f{kFlat, 1, 1 << 30, 0, 0};
  // (the list of all tiles' pieces is counted in 31 bits)
  if (max_q * group <= 32 && packed_tiles(p->q_rows * group, p->sequences, 32) * kMaxPieces * p->kv_heads < (1ll << 31)) f.kind = kFew;
  const int bm = f.kind == kFew ? 32 : 128;
  // tiles that there are: of the tokens, or of so many sequences of the longest one's
  f.tiles = std::min((max_q * group + bm - 1) / bm * p->sequences, p->q_rows * group / bm + p->sequences) * p->kv_heads;
  if (f.kind == kFew) {
    const int64_t all = std::min(max_k * p->sequences, (int64_t)p->k_rows) * p->kv_heads;
    if (max_k >= 512) f.cut(p, max_k, std::max<int64_t>(all / 2048, 256));
    return f;
  }
  const int64_t blocks = (max_k + 31) / 32;
  if (f.tiles > 256) {
    // (tiles of 256 rows that fill their last round)
    const int64_t rounds = (f.tiles + 511) / 512;
    if (p->head_dim == 128 && !p->causal && blocks >= 128 && f.tiles >= rounds * 480) f.kind = kPipe8;
    return f;
  }
  const bool pipe = p->head_dim == 128;
  if (pipe) f.kind = kPipe4;
  // Alone on its CU a workgroup takes so many us per block of 32 keys; in n pieces, of the flat schedule, one n-th of them, and their rows go to
  // memory and back, at some 4 TB/s, through a launch of 5 us.
  const double row_us = (double)p->q_rows * p->heads * p->head_dim * 4 * 2 / 4e6 * (p->causal ? 0.6 : 1.0);
  double best = 0.95 * blocks * (pipe ? 0.56 : 0.75);
  int64_t pieces = 1;
  for (int64_t n = 2; n <= 16 && blocks / n >= 16 && f.tiles * n <= 512; ++n) {
    const double us = (double)blocks / n * (f.tiles * n <= 256 ? 0.75 : 1.06) + n * row_us + 5;
    if (us < best) { best = us; pieces = n; }
  }
  if (pieces > 1) {
    f.kind = kFlat;
    f.cut(p, max_k, (max_k + pieces - 1) / pieces);
  }
  return f;
}

template <int NW>
int launch_pipe(hipStream_t st, const PackedArgs& a, int64_t grid) {
  static LdsOptIn opted;
  if (lds_opt_in(opted, reinterpret_cast<const void*>(packed_pipe_kernel<NW>), kPipeBytes) != MDATTN_OK) return MDATTN_E_LAUNCH;
  MDATTN_LAUNCH(packed_pipe_kernel<NW>, dim3((unsigned)grid), dim3(NW * 64), kPipeBytes, st, a);
  return launch_status();
}

template <int HD, int DC, bool PADDED>
int launch(hipStream_t st, const PackedArgs& a, int kind, int64_t grid) {
  if (kind == kFew) {
    MDATTN_LAUNCH((packed_few_kernel<HD, DC, PADDED>), dim3((unsigned)grid), dim3(256), few_bytes<HD>(), st, a);
  } else if (kind == kFlat || HD != 128 || PADDED) {
    MDATTN_LAUNCH((packed_fwd_kernel<HD, DC, PADDED>), dim3((unsigned)grid, (unsigned)a.pieces), dim3(256), FwdShape<HD>::SLOTS * FwdShape<HD>::Slot, st, a);
  } else {
    return kind == kPipe4 ? launch_pipe<4>(st, a, grid) : launch_pipe<8>(st, a, grid);
  }
  return launch_status();
}

}  // namespace
}  // namespace mdattn

using namespace mdattn;

extern "C" int64_t mdattn_fwd_bf16_packed_workspace_floats(const mdattn_packed* p) {
  return packed_sizes(p) == MDATTN_OK ? fwd_plan(p).floats : 0;
}

extern "C" int mdattn_fwd_bf16_packed(void* stream, const mdattn_packed* p, const void* q, const void* k, const void* v, void* out, float* lse,
                                      const mdattn_strides* q_strides, const mdattn_strides* k_strides, const mdattn_strides* v_strides,
                                      const mdattn_strides* o_strides, float scale, float* workspace, int64_t workspace_floats) {
  const int rc = packed_sizes(p);
  if (rc != MDATTN_OK) return rc;
  if (!(scale > 0.f) || !(scale < INFINITY) || !q_strides || !k_strides || !v_strides || !o_strides) return MDATTN_E_BADARG;
  if (p->q_rows == 0) return MDATTN_OK;  // nothing to be written
  if (!q || !out || (p->k_rows && (!k || !v))) return MDATTN_E_BADARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !packed_aligned(p) || (reinterpret_cast<uintptr_t>(lse) & 3) ||
      !packed_strides_ok(q_strides) || !packed_strides_ok(k_strides) || !packed_strides_ok(v_strides) || !packed_strides_ok(o_strides))
    return MDATTN_E_ALIGN;
  FwdPlan f = fwd_plan(p);
  if (f.pieces > 1 && (!workspace || workspace_floats < f.floats)) {  // (flat or few rows)
    f.pieces = 1;
    f.piece_keys = 1 << 30;
  } else if (f.pieces > 1 && !aligned16(workspace)) {
    return MDATTN_E_ALIGN;
  }
  PackedArgs a{};
  a.q = static_cast<const __bf16*>(q); a.k = static_cast<const __bf16*>(k); a.v = static_cast<const __bf16*>(v);
  a.out = static_cast<__bf16*>(out); a.lse = lse;
  a.seqs = {p->q_offsets, p->k_offsets, p->k_lengths, p->sequences, p->q_rows, p->k_rows, f.kind == kFew ? kAsTheyCome : packed_order(p, f.tiles), 256 / p->kv_heads};
  a.group = divisor((unsigned)(p->heads / p->kv_heads));
  a.kv_heads = p->kv_heads; a.D = p->head_dim; a.causal = p->causal;
  a.qs = {q_strides->seq, q_strides->head}; a.ks = {k_strides->seq, k_strides->head};
  a.vs = {v_strides->seq, v_strides->head}; a.os = {o_strides->seq, o_strides->head};
  a.c = scale * kLog2e;
  a.pieces = f.pieces; a.piece_keys = f.piece_keys;
  const int64_t rows = (int64_t)p->q_rows * p->heads, group_rows = (int64_t)p->q_rows * a.group.d;
  if (f.pieces > 1) {
    a.part = workspace;
    a.ml = reinterpret_cast<float2*>(workspace + f.pieces * rows * a.D);
  }
  int64_t grid = packed_tiles(group_rows, p->sequences, f.kind == kFew ? 32 : f.kind == kPipe8 ? 256 : 128) * p->kv_heads;
  if (f.kind == kFew) {  // two per CU, in whole rounds of the heads, walk what there is
    const int64_t most = (512 + a.kv_heads - 1) / a.kv_heads * a.kv_heads;
    grid = grid * f.pieces < most ? grid * f.pieces : most;
  }
  if (!grid_fits(grid, f.kind == kPipe8 ? 512 : 256) || (f.pieces > 1 && !grid_fits(rows, 256))) return MDATTN_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const int status = a.D == 64   ? launch<64, 64, false>(st, a, f.kind, grid)
                     : a.D < 64  ? launch<64, 64, true>(st, a, f.kind, grid)
                     : a.D <= 96 ? launch<128, 96, true>(st, a, f.kind, grid)
                     : a.D < 128 ? launch<128, 128, true>(st, a, f.kind, grid)
                                 : launch<128, 128, false>(st, a, f.kind, grid);
  if (status != MDATTN_OK || f.pieces == 1) return status;
  MDATTN_LAUNCH(packed_combine_kernel, dim3((unsigned)rows), dim3(256), 0, st, a);
  return launch_status();
}

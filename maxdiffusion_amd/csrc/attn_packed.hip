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
// Few tiles leave CUs idle: two waves then share the keys of 64 rows, or four waves those of 32 (a kernel of its own, that one token meets too).
// Where a tile is all that a sequence has, its keys are cut into pieces besides; each leaves un-normalised f32 rows, joined by another kernel
// in a fixed order.
// Roundings.  Logits, softmax and sums are f32; P goes into its product in bf16, 2^-9 of an element on average, because the matrix pipes take f32 at a
// sixteenth of the rate, and in two parts of bf16 P V would be twice the work: out is off by 1.1 to 1.5 times what its own rounding makes.
// Bound: by the matrix pipes and LDS alike with long sequences (16,384 tokens, 32 heads on 8, causal: 1,895 us, 1.16 PFLOP/s, pipes busy 71 % of the
// cycles; a library's product of 8,192^3 reaches 1.16; other machines 1,811 to 1,885); head dim 64, where a product has half the softmax's work beside
// it, 1,107 us, 0.99; by the keys' way from memory with one token (131,072 keys of 8 heads 101 us, 5.3 TB/s); by the longest walk of a tile, products and
// softmax in turn (prompts of up to 512 tokens 17 us; 4 x 512 tokens against 5,000 to 16,384 keys by two waves 477 us, 0.71 PFLOP/s).
#include <algorithm>

#include "attn_packed.h"
#include "mdattn_host.h"

namespace mdattn {
namespace {

constexpr float kRange = 16777216.f;  // a partial sum of P above 2^24 moves the row's reference point

struct PackedArgs {
  const __bf16 *q, *k, *v;
  __bf16 *out, *rest;
  float* lse;
  PackedSeqs seqs;
  Divisor group;
  int kv_heads, D, causal;
  RowStrides qs, ks, vs, os;
  float c;  // scale * log2(e)
  int pieces, piece_keys, items;  // items: see packed_few_kernel
  float* part;  // [piece][kv_heads][q_rows * group][D]
  float2* ml;   // [piece][kv_heads][q_rows * group]: reference point (log2 units) and sum of P
};

// KW: the waves that deal a slot's keys among them; 4 / KW waves of 32 rows.
template <int HD, int KW>
struct FwdShape {
  static constexpr int NB = HD == 64 ? 2 : 1;               // blocks of 32 keys that a wave computes per slot
  static constexpr int SLOTS = HD == 64 || KW == 2 ? 2 : 3;
  static constexpr int Blocks = NB * KW, Keys = 32 * Blocks, Half = Blocks * PackedBlock<HD>::Bytes, Slot = 2 * Half;
  static constexpr int BM = 128 / KW;
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
// every block of keys, and with that for the keys requested since (16,384 tokens x 32 heads 1,895 -> 1,835 us).
template <int NJ, bool PADDED>
__device__ __forceinline__ void load_row(bf16x8 (&f)[NJ], const __bf16* p, int hh, int D) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) f[j] = !PADDED || j * 16 + hh * 8 < D ? *reinterpret_cast<const bf16x8*>(p + j * 16) : __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
#pragma unroll
  for (int j = 0; j < NJ; ++j) asm volatile("" : "+v"(f[j]));
}

// A pair of bf16 as floats
__device__ __forceinline__ float low_half(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_half(unsigned u) { return __uint_as_float(u & 0xFFFF0000u); }

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
  const int rr = lane / LPR, cc = lane % LPR;
  auto put = [&](__bf16* out, bool rest) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float f[4];
        uint2 u;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = O[db][4 * g + e] * inv;
        u.x = pack2(f[0], f[1]);
        u.y = pack2(f[2], f[3]);
        if (rest) {
          u.x = pack2(f[0] - low_half(u.x), f[1] - high_half(u.x));
          u.y = pack2(f[2] - low_half(u.y), f[3] - high_half(u.y));
        }
        *reinterpret_cast<uint2*>(stage + l32 * RowB + hh * 8 + (db * 32 + g * 8) * 2) = u;
      }
    // LDS accesses of one wave execute in order: the reads below see the writes above, and those of another call the reads
    if (cc * 8 >= (PADDED ? a.D : DC)) return;
#pragma unroll
    for (int j = 0; j < 32 / RPI; ++j) {
      const int row = r0 + j * RPI + rr;
      if (row >= rows) break;
      const int t = (int)div_by((unsigned)row, a.group);
      st_nt(reinterpret_cast<uint4*>(out + (int64_t)(s.q0 + t) * a.os.row + (int64_t)(head * G + row - t * G) * a.os.head + cc * 8),
            *reinterpret_cast<const uint4*>(stage + (j * RPI + rr) * RowB + cc * 16));
    }
  };
  put(a.out, false);
  if (a.rest) put(a.rest, true);
}

template <int HD, int DC, bool PADDED, int KW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(KW == 2 ? 2 : HD == 64 ? 4 : 3, KW == 2 ? 2 : HD == 64 ? 4 : 3)))
void packed_fwd_kernel(PackedArgs a) {
  using T = PackedBlock<HD>;
  using F = FwdShape<HD, KW>;
  constexpr int NJ = DC / 16, ND = (DC + 31) / 32, NB = F::NB, SLOTS = F::SLOTS;
  constexpr int GPW = F::Keys / T::RPI / 4;  // row groups per wave, slot and tensor
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // (fragment addresses are formed by xor)
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // neighbouring workgroups, which go to different dies, take different heads: with eight heads of k and v each die's L2 holds one of them
  const int rank = blockIdx.x / a.kv_heads, head = blockIdx.x - rank * a.kv_heads, G = a.group.d;
  const SeqTile s = find_tile<F::BM, false>(a.seqs, G, rank, lane);
  if (s.none) return;
  const int row_wave = KW == 1 ? wave : wave & 1, key_wave = KW == 1 ? 0 : wave >> 1;
  const int tile = s.tile, rows = s.m * G, r0 = tile * F::BM + row_wave * 32;
  auto token_of = [&](int r) __attribute__((always_inline)) { return (int)div_by((unsigned)r, a.group); };
  if (s.gap) {
    fill_gap<F::BM, HD>(a, s, head, tid);
    return;
  }

  const int r = min(r0 + l32, rows - 1);  // (rows past the end repeat the last one and are not stored)
  const int token = token_of(r);
  auto sees = [&](int t) __attribute__((always_inline)) { return a.causal ? min(max(t + 1 + s.n - s.m, 0), s.n) : s.n; };
  const int lim = sees(token);
  const int all = __builtin_amdgcn_readlane(lim, 0), some = __builtin_amdgcn_readlane(lim, 31);  // keys that all, some rows of the wave see
  const int end = sees(token_of(min(tile * F::BM + F::BM, rows) - 1));                           // some row of the workgroup
  const int nt = (end + F::Keys - 1) / F::Keys;                                                   // slots visited

  const __bf16* kp = a.k + (int64_t)s.k0 * a.ks.row + head * a.ks.head;
  const __bf16* vp = a.v + (int64_t)s.k0 * a.vs.row + head * a.vs.head;
  const unsigned smem_addr = lds_addr_of(smem);
  const int grow = T::row(lane), col0 = T::chunk(lane, wave) * 8;  // (groups wave, wave + 4, ...: the swizzle sees the same)
  const int col = !PADDED || col0 < a.D ? col0 : 0;
  [[maybe_unused]] const uint64_t mask = __builtin_amdgcn_ballot_w64(!PADDED || col0 < a.D);
  const unsigned kofs = (unsigned)(grow * (int)a.ks.row + col) * 2u, vofs = (unsigned)(grow * (int)a.vs.row + col) * 2u;
  auto load = [&](auto... at) __attribute__((always_inline)) {
    if constexpr (PADDED) lds_dma16(at..., mask);
    else lds_dma16(at...);
  };
  auto request = [&](int slot, int t) __attribute__((always_inline)) {
    const unsigned Ks = smem_addr + (unsigned)(slot * F::Slot), Vs = Ks + F::Half;
    if (t * F::Keys + F::Keys <= s.n) {
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
        const int64_t row = min(t * F::Keys + T::RPI * g + grow, s.n - 1);
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

  // a block of 32 keys, the first of them key k0 of the sequence, at `at` (its V a half slot on)
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
      const int i = key_wave * NB + b, k0 = t * F::Keys + 32 * i;
      if (k0 < some) block(at + (unsigned)(i * T::Bytes), k0);
    }
    slot = slot == SLOTS - 1 ? 0 : slot + 1;
    fill = fill == SLOTS - 1 ? 0 : fill + 1;
  }
  __syncthreads();  // every wave has finished reading the ring, and no load into it is in flight: it now stages the output
  float l = xhalf_sum(st.l), mc = st.mc;
  if constexpr (KW == 2) {  // the second waves' shares to the first, by one reference point
    constexpr int Ld = ND * 32 + 4;  // floats of a staged row
    static_assert(2 * 32 * (Ld * 4 + 8) <= SLOTS * F::Slot, "the staged rows fit the ring");
    float* to = reinterpret_cast<float*>(smem) + (row_wave * 32 + l32) * Ld + 4 * hh;
    float2* ml = reinterpret_cast<float2*>(smem + 2 * 32 * Ld * 4) + row_wave * 32 + l32;
    if (key_wave) {
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(to + db * 32 + 8 * g) = f32x4{O[db][4 * g], O[db][4 * g + 1], O[db][4 * g + 2], O[db][4 * g + 3]};
      if (hh == 0) *ml = make_float2(mc, l);
    }
    __syncthreads();
    if (key_wave) return;
    const float2 u = *ml;
    const float top = u.y == 0.f ? mc : l == 0.f ? u.x : fmaxf(mc, u.x);  // (a share without weight carries no reference point)
    const float x = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(mc - top), y = u.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(u.x - top);
    l = l * x + u.y * y;
    mc = top;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 o = *reinterpret_cast<const f32x4*>(to + db * 32 + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) O[db][4 * g + e] = O[db][4 * g + e] * x + o[e] * y;
      }
  }

  constexpr int Behind = KW == 2 ? 2 * 32 * ((ND * 32 + 4) * 4 + 8) : 0;  // (the other wave's share may still be read)
  static_assert(Behind + 4 / KW * 32 * kOutRow<ND> <= SLOTS * F::Slot, "the staged rows fit the ring");
  store_out<ND, DC, PADDED>(a, s, O, l, mc, head, r0, lane, smem + Behind + row_wave * 32 * kOutRow<ND>);
}

// ---------------------------------------------------------------------------------------------------------------------- few rows
// 32 rows of a group (four tokens of eight heads, say) per workgroup, all four waves the same ones.  The keys go by pieces of piece_keys, one to a
// workgroup at a time; in a piece the waves take blocks of 32 keys in turn, each through buffers of its own in LDS, one for K and one for V, so that no
// wave waits for another: the next K is requested once the scores of this one are formed, the next V once its product is.  Four waves and
// two workgroups per CU keep some 64 to 128 KB of keys on their way, what 256 CUs need at 8 TB/s.  The waves' sums are joined through LDS,
// the pieces' by packed_combine_kernel.  The workgroups walk the list of pieces, whose length is known on the device only, up to a.items of them:
// as many as offsets that do not decrease can make.  Offsets that go back and forth name rows many times over; their list would be as much longer, and
// its ranks pass 31 bits.
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

  int from = 0, before = 0;  // (the items' ranks rise)
  for (unsigned item = blockIdx.x; item < (unsigned)a.items; item += gridDim.x) {
    const int rank = item / a.kv_heads, head = item - rank * a.kv_heads;
    int piece;
    const SeqTile s = find_piece(a.seqs, G, rank, lane, a.piece_keys, a.pieces, from, before, piece);
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
      const int64_t to = (int64_t)(s.q0 + t) * a.os.row + (int64_t)h * a.os.head + at;
      const uint4 u = pack8(f);
      *reinterpret_cast<uint4*>(a.out + to) = u;
      if (a.rest) {
        float rounded[8];
        unpack8(u, rounded);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] -= rounded[e];
        *reinterpret_cast<uint4*>(a.rest + to) = pack8(f);
      }
      if (at == 0 && a.lse) a.lse[(int64_t)h * a.seqs.q_rows + s.q0 + t] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
    }
    __syncthreads();  // the next piece's keys go where the rows were staged
  }
}

// The pieces of the keys joined, in their order: a workgroup per row, lane p of each wave with the weight of piece p, each wave the sums of every
// fourth piece.  All loads go out at once, those of pieces without weight among them, whose rows are not used: 64 pieces of 32 rows 8.7 -> 4.7 us.
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
  const int64_t to = (int64_t)t * a.os.row + (int64_t)h * a.os.head + c;
  const unsigned both = pack2(f0 * inv, f1 * inv);
  *reinterpret_cast<unsigned*>(a.out + to) = both;
  if (a.rest) *reinterpret_cast<unsigned*>(a.rest + to) = pack2(f0 * inv - low_half(both), f1 * inv - high_half(both));
  if (c == 0 && a.lse) a.lse[(int64_t)h * a.seqs.q_rows + t] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
}

// How a call is launched.  With few tiles a call's time is the longest walk over the keys by one wave: 0.72 us per block of 32 keys for a
// workgroup alone on its CU with all waves in the rows' direction (flat), about half with two waves to share the keys (half), a quarter with
// four (few); with many it is the CUs' work, which costs half 15 % more than flat, whose workgroups read each key for twice the rows, and few two
// to three times as much.  us at head dim 128, few / half / flat: 512 tokens x 4 heads of k and v with groups of 4 (64 tiles) 11.0 / 11.7 / 15.8, 2,048 x 4
// (256 tiles) 45 / 32 / 48, 4 x 1,024 x 4 (512 tiles) 62 / 33 / 29, causal 4,096 x 4 (512) 129 / 86 / 97, 8,192 x 4 (1,024) 440 / 300 / 257, not causal 4,096
// x 4 210 / 149 / 131; 100 tokens at a time (256 tiles) 16 / 9.7 / 7.4.
enum { kFew, kHalf, kFlat };
struct FwdPlan {
  int kind, pieces, piece_keys;
  int64_t floats, tiles;  // tiles: of 128 rows, of all heads
  int order(const mdattn_packed* p) const { return kind == kFew ? kAsTheyCome : packed_order(p, tiles * (kind == kHalf && p->causal ? 2 : 1)); }
  // tiles with their pieces, of all heads, that the call has at most (few: below 2^31)
  int64_t items(const mdattn_packed* p) const {
    return packed_tiles((int64_t)p->q_rows * (p->heads / p->kv_heads), p->sequences, kind == kFew ? 32 : kind == kHalf ? 64 : 128) * pieces * p->kv_heads;
  }
};
FwdPlan fwd_plan(const mdattn_packed* p) {
  const int64_t group = p->heads / p->kv_heads;
  const int64_t max_q = p->max_q > 0 && p->max_q < p->q_rows ? p->max_q : p->q_rows, max_k = p->max_k > 0 && p->max_k < p->k_rows ? p->max_k : p->k_rows;
  FwdPlan f{kFlat, 1, 1 << 30, 0, 0};
  // tiles that there are: of the tokens, or of so many sequences of the longest one's; blocks of keys that the longest walk has
  f.tiles = std::min((max_q * group + 127) / 128 * p->sequences, p->q_rows * group / 128 + p->sequences) * p->kv_heads;
  const int64_t blocks = (max_k + 31) / 32;
  const bool one_tile = max_q * group <= 32, small = p->head_dim <= 64;
  if (one_tile || (f.tiles <= 64 && blocks >= (small ? 4 : 12)) || (small && f.tiles <= 128 && blocks >= 32)) f.kind = kFew;
  else if (f.tiles <= (p->causal && blocks >= 48 ? 512 : 256) && blocks >= (f.tiles <= 128 ? 4 : 8)) f.kind = kHalf;
  if (f.kind != kFew) return f;
  // (the list of all tiles' pieces is counted in 31 bits)
  if (packed_tiles(p->q_rows * group, p->sequences, 32) * kMaxPieces * p->kv_heads >= (1ll << 31) - (1 << 20)) {
    f.kind = kFlat;
    return f;
  }
  if (!one_tile || max_k < 512) return f;
  // (256 MiB of rows at most, whatever the hints are)
  const int64_t all = std::min(max_k * p->sequences, (int64_t)p->k_rows) * p->kv_heads, piece_floats = (int64_t)p->q_rows * p->heads * (p->head_dim + 2);
  const int64_t most = std::max<int64_t>(std::min<int64_t>(kMaxPieces, (1 << 26) / std::max<int64_t>(piece_floats, 1)), 1);
  // some two workgroups per CU of caches that are half full, or, where the sequences alone are as many, small pieces that even them out: us in pieces of
  // 128 / 256 / 512 / 768 keys, 16 tokens with caches of up to 4,096 keys of 8 heads 18.8 / 15.0 / 14.1 / 16.0; 14 with 1,078 of 4 11.3 / 12.0 / 13.6 /
  // 15.4; 68 with 1,241 of 8 in pieces of 384 31.8, of 768 35.8
  const int64_t share = (int64_t)p->sequences * p->kv_heads <= 512 ? 1024 : 2048;
  const int64_t keys = (std::max({all / share, (int64_t)1, (max_k + most - 1) / most}) + 127) / 128 * 128;
  f.pieces = (int)((max_k + keys - 1) / keys);
  f.piece_keys = (int)keys;
  f.floats = f.pieces > 1 ? f.pieces * piece_floats : 0;
  return f;
}

template <int HD, int DC, bool PADDED>
int launch(hipStream_t st, const PackedArgs& a, int kind, int64_t grid) {
  using H = FwdShape<HD, 2>;
  using F = FwdShape<HD, 1>;
  if (kind == kFew) MDATTN_LAUNCH((packed_few_kernel<HD, DC, PADDED>), dim3((unsigned)grid), dim3(256), few_bytes<HD>(), st, a);
  else if (kind == kHalf) MDATTN_LAUNCH((packed_fwd_kernel<HD, DC, PADDED, 2>), dim3((unsigned)grid), dim3(256), H::SLOTS * H::Slot, st, a);
  else MDATTN_LAUNCH((packed_fwd_kernel<HD, DC, PADDED, 1>), dim3((unsigned)grid), dim3(256), F::SLOTS * F::Slot, st, a);
  return launch_status();
}

}  // namespace
}  // namespace mdattn

using namespace mdattn;

extern "C" int64_t mdattn_fwd_bf16_packed_workspace_floats(const mdattn_packed* p) {
  return packed_sizes(p) == MDATTN_OK ? fwd_plan(p).floats : 0;
}

extern "C" int mdattn_host_packed_fwd_plan(const mdattn_packed* p, mdattn_host_packed_plan* plan) {
  const int rc = packed_sizes(p);
  if (rc != MDATTN_OK) return rc;
  const FwdPlan f = fwd_plan(p);
  *plan = {f.kind == kFew ? 4 : f.kind == kHalf ? 2 : 1, f.order(p), f.pieces, f.piece_keys, f.items(p)};
  return MDATTN_OK;
}

extern "C" int mdattn_fwd_bf16_packed(void* stream, const mdattn_packed* p, const void* q, const void* k, const void* v, void* out, void* rest,
                                      float* lse, const mdattn_strides* q_strides, const mdattn_strides* k_strides, const mdattn_strides* v_strides,
                                      const mdattn_strides* o_strides, float scale, float* workspace, int64_t workspace_floats) {
  const int rc = packed_sizes(p);
  if (rc != MDATTN_OK) return rc;
  if (!(scale > 0.f) || !(scale < INFINITY) || !q_strides || !k_strides || !v_strides || !o_strides) return MDATTN_E_BADARG;
  if (p->q_rows == 0) return MDATTN_OK;  // nothing to be written
  if (!q || !out || (p->k_rows && (!k || !v))) return MDATTN_E_BADARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(rest) || !packed_aligned(p) || (reinterpret_cast<uintptr_t>(lse) & 3) ||
      !packed_strides_ok(q_strides) || !packed_strides_ok(k_strides) || !packed_strides_ok(v_strides) || !packed_strides_ok(o_strides))
    return MDATTN_E_ALIGN;
  FwdPlan f = fwd_plan(p);
  if (f.pieces > 1 && (!workspace || workspace_floats < f.floats)) {
    f.pieces = 1;
    f.piece_keys = 1 << 30;
  } else if (f.pieces > 1 && !aligned16(workspace)) {
    return MDATTN_E_ALIGN;
  }
  PackedArgs a{};
  a.q = static_cast<const __bf16*>(q); a.k = static_cast<const __bf16*>(k); a.v = static_cast<const __bf16*>(v);
  a.out = static_cast<__bf16*>(out); a.rest = static_cast<__bf16*>(rest); a.lse = lse;
  a.seqs = {p->q_offsets, p->k_offsets, p->k_lengths, p->sequences, p->q_rows, p->k_rows, f.order(p), 256 / p->kv_heads};
  a.group = divisor((unsigned)(p->heads / p->kv_heads));
  a.kv_heads = p->kv_heads; a.D = p->head_dim; a.causal = p->causal;
  a.qs = {q_strides->seq, q_strides->head}; a.ks = {k_strides->seq, k_strides->head};
  a.vs = {v_strides->seq, v_strides->head}; a.os = {o_strides->seq, o_strides->head};
  a.c = scale * kLog2e;
  a.pieces = f.pieces; a.piece_keys = f.piece_keys;
  const int64_t rows = (int64_t)p->q_rows * p->heads;
  if (f.pieces > 1) {
    a.part = workspace;
    a.ml = reinterpret_cast<float2*>(workspace + f.pieces * rows * a.D);
  }
  int64_t grid = f.items(p);
  if (f.kind == kFew) {  // two per CU, in whole rounds of the heads, walk what there is
    a.items = (int)grid;
    grid = std::min(grid, (512 + (int64_t)a.kv_heads - 1) / a.kv_heads * a.kv_heads);
  }
  if (!grid_fits(grid, 256) || (f.pieces > 1 && !grid_fits(rows, 256))) return MDATTN_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  // head dims in whole steps of the products' inner axis where it is the larger part: 80 run as 96, 8 x 1,024 tokens of 16 heads, 64.3 us for 62.9
  // (backward 200 for 193)
  const int status = a.D == 64   ? launch<64, 64, false>(st, a, f.kind, grid)
                     : a.D < 64  ? launch<64, 64, true>(st, a, f.kind, grid)
                     : a.D <= 80 ? launch<128, 80, true>(st, a, f.kind, grid)
                     : a.D <= 96 ? launch<128, 96, true>(st, a, f.kind, grid)
                     : a.D < 128 ? launch<128, 128, true>(st, a, f.kind, grid)
                                 : launch<128, 128, false>(st, a, f.kind, grid);
  if (status != MDATTN_OK || f.pieces == 1) return status;
  MDATTN_LAUNCH(packed_combine_kernel, dim3((unsigned)rows), dim3(256), 0, st, a);
  return launch_status();
}

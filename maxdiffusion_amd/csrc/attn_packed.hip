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
// NK: 1: four waves with 32 rows each.  4: four waves that share 32 rows and deal the keys among them, joined through LDS: for one or a few
// tokens, where the time is that of the keys' way from memory.
// With few rows the keys are cut into pieces besides; each leaves un-normalised f32 rows, joined by a second kernel in a fixed order.
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

template <int HD, int NK>
struct FwdShape {
  static constexpr int NB = HD == 64 && NK == 1 ? 2 : 1;        // blocks of 32 keys that a wave computes per slot
  static constexpr int SLOTS = HD == 128 ? (NK == 1 ? 3 : 2) : (NK == 1 ? 2 : 3);
  static constexpr int Blocks = NB * NK, Keys = 32 * Blocks;    // of a slot
  static constexpr int Half = Blocks * PackedBlock<HD>::Bytes, Slot = 2 * Half;
  static constexpr int BM = NK == 1 ? 128 : 32;
};

template <int HD, int DC, bool PADDED, int NK>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NK == 4 ? 1 : HD == 64 ? 4 : 3, NK == 4 ? 2 : HD == 64 ? 4 : 3)))
void packed_fwd_kernel(PackedArgs a) {
  using T = PackedBlock<HD>;
  using F = FwdShape<HD, NK>;
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
  const int tile = s.tiles - 1 - s.tile;  // (causal: the longest first)
  const int rows = s.m * G, r0 = tile * F::BM + (NK == 1 ? wave * 32 : 0);
  const bool split = a.part != nullptr;
  auto token_of = [&](int r) __attribute__((always_inline)) { return (int)div_by((unsigned)r, a.group); };

  if (s.gap) {  // rows of no sequence
    if (blockIdx.y) return;
    for (int i = tid; i < F::BM * (HD / 8); i += 256) {
      const int r = tile * F::BM + i / (HD / 8), col = i % (HD / 8) * 8;
      if (r >= rows) continue;
      const int t = token_of(r), h = head * G + r - t * G;
      if (col < a.D) *reinterpret_cast<uint4*>(a.out + (s.q0 + t) * a.os.row + h * a.os.head + col) = make_uint4(0u, 0u, 0u, 0u);
      if (col == 0 && a.lse) a.lse[(int64_t)h * a.seqs.q_rows + s.q0 + t] = -INFINITY;
    }
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
  bf16x8 qf[NJ];
  {
    const __bf16* p = a.q + (int64_t)(s.q0 + token) * a.qs.row + (int64_t)(head * G + r - token * G) * a.qs.head + hh * 8;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      qf[j] = !PADDED || j * 16 + hh * 8 < a.D ? *reinterpret_cast<const bf16x8*>(p + j * 16) : __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
  }

  f32x16 O[ND];
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[db][i] = 0.f;
  const float c = a.c;
  float m = -1e30f, mc = -1e30f * c, l = 0.f;
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
    auto soft = [&](float rf) __attribute__((always_inline)) {
      float sum = 0.f;
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) {
        unsigned pk[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[8 * hb + e], c, -rf));
          const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[8 * hb + e + 1], c, -rf));
          sum = (hb == 0 && e == 0) ? x0 : sum + x0;
          sum += x1;
          pk[e >> 1] = pack2(x0, x1);
          asm volatile("" : "+v"(pk[e >> 1]), "+v"(sum));  // packed as soon as they exist
        }
        P[hb] = __builtin_bit_cast(bf16x8, u32x4{pk[0], pk[1], pk[2], pk[3]});
      }
      return sum;
    };
    float sum = soft(mc);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum <= kRange)) != 0, 0)) {
      float top = S[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, S[i]);
      const float mnew = fmaxf(m, xhalf_max(top));
      float alpha = __builtin_amdgcn_exp2f((m - mnew) * c);
      m = mnew;
      mc = m * c;
      asm volatile("" : "+v"(alpha));  // keeps the rescale inside this rarely taken branch
      l *= alpha;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) O[db][i] *= alpha;
      sum = soft(mc);
    }
    l += sum;
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

#pragma unroll
  for (int t = 0; t < SLOTS - 1; ++t)
    if (t < nt) request(t, t);
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
      const int i = NK == 1 ? b : wave * NB + b, k0 = t * F::Keys + 32 * i;
      if (k0 < some) block(at + (unsigned)(i * T::Bytes), k0);
    }
    slot = slot == SLOTS - 1 ? 0 : slot + 1;
    fill = fill == SLOTS - 1 ? 0 : fill + 1;
  }
  __syncthreads();  // every wave has finished reading the ring, and no load into it is in flight: it now stages the output
  l = xhalf_sum(l);

  const int64_t part_row = ((int64_t)piece * a.kv_heads + head) * group_rows + (int64_t)s.q0 * G;  // of the sequence's first row
  if constexpr (NK == 1) {
    if (split) {
      if (r0 + l32 < rows) {
        if (hh == 0) a.ml[part_row + r0 + l32] = make_float2(mc, l);
        if (nt > 0) {
          float* p = a.part + (part_row + r0 + l32) * a.D + 4 * hh;
#pragma unroll
          for (int db = 0; db < ND; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
              if (!PADDED || db * 32 + 8 * g < a.D)
                *reinterpret_cast<f32x4*>(p + db * 32 + 8 * g) = f32x4{O[db][4 * g], O[db][4 * g + 1], O[db][4 * g + 2], O[db][4 * g + 3]};
        }
      }
      return;
    }
    // rows that see no key give 0 and -inf; a sum that is not a number stays one
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    if (a.lse && hh == 0 && r0 + l32 < rows)
      a.lse[(int64_t)(head * G + r - token * G) * a.seqs.q_rows + s.q0 + token] = l == 0.f ? -INFINITY : (mc + __log2f(l)) * kLn2;
    constexpr int RowB = ND * 64 + 16, LPR = ND == 3 ? 16 : ND * 4, RPI = 64 / LPR;  // a staged row; lanes per row, rows per store
    static_assert(4 * 32 * RowB <= SLOTS * F::Slot, "the staged rows fit the ring");
    char* stage = smem + wave * 32 * RowB;
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
      const int t = token_of(row);
      st_nt(reinterpret_cast<uint4*>(a.out + (int64_t)(s.q0 + t) * a.os.row + (int64_t)(head * G + row - t * G) * a.os.head + cc * 8),
            *reinterpret_cast<const uint4*>(stage + (j * RPI + rr) * RowB + cc * 16));
    }
  } else {
    // the four waves' shares brought to one reference point
    constexpr int Ld = ND * 32 + 4;  // floats of a staged row
    static_assert((4 * 32 * Ld + 4 * 32 * 2) * 4 <= SLOTS * F::Slot, "the staged rows fit the ring");
    float* stage = reinterpret_cast<float*>(smem);
    float2* ml = reinterpret_cast<float2*>(stage + 4 * 32 * Ld);
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(stage + (wave * 32 + l32) * Ld + db * 32 + 8 * g + 4 * hh) =
            f32x4{O[db][4 * g], O[db][4 * g + 1], O[db][4 * g + 2], O[db][4 * g + 3]};
    if (hh == 0) ml[wave * 32 + l32] = make_float2(mc, l);
    __syncthreads();
    constexpr int CPR = ND * 4;  // chunks of 8 columns of a row
    for (int i = tid; i < 32 * CPR; i += 256) {
      const int lr = i / CPR, cc = i % CPR * 8, row = r0 + lr;
      if (row >= rows || cc >= (PADDED ? a.D : DC)) continue;
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
      if (split) {
        if (cc == 0) a.ml[part_row + row] = make_float2(top, sum);
        if (nt > 0) {
          f32x4* p = reinterpret_cast<f32x4*>(a.part + (part_row + row) * a.D + cc);
          p[0] = f32x4{f[0], f[1], f[2], f[3]};
          p[1] = f32x4{f[4], f[5], f[6], f[7]};
        }
        continue;
      }
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= inv;
      const int t = token_of(row), h = head * G + row - t * G;
      *reinterpret_cast<uint4*>(a.out + (int64_t)(s.q0 + t) * a.os.row + h * a.os.head + cc) = pack8(f);
      if (cc == 0 && a.lse) a.lse[(int64_t)h * a.seqs.q_rows + s.q0 + t] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
    }
  }
}

// The pieces of the keys joined, in their order: one 16-byte store per lane.
__global__ __launch_bounds__(256) void packed_combine_kernel(PackedArgs a, int cpr, int64_t chunks) {  // cpr: chunks of 8 columns per row
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= chunks) return;
  const int64_t row = i / cpr, group_rows = (int64_t)a.seqs.q_rows * a.group.d, rows = group_rows * a.kv_heads;
  const int cc = (int)(i - row * cpr) * 8;
  const int head = (int)(row / group_rows);
  const unsigned rg = (unsigned)(row - head * group_rows), t = div_by(rg, a.group), h = head * a.group.d + rg - t * a.group.d;
  if ((int)t < a.seqs.q_off[0] || (int)t >= a.seqs.q_off[a.seqs.count]) return;  // rows of no sequence: zeros already
  float top = -INFINITY, sum = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < a.pieces; ++p) {
    const float2 u = a.ml[p * rows + row];
    if (u.y != 0.f) top = fmaxf(top, u.x);
  }
  for (int p = 0; p < a.pieces; ++p) {
    const float2 u = a.ml[p * rows + row];
    if (u.y == 0.f) continue;
    const float x = __builtin_amdgcn_exp2f(u.x - top);
    const f32x4* o = reinterpret_cast<const f32x4*>(a.part + (p * rows + row) * a.D + cc);
    const f32x4 o0 = o[0], o1 = o[1];
    sum += x * u.y;
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] += x * o0[e]; f[4 + e] += x * o1[e]; }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] *= inv;
  *reinterpret_cast<uint4*>(a.out + (int64_t)t * a.os.row + (int64_t)h * a.os.head + cc) = pack8(f);
  if (cc == 0 && a.lse) a.lse[(int64_t)h * a.seqs.q_rows + t] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
}

// How a call is launched.
struct FwdPlan {
  int nk, pieces, piece_keys;
  int64_t floats;
};
FwdPlan fwd_plan(const mdattn_packed* p) {
  const int64_t group = p->heads / p->kv_heads;
  const int64_t max_q = p->max_q > 0 && p->max_q < p->q_rows ? p->max_q : p->q_rows, max_k = p->max_k > 0 && p->max_k < p->k_rows ? p->max_k : p->k_rows;
  FwdPlan f{max_q * group <= 32 ? 4 : 1, 1, 1 << 30, 0};
  const int bm = f.nk == 4 ? 32 : 128;
  // tiles that there are: of the tokens, or of so many sequences of the longest one's
  int64_t tiles = (max_q * group + bm - 1) / bm * p->sequences;
  const int64_t most = p->q_rows * group / bm + p->sequences;
  tiles = (tiles < most ? tiles : most) * p->kv_heads;
  const int64_t want = f.nk == 4 ? 1024 : 512, least = f.nk == 4 ? 256 : 512;
  if (tiles <= 0 || tiles >= want / 2 || max_k < 2 * least) return f;
  int64_t pieces = want / tiles;
  if (pieces > max_k / least) pieces = max_k / least;
  if (pieces > 64) pieces = 64;
  if (pieces < 2) return f;
  f.piece_keys = (int)(((max_k + pieces - 1) / pieces + 127) / 128 * 128);
  f.pieces = (int)((max_k + f.piece_keys - 1) / f.piece_keys);
  f.floats = f.pieces * (int64_t)p->q_rows * p->heads * (p->head_dim + 2);
  return f;
}

template <int HD, int DC, bool PADDED, int NK>
int launch(hipStream_t st, const PackedArgs& a, int64_t grid) {
  constexpr int bytes = FwdShape<HD, NK>::SLOTS * FwdShape<HD, NK>::Slot;
  const auto kernel = packed_fwd_kernel<HD, DC, PADDED, NK>;
  if constexpr (bytes > 65536) {
    static LdsOptIn opted;
    if (lds_opt_in(opted, reinterpret_cast<const void*>(kernel), bytes) != MDATTN_OK) return MDATTN_E_LAUNCH;
  }
  MDATTN_LAUNCH(kernel, dim3((unsigned)grid, (unsigned)a.pieces), dim3(256), bytes, st, a);
  return launch_status();
}
template <int NK>
int launch_nk(hipStream_t st, const PackedArgs& a, int64_t grid) {
  if (a.D == 64) return launch<64, 64, false, NK>(st, a, grid);
  if (a.D < 64) return launch<64, 64, true, NK>(st, a, grid);
  if (a.D <= 96) return launch<128, 96, true, NK>(st, a, grid);
  if (a.D < 128) return launch<128, 128, true, NK>(st, a, grid);
  return launch<128, 128, false, NK>(st, a, grid);
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
  if (f.pieces > 1 && (!workspace || workspace_floats < f.floats)) {
    f.pieces = 1;
    f.piece_keys = 1 << 30;
  } else if (f.pieces > 1 && !aligned16(workspace)) {
    return MDATTN_E_ALIGN;
  }
  PackedArgs a{};
  a.q = static_cast<const __bf16*>(q); a.k = static_cast<const __bf16*>(k); a.v = static_cast<const __bf16*>(v);
  a.out = static_cast<__bf16*>(out); a.lse = lse;
  a.seqs = {p->q_offsets, p->k_offsets, p->k_lengths, p->sequences, p->q_rows, p->k_rows};
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
  const int64_t grid = packed_tiles(group_rows, p->sequences, f.nk == 4 ? 32 : 128) * p->kv_heads, chunks = rows * (a.D / 8);
  if (!grid_fits(grid, 256) || (f.pieces > 1 && !grid_fits((chunks + 255) / 256, 256))) return MDATTN_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const int status = f.nk == 4 ? launch_nk<4>(st, a, grid) : launch_nk<1>(st, a, grid);
  if (status != MDATTN_OK || f.pieces == 1) return status;
  MDATTN_LAUNCH(packed_combine_kernel, dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, st, a, a.D / 8, chunks);
  return launch_status();
}

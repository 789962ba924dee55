// What the kernels of attention over packed sequences share: which sequence a workgroup works on, the tiles in LDS, rows of q by group.
#pragma once
#include "mdattn_common.h"
#include "mdpacked.h"

namespace mdattn {

// Division of a row number (below 2^31) by the heads of a group: n / d = n * (2^(31 + l) / d rounded up) >> (31 + l) with 2^l >= d.
struct Divisor {
  unsigned d, mul, shift;
};
inline Divisor divisor(unsigned d) {
  unsigned l = 0;
  while ((1u << l) < d) ++l;
  return {d, (unsigned)((1ull << (31 + l)) / d + 1), l};
}
__device__ __forceinline__ unsigned div_by(unsigned n, const Divisor& d) { return d.d == 1 ? n : __umulhi(n, d.mul) >> (d.shift - 1); }

struct PackedSeqs {
  const int *q_off, *k_off, *k_len;
  int count, q_rows, k_rows;
  int order, half;  // see find_tile
};
enum { kAsTheyCome, kCausal, kByLength };

// A workgroup's tile of a sequence: rows q0 .. q0 + m of q, k0 .. k0 + n of k and v.  Gap: rows of no sequence (m of q, or n of k), to be
// filled with zeros.
struct SeqTile {
  int q0, m, k0, n, tile, tiles;
  bool gap, none;
};

__device__ __forceinline__ int wave_prefix_sum(int x) {  // inclusive, over the 64 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);   // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);   // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);   // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

// Lane i's sequence, of those from i0 on: its rows (of q, and of k) and its tiles of BM rows (KEYS: of k; else of q, `group` rows for each of its
// tokens).  The rows in front of the first sequence and behind the last follow as two more.  Offsets that decrease, or that point outside, are
// brought into the tensors.
template <int BM, bool KEYS>
__device__ __forceinline__ int lane_sequence(const PackedSeqs& s, int group, int i0, int lane, int& qa, int& m, int& ka, int& n) {
  const int i = i0 + lane, at = i < s.count ? i : s.count, next = i < s.count ? i + 1 : i == s.count ? 0 : s.count;
  qa = s.q_off[at];
  ka = s.k_off[at];
  int qb = s.q_off[next], kb = s.k_off[next];
  const int len = s.k_len && i < s.count ? s.k_len[i] : 0x7FFFFFFF;
  if (i == s.count) qa = ka = 0;                           // in front of the first
  if (i == s.count + 1) { qb = s.q_rows; kb = s.k_rows; }  // behind the last
  qa = min(max(qa, 0), s.q_rows);
  ka = min(max(ka, 0), s.k_rows);
  m = min(max(qb, qa), s.q_rows) - qa;
  n = min(min(max(kb, ka), s.k_rows) - ka, max(len, 0));
  return i < s.count + 2 ? (int)(((unsigned)(KEYS ? n : m * group) + (BM - 1)) / BM) : 0;
}

// Moves i0, and `before`, the tiles in front of it, over the groups of 64 sequences whose tiles all lie in front of `rank`.  The four waves of the workgroup
// take turns at the groups, up to AT_ONCE of them at a time: looked through by each for itself they cost a wave 140 cycles each (4,096 sequences of 20
// tokens, 32 heads on 8: 1,137 -> 583 us; one token each, 1,010 -> 392).  tiles_of(i0): a lane's tiles of a group.
template <int AT_ONCE, class TilesOf>
__device__ __forceinline__ void skip_groups(const PackedSeqs& s, int rank, int lane, int& i0, int& before, TilesOf tiles_of) {
  __shared__ int totals[64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  while (i0 + 64 < s.count + 2) {
    const int groups = min((s.count + 2 - i0 + 63) / 64, AT_ONCE);
    __syncthreads();  // an earlier search has read its totals
    constexpr int Each = AT_ONCE < 16 ? AT_ONCE / 4 : 4;  // groups whose loads are on their way together
    for (int g0 = wave; g0 < groups; g0 += 4 * Each) {
      int n[Each];
#pragma unroll
      for (int u = 0; u < Each; ++u) n[u] = tiles_of(i0 + 64 * (g0 + 4 * u));  // (none behind the last)
#pragma unroll
      for (int u = 0; u < Each; ++u) {
        const int total = __builtin_amdgcn_readlane(wave_prefix_sum(n[u]), 63);
        if (lane == 0) totals[g0 + 4 * u] = total;
      }
    }
    __syncthreads();
    const int n = lane < groups ? totals[lane] : 0, upto = wave_prefix_sum(n);
    const uint64_t found = __builtin_amdgcn_ballot_w64(before + upto > rank);
    if (found) {
      const int j = __builtin_ctzll(found);
      before += __builtin_amdgcn_readlane(upto, j) - __builtin_amdgcn_readlane(n, j);
      i0 += 64 * j;
      return;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    i0 += 64 * groups;
  }
}

// Tile `rank` of all sequences' tiles.  Sequences are looked through in their order, each one's last tile first, the last 64 by every wave for itself.  With an
// order (of up to 62 sequences; see packed_order) the tiles go by what they meet, the most first: of a causal batch by their number, over all
// sequences, of others by their sequence's length on the other side.  The second `half` of them, which share their CUs with the first, from
// the other end.
template <int BM, bool KEYS>
__device__ __forceinline__ SeqTile find_tile(const PackedSeqs& s, int group, int rank, int lane) {
  SeqTile t{};
  int before = 0, i0 = 0;
  auto tiles_of = [&](int i0) __attribute__((always_inline)) {
    int qa, m, ka, n;
    return lane_sequence<BM, KEYS>(s, group, i0, lane, qa, m, ka, n);
  };
  skip_groups<64>(s, rank, lane, i0, before, tiles_of);
  for (; i0 < s.count + 2; i0 += 64) {
    int qa, m, ka, n;
    const int tiles = lane_sequence<BM, KEYS>(s, group, i0, lane, qa, m, ka, n);
    const int upto = wave_prefix_sum(tiles), total = __builtin_amdgcn_readlane(upto, 63);
    if (rank - before >= total) {
      before += total;
      continue;
    }
    int j;
    if (s.order == kAsTheyCome) {
      j = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + upto > rank));
      t.tile = before + __builtin_amdgcn_readlane(upto, j) - 1 - rank;
    } else {
      if (rank >= s.half && total <= 2 * s.half) rank = total - 1 - (rank - s.half);
      // the tiles above a level: of each sequence those with a higher number, or all of them where its other side is longer
      const bool causal = s.order == kCausal;
      const int other = KEYS ? m : n;
      auto above = [&](int level) __attribute__((always_inline)) { return causal ? max(tiles - level, 0) : other > level ? tiles : 0; };
      // the highest level that, with what is above it, has more than `rank` tiles
      int lo = -1, hi = causal ? (int)(((unsigned)(KEYS ? s.k_rows : s.q_rows * group)) / BM) + 1 : KEYS ? s.q_rows : s.k_rows;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__builtin_amdgcn_readlane(wave_prefix_sum(above(mid)), 63) > rank) lo = mid;
        else hi = mid;
      }
      // of level lo, the tiles between those above it and those above hi
      const int here = above(lo) - above(hi), sum = wave_prefix_sum(here);
      const int at = rank - __builtin_amdgcn_readlane(wave_prefix_sum(above(hi)), 63);
      j = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > at));
      t.tile = causal ? lo : __builtin_amdgcn_readlane(sum, j) - 1 - at;
    }
    t.q0 = __builtin_amdgcn_readlane(qa, j);
    t.m = __builtin_amdgcn_readlane(m, j);
    t.k0 = __builtin_amdgcn_readlane(ka, j);
    t.n = __builtin_amdgcn_readlane(n, j);
    t.gap = i0 + j >= s.count;
    t.tiles = __builtin_amdgcn_readlane(tiles, j);
    return t;
  }
  t.none = true;
  return t;
}

// Item `rank` of all sequences' tiles of 32 rows with each of its pieces of piece_keys keys (up to `pieces`, the last of which takes the rest; one,
// where there are no keys).  i0 and before: where the search for an earlier item ended, zeros at first.
__device__ __forceinline__ SeqTile find_piece(const PackedSeqs& s, int group, int rank, int lane, int piece_keys, int pieces, int& i0, int& before, int& piece) {
  SeqTile t{};
  auto pieces_of = [&](int i, int n) __attribute__((always_inline)) {
    return i < s.count ? max(min((int)(((unsigned)n + (unsigned)(piece_keys - 1)) / (unsigned)piece_keys), pieces), 1) : 1;
  };
  auto items_of = [&](int i0) __attribute__((always_inline)) {
    int qa, m, ka, n;
    const int tiles = lane_sequence<32, false>(s, group, i0, lane, qa, m, ka, n);
    return pieces == 1 ? tiles : tiles * pieces_of(i0 + lane, n);
  };
  skip_groups<8>(s, rank, lane, i0, before, items_of);
  for (; i0 < s.count + 2; i0 += 64) {
    int qa, m, ka, n;
    const int tiles = lane_sequence<32, false>(s, group, i0, lane, qa, m, ka, n);
    const int each = pieces_of(i0 + lane, n);
    const int upto = wave_prefix_sum(tiles * each), total = __builtin_amdgcn_readlane(upto, 63);
    if (rank - before >= total) {
      before += total;
      continue;
    }
    const int j = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + upto > rank)), per = __builtin_amdgcn_readlane(each, j);
    t.tiles = __builtin_amdgcn_readlane(tiles, j);
    const int at = rank - before - (__builtin_amdgcn_readlane(upto, j) - t.tiles * per);
    t.tile = at / per;
    piece = at - t.tile * per;
    t.q0 = __builtin_amdgcn_readlane(qa, j);
    t.m = __builtin_amdgcn_readlane(m, j);
    t.k0 = __builtin_amdgcn_readlane(ka, j);
    t.n = __builtin_amdgcn_readlane(n, j);
    t.gap = i0 + j >= s.count;
    return t;
  }
  t.none = true;
  return t;
}

// A block of 32 rows of HD elements in LDS, filled by loads of 1 KB: chunk c (16 bytes) of row r sits at position c ^ swizzle(r).  The
// upper part of the swizzle, distinct within 4 rows that follow each other, moves the 64-byte segment, so that the transposing reads
// (4 rows x 64 bytes) cover every bank once; the lower part makes all positions of 16 rows distinct, for the row reads.
template <int HD>
struct PackedBlock {
  static constexpr int RPI = HD == 128 ? 4 : 8;  // rows that one load instruction fills
  static constexpr int Row = HD * 2, Bytes = 32 * Row;
  static __device__ __forceinline__ int swizzle(int r) { return HD == 128 ? 4 * (r & 3) + ((r >> 2) & 3) : 4 * ((r >> 1) & 1) + ((r >> 2) & 3); }
  // the row of its group, and the chunk, that a lane of group g's load brings
  static __device__ __forceinline__ int row(int lane) { return HD == 128 ? lane >> 4 : lane >> 3; }
  static __device__ __forceinline__ int chunk(int lane, int g) { return (lane & (HD / 8 - 1)) ^ swizzle(RPI * g + row(lane)); }
  // where a lane's part of a fragment sits: row read j (chunk 2 j + hh of row l32) at row_at ^ 32 j; transposing read of the 32-column slab sg
  // at trans_at ^ 64 sg for the rows 4 hh + 0..3 and, eight rows on, at that ^ 32
  static __device__ __forceinline__ unsigned row_at(int lane) {
    const int l32 = lane & 31, hh = lane >> 5;
    return (unsigned)(l32 * Row + ((hh ^ swizzle(l32)) * 16));
  }
  static __device__ __forceinline__ unsigned trans_at(int lane) {
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2);
    return (unsigned)(r * Row + ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swizzle(r)) * 16 + (lane & 1) * 8);
  }
};

typedef s16x4 __attribute__((address_space(3))) * lds_s16x4_at;
typedef __attribute__((ext_vector_type(8))) short s16x8_p;
typedef const bf16x8 __attribute__((address_space(3))) * lds_bf16x8_at;
typedef const f32x4 __attribute__((address_space(3))) * lds_f32x4_at;
__device__ __forceinline__ bf16x8 read_row_frag(unsigned at) { return *(lds_bf16x8_at)at; }
__device__ __forceinline__ bf16x8 read_trans_frag(unsigned at0, unsigned at1) {
  const s16x4 r0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_at)at0);
  const s16x4 r1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_at)at1);
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(r0, r1, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Strides of a tensor [rows, heads, head_dim] in elements.
struct RowStrides {
  int64_t row, head;
};

// A few rows' strides are added up in 32 bits; heads' are not.  group: heads of q and out in the backward pass, whose strides the interface limits in
// sum (no count in the kernels needs it).
inline bool packed_strides_ok(const mdattn_strides* s, int64_t group = 0) {
  return s && s->seq % 8 == 0 && s->head % 8 == 0 && s->seq >= 0 && s->head >= 0 && s->seq < (1 << 23) && s->head < (1ll << 40) &&
         group * s->head < (1 << 29);
}
// MDATTN_OK for sizes that the kernels take
inline int packed_sizes(const mdattn_packed* p) {
  if (!p || !p->q_offsets || !p->k_offsets || p->sequences < 0 || p->q_rows < 0 || p->k_rows < 0 || p->heads <= 0 || p->kv_heads <= 0 ||
      p->heads % p->kv_heads || p->head_dim <= 0)
    return MDATTN_E_BADARG;
  if (p->head_dim % 8 || p->head_dim > 128) return MDATTN_E_UNSUPPORTED;
  const int64_t group = p->heads / p->kv_heads;
  // row numbers of a head's group, and the rows of all heads, are counted in 31 bits
  if (group > 1024 || p->sequences > (1 << 24) || (int64_t)p->q_rows * p->heads >= (1ll << 31) - 4096 ||
      (int64_t)p->k_rows * p->kv_heads >= (1ll << 31) - 4096)
    return MDATTN_E_UNSUPPORTED;
  return MDATTN_OK;
}
inline bool packed_aligned(const mdattn_packed* p) {
  return ((reinterpret_cast<uintptr_t>(p->q_offsets) | reinterpret_cast<uintptr_t>(p->k_offsets) | reinterpret_cast<uintptr_t>(p->k_lengths)) & 3) == 0;
}
// Whether the tiles of a call go by what they meet: where they do not all have a CU of their own, what starts last should be short, and what shares a CU
// with a long one too.  The search for a tile costs some 0.5 us.
inline int packed_order(const mdattn_packed* p, int64_t tiles) {
  return p->sequences == 0 || p->sequences > 62 || tiles <= 256 || (p->sequences == 1 && !p->causal) ? kAsTheyCome : p->causal ? kCausal : kByLength;
}
// tiles of BM rows that all sequences of `rows` rows have together at most, and the two gaps
inline int64_t packed_tiles(int64_t rows, int64_t sequences, int BM) { return rows / BM + sequences + 2; }

}  // namespace mdattn

// Prefill kernels of the full attention, varlen and paged, on 32x32x16 MFMA
// tiles, and their launches.
//
// S^T = K Q^T, so that lane l of a wave owns query column l % 32 of the
// accumulator.  The softmax statistics of a query then live in one lane pair
// (l, l ^ 32), and the exponentiated accumulator registers are already the B
// operand of O^T = V^T P^T, whose A operand is read from the row-major V tile
// with ds_read_b64_tr_b16.  The running maximum is re-based only when a new
// tile raises it by more than 2^8 (in exp2 units); O and the row sum always
// share the same base, so the result is the same softmax.
#pragma once

#include <algorithm>

#include <type_traits>

#include "attention_own.h"
#include "fp4.h"

namespace {

struct AttnArgs {
  const void* q;
  int64_t q_st, q_sh;  // element strides: token, head
  KvSource k, v;
  void* o;
  int64_t o_st, o_sh;
  const void* cu;
  const void* ctx;
  PagedTable tab;
  int64_t T, nseq;
  int32_t Hq, Hkv, gh;  // gh: query heads per workgroup (1, 2 or 4)
  int32_t dim;          // head dim (a multiple of 8, at most the kernel's D)
  float c;              // softmax scale * log2(e)
  bool cu64, ctx64, causal;
  // split prefill: (tile, head group) rows of the grid, workgroups for the
  // rows' further pieces, and the pieces' partials (rows + extra slots)
  int64_t rows;
  int32_t extra;
  float* part;
  // kScored: 2 / cap of the tanh cap and 2 cap log2(e) (0: none), slopes of
  // the distance bias (Hq,), and keys of each sequence that all its queries see
  float cap_in, cap_out;
  const float* slopes;
  const void* pfx;
  bool pfx64;
};

// kShared: the shared keys' workgroups, and the decode of the sequences' own
// keys, which takes the grid's first own_wgs workgroups (a multiple of 8)
struct SharedAttnArgs : AttnArgs {
  const SharedWork* work;
  DecodeArgs own;
  uint32_t own_wgs;
};

// kFp4: block scales of the caches' codes
struct Fp4AttnArgs : AttnArgs {
  ScaleSource ks, vs;
};

// Floats of one piece's partial: per wave, the accumulators of its 32 queries
// in register order (lane-contiguous 16-byte pieces), then m and l per lane.
template <int D> constexpr int64_t prefill_part_wave() { return 32 * D + 128; }
template <int D> constexpr int64_t prefill_part_floats() { return 4 * prefill_part_wave<D>(); }

// Element offset in a query row of `dim` dims of the 8 that lane half hh reads
// for k-step s; a piece past the row reads the row's first (its value is
// dropped), so that no lane reads outside the row (dims of 8 have one piece).
__host__ __device__ constexpr int q_piece(int s, int hh, int dim) {
  return 16 * s + 8 * hh < dim ? 16 * s + 8 * hh : 0;
}
constexpr bool q_pieces_inside(int dq) {
  for (int dim = 8; dim <= dq; dim += 8)
    for (int p = 0; p < dq / 8; ++p)
      if (q_piece(p / 2, p % 2, dim) + 8 > dim) return false;
  return true;
}

// ---------------------------------------------------------------------------
// Prefill: one workgroup = 4 waves = `gh` query heads of one kv head x
// (4 / gh) blocks of 32 queries.  K and V tiles of BN keys are staged in LDS
// (double buffered, the next tile prefetched into registers) and shared by
// the four waves.
// PG: 0 packed rows, 1 paged (any page size: a table lookup per row),
// 2 / 3 paged with a page size that is a multiple of 16 and an int32 / int64
// block table (one lookup per 16 rows, a tile ahead, 32-bit arithmetic); kFp4 also 4,
// an int32 table, pages of 16 keys, and v's strides those of k, which holds fewer scalar
// registers: four chunks of up to 2,048 tokens over up to 16,384 keys, 16 / 2 heads of
// 256 950 us, by PG 2 1,110 (16-bit caches 1,005); 16 prompts of up to 4,096 785 and 851;
// the four chunks with 16 heads of 64 293 and 343
// Workgroup id -> (sequence, query tile): tiles of tile_len queries (a power
// of two), laid out sequence after sequence over the tiles that exist (no
// workgroup of a padded grid exits idle).  Below D = 256 batches of up to 64
// sequences go longest first (by keys, ties by index), so that what runs last
// is short: every lane ranks one sequence against the others and sums the
// tiles before it, past eight sequences a quarter of them per wave (a wave
// against all 64 took 10 us of a call: 64 x 100 tokens at D = 64 28.8 us, 18.3
// shared, in index order 17.1).  Six images of 450 to 2,900 patches 143 ->
// 137 us, eight causal prompts of 512 to 4,096 tokens 171 -> 159 (D = 64) and
// 259 -> 247 (128), eight chunks over up to 4,096 cached keys 340 -> 331 (128).
// Past the last tile seq is -1 and tile counts from there.
// Larger batches, and D = 256 (sixteen prompts: 974 in index order, 985
// ranked), are taken in index order by a scan over the workgroup.
struct SeqTile {
  int64_t seq, tile;
};
template <int D, bool PAGED, bool SPLIT>
GDN_DEVICE SeqTile attn_tile_lookup(const AttnArgs& a, int tile_len, int64_t target, int32_t* lds) {
  SeqTile r;
  if (D < 256 && a.nseq <= 64) {
    __shared__ int32_t before[4][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sh = __builtin_ctz(tile_len);
    int nt = 0;
    uint32_t key = 0;
    if (lane < a.nseq) {
      int64_t s, e;
      seq_range(a.cu, a.cu64, lane, a.T, s, e);
      nt = (int)((e - s + tile_len - 1) >> sh);
      key = (uint32_t)clamp64(PAGED ? load_index(a.ctx, lane, a.ctx64) : e - s, 0, (1 << 26) - 1);
    }
    key = key << 6 | (63 - lane);  // (unique, so one comparison ranks)
    const bool share = a.nseq > 8;  // each wave against a quarter of the sequences
    int base = 0;
    for (int j = share ? w : 0; j < (int)a.nseq; j += share ? 4 : 1) {
      const uint32_t kj = (uint32_t)__builtin_amdgcn_readlane((int)key, j);
      const int tj = __builtin_amdgcn_readlane(nt, j);
      base += kj > key ? tj : 0;
    }
    if (share) {
      before[w][lane] = base;
      __syncthreads();
      base = before[0][lane] + before[1][lane] + before[2][lane] + before[3][lane];
    }
    const int t = (int)target - base;
    const uint64_t own = __builtin_amdgcn_ballot_w64(t >= 0 && t < nt);
    r.seq = own ? __builtin_ctzll(own) : -1;
    r.tile = own ? __builtin_amdgcn_readlane(t, (int)r.seq)
                 : target - __builtin_amdgcn_readlane(wave_inclusive_scan_i32(nt), 63);
    return r;
  }
  if (SPLIT && a.nseq <= 64) {  // index order without a barrier: split_tiles has just read the same lengths
    const int lane = threadIdx.x & 63;
    int nt = 0;
    if (lane < a.nseq) {
      int64_t s, e;
      seq_range(a.cu, a.cu64, lane, a.T, s, e);
      nt = (int)((e - s + tile_len - 1) >> __builtin_ctz(tile_len));
    }
    const int incl = wave_inclusive_scan_i32(nt), t = (int)target - (incl - nt);
    const uint64_t own = __builtin_amdgcn_ballot_w64(t >= 0 && t < nt);
    r.seq = own ? __builtin_ctzll(own) : -1;
    r.tile = own ? __builtin_amdgcn_readlane(t, (int)r.seq) : target - __builtin_amdgcn_readlane(incl, 63);
    return r;
  }
  find_seq_tile<256>(a.cu, a.cu64, a.nseq, a.T, tile_len, target, r.seq, r.tile, lds);
  return r;
}

// How a split prefill cuts its rows: into pieces of `tiles` key tiles, the same
// for all rows.  A row's first piece has the row's own workgroup; the further
// ones take floor((n - 1) / tiles) of the extra workgroups per query tile and
// head group of a sequence, n the key tiles of its last query (its other rows
// may need fewer: those left over return).  All second pieces come first, then
// all third ones, so that what runs together reads the same stretch of K and V
// and the rows' short ends run last.
// The length follows from the batch's own lengths.  Lane i prices the longest
// row in i + 1 pieces, in key-tile steps of one workgroup (1.18 us at D = 256,
// 1.05 at 128): the batch's work over the workgroups that run at once, with
// kFixed steps per row (lookup, queries, pipeline fill, output) and kPiece per
// further piece (that, and its share of the merge), and part of the length of
// those that start last; a batch that fits one round takes as long as its
// longest workgroup.  Fitted to 30 batches forced into 1 to 16 pieces: what it
// chooses is 1 % off the best on average, 8 % at most.  A split has to win 3 %
// over one piece per row and to fit the extra workgroups.  The prefill and the
// combine kernel both work it out, in whole numbers, so that they agree.
struct SplitSeq {
  int32_t ntile, n;  // query tiles, key tiles of the last one
};
struct SplitPlan {
  int32_t tiles;  // kWholeRows: not split
  SplitSeq q;     // sequence `lane` of the first 64; the others are read again
};
constexpr int kWholeRows = 1 << 26;  // (32 keys times that: past any row)
constexpr int kMaxPieces = 64;
template <int BN>
GDN_DEVICE SplitSeq split_seq(const AttnArgs& a, int64_t seq, int sh) {
  SplitSeq q{0, 0};
  if (seq < a.nseq) {
    int64_t s, e;
    seq_range(a.cu, a.cu64, seq, a.T, s, e);
    const int64_t keys = clamp64(load_index(a.ctx, seq, a.ctx64), 0, a.tab.cols * a.tab.page);
    q.ntile = (int)((e - s + (1 << sh) - 1) >> sh);
    q.n = q.ntile > 0 ? (int)((keys + BN - 1) / BN) : 0;
  }
  return q;
}
template <int BN>
GDN_DEVICE SplitSeq split_seq(const AttnArgs& a, const SplitPlan& sp, int c, int sh) {
  return c == 0 ? sp.q : split_seq<BN>(a, c + (threadIdx.x & 63), sh);
}
// floor((n - 1) / tiles), at most 2^20: the float quotient is within one of it
GDN_DEVICE int split_further(int n, int tiles, float inv) {
  const int last = n > 0 ? n - 1 : 0;
  int u = (int)((float)last * inv);
  u -= u * tiles > last;
  return u + ((u + 1) * tiles <= last);
}
GDN_DEVICE int wave_top(int x) {  // maximum of non-negative numbers, in the steps of wave_inclusive_scan_i32
  auto up = [&](int y) __attribute__((always_inline)) { x = y > x ? y : x; };
  up(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false));
  up(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false));
  up(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false));
  up(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false));
  up(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false));
  up(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(x, 63);
}
GDN_DEVICE int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_inclusive_scan_i32(x), 63); }

template <int D, int BN>
GDN_DEVICE int split_tiles(const AttnArgs& a, const SplitPlan& sp, int sh) {
  constexpr int kSlots = D == 256 ? 256 : D == 128 ? 512 : 768, kSlots16 = kSlots / 16;  // workgroups that run at once
  constexpr int kFixed = 10, kPiece = D == 256 ? 24 : 16;
  const int lane = threadIdx.x & 63, hg = a.Hq / a.gh, nseq = (int)a.nseq;
  // per head group: query tiles R, work W in units of 16 steps, and what one
  // piece per row takes: the longest (last, these run first) query tile of each
  // sequence starts when the sequences before it have been handed out.  Below
  // D = 256 they are ranked (attn_tile_lookup), so the longest starts first and
  // the shortest last.
  int W = 0, R = 0, top = 0, late = 0, low = kWholeRows;
  for (int c = 0; c < nseq; c += 64) {
    const SplitSeq q = split_seq<BN>(a, sp, c, sh);
    // (the query tiles before the last see 2^sh keys less each)
    const int less = ((q.ntile - 1) << (sh - 5)) / (2 * BN / 32), half = (q.n + 1) >> 1;
    const float w16 = (float)q.ntile * (float)(kFixed + (q.n - less > half ? q.n - less : half)) * 0.0625f;
    const int w = w16 < 0x1p22f ? (int)w16 : 1 << 22, incl = wave_inclusive_scan_i32(w);
    const int end = ((W + incl - w) / kSlots16) * hg + q.n;
    late = q.n > 0 && end > late ? end : late;
    low = q.n > 0 && q.n < low ? q.n : low;
    top = q.n > top ? q.n : top;
    W += __builtin_amdgcn_readlane(incl, 63);
    R += wave_sum(q.ntile);
    if ((int64_t)W * hg > (1 << 28) || (int64_t)R * hg > (1 << 20)) return kWholeRows;  // (past the sums below)
  }
  const int nmax = wave_top(top);
  if (nmax <= 16) return kWholeRows;
  const int rows = hg * R, work = hg * W;
  int whole = kFixed + nmax;
  if (rows > kSlots) {
    const int last = D == 256 ? kFixed + wave_top(late < 1 << 24 ? late : 1 << 24)
                              : work / kSlots16 + kWholeRows - wave_top(kWholeRows - low);
    whole = last > whole ? last : whole;
  }
  int tiles = (int)((float)(nmax + lane) * __builtin_amdgcn_rcpf((float)(lane + 1)));
  tiles += tiles * (lane + 1) < nmax;
  tiles += tiles & 1;
  const float inv = __builtin_amdgcn_rcpf((float)tiles);
  int x = 0;
  for (int c = 0; c < nseq; c += 64) {
    const SplitSeq q = split_seq<BN>(a, sp, c, sh);
    const int m = nseq - c < 64 ? nseq - c : 64;
    for (int j = 0; j < m; ++j)
      x += __mul24(__builtin_amdgcn_readlane(q.ntile, j), split_further(__builtin_amdgcn_readlane(q.n, j), tiles, inv));
  }
  x = x < 1 << 16 ? x * hg : 1 << 24;
  const int tail = D == 256 ? tiles / 2 + tiles / 8 : tiles / 2;
  const int split = rows + x <= kSlots ? kFixed + 4 + tiles + (rows + x) / kSlots16
                                       : (work + kPiece * x / 16) / kSlots16 + tail + kFixed;
  int cost = lane == 0 ? whole - whole / 32 : x > 0 && x <= a.extra && tiles >= 8 ? split : 1 << 24;
  cost = cost < 1 << 24 ? cost : 1 << 24;
  // (the smallest, of equals the one with fewer pieces)
  const int best = 63 - (wave_top(((1 << 24) - cost) << 6 | (63 - lane)) & 63);
  return best > 0 ? __builtin_amdgcn_readlane(tiles, best) : kWholeRows;
}

// Further pieces of index p = lane (1, 2, ...; lane 0: 0) per head group, of
// all sequences and of those before `seq`.
struct SplitCount {
  int32_t all, before;
};
template <int BN>
GDN_DEVICE SplitCount split_count(const AttnArgs& a, const SplitPlan& sp, int sh, int seq) {
  const int lane = threadIdx.x & 63, nseq = (int)a.nseq;
  const float inv = __builtin_amdgcn_rcpf((float)sp.tiles);
  SplitCount k{0, 0};
  for (int c = 0; c < nseq; c += 64) {
    const SplitSeq q = split_seq<BN>(a, sp, c, sh);
    const int f = split_further(q.n, sp.tiles, inv), m = nseq - c < 64 ? nseq - c : 64;
    for (int j = 0; j < m; ++j) {
      const int fj = __builtin_amdgcn_readlane(f, j), nt = __builtin_amdgcn_readlane(q.ntile, j);
      const int x = fj >= lane && lane > 0 ? nt : 0;
      k.all += x;
      k.before += c + j < seq ? x : 0;
    }
  }
  return k;
}

// Of extra workgroup group `target` (per head group): its sequence, query tile
// and piece; seq -1 if it is left over.
struct SplitPiece {
  int64_t seq, tile;
  int piece;
};
template <int BN>
GDN_DEVICE SplitPiece split_piece(const AttnArgs& a, const SplitPlan& sp, int sh, int target) {
  const int nseq = (int)a.nseq;
  const int all = split_count<BN>(a, sp, sh, 0).all, incl = wave_inclusive_scan_i32(all), t = target - (incl - all);
  const uint64_t own = __builtin_amdgcn_ballot_w64(t >= 0 && t < all);
  if (own == 0) return {-1, 0, 0};
  const int p = __builtin_ctzll(own);
  int left = __builtin_amdgcn_readlane(t, p);
  const float inv = __builtin_amdgcn_rcpf((float)sp.tiles);
  for (int c = 0; c < nseq; c += 64) {
    const SplitSeq q = split_seq<BN>(a, sp, c, sh);
    const int x = split_further(q.n, sp.tiles, inv) >= p ? q.ntile : 0;
    const int sum = wave_inclusive_scan_i32(x), u = left - (sum - x);
    const uint64_t mine = __builtin_amdgcn_ballot_w64(u >= 0 && u < x);
    if (mine) {
      const int l = __builtin_ctzll(mine);
      return {c + l, __builtin_amdgcn_readlane(u, l), p};
    }
    left -= __builtin_amdgcn_readlane(sum, 63);
  }
  return {-1, 0, 0};
}

// Output rows that no sequence covers -- [0, cu[0]) and [cu[N], T), clamped
// like seq_range -- are zero, as the reference allocates o zero-filled
// (ops/full_attention.py:467).  The workgroups past the last tile, `wg` of `n`,
// share them (a kernel of their own, launched first, took 3 to 5 us of every
// call; the usual batch covers all rows and has nothing to do here).
template <typename T>
GDN_DEVICE void zero_rows_tail(const AttnArgs& a, uint32_t wg, uint32_t n) {
  int64_t first = load_index(a.cu, 0, a.cu64), last = load_index(a.cu, a.nseq, a.cu64);
  first = clamp64(first, 0, a.T);
  last = clamp64(last, first, a.T);
  const int64_t nrows = first + (a.T - last);
  constexpr int per = 16 / (int)sizeof(T);  // elements of a 16-byte piece
  const int64_t vph = a.dim / per, vpr = a.Hq * vph;
  for (int64_t i = (int64_t)wg * 256 + threadIdx.x; i < nrows * vpr; i += (int64_t)n * 256) {
    const int64_t r = i / vpr, rem = i - r * vpr, h = rem / vph, c = (rem - h * vph) * per;
    const int64_t t = r < first ? r : last + (r - first);
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.o) + t * a.o_st + h * a.o_sh + c) = uint4{0, 0, 0, 0};
  }
}

// SPLIT: the key range of every (query tile, head group) row is cut into
// pieces (split_tiles), one workgroup each.  A row of one piece writes its
// output rows; otherwise every piece writes m, l and the unnormalised O to the
// workspace and attn_prefill_combine_kernel merges them.  It serves batches
// whose rows are few or uneven for 256 CUs (one workgroup per CU at D = 256):
// a workgroup runs 1.2 us per key tile, so 1,000 new tokens over a 15,000-key
// prefix are 128 rows of 550 us each.  Measured (16 / 2 heads, D = 256, one
// piece -> split): four prompts of 260 to 1,900 tokens over prefixes of up to
// 15,800 keys 1,188 -> 957 us, one of 512 over 8,000 keys 309 -> 104, over 2,000
// 88 -> 53, five of 18 over 11,700 444 -> 75; the same with tables of 131,072
// keys (pieces cut from the table's width: 187 us at 8,000 keys, and nothing
// split at 2,000).  Where there is nothing to split, the extra workgroups and
// the second launch cost 1 to 6 us: four prompts of 1,000 tokens without a
// prefix 87 -> 93 us (98 with pieces from the width).
//
// Key tiles: 32 keys, which at D = 64 and 128 leave room for two waves per
// SIMD (at least) whose softmax and MFMAs overlap; D = 96 fits two with 64, and
// at D = 64 few workgroups take 64 (few_workgroups).
// At D = 128 tiles of 64 keys took 259 to 280 registers, one wave per SIMD:
// eight prompts of 512 to 4,096 tokens (16 / 4 heads) 363 -> 254 us, with 64
// keys held to 256 registers 259; eight chunks over up to 4,096 cached keys
// 563 -> 329 us (345).  D = 64: 180 -> 165 us.  D = 96 (vision): 64 keys 142,
// 32 keys 157, three waves per SIMD 158 (32 keys) and 197 (64, spills).
template <typename T, int D, int BN, int PG, bool SPLIT, int DQ = 0, AttnForm FORM = kPlain>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) void attn_prefill_kernel(
    const std::conditional_t<FORM == kShared, SharedAttnArgs,
                             std::conditional_t<FORM == kFp4, Fp4AttnArgs, AttnArgs>> a) {
  constexpr bool PAGED = PG != 0;
  // DQ > 0: head dims of a.dim <= DQ <= D elements (packed rows only), a
  // multiple of 8.  The rows are read as they lie and the 16-byte pieces past
  // a.dim become zeros on the way (query pieces by a select, key and value
  // pieces by an offset past the buffer's range), so nothing is padded in
  // memory; the score product runs over DQ dims, P V over D.  Six images of
  // 450 to 2,900 patches, 16 heads of 72: 306 -> 122 us against padded copies
  // at D = 128 (40 us of copies, and the MFMAs and fragment reads of 56 dims).
  constexpr bool RAG = DQ > 0;
  static_assert(!RAG || (PG == 0 && DQ <= D && DQ % 16 == 0), "ragged head dims are packed rows");
  static_assert(!SPLIT || PG >= 2, "split rows are paged rows of whole 16-row groups");
  static_assert(FORM == kPlain || !RAG, "scored and shared rows are of the kernels' own head dims");
  static_assert(FORM != kShared || (PAGED && !SPLIT), "shared keys are paged, in pieces of their own");
  // kFp4: a thread loads the codes of QE numbers of a row and their scale byte, and
  // turns them into 16 bits where the others store their tile to LDS.  So the
  // tiles in flight take a quarter of the registers, and the products are the
  // 16-bit cache's.
  constexpr bool Q4 = FORM == kFp4;
  constexpr int QE = BN * D / 256, QW = QE >= 8 ? QE / 8 : 1, QL8 = D / QE;  // words of codes, threads per row
  static_assert(!Q4 || (PG >= 2 && QE >= 8 && QE <= 32 && 32 % QL8 == 0), "codes of up to one block a thread");
  typedef Mma<T> M;
  typedef typename M::v8 v8;
  typedef typename M::v4 v4;
  constexpr int LDK = D + 8;   // row stride (elements): 16-byte row skew for the b128 reads
  constexpr int LDV = D == 96 ? D : D + 32;  // 64 bytes of row skew modulo the banks for the transposed reads
  constexpr int NKS = (RAG ? DQ : D) / 16;
  constexpr int NA = BN / 32;
  constexpr int NDT = D / 32;
  constexpr int CH = D / 8;  // 16-byte chunks per row
  constexpr int NLD = BN * CH / 256;
  static_assert(BN % 32 == 0 && (BN * CH) % 256 == 0, "tile");
  __shared__ __align__(16) T ks[2][BN * LDK];
  __shared__ __align__(16) T vs[2][BN * LDV];
  // D = 256: each wave's query fragments sit in LDS (16.5 KB per wave)
  // instead of 64 VGPRs; the registers this frees hold the K, Q and V
  // fragments of the next MFMAs while the current one runs (with Q resident
  // the allocator kept one fragment buffer, so every LDS read was waited for
  // right before its MFMA)
  constexpr bool QL = D == 256;
  // of those, the last QRG stay in registers as well (fewer LDS reads in the
  // score phase for 48 more registers; measured: 12 of 16, all 16 much slower)
  constexpr int QRG = QL ? 12 : 0;
  __shared__ __align__(16) T qs[QL ? 4 * 32 * LDK : 8];

  // (the wave index through readfirstlane: the compiler then knows it, and
  // the wave's query block, causal range and tile tests, to be uniform, so
  // they live in scalar registers and branch without exec masks)
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = a.Hq / a.Hkv, gh = a.gh, qsubs = 4 / gh, groups = R / gh;
  // Workgroup order: sequence after sequence, a sequence's query tiles last
  // first, the head groups of a tile innermost.  The dispatcher deals
  // consecutive workgroups to its 32 queues (8 XCDs x 4 shader engines, 8
  // CUs each) in turn, so every sequence spreads over all of them, and a
  // sequence's workgroups run together and share its K/V rows in L2.
  __shared__ int32_t lookup[8];
  // (kFp4) the first key whose value is NaN in each 32 dims: a probability of 0 would
  // not keep it from the queries before it, so its numbers go to LDS as finite ones
  // and the queries that see it get their NaN at the end (16 prompts of 1,024 tokens, 16 / 2 heads
  // of 256 287 -> 294 us, four chunks of 1,500 behind 7,500 keys 978 -> 989; a branch
  // that writes to LDS at once 298 and 994)
  __shared__ uint32_t nan_at[Q4 ? NDT : 1];
  if (Q4 && tid < NDT) nan_at[tid] = UINT32_MAX;
  const int hg = a.Hq / gh;  // head groups
  // (the grid's rows end with one tile's head groups more than the sequences
  // can have; a split grid's extra workgroups come after them)
  const uint32_t srows = SPLIT ? (uint32_t)a.rows : gridDim.x - hg;
  uint32_t row_id = blockIdx.x, slot = blockIdx.x;  // slot: of the piece's partial
  int ptiles = kWholeRows, piece = 0;
  SeqTile st;
  bool further = false;
  const int sh = __builtin_ctz(32 * qsubs);
  SplitPlan sp;
  if constexpr (SPLIT) {
    sp.q = split_seq<BN>(a, lane, sh);
    further = blockIdx.x >= srows + hg;
    if (further) {
      ptiles = sp.tiles = split_tiles<D, BN>(a, sp, sh);
      if (ptiles == kWholeRows) return;
      row_id = blockIdx.x - (srows + hg);
      slot = srows + row_id;
      const SplitPiece p = split_piece<BN>(a, sp, sh, (int)(row_id / hg));
      if (p.seq < 0) return;
      st.seq = p.seq;
      st.tile = p.tile;
      piece = p.piece;
    }
  }
  // rows from qb on of the `len` of a sequence that begins at s0 (shared: of a
  // group that begins at sequence sb0), their keys, and the position of row 0
  int64_t n, s0, len, qb, Lk, off;
  int kvh, head;
  int64_t pfx = 0;  // keys that every row sees
  int64_t sb0 = 0;
  int stile0 = 0;
  if constexpr (FORM == kShared) {
    if (blockIdx.x < a.own_wgs) {
      // a wave per unit, 16 query heads and kv head (the heads of a unit together:
      // their rows lie side by side); two waves' LDS lies in the key tiles, two in
      // the value tiles
      static_assert(2 * own_lds_per_wave<T, D>() <= sizeof(ks) && sizeof(ks) <= sizeof(vs), "the own keys' LDS");
      const uint32_t id = blockIdx.x * 4 + w, ny = a.Hkv * ((R + 15) / 16), u = id / ny, y = id - u * ny;
      if (u < (uint32_t)a.own.units)
        attn_own_wave<T, D, (PG >= 2)>(a.own,
                                       reinterpret_cast<char*>(w < 2 ? ks[0] : vs[0]) +
                                           (w & 1) * own_lds_per_wave<T, D>(),
                                       u, y % a.Hkv, y / a.Hkv);
      return;
    }
    const SharedWork sw = a.work[blockIdx.x - a.own_wgs];
    if (sw.lead < 0) return;
    n = sw.lead;
    sb0 = sw.b0;
    s0 = 0;
    len = sw.rows;
    qb = sw.row;
    Lk = sw.keys;
    off = 0;
    kvh = sw.kvh;
    head = kvh * R;
    slot = sw.slot;
    stile0 = sw.tile0;
  } else {
    if (!further) {
      st = attn_tile_lookup<D, PAGED, SPLIT>(a, 32 * qsubs, row_id / hg, lookup);
      // (no tile is left past the grid's rows unless the offsets decrease: nothing
      // is kept for it in the workspace)
      if (SPLIT && row_id >= srows && st.seq >= 0) return;
      if (st.seq < 0) {
        const uint32_t tiles = srows / hg + 1;
        zero_rows_tail<T>(a, (uint32_t)st.tile * hg + row_id % hg, (tiles - (row_id / hg - (uint32_t)st.tile)) * hg);
        return;
      }
    }
    n = st.seq;
    const int y = (int)(row_id % hg);
    kvh = y / groups;
    head = kvh * R + (y % groups) * gh + (w % gh);

    int64_t s1;
    seq_range(a.cu, a.cu64, n, a.T, s0, s1);
    len = s1 - s0;
    const int64_t ntile = (len + 32 * qsubs - 1) / (32 * qsubs);
    qb = (ntile - 1 - st.tile) * 32 * qsubs;  // last query tiles first

    if (PAGED) {
      const int64_t ctx = load_index(a.ctx, n, a.ctx64);
      Lk = clamp64(ctx, 0, a.tab.cols * a.tab.page);
      off = ctx - len;  // position of query 0
    } else {
      Lk = len;
      off = 0;
    }
    if (FORM == kScored && a.pfx) pfx = load_index(a.pfx, n, a.pfx64);
  }
  // (causal: the keys that the rows before row `end` see)
  auto seen = [&](int64_t end) __attribute__((always_inline)) {
    const int64_t e = off + end;
    return clamp64(FORM == kScored && e < pfx ? pfx : e, 0, Lk);
  };
  const int64_t q0 = qb + (w / gh) * 32;
  const int64_t wg_qend = qb + 32 * qsubs < len ? qb + 32 * qsubs : len;
  const int64_t w_qend = q0 + 32 < len ? q0 + 32 : len;
  const int64_t kend_row = FORM != kShared && a.causal ? seen(wg_qend) : Lk;
  const int64_t kend_roww = q0 >= len ? 0 : (FORM != kShared && a.causal ? seen(w_qend) : Lk);
  // this piece's key tiles [tile0, ntiles); keys past its end are not loaded
  const int tile0 = FORM == kShared ? stile0 : SPLIT ? piece * ptiles : 0;
  if (SPLIT && piece > 0 && (int64_t)tile0 * BN >= kend_row) return;
  int64_t kend = kend_row, kend_w = kend_roww;
  bool whole = true;  // the row is one piece
  auto cut = [&](int tiles) __attribute__((always_inline)) {
    const int64_t end = (int64_t)(tile0 + tiles) * BN;
    whole = kend_row <= (int64_t)tiles * BN;
    kend = kend_row > end ? end : kend_row;
    kend_w = kend_roww > end ? end : kend_roww;
  };
  if (SPLIT && further) cut(ptiles);

  // query fragments (B operand of S^T = K Q^T): lane holds query q0 + lane % 32,
  // dims 16 ks + 8 (lane / 32) .. +7
  const int col = lane & 31, hh = lane >> 5;
  const int64_t qi = q0 + col;
  const bool qvalid = qi < len;
  // (loaded unconditionally from a clamped row, so the loads stay in flight
  // while tile 0's K/V loads are issued; rows past the sequence are zeroed
  // where the fragments are staged, below)
  v8 qf[NKS];
  {
    static_assert(!RAG || q_pieces_inside(DQ), "query pieces are read inside their row");
    const int64_t row = qvalid ? qi : 0;
    // (shared: row r is head r % R of sequence r / R)
    const uint32_t sb = FORM == kShared ? (uint32_t)row / (uint32_t)R : 0u;
    const T* qp = reinterpret_cast<const T*>(a.q) + (FORM == kShared ? sb0 + sb : s0 + row) * a.q_st +
                  (int64_t)(FORM == kShared ? head + (int)((uint32_t)row - sb * R) : head) * a.q_sh;
#pragma unroll
    for (int s = 0; s < NKS; ++s)
      qf[s] = *reinterpret_cast<const v8*>(qp + (RAG ? q_piece(s, hh, a.dim) : 16 * s + 8 * hh));
  }
  // the softmax below assumes c > 0: a negative scale is folded into q (an
  // exact sign flip), a zero scale is q = 0 with c = 1 (equal weights)
  float c = a.c;
  T* const qw = qs + (QL ? w * 32 * LDK : 0);  // this wave's query rows (only the wave reads them)
  auto stage_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < NKS; ++s) qf[s] = qvalid && (!RAG || 16 * s + 8 * hh < a.dim) ? qf[s] : v8{};
    if (c <= 0.f) {
#pragma unroll
      for (int s = 0; s < NKS; ++s) qf[s] = c < 0.f ? -qf[s] : v8{};
      c = c < 0.f ? -c : 1.f;
    }
    if constexpr (QL) {
#pragma unroll
      for (int s = 0; s < NKS - QRG; ++s) *reinterpret_cast<v8*>(qw + col * LDK + 16 * s + 8 * hh) = qf[s];
    }
  };

  // staging of a K/V tile: global rows -> registers (rows past kend read as
  // zero, so a tile past the range loads nothing) -> LDS
  // packed rows: per key tile, buffer descriptors of the tile's rows of this
  // sequence's kv head whose range ends at the last row before kend (rows
  // past it read as zero, 32-bit offsets): a lane's offsets are the same for
  // every tile, and the tile's position and bound are scalar arithmetic
  const char* const kseq = a.k.base + s0 * a.k.st + kvh * a.k.sh;
  const char* const vseq = a.v.base + s0 * a.v.st + kvh * a.v.sh;
  constexpr int NG = BN / 16;  // 16-row groups of a tile
  static_assert(PG == 0 || (CH >= 8 && 64 % CH == 0), "a wave's rows of a tile lie in one 16-row group");
  // PG 2, 3: each 16-row group of a tile lies in one page.  Its block id is a
  // vector load issued one tile ahead, before the previous tile's data loads,
  // so waiting for it leaves those data loads in flight (a scalar load would
  // be waited for at once, its value forming the addresses, and that wait
  // also drains every LDS access in flight).  The rows then load through a
  // buffer descriptor of the kv head's rows of the page: 32-bit offsets, rows
  // past the range or of an invalid block read zero.
  // The 16-row groups are enumerated in order (load_ids runs for tiles tile0,
  // tile0 + 1, ...), so a group's table column and first page slot are counted up,
  // not divided out.
  // An id is kept as the two raw 32-bit words it was loaded as (an int32
  // table: the entry twice) and decoded only where it is used: converting it
  // at the load would wait for the load, and with it for every load in flight.
  uint32_t idlo[NG], idhi[NG];  // raw block ids of the next tile to load
  bool idin[NG];                // its groups lie inside the range and the table
  uint32_t slots[NG];           // their first page slot
  constexpr bool G16 = PG >= 2, T64 = PG == 3;  // 16-row groups per page lookup; int64 table
  constexpr bool ONE = PG == 4;                               // a page is a 16-row group
  const uint32_t gpp = G16 && !ONE ? (uint32_t)a.tab.page / 16 : 1u;  // 16-row groups per page
  uint32_t gcol = 0, grem = 0;  // table column and group within the page of the next group
  // (G16) this sequence's row of the block table as 32-bit words; the table
  // has columns, and key positions (columns x page), block ids and block
  // strides fit 32 bits (the launcher takes the per-row path otherwise)
  const uint32_t* trow = G16 ? reinterpret_cast<const uint32_t*>(a.tab.table) + (T64 ? 2 : 1) * (n * a.tab.row_stride)
                             : nullptr;
  uint32_t kend32 = (uint32_t)kend;
  auto load_ids = [&](int t, uint32_t* lo, uint32_t* hi, bool* in, uint32_t* sl) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t j0 = (uint32_t)t * BN + 16 * g;
      in[g] = j0 < kend32 && gcol < a.tab.cols;
      // (the index goes through a vector register so the loads stay vector loads)
      uint32_t e = in[g] ? gcol : 0u;
      asm volatile("" : "+v"(e));
      if constexpr (T64) {
        lo[g] = trow[2 * e];
        hi[g] = trow[2 * e + 1];
      } else {
        lo[g] = trow[e];
        hi[g] = 0u;
      }
      sl[g] = ONE ? 0u : 16 * grem;
      if (ONE) {
        ++gcol;
      } else if (++grem == gpp) {
        grem = 0;
        ++gcol;
      }
    }
  };
  if (SPLIT || FORM == kShared) {
    gcol = (uint32_t)tile0 * NG / gpp;
    grem = (uint32_t)tile0 * NG - gcol * gpp;
  }
  if (G16) load_ids(tile0, idlo, idhi, idin, slots);
  const uint32_t kst = (uint32_t)a.k.st, vst = ONE ? kst : (uint32_t)a.v.st;  // row strides in bytes (below 2^31)
  const char* kbase = a.k.base + kvh * a.k.sh;
  const char* vbase = a.v.base + kvh * a.v.sh;
  const uint64_t ksb = (uint32_t)a.k.sb, vsb = ONE ? ksb : (uint32_t)a.v.sb;
  const uint32_t nblk = (uint32_t)(a.tab.num_blocks < 0x7fffffff ? a.tab.num_blocks : 0x7fffffff);
  auto load_tile = [&](int t, uint4* kd, uint4* vd) {
    __amdgpu_buffer_rsrc_t rkg[NG], rvg[NG], rkt, rvt;
    uint32_t r0[NG];
    if (!PAGED) {
      const uint32_t t0 = (uint32_t)t * BN;
      const uint32_t nv = t0 < kend32 ? (kend32 - t0 < (uint32_t)BN ? kend32 - t0 : (uint32_t)BN) : 0u;
      rkt = __builtin_amdgcn_make_buffer_rsrc((void*)(kseq + (uint64_t)t0 * kst), 0, nv * kst, 0x00020000);
      rvt = __builtin_amdgcn_make_buffer_rsrc((void*)(vseq + (uint64_t)t0 * vst), 0, nv * vst, 0x00020000);
    }
    if (G16) {
      uint32_t nlo[NG], nhi[NG], nsl[NG];
      bool nin[NG];
      load_ids(t + 1, nlo, nhi, nin, nsl);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        // valid: inside the range, high word zero (int64) or non-negative (int32), below num_blocks
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)idlo[g]);
        const uint32_t hi = T64 ? (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)idhi[g]) : 0u;
        // (an int32 id below nblk is non-negative: negative ids compare above it unsigned)
        const bool valid = idin[g] && hi == 0u && lo < nblk;
        const uint64_t bb = valid ? lo : 0u;
        r0[g] = slots[g];
        // the group's rows before kend: its range ends after them in the page,
        // so the rows past kend read as zero with no test per row
        const uint32_t j0 = (uint32_t)t * BN + 16u * g;
        const uint32_t ends = slots[g] + (j0 < kend32 ? (kend32 - j0 < 16u ? kend32 - j0 : 16u) : 0u);
        // (block strides below 2^32, checked by the launcher: 32 x 32-bit products)
        rkg[g] = __builtin_amdgcn_make_buffer_rsrc((void*)(kbase + bb * ksb), 0, valid ? ends * kst : 0u, 0x00020000);
        rvg[g] = __builtin_amdgcn_make_buffer_rsrc((void*)(vbase + bb * vsb), 0, valid ? ends * vst : 0u, 0x00020000);
        idlo[g] = nlo[g];
        idhi[g] = nhi[g];
        idin[g] = nin[g];
        slots[g] = nsl[g];
      }
    }
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int c = tid + 256 * i, row = c / CH, ch = c % CH;
      const int64_t j = (int64_t)t * BN + row;
      if (G16) {
        // the row's 16-row group: i * rows-per-pass / 16 when a pass covers at
        // most 16 rows (a constant), else plus the wave's part (uniform)
        constexpr int RPI = 256 / CH;
        __amdgpu_buffer_rsrc_t rkx, rvx;
        uint32_t rx;
        if constexpr (RPI <= 16) {
          rkx = rkg[i * RPI / 16];
          rvx = rvg[i * RPI / 16];
          rx = r0[i * RPI / 16];
        } else {
          const int gu = __builtin_amdgcn_readfirstlane(row >> 4);
          rkx = rkg[0], rvx = rvg[0], rx = r0[0];
#pragma unroll
          for (int g = 1; g < NG; ++g) {
            rkx = gu == g ? rkg[g] : rkx;
            rvx = gu == g ? rvg[g] : rvx;
            rx = gu == g ? r0[g] : rx;
          }
        }
        const uint32_t slot = rx + (uint32_t)(row & 15);
        kd[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rkx, slot * kst + 16u * ch, 0, 0));
        vd[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rvx, slot * vst + 16u * ch, 0, 0));
        continue;
      }
      if (!PAGED) {
        // (the row offset times the stride fits 32 bits: the launcher checks
        // max(max_seqlen, 64) rows of either stride against 2^31)
        // (ranges are below 2^31 bytes, so 2^31 more is past them whatever the row)
        const uint32_t co = !RAG || 8 * ch < a.dim ? 16u * ch : 0x80000000u;
        kd[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rkt, (uint32_t)row * kst + co, 0, 0));
        vd[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rvt, (uint32_t)row * vst + co, 0, 0));
        continue;
      }
      const char* pk = j < kend ? kv_row<PAGED>(a.k, a.tab, n, s0, j, kvh) : nullptr;
      const char* pv = j < kend ? kv_row<PAGED>(a.v, a.tab, n, s0, j, kvh) : nullptr;
      kd[i] = pk ? *reinterpret_cast<const uint4*>(pk + 16 * ch) : uint4{0, 0, 0, 0};
      vd[i] = pv ? *reinterpret_cast<const uint4*>(pv + 16 * ch) : uint4{0, 0, 0, 0};
    }
  };
  auto store_tile = [&](int buf, const uint4* kd, const uint4* vd) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int c = tid + 256 * i, row = c / CH, ch = c % CH;
      *reinterpret_cast<uint4*>(&ks[buf][row * LDK + 8 * ch]) = kd[i];
      *reinterpret_cast<uint4*>(&vs[buf][row * LDV + 8 * ch]) = vd[i];
    }
  };
  // (kFp4) this thread's codes and scale of a row of keys or values, and whether its
  // 16-row group has keys (the wave's rows lie in one group)
  struct Codes {
    uint32_t w[QW], s;
    bool named;
  };
  typedef std::conditional_t<Q4, Codes, uint4> Reg;
  constexpr int NREG = Q4 ? 1 : NLD;
  const uint32_t qrow = (uint32_t)tid / QL8 & 15u, qch = (uint32_t)tid % QL8;
  const uint32_t qko = qrow * kst + qch * (QE / 2), qvo = qrow * vst + qch * (QE / 2);
  auto load = [&](int t, Reg* kd, Reg* vd) __attribute__((always_inline)) {
    if constexpr (Q4) {
      // Scalar bases and one offset per lane (descriptors of four tensors leave too few
      // scalar registers: four chunks of up to 2,048 tokens over up to 16,384 keys took
      // 1,154 us with them, 1,171 with addresses on the vector side, 1,083 so, by PG 2).  Rows past
      // the range are read as the last one in it, a group without keys from block 0,
      // whose codes and scales store() clears.
      uint32_t nlo[NG], nhi[NG], nsl[NG];
      bool nin[NG];
      load_ids(t + 1, nlo, nhi, nin, nsl);
      static_assert(64 / QL8 <= 16, "a wave's rows");
      const int gu = w * (64 / QL8) / 16;
      uint32_t ulo = idlo[0], uhi = idhi[0], usl = slots[0];
      bool uin = idin[0];
#pragma unroll
      for (int g = 1; g < NG; ++g)
        if (gu == g) ulo = idlo[g], uhi = idhi[g], usl = slots[g], uin = idin[g];
      const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)ulo);
      const uint32_t hi = T64 ? (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)uhi) : 0u;
      const uint32_t j0 = (uint32_t)t * BN + 16u * gu;
      const bool named = uin && hi == 0u && lo < nblk;  // (uin: keys of the group lie in the range)
      const uint64_t bb = named ? lo : 0u;
      uint32_t ko = qko, vo = qvo, row = qrow;
      if (named && kend32 - j0 < 16u) {
        const uint32_t last = kend32 - j0 - 1u;
        row = qrow < last ? qrow : last;
        ko = row * kst + qch * (QE / 2), vo = row * vst + qch * (QE / 2);
      }
      const ScaleSource& vss = ONE ? a.ks : a.vs;  // (its strides)
      uint32_t kso = qch * QE / 32 * (uint32_t)a.ks.sd + row, vso = qch * QE / 32 * (uint32_t)vss.sd + row;
      asm("" : "+v"(ko), "+v"(kso));
      if (ONE) vo = ko, vso = kso;
      else asm("" : "+v"(vo), "+v"(vso));
      const char* const kp = kbase + bb * ksb + (uint64_t)(usl * kst);
      const char* const vp = vbase + bb * vsb + (uint64_t)(usl * vst);
      const uint8_t* const ksp = a.ks.base + kvh * a.ks.sh + bb * (uint32_t)a.ks.sb + usl;
      const uint8_t* const vsp = a.vs.base + kvh * vss.sh + bb * (uint32_t)vss.sb + usl;
      auto codes = [](const char* p, Codes& c) __attribute__((always_inline)) {
        if constexpr (QW == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(p);
          c.w[0] = x.x, c.w[1] = x.y, c.w[2] = x.z, c.w[3] = x.w;
        } else if constexpr (QW == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(p);
          c.w[0] = x.x, c.w[1] = x.y;
        } else {
          c.w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
      };
      codes(kp + ko, kd[0]);
      codes(vp + vo, vd[0]);
      kd[0].s = ksp[kso];
      vd[0].s = vsp[vso];
      kd[0].named = vd[0].named = named;
#pragma unroll
      for (int g = 0; g < NG; ++g) idlo[g] = nlo[g], idhi[g] = nhi[g], idin[g] = nin[g], slots[g] = nsl[g];
    } else {
      load_tile(t, kd, vd);
    }
  };
  uint32_t nan_tile = UINT32_MAX;  // (kFp4) the first tile in which this thread's numbers of a value are NaN
  auto store = [&](int t, int buf, const Reg* kd, const Reg* vd) __attribute__((always_inline)) {
    if constexpr (Q4) {
      const int row = tid / QL8, ch = tid % QL8;
      // neighbouring lanes write their words in another order each, so that their
      // 16-byte stores, QE elements apart, fall on different banks
      const int turn = QW == 4 ? (ch + (ch >> 2)) & 3 : QW == 2 ? ch >> 2 & 1 : 0;
      auto put = [&](T* at, const Codes& c, uint32_t scale) __attribute__((always_inline)) {
        uint32_t x[QW], sb = scale;
#pragma unroll
        for (int i = 0; i < QW; ++i) x[i] = c.w[i];
        if (!c.named) {
          sb = 0u;
#pragma unroll
          for (int i = 0; i < QW; ++i) x[i] = 0u;
        }
        const float s = fp4_scale(sb);
        if constexpr (QW >= 2) {  // x[i] <- word (i ^ turn)
#pragma unroll
          for (int i = 0; i < QW; i += 2) {
            const uint32_t p = x[i], q = x[i + 1];
            x[i] = turn & 1 ? q : p;
            x[i + 1] = turn & 1 ? p : q;
          }
        }
        if constexpr (QW == 4) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t p = x[i], q = x[i + 2];
            x[i] = turn & 2 ? q : p;
            x[i + 2] = turn & 2 ? p : q;
          }
        }
#pragma unroll
        for (int i = 0; i < QW; ++i) *reinterpret_cast<uint4*>(at + QE * ch + 8 * (i ^ turn)) = fp4_eight<T>(x[i], s);
      };
      put(&ks[buf][row * LDK], kd[0], kd[0].s);
      const bool nan = vd[0].named && vd[0].s == 255u;
      const uint32_t in = nan ? (uint32_t)t : UINT32_MAX;
      nan_tile = in < nan_tile ? in : nan_tile;
      put(&vs[buf][row * LDV], vd[0], nan ? 0u : vd[0].s);
    } else {
      store_tile(buf, kd, vd);
    }
  };

  f32x16 oacc[NDT];
#pragma unroll
  for (int d = 0; d < NDT; ++d) oacc[d] = f32x16{};
  float m_used = -INFINITY, lsum = 0.f;
  float nb = 0.f;  // -m_used, or 0 while m_used is -inf (the exponent offset)

  // a key tile needs the mask when it reaches past the keys (t BN + BN > Lk)
  // or, causal, past the wave's first query (t BN + BN - 1 > off + q0):
  // t BN > mthr, one 32-bit test per tile (key positions stay below 2^31)
  const int64_t first = FORM == kScored && off + q0 + 1 < pfx ? pfx : off + q0 + 1;  // keys that the first query sees
  const int mthr = (int)clamp64(FORM != kShared && a.causal && first < Lk ? first - BN : Lk - BN, -1, 0x7fffffff);
  const int qpos = FORM == kScored ? (int)clamp64(off + qi, INT32_MIN, INT32_MAX) : 0;
  // tiles up to key `lin` have no visible key past the wave's first query
  const int lin = FORM != kScored            ? 0
                  : a.causal && pfx <= 0 ? INT32_MAX
                                         : (int)clamp64(off + q0 - BN + 1, -1, INT32_MAX);
  const float slope = FORM == kScored && a.slopes ? a.slopes[head] * kLog2e : 0.f;  // in exponents of 2
  // `mid` (the next tiles' LDS stores and global loads) is issued right after
  // the score MFMAs, so that its issue overlaps their execution; a wave with
  // no keys left in this tile still runs it
  // scored rows: what c scales is the capped score where there is a cap, and the
  // bias goes on it in the same units (c > 0 from stage_q on)
  float capk = 0.f, sraw = 0.f, slope4 = 0.f;
  CapNear cn{};
  auto score_consts = [&]() __attribute__((always_inline)) {
    if (a.cap_out > 0.f) {
      capk = fminf(c * a.cap_in, 3e38f);  // (finite: a score of 0 stays 0)
      cn.set(capk);
      c = a.cap_out;
    }
    sraw = slope / c;
    slope4 = slope * (float)(4 * hh);
  };
  auto compute = [&](int t, int buf, auto&& mid) {
    if ((int64_t)t * BN < kend_w) {
      const T* K = ks[buf];
      const T* V = vs[buf];
      f32x16 s[NA];
#pragma unroll
      for (int aa = 0; aa < NA; ++aa) {
        s[aa] = f32x16{};
        const T* kp = K + (32 * aa + col) * LDK + 8 * hh;
        if constexpr (QL) {
          const T* qp = qw + col * LDK + 8 * hh;
#pragma unroll
          for (int k = 0; k < NKS; ++k)
            s[aa] = M::m32(*reinterpret_cast<const v8*>(kp + 16 * k),
                           k >= NKS - QRG ? qf[k] : *reinterpret_cast<const v8*>(qp + 16 * k), s[aa]);
          // schedule: the K and Q fragments of the next k-steps are read while each MFMA runs
          __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // DS reads
#pragma unroll
          for (int k = 0; k < NKS; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            if (k + 2 < NKS - QRG) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            else if (k + 2 < NKS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
        } else {
#pragma unroll
          for (int k = 0; k < NKS; ++k) s[aa] = M::m32(*reinterpret_cast<const v8*>(kp + 16 * k), qf[k], s[aa]);
        }
      }
      mid();
      // scored: the bias of the tile's first key at this lane's query, where the
      // distance from it adds to the scores
      float bias = 0.f;
      if constexpr (FORM == kScored) {
        constexpr bool NEAR = D == 64;
        // one straight run per combination: cap (0 none, 1 any score, 2 near), then
        // bias (0 none, 1 linear, 2 by |i - j|)
        const float d0 = (float)(int)((uint32_t)(t * BN) - (uint32_t)qpos);
        auto form = [&](auto cap, auto dist) __attribute__((always_inline)) {
#pragma unroll
          for (int aa = 0; aa < NA; ++aa)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float j = (float)(32 * aa + 8 * (r >> 2) + (r & 3));
              float x = s[aa][r];
              if constexpr (cap == 1) x = cap_score(x, capk);
              if constexpr (cap == 2) x = cn(x);
              if constexpr (dist == 1) x = __builtin_fmaf(sraw, j, x);
              if constexpr (dist == 2) x = __builtin_fmaf(-sraw, __builtin_fabsf(d0 + (float)(4 * hh) + j), x);
              s[aa][r] = x;
            }
          if constexpr (dist == 1) bias = __builtin_fmaf(slope, d0, slope4);
        };
        typedef std::integral_constant<int, 0> I0;
        typedef std::integral_constant<int, 1> I1;
        typedef std::integral_constant<int, 2> I2;
        // (1: no visible key past the queries, so |i - j| is i - j)
        const int dist = !a.slopes ? 0 : t * BN <= lin ? 1 : 2;
        bool near = false;
        if (NEAR && a.cap_out > 0.f) {
          float top = 0.f;
#pragma unroll
          for (int aa = 0; aa < NA; ++aa)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, __builtin_fabsf(s[aa][r]));
          near = __builtin_amdgcn_ballot_w64(top > cn.lim) == 0;
        }
        if (NEAR && near) {
          if (dist == 0) form(I2(), I0());
          else if (dist == 1) form(I2(), I1());
          else form(I2(), I2());
        } else if (a.cap_out > 0.f) {
          if (dist == 0) form(I1(), I0());
          else if (dist == 1) form(I1(), I1());
          else form(I1(), I2());
        } else if (dist == 1) {
          form(I0(), I1());
        } else if (dist == 2) {
          form(I0(), I2());
        }
      }
      // mask keys past the sequence / context and, if causal, past the query
      const int64_t tk0 = (int64_t)t * BN;
      if (t * BN > mthr) {
        const int64_t own = FORM == kScored && off + qi + 1 < pfx ? pfx : off + qi + 1;
        const int64_t lim = (FORM != kShared && a.causal && own < Lk ? own : Lk) - tk0;
        const int rel = (int)clamp64(lim, -1, BN);  // keys of the tile at or past rel are masked
#pragma unroll
        for (int aa = 0; aa < NA; ++aa)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * aa + 8 * (r >> 2) + 4 * hh + (r & 3) >= rel) s[aa][r] = -INFINITY;
      }
      // tile maximum of the scaled scores (c > 0) over this lane's half of
      // the query's keys; masked scores are -inf and give p = exp2(-inf) = 0
      // below.  The lane pair (l, l ^ 32) shares one base: it moves only when
      // some lane's half exceeds it by 2^8, and then to the maximum over the
      // pair, so the pair's maximum is taken only on that rare path (the
      // same decisions and bases as taking it every tile)
      float mx = -INFINITY;
#pragma unroll
      for (int aa = 0; aa < NA; ++aa)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[aa][r]);
      // (A bias that rises towards the query would move the base on every tile:
      // with P in bf16, of fp32's range, it moves ahead of the maximum by what the
      // bias has still to rise from the tile's last key to the query, at most 2^56,
      // so that P ends near 1.  Four chunks of 256 to 1,024 tokens behind up to 16,384
      // keys, 16 / 4 heads of 128: 525 -> 481 us.  Always 2^56 ahead, and a base that
      // trails by up to 2^24, took 474, but lost values below 1e-21 and above 1e31.)
      constexpr bool WIDE = FORM == kScored && std::is_same<T, bf16_t>::value;
      const float top = FORM == kScored ? __builtin_fmaf(mx, c, bias) : mx * c;
      if (__builtin_amdgcn_ballot_w64(top > m_used + 8.f) != 0) {
        float ahead = 0.f;
        if constexpr (WIDE) {
          const float left = (float)(int)((uint32_t)qpos - (uint32_t)(t * BN + BN - 1));
          ahead = fminf(fmaxf(slope * fmaxf(left, 0.f), 0.f), 56.f);
        }
        const float mn = FORM == kScored ? fmaxf(m_used, max_lane_pair32(top + ahead))
                                         : fmaxf(m_used, max_lane_pair32(mx) * c);
        const float alpha = mn == -INFINITY ? 1.f : exp2_fast(m_used - mn);
#pragma unroll
        for (int d = 0; d < NDT; ++d) oacc[d] *= alpha;
        lsum *= alpha;
        m_used = mn;
        nb = mn == -INFINITY ? 0.f : -mn;
      }
#pragma unroll
      for (int aa = 0; aa < NA; ++aa) {
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
          v8 pf;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = exp2_fast(__builtin_fmaf(s[aa][8 * h2 + e], c, FORM == kScored ? nb + bias : nb));
            lsum += p;
            pf[e] = (T)p;
          }
          // V^T fragment for keys 32 aa + 16 h2 + {4 hh + 0..3, 8 + 4 hh + 0..3}
          const int j16 = lane & 15, qd = lane >> 4;
          const T* vp = V + (32 * aa + 16 * h2 + 4 * (qd >> 1) + (j16 >> 2)) * LDV + 16 * (qd & 1) + 4 * (j16 & 3);
          auto vfrag = [&](int d) __attribute__((always_inline)) {
            const v4 lo = tr4<v4>(vp + 32 * d);
            const v4 hi = tr4<v4>(vp + 32 * d + 8 * LDV);
            return v8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          };
          if constexpr (QL) {
            // the V fragments of two MFMAs ahead are in flight while each
            // MFMA runs; the scheduling barrier keeps the reads ahead
            constexpr int AH = 2;
            v8 vf[AH + 1];
#pragma unroll
            for (int i = 0; i < AH; ++i) vf[i] = vfrag(i);
#pragma unroll
            for (int d = 0; d < NDT; ++d) {
              if (d + AH < NDT) vf[(d + AH) % (AH + 1)] = vfrag(d + AH);
              __builtin_amdgcn_sched_barrier(0);
              oacc[d] = M::m32(vf[d % (AH + 1)], pf, oacc[d]);
            }
          } else {
#pragma unroll
            for (int d = 0; d < NDT; ++d) oacc[d] = M::m32(vfrag(d), pf, oacc[d]);
          }
        }
      }
    } else {
      mid();
    }
  };

  // tile t computes from LDS buffer t % 2 while tile t + 1 waits in registers
  // and tile t + 2 is in flight: two register sets (A: even tiles, B: odd)
  Reg kA[NREG], vA[NREG], kB[NREG], vB[NREG];
  load(tile0, kA, vA);
  // (a row's first piece works out where it ends only now, with the first tile's
  // loads in flight: no piece is shorter than that)
  if constexpr (SPLIT) {
    if (!further) {
      cut(split_tiles<D, BN>(a, sp, sh));
      kend32 = (uint32_t)kend;
    }
  }
  const int ntiles = (int)((kend + BN - 1) / BN);
  stage_q();  // (waits for the query loads with tile 0's loads in flight)
  if constexpr (FORM == kScored) score_consts();
  store(tile0, 0, kA, vA);
  load(tile0 + 1, kB, vB);
  load(tile0 + 2, kA, vA);
  __syncthreads();
  // (packed rows: the next tiles' stores and loads go out between the score
  // MFMAs and the softmax; paged rows: after the tile, since their loads
  // first wait for the block ids, and the longer live ranges cost registers)
  for (int t = tile0; t < ntiles; t += 2) {
    if constexpr (PG == 0) {
      compute(t, 0, [&]() __attribute__((always_inline)) {
        store(t + 1, 1, kB, vB);
        load(t + 3, kB, vB);
      });
      __syncthreads();
      compute(t + 1, 1, [&]() __attribute__((always_inline)) {
        store(t + 2, 0, kA, vA);
        load(t + 4, kA, vA);
      });
      __syncthreads();
    } else {
      const auto after = []() {};  // (one instantiation of compute for both calls)
      compute(t, 0, after);
      store(t + 1, 1, kB, vB);
      load(t + 3, kB, vB);
      __syncthreads();
      compute(t + 1, 1, after);
      store(t + 2, 0, kA, vA);
      load(t + 4, kA, vA);
      __syncthreads();
    }
  }

  if constexpr (Q4) {
    const uint32_t u = 64 * w + lane_anew();
    if (nan_tile != UINT32_MAX)
      __hip_atomic_fetch_min(&nan_at[u % QL8 * QE / 32], nan_tile * BN + u / QL8, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_WORKGROUP);
    __syncthreads();
    const uint32_t keys = (uint32_t)seen(q0 + (u & 31u) + 1);  // that this lane's query sees
#pragma unroll
    for (int d = 0; d < NDT; ++d) {
      const bool nan = nan_at[d] < keys;
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(nan) != 0, 0)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[d][r] = nan ? __builtin_nanf("") : oacc[d][r];
      }
    }
  }
  const float lt = lsum + __shfl_xor(lsum, 32);
  if constexpr (SPLIT || FORM == kShared) {
    if (FORM == kShared || !whole) {
      float* pw = a.part + (int64_t)slot * prefill_part_floats<D>() + w * prefill_part_wave<D>();
#pragma unroll
      for (int d = 0; d < NDT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(pw + ((4 * d + g) * 64 + lane) * 4) =
              f32x4{oacc[d][4 * g], oacc[d][4 * g + 1], oacc[d][4 * g + 2], oacc[d][4 * g + 3]};
      pw[32 * D + lane] = m_used;
      pw[32 * D + 64 + lane] = lt;
      return;
    }
  }
  const float inv = lt > 0.f ? 1.f / lt : 0.f;
  if constexpr (QL) {
    // O goes out through the wave's own query rows in LDS (no longer read):
    // each lane writes its 4-dim pieces of its query's row, then reads back
    // 16-byte row pieces, so that one store instruction covers two whole
    // output rows (512 contiguous bytes each) instead of 32 rows x 16 bytes
#pragma unroll
    for (int d = 0; d < NDT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        v4 ov;
#pragma unroll
        for (int e = 0; e < 4; ++e) ov[e] = (T)(oacc[d][4 * g + e] * inv);
        *reinterpret_cast<v4*>(qw + col * LDK + 32 * d + 8 * g + 4 * hh) = ov;
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int cpos = lane & (CH - 1), rsub = lane / CH;  // 16-byte piece of a row, row within the pass
    constexpr int RPP = 64 / CH;                           // rows per pass
    const int qrem = (int)clamp64(len - q0, 0, 32);  // rows of this wave inside the sequence
    T* const orow = reinterpret_cast<T*>(a.o) + (s0 + q0) * a.o_st + (int64_t)head * a.o_sh + 8 * cpos;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += RPP) {
      const int r = r0 + rsub;
      const v8 ov = *reinterpret_cast<const v8*>(qw + r * LDK + 8 * cpos);
      if (r < qrem && (!RAG || 8 * cpos < a.dim)) *reinterpret_cast<v8*>(orow + (int64_t)r * a.o_st) = ov;
    }
  } else if (qvalid) {
    T* op = reinterpret_cast<T*>(a.o) + (s0 + qi) * a.o_st + (int64_t)head * a.o_sh + 4 * hh;
#pragma unroll
    for (int d = 0; d < NDT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (RAG && 32 * d + 8 * g >= a.dim) break;
        v4 ov;
#pragma unroll
        for (int e = 0; e < 4; ++e) ov[e] = (T)(oacc[d][4 * g + e] * inv);
        *reinterpret_cast<v4*>(op + 32 * d + 8 * g) = ov;
      }
  }
}

// Merge of a split prefill's pieces: workgroup (row, dim group) of the same
// 4 waves x 32 queries as the prefill kernel, each lane reading back its own
// accumulator pieces of DG 32-dim blocks.  Rows of one piece were written by
// the prefill itself.
template <typename T, int D, int BN, int DG, AttnForm FORM = kPlain>
__global__ __launch_bounds__(256) void attn_prefill_combine_kernel(const AttnArgs a) {
  typedef typename Mma<T>::v4 v4;
  __shared__ int32_t lookup[8];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = a.Hq / a.Hkv, gh = a.gh, qsubs = 4 / gh, groups = R / gh, hg = a.Hq / gh;
  const int sh = __builtin_ctz(32 * qsubs);
  SplitPlan sp;
  sp.q = split_seq<BN>(a, lane, sh);
  sp.tiles = split_tiles<D, BN>(a, sp, sh);
  if (sp.tiles == kWholeRows) return;
  const SeqTile st = attn_tile_lookup<D, true, true>(a, 32 * qsubs, blockIdx.x / hg, lookup);
  if (st.seq < 0) return;
  const int y = (int)(blockIdx.x % hg);
  const int head = (y / groups) * R + (y % groups) * gh + (w % gh);
  int64_t s0, s1;
  seq_range(a.cu, a.cu64, st.seq, a.T, s0, s1);
  const int64_t len = s1 - s0;
  const int64_t ntile = (len + 32 * qsubs - 1) / (32 * qsubs);
  const int64_t qb = (ntile - 1 - st.tile) * 32 * qsubs;
  const int64_t ctx = load_index(a.ctx, st.seq, a.ctx64);
  const int64_t Lk = clamp64(ctx, 0, a.tab.cols * a.tab.page);
  const int64_t wg_qend = qb + 32 * qsubs < len ? qb + 32 * qsubs : len;
  int64_t end = ctx - len + wg_qend;
  if (FORM == kScored && a.pfx) {
    const int64_t pfx = load_index(a.pfx, st.seq, a.pfx64);
    end = end < pfx ? pfx : end;
  }
  const int64_t kend = clamp64(end, 0, Lk);
  const int64_t pk = (int64_t)sp.tiles * BN;
  const int np = (int)((kend + pk - 1) / pk);
  const int64_t qi = qb + (w / gh) * 32 + (lane & 31);
  if (np <= 1) return;
  // slots of the row's further pieces, in lane order; the first has the row's own
  const SplitCount k = split_count<BN>(a, sp, sh, (int)st.seq);
  const int extra = wave_inclusive_scan_i32(k.all) - k.all + k.before + (int)st.tile;
  const int slots = lane == 0 ? (int)blockIdx.x : (int)a.rows + extra * hg + y;
  // (lanes past the sequence's end go along: their slots are read by the others)
  const float* const mine = a.part + w * prefill_part_wave<D>();
  for (int g = blockIdx.y; g < D / (32 * DG); g += gridDim.y) {
    f32x4 acc[4 * DG];
#pragma unroll
    for (int i = 0; i < 4 * DG; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float mx = -INFINITY, l = 0.f;
#pragma unroll 2
    for (int p = 0; p < np; ++p) {
      const float* pp = mine + (int64_t)__builtin_amdgcn_readlane(slots, p) * prefill_part_floats<D>();
      const float m = pp[32 * D + lane], lp = pp[32 * D + 64 + lane];
      f32x4 o[4 * DG];
#pragma unroll
      for (int i = 0; i < 4 * DG; ++i) o[i] = *reinterpret_cast<const f32x4*>(pp + ((4 * DG * g + i) * 64 + lane) * 4);
      // (a piece, or all so far, without keys has weight 0)
      const float top = fmaxf(mx, m);
      const float was = mx == -INFINITY ? 0.f : exp2_fast(mx - top), now = m == -INFINITY ? 0.f : exp2_fast(m - top);
      mx = top;
      l = l * was + lp * now;
#pragma unroll
      for (int i = 0; i < 4 * DG; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = acc[i][e] * was + o[i][e] * now;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T* op = reinterpret_cast<T*>(a.o) + (s0 + qi) * a.o_st + (int64_t)head * a.o_sh + 4 * (lane >> 5) + 32 * DG * g;
#pragma unroll
    for (int i = 0; i < 4 * DG; ++i) {
      v4 ov;
#pragma unroll
      for (int e = 0; e < 4; ++e) ov[e] = (T)(acc[i][e] * inv);
      if (qi < len) *reinterpret_cast<v4*>(op + 8 * i) = ov;
    }
  }
}

// Whether the kernels that look a page up once per 16 rows serve the caches:
// whole 16-row groups per page, 32-bit table arithmetic.
bool whole_groups(const AttnArgs& a) {
  return a.tab.page % 16 == 0 && a.k.sb < (int64_t(1) << 32) && a.v.sb < (int64_t(1) << 32) && a.tab.cols > 0 &&
         a.tab.cols * a.tab.page < (int64_t(1) << 31) && a.tab.num_blocks < (int64_t(1) << 31);
}

template <typename T, int D, int BN, bool PAGED, int DQ = 0, AttnForm FORM = kPlain>
hipError_t launch_prefill_t(const AttnArgs& a, int64_t nseq, int64_t max_len, hipStream_t st) {
  const int qsubs = 4 / a.gh;
  // without sequences there are only rows to zero
  if (nseq <= 0 || max_len <= 0)
    zero_uncovered_rows_kernel<(int)sizeof(T)><<<dim3(64), dim3(256), 0, st>>>(a.o, a.o_st, a.o_sh, a.Hq, a.dim, a.cu,
                                                                             a.cu64, a.nseq, a.T);
  if (nseq <= 0 || max_len <= 0) return hipGetLastError();
  // query tiles: at most T / tile_len + one partial tile per sequence, and one
  // that no sequence can have
  const int64_t tiles = a.T / (32 * qsubs) + nseq + 1;
  const dim3 grid((unsigned)(tiles * (a.Hq / a.gh)));
  if constexpr (!PAGED) {
    hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 0, false, DQ, FORM>), grid, dim3(256), 0, st, a);
  } else if (whole_groups(a)) {
    if (a.extra > 0) {
      const dim3 sgrid((unsigned)(a.rows + a.Hq / a.gh + a.extra));
      constexpr int DG = D == 256 ? 2 : 1;  // 32-dim blocks per combine workgroup
      if (a.tab.is64)
        hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 3, true, 0, FORM>), sgrid, dim3(256), 0, st, a);
      else
        hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 2, true, 0, FORM>), sgrid, dim3(256), 0, st, a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      // (many rows fill the chip by themselves)
      hipLaunchKernelGGL((attn_prefill_combine_kernel<T, D, BN, DG, FORM>),
                         dim3((unsigned)a.rows, a.rows >= 256 ? 1 : D / (32 * DG)), dim3(256), 0, st, a);
    } else if (a.tab.is64)
      hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 3, false, 0, FORM>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 2, false, 0, FORM>), grid, dim3(256), 0, st, a);
  } else
    hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 1, false, 0, FORM>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

// Whether packed rows at D = 64 take key tiles of 64 keys rather than 32: 180
// registers and two workgroups a CU against 128 and four, with half the
// barriers per key.  They win while fewer than three workgroups a CU are there
// to run (causal ones are uneven, so a few more), 32 keys with more, or where
// no sequence is longer than a few tiles.  16 heads, us at 64 / 32 keys: causal
// 1 x 1,024 17.6 / 20.8, 1 x 4,096 58 / 67, 3,000 and 2,500 50 / 56, 4 x 1,500
// 45 / 39, 16 x 256 14.7 / 13.6, eight of 512 to 4,096 152 / 139;
// bidirectional 3,000 and 12 x 50 60 / 66, 3,000 and 2,500 88 / 83, 16 x 200
// 12.8 / 12.2.
bool few_workgroups(const AttnArgs& a, int64_t nseq, int64_t max_len) {
  return max_len > 256 && (a.T / (32 * (4 / a.gh)) + nseq) * (a.Hq / a.gh) <= (a.causal ? 736 : 672);
}
template <typename T, int DQ, AttnForm FORM = kPlain>
hipError_t launch_prefill_64(const AttnArgs& a, int64_t nseq, int64_t max_len, hipStream_t st) {
  return few_workgroups(a, nseq, max_len) ? launch_prefill_t<T, 64, 64, false, DQ, FORM>(a, nseq, max_len, st)
                                          : launch_prefill_t<T, 64, 32, false, DQ, FORM>(a, nseq, max_len, st);
}

// Whether a paged prefill over at most `cap` keys per sequence runs split, and
// with how many workgroups for the rows' further pieces (0: not split).  The
// host does not see the context lengths, so it prices the batch as if its rows
// held half the table's capacity on average and the last row to start all of
// it: per workgroup slot rows n / slots pieces of kFixed + nt / 2n steps, the
// last piece's nt / n, and for n > 1 the combine (its launch, and the partials'
// traffic).  The pieces' length is the device's choice, from the lengths
// themselves (split_tiles); what a table wider than its contexts costs is the
// extra workgroups, which find nothing to do, and the combine's launch.  So there
// are no more of them than kMaxExtra, or one per row.
// Not split from about 2,000 rows on (16 prompts of 1,200 tokens over 16
// heads): there the rows themselves fill the chip evenly.
struct PrefillSplit {
  int64_t rows, extra;
};
PrefillSplit prefill_split(int64_t T, int64_t nseq, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap) {
  constexpr double kSlots = 256, kFixed = 10, kCombine = 6, kPiece = 0.03;
  constexpr int64_t kMaxSplits = 64, kMaxFloats = int64_t(1) << 27;  // partials of at most 512 MiB
  PrefillSplit r{0, 0};
  if (T <= 0 || nseq <= 0 || Hkv <= 0 || cap <= 0) return r;
  const int gh = heads_per_group((int)(Hq / Hkv));
  constexpr int BN = 32;
  r.rows = (T / (32 * (4 / gh)) + nseq) * (Hq / gh);
  const int64_t nt = (cap + BN - 1) / BN;
  const double slots = D == 256 ? kSlots : 2 * kSlots;  // D <= 128: two workgroups fit a CU
  const int64_t kMaxExtra = D == 256 ? 1280 : 3584;
  const int64_t per_piece = 4 * (32 * D + 128);
  double best = 0;
  int64_t splits = 1;
  for (int64_t n = 1; n <= kMaxSplits; ++n) {
    if (n > 1 && (nt / n < 8 || r.rows * n * per_piece > kMaxFloats)) break;
    const double step = (double)nt / n;
    const double t = r.rows * n / slots * (kFixed + 0.5 * step) + step +
                     (n > 1 ? kCombine + kPiece * r.rows * n * D / 256 : 0);
    if (n == 1) {
      best = 0.9 * t;  // (a split has to win clearly)
    } else if (t < best) {
      best = t;
      splits = n;
    }
  }
  r.extra = r.rows * std::min(splits - 1, std::max<int64_t>(kMaxExtra / r.rows, 1));
  return r;
}

AttnArgs varlen_args(const gdn_tensor* q, const gdn_tensor* k, const gdn_tensor* v, const gdn_tensor* cu,
                     gdn_tensor* out, float scale, int causal) {
  AttnArgs a{};
  a.q = q->data;
  a.q_st = q->stride[0];
  a.q_sh = q->stride[1];
  a.k = kv_source(k, false);
  a.v = kv_source(v, false);
  a.o = out->data;
  a.o_st = out->stride[0];
  a.o_sh = out->stride[1];
  a.cu = cu->data;
  a.cu64 = cu->dtype == GDN_DTYPE_I64;
  a.T = q->shape[0];
  a.nseq = cu->shape[0] - 1;
  a.Hq = (int32_t)q->shape[1];
  a.dim = (int32_t)q->shape[2];
  a.Hkv = (int32_t)k->shape[1];
  a.gh = heads_per_group(a.Hq / a.Hkv);
  a.c = scale * kLog2e;
  a.causal = causal != 0;
  return a;
}

// workspace: of the split pieces, or null
AttnArgs paged_args(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc, const gdn_tensor* tab,
                    const gdn_tensor* ctx, const gdn_tensor* cu, gdn_tensor* out, float* workspace, float scale) {
  AttnArgs a{};
  if (workspace) {
    const PrefillSplit sp = prefill_split(q->shape[0], cu->shape[0] - 1, q->shape[1], kc->shape[2], q->shape[2],
                                          tab->shape[1] * kc->shape[1]);
    a.rows = sp.rows;
    a.extra = (int32_t)sp.extra;
    a.part = workspace;
  }
  a.q = q->data;
  a.q_st = q->stride[0];
  a.q_sh = q->stride[1];
  a.k = kv_source(kc, true);
  a.v = kv_source(vc, true);
  a.o = out->data;
  a.o_st = out->stride[0];
  a.o_sh = out->stride[1];
  a.cu = cu->data;
  a.cu64 = cu->dtype == GDN_DTYPE_I64;
  a.ctx = ctx->data;
  a.ctx64 = ctx->dtype == GDN_DTYPE_I64;
  a.tab = paged_table(tab, kc);
  a.T = q->shape[0];
  a.nseq = cu->shape[0] - 1;
  a.Hq = (int32_t)q->shape[1];
  a.dim = (int32_t)q->shape[2];
  a.Hkv = (int32_t)kc->shape[2];
  a.gh = heads_per_group(a.Hq / a.Hkv);
  a.c = scale * kLog2e;
  a.causal = true;
  return a;
}

}  // namespace

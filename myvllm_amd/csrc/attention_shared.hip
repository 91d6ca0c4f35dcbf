// Paged decode of sequences that begin with the same keys: the softmax over
// all keys of a sequence is merged from the one over the shared keys and the one
// over its own, (O, m, l) each: m = max, l = sum l_i 2^(m_i - m), O likewise.
//
// Three launches.  A plan, from the lengths on the device: one workgroup.  Then,
// in one grid, the shared keys through the prefill kernel (attention_prefill.h,
// kShared), the queries of a group, sequences x heads of a kv head, being the
// rows of its MFMA tile, so that the group's K and V are read once per 128 of
// them instead of once per sequence; and each sequence's own keys, a wave at a
// time (attention_own.h), on the workgroups beside them: the one is bound by MFMA
// and LDS, the other by HBM.  The third merges their unnormalised pieces.  256
// sequences of 16 / 2 heads of 256, 16,384 shared keys and 128 to 2,048 of their
// own (565 MB, 73 GFLOP): 8 + 174 + 9 us, 178 in a row;
// 64 behind 8,192 (89 MB) 6 + 30 + 7, 43; 4 behind 1,000 6 + 11 + 6, 23.  With the
// plan worked out by every workgroup and the own keys in a launch of their own
// 243, 69 and 33.
#include "attention_decode.h"
#include "attention_prefill.h"

namespace {

constexpr int kSharedTile = 32;  // keys of a tile of the prefill kernel
template <int D> constexpr int kSharedSlots = D == 256 ? 256 : D == 128 ? 512 : 768;  // workgroups that run at once
constexpr int kQueues = 32;         // of workgroups: 8 XCDs x 4 shader engines
constexpr int kMaxPieces11 = 2047;  // pieces of a row, held in 11 bits
constexpr int kOwnPrices = 3;

struct SharedGroup {
  int32_t keys, b0, rows;   // keys that are read once for all, first sequence, rows (sequences x heads of a kv head)
  int32_t rt, pieces;       // 128-row blocks, pieces of the keys
  int32_t slot, lead, pad;  // first slot of a kv head; the sequence through whose table the keys are read
};

struct SharedPlanArgs {
  const void *ctx, *groups, *lens;
  bool ctx64, groups64, lens64;
  int32_t B, n, R, Hkv;  // n groups
  int64_t cap;
  int32_t slots, grid;    // slots of the partials; workgroups of the shared keys
  int32_t units, waves;  // of the own keys: units at most, waves of each
  int32_t* prices;
  int32_t* head;  // slots of a kv head, units of the own keys
  SharedSeq* seqs;
  SharedGroup* group;
  SharedWork* work;
};

// Sequences and keys of group g.  The keys are taken in whole 16-key steps, so
// that each sequence's own begin at one; a group of one sequence shares nothing.
GDN_DEVICE SharedGroup shared_group(const SharedPlanArgs& a, int64_t g) {
  SharedGroup r{};
  int64_t b0 = 0, b1 = a.B;
  const int64_t keys = load_index(a.lens, g, a.lens64);
  if (a.groups) {
    b0 = load_index(a.groups, g, a.groups64);
    b1 = load_index(a.groups, g + 1, a.groups64);
  }
  b0 = clamp64(b0, 0, a.B);
  b1 = clamp64(b1, b0, a.B);
  r.b0 = (int32_t)b0;
  r.rows = (int32_t)(b1 - b0) * a.R;
  r.keys = b1 - b0 > 1 ? (int32_t)(clamp64(keys, 0, a.cap) & ~int64_t(15)) : 0;
  r.rt = r.keys > 0 ? (r.rows + 127) >> 7 : 0;
  return r;
}
// The group that may hold sequence b: the last g with groups[g] <= b.
GDN_DEVICE int32_t shared_group_of(const SharedPlanArgs& a, int64_t b) {
  int32_t lo = 0, hi = a.n;
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) / 2;
    if (load_index(a.groups, mid, a.groups64) <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}
// The keys of sequence b that its group reads for it: all of the group's, or
// none where it is shorter than they are or in no group.
GDN_DEVICE int32_t shared_first(const SharedPlanArgs& a, int32_t b, int64_t L) {
  if (a.n < 1) return 0;
  const SharedGroup g = shared_group(a, shared_group_of(a, b));
  return b >= g.b0 && b - g.b0 < g.rows / a.R && L >= g.keys ? g.keys : 0;
}

// How the chip is shared out, by one wave: units of the own keys, and key tiles
// per piece of the shared ones (0: there are none).
// The own keys get the part of the workgroups that their part of the work is, in
// key-tile steps of a workgroup (a price is 16 keys of one wave, four of which
// a workgroup reads in 1.2 steps), at least kOwnPrices to a unit.
// Consecutive workgroups go to 32 queues of 8 CUs in turn, so both parts are whole
// workgroups of every queue (one more than fits waits for a whole round: 64
// sequences with 64 own keys each 51 us where 40 is due).
// For the pieces lane i prices i + 1 times `mult` of the longest group, in 1/8 of
// a step: the end of the last one where F workgroups of a queue are free at once
// and `own` of them after the own keys' time, each piece taking kFixed steps and
// its tiles; the partials' traffic; the merge's chain.
struct SharedPlan {
  int32_t tiles, units;
};
template <int D>
GDN_DEVICE SharedPlan shared_tiles(const SharedPlanArgs& a, int prices) {
  constexpr int kSlots = kSharedSlots<D>, kDeep = kSlots / kQueues, kFixed = 8, kOwnFixed = 8;
  const int lane = threadIdx.x & 63;
  auto group = [&](int c) { return c + lane < a.n ? shared_group(a, c + lane) : SharedGroup{}; };
  int top = 0, rt = 0;
  float steps = 0.f;  // of the shared keys, per kv head
  for (int c = 0; c < a.n; c += 64) {
    const SharedGroup g = group(c);
    const int n = (g.keys + kSharedTile - 1) / kSharedTile;
    top = n > top ? n : top;
    rt += wave_sum(g.rt);
    steps += (float)g.rt * (float)n;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) steps += __shfl_xor(steps, d);
  steps *= (float)a.Hkv;
  const int most_units = prices / kOwnPrices < a.units ? prices / kOwnPrices : a.units;
  const int nmax = wave_top(top);
  if (nmax == 0) return {0, most_units > 1 ? most_units : 1};
  const float own_steps = 0.3f * (float)prices * (float)a.waves;
  int own = (int)(kDeep * own_steps / (own_steps + steps) + 0.5f);
  own = own > 1 ? own : 1;
  int units = kQueues * 4 * own / a.waves;
  units = units < most_units ? units : most_units;
  units = units > 1 ? units : 1;
  const int64_t least = (int64_t)rt * a.Hkv;
  const int mult = least < kSlots ? (kSlots + 64 * (int)least - 1) / (64 * (int)least) : 1, want = (lane + 1) * mult;
  int tiles = (nmax + want - 1) / want;
  tiles += tiles & 1;
  const float inv = __builtin_amdgcn_rcpf((float)tiles);
  int64_t wgs = 0;
  for (int c = 0; c < a.n; c += 64) {
    const SharedGroup g = group(c);
    const int m = a.n - c < 64 ? a.n - c : 64;
    for (int j = 0; j < m; ++j) {
      const int n = (__builtin_amdgcn_readlane(g.keys, j) + kSharedTile - 1) / kSharedTile;
      wgs += __mul24(__builtin_amdgcn_readlane(g.rt, j), n > 0 ? split_further(n, tiles, inv) + 1 : 0);
    }
  }
  wgs *= a.Hkv;
  const bool fits = wgs <= a.slots;
  const int x = fits ? ((int)wgs + kQueues - 1) / kQueues : 0;
  const float len = 8.f * (float)(kFixed + tiles);
  const int64_t busy = ((int64_t)units * a.waves + 4 * kQueues - 1) / (4 * kQueues);
  own = busy < kDeep ? (int)busy : kDeep;
  const int F = kDeep - own;
  const float t = 8.f * kOwnFixed + 9.6f * (float)prices / (float)units;
  // M: where k rounds of the free workgroups and j of the others make x
  int k = (x + kDeep - 1) / kDeep, j = 0;
  float M = len * (float)k + (F == 0 ? t : 0.f);
  while (F > 0 && __builtin_amdgcn_ballot_w64(k * F + j * own < x)) {
    if (k * F + j * own >= x) continue;
    const float next = (float)(k + 1) * len, next_own = t + (float)(j + 1) * len;
    M = next < next_own ? next : next_own;
    k += next <= next_own;
    j += next_own <= next;
  }
  const float cost = M + (float)x * (kQueues * D / 1400.f) + (float)(nmax / tiles) * 0.25f;
  const int c24 = fits && cost < 0x1p24f ? (int)cost : 1 << 24;
  // (the smallest, of equals the one with fewer pieces: the fewest, which always
  // fit, where all cost 2^24)
  const int best = 63 - (wave_top(((1 << 24) - c24) << 6 | (63 - lane)) & 63);
  return {__builtin_amdgcn_readlane(fits ? tiles : 0, best), units};
}

// Sum over the threads before this one; *all: over all NT.
template <int NT>
GDN_DEVICE int32_t block_exclusive(int32_t x, int32_t* wsum, int32_t* all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int32_t inc = wave_inclusive_scan_i32(x);
  __syncthreads();
  if (lane == 63) wsum[w] = inc;
  __syncthreads();
  int32_t base = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    base += i < w ? wsum[i] : 0;
    sum += wsum[i];
  }
  *all = sum;
  return base + inc - x;
}

// The plan: the price prefix of the own keys (as attn_decode_prices_kernel's),
// the groups' pieces and slots, and what each sequence and workgroup reads.
// Consecutive workgroups go to the 8 XCDs in turn, so an eighth of the slots,
// ordered (kv head, group, piece, block), is dealt to each: the blocks over the
// same keys run on one XCD and read them from its L2.
template <int D, int NT>
__global__ __launch_bounds__(NT) void shared_plan_kernel(const SharedPlanArgs a) {
  __shared__ int32_t wsum[NT / 64], tiles_lds;
  const int tid = threadIdx.x, per = (a.B + NT - 1) / NT;
  auto price_of = [&](int32_t b) -> int32_t {
    if (b >= a.B) return 0;
    const int64_t L = clamp64(load_index(a.ctx, b, a.ctx64), 0, a.cap);
    const int32_t t = (int32_t)((L - shared_first(a, b, L) + 15) / 16);
    return t > 0 ? t + kOwnStartPrice : 0;
  };
  int32_t sum = 0, total;
  for (int i = 0; i < per; ++i) sum += price_of(tid * per + i);
  int32_t run = block_exclusive<NT>(sum, wsum, &total);
  for (int i = 0; i < per; ++i) {
    const int32_t b = tid * per + i;
    if (b >= a.B) break;
    a.prices[b] = run;
    run += per == 1 ? sum : price_of(b);
  }
  if (tid == 0) a.prices[a.B] = total;
  if (tid < 64) {
    const SharedPlan p = shared_tiles<D>(a, total);
    if (tid == 0) {
      tiles_lds = p.tiles;
      a.head[1] = p.units;
    }
  }
  __syncthreads();

  // groups: pieces, slots, and the first sequence that is as long as the shared
  // keys (a padding one may have no table)
  const int tiles = tiles_lds;
  const float inv = __builtin_amdgcn_rcpf((float)tiles);
  int32_t slots = 0;
  for (int32_t c = 0; c < a.n; c += NT) {
    SharedGroup g{};
    if (c + tid < a.n) {
      g = shared_group(a, c + tid);
      if (tiles > 0 && g.keys > 0) g.pieces = split_further((g.keys + kSharedTile - 1) / kSharedTile, tiles, inv) + 1;
      const int32_t nb = g.pieces > 0 ? g.rows / a.R : 0;
      g.lead = -1;
      for (int32_t b = 0; b < nb && g.lead < 0; b += 4) {
        bool ok[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ok[e] = load_index(a.ctx, g.b0 + (b + e < nb ? b + e : 0), a.ctx64) >= g.keys;
        g.lead = ok[0] ? b : ok[1] ? b + 1 : ok[2] ? b + 2 : ok[3] ? b + 3 : -1;
      }
      // (past the end the first sequence was looked at again: not long enough)
      if (g.lead >= 0) g.lead += g.b0;
    }
    int32_t all;
    const int32_t before = block_exclusive<NT>(g.rt * g.pieces, wsum, &all);
    g.slot = slots + before;
    if (c + tid < a.n) a.group[c + tid] = g;
    slots += all;
  }
  if (tid == 0) a.head[0] = slots;
  __syncthreads();

  for (int32_t b = tid; b < a.B; b += NT) {
    SharedSeq s{};
    if (a.n > 0) {
      const SharedGroup g = a.group[shared_group_of(a, b)];
      const int64_t L = clamp64(load_index(a.ctx, b, a.ctx64), 0, a.cap);
      const bool in = b >= g.b0 && b - g.b0 < g.rows / a.R && L >= g.keys;
      s = SharedSeq{in ? g.keys : 0, g.rt << 11 | (in ? g.pieces : 0), g.slot, (b - g.b0) * a.R};
    }
    a.seqs[b] = s;
  }
  const uint32_t all = (uint32_t)slots * a.Hkv, xcd = (all + 7) / 8;
  for (uint32_t id = tid; id < (uint32_t)a.grid; id += NT) {
    SharedWork k{};
    k.lead = -1;
    const uint32_t slot = (id & 7) * xcd + (id >> 3);
    if ((id >> 3) < xcd && slot < all) {
      k.kvh = (int32_t)(slot / (uint32_t)slots);
      const int32_t left = (int32_t)slot - k.kvh * slots;
      int32_t lo = 0, hi = a.n;  // the last group with slot <= left (one without slots has the next one's)
      while (hi - lo > 1) {
        const int32_t mid = (lo + hi) / 2;
        if (a.group[mid].slot <= left) lo = mid;
        else hi = mid;
      }
      const SharedGroup g = a.group[lo];
      const int32_t piece = (left - g.slot) / g.rt, end = (piece + 1) * tiles * kSharedTile;
      k = SharedWork{g.lead, g.b0, g.rows, 128 * (left - g.slot - piece * g.rt), piece * tiles,
                     end < g.keys ? end : g.keys, k.kvh, (int32_t)slot};
    }
    a.work[id] = k;
  }
}

// Merge of the pieces of 32 rows (sequence, head of a kv head) and 32 dims, laid
// out as the prefill kernel's accumulators: lane l has row l % 32 and 4 x 4 dims.
// The four waves take every fourth piece, the shared ones first, and merge
// through LDS.
template <typename T, int D>
__global__ __launch_bounds__(256) void shared_decode_combine_kernel(const SharedAttnArgs a) {
  typedef typename Mma<T>::v4 v4;
  __shared__ float part[4][18][64];
  const DecodeArgs& d = a.own;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = a.Hq / a.Hkv, kvh = blockIdx.z, hh = lane >> 5, dim0 = 32 * blockIdx.y;
  const uint32_t nrows = (uint32_t)a.T * R, row = blockIdx.x * 32 + (lane & 31);
  const bool valid = row < nrows;
  const uint32_t b = (valid ? row : 0u) / (uint32_t)R, h = (valid ? row : 0u) - b * R;
  const int head = kvh * R + (int)h;
  const SharedSeq q = d.seqs[b];
  const int64_t Pt = d.prices[d.B], qb = d.prices[b], qn = d.prices[b + 1], U = d.head[1];
  // shared pieces: np of them, rt slots apart
  const int np = valid ? q.pieces & kMaxPieces11 : 0, rt = q.pieces >> 11, r = q.row + (int)h;
  const int64_t first = (int64_t)kvh * d.head[0] + q.slot + (r >> 7);
  const float* const mine = a.part + prefill_part_wave<D>() * ((r >> 5) & 3);
  const int pl = (r & 31) + 32 * hh;  // the row's lane there
  // own pieces: units u0 .. u0 + ns - 1
  int64_t u0 = 0;
  int ns = 0;
  if (valid && qn > qb) {
    u0 = ((qb + kOwnStartPrice + 1) * U - 1) / Pt;
    ns = (int)((qn * U - 1) / Pt - u0) + 1;
  }
  const bool all_units = Pt >= U;  // every unit has a price range, and a piece

  f32x4 acc[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) acc[g] = f32x4{0.f, 0.f, 0.f, 0.f};
  float mx = -INFINITY, l = 0.f;
  const int most = wave_top(np + ns);
#pragma unroll 2
  for (int i = w; i < most; i += 4) {
    const int64_t u = u0 + i - np;
    const bool own = i >= np;
    if (i >= np + ns || (own && !all_units && (u + 1) * Pt / U <= u * Pt / U)) continue;
    const float* pp = own ? d.part + ((b + u) * d.Hq + head) * (int64_t)(D + 4)
                          : mine + (first + (int64_t)i * rt) * prefill_part_floats<D>();
    const float m = pp[own ? D : 32 * D + pl], lp = pp[own ? D + 1 : 32 * D + 64 + pl];
    const float* po = pp + (own ? dim0 + 4 * hh : 32 * dim0 + 4 * pl);
    f32x4 o[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) o[g] = *reinterpret_cast<const f32x4*>(po + (own ? 8 : 256) * g);
    const float top = fmaxf(mx, m);
    const float was = mx == -INFINITY ? 0.f : exp2_fast(mx - top), now = m == -INFINITY ? 0.f : exp2_fast(m - top);
    mx = top;
    l = l * was + lp * now;
#pragma unroll
    for (int g = 0; g < 4; ++g) acc[g] = acc[g] * was + o[g] * now;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) part[w][e][lane] = acc[e >> 2][e & 3];
  part[w][16][lane] = mx;
  part[w][17][lane] = l;
  __syncthreads();
  // wave w merges dims 8 w + 4 hh .. + 3
  float top = part[0][16][lane];
#pragma unroll
  for (int i = 1; i < 4; ++i) top = fmaxf(top, part[i][16][lane]);
  float lt = 0.f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float m = part[i][16][lane], s = m == -INFINITY ? 0.f : exp2_fast(m - top);
    lt += part[i][17][lane] * s;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += part[i][4 * w + e][lane] * s;
  }
  const float inv = lt > 0.f ? 1.f / lt : 0.f;
  v4 ov;
#pragma unroll
  for (int e = 0; e < 4; ++e) ov[e] = (T)(o[e] * inv);
  if (valid)
    *reinterpret_cast<v4*>(reinterpret_cast<T*>(a.o) + b * a.o_st + (int64_t)head * a.o_sh + dim0 + 8 * w + 4 * hh) =
        ov;
}

// The workspace, in floats: the decode's, the plan, the shared pieces' partials.
// Workgroups that the shared keys may take: one per 128 rows of a group and kv
// head, however few of them a small group has; in pieces up to four times as many
// or one round of the chip, the pieces within 512 MiB of partials.  So many groups
// cost memory: 256 sequences of 16 / 2 heads of 256 in one group 43 MB, in pairs
// 162; 4,096 of 64 / 8 of 128 710 MB and 1.4 GB.
// The own keys are dealt over at most 512 waves' units with the heads (half the
// chip at D = 256, which reads at HBM's rate), and one per four sequences at least,
// which it takes a while to begin with.
struct SharedSpace {
  int64_t units, slots, grid, prices, head, seqs, group, work, part, all;
};
SharedSpace shared_space(int64_t B, int64_t n, int64_t Hq, int64_t Hkv, int64_t D) {
  SharedSpace s{};
  s.units = std::max(std::max<int64_t>(512 / (Hkv * ((Hq / Hkv + 15) / 16)), 1), (B + 3) / 4);
  const int64_t most = std::min(n, B / 2);  // (groups of two sequences at least)
  const int64_t base = Hkv * (B * (Hq / Hkv) / 128 + most), chip = D == 256 ? 256 : D == 128 ? 512 : 768;
  const int64_t fit = (int64_t(1) << 27) / (4 * (32 * D + 128));
  s.slots = most > 0 ? std::max(base, std::min(std::max(4 * base, chip), fit)) : 0;
  s.grid = (s.slots + 7) / 8 * 8;
  s.prices = (B + s.units) * Hq * (D + 4);
  s.head = s.prices + (B + 1 + 3) / 4 * 4;
  s.seqs = s.head + 4;
  s.group = s.seqs + B * 4;
  s.work = s.group + n * 8;
  s.part = s.work + s.grid * 8;
  s.all = s.part + s.slots * 4 * (32 * D + 128);
  return s;
}

template <typename T, int D>
hipError_t launch_shared(const SharedAttnArgs& a, const SharedPlanArgs& p, hipStream_t st) {
  constexpr int BN = kSharedTile;
  if (p.B <= 256)
    shared_plan_kernel<D, 256><<<dim3(1), dim3(256), 0, st>>>(p);
  else
    shared_plan_kernel<D, 1024><<<dim3(1), dim3(1024), 0, st>>>(p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid(a.own_wgs + (unsigned)p.grid);
  if (!whole_groups(a))
    hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 1, false, 0, kShared>), grid, dim3(256), 0, st, a);
  else if (a.tab.is64)
    hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 3, false, 0, kShared>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 2, false, 0, kShared>), grid, dim3(256), 0, st, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t rows = a.T * (a.Hq / a.Hkv);
  hipLaunchKernelGGL((shared_decode_combine_kernel<T, D>),
                     dim3((unsigned)((rows + 31) / 32), D / 32, (unsigned)a.Hkv), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

int64_t attn_shared_slots(int64_t B, int64_t groups, int64_t Hq, int64_t Hkv, int64_t D) {
  return shared_space(B, groups, Hq, Hkv, D).slots;
}

int32_t attn_shared_start_price() { return kOwnStartPrice; }

int64_t attn_shared_floats(int64_t B, int64_t groups, int64_t Hq, int64_t Hkv, int64_t D) {
  return shared_space(B, groups, Hq, Hkv, D).all;
}

// workspace: attn_shared_floats() of them
hipError_t attn_decode_shared_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc,
                                     const gdn_tensor* tab, const gdn_tensor* ctx, const gdn_tensor* lens,
                                     const gdn_tensor* groups, gdn_tensor* out, float* workspace, float scale,
                                     hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  const int64_t n = lens->shape[0], D = q->shape[2];
  const SharedSpace sp = shared_space(q->shape[0], n, q->shape[1], kc->shape[2], D);
  SharedAttnArgs a{};
  DecodeArgs& d = a.own;
  d = decode_args(q, kc, vc, tab, ctx, out, nullptr, 1, scale);
  d.units = (int32_t)sp.units;
  d.part = workspace;
  d.prices = reinterpret_cast<int32_t*>(workspace + sp.prices);
  d.head = reinterpret_cast<const int32_t*>(workspace + sp.head);
  d.seqs = reinterpret_cast<const SharedSeq*>(workspace + sp.seqs);
  a.q = d.q;
  a.q_st = d.q_ss;
  a.q_sh = d.q_sh;
  a.k = d.k;
  a.v = d.v;
  a.o = d.o;
  a.o_st = d.o_ss;
  a.o_sh = d.o_sh;
  a.ctx = d.ctx;
  a.ctx64 = d.ctx64;
  a.tab = d.tab;
  a.T = d.B;
  a.nseq = d.B;
  a.Hq = d.Hq;
  a.Hkv = d.Hkv;
  a.gh = 1;  // a wave per 32 rows
  a.dim = (int32_t)D;
  a.c = d.c;
  a.part = workspace + sp.part;
  a.work = reinterpret_cast<const SharedWork*>(workspace + sp.work);
  const int64_t waves = (int64_t)d.Hkv * ((d.Hq / d.Hkv + 15) / 16);
  a.own_wgs = (uint32_t)((sp.units * waves + 31) / 32 * 8);
  SharedPlanArgs p{};
  p.ctx = d.ctx;
  p.ctx64 = d.ctx64;
  p.lens = lens->data;
  p.lens64 = lens->dtype == GDN_DTYPE_I64;
  if (groups) {
    p.groups = groups->data;
    p.groups64 = groups->dtype == GDN_DTYPE_I64;
  }
  p.B = d.B;
  p.n = (int32_t)n;
  p.R = d.Hq / d.Hkv;
  p.Hkv = d.Hkv;
  p.cap = d.tab.cols * d.tab.page;
  p.slots = (int32_t)sp.slots;
  p.grid = (int32_t)sp.grid;
  p.prices = d.prices;
  p.units = d.units;
  p.waves = (int32_t)waves;
  p.head = reinterpret_cast<int32_t*>(workspace + sp.head);
  p.seqs = reinterpret_cast<SharedSeq*>(workspace + sp.seqs);
  p.group = reinterpret_cast<SharedGroup*>(workspace + sp.group);
  p.work = reinterpret_cast<SharedWork*>(workspace + sp.work);
  if (q->dtype == GDN_DTYPE_BF16) {
    if (D == 64) return launch_shared<bf16_t, 64>(a, p, st);
    if (D == 128) return launch_shared<bf16_t, 128>(a, p, st);
    return launch_shared<bf16_t, 256>(a, p, st);
  }
  if (D == 64) return launch_shared<f16_t, 64>(a, p, st);
  if (D == 128) return launch_shared<f16_t, 128>(a, p, st);
  return launch_shared<f16_t, 256>(a, p, st);
}

// The own keys of a shared decode: a wave per unit, kv head and 16 query heads,
// in the grid of the prefill kernel (attention_prefill.h, kShared).
#pragma once

#include "attention_decode.h"

namespace {

// The start of a piece (its lengths, queries, block ids and first rows, one after
// the other) in the price of a 16-key tile.
constexpr int32_t kOwnStartPrice = 4;

// LDS of one wave: the V rows of a 32-key step, with a 16-byte row skew.
template <typename T, int D> constexpr size_t own_lds_per_wave() { return (size_t)32 * (D + 8) * sizeof(T); }

// Unit u's pieces for kv head kvh and query heads 16 hg .. + 15 of it, each to its
// workspace slot b + u.  A CU reads 36 to 45 GB/s of HBM whatever its waves have
// in flight and however early they read their fragments (548 MB: 32 CUs 377 us,
// 64 205, 96 159), so what counts is that the waves are on many CUs and never
// idle.  As attn_decode_kernel, but made for one wave per SIMD,
// which is all that runs beside the shared keys' tiles at D = 256: 32 keys per
// step, two 16-key halves whose score MFMAs are independent and whose P V is one
// 16x16x32 MFMA per 16 dims (the k-slot 8 g + j of lane group g is key 4 g + j of
// the first half for j < 4, of the second for the others, for P and V alike),
// two steps in flight, the query fragments in registers, and the block ids of
// 64 tiles at a time in a lane each, a batch ahead.
template <typename T, int D, bool PAGE16>
GDN_DEVICE void attn_own_wave(const DecodeArgs& a, char* lds, int64_t u, int kvh, int hg) {
  typedef Mma<T> M;
  typedef typename M::v8 v8;
  typedef typename M::v4 v4;
  constexpr int LDV = D + 8;
  constexpr int NKS = D / 32, NDT = D / 16, CH = D / 8, NLD = 16 * CH / 64;
  T* const vs = reinterpret_cast<T*>(lds);
  const int lane = threadIdx.x & 63, grp = lane >> 4, j16 = lane & 15;
  const int R = a.Hq / a.Hkv, hcol = 16 * hg + j16;
  const bool hvalid = hcol < R;
  const int head = kvh * R + (hvalid ? hcol : 0);
  const int64_t cap = a.tab.cols * a.tab.page;
  const char* const kvk = a.k.base + kvh * a.k.sh;
  const char* const kvv = a.v.base + kvh * a.v.sh;
  const uint32_t kst = (uint32_t)a.k.st, vst = (uint32_t)a.v.st;
  const uint64_t ksb = (uint32_t)a.k.sb, vsb = (uint32_t)a.v.sb;
  const uint32_t gpp = PAGE16 ? (uint32_t)a.tab.page / 16u : 1u;
  const float c = a.c > 0.f ? a.c : (a.c < 0.f ? -a.c : 1.f);

  // the unit's prices [x0, x1), and the sequence that holds x0: the last b < B
  // with Q[b] <= x0, by a 64-ary search (one probe per lane and round)
  const int64_t Pt = load_index_scalar(a.prices, a.B, false), U = load_index_scalar(a.head, 1, false);
  if (u >= U) return;
  const int32_t x0 = (int32_t)(u * Pt / U), x1 = (int32_t)((u + 1) * Pt / U);
  if (x0 >= x1) return;
  int32_t lo = 0, hi = a.B;
  for (;;) {
    const int32_t step = (hi - lo + 63) / 64, i = lo + lane * step;
    const uint64_t le = __builtin_amdgcn_ballot_w64(i < hi && a.prices[i] <= x0);
    lo = __builtin_amdgcn_readfirstlane(lo + ((int32_t)__builtin_popcountll(le) - 1) * step);
    hi = lo + step < hi ? lo + step : hi;
    if (step == 1) break;
  }

  // keys [k_lo, k_hi) of sequence b, k_lo a multiple of 16
  auto piece = [&](int32_t b, uint32_t k_lo, uint32_t k_hi) __attribute__((always_inline)) {
    const int ntiles = (int)((k_hi - k_lo + 15) / 16);
    v8 qf[NKS];
    {
      const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.q_ss + (int64_t)head * a.q_sh + 8 * grp;
#pragma unroll
      for (int s = 0; s < NKS; ++s) {
        const v8 q = *reinterpret_cast<const v8*>(qp + 32 * s);  // (an invalid column's is dropped at the end)
        qf[s] = a.c > 0.f ? q : (a.c < 0.f ? -q : v8{});         // (c > 0 below)
      }
    }
    // tile t is 16-key group k_lo / 16 + t, in page g / gpp at slot 16 (g % gpp);
    // lane i holds tile 64 n + i's block id, -1 past the piece or for an entry
    // outside [0, num_blocks), and slot
    const uint32_t g0 = k_lo / 16u;
    auto load_ids = [&](int n, int32_t& id, uint32_t& slot) __attribute__((always_inline)) {
      const uint32_t t = 64u * n + lane, g = g0 + t, col = gpp == 1u ? g : g / gpp;
      const bool in = (int)t < ntiles;
      const int64_t blk = load_index(a.tab.table, b * a.tab.row_stride + (in ? col : 0u), a.tab.is64);
      id = in && blk >= 0 && blk < a.tab.num_blocks ? (int32_t)blk : -1;
      slot = gpp == 1u ? 0u : 16u * (g - col * gpp);
    };
    int32_t id = -1, id_next = -1;
    uint32_t slot = 0, slot_next = 0;
    if (PAGE16) {
      load_ids(0, id, slot);
      if (ntiles > 64) load_ids(1, id_next, slot_next);
    }
    // (tiles are loaded in order)
    auto load_tile = [&](int t, uint4* kd, uint4* vd) __attribute__((always_inline)) {
      if (PAGE16) {
        if ((t & 63) == 0 && t > 0) {
          id = id_next;
          slot = slot_next;
          if (t + 64 < ntiles) load_ids(t / 64 + 1, id_next, slot_next);
        }
        // one page per tile: descriptors of this kv head's rows of the page,
        // which end after the tile's valid rows (the others read as zero)
        const int32_t blk = __builtin_amdgcn_readlane(id, t & 63);
        const uint32_t r0 = gpp == 1u ? 0u : (uint32_t)__builtin_amdgcn_readlane((int)slot, t & 63);
        const int32_t nv = t < ntiles ? (int32_t)(k_hi - (k_lo + 16u * t)) : 0;
        const uint32_t ends = blk < 0 ? 0u : r0 + (uint32_t)(nv < 16 ? nv : 16);
        const uint64_t bb = blk < 0 ? 0u : (uint32_t)blk;
        const bool none = blk < 0 || nv <= 0;
        const __amdgpu_buffer_rsrc_t rk =
            __builtin_amdgcn_make_buffer_rsrc((void*)(kvk + bb * ksb), 0, none ? 0u : ends * kst, 0x00020000);
        const __amdgpu_buffer_rsrc_t rv =
            __builtin_amdgcn_make_buffer_rsrc((void*)(kvv + bb * vsb), 0, none ? 0u : ends * vst, 0x00020000);
        const uint32_t ko = (r0 + (uint32_t)j16) * kst + 16u * grp;
#pragma unroll
        for (int s = 0; s < NKS; ++s)
          kd[s] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk, ko + 64u * s, 0, 0));
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
          const uint32_t cc = lane + 64 * i, row = cc / CH, ch = cc % CH;
          vd[i] =
              __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rv, (r0 + row) * vst + 16u * ch, 0, 0));
        }
      } else {
        const int64_t j0 = (int64_t)k_lo + 16 * (int64_t)t;
        const char* pk = j0 + j16 < k_hi ? kv_row<true>(a.k, a.tab, b, 0, j0 + j16, kvh) : nullptr;
#pragma unroll
        for (int s = 0; s < NKS; ++s)
          kd[s] = pk ? *reinterpret_cast<const uint4*>(pk + 2 * (32 * s + 8 * grp)) : uint4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
          const int cc = lane + 64 * i, row = cc / CH, ch = cc % CH;
          const char* pv = j0 + row < k_hi ? kv_row<true>(a.v, a.tab, b, 0, j0 + row, kvh) : nullptr;
          vd[i] = pv ? *reinterpret_cast<const uint4*>(pv + 16 * ch) : uint4{0, 0, 0, 0};
        }
      }
    };

    f32x4 oacc[NDT];
#pragma unroll
    for (int d = 0; d < NDT; ++d) oacc[d] = f32x4{};
    float m_used = -INFINITY, lsum = 0.f, nb = 0.f;  // (as in the decode kernel)
    // first half of a step, after which its registers are free: V to LDS (the
    // step before's reads were issued earlier by this wave, and LDS operations
    // of a wave complete in order), scores
    auto scores = [&](const uint4 (*kd)[NKS], const uint4 (*vd)[NLD], f32x4* s) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
          const int cc = lane + 64 * i, row = cc / CH, ch = cc % CH;
          *reinterpret_cast<uint4*>(&vs[(16 * h + row) * LDV + 8 * ch]) = vd[h][i];
        }
      s[0] = s[1] = f32x4{};
#pragma unroll
      for (int k = 0; k < NKS; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[h] = M::m16k32(__builtin_bit_cast(v8, kd[h][k]), qf[k], s[h]);
    };
    auto accumulate = [&](int t, f32x4* s) __attribute__((always_inline)) {
      const uint32_t left = t < ntiles ? k_hi - (k_lo + 16u * t) : 0u;  // keys from the step's first on
      if (left < 32u) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16u * h + 4u * grp + r >= left) s[h][r] = -INFINITY;
      }
      float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
      mx = fmaxf(mx, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      if (__builtin_amdgcn_ballot_w64(mx * c > m_used + 8.f) != 0) {
        float mg = fmaxf(mx, __shfl_xor(mx, 16));
        mg = fmaxf(mg, __shfl_xor(mg, 32));
        const float mn = fmaxf(m_used, mg * c);
        const float alpha = mn == -INFINITY ? 1.f : exp2_fast(m_used - mn);
#pragma unroll
        for (int d = 0; d < NDT; ++d) oacc[d] *= alpha;
        lsum *= alpha;
        m_used = mn;
        nb = mn == -INFINITY ? 0.f : -mn;
      }
      v8 pf;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = exp2_fast(__builtin_fmaf(s[h][r], c, nb));
          lsum += p;
          pf[4 * h + r] = (T)p;
        }
      const T* vp = vs + (4 * grp + (j16 >> 2)) * LDV + 4 * (j16 & 3);
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        const v4 x = tr4<v4>(vp + 16 * d), y = tr4<v4>(vp + 16 * d + 16 * LDV);
        oacc[d] = M::m16k32(v8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, pf, oacc[d]);
      }
    };

    uint4 kA[2][NKS], kB[2][NKS], vA[2][NLD], vB[2][NLD];
    load_tile(0, kA[0], vA[0]);
    load_tile(1, kA[1], vA[1]);
    load_tile(2, kB[0], vB[0]);
    load_tile(3, kB[1], vB[1]);
    for (int t = 0; t < ntiles; t += 4) {
      f32x4 s[2];
      scores(kA, vA, s);
      load_tile(t + 4, kA[0], vA[0]);
      load_tile(t + 5, kA[1], vA[1]);
      accumulate(t, s);
      scores(kB, vB, s);
      load_tile(t + 6, kB[0], vB[0]);
      load_tile(t + 7, kB[1], vB[1]);
      accumulate(t + 2, s);
    }

    float lt = lsum + __shfl_xor(lsum, 16);
    lt += __shfl_xor(lt, 32);
    if (!hvalid) return;
    float* pp = a.part + ((b + u) * a.Hq + head) * (int64_t)(D + 4);
#pragma unroll
    for (int d = 0; d < NDT; ++d) *reinterpret_cast<f32x4*>(pp + 16 * d + 4 * grp) = oacc[d];
    if (grp == 0) {
      pp[D] = m_used;
      pp[D + 1] = lt;
    }
  };

  for (int32_t b = lo; b < a.B; ++b) {
    const int32_t qb = (int32_t)load_index_scalar(a.prices, b, false);
    if (qb >= x1) break;
    const int32_t L = (int32_t)clamp64(load_index(a.ctx, b, a.ctx64), 0, cap), first = a.seqs[b].first;
    const int32_t tb = (L - first + 15) / 16;  // its tiles, at prices [qb + start, ...)
    const int32_t r0 = x0 - qb - kOwnStartPrice, r1 = x1 - qb - kOwnStartPrice;
    const int32_t t0 = r0 < 0 ? 0 : (r0 > tb ? tb : r0), t1 = r1 < 0 ? 0 : (r1 > tb ? tb : r1);
    if (t1 > t0) piece(b, first + 16 * t0, first + 16 * t1 < L ? first + 16 * t1 : L);
  }
}

}  // namespace

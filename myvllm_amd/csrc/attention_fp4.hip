// Attention over paged caches held in 4 bits (fp4.h): the decode kernel, and the
// launches of it and of the prefill (attention_prefill.h, kFp4).
//
// The codes become 16-bit numbers, exactly, in front of the matrix
// instructions, so the result is that of the 16-bit attention over the values that
// the codes stand for.  The scales of a page lie slot by slot for each 32 dims
// (blocks, heads, D / 32, page): one load gives a lane those of four keys.
//
// Bound: HBM in long batches, where each byte of codes and scales is read once: 256
// sequences of U[512, 16384] keys, 16 / 4 heads of 128 (1,106 MB) 205 us and 6 of the
// merge, 5.2 TB/s, 90 % of a streaming copy (by 16-bit caches 690); 64 of U[1024, 8192], 16 / 2
// of 256 (174 MB) 42.3 + 4.8, against 128.  There a start of 9 us shows, which a lone
// sequence takes almost whole (2,943 keys 9.4 + 4.9): instruction fetch, lengths, table,
// codes, the product's chain, the merge.  Heads of 64 dims reach 3.7 TB/s: a tile is 2 KB
// and its conversions and products the work of one of 4 KB.  The scaled products of
// 4-bit operands were not taken: their sums are short of fp32 (7e-5 of the summands'
// magnitudes).
#include "attention_decode.h"
#include "attention_prefill.h"

namespace {

constexpr int32_t kFp4StartPrice = 6;  // of a piece's start, in 16-key groups

// Whether v and its scales lie as k and its do.
template <typename A> bool alike(const A& a) {
  return a.k.sb == a.v.sb && a.k.st == a.v.st && a.ks.sb == a.vs.sb && a.ks.sh == a.vs.sh && a.ks.sd == a.vs.sd;
}

struct Fp4DecodeArgs : DecodeArgs {
  ScaleSource ks, vs;
  uint32_t page_inv;  // floor((2^32 - 1) / 16-key groups of a page)
  int32_t R, hgroups;  // query heads of a kv head, and their groups of 16
  // FEW: tokens of the sequences (offsets, their end, the most of one), and a slot's rows
  const void* cu;
  bool cu64;
  int64_t T;
  int32_t most, rows;
};

// Decode: a workgroup is four waves, of 4 / KS kv heads (and up to 16 query heads of
// each); the KS waves of a head take the 32-key tiles of a piece in turn.  Units,
// pieces and the merge over workgroups are the plain decode's (attention_decode.h).
//
// S^T = K Q^T: lane (c, g) holds dims [CB (4 i + g), + CB) of key c of a 16-key group,
// whole 16-byte loads (a scale each) whose dims the queries' fragments follow.
// O^T = V^T P^T: lane (c, g) holds dims [VE c, + VE) of the keys 4 g + 0..3 of both
// groups, which is where S^T leaves their probabilities, so V reaches the matrix
// instruction without LDS: two numbers of a dim pair at a time are turned into 16
// bits, and byte permutes pair them by keys.
//
// ONE: pages of 16 keys, so a 16-key group is a page and starts at its slot 0, and v's
// strides those of k.
// FEW: a few tokens of each sequence instead of one: the columns are the query heads
// of one token after the other, each with its own last key.  The grid and the slots hold
// the columns of `most` tokens; a sequence that has more of them all the same (the
// caller's number was too small, or is a captured graph's) is read once more for each
// further group of columns, by the workgroups of its first unit.
template <typename T, int D, int KS, bool ONE, bool FEW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attn_decode_fp4_kernel(
    const Fp4DecodeArgs a) {
  typedef Mma<T> M;
  typedef typename M::v8 v8;
  typedef typename M::v4 v4;
  constexpr int CB = D >= 128 ? 32 : 16;  // dims of one load of K
  constexpr int NI = D / (4 * CB);        // loads per key and lane
  constexpr int NQ = CB / 8;              // k-steps per load
  constexpr int VE = D / 16;              // dims of V per lane
  constexpr int VW = VE > 8 ? 2 : 1;      // their words
  constexpr int NT = 2;                   // tiles in flight
  constexpr int LDO = D + 4;
  __shared__ __align__(16) float ob[KS > 1 ? 4 * 16 * LDO : 4];
  __shared__ float ml[4][2][16];
  // FEW: of each wave, the first key whose value is NaN in each 32 dims among those that only
  // some columns see: a probability of 0 would not keep it from the others, so its
  // scale is cleared and the columns that see it get their NaN at the end
  __shared__ uint32_t nan_at[FEW ? 4 * (D / 32) : 1];

  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, grp = lane >> 4, part = wv % KS;
  const int64_t cap = a.tab.cols * a.tab.page;
  const int R = a.R, hgroups = a.hgroups, y = hgroups == 1 ? blockIdx.y : blockIdx.y / hgroups;
  const int kvh = y * (4 / KS) + wv / KS;
  int h0 = ((int)blockIdx.y - y * hgroups) * 16;  // the first column
  int most = FEW ? a.most : 0;                    // tokens whose columns are taken
  const char* const kbase = a.k.base + kvh * a.k.sh;
  const char* const vbase = a.v.base + kvh * a.v.sh;
  const uint8_t* const ksbase = a.ks.base + kvh * a.ks.sh;
  const uint8_t* const vsbase = a.vs.base + kvh * a.vs.sh;
  const uint64_t ksb = (uint32_t)a.k.sb, vsb = ONE ? ksb : (uint32_t)a.v.sb;  // (below 2^32, as all of them, checked by the entry)
  const uint64_t kssb = (uint32_t)a.ks.sb, vssb = ONE ? kssb : (uint32_t)a.vs.sb;
  const uint32_t kst = (uint32_t)a.k.st, vst = ONE ? kst : (uint32_t)a.v.st;
  const uint32_t ksd = (uint32_t)a.ks.sd, vsd = ONE ? ksd : (uint32_t)a.vs.sd;
  const float c = a.c > 0.f ? a.c : (a.c < 0.f ? -a.c : 1.f);
  const uint32_t qsign = a.c < 0.f ? 0x80008000u : 0u;
  const uint32_t gpp = (uint32_t)a.tab.page / 16u, nblk = (uint32_t)a.tab.num_blocks;  // (below 2^31)

  struct Tile {
    uint32_t k[2][NI][CB / 8], ks[2][NI];
    uint32_t v[8][VW], vs[2];
    bool named[2];
  };
  // this lane's place in a group of 16 keys: codes of K, of V, scales of V
  const uint32_t ko = c16 * kst + CB / 2 * grp, vso = VE * c16 / 32 * vsd + 4 * grp;
  uint32_t kso[NI], vo[4];
#pragma unroll
  for (int i = 0; i < NI; ++i) kso[i] = CB * (4 * i + grp) / 32 * ksd + c16;
#pragma unroll
  for (int e = 0; e < 4; ++e) vo[e] = (4 * grp + e) * vst + VE / 2 * c16;

  auto piece = [&](int64_t b_, int64_t lo_, int64_t hi_, int64_t slot_, int64_t) {
    // (the same in all lanes, which the compiler does not see through the lengths'
    // vector loads: descriptors made of it would be looped over)
    // this lane's column: query head cr of the kv head, token ci
    const int ci = FEW ? (int)((uint32_t)(h0 + c16) / (uint32_t)R) : 0, cr = h0 + c16 - ci * R;
    const int32_t b = __builtin_amdgcn_readfirstlane((int32_t)b_), slot = __builtin_amdgcn_readfirstlane((int32_t)slot_);
    const uint32_t k_lo = __builtin_amdgcn_readfirstlane((int32_t)lo_), k_hi = __builtin_amdgcn_readfirstlane((int32_t)hi_);
    // columns of the sequence, its first row of q and out, the keys that this lane's
    // column sees, and those that all of the group's see
    int cols = R;
    int64_t row0 = b;
    uint32_t lim = k_hi, lim0 = k_hi;
    if constexpr (FEW) {
      int64_t s0, s1;
      seq_range(a.cu, a.cu64, b, a.T, s0, s1);
      const int len = __builtin_amdgcn_readfirstlane((int32_t)(s1 - s0 < most ? s1 - s0 : most));
      cols = len * R;
      if (cols <= h0) return;
      row0 = s0;
      const int64_t off = load_index(a.ctx, b, a.ctx64) - (s1 - s0) + 1;  // keys that token 0 sees
      lim = (uint32_t)clamp64(off + ci, 0, k_hi);
      lim0 = __builtin_amdgcn_readfirstlane((int32_t)clamp64(off + (int)((uint32_t)h0 / (uint32_t)R), 0, k_hi));
    }
    const bool hvalid = h0 + c16 < cols;
    const uint32_t qkeep = hvalid && a.c != 0.f ? ~0u : 0u;
    // column h of the group: its row in a slot, and in out
    const int rows = FEW ? a.rows : a.Hq;
    auto slot_row = [&](int h) __attribute__((always_inline)) {
      const int i = FEW ? (int)((uint32_t)(h0 + h) / (uint32_t)R) : 0;
      return i * a.Hq + kvh * R + h0 + h - i * R;
    };
    auto out_row = [&](int h) __attribute__((always_inline)) {
      const int i = FEW ? (int)((uint32_t)(h0 + h) / (uint32_t)R) : 0;
      return reinterpret_cast<T*>(a.o) + (row0 + i) * a.o_ss + (int64_t)(kvh * R + h0 + h - i * R) * a.o_sh;
    };
    if constexpr (FEW) {
      if (lane < D / 32) nan_at[wv * (D / 32) + lane] = UINT32_MAX;
    }
    if (k_hi == 0) {  // no keys: zero rows (and no table column that could be read)
      constexpr int LR = D / 4;
      for (int h = part * (16 / KS) + lane / LR; h < (part + 1) * (16 / KS); h += 64 / LR)
        if (h0 + h < cols) *reinterpret_cast<v4*>(out_row(h) + 4 * (lane % LR)) = v4{};
      return;
    }
    const int ntiles = (int)((k_hi - k_lo + 31) / 32);
    v8 qf[NI][NQ];
    {
      const T* qp = reinterpret_cast<const T*>(a.q) + (row0 + (hvalid ? ci : 0)) * a.q_ss +
                    (int64_t)(kvh * R + (hvalid ? cr : 0)) * a.q_sh;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          // (a negative scale turns q's signs, a zero one clears q, as in the plain decode)
          uint4 x = *reinterpret_cast<const uint4*>(qp + CB * (4 * i + grp) + 8 * q);
          x.x = (x.x & qkeep) ^ qsign, x.y = (x.y & qkeep) ^ qsign, x.z = (x.z & qkeep) ^ qsign, x.w = (x.w & qkeep) ^ qsign;
          qf[i][q] = __builtin_bit_cast(v8, x);
        }
    }
    // 16-key group g of the sequence: its page's block, the slot in it, and whether the
    // table names one.  Groups past the piece stand for its last one (their keys are
    // masked), groups of foreign blocks for block 0 (their words become zero): every load is
    // inside the caches, and none is behind a branch.
    // (a table of 64-bit ids is read as pairs of words, one of 32-bit ids as each word
    // twice: no branch, so the lookups of several groups wait together)
    const uint32_t wide = a.tab.is64 ? 1u : 0u;
    const const_i32_ptr trow = __builtin_bit_cast(const_i32_ptr, a.tab.table) + ((b * a.tab.row_stride) << wide);
    const uint32_t g0 = k_lo / 16u, glast = (k_hi - 1u) / 16u;
    struct Group {
      uint32_t block, slot;
      bool named;
    };
    auto group_of = [&](uint32_t g) -> Group {
      g = g < glast ? g : glast;
      uint32_t col = g, rem = 0;
      if constexpr (!ONE) {
        col = (uint32_t)(((uint64_t)g * a.page_inv) >> 32), rem = g - col * gpp;  // (at most one short)
        if (rem >= gpp) ++col, rem -= gpp;
      }
      const uint32_t low = (uint32_t)trow[col << wide], high = (uint32_t)trow[(col << wide) + wide];
      const bool named = low < nblk && (!wide || high == 0u);
      return {named ? low : 0u, 16u * rem, named};
    };
    // (the offsets are made opaque where they are used: known to be the same in every
    // round they are widened ahead, and each address is then a 64-bit vector sum)
    auto at = [](const auto* base, uint32_t off) __attribute__((always_inline)) {
      asm("" : "+v"(off));
      return reinterpret_cast<const char*>(base) + off;
    };
    auto load = [&](const Group* gr, Tile& x) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t bb = gr[h].block;
        x.named[h] = gr[h].named;
        const char* kp = kbase + bb * ksb;
        const char* vp = vbase + bb * vsb;
        const uint8_t* ksp = ksbase + bb * kssb;
        const uint8_t* vsp = vsbase + bb * vssb;
        if constexpr (!ONE) {
          const uint32_t r0 = gr[h].slot;
          kp += r0 * kst, vp += r0 * vst, ksp += r0, vsp += r0;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          if constexpr (CB == 32) {
            const uint4 w = *reinterpret_cast<const uint4*>(at(kp, ko) + 64 * i);
            x.k[h][i][0] = w.x, x.k[h][i][1] = w.y, x.k[h][i][2] = w.z, x.k[h][i][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(at(kp, ko));
            x.k[h][i][0] = w.x, x.k[h][i][1] = w.y;
          }
          x.ks[h][i] = *reinterpret_cast<const uint8_t*>(at(ksp, kso[i]));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t* const w = x.v[4 * h + e];
          const char* const p = at(vp, vo[e]);
          if constexpr (VE == 16) {
            const uint2 y = *reinterpret_cast<const uint2*>(p);
            w[0] = y.x, w[1] = y.y;
          } else if constexpr (VE == 8) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
          } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
          }
        }
        x.vs[h] = *reinterpret_cast<const uint32_t*>(at(vsp, vso));
      }
    };

    f32x4 oacc[VE];
#pragma unroll
    for (int d = 0; d < VE; ++d) oacc[d] = f32x4{};
    float m_used = -INFINITY, lsum = 0.f, nb = 0.f;  // (as in the plain decode)

    auto compute = [&](int t, Tile& x) {
      if (!(x.named[0] && x.named[1])) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t keep = x.named[h] ? ~0u : 0u;
#pragma unroll
          for (int i = 0; i < NI; ++i) {
#pragma unroll
            for (int w = 0; w < CB / 8; ++w) x.k[h][i][w] &= keep;
            x.ks[h][i] &= keep;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int w = 0; w < VW; ++w) x.v[4 * h + e][w] &= keep;
          x.vs[h] &= keep;
        }
      }
      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4{};
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const float sc = fp4_scale(x.ks[h][i]);
#pragma unroll
          for (int q = 0; q < NQ; ++q)
            s[h] = M::m16k32(__builtin_bit_cast(v8, fp4_eight<T>(x.k[h][i][q], sc)), qf[i][q], s[h]);
        }
      }
      const uint32_t j0 = k_lo + 32u * (uint32_t)t;
      uint32_t vs[2] = {x.vs[0], x.vs[1]};
      if (j0 + 32u > lim0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t j = j0 + 16u * h + 4u * grp + r;
            if (j >= lim) s[h][r] = -INFINITY;
            if (j >= k_hi) vs[h] &= ~(255u << (8 * r));  // (a stale scale may stand for NaN)
          }
        if constexpr (FEW) {
          // (bytes of 255)
          auto full = [](uint32_t x) { return ((x & 0x7F7F7F7Fu) + 0x01010101u) & x & 0x80808080u; };
          if (__builtin_expect(__builtin_amdgcn_ballot_w64((full(vs[0]) | full(vs[1])) != 0) != 0, 0)) {
            const uint32_t l = lane_anew();
            uint32_t at = UINT32_MAX;
#pragma unroll
            for (int h = 1; h >= 0; --h) {
              const uint32_t j = j0 + 16u * h + 4u * (l >> 4);  // the word's first key
              const uint32_t all = lim0 > j ? lim0 - j : 0u;    // of its keys, those that all columns see
              const uint32_t some = all < 4u ? full(vs[h]) >> 7 & ~0u << (8 * all) : 0u;
              at = some != 0u ? j + __builtin_ctz(some) / 8 : at;
              vs[h] &= ~(255u * some);
            }
            __hip_atomic_fetch_min(&nan_at[wv * (D / 32) + VE * (l & 15u) / 32], at, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_WAVEFRONT);
          }
        }
      }
      float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
      mx = fmaxf(mx, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      if (__builtin_amdgcn_ballot_w64(mx * c > m_used + 8.f) != 0) {
        float mg = fmaxf(mx, __shfl_xor(mx, 16));
        mg = fmaxf(mg, __shfl_xor(mg, 32));
        const float mn = fmaxf(m_used, mg * c);
        const float alpha = mn == -INFINITY ? 1.f : exp2_fast(m_used - mn);
        if (__builtin_amdgcn_ballot_w64(m_used != -INFINITY) != 0) {  // (else nothing is summed yet)
#pragma unroll
          for (int d = 0; d < VE; ++d) oacc[d] *= alpha;
          lsum *= alpha;
        }
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
      // (a scale's byte is moved to the exponent; the conversion reads no other bits)
      float sc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        sc[e] = __builtin_bit_cast(float, (e & 3) == 3 ? vs[e >> 2] >> 1 : vs[e >> 2] << (23 - 8 * (e & 3)));
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        constexpr int NP = VE > 8 ? 4 : VE / 2;  // pairs of dims in a word
        uint32_t y[8][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t u = x.v[e][w];
          y[e][0] = Fp4<T>::template pair<0>(u, sc[e]);
          y[e][1] = Fp4<T>::template pair<1>(u, sc[e]);
          if constexpr (NP == 4) {
            y[e][2] = Fp4<T>::template pair<2>(u, sc[e]);
            y[e][3] = Fp4<T>::template pair<3>(u, sc[e]);
          }
        }
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const uint32_t sel = o ? 0x07060302u : 0x05040100u;
            const uint4 vf = {__builtin_amdgcn_perm(y[1][p], y[0][p], sel), __builtin_amdgcn_perm(y[3][p], y[2][p], sel),
                              __builtin_amdgcn_perm(y[5][p], y[4][p], sel), __builtin_amdgcn_perm(y[7][p], y[6][p], sel)};
            const int d = 8 * w + 2 * p + o;
            oacc[d] = M::m16k32(__builtin_bit_cast(v8, vf), pf, oacc[d]);
          }
      }
    };

    // NT tiles in flight, and the groups of the next one to load
    Tile x[NT];
    Group gr[2];
    auto groups = [&](int t) {
      gr[0] = group_of(g0 + 2u * (uint32_t)t);
      gr[1] = group_of(g0 + 2u * (uint32_t)t + 1u);
    };
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      groups(part + u * KS);
      load(gr, x[u]);
    }
    groups(part + NT * KS);
    for (int t = part; t < ntiles; t += NT * KS) {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        compute(t + u * KS, x[u]);
        load(gr, x[u]);
        groups(t + (u + 1 + NT) * KS);
      }
    }

    if constexpr (FEW) {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      const uint32_t l = lane_anew();
      const uint32_t* const at = nan_at + wv * (D / 32) + VE * 4 * (l >> 4) / 32;
      const uint32_t at0 = at[0], at1 = VE == 16 ? at[1] : at0;  // of this lane's rows 0, 1 and 2, 3
      if (__builtin_expect(__builtin_amdgcn_ballot_w64((at0 < at1 ? at0 : at1) < lim) != 0, 0)) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int d = 0; d < VE; ++d) oacc[d][r] = (r < 2 ? at0 : at1) < lim ? __builtin_nanf("") : oacc[d][r];
      }
    }
    float lt = lsum + __shfl_xor(lsum, 16);
    lt += __shfl_xor(lt, 32);
    if constexpr (KS == 1) {
      if (!hvalid) return;
      const float inv = lt > 0.f ? 1.f / lt : 0.f;
      float* const pp = a.part + ((int64_t)slot * rows + slot_row(c16)) * (D + 4);
      T* const op = out_row(c16);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VE; j += 4) {
          const int d = VE * (4 * grp + r) + j;
          const f32x4 o = {oacc[j][r], oacc[j + 1][r], oacc[j + 2][r], oacc[j + 3][r]};
          if (slot < 0) *reinterpret_cast<v4*>(op + d) = v4{(T)(o[0] * inv), (T)(o[1] * inv), (T)(o[2] * inv), (T)(o[3] * inv)};
          else *reinterpret_cast<f32x4*>(pp + d) = o;
        }
      if (slot >= 0 && grp == 0) {
        pp[D] = m_used;
        pp[D + 1] = lt;
      }
    } else {
      // the head's waves meet in LDS: maxima and sums, then O on the common base
      const int w0 = wv - part;  // the head's first wave
      __syncthreads();           // (the previous piece's rows have been read)
      if (grp == 0) {
        ml[wv][0][c16] = m_used;
        ml[wv][1][c16] = lt;
      }
      __syncthreads();
      float mt = ml[w0][0][c16];
#pragma unroll
      for (int p = 1; p < KS; ++p) mt = fmaxf(mt, ml[w0 + p][0][c16]);
      auto weight = [&](float m) { return m == -INFINITY ? 0.f : exp2_fast(m - mt); };
      float l = 0.f;
#pragma unroll
      for (int p = 0; p < KS; ++p) l += ml[w0 + p][1][c16] * weight(ml[w0 + p][0][c16]);
      const float f = weight(m_used) * (slot >= 0 ? 1.f : l > 0.f ? 1.f / l : 0.f);
      float* const mine = ob + (wv * 16 + c16) * LDO;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VE; j += 4)
          *reinterpret_cast<f32x4*>(mine + VE * (4 * grp + r) + j) =
              f32x4{oacc[j][r] * f, oacc[j + 1][r] * f, oacc[j + 2][r] * f, oacc[j + 3][r] * f};
      float* const pp = a.part + (int64_t)slot * rows * (D + 4);
      if (slot >= 0 && part == 0 && grp == 0 && hvalid) {
        float* const mp = pp + (int64_t)slot_row(c16) * (D + 4) + D;
        mp[0] = mt;
        mp[1] = l;
      }
      __syncthreads();
      constexpr int LR = D / 4;    // lanes per row
      constexpr int RW = 16 / KS;  // rows per wave
      static_assert(LR <= 64 && RW % (64 / LR) == 0, "rows of a wave");
#pragma unroll 1
      for (int i = 0; i < RW / (64 / LR); ++i) {
        const int h = part * RW + i * (64 / LR) + lane / LR, d = 4 * (lane % LR);
        if (h0 + h >= cols) break;
        f32x4 o = *reinterpret_cast<const f32x4*>(ob + (w0 * 16 + h) * LDO + d);
#pragma unroll
        for (int p = 1; p < KS; ++p) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(ob + ((w0 + p) * 16 + h) * LDO + d);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] += y[e];
        }
        if (slot < 0) *reinterpret_cast<v4*>(out_row(h) + d) = v4{(T)o[0], (T)o[1], (T)o[2], (T)o[3]};
        else *reinterpret_cast<f32x4*>(pp + (int64_t)slot_row(h) * (D + 4) + d) = o;
      }
    }
  };
  if constexpr (FEW) {
    decode_deal(a, cap, lane, wv == 0, piece, [&]() __attribute__((always_inline)) {
      if (blockIdx.x != 0) return false;
      // (the arguments once more, so that none is held for this in the loops before)
      typedef const Fp4DecodeArgs __attribute__((address_space(4))) * ArgsPtr;
      ArgsPtr args = (ArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();
      asm volatile("" : "+s"(args));
      const int64_t s = clamp64(load_index_scalar(args->cu, blockIdx.z, args->cu64), 0, args->T);
      const int64_t e = clamp64(load_index_scalar(args->cu, (int64_t)blockIdx.z + 1, args->cu64), s, args->T);
      h0 += most != INT32_MAX ? args->most * args->R : args->hgroups * 16;
      most = INT32_MAX;
      return h0 < (int)(e - s) * args->R;
    });
  } else {
    decode_deal(a, cap, lane, wv == 0, piece);
  }
}

// Kv heads of a decode workgroup: one, whose keys its four waves deal among them, for heads
// of 256 dims (a line of the cache a row), and for small batches, where a key split inside
// the workgroup costs less than one that goes through the merge (one sequence of 9,000
// keys, 16 / 4 heads of 128: 14.2 us, with a wave a head 17.0; 8 of 3,000: 12.8 and 15.9; but
// 12 of 9,000 28.8 and 22.2: rows counts sequences, kv heads and groups of 16 columns).
// Else four (or two, or one, as the heads divide), whose rows of a slot share lines (256
// sequences of U[512, 16384] keys, 4 of 128: 230 us, two heads a workgroup 255, one 370).
int fp4_heads(int64_t rows, int Hkv, int D) {
  int n = D == 256 || rows <= 32 ? 1 : 4;
  while (Hkv % n) n /= 2;
  return n;
}

// Merge of the pieces of one token and query head, and (the last kZeroBlocks
// workgroups) the rows of out that no sequence covers, which are zero.
constexpr int kZeroBlocks = 16;
template <typename T, int D>
__global__ __launch_bounds__(64) void attn_few_combine_kernel(const Fp4DecodeArgs a) {
  const int64_t all = (int64_t)a.B * a.rows, id = blockIdx.x;
  if (id >= all) {
    zero_uncovered_rows<(int)sizeof(T)>(a.o, a.o_ss, a.o_sh, a.Hq, D, a.cu, a.cu64, a.B, a.T, id - all, kZeroBlocks,
                                        threadIdx.x, 64);
    return;
  }
  const int64_t b = id / a.rows;
  const int row = (int)(id - b * a.rows), i = row / a.Hq;
  int64_t s0, s1;
  seq_range(a.cu, a.cu64, b, a.T, s0, s1);
  if (i >= s1 - s0) return;
  decode_combine<T, D>(a, b, row, a.rows,
                       reinterpret_cast<T*>(a.o) + (s0 + i) * a.o_ss + (int64_t)(row - i * a.Hq) * a.o_sh);
}

template <typename T, int D, bool ONE, bool FEW>
void launch_decode_fp4_waves(const Fp4DecodeArgs& a, int heads, dim3 grid, hipStream_t st) {
  if constexpr (D < 256) {
    if (heads == 4) return attn_decode_fp4_kernel<T, D, 1, ONE, FEW><<<grid, dim3(256), 0, st>>>(a);
    if (heads == 2) return attn_decode_fp4_kernel<T, D, 2, ONE, FEW><<<grid, dim3(256), 0, st>>>(a);
  }
  attn_decode_fp4_kernel<T, D, 4, ONE, FEW><<<grid, dim3(256), 0, st>>>(a);
}

template <typename T, int D, bool FEW>
hipError_t launch_decode_fp4(const Fp4DecodeArgs& a, hipStream_t st) {
  const int hgroups = a.hgroups, heads = fp4_heads((int64_t)a.B * a.Hkv * hgroups, a.Hkv, D);
  const dim3 grid((unsigned)(a.splits > 1 ? a.units : 1), (unsigned)(a.Hkv / heads * hgroups), (unsigned)a.B);
  if (a.splits > 1 && !a.prices_inline) {
    attn_decode_prices_kernel<<<dim3(1), dim3(1024), 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (a.tab.page == 16 && alike(a)) launch_decode_fp4_waves<T, D, true, FEW>(a, heads, grid, st);
  else launch_decode_fp4_waves<T, D, false, FEW>(a, heads, grid, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  if constexpr (FEW)
    attn_few_combine_kernel<T, D><<<dim3((unsigned)((int64_t)a.B * a.rows + kZeroBlocks)), dim3(64), 0, st>>>(a);
  else
    attn_decode_combine_kernel<T, D><<<dim3((unsigned)((int64_t)a.B * a.Hq)), dim3(64), 0, st>>>(a);
  return hipGetLastError();
}

template <typename T, int D, int PG>
hipError_t launch_prefill_fp4_tiles(const Fp4AttnArgs& a, int64_t nseq, hipStream_t st) {
  constexpr int BN = 32;
  // (the grids of the 16-bit caches, launch_prefill_t)
  const int64_t tiles = a.T / (32 * (4 / a.gh)) + nseq + 1;
  if (a.extra > 0) {
    const dim3 grid((unsigned)(a.rows + a.Hq / a.gh + a.extra));
    attn_prefill_kernel<T, D, BN, PG, true, 0, kFp4><<<grid, dim3(256), 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    constexpr int DG = D == 256 ? 2 : 1;
    attn_prefill_combine_kernel<T, D, BN, DG><<<dim3((unsigned)a.rows, a.rows >= 256 ? 1 : D / (32 * DG)), dim3(256), 0,
                                                st>>>(a);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)(tiles * (a.Hq / a.gh)));
  attn_prefill_kernel<T, D, BN, PG, false, 0, kFp4><<<grid, dim3(256), 0, st>>>(a);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_prefill_fp4(const Fp4AttnArgs& a, int64_t nseq, hipStream_t st) {
  if (nseq <= 0 || a.tab.num_blocks == 0) {
    // (without a block to read every row is zero: those of no sequence are all of them)
    zero_uncovered_rows_kernel<(int)sizeof(T)><<<dim3(64), dim3(256), 0, st>>>(
        a.o, a.o_st, a.o_sh, a.Hq, a.dim, a.cu, a.cu64, a.tab.num_blocks == 0 ? 0 : a.nseq, a.T);
    return hipGetLastError();
  }
  if (a.tab.is64) return launch_prefill_fp4_tiles<T, D, 3>(a, nseq, st);
  if (a.tab.page == 16 && alike(a)) return launch_prefill_fp4_tiles<T, D, 4>(a, nseq, st);
  return launch_prefill_fp4_tiles<T, D, 2>(a, nseq, st);
}

}  // namespace

int32_t attn_fp4_start_price() { return kFp4StartPrice; }

namespace {
template <bool FEW>
hipError_t decode_fp4(const Fp4DecodeArgs& a, int dtype, int D, hipStream_t st) {
  if (dtype == GDN_DTYPE_BF16) {
    if (D == 64) return launch_decode_fp4<bf16_t, 64, FEW>(a, st);
    if (D == 128) return launch_decode_fp4<bf16_t, 128, FEW>(a, st);
    return launch_decode_fp4<bf16_t, 256, FEW>(a, st);
  }
  if (D == 64) return launch_decode_fp4<f16_t, 64, FEW>(a, st);
  if (D == 128) return launch_decode_fp4<f16_t, 128, FEW>(a, st);
  return launch_decode_fp4<f16_t, 256, FEW>(a, st);
}

void set_fp4(Fp4DecodeArgs& a, const gdn_tensor* ks, const gdn_tensor* vs) {
  a.ks = scale_source(ks);
  a.vs = scale_source(vs);
  a.start = kFp4StartPrice;
  a.R = a.Hq / a.Hkv;
  a.hgroups = (a.R + 15) / 16;
  a.page_inv = 0xFFFFFFFFu / (uint32_t)(a.tab.page / 16);
  if (a.tab.num_blocks == 0) a.tab.cols = 0;  // (no page to read: lengths end at 0 keys)
}
}  // namespace

hipError_t attn_decode_fp4_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc,
                                  const gdn_tensor* ks, const gdn_tensor* vs, const gdn_tensor* tab,
                                  const gdn_tensor* ctx, gdn_tensor* out, float* workspace, int32_t splits, float scale,
                                  hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  Fp4DecodeArgs a{};
  static_cast<DecodeArgs&>(a) = decode_args(q, kc, vc, tab, ctx, out, workspace, splits, scale);
  set_fp4(a, ks, vs);
  return decode_fp4<false>(a, q->dtype, (int)q->shape[2], st);
}

// A few tokens (at most `most`) of each sequence by the decode's kernel, split
// (splits >= 2).
hipError_t attn_few_fp4_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc, const gdn_tensor* ks,
                               const gdn_tensor* vs, const gdn_tensor* tab, const gdn_tensor* ctx, const gdn_tensor* cu,
                               gdn_tensor* out, float* workspace, int32_t splits, int32_t most, float scale,
                               hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  Fp4DecodeArgs a{};
  static_cast<DecodeArgs&>(a) = decode_args(q, kc, vc, tab, ctx, out, workspace, splits, scale);
  // (those count q's rows as sequences)
  a.B = (int32_t)tab->shape[0];
  a.rows = most * a.Hq;
  a.unit_inv = 1.0 / ((double)a.B * a.units);
  a.prices = reinterpret_cast<int32_t*>(workspace + (int64_t)a.B * splits * a.rows * (q->shape[2] + 4));
  a.prices_inline = a.B <= 1024;
  set_fp4(a, ks, vs);
  a.hgroups = (int32_t)((most * a.R + 15) / 16);
  a.cu = cu->data;
  a.cu64 = cu->dtype == GDN_DTYPE_I64;
  a.T = q->shape[0];
  a.most = most;
  return decode_fp4<true>(a, q->dtype, (int)q->shape[2], st);
}

hipError_t attn_prefill_fp4_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc,
                                   const gdn_tensor* ks, const gdn_tensor* vs, const gdn_tensor* tab,
                                   const gdn_tensor* ctx, const gdn_tensor* cu, gdn_tensor* out, float* workspace,
                                   float scale, hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  Fp4AttnArgs a{};
  static_cast<AttnArgs&>(a) = paged_args(q, kc, vc, tab, ctx, cu, out, workspace, scale);
  a.ks = scale_source(ks);
  a.vs = scale_source(vs);
  const int D = (int)q->shape[2];
  const int64_t N = cu->shape[0] - 1;
  if (q->dtype == GDN_DTYPE_BF16) {
    if (D == 64) return launch_prefill_fp4<bf16_t, 64>(a, N, st);
    if (D == 128) return launch_prefill_fp4<bf16_t, 128>(a, N, st);
    return launch_prefill_fp4<bf16_t, 256>(a, N, st);
  }
  if (D == 64) return launch_prefill_fp4<f16_t, 64>(a, N, st);
  if (D == 128) return launch_prefill_fp4<f16_t, 128>(a, N, st);
  return launch_prefill_fp4<f16_t, 256>(a, N, st);
}

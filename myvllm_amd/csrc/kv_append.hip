// Append of new keys and values to a paged cache, with the position rotation
// of q and k on the way (gfx950).
//
// Token t of sequence n sits at position p = context_lens[n] - len_n + i and
// goes to slot p % page of block block_tables[n][p / page].  The first `rot`
// dims of q and k are turned by the angle of their frequency at p: with
// (a, b) = dims (j, j + rot / 2), or (2 j, 2 j + 1) when interleaved,
// (a, b) <- (a cos[p][j] - b sin[p][j], b cos[p][j] + a sin[p][j]) in fp32,
// rounded once.  The other dims and v are moved as they are.
//
// Bound: HBM, each row read once and written once.  A wave takes one token and
// kAppendRows x (1024 / D) of its rows (the q, k and v heads in turn); a lane
// takes 16 elements of a row, as two 16-byte pieces that hold whole pairs, and
// the same 16 dims in each of its rows, so the rotation's 8 cosines and sines
// are read once per lane.  The rows are loaded before the sequence lookup and
// the table reads that they do not depend on.  36,696 tokens of
// 16 / 2 heads of 256 (789 MB) 135 us, 5.8 TB/s, 97 % of a streaming copy; with
// 1, 2, 3, 5, 6 rows per lane 134, 138, 135, 141, 142.  Plain stores:
// non-temporal ones take 125 us, but the attention that reads the rows next
// takes 17 us longer.
//
// AXES: the rotation's positions are the caller's, one per token and axis (time,
// height and width of an image's patches), and every frequency turns by the
// position of its own axis: c[j] = cos[p[axis(j)]][j].  The axes of all
// frequencies are two bits each in the arguments; a lane reads the rows of the
// axes that its eight frequencies have.  17,653 tokens of 16 / 4 heads of 128, three axes
// (226 MB) 47 us, one axis of context_lens 42: the positions are one more load that the
// tables' rows wait for (all axes' rows at once, without the branch, 47).
// FP4: the caches hold codes and block scales (fp4.h) of the rows that the
// 16-bit cache would hold.  A block's 32 numbers lie in two to four lanes,
// wherever the rotation's pairs put them, so its largest magnitude is taken by an
// LDS maximum of the wave (30,447 tokens of 16 / 2 heads of 256, 608 MB, 105 us by itself, 5.8
// TB/s, 98 % of a streaming copy, 108 in turn with a read; the 16-bit cache 112; with three axes 121).  Keys are rotated in 64 bits there (products of a
// 16-bit and a 32-bit number are exact in them): next to a border between two
// codes the last bit of a fp32 sum would choose another one now and then.
#include "fp4.h"

namespace {

constexpr int kAppendRows = 3;  // rows in flight per lane

struct AppendArgs {
  const void *k, *v, *q;
  int64_t k_st, k_sh, v_st, v_sh, q_st, q_sh;  // element strides: token, head
  void *kc, *vc, *o;
  int64_t kc_sb, kc_st, kc_sh, vc_sb, vc_st, vc_sh, o_st, o_sh;
  const void *tab, *ctx, *cu;
  const float *cos, *sin;
  int64_t cos_st, sin_st;
  int64_t T, nseq, tab_st, cols, num_blocks, limit;  // limit: positions that have a place and an angle
  int32_t page, Hq, Hkv, rot, chunks;                // chunks: waves per token
  bool tab64, ctx64, cu64, interleaved;
};

// (apart: a launch of the plain form copies no more arguments than it needs)
struct AppendExArgs : AppendArgs {
  // AXES: positions (axes, T), their rows of cos and sin, and the axis of each
  // frequency, eight frequencies a 16-bit half
  const void* pos;
  int64_t pos_st, rows;
  uint32_t axes[8];
  int32_t naxes;
  bool pos64;
  // FP4: the caches' strides are in bytes
  ScaleSource ks, vs;
};

constexpr int kMaxAxes = 4;

// The sequence that holds token t, or -1: the last n with cu[n] <= t, by a
// 64-ary search (one probe per lane and round), if t < cu[n + 1].
GDN_DEVICE int64_t find_seq(const AppendArgs& a, int64_t t, int lane) {
  int64_t lo = 0, hi = a.nseq + 1;  // cu[lo] <= t throughout (or t is before them all)
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 63) / 64, i = lo + lane * step;
    const bool le = i < hi && load_index(a.cu, i, a.cu64) <= t;
    const int c = (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(le));
    if (c == 0) return -1;
    lo += (c - 1) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo < a.nseq ? lo : -1;
}

// A pair turned in fp64, rounded to fp32 and that to T (the compiler, which sees two
// roundings in a row, would round to odd first: other results next to a tie, and ten
// instructions more each).
template <typename T> struct Pair {
  T a, b;
};
template <typename T> GDN_DEVICE Pair<T> turn_exactly(T a, T b, float c, float s) {
  const double x = (float)a, y = (float)b, cd = c, sd = s;
  float p = (float)(x * cd - y * sd), q = (float)(y * cd + x * sd);
  asm("" : "+v"(p), "+v"(q));
  return {(T)p, (T)q};
}

template <typename T, int D, bool AXES = false, bool FP4 = false>
__global__ __launch_bounds__(256) void paged_kv_append_kernel(
    const std::conditional_t<AXES || FP4, AppendExArgs, AppendArgs> a) {
  typedef T v8 __attribute__((ext_vector_type(8)));
  constexpr int U = D / 16;    // lanes per row
  constexpr int RPI = 64 / U;  // rows per wave and step
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t id = blockIdx.x * 4 + w, tok = id / (uint32_t)a.chunks;  // (below 2^31, checked by the entry)
  const int64_t t = tok;
  if (t >= a.T) return;
  const int r0 = (int)(id - tok * a.chunks) * (kAppendRows * RPI) + lane / U;
  const int u = lane % U, nq = a.q ? a.Hq : 0, nrows = nq + 2 * a.Hkv;
  // this lane's two pieces of a row that is rotated: the partners of 8 pairs
  // (halves), or 16 dims in a row
  const bool turns = 16 * u < a.rot, halves = turns && !a.interleaved;
  const int e0 = halves ? 8 * u : 16 * u, e1 = halves ? 8 * u + a.rot / 2 : 16 * u + 8;
  v8 x[kAppendRows], y[kAppendRows];
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int r = r0 + i * RPI < nrows ? r0 + i * RPI : nrows - 1;
    const T* p = r < nq            ? reinterpret_cast<const T*>(a.q) + t * a.q_st + r * a.q_sh
                 : r < nq + a.Hkv ? reinterpret_cast<const T*>(a.k) + t * a.k_st + (r - nq) * a.k_sh
                                   : reinterpret_cast<const T*>(a.v) + t * a.v_st + (r - nq - a.Hkv) * a.v_sh;
    x[i] = *reinterpret_cast<const v8*>(p + e0);
    y[i] = *reinterpret_cast<const v8*>(p + e1);
  }

  int64_t n = t, pos = -1;
  if (a.cu) {
    n = find_seq(a, t, lane);
    if (n >= 0) {
      int64_t s, e;
      seq_range(a.cu, a.cu64, n, a.T, s, e);
      if (t < e) pos = load_index(a.ctx, n, a.ctx64) - e + t;
    }
  } else {
    pos = load_index(a.ctx, n, a.ctx64) - 1;
  }
  bool placed = pos >= 0 && pos < a.limit;
  int64_t turns_by[AXES ? kMaxAxes : 1];
  if constexpr (AXES) {
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x) {
      turns_by[x] = x < a.naxes ? load_index(a.pos, x * a.pos_st + t, a.pos64) : 0;
      placed = placed && turns_by[x] >= 0 && turns_by[x] < a.rows;
    }
  }
  int64_t block = -1;
  int32_t slot = 0;
  if (placed) {
    const int64_t col = (uint32_t)pos / (uint32_t)a.page;  // (positions are below 2^31)
    slot = (int32_t)(pos - col * a.page);
    block = load_index(a.tab, n * a.tab_st + col, a.tab64);
    if (block >= a.num_blocks) block = -1;
  }
  float c[8], s[8];
  if (!AXES && turns && placed) {
    Vec8<float>::load(a.cos + pos * a.cos_st + 8 * u, c);
    Vec8<float>::load(a.sin + pos * a.sin_st + 8 * u, s);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = 1.f, s[j] = 0.f;
  }
  if constexpr (AXES) {
    if (turns && placed) {
      uint32_t of = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) of = u >> 1 == i ? a.axes[i] : of;
      of = u & 1 ? of >> 16 : of & 0xFFFFu;
#pragma unroll
      for (int x = 0; x < kMaxAxes; ++x) {
        // (bit 2 j: frequency j has axis x)
        const uint32_t same = ~(of ^ (0x5555u * (uint32_t)x)), mine = same & (same >> 1) & 0x5555u;
        if (x >= a.naxes || mine == 0) continue;
        float cx[8], sx[8];
        Vec8<float>::load(a.cos + turns_by[x] * a.cos_st + 8 * u, cx);
        Vec8<float>::load(a.sin + turns_by[x] * a.sin_st + 8 * u, sx);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          c[j] = mine >> (2 * j) & 1u ? cx[j] : c[j];
          s[j] = mine >> (2 * j) & 1u ? sx[j] : s[j];
        }
      }
    }
  }

  // (FP4: a largest magnitude per row in flight and block)
  __shared__ uint32_t tops[FP4 ? 4 * kAppendRows * 32 : 1];
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int r = r0 + i * RPI;
    if (r >= nrows) continue;
    if (turns && r < nq + a.Hkv) {
      if (FP4 && r >= nq) {
        if (a.interleaved) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Pair<T> p = turn_exactly(x[i][2 * j], x[i][2 * j + 1], c[j], s[j]);
            const Pair<T> q = turn_exactly(y[i][2 * j], y[i][2 * j + 1], c[j + 4], s[j + 4]);
            x[i][2 * j] = p.a, x[i][2 * j + 1] = p.b;
            y[i][2 * j] = q.a, y[i][2 * j + 1] = q.b;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const Pair<T> p = turn_exactly(x[i][j], y[i][j], c[j], s[j]);
            x[i][j] = p.a, y[i][j] = p.b;
          }
        }
      } else if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a0 = (float)x[i][2 * j], b0 = (float)x[i][2 * j + 1];
          const float a1 = (float)y[i][2 * j], b1 = (float)y[i][2 * j + 1];
          x[i][2 * j] = (T)(a0 * c[j] - b0 * s[j]);
          x[i][2 * j + 1] = (T)(b0 * c[j] + a0 * s[j]);
          y[i][2 * j] = (T)(a1 * c[j + 4] - b1 * s[j + 4]);
          y[i][2 * j + 1] = (T)(b1 * c[j + 4] + a1 * s[j + 4]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float p = (float)x[i][j], q = (float)y[i][j];
          x[i][j] = (T)(p * c[j] - q * s[j]);
          y[i][j] = (T)(q * c[j] + p * s[j]);
        }
      }
    }
    if constexpr (FP4) {
      if (r >= nq) {
        uint32_t* const top = tops + (w * kAppendRows + i) * 32 + lane / U * (D / 32);
        // (LDS operations of a wave complete in order; the lanes of a row, which all write
        // the zeros and take part in the maxima, meet between the steps)
        auto meet = []() __attribute__((always_inline)) {
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };
        top[e0 / 32] = 0u;
        top[e1 / 32] = 0u;
        meet();
        __hip_atomic_fetch_max(top + e0 / 32, top_of_eight(x[i]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
        __hip_atomic_fetch_max(top + e1 / 32, top_of_eight(y[i]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
        meet();
        if (block < 0) continue;
        const uint32_t s0 = fp4_scale_byte<T>(top[e0 / 32]), s1 = fp4_scale_byte<T>(top[e1 / 32]);
        const bool key = r < nq + a.Hkv;
        const int h = r - nq - (key ? 0 : a.Hkv);
        uint8_t* const p = reinterpret_cast<uint8_t*>(key ? a.kc : a.vc) + block * (key ? a.kc_sb : a.vc_sb) +
                           slot * (key ? a.kc_st : a.vc_st) + h * (key ? a.kc_sh : a.vc_sh);
        const uint32_t w0 = fp4_codes<T>(x[i], s0), w1 = fp4_codes<T>(y[i], s1);
        *reinterpret_cast<uint32_t*>(p + e0 / 2) = w0;
        *reinterpret_cast<uint32_t*>(p + e1 / 2) = w1;
        const ScaleSource& sc = key ? a.ks : a.vs;
        uint8_t* const q = sc.base + block * sc.sb + h * sc.sh + slot;
        if (e0 % 32 == 0) q[e0 / 32 * sc.sd] = (uint8_t)s0;
        if (e1 % 32 == 0) q[e1 / 32 * sc.sd] = (uint8_t)s1;
        continue;
      }
    }
    T* p;
    if (r < nq) {
      p = reinterpret_cast<T*>(a.o) + t * a.o_st + r * a.o_sh;
      if (!placed) x[i] = y[i] = v8{};
    } else {
      if (block < 0) continue;
      p = r < nq + a.Hkv
              ? reinterpret_cast<T*>(a.kc) + block * a.kc_sb + slot * a.kc_st + (r - nq) * a.kc_sh
              : reinterpret_cast<T*>(a.vc) + block * a.vc_sb + slot * a.vc_st + (r - nq - a.Hkv) * a.vc_sh;
    }
    *reinterpret_cast<v8*>(p + e0) = x[i];
    *reinterpret_cast<v8*>(p + e1) = y[i];
  }
}

// Keys and values of tokens read back from the caches, as the append found
// their places: one wave per kReadRows x (1024 / D) rows, k and v heads of a
// token in turn, a lane 16 dims of a row.  Rows without a place are zero, and
// so are those of a table entry outside [0, num_blocks).
//
// Bound: HBM, and the chain of offsets, length, table and codes: 30,447 tokens of 2 heads of
// 256 in 4 bits (79 MB) 18 us by itself, 22 in turn with the append, 13.5 at the copy's rate; by
// itself with 1, 4 and 8 rows a lane 18.8, 19.6 and 24.2, and 23.1 where each row waits for
// its own lookup.  From 16-bit caches (125 MB) 21.5, the copy's rate.
struct ReadArgs {
  AppendExArgs in;  // caches, tables, lengths; T, nseq, Hkv
  void *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
};

constexpr int kReadRows = 2;

template <typename T, int D, bool FP4>
__global__ __launch_bounds__(256) void paged_kv_read_kernel(const ReadArgs g) {
  const AppendExArgs& a = g.in;
  constexpr int U = D / 16, RPI = 64 / U;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t first = (blockIdx.x * 4 + w) * (kReadRows * RPI), per = 2 * (uint32_t)a.Hkv;  // (rows below 2^31)
  const uint32_t t0 = first / per;
  if (t0 >= a.T) return;
  // The rows' tokens and places, then their blocks, then their codes: loads of one
  // kind wait together.  As a rule all tokens of the wave are of one sequence.
  int64_t n0 = -1, s0 = 0, e0 = 0, off = 0;
  bool same = false;
  if (a.cu) {
    n0 = find_seq(a, t0, lane);
    if (n0 >= 0) {
      seq_range(a.cu, a.cu64, n0, a.T, s0, e0);
      off = load_index(a.ctx, n0, a.ctx64) - e0;
      same = (first + kReadRows * RPI - 1) / per < (uint64_t)e0;
    }
  }
  const int u = lane % U;
  uint4 x[kReadRows], y[kReadRows];
  uint32_t sc[kReadRows];
  int64_t n[kReadRows], pos[kReadRows], block[kReadRows];
  const int64_t nfirst = n0 < 0 ? 0 : n0;  // (tokens before the first sequence)
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const uint32_t t = (first + i * RPI + lane / U) / per;
    n[i] = same ? n0 : t;
    pos[i] = same ? off + t : -1;
    if (!a.cu && t < a.T) pos[i] = load_index(a.ctx, t, a.ctx64) - 1;
  }
  if (a.cu && !same && a.nseq > 0) {
#pragma unroll 1
    for (int i = 0; i < kReadRows; ++i) {
      const uint32_t t = (first + i * RPI + lane / U) / per;
      if (t >= a.T) break;
      int64_t m = nfirst, s, e;
      while (m < a.nseq - 1 && load_index(a.cu, m + 1, a.cu64) <= t) ++m;
      seq_range(a.cu, a.cu64, m, a.T, s, e);
      const int64_t p = t >= s && t < e ? load_index(a.ctx, m, a.ctx64) - e + t : -1;
#pragma unroll
      for (int k = 0; k < kReadRows; ++k)
        if (k == i) n[k] = m, pos[k] = p;
    }
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    block[i] = -1;
    if (pos[i] >= 0 && pos[i] < a.limit)
      block[i] = load_index(a.tab, n[i] * a.tab_st + (uint32_t)pos[i] / (uint32_t)a.page, a.tab64);
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const uint32_t row = first + i * RPI + lane / U, t = row / per, h2 = row - t * per;
    const bool key = h2 < (uint32_t)a.Hkv;
    const int64_t h = key ? h2 : h2 - a.Hkv;
    x[i] = y[i] = uint4{0, 0, 0, 0};
    sc[i] = 0;
    if (block[i] < 0 || block[i] >= a.num_blocks) continue;
    const int64_t slot = (uint32_t)pos[i] % (uint32_t)a.page, at = block[i];
    const char* p = key ? reinterpret_cast<const char*>(a.kc) + at * a.kc_sb + slot * a.kc_st + h * a.kc_sh
                        : reinterpret_cast<const char*>(a.vc) + at * a.vc_sb + slot * a.vc_st + h * a.vc_sh;
    if constexpr (FP4) {
      const uint2 c = *reinterpret_cast<const uint2*>(p + 8 * u);
      x[i].x = c.x;
      x[i].y = c.y;
      const ScaleSource& ss = key ? a.ks : a.vs;
      sc[i] = ss.base[at * ss.sb + h * ss.sh + (u / 2) * ss.sd + slot];
    } else {
      x[i] = *reinterpret_cast<const uint4*>(p + 32 * u);
      y[i] = *reinterpret_cast<const uint4*>(p + 32 * u + 16);
    }
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const uint32_t row = first + i * RPI + lane / U, t = row / per, h2 = row - t * per;
    if (t >= a.T) continue;
    const bool key = h2 < (uint32_t)a.Hkv;
    const int64_t h = key ? h2 : h2 - a.Hkv;
    T* p = key ? reinterpret_cast<T*>(g.k) + t * g.k_st + h * g.k_sh : reinterpret_cast<T*>(g.v) + t * g.v_st + h * g.v_sh;
    if constexpr (FP4) {
      const float s = fp4_scale(sc[i]);
      y[i] = fp4_eight<T>(x[i].y, s);
      x[i] = fp4_eight<T>(x[i].x, s);
    }
    *reinterpret_cast<uint4*>(p + 16 * u) = x[i];
    *reinterpret_cast<uint4*>(p + 16 * u + 8) = y[i];
  }
}

template <typename T, int D>
hipError_t launch_append(const AppendExArgs& a, bool fp4, hipStream_t st) {
  const dim3 grid((unsigned)((a.T * a.chunks + 3) / 4)), block(256);
  if (fp4) {
    if (a.pos) paged_kv_append_kernel<T, D, true, true><<<grid, block, 0, st>>>(a);
    else paged_kv_append_kernel<T, D, false, true><<<grid, block, 0, st>>>(a);
  } else {
    if (a.pos) paged_kv_append_kernel<T, D, true, false><<<grid, block, 0, st>>>(a);
    else paged_kv_append_kernel<T, D><<<grid, block, 0, st>>>(a);
  }
  return hipGetLastError();
}
template <typename T>
hipError_t launch_append(const AppendExArgs& a, int D, bool fp4, hipStream_t st) {
  if (D == 64) return launch_append<T, 64>(a, fp4, st);
  if (D == 128) return launch_append<T, 128>(a, fp4, st);
  return launch_append<T, 256>(a, fp4, st);
}

template <typename T, int D>
hipError_t launch_read(const ReadArgs& g, bool fp4, hipStream_t st) {
  const int64_t rows = g.in.T * 2 * g.in.Hkv, per = kReadRows * (1024 / D) * 4;
  const dim3 grid((unsigned)((rows + per - 1) / per)), block(256);
  if (fp4) paged_kv_read_kernel<T, D, true><<<grid, block, 0, st>>>(g);
  else paged_kv_read_kernel<T, D, false><<<grid, block, 0, st>>>(g);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_read(const ReadArgs& g, int D, bool fp4, hipStream_t st) {
  if (D == 64) return launch_read<T, 64>(g, fp4, st);
  if (D == 128) return launch_read<T, 128>(g, fp4, st);
  return launch_read<T, 256>(g, fp4, st);
}

// Caches, tables and lengths of an append or a read; byte strides where `bytes`.
void set_caches(AppendArgs& a, const gdn_tensor* kc, const gdn_tensor* vc, const gdn_tensor* tab, const gdn_tensor* ctx,
                const gdn_tensor* cu, int64_t es) {
  a.kc = kc->data;
  a.kc_sb = kc->stride[0] * es;
  a.kc_st = kc->stride[1] * es;
  a.kc_sh = kc->stride[2] * es;
  a.vc = vc->data;
  a.vc_sb = vc->stride[0] * es;
  a.vc_st = vc->stride[1] * es;
  a.vc_sh = vc->stride[2] * es;
  a.num_blocks = kc->shape[0];
  a.page = (int32_t)kc->shape[1];
  a.tab = tab->data;
  a.tab_st = tab->stride[0];
  a.tab64 = tab->dtype == GDN_DTYPE_I64;
  a.cols = tab->shape[1];
  a.limit = a.cols * a.page;
  a.ctx = ctx->data;
  a.ctx64 = ctx->dtype == GDN_DTYPE_I64;
  a.nseq = tab->shape[0];
  a.Hkv = (int32_t)kc->shape[2];
  if (cu) {
    a.cu = cu->data;
    a.cu64 = cu->dtype == GDN_DTYPE_I64;
  }
}

}  // namespace

int64_t paged_kv_append_waves(int64_t T, int64_t rows, int64_t D) {
  const int64_t per = kAppendRows * (1024 / D);
  return T * ((rows + per - 1) / per);
}

// positions (axes, T) and the frequencies of each axis, section after section or
// (dealt) given to the axes in turn while they have some left; k_scales and
// v_scales: caches in 4 bits.
hipError_t paged_kv_append_launch(const gdn_tensor* k, const gdn_tensor* v, gdn_tensor* kc, gdn_tensor* vc,
                                  const gdn_tensor* tab, const gdn_tensor* ctx, const gdn_tensor* q, gdn_tensor* out,
                                  const gdn_tensor* cu, const gdn_tensor* cos, const gdn_tensor* sin,
                                  const gdn_tensor* pos, gdn_tensor* ks, gdn_tensor* vs, int interleaved,
                                  const int32_t* sections, bool dealt, hipStream_t st) {
  if (k->shape[0] == 0) return hipSuccess;
  const int D = (int)k->shape[2];
  AppendExArgs a{};
  a.k = k->data;
  a.k_st = k->stride[0];
  a.k_sh = k->stride[1];
  a.v = v->data;
  a.v_st = v->stride[0];
  a.v_sh = v->stride[1];
  if (q) {
    a.q = q->data;
    a.q_st = q->stride[0];
    a.q_sh = q->stride[1];
    a.o = out->data;
    a.o_st = out->stride[0];
    a.o_sh = out->stride[1];
    a.Hq = (int32_t)q->shape[1];
  }
  set_caches(a, kc, vc, tab, ctx, cu, 1);  // (elements of 16 bits, or bytes of codes)
  a.T = k->shape[0];
  if (cos) {
    a.cos = reinterpret_cast<const float*>(cos->data);
    a.cos_st = cos->stride[0];
    a.sin = reinterpret_cast<const float*>(sin->data);
    a.sin_st = sin->stride[0];
    a.rot = (int32_t)cos->shape[1] * 2;
    if (!pos) a.limit = cos->shape[0] < a.limit ? cos->shape[0] : a.limit;
  }
  if (pos) {
    a.pos = pos->data;
    a.pos_st = pos->stride[0];
    a.pos64 = pos->dtype == GDN_DTYPE_I64;
    a.naxes = (int32_t)pos->shape[0];
    a.rows = cos->shape[0];
    int32_t left[kMaxAxes];
    for (int x = 0; x < kMaxAxes; ++x) left[x] = x < a.naxes ? sections[x] : 0;
    int x = 0;
    for (int32_t j = 0; j < a.rot / 2; ++j) {  // (the sections' sum, checked by the entry)
      while (left[x] == 0) x = (x + 1) % kMaxAxes;
      a.axes[j / 16] |= (uint32_t)x << (2 * (j % 16));
      --left[x];
      if (dealt) x = (x + 1) % kMaxAxes;
    }
  }
  if (ks) {
    a.ks = scale_source(ks);
    a.vs = scale_source(vs);
  }
  a.chunks = (int32_t)paged_kv_append_waves(1, a.Hq + 2 * a.Hkv, D);
  a.interleaved = interleaved != 0;
  return k->dtype == GDN_DTYPE_BF16 ? launch_append<bf16_t>(a, D, ks != nullptr, st)
                                    : launch_append<f16_t>(a, D, ks != nullptr, st);
}

hipError_t paged_kv_read_launch(const gdn_tensor* kc, const gdn_tensor* vc, const gdn_tensor* tab,
                                const gdn_tensor* ctx, gdn_tensor* k, gdn_tensor* v, const gdn_tensor* cu,
                                const gdn_tensor* ks, const gdn_tensor* vs, hipStream_t st) {
  if (k->shape[0] == 0) return hipSuccess;
  ReadArgs g{};
  set_caches(g.in, kc, vc, tab, ctx, cu, ks ? 1 : 2);
  g.in.T = k->shape[0];
  g.k = k->data;
  g.k_st = k->stride[0];
  g.k_sh = k->stride[1];
  g.v = v->data;
  g.v_st = v->stride[0];
  g.v_sh = v->stride[1];
  if (ks) {
    g.in.ks = scale_source(ks);
    g.in.vs = scale_source(vs);
  }
  return k->dtype == GDN_DTYPE_BF16 ? launch_read<bf16_t>(g, (int)k->shape[2], ks != nullptr, st)
                                    : launch_read<f16_t>(g, (int)k->shape[2], ks != nullptr, st);
}

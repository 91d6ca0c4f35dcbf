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
#include "gdn_common.h"

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

template <typename T, int D>
__global__ __launch_bounds__(256) void paged_kv_append_kernel(const AppendArgs a) {
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
  const bool placed = pos >= 0 && pos < a.limit;
  int64_t block = -1;
  int32_t slot = 0;
  if (placed) {
    const int64_t col = (uint32_t)pos / (uint32_t)a.page;  // (positions are below 2^31)
    slot = (int32_t)(pos - col * a.page);
    block = load_index(a.tab, n * a.tab_st + col, a.tab64);
    if (block >= a.num_blocks) block = -1;
  }
  float c[8], s[8];
  if (turns && placed) {
    Vec8<float>::load(a.cos + pos * a.cos_st + 8 * u, c);
    Vec8<float>::load(a.sin + pos * a.sin_st + 8 * u, s);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = 1.f, s[j] = 0.f;
  }

#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int r = r0 + i * RPI;
    if (r >= nrows) continue;
    if (turns && r < nq + a.Hkv) {
      if (a.interleaved) {
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

template <typename T>
hipError_t launch_append(const AppendArgs& a, int D, hipStream_t st) {
  const dim3 grid((unsigned)((a.T * a.chunks + 3) / 4));
  if (D == 64)
    paged_kv_append_kernel<T, 64><<<grid, dim3(256), 0, st>>>(a);
  else if (D == 128)
    paged_kv_append_kernel<T, 128><<<grid, dim3(256), 0, st>>>(a);
  else
    paged_kv_append_kernel<T, 256><<<grid, dim3(256), 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

int64_t paged_kv_append_waves(int64_t T, int64_t rows, int64_t D) {
  const int64_t per = kAppendRows * (1024 / D);
  return T * ((rows + per - 1) / per);
}

hipError_t paged_kv_append_launch(const gdn_tensor* k, const gdn_tensor* v, gdn_tensor* kc, gdn_tensor* vc,
                                  const gdn_tensor* tab, const gdn_tensor* ctx, const gdn_tensor* q, gdn_tensor* out,
                                  const gdn_tensor* cu, const gdn_tensor* cos, const gdn_tensor* sin, int interleaved,
                                  hipStream_t st) {
  if (k->shape[0] == 0) return hipSuccess;
  const int D = (int)k->shape[2];
  AppendArgs a{};
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
  a.kc = kc->data;
  a.kc_sb = kc->stride[0];
  a.kc_st = kc->stride[1];
  a.kc_sh = kc->stride[2];
  a.vc = vc->data;
  a.vc_sb = vc->stride[0];
  a.vc_st = vc->stride[1];
  a.vc_sh = vc->stride[2];
  a.num_blocks = kc->shape[0];
  a.page = (int32_t)kc->shape[1];
  a.tab = tab->data;
  a.tab_st = tab->stride[0];
  a.tab64 = tab->dtype == GDN_DTYPE_I64;
  a.cols = tab->shape[1];
  a.limit = a.cols * a.page;
  a.ctx = ctx->data;
  a.ctx64 = ctx->dtype == GDN_DTYPE_I64;
  a.T = k->shape[0];
  a.nseq = tab->shape[0];
  a.Hkv = (int32_t)k->shape[1];
  if (cu) {
    a.cu = cu->data;
    a.cu64 = cu->dtype == GDN_DTYPE_I64;
  }
  if (cos) {
    a.cos = reinterpret_cast<const float*>(cos->data);
    a.cos_st = cos->stride[0];
    a.sin = reinterpret_cast<const float*>(sin->data);
    a.sin_st = sin->stride[0];
    a.rot = (int32_t)cos->shape[1] * 2;
    a.limit = cos->shape[0] < a.limit ? cos->shape[0] : a.limit;
  }
  a.chunks = (int32_t)paged_kv_append_waves(1, a.Hq + 2 * a.Hkv, D);
  a.interleaved = interleaved != 0;
  return k->dtype == GDN_DTYPE_BF16 ? launch_append<bf16_t>(a, D, st) : launch_append<f16_t>(a, D, st);
}

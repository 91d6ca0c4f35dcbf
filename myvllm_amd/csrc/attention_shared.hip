// Paged decode of sequences that begin with the same keys: the softmax over
// all keys of a sequence is merged from the one over the shared keys and the one
// over its own, (O, m, l) each.
//
// The shared keys run through the prefill kernel (attention_prefill.h, kShared):
// the queries of a group, sequences x heads of one kv head, are the rows of its
// MFMA tile, so the group's K and V are read once per 128 of them instead of once
// per sequence.  Each sequence's own keys run through the decode kernel
// (attention_decode.h, kShared).  Both leave unnormalised pieces, which the
// kernel below merges.
#include "attention_decode.h"
#include "attention_prefill.h"

namespace {

// Merge of the pieces of 32 rows (sequence, head of a kv head) and 32 dims, laid
// out as the prefill kernel's accumulators: lane l has row l % 32 and 4 x 4 dims.
// The four waves take every fourth piece, the shared ones first, and merge
// through LDS.
template <typename T, int D, int BN>
__global__ __launch_bounds__(256) void shared_decode_combine_kernel(const AttnArgs a, const DecodeArgs d) {
  typedef typename Mma<T>::v4 v4;
  __shared__ float part[4][18][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = a.Hq / a.Hkv, kvh = blockIdx.z, hh = lane >> 5;
  const uint32_t nrows = (uint32_t)a.T * R, row = blockIdx.x * 32 + (lane & 31);
  const bool valid = row < nrows;
  const uint32_t b = (valid ? row : 0u) / R;
  const int head = kvh * R + (int)((valid ? row : 0u) - b * R);
  const int64_t cap = a.tab.cols * a.tab.page, L = clamp64(load_index(a.ctx, b, a.ctx64), 0, cap);

  // shared pieces: np of them, rt slots apart
  int np = 0, rt = 0, first = 0, pl = 0;
  const int tiles = shared_tiles<D, BN>(a);
  if (tiles != kWholeRows) {
    const float inv = __builtin_amdgcn_rcpf((float)tiles);
    const int g = shared_group_of(a.sh, b, a.T);
    int per_head = 0;
    for (int c = 0; c < a.sh.n; c += 64) {
      const SharedRows q = shared_rows_lane<BN>(a, c);
      const int x = q.rt * shared_pieces(q.n, tiles, inv), m = a.sh.n - c < 64 ? a.sh.n - c : 64;
      per_head += wave_sum(x);
      for (int j = 0; j < m; ++j) first += c + j < g ? __builtin_amdgcn_readlane(x, j) : 0;
    }
    if (valid && g >= 0) {
      const SharedGroup sg = shared_group(a.sh, g, a.T, cap);
      const SharedRows q = shared_rows<BN>(a, sg);
      const int r = (int)row - (int)sg.b0 * R;
      np = sg.keys > 0 && L >= sg.keys ? shared_pieces(q.n, tiles, inv) : 0;
      rt = q.rt;
      first += kvh * per_head + (r >> 7);
      pl = (int)prefill_part_wave<D>() * ((r >> 5) & 3) + (r & 31) + 32 * hh;  // (m's offset less 32 D)
    }
  }
  // own pieces: units u0 .. u0 + ns - 1
  const int64_t U = (int64_t)d.B * d.units, Pt = d.prices[d.B], qb = d.prices[b], qn = d.prices[b + 1];
  int64_t u0 = 0;
  int ns = 0;
  if (valid && qn > qb) {
    u0 = ((qb + kDecodeStartPrice + 1) * U - 1) / Pt;
    ns = (int)((qn * U - 1) / Pt - u0) + 1;
  }

  const int dim0 = 32 * blockIdx.y;
  f32x4 acc[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) acc[g] = f32x4{0.f, 0.f, 0.f, 0.f};
  float mx = -INFINITY, l = 0.f;
  const int most = wave_top(np + ns);
#pragma unroll 2
  for (int i = w; i < most; i += 4) {
    const int64_t u = u0 + i - np;
    // (a unit without a price range, where there are more units than prices, has no piece)
    const bool own = i >= np, any = i < np + ns && (!own || (u + 1) * Pt / U > u * Pt / U);
    if (!any) continue;
    const float* pp = own ? d.part + ((b + u) * d.Hq + head) * (int64_t)(D + 4)
                          : a.part + (first + (int64_t)i * rt) * prefill_part_floats<D>();
    const float m = own ? pp[D] : pp[pl + 32 * D], lp = own ? pp[D + 1] : pp[pl + 32 * D + 64];
    const float* po = own ? pp + dim0 + 4 * hh : pp + (pl - pl % 64) + 8 * 32 * (int)blockIdx.y * 4 + 4 * (pl % 64);
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
    *reinterpret_cast<v4*>(reinterpret_cast<T*>(a.o) + b * a.o_st + (int64_t)head * a.o_sh + dim0 + 8 * w + 4 * hh) = ov;
}

// Workgroups that the shared keys may take: one per 128 rows of a group and kv
// head, up to four times as many or one round of the chip in pieces, within
// 512 MiB of partials.
int64_t shared_slots(int64_t B, int64_t groups, int64_t Hq, int64_t Hkv, int64_t D) {
  const int64_t most = std::min(groups, B / 2);  // (groups of two sequences at least)
  const int64_t base = Hkv * (B * (Hq / Hkv) / 128 + most), chip = D == 256 ? 256 : D == 128 ? 512 : 768;
  const int64_t fit = (int64_t(1) << 27) / (4 * (32 * D + 128));
  return most > 0 ? std::max(base, std::min(std::max(4 * base, chip), fit)) : 0;
}

template <typename T, int D>
hipError_t launch_shared(const AttnArgs& a, const DecodeArgs& d, hipStream_t st) {
  constexpr int BN = 32;
  if (a.extra > 0) {
    const dim3 grid((unsigned)((a.extra + 7) / 8 * 8));
    if (!whole_groups(a))
      hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 1, false, 0, kShared>), grid, dim3(256), 0, st, a);
    else if (a.tab.is64)
      hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 3, false, 0, kShared>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((attn_prefill_kernel<T, D, BN, 2, false, 0, kShared>), grid, dim3(256), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const hipError_t e = launch_decode_t<T, D, kShared>(d, st);
  if (e != hipSuccess) return e;
  const int64_t rows = a.T * (a.Hq / a.Hkv);
  hipLaunchKernelGGL((shared_decode_combine_kernel<T, D, BN>),
                     dim3((unsigned)((rows + 31) / 32), D / 32, (unsigned)a.Hkv), dim3(256), 0, st, a, d);
  return hipGetLastError();
}

}  // namespace

int64_t attn_shared_slots(int64_t B, int64_t groups, int64_t Hq, int64_t Hkv, int64_t D) {
  return shared_slots(B, groups, Hq, Hkv, D);
}

int64_t attn_shared_partials(int64_t B, int64_t groups, int64_t Hq, int64_t Hkv, int64_t D) {
  return shared_slots(B, groups, Hq, Hkv, D) * 4 * (32 * D + 128);
}

// workspace: the decode kernel's, `own` floats, then the shared pieces'
hipError_t attn_decode_shared_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc,
                                     const gdn_tensor* tab, const gdn_tensor* ctx, const gdn_tensor* lens,
                                     const gdn_tensor* groups, gdn_tensor* out, float* workspace, int64_t own,
                                     int32_t splits, float scale, hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  DecodeArgs d = decode_args(q, kc, vc, tab, ctx, out, workspace, splits, scale);
  d.sh.lens = lens->data;
  d.sh.lens64 = lens->dtype == GDN_DTYPE_I64;
  d.sh.n = (int32_t)lens->shape[0];
  if (groups) {
    d.sh.groups = groups->data;
    d.sh.groups64 = groups->dtype == GDN_DTYPE_I64;
  }
  AttnArgs a{};
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
  a.dim = (int32_t)q->shape[2];
  a.c = d.c;
  a.sh = d.sh;
  a.part = workspace + own;
  a.extra = (int32_t)shared_slots(d.B, d.sh.n, d.Hq, d.Hkv, a.dim);
  if (q->dtype == GDN_DTYPE_BF16) {
    if (a.dim == 64) return launch_shared<bf16_t, 64>(a, d, st);
    if (a.dim == 128) return launch_shared<bf16_t, 128>(a, d, st);
    return launch_shared<bf16_t, 256>(a, d, st);
  }
  if (a.dim == 64) return launch_shared<f16_t, 64>(a, d, st);
  if (a.dim == 128) return launch_shared<f16_t, 128>(a, d, st);
  return launch_shared<f16_t, 256>(a, d, st);
}

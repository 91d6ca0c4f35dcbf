// Attention with another form of scores, in the kernels of attention_prefill.h
// and attention_decode.h: capped by a tanh, biased by the distance of query and
// key, or with a prefix mask.  Against the plain form (us): 8 causal prompts of 256 to
// 4,096 tokens, 16 / 2 heads of 256, capped 483 / 414; 4 chunks behind up to 16,384
// paged keys, 16 / 4 heads of 128, biased 481 / 430; a decode of 64 sequences of
// 1,024 to 8,192 keys, capped, 125 / 120, at 5 TB/s.
#include "attention_decode.h"
#include "attention_prefill.h"

namespace {

template <typename A> void set_scores(A& a, const gdn_tensor* slopes, float cap) {
  a.slopes = slopes ? reinterpret_cast<const float*>(slopes->data) : nullptr;
  a.cap_in = cap > 0.f ? 2.f / cap : 0.f;
  a.cap_out = cap > 0.f ? 2.f * cap * kLog2e : 0.f;
}

template <typename T, bool PAGED>
hipError_t launch_scored(const AttnArgs& a, int64_t nseq, int64_t max_len, hipStream_t st) {
  if (a.dim == 256) return launch_prefill_t<T, 256, 32, PAGED, 0, kScored>(a, nseq, max_len, st);
  if (a.dim == 128) return launch_prefill_t<T, 128, 32, PAGED, 0, kScored>(a, nseq, max_len, st);
  if constexpr (PAGED) return launch_prefill_t<T, 64, 32, true, 0, kScored>(a, nseq, max_len, st);
  else return launch_prefill_64<T, 0, kScored>(a, nseq, max_len, st);
}

template <bool PAGED>
hipError_t launch_scored(AttnArgs a, const gdn_tensor* slopes, const gdn_tensor* pfx, float cap, int dtype,
                         int64_t max_len, hipStream_t st) {
  set_scores(a, slopes, cap);
  if (pfx) {
    a.pfx = pfx->data;
    a.pfx64 = pfx->dtype == GDN_DTYPE_I64;
  }
  return dtype == GDN_DTYPE_BF16 ? launch_scored<bf16_t, PAGED>(a, a.nseq, max_len, st)
                                 : launch_scored<f16_t, PAGED>(a, a.nseq, max_len, st);
}

}  // namespace

hipError_t attn_varlen_scored_launch(const gdn_tensor* q, const gdn_tensor* k, const gdn_tensor* v,
                                     const gdn_tensor* cu, gdn_tensor* out, const gdn_tensor* slopes,
                                     const gdn_tensor* pfx, int64_t max_seqlen, float scale, float cap, int causal,
                                     hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  return launch_scored<false>(varlen_args(q, k, v, cu, out, scale, causal), slopes, pfx, cap, q->dtype, max_seqlen,
                              st);
}

hipError_t attn_paged_scored_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc,
                                    const gdn_tensor* tab, const gdn_tensor* ctx, const gdn_tensor* cu,
                                    gdn_tensor* out, float* workspace, const gdn_tensor* slopes,
                                    const gdn_tensor* pfx, int64_t max_seqlen, float scale, float cap,
                                    hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  return launch_scored<true>(paged_args(q, kc, vc, tab, ctx, cu, out, workspace, scale), slopes, pfx, cap, q->dtype,
                             max_seqlen, st);
}

hipError_t attn_decode_scored_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc,
                                     const gdn_tensor* tab, const gdn_tensor* ctx, gdn_tensor* out, float* workspace,
                                     const gdn_tensor* slopes, int32_t splits, float scale, float cap,
                                     hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  DecodeArgs a = decode_args(q, kc, vc, tab, ctx, out, workspace, splits, scale);
  set_scores(a, slopes, cap);
  const int D = (int)q->shape[2];
  if (q->dtype == GDN_DTYPE_BF16) {
    if (D == 64) return launch_decode_t<bf16_t, 64, kScored>(a, st);
    if (D == 128) return launch_decode_t<bf16_t, 128, kScored>(a, st);
    return launch_decode_t<bf16_t, 256, kScored>(a, st);
  }
  if (D == 64) return launch_decode_t<f16_t, 64, kScored>(a, st);
  if (D == 128) return launch_decode_t<f16_t, 128, kScored>(a, st);
  return launch_decode_t<f16_t, 256, kScored>(a, st);
}

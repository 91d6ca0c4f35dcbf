// Full attention of the hybrid stack for gfx950: the launches of varlen and
// paged prefill (attention_prefill.h) and of split-KV paged decode
// (attention_decode.h).
//
// Reference: ops/full_attention.py of yuyifanbupt/myvllm (flash_attention_prefill
// :114-173, paged_flash_attention_decode :282-335, paged_flash_attention_prefill
// :454-512).  Query head h reads kv head h / (Hq / Hkv); softmax in fp32 with a
// running maximum; P rounded to the input dtype before P V, the row sum taken
// over the unrounded fp32 P (:100-107).
#include <mutex>

#include "attention_decode.h"
#include "attention_prefill.h"

// Split partials of paged_attention_decode_noalloc: a file-scope device array
// (one copy per GPU, for the life of the process) instead of a caller
// workspace.  Host code never passes `scratch` itself to a kernel (on the host
// the name stands for a host-side shadow, not a device address): the address
// is looked up once per device with hipGetSymbolAddress.
static __device__ __align__(256) float scratch[GDN_DECODE_SCRATCH_FLOATS];

namespace {

// Packed rows of any head dim that is a multiple of 8 up to 256: the next
// larger tile (the score product in steps of 16 dims, P V in steps of 32).
template <typename T>
hipError_t launch_prefill_ragged(const AttnArgs& a, int64_t nseq, int64_t max_len, hipStream_t st) {
  if (a.dim <= 64) return launch_prefill_64<T, 64>(a, nseq, max_len, st);
  if (a.dim <= 80) return launch_prefill_t<T, 96, 64, false, 80>(a, nseq, max_len, st);
  if (a.dim <= 96) return launch_prefill_t<T, 96, 64, false, 96>(a, nseq, max_len, st);
  if (a.dim <= 128) return launch_prefill_t<T, 128, 32, false, 128>(a, nseq, max_len, st);
  return launch_prefill_t<T, 256, 32, false, 256>(a, nseq, max_len, st);
}

template <bool PAGED>
hipError_t launch_prefill(const AttnArgs& a, int dtype, int D, int64_t nseq, int64_t max_len, hipStream_t st) {
  if constexpr (!PAGED) {
    if (D != 64 && D != 128 && D != 256)
      return dtype == GDN_DTYPE_BF16 ? launch_prefill_ragged<bf16_t>(a, nseq, max_len, st)
                                     : launch_prefill_ragged<f16_t>(a, nseq, max_len, st);
    if (D == 64)
      return dtype == GDN_DTYPE_BF16 ? launch_prefill_64<bf16_t, 0>(a, nseq, max_len, st)
                                     : launch_prefill_64<f16_t, 0>(a, nseq, max_len, st);
  }
  if (dtype == GDN_DTYPE_BF16) {
    if (D == 64) return launch_prefill_t<bf16_t, 64, 32, PAGED>(a, nseq, max_len, st);
    if (D == 128) return launch_prefill_t<bf16_t, 128, 32, PAGED>(a, nseq, max_len, st);
    return launch_prefill_t<bf16_t, 256, 32, PAGED>(a, nseq, max_len, st);
  }
  if (D == 64) return launch_prefill_t<f16_t, 64, 32, PAGED>(a, nseq, max_len, st);
  if (D == 128) return launch_prefill_t<f16_t, 128, 32, PAGED>(a, nseq, max_len, st);
  return launch_prefill_t<f16_t, 256, 32, PAGED>(a, nseq, max_len, st);
}

}  // namespace

hipError_t attn_varlen_prefill_launch(const gdn_tensor* q, const gdn_tensor* k, const gdn_tensor* v,
                                      const gdn_tensor* cu, gdn_tensor* out, int64_t max_seqlen, float scale,
                                      int causal, hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  return launch_prefill<false>(varlen_args(q, k, v, cu, out, scale, causal), q->dtype, (int)q->shape[2],
                               cu->shape[0] - 1, max_seqlen, st);
}

hipError_t attn_paged_prefill_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc,
                                     const gdn_tensor* tab, const gdn_tensor* ctx, const gdn_tensor* cu,
                                     gdn_tensor* out, float* workspace, int64_t max_seqlen, float scale,
                                     hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  return launch_prefill<true>(paged_args(q, kc, vc, tab, ctx, cu, out, workspace, scale), q->dtype,
                              (int)q->shape[2], cu->shape[0] - 1, max_seqlen, st);
}

int64_t attn_paged_prefill_workspace(int64_t T, int64_t nseq, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap) {
  const PrefillSplit sp = prefill_split(T, nseq, Hq, Hkv, D, cap);
  return sp.extra > 0 ? (sp.rows + sp.extra) * 4 * (32 * D + 128) : 0;
}

namespace {
constexpr int kMaxScratchDevices = 64;
std::mutex g_scratch_mu;
float* g_scratch_ptr[kMaxScratchDevices] = {};
}  // namespace

// Device address of `scratch` on the device that runs stream st, looked up on
// that device's first call (with the device made current for the lookup and
// the caller's current device restored) and cached.
hipError_t attn_decode_scratch(hipStream_t st, float** ptr) {
  int dev = 0;
  hipError_t e = st ? hipStreamGetDevice(st, &dev) : hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev < 0 || dev >= kMaxScratchDevices) return hipErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    int cur = 0;
    if ((e = hipGetDevice(&cur)) != hipSuccess) return e;
    if (cur != dev && (e = hipSetDevice(dev)) != hipSuccess) return e;
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    const hipError_t r = cur != dev ? hipSetDevice(cur) : hipSuccess;
    if (e != hipSuccess) return e;
    if (r != hipSuccess) return r;
    if (!p) return hipErrorInvalidSymbol;
    g_scratch_ptr[dev] = static_cast<float*>(p);
  }
  *ptr = g_scratch_ptr[dev];
  return hipSuccess;
}

int32_t attn_decode_start_price() { return kDecodeStartPrice; }

hipError_t attn_paged_decode_launch(const gdn_tensor* q, const gdn_tensor* kc, const gdn_tensor* vc,
                                    const gdn_tensor* tab, const gdn_tensor* ctx, gdn_tensor* out, float* workspace,
                                    int32_t splits, float scale, hipStream_t st) {
  if (q->shape[0] == 0) return hipSuccess;
  const DecodeArgs a = decode_args(q, kc, vc, tab, ctx, out, workspace, splits, scale);
  const int D = (int)q->shape[2];
  if (q->dtype == GDN_DTYPE_BF16) {
    if (D == 64) return launch_decode_t<bf16_t, 64>(a, st);
    if (D == 128) return launch_decode_t<bf16_t, 128>(a, st);
    return launch_decode_t<bf16_t, 256>(a, st);
  }
  if (D == 64) return launch_decode_t<f16_t, 64>(a, st);
  if (D == 128) return launch_decode_t<f16_t, 128>(a, st);
  return launch_decode_t<f16_t, 256>(a, st);
}

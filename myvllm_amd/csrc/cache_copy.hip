// Copies of blocks inside caches: block dst[i] <- block src[i] of every layer of
// up to four caches (keys and values, their block scales, or the states of
// linear-attention layers) in one launch.  The step behind a fork (the last,
// partly filled page; the states) and behind a compaction.
//
// Bound: HBM, each copied byte read and written once.  The ids come with the
// kernel's arguments, 448 pairs a launch (the limit is 4 KB): the host's allocator
// knows them, so nothing is sent to the device ahead and the entry can check them.
// A workgroup copies 4 KB of a block, 16 bytes a thread: 1,501 pages of 16 KB in eight
// layers of keys and values (787 MB moved) 135 us, 5.8 TB/s, 99 % of a streaming
// copy; with 8, 16 and 32 KB a workgroup 145, 150 and 150.  Calls of 32 MB and more
// store past the caches (164 us without); smaller ones leave what they wrote in the
// L2s for the step that reads it next.
#include "gdn_common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int64_t kStreamBytes = 32 << 20;
constexpr int kCaches = 4, kPairs = 448;

struct CopyCache {
  char* base;
  int64_t layer, block, bytes;  // byte strides; bytes of a block of a layer
  uint32_t chunks, first;       // workgroups per block; first workgroup of this cache
};

struct CopyArgs {
  CopyCache c[kCaches];
  int32_t n, pairs;
  int32_t src[kPairs], dst[kPairs];
};
static_assert(sizeof(CopyArgs) <= 4096, "kernel arguments");

template <typename V, bool STREAM>
__global__ __launch_bounds__(256) void cache_copy_kernel(const CopyArgs a) {
  uint32_t id = blockIdx.x;
  int t = 0;
#pragma unroll
  for (int i = 1; i < kCaches; ++i)
    if (i < a.n && id >= a.c[i].first) t = i;
  const CopyCache& c = a.c[t];
  id -= c.first;
  const uint32_t row = id / c.chunks, chunk = id - row * c.chunks;
  const uint32_t layer = row / (uint32_t)a.pairs, p = row - layer * (uint32_t)a.pairs;
  const char* from = c.base + layer * c.layer + a.src[p] * c.block;
  char* to = c.base + layer * c.layer + a.dst[p] * c.block;
  const int64_t at = ((int64_t)chunk * 256 + threadIdx.x) * sizeof(V);
  if (at >= c.bytes) return;
  const V v = *reinterpret_cast<const V*>(from + at);
  if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<V*>(to + at));
  else *reinterpret_cast<V*>(to + at) = v;
}

int64_t copy_workgroups(const gdn_tensor* t, int64_t es, int64_t vec, int64_t pairs) {
  const int64_t per = 256 * vec;
  return t->shape[0] * pairs * ((t->shape[2] * es + per - 1) / per);
}

}  // namespace

// Whether one launch's workgroups fit a grid axis (checked by the entry).
bool cache_copy_fits(gdn_tensor* const* t, const int64_t* es, int n, int64_t vec, int64_t count) {
  const int64_t most = count < kPairs ? count : kPairs;
  int64_t sum = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t per = 256 * vec, chunks = (t[i]->shape[2] * es[i] + per - 1) / per;
    if (t[i]->shape[0] >= int64_t(1) << 31 || chunks >= int64_t(1) << 31 || t[i]->shape[0] * chunks >= int64_t(1) << 31)
      return false;
    sum += t[i]->shape[0] * most * chunks;
    if (sum >= int64_t(1) << 31) return false;
  }
  return true;
}

// Caches (layers, blocks, elements of a block), es bytes each, 16-byte aligned
// throughout where vec is 16; ids on the host.
hipError_t cache_copy_launch(gdn_tensor* const* t, const int64_t* es, int n, const int32_t* src, const int32_t* dst,
                             int64_t count, int64_t vec, hipStream_t st) {
  CopyArgs a;
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += t[i]->shape[0] * t[i]->shape[2] * es[i] * count;
  for (int64_t p0 = 0; p0 < count; p0 += kPairs) {
    const int64_t m = count - p0 < kPairs ? count - p0 : kPairs;
    a.pairs = (int32_t)m;
    a.n = 0;
    int64_t wgs = 0;
    for (int i = 0; i < n; ++i) {
      const int64_t mine = copy_workgroups(t[i], es[i], vec, m);
      if (mine == 0) continue;
      CopyCache& c = a.c[a.n++];
      c.base = reinterpret_cast<char*>(t[i]->data);
      c.layer = t[i]->stride[0] * es[i];
      c.block = t[i]->stride[1] * es[i];
      c.bytes = t[i]->shape[2] * es[i];
      c.chunks = (uint32_t)(mine / (t[i]->shape[0] * m));
      c.first = (uint32_t)wgs;
      wgs += mine;
    }
    for (int64_t i = 0; i < m; ++i) a.src[i] = src[p0 + i], a.dst[i] = dst[p0 + i];
    if (wgs == 0) continue;
    const dim3 grid((unsigned)wgs), block(256);
    if (vec != 16) cache_copy_kernel<uint8_t, false><<<grid, block, 0, st>>>(a);
    else if (bytes >= kStreamBytes) cache_copy_kernel<u32x4, true><<<grid, block, 0, st>>>(a);
    else cache_copy_kernel<u32x4, false><<<grid, block, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

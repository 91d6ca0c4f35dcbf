// What the full-attention kernels share: the MFMA shapes per 16-bit type, the
// transposed LDS read, key and value rows of packed and paged sources.
#pragma once

#include "gdn_common.h"

namespace {

template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
  typedef bf16x8 v8;
  typedef bf16x4 v4;
  static GDN_DEVICE f32x16 m32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static GDN_DEVICE f32x4 m16k32(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static GDN_DEVICE f32x4 m16k16(v4 a, v4 b, f32x4 c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
  }
};
template <> struct Mma<f16_t> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  static GDN_DEVICE f32x16 m32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static GDN_DEVICE f32x4 m16k32(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static GDN_DEVICE f32x4 m16k16(v4 a, v4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short __attribute__((address_space(3))) lds_short;
typedef s16x4_t __attribute__((address_space(3))) lds_s16x4_t;

// ds_read_b64_tr_b16: in each 16-lane group, lane i supplies the address of
// 4 consecutive 16-bit elements of row (i >> 2), columns 4 (i & 3) .. +3, of
// a 4 x 16 block, and receives column i of that block (rows 0..3).
template <typename V4> GDN_DEVICE V4 tr4(const void* p) {
  return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p)));
}

GDN_DEVICE float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// max(x[l], x[l ^ 32]) in every lane l: one v_permlane32_swap of x with
// itself (lanes 0..31 of one copy trade places with lanes 32..63 of the
// other, so each lane then holds both of the pair's values), no LDS round
// trip as a ds_bpermute would take.  (The two results are copied to scalars
// before they are reinterpreted: this clang reads the first element of the
// vector for __builtin_bit_cast(float, sw[1]).)  The maximum is a select:
// fmaxf would first quiet both operands, two more instructions on the
// softmax's dependency chain (the scores are never NaN).
GDN_DEVICE float max_lane_pair32(float x) {
  const uint32_t v = __builtin_bit_cast(uint32_t, x);
  const auto sw = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t ua = sw[0], ub = sw[1];
  const float a = __builtin_bit_cast(float, ua), b = __builtin_bit_cast(float, ub);
  return a > b ? a : b;
}

GDN_DEVICE int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : (x > hi ? hi : x); }

// An index at a wave-uniform position read through the scalar data cache (a
// constant-address-space load): its wait is on the scalar/LDS counter, so it
// does not drain the vector loads in flight.  Only for read-only inputs.
typedef const int32_t __attribute__((address_space(4))) * const_i32_ptr;
typedef const int64_t __attribute__((address_space(4))) * const_i64_ptr;
GDN_DEVICE int64_t load_index_scalar(const void* p, int64_t i, bool is64) {
  return is64 ? __builtin_bit_cast(const_i64_ptr, p)[i] : (int64_t)__builtin_bit_cast(const_i32_ptr, p)[i];
}

// Row j of a key or value source: packed varlen rows (row s0 + j) or paged
// rows (block table[n][j / page], slot j % page).  nullptr past the valid
// range or for a table entry outside [0, num_blocks): such rows read as zero.
struct KvSource {
  const char* base;
  int64_t sb, st, sh;  // byte strides: block (paged), row, head
};

struct PagedTable {
  const void* table;
  int64_t row_stride, cols, num_blocks;
  int32_t page;
  bool is64;
};

template <bool PAGED>
GDN_DEVICE const char* kv_row(const KvSource& s, const PagedTable& tb, int64_t n, int64_t s0, int64_t j, int kvh) {
  if (PAGED) {
    const int64_t col = j / tb.page;
    if (col >= tb.cols) return nullptr;
    const int64_t blk = load_index(tb.table, n * tb.row_stride + col, tb.is64);
    if (blk < 0 || blk >= tb.num_blocks) return nullptr;
    return s.base + blk * s.sb + (j - col * tb.page) * s.st + kvh * s.sh;
  } else {
    return s.base + (s0 + j) * s.st + kvh * s.sh;
  }
}

// What a prefill or decode kernel computes.
enum AttnForm {
  kPlain,
  kScored,  // capped or biased scores, prefix masks
  kShared,  // decode of sequences that share their first keys: those (prefill kernel), and the others (attention_own.h)
};

// What a shared decode's first launch writes down (attention_shared.hip).  Of a
// sequence: the keys that its group reads for it (its own begin there), its
// group's pieces (0 where it is not read with the group) and 128-row blocks,
// rt << 11 | pieces; the group's first slot of a kv head, and the sequence's
// first row in the group.
struct SharedSeq {
  int32_t first, pieces, slot, row;
};
// Of a workgroup: the sequence through whose table the keys are read (-1: no
// work), the group's first sequence and rows, the workgroup's first row, its
// keys [32 tile0, keys), kv head and slot of the partials.
struct SharedWork {
  int32_t lead, b0, rows, row, tile0, keys, kvh, slot;
};

// A capped score, cap tanh(x) of x = scale s / cap, is cap - 2 cap / (1 + e^(2 x)),
// and a constant on all scores of a row does not change its softmax: the raw score
// s becomes -1 / (1 + 2^(k s)), k = 2 log2(e) scale / cap, which 2 cap log2(e)
// scales to an exponent of 2.  Within 3e-7 cap of the tanh of its fp32 argument:
// twice the exponential's ulp (2^-23 y (1 - y), y the quotient), the sum's half
// (2^-24 y^2) and the reciprocal's (2^-24).
GDN_DEVICE float cap_score(float s, float k) {
  return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(s * k));
}

// The same as tanh(x) / 2 - 1 / 2 by an odd polynomial of degree 9 for |x| <= 0.7
// (|s| <= lim; fitted for the least largest error there, 9.4e-8, 1.9e-7 with the
// fp32 roundings; to 3/4 it would be 2.9e-7): full-rate
// instructions instead of the exponential and the reciprocal, and a test of the
// tile.  It is evaluated in x = h s: folded into the coefficients, the powers of h
// leave fp32's range (h^9 below 1e-4).  It pays where several waves share a SIMD's
// transcendental unit: D = 64, six prompts capped and biased under a prefix mask
// 72 -> 66 us, capped alone 57 -> 55; D = 128 526 -> 533, D = 256, where a wave has
// its SIMD to itself, 481 -> 496.
struct CapNear {
  float lim, h;
  GDN_DEVICE void set(float k) {
    h = k * 0.34657359f;  // x = h s (ln 2 / 2: k is 2 log2(e) scale / cap)
    lim = h < 1e30f ? 0.7f / h : -1.f;
  }
  GDN_DEVICE float operator()(float s) const {
    const float x = s * h, u = x * x;
    float p = 0.5f * 0.01319420f;
    p = __builtin_fmaf(p, u, 0.5f * -0.05019528f);
    p = __builtin_fmaf(p, u, 0.5f * 0.13257456f);
    p = __builtin_fmaf(p, u, 0.5f * -0.33326975f);
    p = __builtin_fmaf(p, u, 0.5f * 0.99999851f);
    return __builtin_fmaf(x, p, -0.5f);
  }
};

constexpr float kLog2e = 1.4426950408889634f;

KvSource kv_source(const gdn_tensor* t, bool paged) {
  const int64_t es = t->dtype == GDN_DTYPE_F32 ? 4 : 2;
  KvSource s;
  s.base = reinterpret_cast<const char*>(t->data);
  if (paged) {
    s.sb = t->stride[0] * es;
    s.st = t->stride[1] * es;
    s.sh = t->stride[2] * es;
  } else {
    s.sb = 0;
    s.st = t->stride[0] * es;
    s.sh = t->stride[1] * es;
  }
  return s;
}

PagedTable paged_table(const gdn_tensor* tab, const gdn_tensor* kc) {
  PagedTable p;
  p.table = tab->data;
  p.row_stride = tab->stride[0];
  p.cols = tab->shape[1];
  p.num_blocks = kc->shape[0];
  p.page = (int32_t)kc->shape[1];
  p.is64 = tab->dtype == GDN_DTYPE_I64;
  return p;
}

int heads_per_group(int R) { return R % 4 == 0 ? 4 : (R % 2 == 0 ? 2 : 1); }

}  // namespace

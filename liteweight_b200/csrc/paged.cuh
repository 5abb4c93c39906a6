// What the paged-cache kernels share: the cache's view on the device, the
// bounds checks of its indexes, the 16-bit types, and the argument checks.
#pragma once

#include <cuda_bf16.h>

#include <atomic>

#include "lw_common.cuh"

namespace lw {

// ------------------------------------------------------------- 16-bit types

template <typename T>
struct Elem;

template <>
struct Elem<__half> {
  static LW_DEV uint32_t pack(float lo, float hi) { return h2_as_u32(__floats2half2_rn(lo, hi)); }
  static LW_DEV float2 unpack(uint32_t u) { return __half22float2(u32_as_h2(u)); }
  static constexpr uint32_t kExpMask = 0x7C00u;   // all ones: infinity or NaN
  // Softmax weights rounded to fp16 may be up to 2^15 (the largest fp16 is just
  // below 2^16): below 2^-14 the type has a fixed step, and with the weights in
  // [0, 1] those under 2^-25 would be 0 in the product and still count in the sum
  // (131070 of e^-18 beside a 1: the result would be 0 instead of 0.002).
  static constexpr float kMaxWeightLog2 = 15.0f;
  // a * 0 + c in each half
  static LW_DEV uint32_t fma0(uint32_t a, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(0u), "r"(c));
    return d;
  }
};

template <>
struct Elem<__nv_bfloat16> {
  static LW_DEV uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static LW_DEV float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  static constexpr uint32_t kExpMask = 0x7F80u;
  static constexpr float kMaxWeightLog2 = 0.0f;   // the range of fp32: small weights keep their precision
  static LW_DEV uint32_t fma0(uint32_t a, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(0u), "r"(c));
    return d;
  }
};

// Either half of the word is an infinity or a NaN.
template <typename T>
LW_DEV bool has_nonfinite(uint32_t u) {
  constexpr uint32_t lo = Elem<T>::kExpMask, hi = lo << 16;
  return (u & lo) == lo || (u & hi) == hi;
}

// D(16x8 f32) += A(16x16, row) * B(16x8, col) in T; fragments as mma16816.
template <typename T>
LW_DEV void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
LW_DEV void mma_16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                              uint32_t b1) {
  mma16816(d, a0, a1, a2, a3, b0, b1);
}
template <>
LW_DEV void mma_16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

LW_DEV void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
LW_DEV void ldmatrix_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

LW_DEV float2 lds_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// 16 bytes global -> shared, zeros instead when !valid (src is not read then).
LW_DEV void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
LW_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
LW_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two fp32 operations in one instruction.
LW_DEV uint64_t as_u64(float2 v) { return *reinterpret_cast<uint64_t*>(&v); }
LW_DEV float2 as_f2(uint64_t v) { return *reinterpret_cast<float2*>(&v); }
LW_DEV float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(as_u64(a)), "l"(as_u64(b)), "l"(as_u64(c)));
  return as_f2(y);
}
LW_DEV float2 add2(float2 a, float2 b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(as_u64(a)), "l"(as_u64(b)));
  return as_f2(y);
}
LW_DEV float2 mul2(float2 a, float2 b) {
  uint64_t y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(as_u64(a)), "l"(as_u64(b)));
  return as_f2(y);
}

// 2^x (a result below the normal range is 0).
LW_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------- the cache

struct PagedView {
  void* k;
  void* v;
  long long kp, kh, ks, vp, vh, vs;   // strides in elements: page, head, slot
  int n_pages, page_size, page_shift, nkv, B;
  const int* table;
  long long table_stride;
  int table_width;
  const int* lens;
};

// Tokens of a sequence of length n that the table can address (a longer length is recorded and cut).
LW_DEV int cut_len(const PagedView& c, int n) {
  const long long most = (long long)c.table_width << c.page_shift;
  if (n > most) {
    lw_record_error(LW_ERR_BAD_INDEX);
    return (int)most;
  }
  return max(n, 0);
}
LW_DEV int seq_len(const PagedView& c, int b) { return cut_len(c, c.lens[b]); }

// Page of token `tok` (0 <= tok < seq_len), or -1 (recorded) for an id outside the pool.
LW_DEV int page_id(const PagedView& c, int b, int tok) {
  const int id = c.table[b * c.table_stride + (tok >> c.page_shift)];
  if ((unsigned)id < (unsigned)c.n_pages) return id;
  lw_record_error(LW_ERR_BAD_INDEX);
  return -1;
}

// The base of a row that sees keys, every score of which is minus infinity: below
// any other, above that of a row (or a part of one) that sees none.
constexpr float kAllBelow = -3.402823466e38f;

// 1 / the sum of the weights; 0 for a row that sees no key, NaN (a softmax of
// minus infinities) for one that sees only keys without weight.
LW_DEV float weight_inverse(float m, float l) {
  return l != 0.f ? 1.f / l : m == -INFINITY ? 0.f : __int_as_float(0x7FFFFFFF);
}

// The first key that position p sees through its window.
LW_DEV int window_start(int p, int window) { return window > 0 ? max(0, p - window + 1) : 0; }

// Sequence of row t: the b with off[b] <= t < off[b + 1], or -1.
LW_DEV int row_sequence(const int* off, int B, int t) {
  if (t < off[0] || t >= off[B]) return -1;
  int lo = 0, hi = B;   // off[lo] <= t < off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace lw

// ------------------------------------------------------------- host

namespace lw_host {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline bool strides8(const long long* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || (s[i] & 7)) return false;
  return true;
}

inline int check_cache(const lw_paged_cache& c) {
  if (c.batch < 0 || c.table_width < 0 || c.n_pages < 0 || c.n_kv_heads <= 0) return LW_ERR_BAD_SHAPE;
  if (c.page_size <= 0 || (c.page_size & (c.page_size - 1))) return LW_ERR_BAD_SHAPE;
  if (c.page_size < 16 || c.page_size > 256 || (c.head_dim != 64 && c.head_dim != 128)) return LW_ERR_UNSUPPORTED;
  if (c.dtype != LW_DTYPE_F16 && c.dtype != LW_DTYPE_BF16) return LW_ERR_UNSUPPORTED;
  if ((long long)c.table_width * c.page_size > 0x7FFFFFFFll - 65536) return LW_ERR_UNSUPPORTED;   // positions are int32
  if (c.batch == 0) return LW_OK;
  if (!c.kv_lens || (c.n_pages && (!c.k_pages || !c.v_pages)) || (c.table_width && !c.page_table))
    return LW_ERR_NULL_POINTER;
  if (!aligned16(c.k_pages) || !aligned16(c.v_pages) || !strides8(c.k_strides, 3) || !strides8(c.v_strides, 3))
    return LW_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(c.kv_lens) & 3u || reinterpret_cast<uintptr_t>(c.page_table) & 3u)
    return LW_ERR_ALIGNMENT;
  return LW_OK;
}

inline lw::PagedView view_of(const lw_paged_cache& c) {
  lw::PagedView v = {};
  v.k = c.k_pages;
  v.v = c.v_pages;
  v.kp = c.k_strides[0];
  v.kh = c.k_strides[1];
  v.ks = c.k_strides[2];
  v.vp = c.v_strides[0];
  v.vh = c.v_strides[1];
  v.vs = c.v_strides[2];
  v.n_pages = c.n_pages;
  v.page_size = c.page_size;
  while ((1 << v.page_shift) < c.page_size) ++v.page_shift;
  v.nkv = c.n_kv_heads;
  v.B = c.batch;
  v.table = c.page_table;
  v.table_stride = c.table_stride;
  v.table_width = c.table_width;
  v.lens = c.kv_lens;
  return v;
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device (asked
// once per kernel and device: it costs as much as a quarter of a launch).
template <auto kKernel>
inline cudaError_t allow_smem(int bytes) {
  static std::atomic<unsigned long long> done{0};   // bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = dev >= 0 && dev < 64 ? 1ull << dev : 0ull;
  if (bit & done.load(std::memory_order_relaxed)) return cudaSuccess;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

inline int sm_count() {
  static int counts[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!counts[dev] && cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    counts[dev] = 148;
  return counts[dev];
}

}  // namespace lw_host

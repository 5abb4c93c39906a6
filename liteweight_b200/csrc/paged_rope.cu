// Norms of queries and keys for each head, rotation by position and the append
// to the paged cache, in one pass (lw_qk_norm_rope).
//
//   y = x * rsqrt(mean(x^2) + eps) * w,   o[d] = y[d] cos[p][d] + r[d] sin[p][d],
//   r = (-y[hd/2:], y[:hd/2])
//
// A group of hd / 16 lanes takes one token's run of up to HPG heads of one kind
// (queries, keys or values): each lane holds dims 8j .. 8j+7 and their rotation
// partners hd/2 + 8j .. + 7, so a head is two 16-byte loads and two 16-byte
// stores a lane, the rotation needs no exchange, and the mean is log2(hd / 16)
// shuffles. Weight and angle make four factors per pair, formed once per run:
//   o_lo = r (x_lo [w_lo cos_lo] - x_hi [w_hi sin_lo]),  r = rsqrt(mean + eps)
//   o_hi = r (x_hi [w_hi cos_hi] + x_lo [w_lo sin_hi])
// All of it in fp32 with one rounding at the store. Memory bound: every element
// is read once and written once. 11064 tokens of 64 + 2x8 heads of 128 (bf16, fp32
// tables): 76 - 78 us on several GPUs, 5.9 - 6.0 TB/s, 0.9 of a copy's rate. One token:
// 2.4 us, a launch.
#include "paged.cuh"

namespace lw {

struct RopeParams {
  PagedView c;
  const void *q, *k, *v;
  long long q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h;
  void* out;
  int T, nq, q_runs, kv_runs;   // runs of heads per token: q_runs + 2 * kv_runs
  const int* off;
  const void *cos, *sin;
  long long rope_stride;
  int rope_rows;
  const void *qw, *kw;
  float eps;
  int zero_tail;
};

// 8 elements as four pairs.
template <typename T>
LW_DEV void unpack8(const uint4& u, float2 (&f)[4]) {
  f[0] = Elem<T>::unpack(u.x);
  f[1] = Elem<T>::unpack(u.y);
  f[2] = Elem<T>::unpack(u.z);
  f[3] = Elem<T>::unpack(u.w);
}
template <typename T>
LW_DEV void load8(const T* p, float2 (&f)[4]) {
  unpack8<T>(*reinterpret_cast<const uint4*>(p), f);
}
template <>
LW_DEV void load8<float>(const float* p, float2 (&f)[4]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = make_float2(a.x, a.y);
  f[1] = make_float2(a.z, a.w);
  f[2] = make_float2(b.x, b.y);
  f[3] = make_float2(b.z, b.w);
}

// 16 bytes that are read once: not kept in L1, where the tables and weights are.
LW_DEV uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

constexpr int kRopeThreads = 256;

// T: element type; TT: type of the rotation table; HPG: heads per run.
template <typename T, typename TT, int HD, int HPG>
__global__ void __launch_bounds__(kRopeThreads, 2) qk_norm_rope_kernel(const RopeParams p) {
  constexpr int LPR = HD / 16;   // lanes per head
  pdl_wait();
  pdl_launch_dependents();
  const int j = threadIdx.x % LPR, runs = p.q_runs + 2 * p.kv_runs;
  const long long item = (long long)blockIdx.x * (kRopeThreads / LPR) + threadIdx.x / LPR;
  const long long t64 = item / runs;
  if (t64 >= p.T) return;   // whole groups: shuffles below stay within a group
  const int t = (int)t64;
  int run = (int)(item - t64 * runs);
  const int kind = run < p.q_runs ? 0 : run < p.q_runs + p.kv_runs ? 1 : 2;   // queries, keys, values
  run -= kind == 0 ? 0 : kind == 1 ? p.q_runs : p.q_runs + p.kv_runs;
  const int h0 = run * HPG, n = min(HPG, (kind ? p.c.nkv : p.nq) - h0);
  const unsigned gmask = ((1u << LPR) - 1u) << ((threadIdx.x & 31) / LPR * LPR);
  const int d_lo = 8 * j, d_hi = HD / 2 + 8 * j;

  // the run's heads, all loads in flight before the first use
  uint4 lo[HPG], hi[HPG];
  {
    const long long st = kind == 0 ? p.q_t : kind == 1 ? p.k_t : p.v_t;
    const long long sh = kind == 0 ? p.q_h : kind == 1 ? p.k_h : p.v_h;
    const T* src = static_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) + t * st + h0 * sh;
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      if (i >= n) break;
      lo[i] = load_once(src + i * sh + d_lo);
      hi[i] = load_once(src + i * sh + d_hi);
    }
  }

  const int b = p.off ? row_sequence(p.off, p.c.B, t) : t;
  int pos = -1;
  if (b >= 0) {
    const int len = p.c.lens[b];
    pos = p.off ? len - p.off[b + 1] + t : len - 1;
  }
  T* dst = kind == 0 ? static_cast<T*>(p.out) + t * p.o_t + h0 * p.o_h : nullptr;
  long long dh = p.o_h;
  if (b < 0 || pos < 0 || pos >= p.rope_rows) {   // a row of no sequence, or a position that there is not
    // past the table, or more new tokens than the length counts
    if (b >= 0 && (pos >= 0 || p.off) && j == 0) lw_record_error(LW_ERR_BAD_INDEX);
    if (kind == 0 && p.zero_tail)
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        *reinterpret_cast<uint4*>(dst + i * dh + d_lo) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + i * dh + d_hi) = make_uint4(0, 0, 0, 0);
      }
    return;
  }
  if (kind) {   // where the token is kept
    const int page = (pos >> p.c.page_shift) < p.c.table_width ? page_id(p.c, b, pos) : -1;
    if (page < 0) {
      if (j == 0) lw_record_error(LW_ERR_BAD_INDEX);
      return;
    }
    const long long slot = pos & (p.c.page_size - 1);
    if (kind == 1) dst = static_cast<T*>(p.c.k) + page * p.c.kp + slot * p.c.ks + h0 * p.c.kh, dh = p.c.kh;
    else dst = static_cast<T*>(p.c.v) + page * p.c.vp + slot * p.c.vs + h0 * p.c.vh, dh = p.c.vh;
    if (kind == 2) {   // values are kept as they are
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        if (i >= n) break;
        *reinterpret_cast<uint4*>(dst + i * dh + d_lo) = lo[i];
        *reinterpret_cast<uint4*>(dst + i * dh + d_hi) = hi[i];
      }
      return;
    }
  }
  // factors of the pairs: own and partner's, for the low and the high half
  float2 own_lo[4], own_hi[4], par_lo[4], par_hi[4];
  {
    const TT* cs = static_cast<const TT*>(p.cos) + pos * p.rope_stride;
    const TT* sn = static_cast<const TT*>(p.sin) + pos * p.rope_stride;
    load8(cs + d_lo, own_lo);
    load8(cs + d_hi, own_hi);
    load8(sn + d_lo, par_lo);
    load8(sn + d_hi, par_hi);
  }
  const T* w = static_cast<const T*>(kind ? p.kw : p.qw);
  const float2 minus = make_float2(-1.f, -1.f);
  if (w) {
    float2 w_lo[4], w_hi[4];
    load8(w + d_lo, w_lo);
    load8(w + d_hi, w_hi);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      own_lo[e] = mul2(own_lo[e], w_lo[e]);
      own_hi[e] = mul2(own_hi[e], w_hi[e]);
      par_lo[e] = mul2(mul2(par_lo[e], minus), w_hi[e]);
      par_hi[e] = mul2(par_hi[e], w_lo[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) par_lo[e] = mul2(par_lo[e], minus);
  }
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    if (i >= n) break;
    float2 x_lo[4], x_hi[4];
    unpack8<T>(lo[i], x_lo);
    unpack8<T>(hi[i], x_hi);
    float r = 1.f;
    if (w) {
      float2 ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = fma2(x_lo[e], x_lo[e], fma2(x_hi[e], x_hi[e], ss));
      float sum = ss.x + ss.y;
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(gmask, sum, o);
      r = rsqrtf(sum * (1.0f / HD) + p.eps);
    }
    const float2 r2 = make_float2(r, r);
    uint32_t y_lo[4], y_hi[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = mul2(r2, fma2(x_lo[e], own_lo[e], mul2(x_hi[e], par_lo[e])));
      const float2 c = mul2(r2, fma2(x_hi[e], own_hi[e], mul2(x_lo[e], par_hi[e])));
      y_lo[e] = Elem<T>::pack(a.x, a.y);
      y_hi[e] = Elem<T>::pack(c.x, c.y);
    }
    *reinterpret_cast<uint4*>(dst + i * dh + d_lo) = make_uint4(y_lo[0], y_lo[1], y_lo[2], y_lo[3]);
    *reinterpret_cast<uint4*>(dst + i * dh + d_hi) = make_uint4(y_hi[0], y_hi[1], y_hi[2], y_hi[3]);
  }
}

}  // namespace lw

namespace {

template <typename T, typename TT, int HD>
cudaError_t rope_launch(lw::RopeParams& p, cudaStream_t s, bool pdl) {
  constexpr int groups = lw::kRopeThreads / (HD / 16);
  auto blocks = [&](int hpg) {
    p.q_runs = (p.nq + hpg - 1) / hpg;
    p.kv_runs = (p.c.nkv + hpg - 1) / hpg;
    return ((long long)p.T * (p.q_runs + 2 * p.kv_runs) + groups - 1) / groups;
  };
  // A run of 8 heads shares one load of the angles and keeps 16 loads in flight
  // a lane (11064 tokens: 76 us, runs of 4 heads 87, of 2 heads 85); a launch too
  // small to give every SM two blocks takes single heads.
  const long long n8 = blocks(8);
  if (n8 > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  if (n8 >= 2 * lw_host::sm_count())
    return lw_launch(lw::qk_norm_rope_kernel<T, TT, HD, 8>, dim3((unsigned)n8), dim3(lw::kRopeThreads), 0, s, pdl, p);
  const long long n1 = blocks(1);
  return lw_launch(lw::qk_norm_rope_kernel<T, TT, HD, 1>, dim3((unsigned)n1), dim3(lw::kRopeThreads), 0, s, pdl, p);
}

template <typename T>
cudaError_t rope_dispatch(lw::RopeParams& p, int hd, bool f32_table, cudaStream_t s, bool pdl) {
  if (hd == 128) return f32_table ? rope_launch<T, float, 128>(p, s, pdl) : rope_launch<T, T, 128>(p, s, pdl);
  return f32_table ? rope_launch<T, float, 64>(p, s, pdl) : rope_launch<T, T, 64>(p, s, pdl);
}

}  // namespace

int lw_paged_rope_take_error() { return lw_tu_take_error(); }

extern "C" int lw_qk_norm_rope(const lw_qk_norm_rope_args* a, lw_stream_t stream) {
  if (!a) return LW_ERR_NULL_POINTER;
  int st = lw_host::check_cache(a->cache);
  if (st) return st;
  if (a->tokens < 0 || a->n_q_heads <= 0 || a->rope_rows < 0) return LW_ERR_BAD_SHAPE;
  if (!a->q_offsets && a->tokens != a->cache.batch) return LW_ERR_BAD_SHAPE;
  if ((a->q_weight == nullptr) != (a->k_weight == nullptr)) return LW_ERR_NULL_POINTER;
  if (a->rope_dtype != LW_DTYPE_F32 && a->rope_dtype != a->cache.dtype) return LW_ERR_UNSUPPORTED;
  if (a->tokens == 0) return LW_OK;
  if (a->cache.batch == 0) return LW_ERR_BAD_SHAPE;
  if (!a->q || !a->k || !a->v || !a->q_out || (a->rope_rows && (!a->rope_cos || !a->rope_sin)))
    return LW_ERR_NULL_POINTER;
  for (const void* ptr : {a->q, a->k, a->v, (const void*)a->q_out, a->rope_cos, a->rope_sin, a->q_weight, a->k_weight})
    if (!lw_host::aligned16(ptr)) return LW_ERR_ALIGNMENT;
  for (const long long* s : {a->q_strides, a->k_strides, a->v_strides, a->out_strides})
    if (!lw_host::strides8(s, 2)) return LW_ERR_ALIGNMENT;
  if (!lw_host::strides8(&a->rope_stride, 1)) return LW_ERR_ALIGNMENT;

  lw::RopeParams p = {};
  p.c = lw_host::view_of(a->cache);
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.q_t = a->q_strides[0];
  p.q_h = a->q_strides[1];
  p.k_t = a->k_strides[0];
  p.k_h = a->k_strides[1];
  p.v_t = a->v_strides[0];
  p.v_h = a->v_strides[1];
  p.out = a->q_out;
  p.o_t = a->out_strides[0];
  p.o_h = a->out_strides[1];
  p.T = a->tokens;
  p.nq = a->n_q_heads;
  p.off = a->q_offsets;
  p.cos = a->rope_cos;
  p.sin = a->rope_sin;
  p.rope_stride = a->rope_stride;
  p.rope_rows = a->rope_rows;
  p.qw = a->q_weight;
  p.kw = a->k_weight;
  p.eps = a->eps;
  p.zero_tail = a->zero_tail;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaGetLastError();
  const bool f32 = a->rope_dtype == LW_DTYPE_F32, pdl = a->pdl != 0;
  cudaError_t e = a->cache.dtype == LW_DTYPE_F16 ? rope_dispatch<__half>(p, a->cache.head_dim, f32, s, pdl)
                                                 : rope_dispatch<__nv_bfloat16>(p, a->cache.head_dim, f32, s, pdl);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? LW_OK : LW_ERR_LAUNCH;
}

// Norms of queries and keys for each head, rotation by position and the append
// to the paged cache, in one pass (lw_qk_norm_rope).
//
//   y = x * rsqrt(mean(x^2) + eps) * w,   o[d] = y[d] cos[p][d] + r[d] sin[p][d],
//   r = (-y[hd/2:], y[:hd/2])
//
// A group of hd / 16 lanes takes one token's run of up to HPG heads (queries,
// then keys, then values): each lane holds dims 8j .. 8j+7 and their rotation
// partners hd/2 + 8j .. + 7, so a head is two 16-byte loads and two 16-byte
// stores a lane, the rotation needs no exchange, and the mean is log2(hd / 16)
// shuffles. The angle's cosines and sines are loaded once per run. All of it in
// fp32 with one rounding at the store. Memory bound: every element is read
// once and written once.
#include "paged.cuh"

namespace lw {

struct RopeParams {
  PagedView c;
  const void *q, *k, *v;
  long long q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h;
  void* out;
  int T, nq, chunks;   // runs of heads per token
  const int* off;
  const void *cos, *sin;
  long long rope_stride;
  int rope_rows;
  const void *qw, *kw;
  float eps;
  int zero_tail;
};

template <typename T>
LW_DEV void load8(const T* p, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = Elem<T>::unpack(w[i]);
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}
template <>
LW_DEV void load8<float>(const float* p, float (&f)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
  f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

template <typename T>
LW_DEV void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = Elem<T>::unpack(w[i]);
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}

template <typename T>
LW_DEV uint4 pack8(const float (&f)[8]) {
  return make_uint4(Elem<T>::pack(f[0], f[1]), Elem<T>::pack(f[2], f[3]), Elem<T>::pack(f[4], f[5]),
                    Elem<T>::pack(f[6], f[7]));
}

constexpr int kRopeThreads = 256;

// T: element type; TT: type of the rotation table; HPG: heads per run.
template <typename T, typename TT, int HD, int HPG>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const RopeParams p) {
  constexpr int LPR = HD / 16;   // lanes per head
  pdl_wait();
  pdl_launch_dependents();
  const int j = threadIdx.x % LPR;
  const long long item = (long long)blockIdx.x * (kRopeThreads / LPR) + threadIdx.x / LPR;
  const long long t64 = item / p.chunks;
  if (t64 >= p.T) return;   // whole groups: shuffles below stay within a group
  const int t = (int)t64, h0 = (int)(item - t64 * p.chunks) * HPG;
  const int heads = p.nq + 2 * p.c.nkv;
  const unsigned gmask = (LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u)) << ((threadIdx.x & 31) / LPR * LPR);
  const int d_lo = 8 * j, d_hi = HD / 2 + 8 * j;

  // the run's heads, all loads in flight before the first use
  uint4 lo[HPG], hi[HPG];
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    const T* src;
    if (h < p.nq) src = static_cast<const T*>(p.q) + t * p.q_t + h * p.q_h;
    else if (h < p.nq + p.c.nkv) src = static_cast<const T*>(p.k) + t * p.k_t + (h - p.nq) * p.k_h;
    else src = static_cast<const T*>(p.v) + t * p.v_t + (h - p.nq - p.c.nkv) * p.v_h;
    lo[i] = *reinterpret_cast<const uint4*>(src + d_lo);
    hi[i] = *reinterpret_cast<const uint4*>(src + d_hi);
  }

  const int b = p.off ? row_sequence(p.off, p.c.B, t) : t;
  int pos = -1;
  if (b >= 0) {
    const int len = p.c.lens[b];
    pos = p.off ? len - p.off[b + 1] + t : len - 1;
  }
  const bool real = b >= 0 && pos >= 0;   // the row is a token of a sequence
  const bool turns = real && pos < p.rope_rows;
  if (!turns) {
    // past the table, or more new tokens than the length counts
    if ((real || (b >= 0 && p.off)) && j == 0) lw_record_error(LW_ERR_BAD_INDEX);
    if (p.zero_tail) {
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        if (h0 + i >= p.nq) break;
        T* dst = static_cast<T*>(p.out) + t * p.o_t + (h0 + i) * p.o_h;
        *reinterpret_cast<uint4*>(dst + d_lo) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + d_hi) = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  // where the token is kept (only the runs that reach keys or values ask)
  long long k_at = -1, v_at = -1;
  if (h0 + HPG > p.nq) {
    const int page = (pos >> p.c.page_shift) < p.c.table_width ? page_id(p.c, b, pos) : -1;
    if (page >= 0) {
      const int slot = pos & (p.c.page_size - 1);
      k_at = page * p.c.kp + slot * p.c.ks;
      v_at = page * p.c.vp + slot * p.c.vs;
    } else if (j == 0) {
      lw_record_error(LW_ERR_BAD_INDEX);
    }
  }
  float c_lo[8], c_hi[8], s_lo[8], s_hi[8];
  {
    const TT* cs = static_cast<const TT*>(p.cos) + pos * p.rope_stride;
    const TT* sn = static_cast<const TT*>(p.sin) + pos * p.rope_stride;
    load8(cs + d_lo, c_lo);
    load8(cs + d_hi, c_hi);
    load8(sn + d_lo, s_lo);
    load8(sn + d_hi, s_hi);
  }
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    if (h >= p.nq + p.c.nkv) {   // values are kept as they are
      if (v_at >= 0) {
        T* dst = static_cast<T*>(p.c.v) + v_at + (h - p.nq - p.c.nkv) * p.c.vh;
        *reinterpret_cast<uint4*>(dst + d_lo) = lo[i];
        *reinterpret_cast<uint4*>(dst + d_hi) = hi[i];
      }
      continue;
    }
    float x_lo[8], x_hi[8];
    unpack8<T>(lo[i], x_lo);
    unpack8<T>(hi[i], x_hi);
    const T* w = static_cast<const T*>(h < p.nq ? p.qw : p.kw);
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x_lo[e], x_lo[e], fmaf(x_hi[e], x_hi[e], ss));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(gmask, ss, o);
      const float r = rsqrtf(ss * (1.0f / HD) + p.eps);
      float w_lo[8], w_hi[8];
      load8(w + d_lo, w_lo);
      load8(w + d_hi, w_hi);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x_lo[e] = x_lo[e] * r * w_lo[e];
        x_hi[e] = x_hi[e] * r * w_hi[e];
      }
    }
    float y_lo[8], y_hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y_lo[e] = x_lo[e] * c_lo[e] - x_hi[e] * s_lo[e];
      y_hi[e] = x_hi[e] * c_hi[e] + x_lo[e] * s_hi[e];
    }
    T* dst;
    if (h < p.nq) {
      dst = static_cast<T*>(p.out) + t * p.o_t + h * p.o_h;
    } else {
      if (k_at < 0) continue;
      dst = static_cast<T*>(p.c.k) + k_at + (h - p.nq) * p.c.kh;
    }
    *reinterpret_cast<uint4*>(dst + d_lo) = pack8<T>(y_lo);
    *reinterpret_cast<uint4*>(dst + d_hi) = pack8<T>(y_hi);
  }
}

}  // namespace lw

namespace {

template <typename T, typename TT, int HD>
cudaError_t rope_launch(lw::RopeParams& p, cudaStream_t s, bool pdl) {
  constexpr int groups = lw::kRopeThreads / (HD / 16);
  const int heads = p.nq + 2 * p.c.nkv;
  auto blocks = [&](int hpg) {
    p.chunks = (heads + hpg - 1) / hpg;
    return ((long long)p.T * p.chunks + groups - 1) / groups;
  };
  // A run of 8 heads shares one load of the angles and keeps 16 loads in flight
  // a lane; a launch too small to give every SM work takes single heads.
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

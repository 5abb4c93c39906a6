// Attention of prompt chunks over the paged cache (lw_paged_attention with
// q_offsets): the newest tokens of every sequence against all it keeps, causal,
// with an optional window and first keys that stay visible.
//
// A CTA takes a tile of 64 rows = consecutive positions x the query heads of
// one kv head's group, so K and V are read once for the whole group, and
// walks the 64-key tiles any of its rows sees. S = Q K^T and O += P V with
// mma.sync, online softmax in fp32 per row.
//
// Keys that no row of the tile sees are zero-filled by the copy. A key that
// some rows see and others do not (the diagonal, the window's edge) meets the
// other rows with weight 0; if its value holds an infinity or a NaN, 0 * v would
// reach them, so the values of such tiles are scanned, non-finite ones are
// replaced by 0 and added afterwards to the rows that see them.
#include "paged.cuh"

namespace lw {

struct PromptParams {
  PagedView c;
  const void* q;
  void* out;
  long long q_t, q_h, o_t, o_h;
  int T, nq, group, rp;   // rp: positions per row tile
  const int* off;
  int window, sinks;
  float scale_log2;
  int zero_tail;
};

// Row tiles of the ragged batch: sequence b owns the slots from off[b] / rp + b
// on, at least as many as its rows need (ceil(n / rp) <= floor((off + n) / rp) -
// floor(off / rp) + 1), so a slot finds its sequence by bisection and the grid
// needs only T and B. Slots without rows exit.
LW_DEV bool find_row_tile(const PromptParams& p, int slot, int& b, int& i0, int& n) {
  int lo = 0, hi = p.c.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.off[mid] / p.rp + mid <= slot) lo = mid;
    else hi = mid;
  }
  b = lo;
  const int o = p.off[b];
  n = p.off[b + 1] - o;
  i0 = (slot - (o / p.rp + b)) * p.rp;
  return i0 >= 0 && i0 < n && o >= 0 && (long long)o + n <= p.T;
}

constexpr int kPmRows = 64, kPmKeys = 64, kPmThreads = 128;

template <typename T, int HD>
__global__ void __launch_bounds__(kPmThreads) paged_prompt_kernel(const PromptParams p) {
  constexpr int CPR = HD / 8;
  constexpr int kTileBytes = kPmKeys * HD * 2;
  extern __shared__ __align__(128) uint8_t smem[];   // 2 x (K tile, V tile)
  __shared__ uint8_t lost[2][kPmKeys / 16];          // 16-key groups whose page id is outside the pool
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  if (p.zero_tail) {
    for (int r = max(0, p.off[p.c.B]) + blockIdx.x; r < p.T; r += gridDim.x)
      for (int i = tid; i < p.group * CPR; i += kPmThreads)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + r * p.o_t + (kvh * p.group + i / CPR) * p.o_h +
                                  (i % CPR) * 8) = make_uint4(0, 0, 0, 0);
  }
  int b, i0, n;
  if (!find_row_tile(p, gridDim.x - 1 - blockIdx.x, b, i0, n)) return;   // the longest rows first
  const int tok0 = p.off[b] + i0;
  const int np = min(p.rp, n - i0);                  // positions of this tile
  const int len = seq_len(p.c, b);
  const int pos0 = p.c.lens[b] - n + i0;             // position of the first (negative: more rows than tokens)
  const int last = min(pos0 + np, len) - 1;          // the last position any row has
  const int lo0 = window_start(max(pos0, 0), p.window);
  if (pos0 < 0 && tid == 0) lw_record_error(LW_ERR_BAD_INDEX);
  const int hi_tile = last < 0 ? 0 : last / kPmKeys + 1;
  const int ns = min((p.sinks + kPmKeys - 1) / kPmKeys, lo0 / kPmKeys);
  const int w0 = lo0 / kPmKeys;
  const int nt = p.window > 0 ? ns + max(0, hi_tile - w0) : hi_tile;

  // rows of this lane: packed row r = (position r / group, head r % group)
  int row[2], pos[2];
  bool have[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    row[e] = warp * 16 + g + 8 * e;
    have[e] = row[e] < np * p.group;
    pos[e] = have[e] ? min(pos0 + row[e] / p.group, len - 1) : -1;
  }
  uint32_t qa[HD / 16][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const T* qp = static_cast<const T*>(p.q) + (long long)(tok0 + (have[e] ? row[e] / p.group : 0)) * p.q_t +
                  (long long)(kvh * p.group + (have[e] ? row[e] % p.group : 0)) * p.q_h + 2 * t;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      qa[k][e] = have[e] ? *reinterpret_cast<const uint32_t*>(qp + k * 16) : 0u;
      qa[k][2 + e] = have[e] ? *reinterpret_cast<const uint32_t*>(qp + k * 16 + 8) : 0u;
    }
  }
  auto key_of = [&](int i) { return (p.window > 0 && i >= ns ? w0 + i - ns : i) * kPmKeys; };
  auto tile_sees = [&](int key) { return key <= last && (p.window <= 0 || key >= lo0 || key < p.sinks); };
  const uint32_t sm = smem_u32(smem);
  auto load = [&](int i) {
    if (i < nt) {
      const int key0 = key_of(i);
      const uint32_t dst = sm + (i & 1) * 2 * kTileBytes;
      if (tid < kPmKeys / 16) {
        bool bad = false;
        const int first = key0 + tid * 16;   // the group's first key that some row sees
        for (int k = first; k < first + 16; ++k)
          if (tile_sees(k)) {
            bad = page_id(p.c, b, k) < 0;
            break;
          }
        lost[i & 1][tid] = bad;
      }
      for (int x = tid; x < kPmKeys * CPR; x += kPmThreads) {
        const int r = x / CPR, c = x % CPR, key = key0 + r;
        const int page = tile_sees(key) ? page_id(p.c, b, key) : -1;
        const int slot = key & (p.c.page_size - 1);
        const T *kp = static_cast<const T*>(p.q), *vp = kp;   // not read when there is no page
        if (page >= 0) {
          kp = static_cast<const T*>(p.c.k) + page * p.c.kp + kvh * p.c.kh + slot * p.c.ks + c * 8;
          vp = static_cast<const T*>(p.c.v) + page * p.c.vp + kvh * p.c.vh + slot * p.c.vs + c * 8;
        }
        const uint32_t at = dst + (uint32_t)(r * (HD * 2) + ((c ^ (r & 7)) << 4));
        cp_async16(at, kp, page >= 0);
        cp_async16(at + kTileBytes, vp, page >= 0);
      }
    }
    cp_async_commit();
  };
  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  load(0);
  for (int i = 0; i < nt; ++i) {
    load(i + 1);
    cp_async_wait<1>();
    __syncthreads();
    const int key0 = key_of(i);
    const uint32_t kt = sm + (i & 1) * 2 * kTileBytes, vt = kt + kTileBytes;
    uint8_t* vptr = smem + (i & 1) * 2 * kTileBytes + kTileBytes;
    // a tile that some row does not see whole
    const bool partial = key0 + kPmKeys - 1 > pos0 || (p.window > 0 && key0 <= last - p.window);
    bool odd = false;
    if (partial) {
      bool mine = false;
      for (int x = tid; x < kPmKeys * CPR; x += kPmThreads) {
        const uint4 v = lds128(vptr + x * 16);
        mine |= has_nonfinite<T>(v.x) || has_nonfinite<T>(v.y) || has_nonfinite<T>(v.z) || has_nonfinite<T>(v.w);
      }
      odd = __syncthreads_or(mine);
    }
    const uint8_t* gone = lost[i & 1];
    auto sees = [&](int key, int e) {
      return key <= pos[e] && !gone[(key - key0) >> 4] && (p.window <= 0 || pos[e] - key < p.window || key < p.sinks);
    };
    if (odd) {
      // each lane adds its rows' and columns' non-finite values, then they are cleared
#pragma unroll
      for (int d8 = 0; d8 < HD / 8; ++d8) {
        for (int r = 0; r < kPmKeys; ++r) {
          const uint32_t u = *reinterpret_cast<const uint32_t*>(vptr + r * (HD * 2) + ((d8 ^ (r & 7)) << 4) + 4 * t);
          if (!has_nonfinite<T>(u)) continue;
          const float2 v = Elem<T>::unpack(u);
          for (int e = 0; e < 2; ++e)
            if (sees(key0 + r, e)) {
              if (!isfinite(v.x)) o[d8][2 * e] += v.x;
              if (!isfinite(v.y)) o[d8][2 * e + 1] += v.y;
            }
        }
      }
      __syncthreads();
      for (int x = tid; x < kPmKeys * CPR * 8; x += kPmThreads) {
        uint16_t* h = reinterpret_cast<uint16_t*>(vptr) + x;
        if ((*h & Elem<T>::kExpMask) == Elem<T>::kExpMask) *h = 0;
      }
      __syncthreads();
    }
    float sc[kPmKeys / 8][4];
#pragma unroll
    for (int x = 0; x < kPmKeys / 8; ++x) sc[x][0] = sc[x][1] = sc[x][2] = sc[x][3] = 0.f;
    {
      const int r8 = (lane >> 4) * 8 + (lane & 7), cb = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int x = 0; x < kPmKeys / 16; ++x) {
          const int r = x * 16 + r8;
          uint32_t f[4];
          ldmatrix_x4(kt + (uint32_t)(r * (HD * 2) + (((2 * k + cb) ^ (r & 7)) << 4)), f);
          mma_16816<T>(sc[2 * x], qa[k][0], qa[k][1], qa[k][2], qa[k][3], f[0], f[1]);
          mma_16816<T>(sc[2 * x + 1], qa[k][0], qa[k][1], qa[k][2], qa[k][3], f[2], f[3]);
        }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int x = 0; x < kPmKeys / 8; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[x][e] = sees(key0 + x * 8 + 2 * t + (e & 1), e >> 1) ? sc[x][e] * p.scale_log2 : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], sc[x][e]);
      }
    float corr[2], base[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
      const float mn = fmaxf(m[e], mx[e]);
      corr[e] = m[e] == -INFINITY ? 1.f : exp2f(m[e] - mn);
      base[e] = mn == -INFINITY ? 0.f : mn;
      m[e] = mn;
      l[e] *= corr[e];
    }
#pragma unroll
    for (int x = 0; x < kPmKeys / 8; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[x][e] = exp2f(sc[x][e] - base[e >> 1]);
        l[e >> 1] += sc[x][e];
      }
#pragma unroll
    for (int x = 0; x < HD / 8; ++x) {
      o[x][0] *= corr[0];
      o[x][1] *= corr[0];
      o[x][2] *= corr[1];
      o[x][3] *= corr[1];
    }
    {
      const int r8 = ((lane >> 3) & 1) * 8 + (lane & 7), cb = lane >> 4;
#pragma unroll
      for (int x = 0; x < kPmKeys / 16; ++x) {
        const uint32_t a0 = Elem<T>::pack(sc[2 * x][0], sc[2 * x][1]), a1 = Elem<T>::pack(sc[2 * x][2], sc[2 * x][3]);
        const uint32_t a2 = Elem<T>::pack(sc[2 * x + 1][0], sc[2 * x + 1][1]);
        const uint32_t a3 = Elem<T>::pack(sc[2 * x + 1][2], sc[2 * x + 1][3]);
        const int r = x * 16 + r8;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          uint32_t f[4];
          ldmatrix_x4_t(vt + (uint32_t)(r * (HD * 2) + (((2 * d + cb) ^ (r & 7)) << 4)), f);
          mma_16816<T>(o[2 * d], a0, a1, a2, a3, f[0], f[1]);
          mma_16816<T>(o[2 * d + 1], a0, a1, a2, a3, f[2], f[3]);
        }
      }
    }
    __syncthreads();   // the stage is free for tile i + 2
  }
  cp_async_wait<0>();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    if (!have[e]) continue;
    const float inv = l[e] == 0.f ? 0.f : 1.f / l[e];
    T* dst = static_cast<T*>(p.out) + (long long)(tok0 + row[e] / p.group) * p.o_t +
             (long long)(kvh * p.group + row[e] % p.group) * p.o_h + 2 * t;
#pragma unroll
    for (int x = 0; x < HD / 8; ++x)
      *reinterpret_cast<uint32_t*>(dst + x * 8) = Elem<T>::pack(o[x][2 * e] * inv, o[x][2 * e + 1] * inv);
  }
}

}  // namespace lw

size_t lw_paged_decode_workspace(const lw_paged_attention_args* a);
int lw_paged_decode(const lw_paged_attention_args* a, cudaStream_t s);

namespace {

int check(const lw_paged_attention_args* a) {
  if (!a) return LW_ERR_NULL_POINTER;
  int st = lw_host::check_cache(a->cache);
  if (st) return st;
  if (a->tokens < 0 || a->n_q_heads <= 0 || a->n_q_heads % a->cache.n_kv_heads || a->sinks < 0) return LW_ERR_BAD_SHAPE;
  if (!a->q_offsets && a->tokens != a->cache.batch) return LW_ERR_BAD_SHAPE;
  if (a->q_offsets && a->n_q_heads / a->cache.n_kv_heads > lw::kPmRows) return LW_ERR_UNSUPPORTED;
  if (a->tokens == 0) return LW_OK;
  if (a->cache.batch == 0) return LW_ERR_BAD_SHAPE;
  if (!a->q || !a->out) return LW_ERR_NULL_POINTER;
  if (!lw_host::aligned16(a->q) || !lw_host::aligned16(a->out) || !lw_host::strides8(a->q_strides, 2) ||
      !lw_host::strides8(a->out_strides, 2) || (reinterpret_cast<uintptr_t>(a->q_offsets) & 3u))
    return LW_ERR_ALIGNMENT;
  return LW_OK;
}

template <typename T, int HD>
cudaError_t prompt_launch(const lw::PromptParams& p, cudaStream_t s, bool pdl) {
  constexpr int smem = 4 * lw::kPmKeys * HD * 2;
  auto kern = lw::paged_prompt_kernel<T, HD>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return lw_launch(kern, dim3((unsigned)(p.T / p.rp + p.c.B), (unsigned)p.c.nkv), dim3(lw::kPmThreads), smem, s, pdl,
                   p);
}

}  // namespace

int lw_paged_prompt_take_error() { return lw_tu_take_error(); }

extern "C" {

size_t lw_paged_attention_workspace_size(const lw_paged_attention_args* a) {
  if (check(a) != LW_OK || a->tokens == 0) return 0;
  return a->q_offsets ? 0 : lw_paged_decode_workspace(a);
}

int lw_paged_attention(const lw_paged_attention_args* a, lw_stream_t stream) {
  const int st = check(a);
  if (st || a->tokens == 0) return st;
  const size_t need = lw_paged_attention_workspace_size(a);
  if (need && (!a->workspace || a->workspace_bytes < need)) return LW_ERR_WORKSPACE;
  if (need && (reinterpret_cast<uintptr_t>(a->workspace) & 255u)) return LW_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaGetLastError();
  if (!a->q_offsets) return lw_paged_decode(a, s);
  if (a->cache.n_kv_heads > 65535) return LW_ERR_UNSUPPORTED;
  lw::PromptParams p = {};
  p.c = lw_host::view_of(a->cache);
  p.q = a->q;
  p.out = a->out;
  p.q_t = a->q_strides[0];
  p.q_h = a->q_strides[1];
  p.o_t = a->out_strides[0];
  p.o_h = a->out_strides[1];
  p.T = a->tokens;
  p.nq = a->n_q_heads;
  p.group = a->n_q_heads / a->cache.n_kv_heads;
  p.rp = lw::kPmRows / p.group;
  p.off = a->q_offsets;
  p.window = a->window;
  p.sinks = a->sinks;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.zero_tail = a->zero_tail;
  const bool pdl = a->pdl != 0;
  cudaError_t e;
  if (a->cache.dtype == LW_DTYPE_F16)
    e = a->cache.head_dim == 128 ? prompt_launch<__half, 128>(p, s, pdl) : prompt_launch<__half, 64>(p, s, pdl);
  else
    e = a->cache.head_dim == 128 ? prompt_launch<__nv_bfloat16, 128>(p, s, pdl)
                                 : prompt_launch<__nv_bfloat16, 64>(p, s, pdl);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? LW_OK : LW_ERR_LAUNCH;
}

}  // extern "C"

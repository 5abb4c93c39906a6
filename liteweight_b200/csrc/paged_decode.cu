// Attention of one new token per sequence over the paged cache
// (lw_paged_attention without q_offsets): split over the cache's length, joined.
//
//   out[b][h] = sum_j softmax_j(scale * q[b][h] . k_j) v_j  over the keys j that
//   position p = kv_lens[b] - 1 sees.
//
// Bound by reading the visible keys and values once. The work is cut into
// tiles of 16 consecutive token positions (one page each: a page is a multiple
// of 16 slots) of one item = (sequence, kv head, block of up to 16 query heads
// of its group). All items' tiles form one line, and every CTA of a grid of one
// per SM takes an equal run of it, so sequences of any lengths keep all SMs
// equally busy; a run's eight warps take its tiles in turn. A warp streams its
// tiles through a private ring of shared-memory stages (cp.async, no CTA
// barrier), computes S = Q K^T and O += P V with mma.sync (the query heads of
// the group are the MMA's rows, so K and V are read once for all of them) and
// keeps an online softmax in fp32. At the end of an item the warps merge in
// shared memory; an item that lies in one run is written at once, otherwise each
// run leaves (max, sum, fp32 accumulator) in the workspace and a second kernel
// joins them in order: the same bits on every call.
//
// Hidden keys of a tile are zero-filled by the copy, so what their slots hold
// (NaN included) never meets the tensor cores.
#include "paged.cuh"

namespace lw {

constexpr int kPdWarps = 8;
constexpr int kPdThreads = kPdWarps * 32;
constexpr int kPdTile = 16;      // keys per tile
constexpr int kPdRows = 16;      // query heads per item (MMA rows)
constexpr int kPdMinRun = 8;     // tiles a CTA takes at least: one per warp

struct PagedDecodeParams {
  PagedView c;
  const void* q;
  void* out;
  long long q_b, q_h, o_b, o_h;
  int nq, group, hblocks;   // group = nq / nkv; hblocks = blocks of kPdRows heads in it
  int window, sinks;
  float scale_log2;
  int grid;                 // CTAs of the first kernel
  int2* meta;               // [items]: first run << 1 | starts inside it, runs (0: nothing to join)
  float* part;              // [2 * grid][kPdRows][HD + 2]
};

// The tiles a sequence's newest position sees: [0, ns) and [w0, w0 + nt - ns).
struct TileSpan {
  int len, lo, sinks;   // keys [lo, len) and [0, sinks) are visible
  int ns, w0, nt;
};

LW_DEV TileSpan tile_span(const PagedDecodeParams& p, int len) {
  TileSpan s;
  s.len = len;
  s.lo = window_start(len - 1, p.window);
  s.sinks = min(p.sinks, s.lo);
  s.w0 = s.lo / kPdTile;
  s.ns = min((s.sinks + kPdTile - 1) / kPdTile, s.w0);
  s.nt = len > 0 ? s.ns + (len + kPdTile - 1) / kPdTile - s.w0 : 0;
  return s;
}

// A place on the line of tiles: sequence b, its span, item within it.
struct LineCursor {
  int b, hh;            // hh: (kv head, head block) within the sequence
  long long item0;      // first tile of the item on the line
  TileSpan span;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kPdThreads, 1) paged_decode_kernel(const PagedDecodeParams p) {
  constexpr int CPR = HD / 8;                      // 16-byte chunks per row
  constexpr int kTileBytes = kPdTile * HD * 2;     // K or V of a tile
  constexpr int kStages = 24576 / (2 * kTileBytes);   // 24 KB of ring per warp: 3 stages (hd 128), 6 (hd 64)
  constexpr int ROWS_PER_INSTR = 32 / CPR;         // rows one cp.async of the warp covers
  constexpr int COPIES = kPdTile / ROWS_PER_INSTR;
  extern __shared__ __align__(128) uint8_t smem[];
  float* sm_o = reinterpret_cast<float*>(smem + kPdWarps * kStages * 2 * kTileBytes);   // [warps][8][HD]
  __shared__ float sm_m[kPdWarps][kPdRows], sm_l[kPdWarps][kPdRows];
  __shared__ long long sm_scan[kPdWarps];
  __shared__ long long sm_first;   // tiles before sm_b
  __shared__ int sm_b;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int H = p.c.nkv * p.hblocks;
  pdl_wait();
  pdl_launch_dependents();

  // ---- this CTA's run of the line: a scan of the sequences' tile counts
  const int per_thread = (p.c.B + kPdThreads - 1) / kPdThreads;
  const int b_lo = min(p.c.B, tid * per_thread), b_hi = min(p.c.B, b_lo + per_thread);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += (long long)tile_span(p, seq_len(p.c, b)).nt * H;
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sm_scan[warp] = incl;
  __syncthreads();
  long long total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kPdWarps; ++w) {
    if (w < warp) before += sm_scan[w];
    total += sm_scan[w];
  }
  long long run = (total + p.grid - 1) / p.grid;
  if (run < kPdMinRun) run = kPdMinRun;
  const long long r0 = blockIdx.x * run, r1 = min(total, r0 + run);
  if (r0 >= r1) return;   // the whole CTA
  {
    long long excl = before + incl - mine;
    if (mine > 0 && excl <= r0 && r0 < excl + mine) {
      int b = b_lo;
      for (; b < b_hi - 1; ++b) {
        const long long n = (long long)tile_span(p, seq_len(p.c, b)).nt * H;
        if (r0 < excl + n) break;
        excl += n;
      }
      sm_b = b;
      sm_first = excl;
    }
  }
  __syncthreads();

  LineCursor start;
  start.b = sm_b;
  start.span = tile_span(p, seq_len(p.c, start.b));
  start.hh = (int)((r0 - sm_first) / start.span.nt);
  start.item0 = sm_first + (long long)start.hh * start.span.nt;
  auto advance = [&](LineCursor& c) {   // to the next item with tiles (one exists while its first tile < total)
    c.item0 += c.span.nt;
    if (++c.hh == H) {
      c.hh = 0;
      do {
        ++c.b;
        c.span = tile_span(p, seq_len(p.c, c.b));
      } while (c.span.nt == 0);
    }
  };

  // ---- the warp's copies: tile `tile` of the line into ring stage `st`
  const uint32_t ring = smem_u32(smem) + warp * (kStages * 2 * kTileBytes);
  const int c_row = lane / CPR, c_chunk = lane % CPR;
  LineCursor ahead = start;
  uint32_t lost = 0;   // bit st: the stage's page id was outside the pool, its keys are hidden
  auto issue = [&](long long tile, int st) {
    lost &= ~(1u << st);
    if (tile < r1) {
      while (tile >= ahead.item0 + ahead.span.nt) advance(ahead);
      const int ti = (int)(tile - ahead.item0);
      const TileSpan& sp = ahead.span;
      const int key0 = (ti < sp.ns ? ti : sp.w0 + ti - sp.ns) * kPdTile;
      const int page = page_id(p.c, ahead.b, key0);
      const int slot0 = key0 & (p.c.page_size - 1);
      if (page < 0) lost |= 1u << st;
      const int kvh = ahead.hh / p.hblocks;
      const T* kp = static_cast<const T*>(p.c.k) + page * p.c.kp + kvh * p.c.kh + slot0 * p.c.ks + c_chunk * 8;
      const T* vp = static_cast<const T*>(p.c.v) + page * p.c.vp + kvh * p.c.vh + slot0 * p.c.vs + c_chunk * 8;
      const uint32_t dst = ring + st * (2 * kTileBytes);
#pragma unroll
      for (int i = 0; i < COPIES; ++i) {
        const int r = c_row + i * ROWS_PER_INSTR, key = key0 + r;
        const bool ok = page >= 0 && key < sp.len && (key >= sp.lo || key < sp.sinks);
        const uint32_t at = dst + (uint32_t)(r * (HD * 2) + ((c_chunk ^ (r & 7)) << 4));
        cp_async16(at, ok ? kp + r * p.c.ks : static_cast<const T*>(p.q), ok);
        cp_async16(at + kTileBytes, ok ? vp + r * p.c.vs : static_cast<const T*>(p.q), ok);
      }
    }
    cp_async_commit();   // one group per call, empty past the run's end
  };
  long long next = r0 + warp;   // next tile to issue
#pragma unroll
  for (int s = 0; s < kStages; ++s, next += kPdWarps) issue(next, s);

  // ---- items of the run
  LineCursor cur = start;
  long long tile = r0 + warp;
  int st = 0;
  for (;;) {
    const long long seg0 = max(cur.item0, r0), seg1 = min(cur.item0 + cur.span.nt, r1);
    const int kvh = cur.hh / p.hblocks, hb = cur.hh - kvh * p.hblocks;
    const int rows = min(kPdRows, p.group - hb * kPdRows);
    const int head0 = kvh * p.group + hb * kPdRows;

    uint32_t qa[HD / 16][4];
    {
      const T* qp = static_cast<const T*>(p.q) + cur.b * p.q_b + (long long)head0 * p.q_h + 2 * t;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        qa[k][0] = g < rows ? *reinterpret_cast<const uint32_t*>(qp + g * p.q_h + k * 16) : 0u;
        qa[k][2] = g < rows ? *reinterpret_cast<const uint32_t*>(qp + g * p.q_h + k * 16 + 8) : 0u;
        qa[k][1] = g + 8 < rows ? *reinterpret_cast<const uint32_t*>(qp + (g + 8) * p.q_h + k * 16) : 0u;
        qa[k][3] = g + 8 < rows ? *reinterpret_cast<const uint32_t*>(qp + (g + 8) * p.q_h + k * 16 + 8) : 0u;
      }
    }
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};   // rows g, g + 8

    for (; tile < seg1; tile += kPdWarps) {
      cp_async_wait<kStages - 1>();   // the oldest group has landed
      __syncwarp();
      const uint32_t kt = ring + st * (2 * kTileBytes), vt = kt + kTileBytes;
      const int ti = (int)(tile - cur.item0);
      const TileSpan& sp = cur.span;
      const int key0 = (ti < sp.ns ? ti : sp.w0 + ti - sp.ns) * kPdTile;
      const bool kept = !((lost >> st) & 1u);
      auto sees = [&](int key) { return kept && key < sp.len && (key >= sp.lo || key < sp.sinks); };
      float sc[2][4] = {};
      {
        // matrices of 8 keys x 8 dims: (keys 0-7 | 8-15) x (dims 0-7 | 8-15) of a k-step
        const int r = (lane >> 4) * 8 + (lane & 7), cb = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t b[4];
          ldmatrix_x4(kt + (uint32_t)(r * (HD * 2) + (((2 * k + cb) ^ (r & 7)) << 4)), b);
          mma_16816<T>(sc[0], qa[k][0], qa[k][1], qa[k][2], qa[k][3], b[0], b[1]);
          mma_16816<T>(sc[1], qa[k][0], qa[k][1], qa[k][2], qa[k][3], b[2], b[3]);
        }
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n * 8 + 2 * t + (e & 1);
          sc[n][e] = sees(key) ? sc[n][e] * p.scale_log2 : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], sc[n][e]);
        }
      float corr[2], base[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float mn = fmaxf(m[r], mx[r]);
        corr[r] = m[r] == -INFINITY ? 0.f : exp2f(m[r] - mn);   // nothing summed yet: nothing to keep
        base[r] = mn == -INFINITY ? 0.f : mn;   // no key seen yet: every weight is 0
        m[r] = mn;
        l[r] *= corr[r];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[n][e] = exp2f(sc[n][e] - base[e >> 1]);
          l[e >> 1] += sc[n][e];
        }
      // the weights lie in [0, 1]: rounded to T for the second product, half a
      // step each, averaged over the keys; their sum stays in fp32
      const uint32_t a0 = Elem<T>::pack(sc[0][0], sc[0][1]), a1 = Elem<T>::pack(sc[0][2], sc[0][3]);
      const uint32_t a2 = Elem<T>::pack(sc[1][0], sc[1][1]), a3 = Elem<T>::pack(sc[1][2], sc[1][3]);
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        o[i][0] *= corr[0];
        o[i][1] *= corr[0];
        o[i][2] *= corr[1];
        o[i][3] *= corr[1];
      }
      {
        const int r = ((lane >> 3) & 1) * 8 + (lane & 7), cb = lane >> 4;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          uint32_t b[4];
          ldmatrix_x4_t(vt + (uint32_t)(r * (HD * 2) + (((2 * d + cb) ^ (r & 7)) << 4)), b);
          mma_16816<T>(o[2 * d], a0, a1, a2, a3, b[0], b[1]);
          mma_16816<T>(o[2 * d + 1], a0, a1, a2, a3, b[2], b[3]);
        }
      }
      __syncwarp();   // every lane has read the stage
      issue(next, st);
      next += kPdWarps;
      if (++st == kStages) st = 0;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }

    // ---- the item's end in this run: the warps merge, eight rows at a time
    const bool whole = seg0 == cur.item0 && seg1 == cur.item0 + cur.span.nt;
    const int item = cur.b * H + cur.hh;
    const bool head_slot = seg0 == r0;
    float* slot = p.part + (long long)(2 * blockIdx.x + (head_slot ? 0 : 1)) * kPdRows * (HD + 2);
    if (tid == 0 && seg0 == cur.item0) {
      const long long last = (cur.item0 + cur.span.nt - 1) / run;
      p.meta[item] = make_int2((int)blockIdx.x * 2 + (head_slot ? 0 : 1), whole ? 0 : (int)(last - blockIdx.x) + 1);
    }
    if (t == 0) {
      sm_m[warp][g] = m[0];
      sm_m[warp][g + 8] = m[1];
      sm_l[warp][g] = l[0];
      sm_l[warp][g + 8] = l[1];
    }
    for (int half = 0; half < 2 && half * 8 < rows; ++half) {
      float* mine_o = sm_o + (warp * 8 + g) * HD + 2 * t;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
        *reinterpret_cast<float2*>(mine_o + i * 8) =
            half ? make_float2(o[i][2], o[i][3]) : make_float2(o[i][0], o[i][1]);
      __syncthreads();
      const int n = min(8, rows - half * 8);
      for (int i = tid; i < n * (HD / 2); i += kPdThreads) {
        const int r = i / (HD / 2), d = (i - r * (HD / 2)) * 2, row = half * 8 + r;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kPdWarps; ++w) M = fmaxf(M, sm_m[w][row]);
        float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kPdWarps; ++w) {
          const float f = sm_m[w][row] == -INFINITY ? 0.f : exp2f(sm_m[w][row] - M);   // a warp without tiles adds nothing
          const float2 v = *reinterpret_cast<const float2*>(sm_o + (w * 8 + r) * HD + d);
          L = fmaf(sm_l[w][row], f, L);
          x = fmaf(v.x, f, x);
          y = fmaf(v.y, f, y);
        }
        if (whole) {
          T* dst = static_cast<T*>(p.out) + cur.b * p.o_b + (long long)(head0 + row) * p.o_h + d;
          *reinterpret_cast<uint32_t*>(dst) = L == 0.f ? 0u : Elem<T>::pack(x / L, y / L);
        } else {
          float* dst = slot + row * (HD + 2);
          *reinterpret_cast<float2*>(dst + 2 + d) = make_float2(x, y);
          if (d == 0) {
            dst[0] = M;
            dst[1] = L;
          }
        }
      }
      __syncthreads();   // the buffers are free again
    }
    if (seg1 == r1) break;
    advance(cur);
  }
}

// Joins the runs of every item that was split, in the order of the line, and
// writes zeros for sequences without a visible key. One block per item.
template <typename T, int HD>
__global__ void __launch_bounds__(HD) paged_join_kernel(const PagedDecodeParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int H = p.c.nkv * p.hblocks;
  const int b = blockIdx.x / H, hh = blockIdx.x - b * H;
  const int kvh = hh / p.hblocks, hb = hh - kvh * p.hblocks;
  const int rows = min(kPdRows, p.group - hb * kPdRows);
  T* dst = static_cast<T*>(p.out) + b * p.o_b + (long long)(kvh * p.group + hb * kPdRows) * p.o_h;
  const int d = (threadIdx.x % (HD / 2)) * 2;
  if (seq_len(p.c, b) == 0) {
    for (int r = threadIdx.x / (HD / 2); r < rows; r += 2) *reinterpret_cast<uint32_t*>(dst + r * p.o_h + d) = 0u;
    return;
  }
  const int2 mt = p.meta[blockIdx.x];
  if (mt.y == 0) return;   // written by the one run that holds it
  for (int r = threadIdx.x / (HD / 2); r < rows; r += 2) {
    auto slot = [&](int i) {
      const int s = i == 0 ? mt.x : 2 * ((mt.x >> 1) + i);
      return p.part + ((long long)s * kPdRows + r) * (HD + 2);
    };
    float M = -INFINITY;
    for (int i = 0; i < mt.y; ++i) M = fmaxf(M, slot(i)[0]);
    float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll 4
    for (int i = 0; i < mt.y; ++i) {
      const float* s = slot(i);
      const float f = s[0] == -INFINITY ? 0.f : exp2f(s[0] - M);
      const float2 v = *reinterpret_cast<const float2*>(s + 2 + d);
      L = fmaf(s[1], f, L);
      x = fmaf(v.x, f, x);
      y = fmaf(v.y, f, y);
    }
    *reinterpret_cast<uint32_t*>(dst + r * p.o_h + d) = L == 0.f ? 0u : Elem<T>::pack(x / L, y / L);
  }
}

}  // namespace lw

namespace {

struct DecodePlan {
  int group, hblocks, grid;
  long long items;
  size_t part_off, bytes;
};

DecodePlan decode_plan(const lw_paged_attention_args* a) {
  DecodePlan d;
  d.group = a->n_q_heads / a->cache.n_kv_heads;
  d.hblocks = (d.group + lw::kPdRows - 1) / lw::kPdRows;
  d.items = (long long)a->cache.batch * a->cache.n_kv_heads * d.hblocks;
  d.grid = lw_host::sm_count();
  d.part_off = ((size_t)d.items * sizeof(int2) + 255) & ~(size_t)255;
  d.bytes = d.part_off + (size_t)2 * d.grid * lw::kPdRows * (a->cache.head_dim + 2) * sizeof(float);
  return d;
}

template <typename T, int HD>
cudaError_t decode_launch(const lw::PagedDecodeParams& p, long long items, cudaStream_t s, bool pdl) {
  constexpr int smem = lw::kPdWarps * 24576 + lw::kPdWarps * 8 * HD * (int)sizeof(float);
  auto kern = lw::paged_decode_kernel<T, HD>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  e = lw_launch(kern, dim3(p.grid), dim3(lw::kPdThreads), smem, s, pdl, p);
  if (e != cudaSuccess) return e;
  return lw_launch(lw::paged_join_kernel<T, HD>, dim3((unsigned)items), dim3(HD), 0, s, true, p);
}

}  // namespace

int lw_paged_decode_take_error() { return lw_tu_take_error(); }

// The form without q_offsets (arguments checked by lw_paged_attention).
size_t lw_paged_decode_workspace(const lw_paged_attention_args* a) { return decode_plan(a).bytes; }

int lw_paged_decode(const lw_paged_attention_args* a, cudaStream_t s) {
  const DecodePlan d = decode_plan(a);
  if (d.items > 0x7FFFFFFFll) return LW_ERR_BAD_SHAPE;
  lw::PagedDecodeParams p = {};
  p.c = lw_host::view_of(a->cache);
  p.q = a->q;
  p.out = a->out;
  p.q_b = a->q_strides[0];
  p.q_h = a->q_strides[1];
  p.o_b = a->out_strides[0];
  p.o_h = a->out_strides[1];
  p.nq = a->n_q_heads;
  p.group = d.group;
  p.hblocks = d.hblocks;
  p.window = a->window;
  p.sinks = a->sinks;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.grid = d.grid;
  p.meta = static_cast<int2*>(a->workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + d.part_off);
  const bool pdl = a->pdl != 0;
  cudaError_t e;
  if (a->cache.dtype == LW_DTYPE_F16)
    e = a->cache.head_dim == 128 ? decode_launch<__half, 128>(p, d.items, s, pdl)
                                 : decode_launch<__half, 64>(p, d.items, s, pdl);
  else
    e = a->cache.head_dim == 128 ? decode_launch<__nv_bfloat16, 128>(p, d.items, s, pdl)
                                 : decode_launch<__nv_bfloat16, 64>(p, d.items, s, pdl);
  return e == cudaSuccess ? LW_OK : LW_ERR_LAUNCH;
}

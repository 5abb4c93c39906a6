// Attention of one new token per sequence over the paged cache
// (lw_paged_attention without q_offsets): split over the cache's length, joined.
//
//   out[b][h] = sum_j softmax_j(scale * q[b][h] . k_j) v_j  over the keys j that
//   position p = kv_lens[b] - 1 sees.
//
// Bound by reading the visible keys and values once. The work is cut into
// tiles of 16 consecutive token positions (one page each: a page is a multiple
// of 16 slots) of one item = (sequence, kv head, block of up to ROWS query
// heads of its group). A warp streams tiles through a private ring of
// shared-memory stages (cp.async, no CTA barrier), computes S = Q K^T and
// O += P V with mma.sync (the query heads are the MMA's rows, so K and V are
// read once for all of them) and keeps an online softmax in fp32.
//
// Long or many sequences: all items' tiles form one line, and every warp of a
// grid of one CTA per SM takes an equal run of it, so sequences of any lengths
// keep all SMs equally busy. An item that lies in one run is written by its
// warp. Other pieces wait in shared memory until the CTA's warps are done; those
// of one item are merged there, and what continues in another CTA is left as
// (max, sum, fp32 accumulator) in the workspace, which a second kernel joins in
// order: the same bits on every call.
//
// Few short sequences: a cluster of up to eight CTAs takes an item and merges
// through distributed shared memory: one launch, no workspace.
//
// Hidden keys of a tile are zero-filled by the copy, so what their slots hold
// (NaN included) never meets the tensor cores.
#include <cooperative_groups.h>

#include <algorithm>

#include "paged.cuh"

namespace lw {

constexpr int kPdWarps = 8;
constexpr int kPdThreads = kPdWarps * 32;
constexpr int kPdTile = 16;      // keys per tile

struct PagedDecodeParams {
  PagedView c;
  const void* q;
  void* out;
  long long q_b, q_h, o_b, o_h;
  int group, hblocks;       // group = query heads per kv head; hblocks = blocks of ROWS heads in it
  int window, sinks;
  float scale_log2;
  int2* meta;               // [grid]: the item that begins in this CTA and ends in another, CTAs that hold it (or 0)
  float* part;              // [2 * grid][ROWS][HD + 8]
};

// The tiles a sequence's newest position sees: [0, ns) and [w0, w0 + nt - ns).
struct TileSpan {
  int len, lo, sinks;   // keys [lo, len) and [0, sinks) are visible
  int ns, w0, nt;
  LW_DEV int key0(int tile) const { return (tile < ns ? tile : w0 + tile - ns) * kPdTile; }
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

// Sizes of a kernel's shared memory: a ring per warp, then pieces [warps][ROWS][HD + 8]
// (accumulator, maximum, sum; the stride keeps the fragment stores off each other's banks).
template <int HD, int ROWS>
struct DecodeShape {
  static constexpr int kTileBytes = kPdTile * HD * 2;           // K or V of a tile
  static constexpr int kRing = ROWS == 8 ? 24576 : 16384;       // per warp
  static constexpr int kStages = kRing / (2 * kTileBytes);
  static constexpr int kStride = HD + 8;
  static constexpr int kPiece = ROWS * kStride;                 // floats
  static constexpr int kBytes = kPdWarps * (kRing + kPiece * 4);
};

// One warp's share of an item: queries as MMA fragments, the online softmax of
// rows g and g + 8 (g + 8 with ROWS = 16 only), the accumulator.
template <typename T, int HD, int ROWS>
struct WarpItem {
  using S = DecodeShape<HD, ROWS>;
  static constexpr int R = ROWS / 8;
  uint32_t qa[HD / 16][2 * R];
  float o[HD / 8][4];
  float m[R], l[R];

  LW_DEV static void load_q(const PagedDecodeParams& p, int b, int head0, int rows, int lane,
                            uint32_t (&f)[HD / 16][2 * R]) {
    const int g = lane >> 2, t = lane & 3;
    const T* qp = static_cast<const T*>(p.q) + b * p.q_b + (long long)head0 * p.q_h + 2 * t;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool ok = g + 8 * r < rows;
        const T* at = qp + (g + 8 * r) * p.q_h + k * 16;
        f[k][r] = ok ? *reinterpret_cast<const uint32_t*>(at) : 0u;
        f[k][R + r] = ok ? *reinterpret_cast<const uint32_t*>(at + 8) : 0u;
      }
  }

  LW_DEV void clear() {
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = -INFINITY, l[r] = 0.f;
  }

  // Keys key0 .. key0 + 15 of the stage at `kt` (K tile, then V tile; 16-byte
  // chunk c of row r at chunk c ^ (r & 7)).
  LW_DEV void tile(const PagedDecodeParams& p, const TileSpan& sp, int key0, bool kept, uint32_t kt, int lane) {
    const int t = lane & 3;
    float sc[2][4] = {};
    {
      // matrices of 8 keys x 8 dims: (keys 0-7 | 8-15) x (dims 0-7 | 8-15) of a k-step
      const int r = (lane >> 4) * 8 + (lane & 7), cb = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t b[4];
        ldmatrix_x4(kt + (uint32_t)(r * (HD * 2) + (((2 * k + cb) ^ (r & 7)) << 4)), b);
        const uint32_t a1 = R == 2 ? qa[k][R - 1] : 0u, a3 = R == 2 ? qa[k][2 * R - 1] : 0u;
        mma_16816<T>(sc[0], qa[k][0], a1, qa[k][R], a3, b[0], b[1]);
        mma_16816<T>(sc[1], qa[k][0], a1, qa[k][R], a3, b[2], b[3]);
      }
    }
    const bool whole = kept && key0 + kPdTile <= sp.len && (key0 >= sp.lo || key0 + kPdTile <= sp.sinks);
    if (!whole) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n * 8 + 2 * t + (e & 1);
          if (!(kept && key < sp.len && (key >= sp.lo || key < sp.sinks))) sc[n][e] = -INFINITY;
        }
    }
    float corr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[r], mx * p.scale_log2);
      const float base = mn == -INFINITY ? 0.f : mn;   // no key seen yet: every weight is 0
      corr[r] = ex2(m[r] - base);
      m[r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 2 * r; e < 2 * r + 2; ++e) {
          sc[n][e] = ex2(fmaf(sc[n][e], p.scale_log2, -base));
          sum += sc[n][e];
        }
      l[r] = fmaf(l[r], corr[r], sum);
    }
    // the weights lie in [0, 1]: rounded to T for the second product, half a
    // step each, averaged over the keys; their sum stays in fp32
    const uint32_t a0 = Elem<T>::pack(sc[0][0], sc[0][1]), a2 = Elem<T>::pack(sc[1][0], sc[1][1]);
    const uint32_t a1 = R == 2 ? Elem<T>::pack(sc[0][2], sc[0][3]) : 0u;
    const uint32_t a3 = R == 2 ? Elem<T>::pack(sc[1][2], sc[1][3]) : 0u;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      o[i][0] *= corr[0];
      o[i][1] *= corr[0];
      if constexpr (R == 2) {
        o[i][2] *= corr[R - 1];
        o[i][3] *= corr[R - 1];
      }
    }
    const uint32_t vt = kt + S::kTileBytes;
    const int r = ((lane >> 3) & 1) * 8 + (lane & 7), cb = lane >> 4;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) {
      uint32_t b[4];
      ldmatrix_x4_t(vt + (uint32_t)(r * (HD * 2) + (((2 * d + cb) ^ (r & 7)) << 4)), b);
      mma_16816<T>(o[2 * d], a0, a1, a2, a3, b[0], b[1]);
      mma_16816<T>(o[2 * d + 1], a0, a1, a2, a3, b[2], b[3]);
    }
  }

  LW_DEV void finish_sums() {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
  }

  // The piece to shared memory: accumulator, maximum and sum of every row.
  LW_DEV void store_piece(float* piece, int lane) const {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float* row = piece + (g + 8 * r) * S::kStride;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
        *reinterpret_cast<float2*>(row + i * 8 + 2 * t) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
      if (t == 0) {
        row[HD] = m[r];
        row[HD + 1] = l[r];
      }
    }
  }

  LW_DEV void store_out(const PagedDecodeParams& p, int b, int head0, int rows, int lane) const {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (g + 8 * r >= rows) continue;
      const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
      T* dst = static_cast<T*>(p.out) + b * p.o_b + (long long)(head0 + g + 8 * r) * p.o_h + 2 * t;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
        *reinterpret_cast<uint32_t*>(dst + i * 8) = Elem<T>::pack(o[i][2 * r] * inv, o[i][2 * r + 1] * inv);
    }
  }
};

// The warp's copy of a tile into a ring stage: zeros for keys nobody sees.
template <typename T, int HD, int ROWS>
LW_DEV void copy_tile(const PagedDecodeParams& p, const TileSpan& sp, int key0, int page, int kvh, uint32_t dst,
                      int lane) {
  using S = DecodeShape<HD, ROWS>;
  constexpr int CPR = HD / 8, ROWS_PER_INSTR = 32 / CPR, COPIES = kPdTile / ROWS_PER_INSTR;
  const int c_row = lane / CPR, c_chunk = lane % CPR;
  const int slot0 = key0 & (p.c.page_size - 1);
  const T* kp = static_cast<const T*>(p.c.k) + page * p.c.kp + kvh * p.c.kh + slot0 * p.c.ks + c_chunk * 8;
  const T* vp = static_cast<const T*>(p.c.v) + page * p.c.vp + kvh * p.c.vh + slot0 * p.c.vs + c_chunk * 8;
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    const int r = c_row + i * ROWS_PER_INSTR, key = key0 + r;
    const bool ok = page >= 0 && key < sp.len && (key >= sp.lo || key < sp.sinks);
    const uint32_t at = dst + (uint32_t)(r * (HD * 2) + ((c_chunk ^ (r & 7)) << 4));
    cp_async16(at, ok ? kp + r * p.c.ks : static_cast<const T*>(p.q), ok);
    cp_async16(at + S::kTileBytes, ok ? vp + r * p.c.vs : static_cast<const T*>(p.q), ok);
  }
}

// A place on the line of tiles: sequence b, its span, item (kv head, head block) within it.
struct LineCursor {
  int b, hh;
  long long item0;      // first tile of the item on the line
  TileSpan span;
};

template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(kPdThreads, 1) paged_decode_kernel(const PagedDecodeParams p) {
  using S = DecodeShape<HD, ROWS>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long sm_scan[kPdWarps];
  __shared__ long long sm_first[kPdWarps];   // tiles before sm_b
  __shared__ int sm_b[kPdWarps];
  // pieces of items that do not lie in one run: entry 2w the one warp w's run
  // begins in, entry 2w + 1 the one it ends in
  __shared__ int sm_item[2 * kPdWarps], sm_runs[2 * kPdWarps];   // item or -1; CTAs its rest covers (0: it ends here)
  __shared__ int sm_b_of[2 * kPdWarps];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int H = p.c.nkv * p.hblocks;
  float* head_piece = reinterpret_cast<float*>(smem + kPdWarps * S::kRing) + warp * S::kPiece;
  float* tail_piece = reinterpret_cast<float*>(smem + warp * S::kRing);   // the ring, once it is drained
  static_assert(S::kPiece * 4 <= S::kRing, "a piece fits in the ring");
  pdl_wait();
  pdl_launch_dependents();

  // ---- the warps' runs of the line: a scan of the sequences' tile counts
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
  if (tid < 2 * kPdWarps) sm_item[tid] = -1;
  __syncthreads();
  long long total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kPdWarps; ++w) {
    if (w < warp) before += sm_scan[w];
    total += sm_scan[w];
  }
  const long long lanes_of_work = (long long)gridDim.x * kPdWarps;
  const long long run = max(1ll, (total + lanes_of_work - 1) / lanes_of_work);
  const long long cta0 = (long long)blockIdx.x * kPdWarps * run;
  if (cta0 >= total) {   // the whole CTA
    if (tid == 0) p.meta[blockIdx.x] = make_int2(0, 0);
    return;
  }
  if (mine > 0) {
    const long long mine0 = before + incl - mine;
    for (int w = 0; w < kPdWarps; ++w) {
      const long long at = cta0 + w * run;
      if (at < mine0 || at >= mine0 + mine) continue;
      long long excl = mine0;
      int b = b_lo;
      for (; b < b_hi - 1; ++b) {
        const long long n = (long long)tile_span(p, seq_len(p.c, b)).nt * H;
        if (at < excl + n) break;
        excl += n;
      }
      sm_b[w] = b;
      sm_first[w] = excl;
    }
  }
  __syncthreads();

  const long long r0 = cta0 + warp * run, r1 = min(total, r0 + run);
  if (r0 < r1) {
    LineCursor cur;
    cur.b = sm_b[warp];
    cur.span = tile_span(p, seq_len(p.c, cur.b));
    cur.hh = (int)((r0 - sm_first[warp]) / cur.span.nt);
    cur.item0 = sm_first[warp] + (long long)cur.hh * cur.span.nt;
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
    const uint32_t ring = smem_u32(smem) + warp * S::kRing;
    LineCursor ahead = cur;
    uint32_t lost = 0;   // bit st: the stage's page id was outside the pool, its keys are hidden
    auto issue = [&](long long tile, int st) {
      if (tile < r1) {
        if (tile >= ahead.item0 + ahead.span.nt) advance(ahead);
        const int key0 = ahead.span.key0((int)(tile - ahead.item0));
        const int page = page_id(p.c, ahead.b, key0);
        lost = page < 0 ? lost | (1u << st) : lost & ~(1u << st);
        copy_tile<T, HD, ROWS>(p, ahead.span, key0, page, ahead.hh / p.hblocks, ring + st * (2 * S::kTileBytes), lane);
      }
      cp_async_commit();   // one group per call, empty past the run's end
    };
    long long next = r0;   // next tile to copy
#pragma unroll
    for (int s = 0; s < S::kStages; ++s) issue(next++, s);

    using Item = WarpItem<T, HD, ROWS>;
    Item w;
    auto head_of = [&](const LineCursor& c) {
      const int kvh = c.hh / p.hblocks;
      return kvh * p.group + (c.hh - kvh * p.hblocks) * ROWS;
    };
    auto rows_of = [&](const LineCursor& c) { return min(ROWS, p.group - c.hh % p.hblocks * ROWS); };
    Item::load_q(p, cur.b, head_of(cur), rows_of(cur), lane, w.qa);
    long long tile = r0;
    int st = 0;
    for (;;) {
      const long long end = min(cur.item0 + cur.span.nt, r1);
      const bool starts = cur.item0 >= r0, ends = cur.item0 + cur.span.nt <= r1;
      LineCursor nxt = cur;
      uint32_t qn[HD / 16][2 * Item::R];   // the next item's queries arrive meanwhile
      if (end < r1) {
        advance(nxt);
        Item::load_q(p, nxt.b, head_of(nxt), rows_of(nxt), lane, qn);
      }
      w.clear();
      for (; tile < end; ++tile) {
        cp_async_wait<S::kStages - 1>();   // the oldest group has landed
        __syncwarp();
        w.tile(p, cur.span, cur.span.key0((int)(tile - cur.item0)), !((lost >> st) & 1u),
               ring + st * (2 * S::kTileBytes), lane);
        __syncwarp();   // every lane has read the stage
        issue(next++, st);
        if (++st == S::kStages) st = 0;
      }
      w.finish_sums();
      const int item = cur.b * H + cur.hh;
      if (starts && ends) {
        w.store_out(p, cur.b, head_of(cur), rows_of(cur), lane);
      } else {
        const int e = 2 * warp + (starts ? 1 : 0);
        if (lane == 0) {
          sm_item[e] = item;
          sm_b_of[e] = cur.b;
          // CTAs after this one that hold tiles of the item
          sm_runs[e] = (int)((cur.item0 + cur.span.nt - 1) / (run * kPdWarps) - blockIdx.x);
        }
        if (starts) {
          cp_async_wait<0>();   // the run's last item: the ring is drained
          __syncwarp();
          w.store_piece(tail_piece, lane);
        } else {
          w.store_piece(head_piece, lane);
        }
      }
      if (end == r1) break;
      cur = nxt;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int r = 0; r < 2 * Item::R; ++r) w.qa[k][r] = qn[k][r];
    }
  }
  __syncthreads();

  // ---- pieces of one item follow one another in the entries
  int2 open = make_int2(0, 0);
  for (int e = 0; e < 2 * kPdWarps;) {
    const int item = sm_item[e];
    if (item < 0) {
      ++e;
      continue;
    }
    int end = e + 1;
    while (end < 2 * kPdWarps && (sm_item[end] < 0 || sm_item[end] == item)) ++end;
    const int b = sm_b_of[e], hh = item - b * H, kvh = hh / p.hblocks, hb = hh - kvh * p.hblocks;
    const int rows = min(ROWS, p.group - hb * ROWS);
    const int more = sm_runs[e];
    const bool starts = e & 1;
    if (starts && more) open = make_int2(item, more + 1);
    float* slot = p.part + (long long)(2 * blockIdx.x + (starts ? 1 : 0)) * S::kPiece;
    auto piece = [&](int i) {
      return reinterpret_cast<const float*>(smem + ((i & 1) ? (i >> 1) * S::kRing : kPdWarps * S::kRing +
                                                                                        (i >> 1) * S::kPiece * 4));
    };
    for (int i = tid; i < rows * (HD / 2); i += kPdThreads) {
      const int r = i / (HD / 2), d = (i - r * (HD / 2)) * 2;
      float M = -INFINITY;
      for (int x = e; x < end; ++x)
        if (sm_item[x] >= 0) M = fmaxf(M, piece(x)[r * S::kStride + HD]);
      float L = 0.f, x0 = 0.f, x1 = 0.f;
      for (int x = e; x < end; ++x) {
        if (sm_item[x] < 0) continue;
        const float* row = piece(x) + r * S::kStride;
        const float f = row[HD] == -INFINITY ? 0.f : ex2(row[HD] - M);   // no key seen in this piece
        const float2 v = *reinterpret_cast<const float2*>(row + d);
        L = fmaf(row[HD + 1], f, L);
        x0 = fmaf(v.x, f, x0);
        x1 = fmaf(v.y, f, x1);
      }
      if (starts && !more) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        T* dst = static_cast<T*>(p.out) + b * p.o_b + (long long)(kvh * p.group + hb * ROWS + r) * p.o_h + d;
        *reinterpret_cast<uint32_t*>(dst) = Elem<T>::pack(x0 * inv, x1 * inv);
      } else {
        float* dst = slot + r * S::kStride;
        *reinterpret_cast<float2*>(dst + d) = make_float2(x0, x1);
        if (d == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(M, L);
      }
    }
    e = end;
  }
  if (tid == 0) p.meta[blockIdx.x] = open;
}

// Joins the pieces of the items that several CTAs hold, in the order of the
// line: block (c, r) row r of the one that begins in CTA c, if there is one (a
// CTA's end cuts one item at most). Its warps take the pieces in turn, then merge.
// The blocks also write zeros for sequences without a visible key.
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(kPdThreads) paged_join_kernel(const PagedDecodeParams p) {
  using S = DecodeShape<HD, ROWS>;
  constexpr int V = HD / 32;   // dims per lane
  __shared__ float sm_acc[kPdWarps][HD], sm_m[kPdWarps], sm_l[kPdWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane * V;
  const int H = p.c.nkv * p.hblocks, r = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  const int2 mt = p.meta[blockIdx.x];
  for (int b = blockIdx.x + (int)gridDim.x * warp; b < p.c.B; b += (int)gridDim.x * kPdWarps)
    if (seq_len(p.c, b) == 0)
      for (int h = r; h < p.c.nkv * p.group; h += gridDim.y) {
        T* dst = static_cast<T*>(p.out) + b * p.o_b + h * p.o_h + d;
        if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(0, 0);
        else *reinterpret_cast<uint32_t*>(dst) = 0u;
      }
  const int b = mt.x / H, hh = mt.x - b * H, kvh = hh / p.hblocks, hb = hh - kvh * p.hblocks;
  if (mt.y == 0 || r >= p.group - hb * ROWS) return;
  constexpr int kAtOnce = 4;
  float M = -INFINITY, L = 0.f, acc[V] = {};
  for (int i0 = warp; i0 < mt.y; i0 += kPdWarps * kAtOnce) {
    float2 ml[kAtOnce];
    float v[kAtOnce][V];
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      const int i = i0 + x * kPdWarps;
      ml[x] = make_float2(-INFINITY, 0.f);
      if (i < mt.y) {
        const float* s = p.part + (long long)(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * S::kPiece +
                         r * S::kStride;
        ml[x] = *reinterpret_cast<const float2*>(s + HD);
        if constexpr (V == 4) *reinterpret_cast<float4*>(v[x]) = *reinterpret_cast<const float4*>(s + d);
        else *reinterpret_cast<float2*>(v[x]) = *reinterpret_cast<const float2*>(s + d);
      }
    }
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      if (ml[x].x == -INFINITY && ml[x].y == 0.f) continue;   // past the end, or no key seen in the piece
      const float mn = fmaxf(M, ml[x].x);
      const float f0 = ex2(M - mn), f1 = ex2(ml[x].x - mn);
      M = mn;
      L = fmaf(L, f0, ml[x].y * f1);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(acc[e], f0, v[x][e] * f1);
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) sm_acc[warp][d + e] = acc[e];
  if (lane == 0) {
    sm_m[warp] = M;
    sm_l[warp] = L;
  }
  __syncthreads();
  if (warp) return;
  M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kPdWarps; ++w) M = fmaxf(M, sm_m[w]);
  L = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
#pragma unroll
  for (int w = 0; w < kPdWarps; ++w) {
    const float f = sm_m[w] == -INFINITY ? 0.f : ex2(sm_m[w] - M);   // a warp without pieces
    L = fmaf(sm_l[w], f, L);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = fmaf(sm_acc[w][d + e], f, acc[e]);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* dst = static_cast<T*>(p.out) + b * p.o_b + (long long)(kvh * p.group + hb * ROWS + r) * p.o_h + d;
  if constexpr (V == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::pack(acc[0] * inv, acc[1] * inv),
                                                Elem<T>::pack(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = Elem<T>::pack(acc[0] * inv, acc[1] * inv);
}

// An item per cluster: its CTAs' warps take the tiles in turn.
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(kPdThreads, 1) paged_decode_cluster_kernel(const PagedDecodeParams p) {
  namespace cg = cooperative_groups;
  using S = DecodeShape<HD, ROWS>;
  using Item = WarpItem<T, HD, ROWS>;
  extern __shared__ __align__(128) uint8_t smem[];
  float* pieces = reinterpret_cast<float*>(smem + kPdWarps * S::kRing);
  float* joined = reinterpret_cast<float*>(smem);   // this CTA's piece, once the rings are drained
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int H = p.c.nkv * p.hblocks;
  const int item = blockIdx.y, b = item / H, hh = item - b * H, kvh = hh / p.hblocks, hb = hh - kvh * p.hblocks;
  const int head0 = kvh * p.group + hb * ROWS, rows = min(ROWS, p.group - hb * ROWS);
  pdl_wait();
  pdl_launch_dependents();
  Item w;
  Item::load_q(p, b, head0, rows, lane, w.qa);
  const TileSpan sp = tile_span(p, seq_len(p.c, b));
  const int step = CL * kPdWarps;
  const uint32_t ring = smem_u32(smem) + warp * S::kRing;
  uint32_t lost = 0;
  auto issue = [&](int tile, int st) {
    if (tile < sp.nt) {
      const int key0 = sp.key0(tile), page = page_id(p.c, b, key0);
      lost = page < 0 ? lost | (1u << st) : lost & ~(1u << st);
      copy_tile<T, HD, ROWS>(p, sp, key0, page, kvh, ring + st * (2 * S::kTileBytes), lane);
    }
    cp_async_commit();
  };
  int tile = rank * kPdWarps + warp, next = tile, st = 0;
#pragma unroll
  for (int s = 0; s < S::kStages; ++s, next += step) issue(next, s);
  w.clear();
  for (; tile < sp.nt; tile += step) {
    cp_async_wait<S::kStages - 1>();
    __syncwarp();
    w.tile(p, sp, sp.key0(tile), !((lost >> st) & 1u), ring + st * (2 * S::kTileBytes), lane);
    __syncwarp();
    issue(next, st);
    next += step;
    if (++st == S::kStages) st = 0;
  }
  w.finish_sums();
  w.store_piece(pieces + warp * S::kPiece, lane);
  cp_async_wait<0>();
  __syncthreads();
  for (int i = tid; i < rows * (HD / 2); i += kPdThreads) {
    const int r = i / (HD / 2), d = (i - r * (HD / 2)) * 2;
    const float* row = pieces + r * S::kStride;
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < kPdWarps; ++x) M = fmaxf(M, row[x * S::kPiece + HD]);
    float L = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int x = 0; x < kPdWarps; ++x) {
      const float* s = row + x * S::kPiece;
      const float f = s[HD] == -INFINITY ? 0.f : ex2(s[HD] - M);   // a warp without tiles adds nothing
      L = fmaf(s[HD + 1], f, L);
      x0 = fmaf(s[d], f, x0);
      x1 = fmaf(s[d + 1], f, x1);
    }
    float* dst = joined + r * S::kStride;
    *reinterpret_cast<float2*>(dst + d) = make_float2(x0, x1);
    if (d == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(M, L);
  }
  cluster.sync();
  for (int i = rank * kPdThreads + tid; i < rows * (HD / 2); i += CL * kPdThreads) {
    const int r = i / (HD / 2), d = (i - r * (HD / 2)) * 2;
    float2 ml[8], v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {   // the remote reads together
      const float* s = cluster.map_shared_rank(joined, c < CL ? c : 0) + r * S::kStride;
      ml[c] = *reinterpret_cast<const float2*>(s + HD);
      v[c] = *reinterpret_cast<const float2*>(s + d);
    }
    float M = -INFINITY;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < CL) M = fmaxf(M, ml[c].x);
    float L = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (c >= CL) break;
      const float f = ml[c].x == -INFINITY ? 0.f : ex2(ml[c].x - M);
      L = fmaf(ml[c].y, f, L);
      x0 = fmaf(v[c].x, f, x0);
      x1 = fmaf(v[c].y, f, x1);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* dst = static_cast<T*>(p.out) + b * p.o_b + (long long)(head0 + r) * p.o_h + d;
    *reinterpret_cast<uint32_t*>(dst) = Elem<T>::pack(x0 * inv, x1 * inv);
  }
  cluster.sync();   // this CTA's shared memory lives until every remote read is done
}

}  // namespace lw

namespace {

struct DecodePlan {
  int group, rows, hblocks, grid, cluster;   // cluster 0: runs and a join
  long long items;
  size_t part_off, bytes;
};

DecodePlan decode_plan(const lw_paged_attention_args* a) {
  DecodePlan d;
  d.group = a->n_q_heads / a->cache.n_kv_heads;
  d.rows = d.group <= 8 ? 8 : 16;
  d.hblocks = (d.group + d.rows - 1) / d.rows;
  d.items = (long long)a->cache.batch * a->cache.n_kv_heads * d.hblocks;
  d.grid = lw_host::sm_count();
  // Clusters of as many CTAs as the SMs hold beside each other (up to 8), when
  // no sequence can give one of their CTAs more than 32 tiles (four per warp).
  long long keys = (long long)a->cache.table_width * a->cache.page_size;
  if (a->window > 0) keys = std::min(keys, (long long)a->window + a->sinks);
  d.cluster = 8;
  while (d.cluster > 1 && d.items * d.cluster > d.grid) d.cluster /= 2;
  if (d.items * d.cluster > d.grid || keys > 32ll * lw::kPdTile * d.cluster) d.cluster = 0;
  d.part_off = ((size_t)d.grid * sizeof(int2) + 255) & ~(size_t)255;
  d.bytes = d.cluster ? 0 : d.part_off + (size_t)2 * d.grid * d.rows * (a->cache.head_dim + 8) * sizeof(float);
  return d;
}

template <typename Kernel>
cudaError_t allow_smem(Kernel kern, int bytes) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename T, int HD, int ROWS>
cudaError_t decode_launch(const lw::PagedDecodeParams& p, const DecodePlan& d, cudaStream_t s, bool pdl) {
  constexpr int smem = lw::DecodeShape<HD, ROWS>::kBytes;
  if (d.cluster) {
    auto kern = lw::paged_decode_cluster_kernel<T, HD, ROWS>;
    cudaError_t e = allow_smem(kern, smem);
    if (e != cudaSuccess) return e;
    lw_count_launch();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)d.cluster, (unsigned)d.items);
    cfg.blockDim = dim3(lw::kPdThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)d.cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
  }
  auto kern = lw::paged_decode_kernel<T, HD, ROWS>;
  cudaError_t e = allow_smem(kern, smem);
  if (e != cudaSuccess) return e;
  e = lw_launch(kern, dim3(d.grid), dim3(lw::kPdThreads), smem, s, pdl, p);
  if (e != cudaSuccess) return e;
  return lw_launch(lw::paged_join_kernel<T, HD, ROWS>, dim3(d.grid, std::min(ROWS, d.group)), dim3(lw::kPdThreads), 0, s,
                   true, p);
}

template <typename T>
cudaError_t decode_dispatch(const lw::PagedDecodeParams& p, int hd, const DecodePlan& d, cudaStream_t s, bool pdl) {
  if (hd == 128) return d.rows == 8 ? decode_launch<T, 128, 8>(p, d, s, pdl) : decode_launch<T, 128, 16>(p, d, s, pdl);
  return d.rows == 8 ? decode_launch<T, 64, 8>(p, d, s, pdl) : decode_launch<T, 64, 16>(p, d, s, pdl);
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
  p.group = d.group;
  p.hblocks = d.hblocks;
  p.window = a->window;
  p.sinks = a->sinks;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.meta = static_cast<int2*>(a->workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + d.part_off);
  const bool pdl = a->pdl != 0;
  const cudaError_t e = a->cache.dtype == LW_DTYPE_F16 ? decode_dispatch<__half>(p, a->cache.head_dim, d, s, pdl)
                                                       : decode_dispatch<__nv_bfloat16>(p, a->cache.head_dim, d, s, pdl);
  return e == cudaSuccess ? LW_OK : LW_ERR_LAUNCH;
}

// Attention of one new token per sequence over the paged cache
// (lw_paged_attention without q_offsets): split over the cache's length, joined.
//
//   out[b][h] = sum_j softmax_j(scale * q[b][h] . k_j) v_j  over the keys j that
//   position p = kv_lens[b] - 1 sees.
//
// Bound by reading the visible keys and values once. The work is cut into
// tiles of 16 (head_dim 128) or 32 (64) consecutive token positions, 8 KB of keys
// and values, of one item = (sequence, kv head, block of up to ROWS query
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
// Measured (device time, several GPUs): 64 sequences of 131 to 16384 tokens, 32 / 8
// heads of 128, 0.90 GB: 144-152 us, 5.9-6.3 TB/s; one of 131071 tokens, 0.54 GB: 89-95
// us, 5.7-6.0 TB/s; one of 517 tokens: 5.4 us. The stream itself runs at 7.0 TB/s; the rest is
// the start (3 us), SMs that end later than others, the merge and the join (5 us).
// A warp's tile takes 0.5 us of work against 1.5 us of its share of the memory.
//
// Hidden keys of a tile are zero-filled by the copy, so what their slots hold
// (NaN included) never meets the tensor cores.
#include <cooperative_groups.h>

#include <algorithm>

#include "paged.cuh"

namespace lw {

constexpr int kPdWarps = 8;
constexpr int kPdThreads = kPdWarps * 32;

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
};

template <int TILE>
LW_DEV TileSpan tile_span(const PagedDecodeParams& p, int len) {
  TileSpan s;
  s.len = len;
  s.lo = window_start(len - 1, p.window);
  s.sinks = min(p.sinks, s.lo);
  s.w0 = s.lo / TILE;
  s.ns = min((s.sinks + TILE - 1) / TILE, s.w0);
  s.nt = len > 0 ? s.ns + (len + TILE - 1) / TILE - s.w0 : 0;
  return s;
}
// First key of a span's tile.
template <int TILE>
LW_DEV int tile_key(const TileSpan& s, int tile) {
  return (tile < s.ns ? tile : s.w0 + tile - s.ns) * TILE;
}

// Whether tiles t0, t0 + step, .. below t1 hold a visible key. Asked only for a row
// that has no weight, so that the tiles' loop does not track it.
template <int TILE>
LW_DEV bool sees_key(const PagedDecodeParams& p, const TileSpan& sp, int b, int t0, int t1, int step) {
#pragma unroll 1
  for (int tile = t0; tile < t1; tile += step)
#pragma unroll 1
    for (int x = 0; x < TILE; x += 16) {   // 16 keys are of one page
      const int key = tile_key<TILE>(sp, tile) + x;
      if (key < sp.len && (key + 16 > sp.lo || key < sp.sinks) && page_id(p.c, b, key) >= 0) return true;
    }
  return false;
}

// Sizes of a kernel's shared memory: a ring per warp, then pieces [warps][ROWS][HD + 8]
// (accumulator, maximum, sum; the stride keeps the fragment stores off each other's banks).
template <int HD, int ROWS>
struct DecodeShape {
  static constexpr int kTile = 2048 / HD;                       // keys per tile
  static constexpr int kGroups = kTile / 16;                    // of 16 keys: one page each
  static constexpr int kTileBytes = kTile * HD * 2;             // K or V of a tile
  static constexpr int kRing = ROWS == 8 ? 24576 : 16384;       // per warp
  static constexpr int kStages = kRing / (2 * kTileBytes);
  static constexpr int kStride = HD + 8;
  static constexpr int kPiece = ROWS * kStride;                 // floats
  static constexpr int kBytes = kPdWarps * (kRing + kPiece * 4);
};

// One warp's share of an item: queries as MMA fragments, the online softmax of
// rows g and g + 8 (g + 8 with ROWS = 16 only), the accumulator. m is the base of
// the weights: the maximum so far less kMaxWeightLog2.
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

  // The keys from key0 on, in the stage at `kt` (K tile, then V tile; 16-byte chunk
  // c of row r at chunk c ^ (r & 7)); bit i of `lost`: the 16-key group i is hidden.
  LW_DEV void tile(const PagedDecodeParams& p, const TileSpan& sp, int key0, uint32_t lost, uint32_t kt, int lane) {
    constexpr int N = S::kTile / 8;   // score fragments of 8 keys
    const int t = lane & 3;
    float sc[N][4];
#pragma unroll
    for (int n = 0; n < N; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
    {
      // matrices of 8 keys x 8 dims: (keys 0-7 | 8-15) x (dims 0-7 | 8-15) of a k-step
      const int r0 = (lane >> 4) * 8 + (lane & 7), cb = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int x = 0; x < S::kGroups; ++x) {
          const int r = 16 * x + r0;
          uint32_t b[4];
          ldmatrix_x4(kt + (uint32_t)(r * (HD * 2) + (((2 * k + cb) ^ (r & 7)) << 4)), b);
          const uint32_t a1 = R == 2 ? qa[k][R - 1] : 0u, a3 = R == 2 ? qa[k][2 * R - 1] : 0u;
          mma_16816<T>(sc[2 * x], qa[k][0], a1, qa[k][R], a3, b[0], b[1]);
          mma_16816<T>(sc[2 * x + 1], qa[k][0], a1, qa[k][R], a3, b[2], b[3]);
        }
    }
    const bool whole = !lost && key0 + S::kTile <= sp.len && (key0 >= sp.lo || key0 + S::kTile <= sp.sinks);
    if (!whole) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n * 8 + 2 * t + (e & 1);
          if (((lost >> (n / 2)) & 1u) || key >= sp.len || (key < sp.lo && key >= sp.sinks)) sc[n][e] = -INFINITY;
        }
    }
    float corr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = fmaxf(sc[0][2 * r], sc[0][2 * r + 1]);
#pragma unroll
      for (int n = 1; n < N; ++n) mx = fmaxf(mx, fmaxf(sc[n][2 * r], sc[n][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // the base that weights are taken from: the maximum less the largest weight's
      // exponent, rounded up, so that no weight is above 2^kMaxWeightLog2 however
      // coarse fp32 is at the scores' size. Sums and accumulators carry the factor.
      const float mn = fmaxf(m[r], __fmaf_ru(mx, p.scale_log2, -Elem<T>::kMaxWeightLog2));
      const float base = mn == -INFINITY ? 0.f : mn;   // no key seen yet: every weight is 0
      corr[r] = ex2(m[r] - base);
      m[r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 2 * r; e < 2 * r + 2; ++e) {
          sc[n][e] = ex2(fmaf(sc[n][e], p.scale_log2, -base));
          sum += sc[n][e];
        }
      l[r] = fmaf(l[r], corr[r], sum);
    }
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
    const int r0 = ((lane >> 3) & 1) * 8 + (lane & 7), cb = lane >> 4;
#pragma unroll
    for (int x = 0; x < S::kGroups; ++x) {
      // rounded to T for the second product, half a step each, averaged over the
      // keys (fp16: weights under 2^-29 of the largest so far by up to 2^-40 of it);
      // their sum stays in fp32
      const uint32_t a0 = Elem<T>::pack(sc[2 * x][0], sc[2 * x][1]);
      const uint32_t a2 = Elem<T>::pack(sc[2 * x + 1][0], sc[2 * x + 1][1]);
      const uint32_t a1 = R == 2 ? Elem<T>::pack(sc[2 * x][2], sc[2 * x][3]) : 0u;
      const uint32_t a3 = R == 2 ? Elem<T>::pack(sc[2 * x + 1][2], sc[2 * x + 1][3]) : 0u;
      const int r = 16 * x + r0;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        uint32_t b[4];
        ldmatrix_x4_t(vt + (uint32_t)(r * (HD * 2) + (((2 * d + cb) ^ (r & 7)) << 4)), b);
        mma_16816<T>(o[2 * d], a0, a1, a2, a3, b[0], b[1]);
        mma_16816<T>(o[2 * d + 1], a0, a1, a2, a3, b[2], b[3]);
      }
    }
  }

  // Of tiles t0, t0 + step, .. below t1 of sequence b.
  LW_DEV void finish(const PagedDecodeParams& p, const TileSpan& sp, int b, int t0, int t1, int step) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (m[r] == -INFINITY && sees_key<S::kTile>(p, sp, b, t0, t1, step)) m[r] = kAllBelow;
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
      const float inv = weight_inverse(m[r], l[r]);
      T* dst = static_cast<T*>(p.out) + b * p.o_b + (long long)(head0 + g + 8 * r) * p.o_h + 2 * t;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
        *reinterpret_cast<uint32_t*>(dst + i * 8) = Elem<T>::pack(o[i][2 * r] * inv, o[i][2 * r + 1] * inv);
    }
  }
};

// The warp's copy of a tile into a ring stage, zeros for keys nobody sees. Returns
// the 16-key groups whose page id is outside the pool: their keys are hidden.
template <typename T, int HD, int ROWS>
LW_DEV uint32_t copy_tile(const PagedDecodeParams& p, const TileSpan& sp, int b, int key0, int kvh, uint32_t dst,
                          int lane) {
  using S = DecodeShape<HD, ROWS>;
  constexpr int CPR = HD / 8, ROWS_PER_INSTR = 32 / CPR, COPIES = 16 / ROWS_PER_INSTR;
  const int c_row = lane / CPR, c_chunk = lane % CPR;
  int page[S::kGroups];
  uint32_t lost = 0;
#pragma unroll
  for (int x = 0; x < S::kGroups; ++x) {
    const int first = key0 + 16 * x;   // a group may lie outside what is seen: its table entry is not read
    const bool seen = S::kGroups == 1 || (first < sp.len && (first + 16 > sp.lo || first < sp.sinks));
    page[x] = seen ? page_id(p.c, b, first) : 0;
    if (page[x] < 0) lost |= 1u << x;
  }
#pragma unroll
  for (int x = 0; x < S::kGroups; ++x) {
    const int first = key0 + 16 * x, slot0 = first & (p.c.page_size - 1);
    const T* kp = static_cast<const T*>(p.c.k) + page[x] * p.c.kp + kvh * p.c.kh + slot0 * p.c.ks + c_chunk * 8;
    const T* vp = static_cast<const T*>(p.c.v) + page[x] * p.c.vp + kvh * p.c.vh + slot0 * p.c.vs + c_chunk * 8;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int r = c_row + i * ROWS_PER_INSTR, key = first + r;
      const bool ok = page[x] >= 0 && key < sp.len && (key >= sp.lo || key < sp.sinks);
      const uint32_t at = dst + (uint32_t)((16 * x + r) * (HD * 2) + ((c_chunk ^ (r & 7)) << 4));
      cp_async16(at, ok ? kp + r * p.c.ks : static_cast<const T*>(p.q), ok);
      cp_async16(at + S::kTileBytes, ok ? vp + r * p.c.vs : static_cast<const T*>(p.q), ok);
    }
  }
  return lost;
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
  constexpr uint32_t kGroupBits = (1u << S::kGroups) - 1u;
  pdl_wait();
  pdl_launch_dependents();

  // ---- the warps' runs of the line: a scan of the sequences' tile counts
  const int per_thread = (p.c.B + kPdThreads - 1) / kPdThreads;
  const int b_lo = min(p.c.B, tid * per_thread), b_hi = min(p.c.B, b_lo + per_thread);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += (long long)tile_span<S::kTile>(p, seq_len(p.c, b)).nt * H;
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
        const long long n = (long long)tile_span<S::kTile>(p, seq_len(p.c, b)).nt * H;
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
    cur.span = tile_span<S::kTile>(p, seq_len(p.c, cur.b));
    cur.hh = (int)((r0 - sm_first[warp]) / cur.span.nt);
    cur.item0 = sm_first[warp] + (long long)cur.hh * cur.span.nt;
    auto advance = [&](LineCursor& c) {   // to the next item with tiles (one exists while its first tile < total)
      c.item0 += c.span.nt;
      if (++c.hh == H) {
        c.hh = 0;
        do {
          ++c.b;
          c.span = tile_span<S::kTile>(p, seq_len(p.c, c.b));
        } while (c.span.nt == 0);
      }
    };
    const uint32_t ring = smem_u32(smem) + warp * S::kRing;
    LineCursor ahead = cur;
    uint32_t lost = 0;   // kGroups bits per stage: page ids outside the pool
    auto issue = [&](long long tile, int st) {
      if (tile < r1) {
        if (tile >= ahead.item0 + ahead.span.nt) advance(ahead);
        const int key0 = tile_key<S::kTile>(ahead.span, (int)(tile - ahead.item0));
        const uint32_t bad = copy_tile<T, HD, ROWS>(p, ahead.span, ahead.b, key0, ahead.hh / p.hblocks,
                                                    ring + st * (2 * S::kTileBytes), lane);
        lost = (lost & ~(kGroupBits << (st * S::kGroups))) | (bad << (st * S::kGroups));
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
      const int t0 = (int)(tile - cur.item0);
      for (; tile < end; ++tile) {
        cp_async_wait<S::kStages - 1>();   // the oldest group has landed
        __syncwarp();
        w.tile(p, cur.span, tile_key<S::kTile>(cur.span, (int)(tile - cur.item0)),
               (lost >> (st * S::kGroups)) & kGroupBits, ring + st * (2 * S::kTileBytes), lane);
        __syncwarp();   // every lane has read the stage
        issue(next++, st);
        if (++st == S::kStages) st = 0;
      }
      w.finish(p, cur.span, cur.b, t0, (int)(end - cur.item0), 1);
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

  // ---- pieces of one item follow one another in the entries; `firsts` marks the
  // first of each item's. A warp takes an item's row at a time: lane e has the
  // weight of entry e, then a lane has HD / 32 dims.
  const int my_item = lane < 2 * kPdWarps ? sm_item[lane] : -1, my_runs = lane < 2 * kPdWarps ? sm_runs[lane] : 0;
  const uint32_t valid = __ballot_sync(0xffffffffu, my_item >= 0);
  uint32_t firsts;
  {
    const uint32_t before_me = valid & ((1u << lane) - 1u);
    const int prev = __shfl_sync(0xffffffffu, my_item, before_me ? 31 - __clz(before_me) : lane);
    firsts = __ballot_sync(0xffffffffu, my_item >= 0 && (!before_me || prev != my_item));
  }
  // only the last item can go on in the next CTA; an odd entry: it begins in this one
  if (tid == 31 - __clz(firsts | 1u))
    p.meta[blockIdx.x] = (tid & 1) && my_item >= 0 && my_runs ? make_int2(my_item, my_runs + 1) : make_int2(0, 0);
  auto piece = [&](int e) {   // entry e's first byte
    return smem_u32(smem) + (uint32_t)((e & 1) ? (e >> 1) * S::kRing : kPdWarps * S::kRing + (e >> 1) * S::kPiece * 4);
  };
  constexpr int V = HD / 32;
  const int rows_max = min(ROWS, p.group), tasks = __popc(firsts) * rows_max;
  for (int task = warp; task < tasks; task += kPdWarps) {
    const int k = task / rows_max, r = task - k * rows_max;
    uint32_t rest = firsts;
    for (int x = 0; x < k; ++x) rest &= rest - 1u;
    const int e0 = __ffs(rest) - 1;
    rest &= rest - 1u;
    const uint32_t mine = valid & (~0u << e0) & (rest ? (rest & (0u - rest)) - 1u : ~0u);   // the item's entries
    const int item = __shfl_sync(0xffffffffu, my_item, e0), b = sm_b_of[e0], hh = item - b * H;
    const int kvh = hh / p.hblocks, hb = hh - kvh * p.hblocks;
    if (r >= p.group - hb * ROWS) continue;
    float2 ml = make_float2(-INFINITY, 0.f);
    if ((mine >> lane) & 1u) ml = lds_f2(piece(lane) + (uint32_t)(r * S::kStride + HD) * 4u);
    const float M = warp_max(ml.x);
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);   // no key seen in this piece
    const float L = warp_sum(ml.y * f);
    float2 acc[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) acc[i] = make_float2(0.f, 0.f);
#pragma unroll
    for (int x = 0; x < 2 * kPdWarps; ++x) {
      if (!((mine >> x) & 1u)) continue;
      const float g = __shfl_sync(0xffffffffu, f, x);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 v = lds_f2(piece(x) + (uint32_t)(r * S::kStride + lane * V + 2 * i) * 4u);
        acc[i].x = fmaf(v.x, g, acc[i].x);
        acc[i].y = fmaf(v.y, g, acc[i].y);
      }
    }
    const bool starts = e0 & 1;
    if (starts && !__shfl_sync(0xffffffffu, my_runs, e0)) {
      const float inv = weight_inverse(M, L);
      T* out = static_cast<T*>(p.out) + b * p.o_b + (long long)(kvh * p.group + hb * ROWS + r) * p.o_h + lane * V;
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        *reinterpret_cast<uint32_t*>(out + 2 * i) = Elem<T>::pack(acc[i].x * inv, acc[i].y * inv);
    } else {
      float* part = p.part + (long long)(2 * blockIdx.x + (starts ? 1 : 0)) * S::kPiece + r * S::kStride;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) *reinterpret_cast<float2*>(part + lane * V + 2 * i) = acc[i];
      if (lane == 0) *reinterpret_cast<float2*>(part + HD) = make_float2(M, L);
    }
  }
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
  // piece i of the item that may begin here; a warp's first is asked for before it
  // is known whether there is one (what is read for nothing is thrown away)
  float2 ml[4];
  float v[4][V];
  auto load = [&](int x, int i) {
    const float* s = p.part + (long long)(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * S::kPiece +
                     r * S::kStride;
    ml[x] = *reinterpret_cast<const float2*>(s + HD);
    if constexpr (V == 4) *reinterpret_cast<float4*>(v[x]) = *reinterpret_cast<const float4*>(s + d);
    else *reinterpret_cast<float2*>(v[x]) = *reinterpret_cast<const float2*>(s + d);
  };
  const int2 mt = p.meta[blockIdx.x];
  if (blockIdx.x + warp < gridDim.x) load(0, warp);
  for (int b = blockIdx.x + (int)gridDim.x * warp; b < p.c.B; b += (int)gridDim.x * kPdWarps)
    if (seq_len(p.c, b) == 0)
      for (int h = r; h < p.c.nkv * p.group; h += gridDim.y) {
        T* dst = static_cast<T*>(p.out) + b * p.o_b + h * p.o_h + d;
        if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(0, 0);
        else *reinterpret_cast<uint32_t*>(dst) = 0u;
      }
  const int b = mt.x / H, hh = mt.x - b * H, kvh = hh / p.hblocks, hb = hh - kvh * p.hblocks;
  if (mt.y == 0 || r >= p.group - hb * ROWS) return;
  float M = -INFINITY, L = 0.f, acc[V] = {};
  for (int i0 = warp; i0 < mt.y; i0 += kPdWarps * 4) {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if ((x > 0 || i0 != warp) && i0 + x * kPdWarps < mt.y) load(x, i0 + x * kPdWarps);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      // past the last, or no key seen in the piece
      if (i0 + x * kPdWarps >= mt.y || (ml[x].x == -INFINITY && ml[x].y == 0.f)) continue;
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
  const float inv = weight_inverse(M, L);
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
  const TileSpan sp = tile_span<S::kTile>(p, seq_len(p.c, b));
  constexpr uint32_t kGroupBits = (1u << S::kGroups) - 1u;
  const int step = CL * kPdWarps;
  const uint32_t ring = smem_u32(smem) + warp * S::kRing;
  uint32_t lost = 0;
  auto issue = [&](int tile, int st) {
    if (tile < sp.nt) {
      const uint32_t bad =
          copy_tile<T, HD, ROWS>(p, sp, b, tile_key<S::kTile>(sp, tile), kvh, ring + st * (2 * S::kTileBytes), lane);
      lost = (lost & ~(kGroupBits << (st * S::kGroups))) | (bad << (st * S::kGroups));
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
    w.tile(p, sp, tile_key<S::kTile>(sp, tile), (lost >> (st * S::kGroups)) & kGroupBits,
           ring + st * (2 * S::kTileBytes), lane);
    __syncwarp();
    issue(next, st);
    next += step;
    if (++st == S::kStages) st = 0;
  }
  w.finish(p, sp, b, rank * kPdWarps + warp, sp.nt, step);
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
    const float inv = weight_inverse(M, L);
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

// Clusters of `size` CTAs with a kernel's shared memory that run at once on the current device.
int resident_clusters(int size) {
  static std::atomic<int> known[64][4];   // by device and size, 0: not asked yet
  int dev = 0, log = 0, n = 0;
  while ((1 << log) < size) ++log;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if ((n = known[dev][log].load(std::memory_order_relaxed)) != 0) return std::max(n, 0);
  constexpr auto kern = lw::paged_decode_cluster_kernel<__half, 128, 8>;
  constexpr int smem = lw::DecodeShape<128, 8>::kBytes;   // the largest of all forms
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)size, 148);
  cfg.blockDim = dim3(lw::kPdThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (lw_host::allow_smem<kern>(smem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();   // no device: no clusters
    return 0;
  }
  known[dev][log].store(n > 0 ? n : -1, std::memory_order_relaxed);
  return n;
}

DecodePlan decode_plan(const lw_paged_attention_args* a) {
  DecodePlan d;
  d.group = a->n_q_heads / a->cache.n_kv_heads;
  d.rows = d.group <= 8 ? 8 : 16;
  d.hblocks = (d.group + d.rows - 1) / d.rows;
  d.items = (long long)a->cache.batch * a->cache.n_kv_heads * d.hblocks;
  // Runs: a CTA per SM. Some groups of neighbouring SMs end 10 to 20 % after the
  // others, which ones differs from GPU to GPU: 128 CTAs instead of 148 took 145 us
  // instead of 153 for 64 ragged sequences on one B200 and 159 instead of 150 on another.
  d.grid = lw_host::sm_count();
  // Clusters: the largest of 8, 4, 2 or 1 CTAs of which one per item runs at once,
  // when no sequence can give a CTA more than 1024 keys, or 512 where the items
  // fill less than 64 SMs (the runs then use more of them). Cluster / runs, us: 8 items of 2048 keys
  // 6.7 / 9.5, of 8192 14.4 / 15.3, of 16384 22.8 / 19.6; 1 item of 4096 8.9 / 10.0,
  // of 8192 13.4 / 10.7; 32 items of 4096 15.9 / 19.9; 128 items of 512 9.2 / 14.6.
  long long keys = (long long)a->cache.table_width * a->cache.page_size;
  if (a->window > 0) keys = std::min(keys, (long long)a->window + a->sinks);
  d.cluster = 8;
  while (d.cluster > 0 && d.items > resident_clusters(d.cluster)) d.cluster /= 2;
  if (keys > (d.items * d.cluster >= 64 ? 1024ll : 512ll) * d.cluster) d.cluster = 0;
  d.part_off = ((size_t)d.grid * sizeof(int2) + 255) & ~(size_t)255;
  d.bytes = d.cluster ? 0 : d.part_off + (size_t)2 * d.grid * d.rows * (a->cache.head_dim + 8) * sizeof(float);
  return d;
}

template <typename T, int HD, int ROWS>
cudaError_t decode_launch(const lw::PagedDecodeParams& p, const DecodePlan& d, cudaStream_t s, bool pdl) {
  constexpr int smem = lw::DecodeShape<HD, ROWS>::kBytes;
  if (d.cluster) {
    auto kern = lw::paged_decode_cluster_kernel<T, HD, ROWS>;
    cudaError_t e = lw_host::allow_smem<lw::paged_decode_cluster_kernel<T, HD, ROWS>>(smem);
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
  cudaError_t e = lw_host::allow_smem<lw::paged_decode_kernel<T, HD, ROWS>>(smem);
  if (e != cudaSuccess) return e;
  e = lw_launch(kern, dim3(d.grid), dim3(lw::kPdThreads), smem, s, pdl, p);
  if (e != cudaSuccess) return e;
  return lw_launch(lw::paged_join_kernel<T, HD, ROWS>, dim3(d.grid, std::min(ROWS, d.group)), dim3(lw::kPdThreads), 0,
                   s, true, p);
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
  const int hd = a->cache.head_dim;
  const cudaError_t e = a->cache.dtype == LW_DTYPE_F16 ? decode_dispatch<__half>(p, hd, d, s, pdl)
                                                       : decode_dispatch<__nv_bfloat16>(p, hd, d, s, pdl);
  return e == cudaSuccess ? LW_OK : LW_ERR_LAUNCH;
}

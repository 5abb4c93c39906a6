// Attention of prompt chunks over the paged cache (lw_paged_attention with
// q_offsets): the newest tokens of every sequence against all it keeps, causal,
// with an optional window and first keys that stay visible.
//
//   S = scale Q K^T, P = exp2(S log2(e) - m), O = sum P V / sum P
//
// on the 5th-generation tensor cores. A piece of work is two tiles of 128 rows; a
// row is a position x a query head of one kv head's group, so K and V are read
// once for the group and a tile spans only 128 / group positions (few masked
// keys on the diagonal and at a window's edges). It walks the 128-key tiles that
// any of its rows sees. Tensor memory holds, for each of the two row tiles, S
// (128 fp32 columns; P in 16 bits overwrites its first 64) and O (head_dim fp32
// columns). One CTA per SM; warps are specialised:
//   warps 0-3, 4-7  softmax of row tile 0 / 1, one row per thread: read S, mask,
//                   keep the running maximum and sum in fp32, write P. The
//                   accumulator is rescaled only when a row's maximum has grown
//                   by more than 2^8 (P stays within the type's range; the sum
//                   and O carry the same factor), so O rarely moves.
//   warp 8          TMA copies: Q once, K and V tiles page by page into a ring.
//   warp 9          issues tcgen05.mma: S_g = Q_g K^T (both from shared memory),
//                   O_g += P_g V (P from tensor memory). While one row tile is in
//                   its softmax the tensor cores work on the other.
//   warp 10         finds the work: its own block's first, then that of blocks
//                   not yet launched, which it takes over (cluster launch
//                   control), so copies and products of the next piece run
//                   beside the end of this one and SMs share the work evenly.
// tcgen05.mma instructions of one thread run in the order they are issued, so S of
// the next keys may overwrite P as soon as the product that reads P is issued,
// and the barrier of S(j) covers O's update j - 1 too. P is handed over in two
// parts, so most of the second product runs beside the last exponentials.
//
// When the row tiles alone leave SMs idle (few rows, a long cache) the keys are
// cut into slices as well; each writes (m, sum, fp32 O) to the workspace and a
// second kernel joins them in order. The launch knows only how long a context the
// table can hold; a row tile that sees fewer keys takes fewer slices, or none.
//
// What hidden slots hold never reaches a result. Pages that no row sees are
// zero-filled by the copy (their table entries are not read). In a tile that
// some row does not see whole, the values are scanned: rows of V that nobody
// sees are cleared, and where a value that some rows see is an infinity or a NaN
// it is cleared too (0 * it would reach the others) and added at the end to the
// rows that see it.
//
// Every wait is bounded; on expiry LW_ERR_TIMEOUT is recorded and the CTA ends.
//
// Measured (32 / 8 heads of 128; several GPUs): one prompt of 8192 tokens 547 - 566
// us, 0.97 - 1.0 PFLOP/s, 0.6 of the measured burst of a bf16 GEMM at an SM clock of
// 1.6 to 1.75 GHz under the power limit; six prompts of 129 to 2111 tokens 249 - 255
// us, 0.90 - 0.92 PFLOP/s. Per key tile the tensor cores and the special-function
// unit (exponentials) need 2048 cycles each for the two row tiles; a tile takes
// 3480. No unit is full (tensor and special function 58 %, issue 36 %): the period is
// a chain, a row tile's softmax (2300: read and mask 260, maximum 250, rescale check
// 155, exponentials 1450) and then its way through the tensor cores (1160). Making S
// before it is waited for (526 -> 575 us) and two threads per row (685) did not
// shorten it; weights formed before the tile's maximum is known are not built.
#include <algorithm>
#include <cmath>

#include "paged.cuh"
#include "tcgen05.cuh"
#include "tma_host.cuh"

namespace lw {

constexpr int kPmRows = 128;                 // rows per tile (UMMA M)
constexpr int kPmKeys = 128;                 // keys per tile
constexpr int kPmThreads = 384;              // three warpgroups: softmax, softmax, copies and MMA
// Registers per thread after the split: a softmax row holds 128 scores. The sum
// is what the block is launched with (168 x 384).
constexpr int kPmSoftmaxRegs = 224, kPmOtherRegs = 56;
static_assert(2 * 128 * kPmSoftmaxRegs + 128 * kPmOtherRegs <= 168 * kPmThreads, "registers of the launch");
constexpr int kPmTmaWarp = 8, kPmMmaWarp = 9, kPmWorkWarp = 10;
constexpr int kPmSliceTiles = 4;             // key tiles of a slice at least
constexpr long long kPmWaitNs = 2000000000;
constexpr float kPmGrow = 8.0f;              // log2 of what a row's maximum may grow by before O is rescaled
// log2 of the largest P against the maximum it was taken from: fp16 leaves the
// range above 1 that growth does not need to small weights
template <typename T>
constexpr float kPmMaxWeightLog2 = Elem<T>::kMaxWeightLog2 > kPmGrow ? Elem<T>::kMaxWeightLog2 - kPmGrow : 0.0f;
constexpr int kPmPart = 96;                  // keys of P's first part

struct PromptParams {
  CUtensorMap tm_q;   // {head_dim, heads, tokens}, box {64, group, rp}
  CUtensorMap tm_k;   // {head_dim, slots, kv heads, pages}, box {64, min(page, 128), 1, 1}
  CUtensorMap tm_v;
  PagedView c;
  void* out;
  long long o_t, o_h;
  int T, nq, group, rp;   // rp: positions per row tile
  int no_page;            // a page index past the pool: its copy is zeros
  const int* off;
  int window, sinks;
  float scale_log2;
  int zero_tail;
  int slices;
  int* part_n;            // [T][nq]: slices of the row (1: its result is written)
  float2* part_ml;        // [slices][T][nq]
  float* part_o;          // [slices][T][nq][head_dim]
};

// A piece of work: up to 2 * rp positions of one sequence x one kv head's group,
// against a slice of the key tiles they see.
struct PromptWork {
  int valid;           // 0: there is no more; -1: rows tok0 .. of a sequence that is refused (never published)
  int kvh, slice, slices, b;
  int tok0, np;        // first row of q, positions
  int pos0, last;      // position of the first, of the last
  int lo0;             // first key that the window of any row reaches
  int ns, w0, t0, nt;  // tiles 0 .. ns - 1 and w0 .. are seen; the slice is the nt from the t0-th on
  LW_DEV int key_of(int i) const { return (t0 + i < ns ? t0 + i : w0 + t0 + i - ns) * kPmKeys; }
};

// The row tiles of a slot: sequence b owns the slots from off[b] / R + b on (R
// positions per slot), at least as many as its rows need (ceil(n / R) <=
// floor((off + n) / R) - floor(off / R) + 1), so a slot finds its sequence by
// bisection and the grid needs only T and B. Some slots have no rows. A whole warp
// looks, 32 sequences at a time.
LW_DEV bool find_work(const PromptParams& p, int slot, int kvh, int slice, PromptWork& w) {
  const int R = 2 * p.rp;
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.c.B, o, n, len;   // off[lo] / R + lo <= slot, and hi's is past it
  for (;;) {
    const int step = (hi - lo + 31) / 32, at = min(lo + lane * step, hi - 1);
    const int off_at = p.off[at], off_next = p.off[at + 1], len_at = p.c.lens[at];
    const uint32_t ok = __ballot_sync(0xffffffffu, lo + lane * step < hi && off_at / R + at <= slot);
    const int last = ok ? 31 - __clz(ok) : 0;   // the offsets do not fall, so these are the first lanes
    if (step == 1) {
      lo += last;
      o = __shfl_sync(0xffffffffu, off_at, last);
      n = __shfl_sync(0xffffffffu, off_next, last) - o;
      len = __shfl_sync(0xffffffffu, len_at, last);
      break;
    }
    lo += last * step;
    hi = min(hi, lo + step);
  }
  const int i0 = (slot - (o / R + lo)) * R;
  w.valid = 0;
  if (i0 < 0 || i0 >= n) return false;
  w.tok0 = o + i0;
  w.np = min(R, n - i0);
  if (o < 0 || (long long)o + n > p.T) {   // rows that q does not have
    lw_record_error(LW_ERR_BAD_INDEX);
    w.valid = -1;
    return false;
  }
  w.valid = 1;
  w.kvh = kvh;
  w.slice = slice;
  w.b = lo;
  w.pos0 = cut_len(p.c, len) - n + i0;   // negative: more rows than tokens
  if (w.pos0 < 0) lw_record_error(LW_ERR_BAD_INDEX);
  w.last = w.pos0 + w.np - 1;
  w.lo0 = window_start(max(w.pos0, 0), p.window);
  w.w0 = w.lo0 / kPmKeys;
  w.ns = p.window > 0 ? min((min(p.sinks, w.lo0) + kPmKeys - 1) / kPmKeys, w.w0) : 0;
  const int all = w.last < 0 ? 0 : w.ns + w.last / kPmKeys + 1 - w.w0;
  w.slices = max(1, min(p.slices, all / kPmSliceTiles));
  if (slice >= w.slices) return false;
  w.t0 = (int)((long long)all * slice / w.slices);
  w.nt = (int)((long long)all * (slice + 1) / w.slices) - w.t0;
  return true;
}

// Bits 0 .. n - 1 (all of them from n = 32 on, none up to 0).
LW_DEV uint32_t low_bits(int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; }

// The largest of three; NaN if one is.
LW_DEV float max3(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Zeros in the place of the infinities and NaNs of a row of V (128 bytes in each half).
template <typename T>
__device__ __noinline__ void clear_nonfinite(uint8_t* row, int halves, int half_bytes) {
  for (int h = 0; h < halves; ++h)
    for (int c = 0; c < 32; ++c) {
      uint32_t* at = reinterpret_cast<uint32_t*>(row + h * half_bytes) + c;
      constexpr uint32_t kLo = Elem<T>::kExpMask, kHi = kLo << 16;
      uint32_t u = *at;
      if ((u & kLo) == kLo) u &= 0xFFFF0000u;
      if ((u & kHi) == kHi) u &= 0x0000FFFFu;
      *at = u;
    }
}

// What was cleared and the row sees, added to its accumulator (whole warps).
template <typename T, int HD>
__device__ __noinline__ void add_nonfinite(const PromptParams& p, const PromptWork& w, int pos, int lo, int sinks,
                                           uint32_t to) {
  for (int x = 0; x < HD / 8; ++x) {
    uint32_t o[8];
    tmem_ld8(to + 8 * x, o);
    for (int i = 0; i < w.nt; ++i) {
      const int key0 = w.key_of(i);
      if (!(key0 + kPmKeys - 1 > w.pos0 || (p.window > 0 && key0 <= w.last - p.window && key0 + kPmKeys > sinks)))
        continue;   // every row sees the tile whole
      for (int key = key0; key < key0 + kPmKeys; ++key) {
        if (!(key <= pos && (key > lo || key < sinks))) continue;
        const int page = page_id(p.c, w.b, key);
        if (page < 0) continue;
        const T* v = static_cast<const T*>(p.c.v) + page * p.c.vp + w.kvh * p.c.vh +
                     (key & (p.c.page_size - 1)) * p.c.vs + 8 * x;
        for (int e = 0; e < 8; ++e) {
          const float f = static_cast<float>(v[e]);
          if (!isfinite(f)) o[e] = __float_as_uint(__uint_as_float(o[e]) + f);
        }
      }
    }
    __syncwarp();
    tmem_st8(to + 8 * x, o);
  }
  tmem_wait_st();
}

// Whether the piece's tiles hold a key that the row sees (asked for a row without a weight).
__device__ __noinline__ bool sees_key(const PromptParams& p, const PromptWork& w, int pos, int lo, int sinks) {
  for (int i = 0; i < w.nt; ++i) {
    const int key0 = w.key_of(i);
    for (int key = key0; key < key0 + kPmKeys && key <= pos; key += 16)   // 16 keys are of one page
      if ((min(key + 15, pos) > lo || key < sinks) && page_id(p.c, w.b, key) >= 0) return true;
  }
  return false;
}

template <int HD>
struct PromptSmem {
  static constexpr int kTile = kPmKeys * HD * 2;              // a K, V or Q tile
  static constexpr int kSlots = HD == 128 ? 4 : 8;            // K and V tiles in the ring
  static constexpr int kStage = 32 * 128;                     // a softmax warp's rows on their way out, 128 bytes at a time
  static constexpr int kBytes = 1024 + (2 + kSlots) * kTile + 8 * kStage;
};

template <typename T, int HD>
__global__ void __launch_bounds__(kPmThreads, 1) paged_prompt_kernel(const __grid_constant__ PromptParams p) {
  using S = PromptSmem<HD>;
  constexpr int NS = S::kSlots, HALVES = HD / 64, HALF = kPmKeys * 128;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(16) uint4 clc_s;
  __shared__ __align__(8) unsigned long long bar_q, bar_qfree, bar_full[NS], bar_empty[NS], bar_s[2], bar_p[2][2],
      bar_o[2], bar_work, bar_taken, bar_clc, bar_done;
  __shared__ PromptWork work_s;
  __shared__ uint32_t tmem_s;
  __shared__ volatile int abort_s, odd_s[4];   // odd_s[piece mod 4]: a value was cleared that rows see
  __shared__ volatile uint8_t lost_s[8];       // key tile mod 8: its 16-key groups whose page id is outside the pool

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  auto slot_at = [&](int s) { return (uint32_t)(2 + s) * S::kTile; };

  if (tid == 0) {
    mbar_init(smem_u32(&bar_q), 1);
    mbar_init(smem_u32(&bar_qfree), 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(smem_u32(&bar_s[g]), 1);
      for (int h = 0; h < 2; ++h) mbar_init(smem_u32(&bar_p[g][h]), 4);
      mbar_init(smem_u32(&bar_o[g]), 1);
    }
    mbar_init(smem_u32(&bar_work), 1);
    mbar_init(smem_u32(&bar_taken), 10);   // the softmax, copy and MMA warps
    mbar_init(smem_u32(&bar_clc), 1);
    mbar_init(smem_u32(&bar_done), 1);
    abort_s = 0;
    for (int i = 0; i < 4; ++i) odd_s[i] = 0;
    fence_mbar_init();
  }
  if (warp == kPmMmaWarp) {
    tmem_alloc(smem_u32(&tmem_s), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  pdl_wait();
  pdl_launch_dependents();

  // Bounded waits: the first to give up makes the others stop at their next one.
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    if (abort_s) return false;
    if (mbar_wait_bounded(bar, parity, kPmWaitNs)) return true;
    abort_s = 1;
    return false;
  };
  auto warp_wait = [&](uint32_t bar, uint32_t parity) -> bool {
    return __shfl_sync(0xffffffffu, wait(bar, parity) ? 1u : 0u, 0) != 0;
  };
  // The warp's copy of piece `it` (false: no more, or a wait gave up).
  auto take = [&](int it, PromptWork& w) -> bool {
    if (!warp_wait(smem_u32(&bar_work), it & 1)) return false;
    w = work_s;
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bar_taken));
    return w.valid != 0;
  };
  const bool windowed = p.window > 0;

  if (warp >= kPmTmaWarp) {
    // the third warpgroup gives registers to the other two
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPmOtherRegs));
    if (warp == kPmTmaWarp) {
      // ---- copies. Tile i's K is copy 2i of the ring, its V copy 2i + 1 (i
      // counts through all pieces). Lane (page of the tile, half of the head
      // dim) issues one box each.
      const int pg = min(p.c.page_size, kPmKeys), npg = kPmKeys / pg;   // slots per box, boxes per tile and half
      const int my_pg = lane % npg, my_half = lane / npg;
      const bool mine = my_half < HALVES;
      if (lane == 0) {
        tma_prefetch_map(&p.tm_q);
        tma_prefetch_map(&p.tm_k);
        tma_prefetch_map(&p.tm_v);
      }
      int x = 0, s = 0, nq = 0;      // copies issued, the next one's slot, Q loads issued
      uint32_t phase = 1;            // of the slots' emptiness (the first pass over the ring does not wait)
      bool ok = true;
      PromptWork w;
      for (int it = 0; ok && take(it, w); ++it) {
        auto page_at = [&](int i) {   // page of this lane's part of tile i (no_page: zeros)
          const int first = w.key_of(i) + my_pg * pg, end = first + pg - 1;
          if (!(first <= w.last && (!windowed || end >= w.lo0 || first < p.sinks))) return p.no_page;
          return page_id(p.c, w.b, first);
        };
        int page = w.nt > 0 ? page_at(0) : 0;
        for (int i = 0; i < w.nt && ok; ++i) {
          const int key0 = w.key_of(i);
          const int next = i + 1 < w.nt ? page_at(i + 1) : 0;   // asked for a tile ahead
          // a page id outside the pool: its keys (16-key groups) are hidden, its copy is zeros
          const uint32_t bad_boxes = __ballot_sync(0xffffffffu, page < 0) & ((1u << npg) - 1u);
          if (lane == 0) {
            uint32_t groups = 0;
            for (int y = 0; y < npg; ++y)
              if ((bad_boxes >> y) & 1u) groups |= ((1u << (pg / 16)) - 1u) << (y * (pg / 16));
            lost_s[(x >> 1) & 7] = (uint8_t)groups;
          }
          const int from = page < 0 ? p.no_page : page;
          const int slot = key0 & (p.c.page_size - 1);   // within a page of more than 128 slots
          for (int kv = 0; kv < 2; ++kv) {
            if (!(ok = warp_wait(smem_u32(&bar_empty[s]), phase))) break;
            const uint32_t bar = smem_u32(&bar_full[s]);
            if (lane == 0) mbar_arrive_expect_tx(bar, S::kTile);
            __syncwarp();
            if (mine)
              tma_load_4d(base + slot_at(s) + my_half * HALF + my_pg * pg * 128, kv ? &p.tm_v : &p.tm_k, my_half * 64,
                          slot, w.kvh, from, bar);
            __syncwarp();
            ++x;
            if (++s == NS) s = 0, phase ^= 1u;
            if (kv == 0 && i == 0) {   // Q once the last scores of the piece before are done
              if (nq > 0 && !(ok = warp_wait(smem_u32(&bar_qfree), (nq - 1) & 1))) break;
              if (lane == 0) {
                const int ng = w.np > p.rp ? 2 : 1;
                mbar_arrive_expect_tx(smem_u32(&bar_q), (uint32_t)(HALVES * 128 * p.group * p.rp) * ng);
                for (int g = 0; g < ng; ++g)
                  for (int h = 0; h < HALVES; ++h)
                    tma_load_3d(base + g * S::kTile + h * HALF, &p.tm_q, h * 64, w.kvh * p.group, w.tok0 + g * p.rp,
                                smem_u32(&bar_q));
              }
              __syncwarp();
              ++nq;
            }
          }
          page = next;
        }
      }
      // no copy may land after the CTA has ended (immediate unless a wait gave up)
      if (lane == 0) {
        if (nq > 0) mbar_wait_bounded(smem_u32(&bar_q), (nq - 1) & 1, kPmWaitNs);
        for (int y = max(0, x - NS); y < x; ++y)
          mbar_wait_bounded(smem_u32(&bar_full[y % NS]), (y / NS) & 1, kPmWaitNs);
      }
      __syncwarp();
    } else if (warp == kPmMmaWarp) {
      // ---- tensor cores
      const bool leader = elect_one_sync();   // one thread issues everything: commits follow its instructions
      constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
      constexpr uint32_t kCommon = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((uint32_t)(kPmRows >> 4) << 24);
      constexpr uint32_t kDescS = kCommon | ((uint32_t)(kPmKeys >> 3) << 17);              // B = K, K-major
      constexpr uint32_t kDescO = kCommon | ((uint32_t)(HD >> 3) << 17) | (1u << 16);      // B = V, N-major
      auto scores = [&](int g, int s) {   // S_g = Q_g K^T
        const uint64_t a = sw128_desc(base + g * S::kTile), k = sw128_desc(base + slot_at(s));
#pragma unroll
        for (int x = 0; x < HD / 16; ++x) {
          const uint64_t o = (uint64_t)((x / 4) * (HALF >> 4) + (x % 4) * 2);
          tc_mma_f16(tmem + g * kPmKeys, a + o, k + o, kDescS, x != 0);
        }
      };
      auto values = [&](int g, int s, int x0, int x1, bool first) {   // O_g += P_g V, keys 16 x0 .. 16 x1 - 1
        const uint64_t v = sw128_mn_desc(base + slot_at(s), HALF);
#pragma unroll
        for (int x = x0; x < x1; ++x)
          tc_mma_f16_ts(tmem + 2 * kPmKeys + g * HD, tmem + g * kPmKeys + 8 * x, v + (uint64_t)(x * (2048 >> 4)),
                        kDescO, !first || x != 0);
      };
      int s = 0, nq = 0, np[2] = {0, 0};   // ring slot, Q loads awaited, P tiles of each row tile awaited
      uint32_t phase = 0;
      auto step = [&] {
        if (++s == NS) s = 0, phase ^= 1u;
      };
      bool ok = true;
      PromptWork w;
      for (int it = 0; ok && take(it, w); ++it) {
        if (w.nt == 0) continue;
        const int ng = w.np > p.rp ? 2 : 1;
        ok = warp_wait(smem_u32(&bar_full[s]), phase) && warp_wait(smem_u32(&bar_q), nq++ & 1);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          for (int g = 0; g < ng; ++g) {
            scores(g, s);
            tc_commit(smem_u32(&bar_s[g]));
          }
          tc_commit(smem_u32(&bar_empty[s]));
          if (w.nt == 1) tc_commit(smem_u32(&bar_qfree));
        }
        __syncwarp();
        step();
        for (int i = 0; i < w.nt && ok; ++i) {
          const int sv = s;
          if (!(ok = warp_wait(smem_u32(&bar_full[sv]), phase))) break;
          step();   // at the next tile's K
          for (int g = 0; g < ng; ++g) {
            const uint32_t par = np[g]++ & 1;
            if (!(ok = warp_wait(smem_u32(&bar_p[g][0]), par))) break;
            tc_fence_after();
            if (leader) values(g, sv, 0, kPmPart / 16, i == 0);
            __syncwarp();
            ok = warp_wait(smem_u32(&bar_p[g][1]), par);
            if (ok && g == 0 && i + 1 < w.nt) ok = warp_wait(smem_u32(&bar_full[s]), phase);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
              values(g, sv, kPmPart / 16, kPmKeys / 16, i == 0);
              if (g == ng - 1) tc_commit(smem_u32(&bar_empty[sv]));
              if (i + 1 < w.nt) {
                scores(g, s);
                tc_commit(smem_u32(&bar_s[g]));
                if (g == ng - 1) {
                  tc_commit(smem_u32(&bar_empty[s]));
                  if (i + 2 == w.nt) tc_commit(smem_u32(&bar_qfree));
                }
              } else {
                tc_commit(smem_u32(&bar_o[g]));
              }
            }
            __syncwarp();
          }
          if (ok && i + 1 < w.nt) step();
        }
      }
      // tensor memory may not be released under a running instruction
      if (leader) {
        tc_commit(smem_u32(&bar_done));
        mbar_wait_bounded(smem_u32(&bar_done), 0, kPmWaitNs);
      }
      __syncwarp();
    } else if (warp == kPmWorkWarp) {
      // ---- work: publish a piece, and when every warp has taken it, ask for another
      // Block x: kv head x % heads of slot x / heads from the end. The last positions
      // see the most keys, so the longest pieces of all heads come first and the
      // short ones even out the end (head by head, the last head's long pieces were
      // the end: 8192 tokens 597 us instead of 545).
      int x = blockIdx.x, y, z = blockIdx.z, it = 0;
      const int slots = (int)(gridDim.x / (unsigned)p.c.nkv);
      uint32_t asked = 0;
      bool more = true;
      PromptWork w;
      auto publish = [&]() -> bool {
        if (lane == 0) {
          work_s = w;
          mbar_arrive(smem_u32(&bar_work));
        }
        __syncwarp();
        // most of a piece's time: asleep, not polling beside the softmax warps
        const uint32_t bar = smem_u32(&bar_taken), parity = it++ & 1;
        const unsigned long long t0 = globaltimer_ns();
        bool ok = true;
        while (ok && !mbar_try_wait_sleep(bar, parity, 20000)) {
          if (abort_s || (long long)(globaltimer_ns() - t0) > kPmWaitNs) {
            lw_record_error(LW_ERR_TIMEOUT);
            abort_s = 1;
            ok = false;
          }
        }
        return __shfl_sync(0xffffffffu, ok ? 1u : 0u, 0) != 0;
      };
      while (more) {
        const int slot = slots - 1 - x / p.c.nkv, kvh = x % p.c.nkv, slice = z;
        const bool found = find_work(p, slot, kvh, slice, w);
        // rows refused_0 .. of a sequence whose rows run past q's
        const int refused = slice == 0 && w.valid < 0 ? min(w.np, p.T - w.tok0) : 0, refused_0 = w.tok0;
        if (found && !publish()) break;
        if (lane == 0) {
          fence_proxy_async_smem();   // the answer before has been read
          mbar_arrive_expect_tx(smem_u32(&bar_clc), 16);
          clc_try_cancel(smem_u32(&clc_s), smem_u32(&bar_clc));
        }
        __syncwarp();
        if (!warp_wait(smem_u32(&bar_clc), asked++ & 1)) break;
        more = clc_answer(smem_u32(&clc_s), x, y, z);
        __syncwarp();
        auto clear_row = [&](int r) {
          for (int i = lane; i < p.group * (HD / 8); i += 32)
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + r * p.o_t + (kvh * p.group + i / (HD / 8)) * p.o_h +
                                      (i % (HD / 8)) * 8) = make_uint4(0, 0, 0, 0);
        };
        for (int r = max(0, refused_0); r < refused_0 + refused; ++r) {
          if (p.zero_tail) clear_row(r);
          if (p.slices > 1)   // nothing to join
            for (int i = lane; i < p.group; i += 32) p.part_n[(long long)r * p.nq + kvh * p.group + i] = 1;
        }
        if (p.zero_tail && slice == 0) {   // rows of no sequence: before the first, behind the last
          const int first = max(0, min(p.T, p.off[0])), behind = max(first, p.off[p.c.B]);
          for (int x0 = slot; x0 < first + max(0, p.T - behind); x0 += slots)
            clear_row(x0 < first ? x0 : behind + x0 - first);
        }
      }
      w.valid = 0;
      if (!more) publish();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPmSoftmaxRegs));
    // ---- softmax of row tile g, row r
    const int g = warp >> 2, r = tid & 127, r_pos = r / p.group, r_head = r - r_pos * p.group;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + g * kPmKeys, to = tmem + lanes + 2 * kPmKeys + g * HD;
    uint8_t* stage = base_ptr + slot_at(NS) + warp * S::kStage;
    int tiles = 0, ns = 0, no = 0;   // key tiles of all pieces, S tiles and O tiles of this row tile
    bool ok = true;
    PromptWork w;
    for (int it = 0; ok && take(it, w); ++it) {
      if (tid == 0) odd_s[(it + 2) & 3] = 0;
      if (g == 1 && w.np <= p.rp) {   // no second row tile
        tiles += w.nt;
        continue;
      }
      const int npos = min(p.rp, w.np - g * p.rp);
      const bool have = r < npos * p.group;
      const int first_pos = w.pos0 + g * p.rp, last_pos = first_pos + npos - 1;
      const int pos = have ? first_pos + r_pos : -1;
      const int lo = windowed ? pos - p.window : -1;   // keys above lo, or below sinks
      const int sinks = windowed ? p.sinks : 0;
      float m = -INFINITY, l = 0.f;
      // key tiles that a row of this row tile / of the piece does not see whole:
      // past the one, or up to the other and not among the first keys alone
      const int mask_hi = first_pos - (kPmKeys - 1), mask_lo = windowed ? last_pos - p.window : -1;
      const int cut_hi = w.pos0 - (kPmKeys - 1), cut_lo = windowed ? w.last - p.window : -1;
      int key0 = w.key_of(0);
      for (int i = 0; i < w.nt; ++i, ++tiles, key0 = w.t0 + i == w.ns ? w.w0 * kPmKeys : key0 + kPmKeys) {
        if (!(ok = warp_wait(smem_u32(&bar_s[g]), ns++ & 1))) break;
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_ld32(ts + 32 * x, s[x]);
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_regs_ready(s[x]);
        const uint32_t lost = lost_s[tiles & 7];
        const bool past_sinks = key0 + kPmKeys > sinks;
        if (key0 > mask_hi || (key0 <= mask_lo && past_sinks) || lost) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            // bit e: the row sees key k0 + e
            const int k0 = key0 + 32 * x;
            const uint32_t gone = ((lost >> (2 * x)) & 1u ? 0xFFFFu : 0u) | ((lost >> (2 * x)) & 2u ? 0xFFFF0000u : 0u);
            const uint32_t seen = low_bits(pos + 1 - k0) & (~low_bits(lo + 1 - k0) | low_bits(sinks - k0)) & ~gone;
#pragma unroll
            for (int e = 0; e < 32; ++e) s[x][e] = (seen >> e) & 1u ? s[x][e] : 0xFF800000u;   // -infinity
          }
        }
        float mx[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          mx[x] = max3(__uint_as_float(s[x][0]), __uint_as_float(s[x][1]), __uint_as_float(s[x][2]));
#pragma unroll
          for (int e = 3; e < 31; e += 2) mx[x] = max3(mx[x], __uint_as_float(s[x][e]), __uint_as_float(s[x][e + 1]));
          mx[x] = max3(mx[x], mx[x], __uint_as_float(s[x][31]));
        }
        // a NaN among the row's scores makes its maximum, and so all of the row, NaN
        // (the base of the weights, rounded up: none is above 2^kPmMaxWeightLog2)
        const float mt = __fmaf_ru(max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]), p.scale_log2, -kPmMaxWeightLog2<T>);
        if (i == 0) {
          m = have ? mt : 0.f;   // a row that is none holds anything
        } else {
          const bool grow = have && !(mt <= __fadd_rd(m, kPmGrow));
          if (__any_sync(0xffffffffu, grow)) {
            // O's update i - 1 is complete (S(i) was issued after it)
            const float f = !grow ? 1.f : (m == -INFINITY ? 0.f : ex2(m - mt));
            if (grow) m = mt;
            l *= f;
#pragma unroll
            for (int x = 0; x < HD / 32; ++x) {
              uint32_t o[32];
              tmem_ld32(to + 32 * x, o);
              tmem_wait_ld();
              tmem_regs_ready(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(to + 32 * x, o);
            }
          }
        }
        if (g == 0 && (key0 > cut_hi || (key0 <= cut_lo && past_sinks))) {
          // row r of V
          const int xv = 2 * tiles + 1;
          if (!(ok = warp_wait(smem_u32(&bar_full[xv % NS]), (xv / NS) & 1))) break;
          const uint8_t* row = base_ptr + slot_at(xv % NS) + r * 128;
          uint32_t any = 0u;   // NaN in either half once an infinity or a NaN has passed: 0 * it
#pragma unroll
          for (int c = 0; c < HALVES * 8; ++c) {
            const uint4 v = lds128(row + (c / 8) * HALF + (((c + r) & 7) << 4));   // an order that spreads over the banks
            any = Elem<T>::fma0(v.x, Elem<T>::fma0(v.y, Elem<T>::fma0(v.z, Elem<T>::fma0(v.w, any))));
          }
          if (has_nonfinite<T>(any)) {
            const int key = key0 + r;
            clear_nonfinite<T>(base_ptr + slot_at(xv % NS) + r * 128, HALVES, HALF);
            if (key <= w.last && (!windowed || key >= w.lo0 || key < p.sinks)) odd_s[it & 3] = 1;
          }
          fence_proxy_async_smem();   // before the tensor cores read it
        }
        const float sub = m == -INFINITY ? 0.f : m;   // no key seen yet: every weight is 0
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), sub2 = make_float2(-sub, -sub);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // weights rounded to T for the second product: half a step each, averaged
        // over the keys (fp16: weights under 2^-21 of the base's maximum by up to
        // 2^-32 of it); their sum is that of the unrounded ones
        auto weights = [&](int e) {
          const int x = e / 16, y = (2 * e) % 32;
          float2 a = fma2(make_float2(__uint_as_float(s[x][y]), __uint_as_float(s[x][y + 1])), scale2, sub2);
          a.x = ex2(a.x);
          a.y = ex2(a.y);
          sum[e & 1] = add2(sum[e & 1], a);
          return Elem<T>::pack(a.x, a.y);
        };
        static_assert(kPmPart == 96, "the stores below");
        {
          uint32_t u[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) u[e] = weights(e);
          tmem_st32(ts, u);
        }
        uint32_t u[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) u[e] = weights(32 + e);
        tmem_st16(ts + 32, u);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_p[g][0]));
#pragma unroll
        for (int e = 0; e < 16; ++e) u[e] = weights(48 + e);
        tmem_st16(ts + 48, u);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_p[g][1]));
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      if (!ok) break;
      // ---- the row's result
      if (w.nt > 0) {
        if (!(ok = warp_wait(smem_u32(&bar_o[g]), no++ & 1))) break;
        tc_fence_after();
      }
      if (odd_s[it & 3]) add_nonfinite<T, HD>(p, w, pos, lo, sinks, to);
      if (have && m == -INFINITY && sees_key(p, w, pos, lo, sinks)) m = kAllBelow;
      const int tok = w.tok0 + g * p.rp + r_pos, head = w.kvh * p.group + r_head;
      // 128 bytes of each of the warp's 32 rows at a time go through shared memory
      // (16-byte chunk c of a row at chunk c ^ (row & 7)), so that eight lanes
      // write a row's 128 bytes together. row_at: this lane's row, in bytes, or -1.
      auto write_out = [&](uint8_t* out, long long row_at) {
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int row = 4 * k + lane / 8, c = lane % 8;
          const long long at = __shfl_sync(0xffffffffu, row_at, row);
          const uint4 v = lds128(stage + row * 128 + ((c ^ (row & 7)) << 4));
          if (at >= 0) *reinterpret_cast<uint4*>(out + at + c * 16) = v;
        }
        __syncwarp();
      };
      auto put = [&](int c, uint4 v) { sts128(stage + lane * 128 + ((c ^ (lane & 7)) << 4), v); };
      if (p.slices > 1 && w.slice == 0 && have) p.part_n[(long long)tok * p.nq + head] = w.slices;
      if (w.slices == 1) {
        const float inv = weight_inverse(m, l);
        const long long row_at = have ? (tok * p.o_t + head * p.o_h) * 2 : -1ll;
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += 64) {
          uint32_t o[2][32];
          if (w.nt > 0) {
            tmem_ld32(to + c0, o[0]);
            tmem_ld32(to + c0 + 32, o[1]);
            tmem_wait_ld();
            tmem_regs_ready(o[0]);
            tmem_regs_ready(o[1]);
          } else {
#pragma unroll
            for (int e = 0; e < 64; ++e) o[e / 32][e % 32] = 0u;
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              u[e] = Elem<T>::pack(__uint_as_float(o[c / 4][8 * (c % 4) + 2 * e]) * inv,
                                   __uint_as_float(o[c / 4][8 * (c % 4) + 2 * e + 1]) * inv);
            put(c, make_uint4(u[0], u[1], u[2], u[3]));
          }
          write_out(static_cast<uint8_t*>(p.out) + c0 * 2, row_at);
        }
      } else {
        const long long part = ((long long)w.slice * p.T + tok) * p.nq + head;
        if (have) p.part_ml[part] = make_float2(m, l);
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += 32) {
          uint32_t o[32];
          tmem_ld32(to + c0, o);
          tmem_wait_ld();
          tmem_regs_ready(o);
#pragma unroll
          for (int c = 0; c < 8; ++c) put(c, make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]));
          write_out(reinterpret_cast<uint8_t*>(p.part_o) + c0 * 4, have ? part * HD * 4 : -1ll);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kPmMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the key slices of every row, in order. A row per HD / 4 threads.
template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_prompt_join_kernel(const __grid_constant__ PromptParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int TPR = HD / 4;
  const long long row = (long long)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (row >= (long long)p.T * p.nq) return;
  const int tok = (int)(row / p.nq), head = (int)(row - (long long)tok * p.nq), d = (threadIdx.x % TPR) * 4;
  // four slices at a time; the first four are asked for before it is known how
  // many there are (what is read for nothing is thrown away)
  const long long step = (long long)p.T * p.nq;
  const int said = p.part_n[row];
  float2 ml[4];
  float4 o[4];
  auto load = [&](int i0, int n) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      ml[x] = make_float2(-INFINITY, 0.f);
      if (i0 + x < n) {
        ml[x] = p.part_ml[(i0 + x) * step + row];
        o[x] = *reinterpret_cast<const float4*>(p.part_o + ((i0 + x) * step + row) * HD + d);
      }
    }
  };
  load(0, p.slices);
  const int n = min(said, p.slices);
  // its one slice wrote the result; behind the last sequence: not ours
  if (n <= 1 || row_sequence(p.off, p.c.B, tok) < 0) return;
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 4) {
    if (i0) load(i0, n);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (i0 + x >= n || (ml[x].x == -INFINITY && ml[x].y == 0.f)) continue;   // a slice without a key for this row
      const float mn = fmaxf(M, ml[x].x), f0 = ex2(M - mn), f1 = ex2(ml[x].x - mn);
      M = mn;
      L = fmaf(L, f0, ml[x].y * f1);
      acc.x = fmaf(acc.x, f0, o[x].x * f1);
      acc.y = fmaf(acc.y, f0, o[x].y * f1);
      acc.z = fmaf(acc.z, f0, o[x].z * f1);
      acc.w = fmaf(acc.w, f0, o[x].w * f1);
    }
  }
  const float inv = weight_inverse(M, L);
  uint2 u = make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + tok * p.o_t + head * p.o_h + d) = u;
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
  // above 0: the maximum is taken before scaling; finite times log2(e), as the kernels use it
  if (!(a->scale > 0.f) || !std::isfinite(a->scale * 1.4426950408889634f)) return LW_ERR_BAD_SHAPE;
  if (!a->q_offsets && a->tokens != a->cache.batch) return LW_ERR_BAD_SHAPE;
  if (a->q_offsets && a->n_q_heads / a->cache.n_kv_heads > 64) return LW_ERR_UNSUPPORTED;
  if (a->tokens == 0) return LW_OK;
  if (a->cache.batch == 0) return LW_ERR_BAD_SHAPE;
  if (!a->q || !a->out) return LW_ERR_NULL_POINTER;
  if (!lw_host::aligned16(a->q) || !lw_host::aligned16(a->out) || !lw_host::strides8(a->q_strides, 2) ||
      !lw_host::strides8(a->out_strides, 2) || (reinterpret_cast<uintptr_t>(a->q_offsets) & 3u))
    return LW_ERR_ALIGNMENT;
  return LW_OK;
}

struct PromptPlan {
  int group, rp, slices;
  size_t ml_off, o_off, bytes;
};

PromptPlan prompt_plan(const lw_paged_attention_args* a) {
  PromptPlan d;
  d.group = a->n_q_heads / a->cache.n_kv_heads;
  d.rp = lw::kPmRows / d.group;
  // Keys are cut into slices only where the row tiles leave SMs idle, as many
  // slices as fill them, none below four key tiles.
  const long long R = 2 * d.rp;
  const long long ctas = ((long long)a->tokens + a->cache.batch * (R - 1)) / R * a->cache.n_kv_heads;
  long long keys = (long long)a->cache.table_width * a->cache.page_size;
  if (a->window > 0) keys = std::min(keys, (long long)a->window + a->sinks + R);
  const long long most = std::min(keys / (lw::kPmSliceTiles * lw::kPmKeys), lw_host::sm_count() / std::max(1ll, ctas));
  d.slices = (int)std::max(1ll, std::min(most, 64ll));
  const size_t rows = (size_t)a->tokens * a->n_q_heads * d.slices;
  d.ml_off = ((size_t)a->tokens * a->n_q_heads * sizeof(int) + 255) & ~(size_t)255;
  d.o_off = d.ml_off + ((rows * sizeof(float2) + 255) & ~(size_t)255);
  d.bytes = d.slices > 1 ? d.o_off + rows * a->cache.head_dim * sizeof(float) : 0;
  return d;
}

template <typename T, int HD>
cudaError_t prompt_launch(const lw::PromptParams& p, cudaStream_t s, bool pdl) {
  constexpr int smem = lw::PromptSmem<HD>::kBytes;
  auto kern = lw::paged_prompt_kernel<T, HD>;
  cudaError_t e = lw_host::allow_smem<lw::paged_prompt_kernel<T, HD>>(smem);
  if (e != cudaSuccess) return e;
  e = lw_launch(kern, dim3((unsigned)((p.T / (2 * p.rp) + p.c.B) * p.c.nkv), 1, (unsigned)p.slices),
                dim3(lw::kPmThreads), smem, s, pdl, p);
  if (e != cudaSuccess || p.slices == 1) return e;
  const long long rows = (long long)p.T * p.nq, per = 256 / (HD / 4);
  if ((rows + per - 1) / per > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  return lw_launch(lw::paged_prompt_join_kernel<T, HD>, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, true,
                   p);
}

// Tensor map of a pool [pages][heads][slots][head_dim] by its strides.
bool pool_map(CUtensorMap* m, CUtensorMapDataType type, const void* base, const lw_paged_cache& c,
              const long long* st) {
  const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)c.page_size, (uint64_t)c.n_kv_heads,
                            (uint64_t)std::max(1, c.n_pages)};
  const uint64_t strides[3] = {(uint64_t)st[2] * 2, (uint64_t)st[1] * 2, (uint64_t)st[0] * 2};
  const uint32_t box[4] = {64, (uint32_t)std::min(c.page_size, lw::kPmKeys), 1, 1};
  return lw::encode_nd_sw128(m, type, base, 4, dims, strides, box);
}

}  // namespace

int lw_paged_prompt_take_error() { return lw_tu_take_error(); }

extern "C" {

size_t lw_paged_attention_workspace_size(const lw_paged_attention_args* a) {
  if (check(a) != LW_OK || a->tokens == 0) return 0;
  return a->q_offsets ? prompt_plan(a).bytes : lw_paged_decode_workspace(a);
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
  const PromptPlan d = prompt_plan(a);
  lw::PromptParams p = {};
  p.c = lw_host::view_of(a->cache);
  p.out = a->out;
  p.o_t = a->out_strides[0];
  p.o_h = a->out_strides[1];
  p.T = a->tokens;
  p.nq = a->n_q_heads;
  p.group = d.group;
  p.rp = d.rp;
  p.no_page = std::max(1, a->cache.n_pages);
  p.off = a->q_offsets;
  p.window = a->window;
  p.sinks = a->sinks;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.zero_tail = a->zero_tail;
  p.slices = d.slices;
  p.part_n = static_cast<int*>(a->workspace);
  p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(a->workspace) + d.ml_off);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + d.o_off);
  const CUtensorMapDataType type =
      a->cache.dtype == LW_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t dims[3] = {(uint64_t)a->cache.head_dim, (uint64_t)a->n_q_heads, (uint64_t)a->tokens};
  const uint64_t strides[2] = {(uint64_t)a->q_strides[1] * 2, (uint64_t)a->q_strides[0] * 2};
  const uint32_t box[3] = {64, (uint32_t)d.group, (uint32_t)d.rp};
  // an empty pool has no address: every copy is past its end then
  const void* kb = a->cache.n_pages ? a->cache.k_pages : a->q;
  const void* vb = a->cache.n_pages ? a->cache.v_pages : a->q;
  if (((long long)p.T / (2 * p.rp) + p.c.B) * p.c.nkv > 0x7FFFFFFFll) return LW_ERR_UNSUPPORTED;   // blocks of the grid
  if (!lw::encode_nd_sw128(&p.tm_q, type, a->q, 3, dims, strides, box) ||
      !pool_map(&p.tm_k, type, kb, a->cache, a->cache.k_strides) ||
      !pool_map(&p.tm_v, type, vb, a->cache, a->cache.v_strides))
    return LW_ERR_UNSUPPORTED;   // strides that a tensor map does not take
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

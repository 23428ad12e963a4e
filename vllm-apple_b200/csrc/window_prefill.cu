// Attention of chunks of new tokens over a paged cache under a sliding window with sinks
// (visibility rule: window.cuh), fp16 or e4m3 cache (row format: kv_q8.cuh), on the
// 5th-generation tensor cores.
//
// One CTA takes a pair of 128-row tiles of one sequence and one kv head.  A row is a
// (token, query head of the group) pair, so every staged key serves all heads of the
// group and both tiles; the tiles' keys are the pair's key tiles of 128 (window.cuh), and
// no block without a key that some row sees is read, no tile without one multiplied.
//   * warps 0-7: softmax, one thread per row (TMEM lane = row), warps 0-3 tile 0 and 4-7
//     tile 1.  A row's 128 scores sit in the thread's registers (the other warps hand
//     theirs over with setmaxnreg); P goes back over S as fp16 and feeds the second product
//     from TMEM.  The maximum a row's powers are taken against only moves when a power
//     would pass 2^12 (fp16 ends at 2^16), so O is rarely rescaled: 494 us (of 8192 tokens,
//     below) with 2^6, 480 with 2^8, 476 from 2^10 on (before the waits were a warp's).  Rows
//     whose maximum does move cost what they rescale: 440 us become 488 to 494 with queries 4
//     to 32 times as large, 65 us (fp16, below) 71 to 72.
//   * warp 8, one thread: issues tcgen05.mma for both tiles in turn -- PV_0(j-1), S_0(j),
//     PV_1(j-1), S_1(j) -- so one tile's products run while the other is in its softmax.
//   * fp16 cache: warp 9 brings K and V key tiles into a ring of shared-memory slots by TMA,
//     one copy per block of the cache and 64 columns, in the 128-byte-swizzled layout of the
//     tensor core.  Blocks that no row of the pair sees are copied from past the tensor's end,
//     which gives zeros.  Block sizes that do not tile 128 keys (and cache layouts without a
//     tensor map) take 16-byte cp.async from warps 12-15 instead, whose issue takes as long as
//     a tile's products and softmax: four chunks of 512 under a window of 1024 (32 heads of 128
//     over 8) 65.1 us by TMA, 74.3 by cp.async.
//   * e4m3 cache: warps 12-19 copy rows by cp.async into a raw buffer two items ahead, and turn
//     them into fp16 (exactly) in the slot.  TMA into a raw ring was 2 % faster on 8192 tokens
//     and 2 % slower on short ones; four converting warps took 525 us where eight took 502
//     (before the waits were a warp's).
//   Keys that no row of the pair sees are never part of a result: they are zeros, or their
//   scores are masked for every row.
// What bounds it: 8192 tokens under a window of 4096 over an e4m3 cache take 440 us (57 % of
// the measured tensor peak for the visible products) in a graph's replay, 473 called one by one
// with other inputs each time; an fp16 cache 398.  Alone, on the same grid, the products take
// 342 us, the softmax 345, the conversion 369 and the barriers 237; the products of one tile
// wait for its softmax, and the overlap of the two tiles hides some of it.  Half-tile double
// buffering of S, P published in halves and polynomial powers were slower; TMEM is full, so no
// third tile fits.
// A key masked for one row but seen by another may hold an infinity or a NaN in V, and
// 0 * inf would reach the masked row.  In key tiles that are masked in part (at most a
// few per pair) warps 12 on replace such values by 0, and rows that do see them get
// them added at the end.
// Scores, statistics and O are fp32; P is rounded to fp16, the type of the V that the second
// product reads (error against 64 bits 2.6e-4 to 2.9e-4 of the result's size, where its own
// rounding to fp16 is 2.0e-4).
// Bounded waits: after a time-out every role runs its loop to the end without waiting or
// issuing (so the roles still meet at their barriers), nothing is written and
// VA_FLAG_WAIT_TIMEOUT is set.
#include <cudaTypedefs.h>
#include <limits.h>

#include "prefill_tc.cuh"
#include "window.cuh"

namespace {

constexpr int kRows = 128, kKeys = 128, kTiles = 2;
constexpr int kSoftmax = kTiles * kRows;
constexpr int kMmaWarp = kSoftmax / 32;
constexpr int kLoadWarp = kMmaWarp + 1;       // warps 10 and 11 only lend their registers
constexpr int kFirstProducer = kSoftmax + 128;
constexpr int kLag = 2;  // fp16 cp.async copies in flight behind the newest
constexpr int kScrub = 4;  // barriers of V tiles that wait to be scrubbed (TMA)
constexpr uint32_t kWaitLimit = 1u << 22;
constexpr uint32_t kTmemO = kTiles * kKeys;  // TMEM: S of both tiles, then O of both

template <int D, bool Q8, bool TMA>
struct Shape {
  // An e4m3 cache takes eight warps to convert, an fp16 one four for what is left to do.
  static constexpr int kProducers = Q8 ? 256 : 128;
  static constexpr int kThreads = kFirstProducer + kProducers;
  // Registers: the threads launch with kRegsLaunch each; the warpgroups past the softmax
  // ones go down to kRegsOther and the softmax warpgroups take what they give up.  e4m3, 8192
  // tokens (before the waits were a warp's): 502 us with 168 and 48, 480 with 176 and 40, 510
  // with 184 and 32; fp16 does not change from 184 to 208.  Held to 96 registers at launch, the
  // e4m3 kernels spill 12 bytes at head size 128 and 8 at 96, the others none.
  static constexpr int kRegsLaunch = Q8 ? 96 : 128, kRegsSoftmax = Q8 ? 176 : 192;
  static constexpr int kRegsOther = Q8 ? 40 : 64;
  static_assert(kThreads * kRegsLaunch <= 65536 &&
                    kSoftmax * kRegsSoftmax + (kThreads - kSoftmax) * kRegsOther <=
                        kThreads * kRegsLaunch,
                "register shares");
  static constexpr int NB = (D + 63) / 64;            // 64-column blocks of a row
  static constexpr uint32_t kTileBytes = NB * 128 * 128;
  // fp16 key tiles of K or V; an e4m3 cache keeps two more as they come
  static constexpr int kSlots = NB == 2 ? (Q8 ? 4 : 5) : 8;
  static constexpr uint32_t kRawBytes = Q8 ? kKeys * D : 0;
  static constexpr uint32_t oSlot = kTiles * kTileBytes;
  static constexpr uint32_t oRaw = oSlot + kSlots * kTileBytes;
  static constexpr uint32_t oInfo = oRaw + 2 * kRawBytes;  // int64 [128] row offsets (cp.async)
  static constexpr uint32_t oExp = oInfo + (TMA ? 0 : 128 * 8);  // fp16 scales: K [128], V [2][128]
  static constexpr uint32_t oBar = oExp + (Q8 ? 3 * 128 * 2 : 0);
  static constexpr uint32_t kBars = 2 * kSlots + (TMA ? kScrub : 0) + 3 * kTiles + 2;
  static constexpr uint32_t kBytes = oBar + kBars * 8 + 16 + 1024;  // + alignment slack
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

struct Args {
  CUtensorMap mk, mv;  // boxes of one block of one head, or 128 tokens of it (TMA)
  __half *out;
  const __half *q;
  const uint8_t *kc, *vc, *ks, *vs;
  const int32_t *bt, *qsl, *sl;
  int32_t *err;
  int64_t T, max_blocks, num_blocks;
  int S, Hkv, G, TQ, window, sinks;
  win::FastDiv bs, g;
  float scale_log2;
  int64_t s_block, s_head, s_token, c_block, c_head, c_token;
  int64_t q_s_token, q_s_head, o_s_token, o_s_head;
};

// The MMA warp's instructions, issued by the lane with `go` set.  (A branch around them
// would have every descriptor moved to uniform registers one by one.)
VA_DEVINL uint32_t elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one;
}
VA_DEVINL void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                       uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(go)
      : "memory");
}
VA_DEVINL void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                       uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(go)
      : "memory");
}
VA_DEVINL void umma_commit(uint64_t *bar, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          va::smem_addr(bar)),
      "r"(go)
      : "memory");
}

// 4-D tiled TMA load global -> shared, completion as tx bytes on `bar`.
VA_DEVINL void tma_load_4d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, int c3,
                           uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(va::smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3),
      "r"(va::smem_addr(bar))
      : "memory");
}

// What a pair of tiles reads, in key tiles.
struct Pair {
  int n_sink;             // key tiles 0 .. n_sink - 1 hold sinks
  int first[kTiles], last[kTiles];  // key tiles of each tile's run; last < 0: no rows
  int full_from[kTiles], full_to[kTiles], full_sink;  // those that every row sees whole

  VA_DEVINL Pair(const int (&pmin)[kTiles], const int (&pmax)[kTiles], int window, int sinks) {
    n_sink = (sinks + kKeys - 1) / kKeys;
    full_sink = sinks / kKeys;
#pragma unroll
    for (int h = 0; h < kTiles; ++h) {
      first[h] = win::run_start(pmin[h], window) / kKeys;
      last[h] = pmax[h] >= 0 ? pmax[h] / kKeys : -1;
      full_from[h] = (win::run_start(pmax[h], window) + kKeys - 1) / kKeys;
      full_to[h] = (pmin[h] + 1) / kKeys - 1;
    }
  }
  // key tile c holds a key that some row of tile h sees (h known at compile time, so that
  // nothing here is an indexed array)
  VA_DEVINL bool need(int h, int c) const {
    return c <= last[h] && (c >= first[h] || c < n_sink);
  }
  // every row of tile h sees every key of c
  VA_DEVINL bool full(int h, int c) const {
    return c <= full_to[h] && (c >= full_from[h] || c < full_sink);
  }
  // masked in part for a tile that reads it
  VA_DEVINL bool partial(int c) const {
    return (need(0, c) && !full(0, c)) || (need(1, c) && !full(1, c));
  }
};

VA_DEVINL bool not_finite(uint32_t h) { return (h & 0x7c00u) == 0x7c00u; }

// Whether every block with a key that the query at p sees is a block of the cache.
__noinline__ __device__ bool blocks_ok(const Args &a, const int32_t *bt, int p) {
  const int lo = win::run_start(p, a.window);
  for (int b = a.bs.div(lo); b <= a.bs.div(p); ++b) {
    const int32_t id = __ldg(bt + b);
    if (id < 0 || id >= a.num_blocks) return false;
  }
  const int ns = min(a.sinks, lo);
  for (int b = 0; b * (int64_t)a.bs.d < ns; ++b) {
    const int32_t id = __ldg(bt + b);
    if (id < 0 || id >= a.num_blocks) return false;
  }
  return true;
}

// Adds the values of V at (key tile c, columns col..col+31) that are not finite and
// belong to keys that the query at p sees (they are zeros in shared memory).
template <bool Q8>
__noinline__ __device__ void add_not_finite(const Args &a, const int32_t *bt, int kvh, int p, int c,
                                            int col, float *o) {
  for (int key = c * kKeys; key < (c + 1) * kKeys; ++key) {
    if (key > p || (a.window > 0 && key <= p - a.window && key >= a.sinks)) continue;
    const int32_t blk = __ldg(bt + a.bs.div(key));
    if (blk < 0 || blk >= a.num_blocks) continue;
    const int64_t row = blk * a.s_block + kvh * a.s_head + a.bs.mod(key) * a.s_token + col;
    for (int i = 0; i < 32; ++i) {
      if constexpr (Q8) {
        if ((a.vc[row + i] & 0x7f) == 0x7f) o[i] = NAN;
      } else {
        const __half v = reinterpret_cast<const __half *>(a.vc)[row + i];
        if (not_finite(__half_as_ushort(v))) o[i] += __half2float(v);
      }
    }
  }
}

template <int D, bool Q8, bool TMA>
__global__ void __launch_bounds__(Shape<D, Q8, TMA>::kThreads, 1)
    window_prefill_kernel(const __grid_constant__ Args a) {
  using S = Shape<D, Q8, TMA>;
  static_assert(!(Q8 && TMA), "e4m3 rows go through registers");
  constexpr int NB = S::NB, kSlots = S::kSlots, kProducers = S::kProducers;
  constexpr int kRegsSoftmax = S::kRegsSoftmax, kRegsOther = S::kRegsOther;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  // 128-byte swizzle atoms must sit on 1024-byte boundaries of the shared window
  unsigned char *smem = smem_raw + ((1024u - (va::smem_addr(smem_raw) & 1023u)) & 1023u);
  uint64_t *bar_full = reinterpret_cast<uint64_t *>(smem + S::oBar);  // [kSlots] tile landed
  uint64_t *bar_empty = bar_full + kSlots;   // [kSlots] MMAs that read the slot are done
  uint64_t *bar_scrub = bar_empty + kSlots;  // [kScrub] a V tile to scrub landed (TMA)
  uint64_t *bar_s = bar_scrub + (TMA ? kScrub : 0);  // [kTiles] S written
  uint64_t *bar_p = bar_s + kTiles;          // [kTiles] P published (one arrival per warp)
  uint64_t *bar_o = bar_p + kTiles;          // [kTiles] PV done
  uint64_t *bar_q = bar_o + kTiles;          // Q staged
  uint64_t *bar_end = bar_q + 1;             // every MMA retired
  int *state = reinterpret_cast<int *>(bar_end + 1);
  int &s_dead = state[0], &s_bad = state[1], &s_poison = state[2];
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(state + 3);

  va::pdl_enter();
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  // ---- the pair: pairs of sequence s start at index qsl[s] / TP + s (strictly
  // increasing, and far enough apart for ceil(len / TP) pairs), so a binary search finds
  // the sequence.  Last pairs first: the longest contexts of a prompt start first. ----
  const int TP = kTiles * a.TQ;
  const int kvh = blockIdx.x % a.Hkv;
  const int64_t unit = (gridDim.x - 1 - blockIdx.x) / a.Hkv;
  const int64_t first = __ldg(a.qsl);
  int s0 = 0, s1 = a.S - 1;
  while (s0 < s1) {
    const int mid = (s0 + s1 + 1) >> 1;
    const int64_t at = (__ldg(a.qsl + mid) - first) / TP + mid;
    if (at <= unit) s0 = mid;
    else s1 = mid - 1;
  }
  const int seq = s0;
  const int t_begin = __ldg(a.qsl + seq), t_end = __ldg(a.qsl + seq + 1);
  const int64_t local = unit - ((t_begin - first) / TP + seq);
  const int64_t t0l = t_begin + local * TP;
  if (local < 0 || t0l >= t_end) return;
  const int L = __ldg(a.sl + seq);
  if (t_begin < 0 || t_end > a.T || (L > 0 && a.bs.div(L - 1) >= a.max_blocks)) {
    if (tid == 0 && local == 0 && kvh == 0) va::raise_flag(a.err, VA_FLAG_CTX_OVERFLOW);
    return;
  }
  if (L <= 0) return;
  const int t0 = (int)t0l, nq = min(TP, t_end - t0);
  const int p0 = L - (t_end - t0);  // position of token t0 (may be negative: skipped)
  int pmin[kTiles], pmax[kTiles];  // query positions of each tile; pmax < 0: none
#pragma unroll
  for (int h = 0; h < kTiles; ++h) {
    const int n = min(a.TQ, nq - h * a.TQ);
    pmin[h] = max(p0 + h * a.TQ, 0);
    pmax[h] = n > 0 ? max(p0 + h * a.TQ + n - 1, -1) : -1;
  }
  const int plast = max(pmax[0], pmax[1]);
  if (plast < 0) return;
  const int pfirst = pmax[0] >= 0 ? pmin[0] : pmin[1];
  const Pair pr(pmin, pmax, a.window, a.sinks);
  const win::Tiles tl = win::key_tiles(pfirst, plast, a.window, a.sinks, kKeys);
  const int nch = tl.count;
  const int32_t *bt = a.bt + seq * a.max_blocks;

  if (tid == 0) {
    s_dead = s_bad = s_poison = 0;
    for (int i = 0; i < kSlots; ++i) {
      va::mbar_init(&bar_full[i], TMA ? 1 : kProducers / 32);
      va::mbar_init(&bar_empty[i], 1);
    }
    for (int i = 0; TMA && i < kScrub; ++i) va::mbar_init(&bar_scrub[i], 1);
    for (int h = 0; h < kTiles; ++h) {
      va::mbar_init(&bar_s[h], 1);
      va::mbar_init(&bar_p[h], kRows / 32);
      va::mbar_init(&bar_o[h], 1);
    }
    va::mbar_init(bar_q, kSoftmax / 32);
    va::mbar_init(bar_end, 1);
    va::fence_barrier_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(tmem_slot, tc::kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();

  auto dead = [&]() { return *(volatile int *)&s_dead != 0; };
  // Whole warps wait, and all lanes take one answer: what follows (a named barrier, TMEM
  // accesses, another wait) is the warp's.  The phase that a warp waits for cannot pass while
  // a lane has not seen it, since the next one needs that warp's own arrivals.  A wait that
  // runs out gives up for good, and so does one that runs long after another warp's has: every
  // wait ends, and those that need not wait do not look at s_dead.  (The lanes' own answers
  // let them run apart, and took 477 us for 8192 e4m3 tokens where this takes 440.)
  bool gone = *tmem_slot != 0;  // all 512 columns are this CTA's: its TMEM begins at column 0
  auto wait_bar = [&](uint64_t *bar, uint32_t parity) {
    bool ok = __all_sync(0xffffffffu, gone || va::mbar_try_wait(bar, parity));
    for (uint32_t i = 1; !ok && i < kWaitLimit; ++i) {
      ok = __all_sync(0xffffffffu, va::mbar_try_wait(bar, parity));
      if ((i & 255) == 0 && __any_sync(0xffffffffu, dead())) break;
    }
    if (!ok) {
      gone = true;
      if (atomicExch(&s_dead, 1) == 0) va::raise_flag(a.err, VA_FLAG_WAIT_TIMEOUT);
    }
  };

  // A barrier counts warps: each thread's part is done, one lane arrives.
  auto warp_arrive = [&](uint64_t *bar) {
    __syncwarp();
    if ((tid & 31) == 0) va::mbar_arrive(bar);
  };
  const int klo = win::run_start(pfirst, a.window);
  // whether some row of the pair sees the key (a sink that only a later row's window has
  // passed is inside the run [klo, plast])
  auto seen = [&](int key) { return key <= plast && (key >= klo || key < a.sinks); };
  auto slot_of = [&](int item) { return smem + S::oSlot + (item % kSlots) * S::kTileBytes; };
  // whether the MMAs that read the item's slot before are done (without waiting; the warp's
  // answer, as above), and a wait
  auto is_empty = [&](int item) {
    uint64_t *bar = &bar_empty[item % kSlots];
    return item < kSlots ||
           __all_sync(0xffffffffu, gone || va::mbar_try_wait(bar, ((item / kSlots) - 1) & 1));
  };
  auto wait_empty = [&](int item) {
    if (item >= kSlots) wait_bar(&bar_empty[item % kSlots], ((item / kSlots) - 1) & 1);
  };

  if (tid >= kFirstProducer) {
    // =================== producers ===================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    const int pt = tid - kFirstProducer, kr = pt & (kKeys - 1);  // kr: its key row
    // element offset of each row of the key tile in the cache, | 1; 0: zeros
    int64_t *info = reinterpret_cast<int64_t *>(smem + S::oInfo);
    auto producer_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(kProducers) : "memory"); };
    const int64_t head_off = kvh * a.s_head;
    // block of key row kr of key tile j (-1: zeros)
    auto block_of = [&](int j) -> int32_t {
      if (j >= nch) return -1;
      const int key = win::tile_at(tl, j) * kKeys + kr;
      if (!seen(key)) return -1;
      const int32_t b = __ldg(bt + a.bs.div(key));
      if (b < 0 || b >= a.num_blocks) {
        va::raise_flag(a.err, VA_FLAG_BAD_BLOCK);
        *(volatile int *)&s_bad = 1;
        return -1;
      }
      return b;
    };
    auto off_of = [&](int j) { return a.bs.mod(win::tile_at(tl, j) * kKeys + kr); };
    // (offsets are multiples of 8)
    auto row_of = [&](int32_t blk, int j) {
      return blk >= 0 ? (blk * a.s_block + head_off + off_of(j) * a.s_token) | 1 : int64_t(0);
    };
    auto publish = [&](int item) {  // this thread's stores to the item's slot are visible
      va::fence_proxy_async_smem();
      warp_arrive(&bar_full[item % kSlots]);
    };

    if constexpr (!Q8) {
      constexpr int P = D / 8;  // 16-byte pieces per row; each thread copies P of a tile
      // piece k of this thread: row, column and place in a slot; rows a multiple of 8 apart
      // unless P = 12, so that the places are one base and a constant
      auto piece_row = [&](int k) {
        return P == 12 ? (pt + k * kProducers) / 12 : pt / P + k * (kProducers / P);
      };
      auto piece_col = [&](int k) { return P == 12 ? (pt + k * kProducers) % 12 : pt % P; };
      const uint32_t place0 = tc::sw128_off(pt / P, pt % P * 8, kKeys);
      auto place = [&](int k) {
        return P == 12 ? tc::sw128_off(piece_row(k), piece_col(k) * 8, kKeys)
                       : place0 + k * (kProducers / P) * 128;
      };
      // V of a partly masked tile: no infinity or NaN stays
      auto scrub = [&](int item) {
        unsigned char *sl = slot_of(item);
        const int key0 = win::tile_at(tl, item >> 1) * kKeys;
        bool hit = false;
#pragma unroll 4
        for (int k = 0; k < P; ++k) {
          uint4 *w = reinterpret_cast<uint4 *>(sl + place(k));
          uint32_t x[4] = {w->x, w->y, w->z, w->w};
          uint32_t h = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bad = __vcmpgeu2(x[i] & 0x7fff7fffu, 0x7c007c00u);
            h |= bad;
            x[i] &= ~bad;
          }
          if (h) {
            *w = make_uint4(x[0], x[1], x[2], x[3]);
            hit = hit || seen(key0 + piece_row(k));
          }
        }
        if (hit) *(volatile int *)&s_poison = 1;
      };
      if constexpr (TMA) {
        int n = 0;
#pragma unroll 1
        for (int j = 0; j < nch; ++j) {
          if (!pr.partial(win::tile_at(tl, j))) continue;
          wait_bar(&bar_scrub[n % kScrub], (n / kScrub) & 1);
          scrub(2 * j + 1);
          va::fence_proxy_async_smem();
          producer_sync();
          if (pt == 0) va::mbar_arrive(&bar_full[(2 * j + 1) % kSlots]);
          ++n;
        }
      } else {
        int32_t blk = block_of(0);
        // an item's copies have landed -> scrub, publish
        auto finish = [&](int item) {
          if ((item & 1) && pr.partial(win::tile_at(tl, item >> 1))) scrub(item);
          publish(item);
        };
        int done = 0;  // items published
        // Copies the item into its slot.  At most kLag items stay unpublished behind the newest
        // one, and none while this thread waits for a slot.
        auto copy = [&](int item) {
          if (!is_empty(item)) {
            if (item - done == 2) {
              win::cp_async_wait<1>();
              finish(done++);
            }
            if (item - done == 1) {
              win::cp_async_wait<0>();
              finish(done++);
            }
            wait_empty(item);
          }
          const __half *src = reinterpret_cast<const __half *>(item & 1 ? a.vc : a.kc);
          const uint32_t sl = va::smem_addr(slot_of(item));
#pragma unroll P == 12 ? 4 : P
          for (int k = 0; k < P; ++k) {
            const int64_t e = info[piece_row(k)];
            win::cp_async_zfill<16>(sl + place(k), src + (e & ~int64_t(7)) + piece_col(k) * 8, e & 1);
          }
          win::cp_async_commit();
          if (item - done == kLag) {
            win::cp_async_wait<kLag>();
            finish(done++);
          }
        };
#pragma unroll 1
        for (int j = 0; j < nch; ++j) {
          producer_sync();  // everyone is done with the rows of the tile before
          info[pt] = row_of(blk, j);
          producer_sync();
          blk = block_of(j + 1);
          copy(2 * j);
          copy(2 * j + 1);
        }
        win::cp_async_wait<0>();
        while (done < 2 * nch) finish(done++);
      }
    } else {
      // The codes of an item come by cp.async into one of two raw buffers, two items ahead;
      // each thread turns the pieces it copied itself into fp16 in the item's slot.
      constexpr int P = D / 16, N = P * kKeys / kProducers;  // 16-code pieces of a row, of a thread
      // Piece k of this thread: row and column; rows a multiple of 8 apart unless P = 6, so
      // that every address below is one base and a constant.  With P = 8 eight lanes take
      // half of a row and the other half of the next: their codes lie in all banks, and so do
      // their chunks 2c (and 2c + 1) in the swizzled slot, where the two halves of one row
      // would share banks (546 -> 525 us for 8192 tokens under a window of 4096).
      const int row0 = P == 8 ? (pt >> 4) * 2 + (pt >> 2 & 1) : pt / P;
      const int col0 = P == 8 ? ((pt >> 1 ^ pt) & 4) + (pt & 3) : pt % P;
      auto piece_row = [&](int k) {
        return P == 6 ? (pt + k * kProducers) / 6 : row0 + k * (kProducers / P);
      };
      auto piece_col = [&](int k) { return P == 6 ? (pt + k * kProducers) % 6 : col0; };
      unsigned char *raw = smem + S::oRaw + row0 * D + col0 * 16;  // + k * kProducers * 16
      __half *scale_k = reinterpret_cast<__half *>(smem + S::oExp), *scale_v = scale_k + kKeys;
      const bool is_k = pt < kKeys;  // whose exponents this thread brings
      int32_t blk0 = block_of(0), blk1 = block_of(1);
      auto load_exp = [&](int32_t blk, int j) -> uint32_t {
        if (blk < 0) return va::kQ8ExpBias;
        return __ldg((is_k ? a.ks : a.vs) + blk * a.c_block + kvh * a.c_head + off_of(j) * a.c_token);
      };
      uint32_t e0 = load_exp(blk0, 0);
      // rows of key tile j and their scales for everyone; the next tile's exponents and block
      // are on their way
      auto announce = [&](int j) {
        producer_sync();  // K(j-1) is converted, V(j-1) on its way
        if (is_k) info[kr] = row_of(blk0, j);
        (is_k ? scale_k : scale_v + (j & 1) * kKeys)[kr] =
            __ushort_as_half((unsigned short)va::q8_scale_h2(e0));
        producer_sync();
        blk0 = blk1;
        if (j + 1 < nch) e0 = load_exp(blk0, j + 1);
        blk1 = block_of(j + 2);
      };
      auto fetch = [&](int item) {
        const uint8_t *src = item & 1 ? a.vc : a.kc;
        const uint32_t to = va::smem_addr(raw + (item & 1) * S::kRawBytes);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int64_t e = info[piece_row(k)];
          win::cp_async_zfill<16>(to + k * kProducers * 16, src + (e & ~int64_t(15)) + piece_col(k) * 16,
                                  e & 1);
        }
        win::cp_async_commit();
      };
      auto convert = [&](int item) {
        const unsigned char *from = raw + (item & 1) * S::kRawBytes;
        unsigned char *sl = slot_of(item);
        const __half *scale = item & 1 ? scale_v + (item >> 1 & 1) * kKeys : scale_k;
        const int c = win::tile_at(tl, item >> 1);
        const bool scrub = (item & 1) && pr.partial(c);
        uint32_t hit = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const uint4 r = *reinterpret_cast<const uint4 *>(from + k * kProducers * 16);
          const uint32_t f = (uint32_t)__half_as_ushort(scale[piece_row(k)]) * 0x10001u;
          uint32_t w[4] = {r.x, r.y, r.z, r.w}, o[8];
          if (scrub) {
            uint32_t any = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t bad = __vcmpeq4(w[x] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              any |= bad;
              w[x] &= ~bad;
            }
            if (any && seen(c * kKeys + piece_row(k))) hit = 1;
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            va::q8_decode4(w[x], o[2 * x], o[2 * x + 1]);
            o[2 * x] = va::hmul2(o[2 * x], f);
            o[2 * x + 1] = va::hmul2(o[2 * x + 1], f);
          }
          // 16-byte chunks 2c, 2c + 1 of the row; the first one's place differs by bit 4
          const uint32_t to = P == 6 ? tc::sw128_off(piece_row(k), piece_col(k) * 16, kKeys)
                                     : tc::sw128_off(row0, col0 * 16, kKeys) +
                                           k * (kProducers / P) * 128;
          *reinterpret_cast<uint4 *>(sl + to) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4 *>(sl + (to ^ 16)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        if (hit) *(volatile int *)&s_poison = 1;
        publish(item);
      };
      announce(0);
      fetch(0);
      fetch(1);
#pragma unroll 1
      for (int item = 0; item < 2 * nch; ++item) {
        win::cp_async_wait<1>();
        wait_empty(item);
        convert(item);
        if (item + 2 < 2 * nch) {
          if ((item & 1) == 0) announce((item >> 1) + 1);
          fetch(item + 2);
        } else {
          win::cp_async_commit();  // keeps the count of groups
        }
      }
    }
  } else if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kMmaWarp) {
      // =================== MMA issue ===================
      // The whole warp walks the loop, so that the descriptors are uniform values; the one
      // elected lane issues.
      const uint32_t one = elect_one();
      const uint32_t sQ = va::smem_addr(smem);
      constexpr uint32_t IDESC_S = tc::idesc_f16(kRows, kKeys, false);
      constexpr uint32_t IDESC_O = tc::idesc_f16(kRows, NB * 64, true);
      // descriptors differ in their address field (16-byte units) alone
      const uint64_t dQK = tc::sdesc(sQ, 16, 1024);                   // K-major
      const uint64_t dV = tc::sdesc(sQ + S::oSlot, kKeys * 128, 1024);  // MN-major: LBO = next
                                                                      // 64 columns, SBO = 8 keys
      constexpr uint32_t kTile16 = S::kTileBytes / 16, kSlot16 = S::oSlot / 16;
      int np[kTiles] = {0, 0};  // PVs issued per tile
      int sk = 0, sv = kSlots - 1;  // slots of K(j) and V(j-1): items 2j and 2j - 1
      uint32_t fk = 0, fv = 1;      // phases of their "full" barriers
      // O_h (+)= P_h V: A = P_h [128 x 128] from TMEM, B = V [128 keys x NB*64]
      auto issue_pv = [&](int h) {
        wait_bar(&bar_p[h], np[h] & 1);
        tc::fence_after_sync();
        const uint32_t go = gone ? 0 : one, acc = np[h] > 0;
        const uint64_t v = dV + sv * kTile16;
#pragma unroll
        for (int ks = 0; ks < kKeys / 16; ++ks)
          umma_ts(kTmemO + h * NB * 64, h * 128 + ks * 8, v + ks * 128, IDESC_O, ks ? 1u : acc, go);
        umma_commit(&bar_o[h], go);
        ++np[h];
      };
      // S_h = Q_h K^T.  It overwrites P_h, read by the PV before it: one thread's
      // tcgen05.mma run in issue order.
      auto issue_s = [&](int h) {
        const uint32_t go = gone ? 0 : one;
        const uint64_t q = dQK + h * kTile16, k = dQK + kSlot16 + sk * kTile16;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          constexpr uint32_t kBlock16 = 128 * 128 / 16;
          const uint32_t o = (ks >> 2) * kBlock16 + (ks & 3) * 2;
          umma_ss(h * 128, q + o, k + o, IDESC_S, ks > 0, go);
        }
        umma_commit(&bar_s[h], go);
      };
      wait_bar(bar_q, 0);
      wait_bar(&bar_full[0], 0);
      tc::fence_after_sync();
      bool pv0 = pr.need(0, win::tile_at(tl, 0)), pv1 = pr.need(1, win::tile_at(tl, 0));
      if (pv0) issue_s(0);
      if (pv1) issue_s(1);
      umma_commit(&bar_empty[0], gone ? 0 : one);
#pragma unroll 1
      for (int j = 1; j <= nch; ++j) {
        // items advance by two
        sk += 2;
        sv += 2;
        if (sk >= kSlots) { sk -= kSlots; fk ^= 1; }
        if (sv >= kSlots) { sv -= kSlots; fv ^= 1; }
        const int c = win::tile_at(tl, j);
        const bool s0 = j < nch && pr.need(0, c), s1 = j < nch && pr.need(1, c);
        wait_bar(&bar_full[sv], fv);
        if (pv0) issue_pv(0);
        if (j < nch) {
          wait_bar(&bar_full[sk], fk);
          tc::fence_after_sync();
        }
        if (s0) issue_s(0);
        if (pv1) issue_pv(1);
        umma_commit(&bar_empty[sv], gone ? 0 : one);
        if (s1) issue_s(1);
        if (j < nch) umma_commit(&bar_empty[sk], gone ? 0 : one);
        pv0 = s0;
        pv1 = s1;
      }
      // every MMA issued above has retired before TMEM is freed
      umma_commit(bar_end, one);
      if (!va::mbar_wait_bounded(bar_end, 0, kWaitLimit) && atomicExch(&s_dead, 1) == 0)
        va::raise_flag(a.err, VA_FLAG_WAIT_TIMEOUT);
      __syncwarp();
    } else if (TMA && warp == kLoadWarp) {
      // =================== TMA: one copy per block of a key tile ===================
      const int lane = tid & 31;
      const int rows = min((int)a.bs.d, kKeys), copies = kKeys / rows;  // lanes 0 .. copies - 1 copy
      // block of the lane's copy for key tile j; num_blocks, past the tensor, gives zeros
      auto block_of = [&](int j) -> int32_t {
        const int key = win::tile_at(tl, j) * kKeys + lane * rows;
        // some row sees one of its keys
        if (lane >= copies || key > plast || (key + rows <= klo && key >= a.sinks))
          return (int32_t)a.num_blocks;
        const int32_t b = __ldg(bt + a.bs.div(key));
        if (b >= 0 && b < a.num_blocks) return b;
        va::raise_flag(a.err, VA_FLAG_BAD_BLOCK);
        *(volatile int *)&s_bad = 1;
        return (int32_t)a.num_blocks;
      };
      int items = 0, n = 0;  // issued; those that wait to be scrubbed
      int32_t next = block_of(0);
#pragma unroll 1
      for (int j = 0; j < nch; ++j) {
        const int c = win::tile_at(tl, j);
        const int32_t blk = next;
        const int off = a.bs.mod(c * kKeys + lane * rows);  // token of the block
        if (j + 1 < nch) next = block_of(j + 1);
        const bool part = pr.partial(c);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int item = 2 * j + v;
          wait_empty(item);
          if (gone) continue;
          uint64_t *bar = v && part ? &bar_scrub[n++ % kScrub] : &bar_full[item % kSlots];
          if (lane == 0) va::mbar_arrive_expect_tx(bar, S::kTileBytes);
          __syncwarp();
          if (lane < copies) {
            unsigned char *to = slot_of(item) + lane * rows * 128;
#pragma unroll
            for (int b = 0; b < NB; ++b)
              tma_load_4d(to + b * (kKeys * 128), v ? &a.mv : &a.mk, b * 64, off, kvh, blk, bar);
          }
          items = item + 1;
        }
      }
      // After a time-out nobody else may wait for the copies in flight: they land (within a
      // bounded wait) before the CTA's shared memory is given back.
      if (gone || dead()) {
        bool landed = true;
        auto land = [&](uint64_t *bar, uint32_t parity) {
          landed = va::mbar_wait_bounded(bar, parity, kWaitLimit) && landed;
        };
        for (int i = 0, m = 0; i < items; ++i) {
          if ((i & 1) && pr.partial(win::tile_at(tl, i >> 1))) {
            if (m >= n - kScrub) land(&bar_scrub[m % kScrub], (m / kScrub) & 1);
            ++m;
          } else if (i >= items - kSlots) {
            land(&bar_full[i % kSlots], (i / kSlots) & 1);
          }
        }
        if (!landed) va::raise_flag(a.err, VA_FLAG_WAIT_TIMEOUT);
      }
    }
  } else {
    // =================== Q, then softmax of tile h, one thread per row ===================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int h = warp >> 2, row = tid & (kRows - 1);
    const int head0 = kvh * a.G;
    {
      constexpr int P = D / 8;
#pragma unroll 4
      for (int i = tid; i < kTiles * kRows * P; i += kSoftmax) {
        const int r2 = i / P, c = i - r2 * P, hh = r2 / kRows, r = r2 - hh * kRows;
        const int tk = a.g.div(r), g = r - tk * a.G, ti = hh * a.TQ + tk;
        const bool on = tk < a.TQ && ti < nq;
        win::cp_async_zfill<16>(
            va::smem_addr(smem + hh * S::kTileBytes + tc::sw128_off(r, c * 8, kRows)),
            a.q + (on ? (t0 + ti) * a.q_s_token + (int64_t)(head0 + g) * a.q_s_head + c * 8 : 0),
            on);
      }
      win::cp_async_commit();
      win::cp_async_wait<0>();
      va::fence_proxy_async_smem();
      warp_arrive(bar_q);
    }
    const int tk = a.g.div(row), g = row - tk * a.G, ti = h * a.TQ + tk;
    const bool row_ok = tk < a.TQ && ti < nq && p0 + ti >= 0;
    // rows of no token take the tile's last position: their result is dropped
    const int pos = row_ok ? p0 + ti : (h ? pmax[1] : pmax[0]);
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = h * 128 + lane_base;
    const uint32_t tO = kTmemO + h * NB * 64 + lane_base;
    const float sc = a.scale_log2;
    float m = -INFINITY, l = 0.f;
    int n = 0;  // key tiles of this tile so far
#pragma unroll 1
    for (int j = 0; j < nch; ++j) {
      const int c = win::tile_at(tl, j);
      if (!(h ? pr.need(1, c) : pr.need(0, c))) continue;
      // columns [vlo, vhi] and [0, vsk) of the key tile are visible
      const bool masked = !(h ? pr.full(1, c) : pr.full(0, c));
      const int vhi = pos - c * kKeys;
      const int vlo = a.window > 0 ? pos - a.window + 1 - c * kKeys : 0;
      const int vsk = a.sinks - c * kKeys;
      wait_bar(&bar_s[h], n & 1);
      tc::fence_after_sync();
      float p[kKeys];
      {
        uint32_t x[4][32];
#pragma unroll
        for (int k = 0; k < 4; ++k) tc::tmem_ld32(tS + k * 32, x[k]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < kKeys; ++i) p[i] = __uint_as_float(x[i >> 5][i & 31]);
      }
      if (masked) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // bits [vlo, vhi] and [0, vsk) of columns 32k .. 32k + 31
          auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };
          const uint32_t see =
              below(vhi + 1 - 32 * k) & (~below(vlo - 32 * k) | below(vsk - 32 * k));
#pragma unroll
          for (int i = 0; i < 32; ++i) p[32 * k + i] = see >> i & 1 ? p[32 * k + i] : -INFINITY;
        }
      }
      float mx[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
      for (int i = 4; i < kKeys - 4; i += 8) {
        mx[0] = tc::fmax3(mx[0], p[i], p[i + 1]);
        mx[1] = tc::fmax3(mx[1], p[i + 2], p[i + 3]);
        mx[2] = tc::fmax3(mx[2], p[i + 4], p[i + 5]);
        mx[3] = tc::fmax3(mx[3], p[i + 6], p[i + 7]);
      }
      mx[0] = tc::fmax3(mx[0], p[kKeys - 4], p[kKeys - 3]);
      mx[1] = tc::fmax3(mx[1], p[kKeys - 2], p[kKeys - 1]);
      float rmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      rmax *= sc;  // the scale is positive
      const float mn = (m == -INFINITY || rmax > m + 12.f) ? fmaxf(m, rmax) : m;
      const bool none = mn == -INFINITY;  // no visible key so far
      const float alpha = (none || mn == m) ? 1.f : va::fast_exp2(m - mn);
      const float nm = none ? 0.f : -mn;
      m = mn;
      if (n > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        // the warp's rows of O are rescaled once the PV before has left them
        wait_bar(&bar_o[h], (n - 1) & 1);
        tc::fence_after_sync();
#pragma unroll 1
        for (int k = 0; k < NB * 64; k += 32) {
          uint32_t o[32];
          tc::tmem_ld32(tO + k, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tc::tmem_st32(tO + k, o);
        }
        tc::tmem_wait_st();
      }
      const uint64_t sc2 = tc::pk2(sc, sc), nm2 = tc::pk2(nm, nm);
      uint64_t sum2[2] = {tc::pk2(0.f, 0.f), tc::pk2(0.f, 0.f)};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int k = half * 64 + 2 * i;
          float x0, x1;
          tc::upk2(tc::ffma2(tc::pk2(p[k], p[k + 1]), sc2, nm2), x0, x1);
          x0 = va::fast_exp2(x0);
          x1 = va::fast_exp2(x1);
          sum2[i & 1] = tc::fadd2(sum2[i & 1], tc::pk2(x0, x1));
          w[i] = va::pack_h2(x0, x1);
        }
        tc::tmem_st32(tS + half * 32, w);  // over S, which is in registers
      }
      float y0, y1, y2, y3;
      tc::upk2(sum2[0], y0, y1);
      tc::upk2(sum2[1], y2, y3);
      l = l * alpha + ((y0 + y1) + (y2 + y3));
      tc::tmem_wait_st();
      tc::fence_before_sync();
      warp_arrive(&bar_p[h]);
      ++n;
    }
    if (n > 0) {
      wait_bar(&bar_o[h], (n - 1) & 1);
      tc::fence_after_sync();
      const bool poison = *(volatile int *)&s_poison != 0;  // some V value was scrubbed
      bool write = row_ok && !gone && !dead();
      if (*(volatile int *)&s_bad != 0) write = write && blocks_ok(a, bt, pos);
      const float inv = 1.f / l;
      __half *orow = a.out + (t0 + ti) * a.o_s_token + (int64_t)(head0 + g) * a.o_s_head;
#pragma unroll 1
      for (int k = 0; k < D; k += 32) {
        uint32_t x[32];
        tc::tmem_ld32(tO + k, x);
        tc::tmem_wait_ld();
        if (write) {
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(x[i]) * inv;
          if (poison) {
            float fix[32];
            for (int i = 0; i < 32; ++i) fix[i] = 0.f;
            for (int j = 0; j < nch; ++j) {
              const int c = win::tile_at(tl, j);
              if (pr.partial(c)) add_not_finite<Q8>(a, bt, kvh, pos, c, k, fix);
            }
            for (int i = 0; i < 32; ++i) o[i] += fix[i];
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            *reinterpret_cast<uint4 *>(orow + k + i) =
                make_uint4(va::pack_h2(o[i], o[i + 1]), va::pack_h2(o[i + 2], o[i + 3]),
                           va::pack_h2(o[i + 4], o[i + 5]), va::pack_h2(o[i + 6], o[i + 7]));
        }
        __syncwarp();  // the next load from TMEM is a whole warp's
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(*tmem_slot, tc::kTmemCols);
  }
}

template <int D, bool Q8, bool TMA>
int launch_t(const Args &a, unsigned grid, cudaStream_t st) {
  using S = Shape<D, Q8, TMA>;
  constexpr auto kernel = window_prefill_kernel<D, Q8, TMA>;
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> regs{0};
  if (!win::allow_smem(kernel, (int)S::kBytes, done)) return VA_ERR_LAUNCH;
  // the register shares only add up when the build gave every thread kRegsLaunch: with fewer
  // the softmax warps would wait for registers for good
  int r = regs.load(std::memory_order_relaxed);
  if (!r) {
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, kernel) != cudaSuccess) return VA_ERR_LAUNCH;
    regs.store(r = at.numRegs, std::memory_order_relaxed);
  }
  if (r != S::kRegsLaunch) return VA_ERR_LAUNCH;
  if (va_host::launch_pdl_smem(kernel, grid, S::kThreads, S::kBytes, st, a)) return VA_ERR_LAUNCH;
  return va_host::launch_status();
}

using Encode = PFN_cuTensorMapEncodeTiled_v12000;
Encode encoder() {
  static const Encode fn = [] {
    cudaDriverEntryPointQueryResult q;
    void *f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  return fn;
}

// Tensor maps over (head dim, token of the block, kv head, block) of the fp16 caches: a box is
// 64 columns of one block of one head, or of 128 tokens of a longer block, and lands in the
// tensor core's 128-byte swizzle (columns past the head size are zeros).  Blocks that do not
// tile 128 keys in pieces of at least 8 rows (one swizzle atom), and layouts that the encoder
// does not take, leave the copies to cp.async.
bool encode_maps(Args &a, int D) {
  const int bs = (int)a.bs.d, rows = bs < kKeys ? bs : kKeys;
  if (bs < 8 || (bs < kKeys ? kKeys % bs : bs % kKeys) || a.num_blocks == 0 ||
      a.num_blocks >= INT32_MAX)
    return false;
  const Encode enc = encoder();
  if (!enc) return false;
  const int64_t extent[3] = {bs, a.Hkv, a.num_blocks}, stride[3] = {a.s_token, a.s_head, a.s_block};
  cuuint64_t dims[4] = {(cuuint64_t)D}, strides[3];
  for (int i = 0; i < 3; ++i) {
    if (extent[i] > 1 && (stride[i] <= 0 || stride[i] >= int64_t(1) << 38)) return false;
    dims[i + 1] = (cuuint64_t)extent[i];
    strides[i] = (cuuint64_t)(extent[i] > 1 ? stride[i] : D) * 2;  // of one element: never used
  }
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, one[4] = {1, 1, 1, 1};
  for (int v = 0; v < 2; ++v)
    if (enc(v ? &a.mv : &a.mk, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<uint8_t *>(v ? a.vc : a.kc), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            D > 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  return true;
}

template <int D>
int launch_d(Args &a, bool q8, unsigned grid, cudaStream_t st) {
  if (q8) return launch_t<D, true, false>(a, grid, st);
  return encode_maps(a, D) ? launch_t<D, false, true>(a, grid, st)
                           : launch_t<D, false, false>(a, grid, st);
}

}  // namespace

extern "C" int va_window_prefill(void *out, const void *q, const void *k_cache,
                                 const void *v_cache, const void *k_scale, const void *v_scale,
                                 int kv_e4m3, const int32_t *block_table,
                                 const int32_t *query_start_loc, const int32_t *seq_lens,
                                 int64_t num_tokens, int64_t num_seqs, int num_query_heads,
                                 int num_kv_heads, int head_size, int block_size,
                                 int64_t max_blocks_per_seq, int64_t num_blocks, float scale,
                                 int window, int sink_tokens, int64_t s_block, int64_t s_head,
                                 int64_t s_token, int64_t sc_block, int64_t sc_head,
                                 int64_t sc_token, int64_t q_s_token, int64_t q_s_head,
                                 int64_t o_s_token, int64_t o_s_head, int32_t *err_flag,
                                 void *stream) {
  if (num_tokens < 0 || num_seqs < 0 || num_blocks < 0 || max_blocks_per_seq < 0 ||
      sink_tokens < 0 || !win::scale_ok(scale))
    return VA_ERR_INVALID_ARG;
  if (num_kv_heads <= 0 || num_query_heads <= 0 || num_query_heads % num_kv_heads ||
      block_size <= 0)
    return VA_ERR_INVALID_ARG;
  if (num_tokens == 0 || num_seqs == 0) return VA_OK;
  if (!out || !q || !k_cache || !v_cache || !block_table || !query_start_loc || !seq_lens ||
      (kv_e4m3 && (!k_scale || !v_scale)))
    return VA_ERR_INVALID_ARG;
  const int G = num_query_heads / num_kv_heads;
  if (!win::head_size_ok(head_size) || G > kRows) return VA_ERR_UNSUPPORTED;
  // positions and token indexes are 32-bit on the device, with room for a tile
  if (num_tokens > INT32_MAX / 2 || num_seqs > INT32_MAX / 2 ||
      max_blocks_per_seq > (INT32_MAX / 2) / block_size)
    return VA_ERR_UNSUPPORTED;
  if (!va_host::aligned16(k_cache) || !va_host::aligned16(v_cache) ||
      !win::strides_ok(kv_e4m3, s_block, s_head, s_token) ||
      !win::rows_ok(q, q_s_token, q_s_head) || !win::rows_ok(out, o_s_token, o_s_head))
    return VA_ERR_INVALID_ARG;
  Args a{};
  a.out = static_cast<__half *>(out);
  a.q = static_cast<const __half *>(q);
  a.kc = static_cast<const uint8_t *>(k_cache);
  a.vc = static_cast<const uint8_t *>(v_cache);
  a.ks = static_cast<const uint8_t *>(k_scale);
  a.vs = static_cast<const uint8_t *>(v_scale);
  a.bt = block_table;
  a.qsl = query_start_loc;
  a.sl = seq_lens;
  a.err = err_flag;
  a.T = num_tokens;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = num_blocks;
  a.S = (int)num_seqs;
  a.Hkv = num_kv_heads;
  a.G = G;
  a.g = win::fast_div(G);
  a.TQ = kRows / G;
  a.bs = win::fast_div(block_size);
  a.window = win::window_of(window);
  a.sinks = win::sinks_of(sink_tokens);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.s_block = s_block; a.s_head = s_head; a.s_token = s_token;
  a.c_block = sc_block; a.c_head = sc_head; a.c_token = sc_token;
  a.q_s_token = q_s_token; a.q_s_head = q_s_head;
  a.o_s_token = o_s_token; a.o_s_head = o_s_head;
  // pairs of sequence s start at index qsl[s] / TP + s: at most this many in all
  const int64_t pairs = num_tokens / (kTiles * a.TQ) + num_seqs;
  if (pairs * num_kv_heads > INT32_MAX) return VA_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)(pairs * num_kv_heads);
  auto st = static_cast<cudaStream_t>(stream);
  const bool q8 = kv_e4m3 != 0;
  switch (head_size) {
    case 32: return launch_d<32>(a, q8, grid, st);
    case 64: return launch_d<64>(a, q8, grid, st);
    case 96: return launch_d<96>(a, q8, grid, st);
    case 128: return launch_d<128>(a, q8, grid, st);
  }
  return VA_ERR_UNSUPPORTED;
}

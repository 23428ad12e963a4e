// Attention of chunks of new tokens over a paged cache under a sliding window with sinks
// (visibility rule: window.cuh), fp16 or e4m3 cache (row format: kv_q8.cuh), on the
// 5th-generation tensor cores.
//
// One CTA takes a pair of 128-row tiles of one sequence and one kv head.  A row is a
// (token, query head of the group) pair, so every staged key serves all heads of the
// group and both tiles; the tiles' keys are the pair's key tiles of 128 (window.cuh), and
// nothing outside the window and the sinks is read or multiplied.
//   * warps 0-7: softmax, one thread per row (TMEM lane = row), warps 0-3 tile 0 and 4-7
//     tile 1.  S comes from TMEM twice, 64 columns at a time (the row maximum, then the
//     powers), so a row's 128 scores never sit in registers at once.  P goes back over S
//     as fp16 and feeds the second product from TMEM.  The maximum a row's powers are
//     taken against only moves when it grows by more than 2^8, so O is rarely rescaled.
//   * warp 8: issues tcgen05.mma for both tiles in turn -- PV_0(j-1), S_0(j), PV_1(j-1),
//     S_1(j) -- so one tile's products run while the other tile is in its softmax.
//   * warps 9-12: bring K and V key tiles into a ring of shared-memory slots in the
//     128-byte-swizzled layout of the tensor core.  fp16 rows go by 16-byte cp.async; e4m3
//     rows are loaded one key tile ahead into registers, turned into fp16 (exactly) and
//     stored.  Row addresses come from the block table once per key tile, so any block
//     size and any strides work; keys that no row of the pair sees are zeros, unread.
// A key masked for one row but seen by another may hold an infinity or a NaN in V, and
// 0 * inf would reach the masked row.  In key tiles that are masked in part (at most a
// few per pair) the producers replace such values by 0, and rows that do see them get
// them added at the end.
// Scores, statistics and O are fp32; P is rounded to fp16.
// Bounded waits: after a time-out every role runs its loop to the end without waiting or
// issuing (so the roles still meet at their barriers), nothing is written and
// VA_FLAG_WAIT_TIMEOUT is set.
#include <limits.h>

#include "prefill_tc.cuh"
#include "window.cuh"

namespace {

constexpr int kRows = 128, kKeys = 128, kTiles = 2;
constexpr int kSoftmax = kTiles * kRows;
constexpr int kMmaWarp = kSoftmax / 32;
constexpr int kProducers = 128;
constexpr int kThreads = kSoftmax + 32 + kProducers;
constexpr int kLag = 2;  // fp16 copies in flight behind the newest
constexpr uint32_t kWaitLimit = 1u << 22;

template <int D>
struct Shape {
  static constexpr int NB = (D + 63) / 64;            // 64-column blocks of a row
  static constexpr uint32_t kTileBytes = NB * 128 * 128;
  static constexpr int kSlots = NB == 2 ? 5 : 8;      // K/V key tiles in flight
  static constexpr uint32_t oSlot = kTiles * kTileBytes;
  static constexpr uint32_t oInfo = oSlot + kSlots * kTileBytes;  // int2 [128] {block, offset}
  static constexpr uint32_t oExp = oInfo + 128 * 8;   // uchar2 [2][128] exponents of K, V
  static constexpr uint32_t oBar = oExp + 2 * 128 * 2;
  static constexpr uint32_t kBytes = oBar + 256 + 1024;  // + alignment slack
};

struct Args {
  __half *out;
  const __half *q;
  const uint8_t *kc, *vc, *ks, *vs;
  const int32_t *bt, *qsl, *sl;
  int32_t *err;
  int64_t T, max_blocks, num_blocks;
  int S, Hkv, G, TQ, bs, window, sinks;
  float scale_log2;
  int64_t s_block, s_head, s_token, c_block, c_head, c_token;
  int64_t q_s_token, q_s_head, o_s_token, o_s_head;
};

VA_DEVINL void producer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kProducers) : "memory"); }

// What a pair of tiles reads.
struct Pair {
  int pmin[kTiles], pmax[kTiles];  // query positions of each tile; pmax < pmin: empty
  int window, sinks;
  // key tile c holds a key that some row of tile h sees
  VA_DEVINL bool need(int h, int c) const {
    return c * kKeys <= pmax[h] &&
           ((c + 1) * kKeys > win::run_start(pmin[h], window) || c * kKeys < sinks);
  }
  // every row of tile h sees every key of c
  VA_DEVINL bool full(int h, int c) const {
    return (c + 1) * kKeys - 1 <= pmin[h] &&
           (window <= 0 || c * kKeys > pmax[h] - window || (c + 1) * kKeys <= sinks);
  }
  // masked in part for a tile that reads it
  VA_DEVINL bool partial(int c) const {
    return (need(0, c) && !full(0, c)) || (need(1, c) && !full(1, c));
  }
  VA_DEVINL bool sees(int p, int key) const {
    return key <= p && (window <= 0 || key > p - window || key < sinks);
  }
};

VA_DEVINL bool not_finite(uint32_t h) { return (h & 0x7c00u) == 0x7c00u; }

// Whether every block with a key that the query at p sees is a block of the cache.
__noinline__ __device__ bool blocks_ok(const Args &a, const int32_t *bt, int p) {
  const int lo = win::run_start(p, a.window);
  for (int b = lo / a.bs; b <= p / a.bs; ++b) {
    const int32_t id = __ldg(bt + b);
    if (id < 0 || id >= a.num_blocks) return false;
  }
  const int ns = min(a.sinks, lo);
  for (int b = 0; b * (int64_t)a.bs < ns; ++b) {
    const int32_t id = __ldg(bt + b);
    if (id < 0 || id >= a.num_blocks) return false;
  }
  return true;
}

// Adds the values of V at (key tile c, columns col..col+31) that are not finite and
// belong to keys that the query at p sees (they are zeros in shared memory).
template <bool Q8>
__noinline__ __device__ void add_not_finite(const Args &a, const int32_t *bt, int kvh, int p,
                                            const Pair &pr, int c, int col, float *o) {
  for (int key = c * kKeys; key < (c + 1) * kKeys; ++key) {
    if (!pr.sees(p, key)) continue;
    const int32_t blk = __ldg(bt + key / a.bs);
    if (blk < 0 || blk >= a.num_blocks) continue;
    const int64_t row = blk * a.s_block + kvh * a.s_head + (key % a.bs) * a.s_token + col;
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

template <int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 1) window_prefill_kernel(const Args a) {
  using S = Shape<D>;
  constexpr int NB = S::NB, kSlots = S::kSlots;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  // 128-byte swizzle atoms must sit on 1024-byte boundaries of the shared window
  unsigned char *smem = smem_raw + ((1024u - (va::smem_addr(smem_raw) & 1023u)) & 1023u);
  uint64_t *bar_full = reinterpret_cast<uint64_t *>(smem + S::oBar);  // [kSlots] tile landed
  uint64_t *bar_empty = bar_full + kSlots;   // [kSlots] MMAs that read the slot are done
  uint64_t *bar_s = bar_empty + kSlots;      // [kTiles] S written
  uint64_t *bar_p = bar_s + kTiles;          // [kTiles] P published (kRows arrivals)
  uint64_t *bar_o = bar_p + kTiles;          // [kTiles] PV done
  uint64_t *bar_q = bar_o + kTiles;          // Q staged
  uint64_t *bar_end = bar_q + 1;             // every MMA retired
  int *state = reinterpret_cast<int *>(bar_end + 1);
  int &s_dead = state[0], &s_bad = state[1], &s_poison = state[2];
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(state + 3);
  static_assert((2 * kSlots + 3 * kTiles + 2) * 8 + 16 <= 256, "barrier space");

  va::pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
  if (t_begin < 0 || t_end > a.T || (L > 0 && (L + (int64_t)a.bs - 1) / a.bs > a.max_blocks)) {
    if (tid == 0 && local == 0 && kvh == 0) va::raise_flag(a.err, VA_FLAG_CTX_OVERFLOW);
    return;
  }
  if (L <= 0) return;
  const int t0 = (int)t0l, nq = min(TP, t_end - t0);
  const int p0 = L - (t_end - t0);  // position of token t0 (may be negative: skipped)
  Pair pr;
  pr.window = a.window;
  pr.sinks = a.sinks;
#pragma unroll
  for (int h = 0; h < kTiles; ++h) {
    const int n = min(a.TQ, nq - h * a.TQ);
    pr.pmin[h] = max(p0 + h * a.TQ, 0);
    pr.pmax[h] = n > 0 ? p0 + h * a.TQ + n - 1 : -1;
  }
  const int plast = max(pr.pmax[0], pr.pmax[1]);
  if (plast < 0) return;
  const int pfirst = pr.pmax[0] >= 0 ? pr.pmin[0] : pr.pmin[1];
  const win::Tiles tl = win::key_tiles(pfirst, plast, a.window, a.sinks, kKeys);
  const int nch = tl.count;
  const int32_t *bt = a.bt + seq * a.max_blocks;

  if (tid == 0) {
    s_dead = s_bad = s_poison = 0;
    for (int i = 0; i < kSlots; ++i) {
      va::mbar_init(&bar_full[i], kProducers);
      va::mbar_init(&bar_empty[i], 1);
    }
    for (int h = 0; h < kTiles; ++h) {
      va::mbar_init(&bar_s[h], 1);
      va::mbar_init(&bar_p[h], kRows);
      va::mbar_init(&bar_o[h], 1);
    }
    va::mbar_init(bar_q, kSoftmax);
    va::mbar_init(bar_end, 1);
    va::fence_barrier_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc(tmem_slot, tc::kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  auto dead = [&]() { return *(volatile int *)&s_dead != 0; };
  auto wait_bar = [&](uint64_t *bar, uint32_t parity) {
    if (dead()) return;
    if (!va::mbar_wait_bounded(bar, parity, kWaitLimit) && atomicExch(&s_dead, 1) == 0)
      va::raise_flag(a.err, VA_FLAG_WAIT_TIMEOUT);
  };

  if (warp > kMmaWarp) {
    // =================== producers ===================
    const int pt = tid - kSoftmax - 32;
    int2 *info = reinterpret_cast<int2 *>(smem + S::oInfo);
    uchar2 *exps = reinterpret_cast<uchar2 *>(smem + S::oExp);
    const int klo = win::run_start(pfirst, a.window);
    const int64_t head_off = kvh * a.s_head;
    // block of key row pt of key tile j (-1: zeros)
    auto block_of = [&](int j) -> int32_t {
      if (j >= nch) return -1;
      const int key = win::tile_at(tl, j) * kKeys + pt;
      // a sink that only a later row's window has passed is inside the run [klo, plast]
      if (key > plast || (key < klo && key >= a.sinks)) return -1;
      const int32_t b = __ldg(bt + key / a.bs);
      if (b < 0 || b >= a.num_blocks) {
        va::raise_flag(a.err, VA_FLAG_BAD_BLOCK);
        *(volatile int *)&s_bad = 1;
        return -1;
      }
      return b;
    };
    auto off_of = [&](int j) { return (win::tile_at(tl, j) * kKeys + pt) % a.bs; };
    auto row_base = [&](int2 r) { return r.x * a.s_block + head_off + r.y * a.s_token; };
    auto slot_of = [&](int item) { return smem + S::oSlot + (item % kSlots) * S::kTileBytes; };
    auto wait_empty = [&](int item) {
      if (item >= kSlots) wait_bar(&bar_empty[item % kSlots], ((item / kSlots) - 1) & 1);
    };
    auto publish = [&](int item) {  // this thread's stores to the item's slot are visible
      va::fence_proxy_async_smem();
      va::mbar_arrive(&bar_full[item % kSlots]);
    };

    if constexpr (!Q8) {
      constexpr int P = D / 8;  // 16-byte pieces per row; each thread copies P of a tile
      int32_t blk = block_of(0);
      // item i: its copies have landed -> scrub (V of a partly masked tile), publish
      auto finish = [&](int item) {
        const int j = item >> 1;
        if ((item & 1) && pr.partial(win::tile_at(tl, j))) {
          unsigned char *sl = slot_of(item);
          bool hit = false;
#pragma unroll 4
          for (int i = pt; i < kKeys * P; i += kProducers) {
            uint4 *w = reinterpret_cast<uint4 *>(sl + tc::sw128_off(i / P, (i % P) * 8, kKeys));
            uint32_t x[4] = {w->x, w->y, w->z, w->w};
            bool h = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t bad = __vcmpgeu2(x[k] & 0x7fff7fffu, 0x7c007c00u);
              h = h || bad;
              x[k] &= ~bad;
            }
            if (h) *w = make_uint4(x[0], x[1], x[2], x[3]);
            hit = hit || h;
          }
          if (hit) *(volatile int *)&s_poison = 1;
        }
        publish(item);
      };
      auto copy = [&](int item) {
        wait_empty(item);
        const __half *src = reinterpret_cast<const __half *>(item & 1 ? a.vc : a.kc);
        const uint32_t sl = va::smem_addr(slot_of(item));
#pragma unroll 4
        for (int i = pt; i < kKeys * P; i += kProducers) {
          const int r = i / P, c = i % P;
          const int2 e = info[r];
          const bool on = e.x >= 0;
          win::cp_async_zfill<16>(sl + tc::sw128_off(r, c * 8, kKeys),
                                  src + (on ? row_base(e) + c * 8 : 0), on);
        }
        win::cp_async_commit();
      };
#pragma unroll 1
      for (int j = 0; j < nch; ++j) {
        producer_sync();  // everyone is done with the rows of the tile before
        info[pt] = make_int2(blk, off_of(j));
        producer_sync();
        blk = block_of(j + 1);
        copy(2 * j);
        if (j > 0) {
          win::cp_async_wait<kLag>();
          finish(2 * j - kLag);
        }
        copy(2 * j + 1);
        if (j > 0) {
          win::cp_async_wait<kLag>();
          finish(2 * j + 1 - kLag);
        }
      }
      win::cp_async_wait<0>();
      finish(2 * nch - 2);
      finish(2 * nch - 1);
    } else {
      constexpr int P = D / 16;  // 16-code pieces per row; each thread takes P of a tile
      int32_t blk0 = block_of(0), blk1 = block_of(1);
      auto load_exps = [&](int32_t blk, int j) {
        uchar2 e = make_uchar2(va::kQ8ExpBias, va::kQ8ExpBias);
        if (blk >= 0) {
          const int64_t at = blk * a.c_block + kvh * a.c_head + off_of(j) * a.c_token;
          e.x = __ldg(a.ks + at);
          e.y = __ldg(a.vs + at);
        }
        return e;
      };
      uchar2 e0 = load_exps(blk0, 0);
      auto load = [&](const uint8_t *src, uint4 (&r)[P]) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const int i = pt + k * kProducers, row = i / P, c = i % P;
          const int2 e = info[row];
          r[k] = make_uint4(0, 0, 0, 0);
          if (e.x >= 0) r[k] = __ldg(reinterpret_cast<const uint4 *>(src + row_base(e) + c * 16));
        }
      };
      auto store = [&](int item, uint4 (&r)[P], bool scrub) {
        unsigned char *sl = slot_of(item);
        const uchar2 *ex = exps + ((item >> 1) & 1) * kKeys;
        bool hit = false;
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const int i = pt + k * kProducers, row = i / P, c = i % P;
          const uint32_t f = va::q8_scale_h2(item & 1 ? ex[row].y : ex[row].x);
          uint32_t w[4] = {r[k].x, r[k].y, r[k].z, r[k].w}, o[8];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (scrub) {
              const uint32_t bad = __vcmpeq4(w[x] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              hit = hit || bad;
              w[x] &= ~bad;
            }
            o[2 * x] = va::hmul2(va::q8_decode2(w[x]), f);
            o[2 * x + 1] = va::hmul2(va::q8_decode2(w[x] >> 16), f);
          }
          *reinterpret_cast<uint4 *>(sl + tc::sw128_off(row, c * 16, kKeys)) =
              make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4 *>(sl + tc::sw128_off(row, c * 16 + 8, kKeys)) =
              make_uint4(o[4], o[5], o[6], o[7]);
        }
        if (hit) *(volatile int *)&s_poison = 1;
        publish(item);
      };
      // rows of key tile j for everyone; the next tile's exponents and block are on their way
      auto announce = [&](int j) {
        producer_sync();  // everyone has issued the loads of the tile before
        info[pt] = make_int2(blk0, j < nch ? off_of(j) : 0);
        exps[(j & 1) * kKeys + pt] = e0;
        producer_sync();
        blk0 = blk1;
        if (j + 1 < nch) e0 = load_exps(blk0, j + 1);
        blk1 = block_of(j + 2);
      };
      uint4 rk[P], rv[P];
      announce(0);
      load(a.kc, rk);
#pragma unroll 1
      for (int j = 0; j < nch; ++j) {
        load(a.vc, rv);
        wait_empty(2 * j);
        store(2 * j, rk, false);
        if (j + 1 < nch) {
          announce(j + 1);
          load(a.kc, rk);
        }
        wait_empty(2 * j + 1);
        store(2 * j + 1, rv, pr.partial(win::tile_at(tl, j)));
      }
    }
  } else if (warp == kMmaWarp) {
    // =================== MMA issue (lane 0) ===================
    const uint32_t sQ = va::smem_addr(smem), sSlot = sQ + S::oSlot;
    constexpr uint32_t IDESC_S = tc::idesc_f16(kRows, kKeys, false);
    constexpr uint32_t IDESC_O = tc::idesc_f16(kRows, NB * 64, true);
    auto wait_item = [&](int item) {
      wait_bar(&bar_full[item % kSlots], (item / kSlots) & 1);
      tc::fence_after_sync();
    };
    auto release = [&](int item) {
      if (lane == 0 && !dead()) tc::umma_commit(&bar_empty[item % kSlots]);
      __syncwarp();
    };
    int np[kTiles] = {0, 0};  // PVs issued per tile
    wait_bar(bar_q, 0);
#pragma unroll 1
    for (int j = 0; j <= nch; ++j) {
      const int c = j < nch ? win::tile_at(tl, j) : 0, cp = j > 0 ? win::tile_at(tl, j - 1) : 0;
      if (j < nch) wait_item(2 * j);
      if (j > 0) wait_item(2 * j - 1);
#pragma unroll
      for (int h = 0; h < kTiles; ++h) {
        if (j > 0 && pr.need(h, cp)) {
          // O_h (+)= P_h V: A = P_h [128 x 128] from TMEM, B = V [128 keys x NB*64] MN-major
          // (LBO = next 64 columns, SBO = next 8 keys)
          wait_bar(&bar_p[h], np[h] & 1);
          if (lane == 0 && !dead()) {
            tc::fence_after_sync();
            const uint32_t v = sSlot + ((2 * j - 1) % kSlots) * S::kTileBytes;
#pragma unroll
            for (int ks = 0; ks < kKeys / 16; ++ks)
              tc::umma_f16_ts(tmem + 256 + h * NB * 64, tmem + h * 128 + ks * 8,
                              tc::sdesc(v + ks * 2048, kKeys * 128, 1024), IDESC_O,
                              (np[h] > 0 || ks > 0) ? 1u : 0u);
            tc::umma_commit(&bar_o[h]);
          }
          __syncwarp();
          ++np[h];
        }
        if (h == kTiles - 1 && j > 0) release(2 * j - 1);
        if (j < nch && pr.need(h, c)) {
          // S_h = Q_h K^T, K-major operands.  It overwrites P_h, read by the PV before it:
          // one thread's tcgen05.mma run in issue order.
          if (lane == 0 && !dead()) {
            const uint32_t q = sQ + h * S::kTileBytes;
            const uint32_t k = sSlot + ((2 * j) % kSlots) * S::kTileBytes;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint32_t o = (ks >> 2) * 128 * 128 + (ks & 3) * 32;
              tc::umma_f16(tmem + h * 128, tc::sdesc(q + o, 16, 1024), tc::sdesc(k + o, 16, 1024),
                           IDESC_S, ks > 0);
            }
            tc::umma_commit(&bar_s[h]);
          }
          __syncwarp();
        }
      }
      if (j < nch) release(2 * j);
    }
    // every MMA issued above has retired before TMEM is freed
    if (lane == 0) {
      tc::umma_commit(bar_end);
      if (!va::mbar_wait_bounded(bar_end, 0, kWaitLimit) && atomicExch(&s_dead, 1) == 0)
        va::raise_flag(a.err, VA_FLAG_WAIT_TIMEOUT);
    }
    __syncwarp();
  } else {
    // =================== Q, then softmax of tile h, one thread per row ===================
    const int h = warp >> 2, row = tid & (kRows - 1);
    const int head0 = kvh * a.G;
    {
      constexpr int P = D / 8;
#pragma unroll 4
      for (int i = tid; i < kTiles * kRows * P; i += kSoftmax) {
        const int r2 = i / P, c = i - r2 * P, hh = r2 / kRows, r = r2 - hh * kRows;
        const int tk = r / a.G, g = r - tk * a.G, ti = hh * a.TQ + tk;
        const bool on = tk < a.TQ && ti < nq;
        win::cp_async_zfill<16>(
            va::smem_addr(smem + hh * S::kTileBytes + tc::sw128_off(r, c * 8, kRows)),
            a.q + (on ? (t0 + ti) * a.q_s_token + (int64_t)(head0 + g) * a.q_s_head + c * 8 : 0),
            on);
      }
      win::cp_async_commit();
      win::cp_async_wait<0>();
      va::fence_proxy_async_smem();
      va::mbar_arrive(bar_q);
    }
    const int tk = row / a.G, g = row - tk * a.G, ti = h * a.TQ + tk;
    const bool row_ok = tk < a.TQ && ti < nq && p0 + ti >= 0;
    // rows of no token take the tile's last position: their result is dropped
    const int pos = row_ok ? p0 + ti : pr.pmax[h];
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + h * 128 + lane_base;
    const uint32_t tO = tmem + 256 + h * NB * 64 + lane_base;
    const float sc = a.scale_log2;
    float m = -INFINITY, l = 0.f;
    int n = 0;  // key tiles of this tile so far
#pragma unroll 1
    for (int j = 0; j < nch; ++j) {
      const int c = win::tile_at(tl, j);
      if (!pr.need(h, c)) continue;
      // columns [vlo, vhi] and [0, vsk) of the key tile are visible
      const bool masked = !pr.full(h, c);
      const int vhi = pos - c * kKeys;
      const int vlo = a.window > 0 ? pos - a.window + 1 - c * kKeys : INT_MIN;
      const int vsk = a.sinks - c * kKeys;
      wait_bar(&bar_s[h], n & 1);
      tc::fence_after_sync();
      auto load64 = [&](int half, float (&p)[64]) {
        uint32_t x[32], y[32];
        tc::tmem_ld32(tS + half * 64, x);
        tc::tmem_ld32(tS + half * 64 + 32, y);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          p[i] = __uint_as_float(x[i]);
          p[32 + i] = __uint_as_float(y[i]);
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            const int k = half * 64 + i;
            p[i] = k <= vhi && (k >= vlo || k < vsk) ? p[i] : -INFINITY;
          }
        }
      };
      float rmax = -INFINITY;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float p[64];
        load64(half, p);
        float x[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
        for (int i = 4; i < 60; i += 8) {
          x[0] = tc::fmax3(x[0], p[i], p[i + 1]);
          x[1] = tc::fmax3(x[1], p[i + 2], p[i + 3]);
          x[2] = tc::fmax3(x[2], p[i + 4], p[i + 5]);
          x[3] = tc::fmax3(x[3], p[i + 6], p[i + 7]);
        }
        x[0] = tc::fmax3(x[0], p[60], p[61]);
        x[1] = tc::fmax3(x[1], p[62], p[63]);
        rmax = fmaxf(rmax, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
      }
      rmax *= sc;  // the scale is positive
      const float mn = (m == -INFINITY || rmax > m + 8.f) ? fmaxf(m, rmax) : m;
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
        float p[64];
        load64(half, p);
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float x0, x1;
          tc::upk2(tc::ffma2(tc::pk2(p[2 * i], p[2 * i + 1]), sc2, nm2), x0, x1);
          x0 = va::fast_exp2(x0);
          x1 = va::fast_exp2(x1);
          sum2[i & 1] = tc::fadd2(sum2[i & 1], tc::pk2(x0, x1));
          w[i] = va::pack_h2(x0, x1);
        }
        // over S columns that this thread has read already
        tc::tmem_st32(tS + half * 32, w);
      }
      float y0, y1, y2, y3;
      tc::upk2(sum2[0], y0, y1);
      tc::upk2(sum2[1], y2, y3);
      l = l * alpha + ((y0 + y1) + (y2 + y3));
      tc::tmem_wait_st();
      tc::fence_before_sync();
      va::mbar_arrive(&bar_p[h]);
      ++n;
    }
    if (n > 0) {
      wait_bar(&bar_o[h], (n - 1) & 1);
      tc::fence_after_sync();
      const bool poison = *(volatile int *)&s_poison != 0;  // some V value was scrubbed
      bool write = row_ok && !dead();
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
              if (pr.partial(c)) add_not_finite<Q8>(a, bt, kvh, pos, pr, c, k, fix);
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
    tc::tmem_dealloc(tmem, tc::kTmemCols);
  }
}

template <int D, bool Q8>
int launch_t(const Args &a, unsigned grid, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (!win::allow_smem(window_prefill_kernel<D, Q8>, (int)Shape<D>::kBytes, done))
    return VA_ERR_LAUNCH;
  if (va_host::launch_pdl_smem(window_prefill_kernel<D, Q8>, grid, kThreads, Shape<D>::kBytes, st,
                               a))
    return VA_ERR_LAUNCH;
  return va_host::launch_status();
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
  a.TQ = kRows / G;
  a.bs = block_size;
  a.window = win::window_of(window);
  a.sinks = sink_tokens;
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
  switch (head_size + (kv_e4m3 ? 1 : 0)) {
    case 32: return launch_t<32, false>(a, grid, st);
    case 33: return launch_t<32, true>(a, grid, st);
    case 64: return launch_t<64, false>(a, grid, st);
    case 65: return launch_t<64, true>(a, grid, st);
    case 96: return launch_t<96, false>(a, grid, st);
    case 97: return launch_t<96, true>(a, grid, st);
    case 128: return launch_t<128, false>(a, grid, st);
    case 129: return launch_t<128, true>(a, grid, st);
  }
  return VA_ERR_UNSUPPORTED;
}

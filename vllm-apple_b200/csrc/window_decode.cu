// Single-token attention over a paged cache under a sliding window with sinks
// (visibility rule: window.cuh), fp16 or e4m3 cache (row format: kv_q8.cuh), with the
// write of the new row.
//
//   out_h = sum_j p_hj v_j / sum_j p_hj,   p_hj = 2^(scale log2(e) q_h.k_j - m_h)
//
// Every K/V byte of a sequence is read once per kv head and serves all query heads of
// its group, so the kernel is bound by HBM; everything else is kept off its way:
//   * The products run on mma.sync m16n8k16 with the KEYS as the 16 rows and the query
//     heads as the 8 columns (S^T = K Q^T, then O^T = V^T P^T), so a group of up to 8
//     heads fills the instruction's columns and an e4m3 cache (half the bytes per key)
//     does not run into the FP32 pipe, as one FMA per head and value would.
//   * The order of a contraction's terms is free, so a lane's fragments of K are consecutive
//     values of a row, and those of V consecutive values of four rows: 16-byte reads.  The
//     rows come in by cp.async, 16 bytes a lane and whole 128-byte lines a request (with
//     requests of 64 bytes, a fragment's own share of a row, the L2 limited the kernel), into
//     a ring that belongs to the warp alone: no barrier, only cp.async.wait_group.
//   * A warp takes every 4th tile of 16 keys of its CTA's range; kStages tiles per warp
//     are in flight.  S^T comes out of the MMA with keys in rows; P^T is wanted with keys
//     in columns: one 8x8 transpose (movmatrix) per 8 keys.
//   * Statistics, sums and O are fp32; P is rounded to fp16 (2^-11 of a value <= 1) for
//     the second product, whose instruction takes nothing wider beside fp16 values.  The
//     result's error against 64 bits is 2.3e-4 to 2.7e-4 of its size; with P in fp32 it is the
//     result's own rounding, 2.0e-4.  An e4m3 code becomes fp16 exactly; the exponent of a K row
//     scales its fp32 score, that of a V row its fp16 values (both exact).
//   * Long lists of keys: all tiles of the call, in (sequence, head group, tile) order, are one
//     list that is cut into equal ranges, one per CTA that fits the GPU, so that ragged lengths
//     and one long sequence make one even wave.  A range holds whole (sequence, head group)
//     lists, written at once, and at most two parts of lists, whose (O, m, l) a second
//     kernel, launched as a programmatic dependent, merges in list order.  Short lists and very
//     many of them have a CTA each instead (make_plan).
//   * Keys that the query does not see are zero-filled, never read: what lies in the
//     cache behind a sequence, before its window or in a freed block does not matter.
// Measured (32 heads of 128 over 8): 128 sequences under a window of 1024, fp16, 94-96 us (5.6
// TB/s); 128 ragged e4m3 contexts of up to 8192 tokens 207 us (5.4 TB/s; 218-224 called one by
// one with other inputs each time), one of 131000 59 us (4.6 TB/s).  The copies alone, without
// products, took 210 and 53 us of the last two when they took 212 and 60, the products alone 132
// and 42.  A stream of tiles per warp instead of per CTA took 273 and 74 us, two or eight warps
// per CTA 269 and 251 us for the contexts, two waves of ranges more than one.  Groups of 9 to 16
// heads (two tiles of columns; 247 to 249 registers at head size 128, so two CTAs per SM where
// an e4m3 group of up to 8 has three): the same contexts take 361-371 us in fp16 (349 with
// groups of 4) and 282-294 in e4m3 (207).  Groups of 32 read every key twice: 727 and 577.
// Small calls (4 sequences under a window of 128, 14 heads of 64 over 2: 4.6 us) are one launch
// and one chain of dependent loads on a few CTAs.
#include <float.h>

#include "window.cuh"

namespace {

constexpr int kNW = 4;  // warps per CTA
constexpr int kKeys = 16;
// Where a maximum begins.  Scores that are -inf (masked keys, an infinity in a K row) do not
// move it, and their powers are 0; from -inf they would be the NaN of -inf - -inf, which other
// keys' results could not take back.  No finite score lies below.
constexpr float kLowest = -FLT_MAX;

template <int D, bool Q8>
struct Shape {
  static constexpr int ES = Q8 ? 1 : 2;                    // bytes per value
  static constexpr int KB = (D / 4 * ES) % 16 ? 8 : 16;    // K: bytes per read
  static constexpr int KN = D / 4 * ES / KB;               // reads per row and lane
  static constexpr int KE = KB / ES;                       // values per read
  static constexpr int VB = (D / 8 * ES) % 16 == 0 ? 16 : (D / 8 * ES) % 8 == 0 ? 8 : 4;
  static constexpr int VN = D / 8 * ES / VB;
  static constexpr int VE = VB / ES;
  static constexpr int RB = D * ES;                        // bytes of a row
  static constexpr int P = RB / 16;                        // 16-byte pieces of a row
  static constexpr int oV = kKeys * RB;                    // stage: K rows, V rows, exponents
  static constexpr int oS = 2 * kKeys * RB;
  // The rows of a stage lie one after the other, their pieces exchanged inside 128-byte
  // lines so that the fragment reads below hit every bank once (row sizes 32 to 256; the
  // rows of 96 and 192 bytes stay as they are).
  static VA_DEVINL int k_swz(int r) { return RB % 128 == 0 ? (r & 1) << 6 : 0; }
  static VA_DEVINL int v_swz(int r) {
    return RB == 32 ? (r >> 2 & 1) << 5 : RB % 64 == 0 && RB != 192 ? (r >> 1 & 3) << 5 : 0;
  }
  static constexpr int kStage = oS + (Q8 ? 128 : 0);
  // tiles per pass: an e4m3 tile is half the bytes, so two share a pass's reductions
  static constexpr int KT = Q8 ? 2 : 1;
  static constexpr int kStages = D * ES >= 256 ? 3 : 4;  // a multiple of KT
  static constexpr int kHead = D + 4;  // floats of a head's row in the warps' merge
  static constexpr int kRing = kNW * kStages * kStage;
};

struct Args {
  __half *out;
  const __half *q;
  uint8_t *kc, *vc;   // cache bytes (fp16 or e4m3)
  uint8_t *ks, *vs;   // exponent bytes (e4m3 caches)
  const __half *nk, *nv;
  const int32_t *bt, *sl;
  float *ws_acc;     // [2 * ranges][gc][D] un-normalised O of the ranges' first and last parts
  float2 *ws_ml;     // [2 * ranges][gc] (m, l) of them; l < 0: a block could not be read
  int64_t *ws_plan;  // {places per range, open, places before sequence 0, 1, ...}
  int32_t *err;
  int64_t max_blocks, num_blocks, max_len;
  int B, Hq, G, hg, gc, Hk, window, sinks, ranges;
  win::FastDiv bs;
  float scale_log2;
  int64_t s_block, s_head, s_token, c_block, c_head, c_token;
  int64_t q_s_token, q_s_head, o_s_token, o_s_head, n_s_token, n_s_head;
};

VA_DEVINL void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                   uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
VA_DEVINL uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <int V>
VA_DEVINL void lds(uint32_t (&w)[V / 4], const unsigned char *p) {
  if constexpr (V == 16) {
    const uint4 x = *reinterpret_cast<const uint4 *>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (V == 8) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  }
}

// Length of a sequence, 0 when it is skipped.
VA_DEVINL int seq_len(const Args &a, int seq, bool flag) {
  const int L = __ldg(a.sl + seq);
  if (L <= 0) return 0;
  if (L > a.max_len || a.bs.div(L - 1) >= a.max_blocks) {
    if (flag) va::raise_flag(a.err, VA_FLAG_CTX_OVERFLOW);
    return 0;
  }
  return L;
}
VA_DEVINL win::Tiles seq_tiles(const Args &a, int L) {
  return win::key_tiles(L - 1, L - 1, a.window, a.sinks, kKeys);
}
VA_DEVINL int num_tiles(const Args &a, int L) { return L > 0 ? seq_tiles(a, L).count : 0; }

// Fewest tiles of a range: two per warp.
constexpr int kMinRange = 2 * kNW;

// Beginning another list of tiles (its length, block ids, first copies, the merge of the
// warps) costs a CTA about as long as 28 tiles, so when the ranges are cut every list
// counts for that many more: its first `open` places hold no tile.  Three quarters of a range at
// most, since every range begins one list in any case.  Measured at 0, 4, 16, 28 and 48: 128
// ragged e4m3 contexts 270, 226, 220, 211 and 222 us (a build that took 211); 64 shorter ones,
// whose ranges are some 30 tiles, 29 us (0), 24 (a quarter of a range), 19.5 (three quarters),
// 23 (28).
constexpr int kOpenMost = 28;
VA_DEVINL int places(int tiles, int open) { return tiles > 0 ? tiles + open : 0; }

// The range of this CTA in the list of all places in (sequence, head group, tile) order.
struct Range {
  int64_t begin, end;  // places of the list
  int64_t before;      // places of one head group before sequence `seq`
  int seq;             // sequence of the first place
  int open;
};
// Every CTA sums the sequences' tiles for itself (their lengths are few and in L2), so no
// planning kernel runs before; CTA 0 leaves the sums for the merge.
VA_DEVINL Range find_range(const Args &a) {
  __shared__ int64_t s_warp[kNW];
  __shared__ int64_t s_before;
  __shared__ int s_seq;
  constexpr int kCount = 17;  // sums hold tiles << 17 | sequences (at most 65535) with tiles
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + kNW * 32 - 1) / (kNW * 32);
  const int q0 = min(tid * per, a.B), q1 = min(q0 + per, a.B);
  int64_t mine = 0;
  for (int q = q0; q < q1; ++q) {
    const int n = num_tiles(a, seq_len(a, q, blockIdx.x == 0));
    if (n > 0) mine += (int64_t)n << kCount | 1;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int64_t sum = 0, excl = incl - mine;
#pragma unroll
  for (int w = 0; w < kNW; ++w) {
    if (w < warp) excl += s_warp[w];
    sum += s_warp[w];
  }
  Range r;
  r.open = (int)min((sum >> kCount) * a.Hk * 3 / a.ranges / 4, (int64_t)kOpenMost);
  auto to_places = [&](int64_t x) {
    return (x >> kCount) + (x & ((1 << kCount) - 1)) * r.open;
  };
  const int64_t total = to_places(sum) * a.Hk;
  const int64_t w = max((total + a.ranges - 1) / a.ranges, (int64_t)kMinRange);
  r.begin = blockIdx.x * w;
  r.end = min(r.begin + w, total);
  int64_t at = to_places(excl);
  if (r.begin >= at * a.Hk && r.begin < to_places(excl + mine) * a.Hk) {
    int q = q0;  // this thread's sequences hold the first place
    int64_t x = at;
    for (int n; x + (n = places(num_tiles(a, seq_len(a, q, false)), r.open)) <= r.begin / a.Hk; ++q)
      x += n;
    s_before = x;
    s_seq = q;
  }
  if (blockIdx.x == 0) {
    if (tid == 0) {
      a.ws_plan[0] = w;
      a.ws_plan[1] = r.open;
    }
    for (int q = q0; q < q1; ++q) {
      a.ws_plan[2 + q] = at;
      at += places(num_tiles(a, seq_len(a, q, false)), r.open);
    }
  }
  __syncthreads();
  r.before = s_before;  // not set, and not used, where the range is empty
  r.seq = s_seq;
  return r;
}

// The new K (lanes 0..15) and V (lanes 16..31) row of one kv head into the cache.
template <int D, bool Q8>
VA_DEVINL void write_new_row(const Args &a, int seq, int kvh, int64_t blk, int off) {
  const int sub = threadIdx.x & 15;
  const bool is_v = threadIdx.x & 16, on = sub * 8 < D;
  const __half *src = (is_v ? a.nv : a.nk) + seq * a.n_s_token + kvh * a.n_s_head + sub * 8;
  uint4 w = make_uint4(0, 0, 0, 0);
  if (on) w = *reinterpret_cast<const uint4 *>(src);
  const int64_t dst = blk * a.s_block + kvh * a.s_head + off * a.s_token + sub * 8;
  uint8_t *cache = is_v ? a.vc : a.kc;
  if constexpr (!Q8) {
    if (on) *reinterpret_cast<uint4 *>(cache + 2 * dst) = w;
  } else {
    uint32_t m = va::q8_absmax2_finite(
        va::q8_absmax2_finite(va::q8_absmax2_finite(va::q8_absmax2_finite(0, w.x), w.y), w.z), w.w);
    m = max(m & 0xffffu, m >> 16);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int e = va::q8_exponent(m);
    const uint32_t inv = va::q8_inv_h2(e);
    if (on)
      *reinterpret_cast<uint2 *>(cache + dst) =
          make_uint2(va::q8_encode4(w.x, w.y, inv), va::q8_encode4(w.z, w.w, inv));
    if (sub == 0)
      (is_v ? a.vs : a.ks)[blk * a.c_block + kvh * a.c_head + off * a.c_token] =
          (uint8_t)(e + va::kQ8ExpBias);
  }
}

// One part: tiles [t_begin, t_end) of one head group of one sequence.  `slot` >= 0: not
// the whole list of its tiles, so the result goes to that slot of the workspace.
template <int D, bool Q8, int NT>
VA_DEVINL void decode_part(const Args &a, unsigned char *smem, int *s_bad, int seq, int hk, int L,
                           const win::Tiles &tl, int t_begin, int t_end, int64_t slot) {
  using S = Shape<D, Q8>;
  const int kvh = hk / a.hg, head0 = kvh * a.G + (hk - kvh * a.hg) * a.gc;
  const int nheads = min(a.gc, (kvh + 1) * a.G - head0);
  const int lo = win::run_start(L - 1, a.window);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int32_t *bt = a.bt + seq * a.max_blocks;
  // Q^T fragments: columns = heads, rows in the order of the K fragments below
  uint32_t qf[NT][D / 16][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int e = 4 * ks, d = e / S::KE * (4 * S::KE) + t * S::KE + e % S::KE;
      uint2 w = make_uint2(0, 0);
      if (n * 8 + g < nheads)
        w = __ldg(reinterpret_cast<const uint2 *>(a.q + seq * a.q_s_token +
                                                  (int64_t)(head0 + n * 8 + g) * a.q_s_head + d));
      qf[n][ks][0] = w.x;
      qf[n][ks][1] = w.y;
    }

  // ---- copy pipeline: tile i of this warp is key tile t_begin + warp + i * kNW ----
  constexpr int KT = S::KT, R = S::kStages;
  const int ntiles = max(0, (t_end - t_begin - warp + kNW - 1) / kNW);
  const int npass = (ntiles + KT - 1) / KT;  // tiles past ntiles are zeros
  unsigned char *ring = smem + warp * R * S::kStage;
  const bool one_block = a.bs.d % kKeys == 0;  // a tile never straddles two blocks
  // this lane's pieces lane, lane + 32, ... of a tile, in row order
  const int64_t tok = a.s_token * S::ES;
  const uint8_t *k_head = a.kc + kvh * a.s_head * S::ES, *v_head = a.vc + kvh * a.s_head * S::ES;
  const uint8_t *s_lane = Q8 ? (lane < 16 ? a.ks : a.vs) + kvh * a.c_head : nullptr;
  bool bad = false;
  auto key_tile = [&](int i) { return win::tile_at(tl, t_begin + warp + i * kNW); };
  auto seen = [&](int key) { return key < L && (key >= lo || key < a.sinks); };
  // block id of tile i (one_block), or of this lane's key (lane & 15) of it, as the table
  // has it: it is looked at a pass later, when it has arrived
  auto block_of = [&](int i) -> int32_t {
    if (i >= ntiles) return -1;
    const int key0 = key_tile(i) * kKeys, key = key0 + (lane & 15);
    if (!one_block && !seen(key)) return -1;
    return __ldg(bt + a.bs.div(one_block ? key0 : key));
  };
  // block ids of the next pass to be copied, asked for a pass ahead; exponent bytes of the
  // pass copied last, stored when the next is copied (nothing waits for either)
  int32_t blk[KT];
  uint32_t sc[KT];
  unsigned char *sc_at = nullptr;
#pragma unroll
  for (int u = 0; u < KT; ++u) {
    blk[u] = block_of(u);
    sc[u] = va::kQ8ExpBias;
  }
  auto copy_tile = [&](int i, unsigned char *st, int32_t blk, uint32_t &sc_prev) {
    const int key0 = i < ntiles ? key_tile(i) * kKeys : 0;
    const bool in = blk >= 0 && blk < a.num_blocks;
    if (one_block && in && key0 + kKeys <= L &&
        (key0 >= lo || key0 + kKeys <= a.sinks)) {
      // every key is seen and the rows are evenly spaced
      const int off = a.bs.mod(key0);
      const int64_t base = blk * a.s_block * S::ES + off * tok;
#pragma unroll
      for (int i = 0; i < S::P / 2; ++i) {
        const int r = (lane + 32 * i) / S::P, c = (lane + 32 * i) % S::P * 16;
        const int64_t src = base + r * tok + c;
        win::cp_async<16>(va::smem_addr(st + ((r * S::RB + c) ^ S::k_swz(r))), k_head + src);
        win::cp_async<16>(va::smem_addr(st + S::oV + ((r * S::RB + c) ^ S::v_swz(r))),
                          v_head + src);
      }
      if constexpr (Q8)
        sc_prev = s_lane[blk * a.c_block + (off + (lane & 15)) * a.c_token];
    } else {
      const int key = key0 + (lane & 15), off = a.bs.mod(key);
      const bool want = i < ntiles && seen(key), on = want && in;
      bad = bad || (want && !in);
      const int64_t row = on ? blk * a.s_block * S::ES + off * tok : 0;
#pragma unroll
      for (int i = 0; i < S::P / 2; ++i) {
        const int r = (lane + 32 * i) / S::P, c = (lane + 32 * i) % S::P * 16;
        const int64_t src = __shfl_sync(0xffffffffu, row, r) + c;
        const bool ro = __shfl_sync(0xffffffffu, (int)on, r);
        win::cp_async_zfill<16>(va::smem_addr(st + ((r * S::RB + c) ^ S::k_swz(r))),
                                ro ? k_head + src : a.kc, ro);
        win::cp_async_zfill<16>(va::smem_addr(st + S::oV + ((r * S::RB + c) ^ S::v_swz(r))),
                                ro ? v_head + src : a.vc, ro);
      }
      if constexpr (Q8)
        sc_prev = on ? s_lane[blk * a.c_block + off * a.c_token] : va::kQ8ExpBias;
    }
  };
  int wslot = 0;  // ring slot of the next pass
  auto copy_pass = [&](int p) {
    if constexpr (Q8) {
      if (sc_at) {
#pragma unroll
        for (int u = 0; u < KT; ++u) {
          unsigned char *at = sc_at + u * S::kStage;
          if (lane < 16)  // K: fp32 2^e; V: fp16 2^e
            reinterpret_cast<uint32_t *>(at)[lane] = sc[u] << 23;
          else
            reinterpret_cast<uint16_t *>(at)[lane + 16] = (uint16_t)va::q8_scale_h2(sc[u]);
        }
      }
      sc_at = nullptr;
    }
    if (p < npass) {
      unsigned char *st = ring + wslot * S::kStage;
#pragma unroll
      for (int u = 0; u < KT; ++u) copy_tile(p * KT + u, st + u * S::kStage, blk[u], sc[u]);
      if constexpr (Q8) sc_at = st + S::oS;
#pragma unroll
      for (int u = 0; u < KT; ++u) blk[u] = block_of((p + 1) * KT + u);
      wslot = wslot + KT == R ? 0 : wslot + KT;
    }
    win::cp_async_commit();
  };
  // The warp that reads the newest key (its last tile) writes it before, and reads it back
  // with the rest; its first copies are on their way by then where they do not hold it.
  constexpr int kAhead = R / KT - 1;  // passes
  const bool writes = a.nk && t_end == tl.count && warp == (t_end - 1 - t_begin) % kNW;
  auto write = [&]() {
    const int page = a.bs.div(L - 1);
    const int32_t to = __ldg(bt + page);
    if (to >= 0 && to < a.num_blocks)
      write_new_row<D, Q8>(a, seq, kvh, to, L - 1 - page * (int)a.bs.d);
    __syncwarp();  // for the lanes that copy it
  };
  if (writes && npass <= kAhead) write();
#pragma unroll
  for (int p = 0; p < kAhead; ++p) copy_pass(p);
  if (writes && npass > kAhead) write();

  float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = kLowest;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }

  int rslot = 0;
#pragma unroll 1
  for (int i = 0; i < npass; ++i) {
    copy_pass(i + kAhead);
    win::cp_async_wait<kAhead>();
    __syncwarp();  // other lanes' copies and exponents
    const unsigned char *st0 = ring + rslot * S::kStage;
    // ---- S^T = K Q^T ----
    float s[KT][NT][4];
#pragma unroll
    for (int u = 0; u < KT; ++u) {
      const unsigned char *st = st0 + u * S::kStage;
#pragma unroll
      for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < S::KN; ++c) {
        uint32_t wa[S::KB / 4], wb[S::KB / 4];
        const int at = (g * S::RB + c * 4 * S::KB + t * S::KB) ^ S::k_swz(g);
        lds<S::KB>(wa, st + at);
        lds<S::KB>(wb, st + at + 8 * S::RB);  // row g + 8 is exchanged like row g
#pragma unroll
        for (int x = 0; x < S::KE / 4; ++x) {
          uint32_t a0, a1, a2, a3;
          if constexpr (Q8) {
            va::q8_decode4(wa[x], a0, a2);
            va::q8_decode4(wb[x], a1, a3);
          } else {
            a0 = wa[2 * x];
            a2 = wa[2 * x + 1];
            a1 = wb[2 * x];
            a3 = wb[2 * x + 1];
          }
          const int ks = c * (S::KE / 4) + x;
#pragma unroll
          for (int n = 0; n < NT; ++n) mma(s[u][n], a0, a1, a2, a3, qf[n][ks][0], qf[n][ks][1]);
        }
      }
      // ---- scale, mask (rows g, g + 8 of the tile; columns 2t, 2t + 1) ----
      float fa = a.scale_log2, fb = a.scale_log2;
      if constexpr (Q8) {
        const float *f = reinterpret_cast<const float *>(st + S::oS);
        fa *= f[g];
        fb *= f[g + 8];
      }
      const int key0 = i * KT + u < ntiles ? key_tile(i * KT + u) * kKeys : L;
      const bool sa = seen(key0 + g), sb = seen(key0 + g + 8);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[u][n][0] = sa ? s[u][n][0] * fa : -INFINITY;
        s[u][n][1] = sa ? s[u][n][1] * fa : -INFINITY;
        s[u][n][2] = sb ? s[u][n][2] * fb : -INFINITY;
        s[u][n][3] = sb ? s[u][n][3] * fb : -INFINITY;
      }
    }
    // ---- online softmax ----
    uint32_t pb[KT][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float m0 = m[n][0], m1 = m[n][1];
#pragma unroll
      for (int u = 0; u < KT; ++u) {
        m0 = fmaxf(m0, fmaxf(s[u][n][0], s[u][n][2]));
        m1 = fmaxf(m1, fmaxf(s[u][n][1], s[u][n][3]));
      }
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, w));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, w));
      }
      if (__any_sync(0xffffffffu, m0 != m[n][0] || m1 != m[n][1])) {
        const float f0 = m0 == m[n][0] ? 1.f : va::fast_exp2(m[n][0] - m0);
        const float f1 = m1 == m[n][1] ? 1.f : va::fast_exp2(m[n][1] - m1);
        m[n][0] = m0;
        m[n][1] = m1;
        l[n][0] *= f0;
        l[n][1] *= f1;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          o[n][k][0] *= f0;
          o[n][k][1] *= f1;
          o[n][k][2] *= f0;
          o[n][k][3] *= f1;
        }
      }
#pragma unroll
      for (int u = 0; u < KT; ++u) {
        const float x0 = va::fast_exp2(s[u][n][0] - m0), x1 = va::fast_exp2(s[u][n][1] - m1);
        const float y0 = va::fast_exp2(s[u][n][2] - m0), y1 = va::fast_exp2(s[u][n][3] - m1);
        l[n][0] += x0 + y0;
        l[n][1] += x1 + y1;
        pb[u][n][0] = transpose8x8(va::pack_h2(x0, x1));
        pb[u][n][1] = transpose8x8(va::pack_h2(y0, y1));
      }
    }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int u = 0; u < KT; ++u) {
      const unsigned char *st = st0 + u * S::kStage;
      uint32_t f01 = 0, f89 = 0;
      if constexpr (Q8) {
        const uint32_t *f = reinterpret_cast<const uint32_t *>(st + S::oS + 64);
        f01 = f[t];
        f89 = f[t + 4];
      }
#pragma unroll
      for (int c = 0; c < S::VN; ++c) {
        uint32_t w[4][S::VB / 4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          // rows 2t, 2t + 1, 2t + 8, 2t + 9 are exchanged alike
          lds<S::VB>(w[r], st + S::oV + (((2 * t + (r & 1)) * S::RB + c * 8 * S::VB + g * S::VB) ^
                                         S::v_swz(2 * t)) +
                               (r >> 1) * 8 * S::RB);
#pragma unroll
        for (int x = 0; x < S::VE / 2; ++x) {  // values 2x, 2x + 1 of the copy
          uint32_t a0, a1, a2, a3;
          if constexpr (Q8) {
            const uint32_t sel = x & 1 ? 0x7362 : 0x5140;
            const uint32_t p = __byte_perm(w[0][x / 2], w[1][x / 2], sel);
            const uint32_t q = __byte_perm(w[2][x / 2], w[3][x / 2], sel);
            va::q8_decode4(p, a0, a1);
            va::q8_decode4(q, a2, a3);
            a0 = va::hmul2(a0, f01);
            a1 = va::hmul2(a1, f01);
            a2 = va::hmul2(a2, f89);
            a3 = va::hmul2(a3, f89);
          } else {
            a0 = __byte_perm(w[0][x], w[1][x], 0x5410);
            a1 = __byte_perm(w[0][x], w[1][x], 0x7632);
            a2 = __byte_perm(w[2][x], w[3][x], 0x5410);
            a3 = __byte_perm(w[2][x], w[3][x], 0x7632);
          }
          const int k = c * (S::VE / 2) + x;
#pragma unroll
          for (int n = 0; n < NT; ++n) mma(o[n][k], a0, a1, a2, a3, pb[u][n][0], pb[u][n][1]);
        }
      }
    }
    rslot = rslot + KT == R ? 0 : rslot + KT;
    __syncwarp();  // the next copies go over this pass's slots
  }
  win::cp_async_wait<0>();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) {
      l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], w);
      l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], w);
    }
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) s_bad[warp] = bad;
  __syncthreads();  // the ring is free: the warps' results go there

  // value e of lane g lies at e * 8 + g of its head's row: stores hit every bank once
  constexpr int NH = 8 * NT, HS = S::kHead;
  float *so = reinterpret_cast<float *>(smem);          // [kNW][NH][HS]
  float *sm = so + kNW * NH * HS, *sl = sm + kNW * NH;  // [kNW][NH]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        so[(warp * NH + n * 8 + 2 * t) * HS + (2 * k + y) * 8 + g] = o[n][k][2 * y];
        so[(warp * NH + n * 8 + 2 * t + 1) * HS + (2 * k + y) * 8 + g] = o[n][k][2 * y + 1];
      }
    if (g == 0) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        sm[warp * NH + n * 8 + 2 * t + y] = m[n][y];
        sl[warp * NH + n * 8 + 2 * t + y] = l[n][y];
      }
    }
  }
  __syncthreads();
  bool skip = false;
#pragma unroll
  for (int w = 0; w < kNW; ++w) skip = skip || s_bad[w] != 0;
  if (skip && threadIdx.x == 0) va::raise_flag(a.err, VA_FLAG_BAD_BLOCK);
  for (int i = threadIdx.x; i < nheads * D; i += kNW * 32) {
    const int h = i / D, d = i - h * D;
    const int at = (d / (8 * S::VE) * S::VE + d % S::VE) * 8 + d / S::VE % 8;
    float M = sm[h];
#pragma unroll
    for (int w = 1; w < kNW; ++w) M = fmaxf(M, sm[w * NH + h]);
    float A = 0.f, Ls = 0.f;
#pragma unroll
    for (int w = 0; w < kNW; ++w) {
      // (a warp without tiles adds zeros)
      const float f = va::fast_exp2(sm[w * NH + h] - M);
      A += so[(w * NH + h) * HS + at] * f;
      Ls += sl[w * NH + h] * f;
    }
    if (slot < 0) {
      if (!skip)
        a.out[seq * a.o_s_token + (int64_t)(head0 + h) * a.o_s_head + d] = __float2half_rn(A / Ls);
    } else {
      const int64_t p = slot * a.gc + h;
      a.ws_acc[p * D + d] = A;
      // l < 0 marks a part with an unreadable block: its sequence is left alone
      if (d == 0) a.ws_ml[p] = make_float2(M, skip ? -1.f : Ls);
    }
  }
}

// NT: tiles of 8 query heads per warp (1 for groups of up to 8, 2 up to 16).
template <int D, bool Q8, int NT>
__global__ void __launch_bounds__(kNW * 32) window_decode_kernel(const Args a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int s_bad[kNW];
  va::pdl_enter();
  if (a.ranges == 0) {  // a CTA per (sequence, head group)
    const int seq = blockIdx.x / a.Hk, hk = blockIdx.x - seq * a.Hk;
    const int L = seq_len(a, seq, hk == 0 && threadIdx.x == 0);
    if (L == 0) return;
    const win::Tiles tl = seq_tiles(a, L);
    decode_part<D, Q8, NT>(a, smem, s_bad, seq, hk, L, tl, 0, tl.count, -1);
    return;
  }
  const Range r = find_range(a);
  int seq = r.seq;
  int64_t before = r.before;
#pragma unroll 1
  for (int64_t at = r.begin; at < r.end;) {
    const int L = seq_len(a, seq, false), n = num_tiles(a, L), np = places(n, r.open);
    const int64_t rel = at - before * a.Hk;
    if (rel >= (int64_t)np * a.Hk) {  // past this sequence (also where it has no tiles)
      before += np;
      ++seq;
      continue;
    }
    const int hk = (int)(rel / np), p_begin = (int)(rel - (int64_t)hk * np);
    const int p_end = (int)min((int64_t)np, p_begin + (r.end - at));
    const int t_begin = max(p_begin - r.open, 0), t_end = max(p_end - r.open, 0);
    if (t_end > t_begin) {
      // a part of a list is the range's first (slot 0) or, where its list begins, last (1)
      const int64_t slot = t_begin == 0 && t_end == n
                               ? -1
                               : 2 * (int64_t)blockIdx.x + (t_begin == 0 ? 1 : 0);
      decode_part<D, Q8, NT>(a, smem, s_bad, seq, hk, L, seq_tiles(a, L), t_begin, t_end, slot);
      __syncthreads();  // the merged sums have been read
    }
    at += p_end - p_begin;
  }
}

// Merges the parts of a (sequence, query head) that lies in more than one range, in an
// order that only the lengths set: a CTA per pair, warp w takes parts w, w + 4, ..., each
// lane D / 32 of the values, then the warps' sums are added in warp order.
template <int D>
__global__ void __launch_bounds__(128) window_decode_merge_kernel(const Args a) {
  constexpr int E = D / 32;
  __shared__ float s_acc[4][D], s_l[4];
  va::pdl_enter();
  const int seq = blockIdx.x, h = blockIdx.y;
  const int n = num_tiles(a, seq_len(a, seq, false));
  if (n == 0) return;
  const int kvh = h / a.G, j = (h - kvh * a.G) / a.gc, hl = h - kvh * a.G - j * a.gc;
  const int64_t width = a.ws_plan[0];
  const int open = (int)a.ws_plan[1];
  const int64_t first =  // place of the pair's first tile
      a.ws_plan[2 + seq] * a.Hk + (int64_t)(kvh * a.hg + j) * places(n, open) + open;
  const int64_t c0 = first / width;
  const int nsplit = (int)((first + n - 1) / width - c0) + 1;
  if (nsplit == 1) return;  // written whole
  // the pair's first part is the last of its range (slot 1), the others their range's first
  auto part = [&](int s) -> int64_t { return (2 * (c0 + s) + (s == 0 ? 1 : 0)) * a.gc + hl; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // every warp finds the common maximum, 32 ranges at a time
  float M = kLowest;
  bool skip = false;
  for (int s = lane; s < nsplit; s += 32) {
    const float2 v = a.ws_ml[part(s)];
    skip = skip || v.y < 0.f;
    M = fmaxf(M, v.x);
  }
  if (__any_sync(0xffffffffu, skip)) return;  // uniform: every warp sees every range
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
  float A[E], Ls = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) A[e] = 0.f;
#pragma unroll 8
  for (int s = warp; s < nsplit; s += 4) {
    const int64_t p = part(s);
    const float2 v = a.ws_ml[p];
    const float f = va::fast_exp2(v.x - M);
    Ls = fmaf(v.y, f, Ls);
#pragma unroll
    for (int e = 0; e < E; ++e)
      A[e] = fmaf(a.ws_acc[p * D + e * 32 + lane], f, A[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_acc[warp][e * 32 + lane] = A[e];
  if (lane == 0) s_l[warp] = Ls;
  __syncthreads();
  const int d = threadIdx.x;
  if (d < D) {
    const float acc = (s_acc[0][d] + s_acc[1][d]) + (s_acc[2][d] + s_acc[3][d]);
    const float sum = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    a.out[seq * a.o_s_token + (int64_t)h * a.o_s_head + d] = __float2half_rn(acc / sum);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct Plan {
  int gc, hg, most;  // most: ranges, 0 where every (sequence, head group) has its own CTA
  size_t o_ml, o_plan, total;
};

// CTAs per SM that the workspace is sized for (the kernels fit 2 to 4).
constexpr int kMaxPerSm = 4;

// Head groups of up to 16.  All tiles of the call are one list that is cut into equal
// ranges, one per CTA that fits the GPU at once: one even wave, whatever the lengths.
// Two cases gain nothing from the cut, its search and its merge kernel.  Sequences of at most
// 40 tiles, which a CTA reads in about that time: 1 to 128 sequences of up to 600 keys, of one
// length or ragged, take 0.40 to 0.99 of the time cut; of 800 keys 0.72 to 1.18, of 1200 0.84
// to 1.44.  And so many lists that whole ones balance, ragged ones too, and a CTA that ends
// makes room for the next one's copies: up to 8192 tokens ragged, fp16 / e4m3 heads of 128,
// 512 lists 1.20 / 1.33 of the time cut, 1024 1.03 / 1.15, 2048 0.96 / 1.01, 2560 0.95 / 0.99,
// 4096 0.93 / 0.96, 8192 (1024 sequences of 8 kv heads) 2385 us for 2616 and 1382 for 1506.
Plan make_plan(int64_t num_seqs, int Hq, int Hkv, int D, int64_t max_len, int window, int sinks) {
  Plan p{};
  const int G = Hq / Hkv;
  p.hg = (G + 15) / 16;
  p.gc = (G + p.hg - 1) / p.hg;
  window = win::window_of(window);
  sinks = win::sinks_of(sinks);
  int64_t keys = max_len;
  if (window > 0 && (int64_t)window + sinks < keys) keys = (int64_t)window + sinks;
  // an unaligned run and the sinks each reach into one more tile
  const int64_t tiles = (keys + kKeys - 1) / kKeys + 2;
  const int64_t units = num_seqs * Hkv * p.hg, slots = (int64_t)kMaxPerSm * va_host::sm_count();
  if (tiles <= 5 * kMinRange || units >= 4 * slots) return p;
  const int64_t most = units * ((tiles + kOpenMost + kMinRange - 1) / kMinRange);
  p.most = (int)(most < slots ? most : slots);
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  p.o_ml = up((size_t)p.most * 2 * p.gc * D * 4);
  p.o_plan = p.o_ml + up((size_t)p.most * 2 * p.gc * 8);
  p.total = p.o_plan + up((size_t)(num_seqs + 2) * 8);
  return p;
}

template <int D, bool Q8, int NT>
int launch_t(Args &a, cudaStream_t st) {
  constexpr int merge = kNW * 8 * NT * (Shape<D, Q8>::kHead + 2) * 4;
  constexpr int smem = Shape<D, Q8>::kRing > merge ? Shape<D, Q8>::kRing : merge;
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> per_sm{0};
  if (!win::allow_smem(window_decode_kernel<D, Q8, NT>, smem, done)) return VA_ERR_LAUNCH;
  int64_t grid = (int64_t)a.B * a.Hk;
  if (a.ranges) {
    int n = per_sm.load(std::memory_order_relaxed);
    if (!n) {
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, window_decode_kernel<D, Q8, NT>,
                                                        kNW * 32, smem) != cudaSuccess ||
          n < 1)
        return VA_ERR_LAUNCH;
      per_sm.store(n = n < kMaxPerSm ? n : kMaxPerSm, std::memory_order_relaxed);
    }
    const int fit = n * va_host::sm_count();
    if (fit < a.ranges) a.ranges = fit;
    grid = a.ranges;
  }
  if (va_host::launch_pdl_smem(window_decode_kernel<D, Q8, NT>, (unsigned)grid, kNW * 32, smem, st,
                               a))
    return VA_ERR_LAUNCH;
  if (a.ranges && va_host::launch_pdl(window_decode_merge_kernel<D>,
                                      dim3((unsigned)a.B, (unsigned)a.Hq), 128, st, a))
    return VA_ERR_LAUNCH;
  return va_host::launch_status();
}

template <int D>
int launch_d(bool q8, Args &a, cudaStream_t st) {
  if (q8) return a.gc <= 8 ? launch_t<D, true, 1>(a, st) : launch_t<D, true, 2>(a, st);
  return a.gc <= 8 ? launch_t<D, false, 1>(a, st) : launch_t<D, false, 2>(a, st);
}

}  // namespace

extern "C" size_t va_window_decode_workspace_size(int64_t num_seqs, int num_query_heads,
                                                  int num_kv_heads, int head_size,
                                                  int64_t max_seq_len, int window,
                                                  int sink_tokens) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || num_query_heads <= 0 || head_size <= 0 ||
      num_query_heads % num_kv_heads || max_seq_len <= 0 || sink_tokens < 0)
    return 0;
  return make_plan(num_seqs, num_query_heads, num_kv_heads, head_size, max_seq_len, window,
                   sink_tokens)
      .total;
}

extern "C" int va_window_decode(void *out, const void *q, void *k_cache, void *v_cache,
                                void *k_scale, void *v_scale, int kv_e4m3,
                                const int32_t *block_table, const int32_t *seq_lens,
                                const void *new_k, const void *new_v, int64_t num_seqs,
                                int num_query_heads, int num_kv_heads, int head_size,
                                int block_size, int64_t max_blocks_per_seq, int64_t max_seq_len,
                                int64_t num_blocks, float scale, int window, int sink_tokens,
                                int64_t s_block, int64_t s_head, int64_t s_token,
                                int64_t sc_block, int64_t sc_head, int64_t sc_token,
                                int64_t q_s_token, int64_t q_s_head, int64_t o_s_token,
                                int64_t o_s_head, int64_t new_s_token, int64_t new_s_head,
                                void *workspace, size_t workspace_bytes, int32_t *err_flag,
                                void *stream) {
  if (num_seqs < 0 || max_seq_len < 0 || num_blocks < 0 || max_blocks_per_seq < 0 ||
      sink_tokens < 0 || !win::scale_ok(scale))
    return VA_ERR_INVALID_ARG;
  if (num_kv_heads <= 0 || num_query_heads <= 0 || num_query_heads % num_kv_heads ||
      block_size <= 0)
    return VA_ERR_INVALID_ARG;
  if (num_seqs == 0 || max_seq_len == 0) return VA_OK;
  if (!out || !q || !k_cache || !v_cache || !block_table || !seq_lens ||
      (kv_e4m3 && (!k_scale || !v_scale)) || (new_k == nullptr) != (new_v == nullptr))
    return VA_ERR_INVALID_ARG;
  if (!win::head_size_ok(head_size) || num_seqs > 65535) return VA_ERR_UNSUPPORTED;
  if (max_seq_len > INT32_MAX / 2) return VA_ERR_UNSUPPORTED;
  if (!va_host::aligned16(k_cache) || !va_host::aligned16(v_cache) ||
      !win::strides_ok(kv_e4m3, s_block, s_head, s_token) ||
      !win::rows_ok(q, q_s_token, q_s_head) || (reinterpret_cast<uintptr_t>(out) & 1))
    return VA_ERR_INVALID_ARG;
  if (new_k && (!win::rows_ok(new_k, new_s_token, new_s_head) || !va_host::aligned16(new_v)))
    return VA_ERR_INVALID_ARG;
  const Plan p = make_plan(num_seqs, num_query_heads, num_kv_heads, head_size, max_seq_len,
                           window, sink_tokens);
  if (num_query_heads > 65535 || num_seqs * num_kv_heads * p.hg > INT32_MAX)
    return VA_ERR_UNSUPPORTED;
  if (p.total && (!workspace || workspace_bytes < p.total || !va_host::aligned16(workspace)))
    return VA_ERR_WORKSPACE;
  Args a{};
  a.out = static_cast<__half *>(out);
  a.q = static_cast<const __half *>(q);
  a.kc = static_cast<uint8_t *>(k_cache);
  a.vc = static_cast<uint8_t *>(v_cache);
  a.ks = static_cast<uint8_t *>(k_scale);
  a.vs = static_cast<uint8_t *>(v_scale);
  a.nk = static_cast<const __half *>(new_k);
  a.nv = static_cast<const __half *>(new_v);
  a.bt = block_table;
  a.sl = seq_lens;
  if (p.total) {
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    a.ws_acc = reinterpret_cast<float *>(ws);
    a.ws_ml = reinterpret_cast<float2 *>(ws + p.o_ml);
    a.ws_plan = reinterpret_cast<int64_t *>(ws + p.o_plan);
  }
  a.err = err_flag;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = num_blocks;
  a.max_len = max_seq_len;
  a.Hq = num_query_heads;
  a.G = num_query_heads / num_kv_heads;
  a.hg = p.hg;
  a.gc = p.gc;
  a.bs = win::fast_div(block_size);
  a.window = win::window_of(window);
  a.sinks = win::sinks_of(sink_tokens);
  a.ranges = p.most;
  a.B = (int)num_seqs;
  a.Hk = num_kv_heads * p.hg;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.s_block = s_block; a.s_head = s_head; a.s_token = s_token;
  a.c_block = sc_block; a.c_head = sc_head; a.c_token = sc_token;
  a.q_s_token = q_s_token; a.q_s_head = q_s_head;
  a.o_s_token = o_s_token; a.o_s_head = o_s_head;
  a.n_s_token = new_s_token; a.n_s_head = new_s_head;
  auto st = static_cast<cudaStream_t>(stream);
  switch (head_size) {
    case 32: return launch_d<32>(kv_e4m3 != 0, a, st);
    case 64: return launch_d<64>(kv_e4m3 != 0, a, st);
    case 96: return launch_d<96>(kv_e4m3 != 0, a, st);
    case 128: return launch_d<128>(kv_e4m3 != 0, a, st);
  }
  return VA_ERR_UNSUPPORTED;
}

// The 8-bit KV cache: rows quantised as they are written, and read back to fp16.
// (Row format and its reasons: kv_q8.cuh.)
//
// Both kernels move each byte once and are bound by HBM, small calls by the launch.
#include "window.cuh"

namespace {

constexpr int kThreads = 128;

// ---------------------------------------------------------------------------
// write: fp16 rows -> codes + exponent byte, scattered by slot
// ---------------------------------------------------------------------------
struct QWriteArgs {
  uint8_t *kc, *vc, *ks, *vs;
  const __half *nk, *nv;
  const void *slots;
  int slot64;
  win::FastDiv heads, bs;
  int64_t rows, num_slots;  // rows = tokens * heads
  int64_t s_block, s_head, s_token, c_block, c_head, c_token, n_token, n_head;
  int32_t *err;
};

// A group of L lanes owns one (token, head): every lane takes 8 values (16 bytes) of the
// K row and of the V row, so a row is read once, its maximum is a shuffle reduction and
// the codes never leave registers.  head_size 96 leaves 4 of 16 lanes idle.  16384 rows of
// 8 heads of 128 take 19.0 us (5.3 TB/s), 64 rows of 2 heads of 64 1.7 us, a launch.  A group takes
// kPair rows at a time and reads them without waiting for their slots (rows of padding are
// read too), so that one latency covers slots and rows.
template <int D>
__global__ void __launch_bounds__(kThreads) kv_quant_write_kernel(const QWriteArgs a) {
  constexpr int L = D > 64 ? 16 : D / 8, kPair = 2;
  constexpr int kRowsCta = kThreads / L * kPair;
  va::pdl_enter();
  const int sub = threadIdx.x % L;
  const bool on = sub * 8 < D;
  for (int64_t row0 = (int64_t)blockIdx.x * kRowsCta; row0 < a.rows;
       row0 += (int64_t)gridDim.x * kRowsCta) {
    int64_t slot[kPair];
    int head[kPair];
    uint4 k[kPair], v[kPair];
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      const int64_t row = row0 + u * (kThreads / L) + threadIdx.x / L;
      slot[u] = -1;
      k[u] = v[u] = make_uint4(0, 0, 0, 0);
      if (row >= a.rows) continue;
      const int64_t tok = a.rows <= INT32_MAX ? a.heads.div((int)row) : row / a.heads.d;
      head[u] = (int)(row - tok * a.heads.d);
      slot[u] = a.slot64 ? __ldg(static_cast<const int64_t *>(a.slots) + tok)
                         : (int64_t)__ldg(static_cast<const int32_t *>(a.slots) + tok);
      if (on) {
        const int64_t src = tok * a.n_token + (int64_t)head[u] * a.n_head + sub * 8;
        k[u] = __ldcs(reinterpret_cast<const uint4 *>(a.nk + src));
        v[u] = __ldcs(reinterpret_cast<const uint4 *>(a.nv + src));
      }
    }
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      auto absmax = [](const uint4 &w) {
        const uint32_t m = va::q8_absmax2(
            va::q8_absmax2(va::q8_absmax2(va::q8_absmax2(0, w.x), w.y), w.z), w.w);
        return max(m & 0xffffu, m >> 16);
      };
      // one 16-bit maximum each, K in the low half and V in the high half
      uint32_t m = absmax(k[u]) | absmax(v[u]) << 16;
#pragma unroll
      for (int o = 1; o < L; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
      // an infinity or a NaN in some row of the warp: the finite maxima
      if (__any_sync(0xffffffffu, __vcmpgeu2(m, 0x7c007c00u))) {
        auto finite = [](const uint4 &w) {
          const uint32_t m = va::q8_absmax2_finite(
              va::q8_absmax2_finite(va::q8_absmax2_finite(va::q8_absmax2_finite(0, w.x), w.y), w.z),
              w.w);
          return max(m & 0xffffu, m >> 16);
        };
        m = finite(k[u]) | finite(v[u]) << 16;
#pragma unroll
        for (int o = 1; o < L; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
      }
      if (slot[u] < 0 || slot[u] >= a.num_slots) {
        if (slot[u] != -1 && head[u] == 0 && sub == 0) va::raise_flag(a.err, VA_FLAG_BAD_SLOT);
        continue;
      }
      const int ek = va::q8_exponent(m & 0xffffu), ev = va::q8_exponent(m >> 16);
      const uint32_t ik = va::q8_inv_h2(ek), iv = va::q8_inv_h2(ev);
      const int64_t blk =
          a.num_slots <= INT32_MAX ? a.bs.div((int)slot[u]) : slot[u] / a.bs.d;
      const int64_t off = slot[u] - blk * a.bs.d;
      if (on) {
        const int64_t dst = blk * a.s_block + head[u] * a.s_head + off * a.s_token + sub * 8;
        const uint2 ck = make_uint2(va::q8_encode4(k[u].x, k[u].y, ik),
                                    va::q8_encode4(k[u].z, k[u].w, ik));
        const uint2 cv = make_uint2(va::q8_encode4(v[u].x, v[u].y, iv),
                                    va::q8_encode4(v[u].z, v[u].w, iv));
        *reinterpret_cast<uint2 *>(a.kc + dst) = ck;
        *reinterpret_cast<uint2 *>(a.vc + dst) = cv;
      }
      if (sub == 0) {
        const int64_t c = blk * a.c_block + head[u] * a.c_head + off * a.c_token;
        a.ks[c] = (uint8_t)(ek + va::kQ8ExpBias);
        a.vs[c] = (uint8_t)(ev + va::kQ8ExpBias);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// read: active blocks -> fp16 cache
// ---------------------------------------------------------------------------
struct QReadArgs {
  const uint8_t *kc, *vc, *ks, *vs;
  __half *dk, *dv;
  const int32_t *bt, *dbt, *sl;
  win::FastDiv inner, rows_blk;  // rows of the inner axis, rows of a block
  int head_minor;      // heads are the inner axis (rows of one token lie together)
  int bs, bpu, parts;  // blocks per unit, or units per block
  int64_t num_seqs, max_blocks, units_per_seq, src_nb, dst_nb;
  int64_t s_block, s_head, s_token, c_block, c_head, c_token, d_block, d_head, d_token;
  int32_t *err;
};

// A CTA takes `bpu` consecutive blocks of one sequence (or one of `parts` parts of a block)
// and walks them in pieces of 16 codes in the order the source stores them, one piece of K
// and the same piece of V per thread and step, two steps unrolled.  Eight small CTAs on an SM
// keep enough in flight: a batch of 64 contexts with 1.69 GB to move takes 272 us, against 284
// us with five CTAs of 256 threads, 331 us with four steps unrolled (80 registers, 3 CTAs).
template <int D>
__global__ void __launch_bounds__(kThreads, 8) kv_dequant_kernel(const QReadArgs a) {
  constexpr int P = D / 16;  // pieces per row
  va::pdl_enter();
  const int64_t units = a.num_seqs * a.units_per_seq;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t seq = u / a.units_per_seq, v = u - seq * a.units_per_seq;
    const int64_t g = a.parts > 1 ? v / a.parts : v;
    const int part = (int)(v - g * a.parts);
    const int64_t b0 = g * a.bpu, n = __ldg(a.sl + seq);
    if (n <= b0 * a.bs) continue;
    const int64_t nblk = (n + a.bs - 1) / a.bs;
    if (nblk > a.max_blocks) {
      if (v == 0 && threadIdx.x == 0) va::raise_flag(a.err, VA_FLAG_CTX_OVERFLOW);
      continue;
    }
    const int rows = (int)min((int64_t)a.bpu, nblk - b0) * (int)a.rows_blk.d;
#pragma unroll 2
    for (int i = threadIdx.x + part * kThreads; i < rows * P; i += kThreads * a.parts) {
      const int r = i / P, c = i - r * P;
      const int b = a.rows_blk.div(r), rb = r - b * (int)a.rows_blk.d;
      const int outer = a.inner.div(rb), in = rb - outer * (int)a.inner.d;
      const int h = a.head_minor ? in : outer, t = a.head_minor ? outer : in;
      if ((b0 + b) * a.bs + t >= n) continue;
      const int64_t e = seq * a.max_blocks + b0 + b;
      const int32_t sb = __ldg(a.bt + e), db = a.dbt ? __ldg(a.dbt + e) : sb;
      if (sb < 0 || sb >= a.src_nb || db < 0 || db >= a.dst_nb) {
        if (rb == 0 && c == 0) va::raise_flag(a.err, VA_FLAG_BAD_BLOCK);
        continue;
      }
      const int64_t src = sb * a.s_block + h * a.s_head + t * a.s_token + c * 16;
      const int64_t sc = sb * a.c_block + h * a.c_head + t * a.c_token;
      const uint4 k = __ldcs(reinterpret_cast<const uint4 *>(a.kc + src));
      const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(a.vc + src));
      const uint32_t fk = __ldg(a.ks + sc), fv = __ldg(a.vs + sc);
      const int64_t dst = db * a.d_block + h * a.d_head + t * a.d_token + c * 16;
      auto put = [](__half *p, const uint4 &w, uint32_t f) {
        uint4 lo, hi;
        va::q8_decode4(w.x, lo.x, lo.y);
        va::q8_decode4(w.y, lo.z, lo.w);
        va::q8_decode4(w.z, hi.x, hi.y);
        va::q8_decode4(w.w, hi.z, hi.w);
        lo = make_uint4(va::hmul2(lo.x, f), va::hmul2(lo.y, f), va::hmul2(lo.z, f),
                        va::hmul2(lo.w, f));
        hi = make_uint4(va::hmul2(hi.x, f), va::hmul2(hi.y, f), va::hmul2(hi.z, f),
                        va::hmul2(hi.w, f));
        __stcs(reinterpret_cast<uint4 *>(p), lo);
        __stcs(reinterpret_cast<uint4 *>(p) + 1, hi);
      };
      put(a.dk + dst, k, va::q8_scale_h2(fk));
      put(a.dv + dst, w, va::q8_scale_h2(fv));
    }
  }
}

bool head_size_ok(int D) { return D == 32 || D == 64 || D == 96 || D == 128; }
bool mult(int64_t s, int64_t m) { return s % m == 0; }

}  // namespace

extern "C" int va_kv_quant_write_slots(void *k_cache, void *v_cache, void *k_scale, void *v_scale,
                                       const void *new_k, const void *new_v,
                                       const void *slot_mapping, int slot_is_i64,
                                       int64_t num_tokens, int num_kv_heads, int head_size,
                                       int block_size, int64_t num_blocks, int64_t s_block,
                                       int64_t s_head, int64_t s_token, int64_t sc_block,
                                       int64_t sc_head, int64_t sc_token, int64_t new_s_token,
                                       int64_t new_s_head, int32_t *err_flag, void *stream) {
  if (num_tokens < 0 || num_blocks < 0 || num_kv_heads <= 0 || block_size <= 0)
    return VA_ERR_INVALID_ARG;
  if (num_tokens == 0) return VA_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !new_k || !new_v || !slot_mapping)
    return VA_ERR_INVALID_ARG;
  if (!head_size_ok(head_size)) return VA_ERR_UNSUPPORTED;
  if (num_tokens > (INT64_MAX >> 16) / num_kv_heads) return VA_ERR_UNSUPPORTED;
  if (!va_host::aligned16(k_cache) || !va_host::aligned16(v_cache) ||
      !va_host::aligned16(new_k) || !va_host::aligned16(new_v) || !mult(s_block, 16) ||
      !mult(s_head, 16) || !mult(s_token, 16) || !mult(new_s_token, 8) || !mult(new_s_head, 8))
    return VA_ERR_INVALID_ARG;
  QWriteArgs a{};
  a.kc = static_cast<uint8_t *>(k_cache);
  a.vc = static_cast<uint8_t *>(v_cache);
  a.ks = static_cast<uint8_t *>(k_scale);
  a.vs = static_cast<uint8_t *>(v_scale);
  a.nk = static_cast<const __half *>(new_k);
  a.nv = static_cast<const __half *>(new_v);
  a.slots = slot_mapping;
  a.slot64 = slot_is_i64;
  a.heads = win::fast_div(num_kv_heads);
  a.bs = win::fast_div(block_size);
  a.rows = num_tokens * num_kv_heads;
  a.num_slots = num_blocks * block_size;
  a.s_block = s_block; a.s_head = s_head; a.s_token = s_token;
  a.c_block = sc_block; a.c_head = sc_head; a.c_token = sc_token;
  a.n_token = new_s_token; a.n_head = new_s_head;
  a.err = err_flag;
  const int per = 2 * kThreads / (head_size > 64 ? 16 : head_size / 8);  // rows of a CTA
  const int64_t want = (a.rows + per - 1) / per;
  const dim3 grid((unsigned)(want < (1 << 20) ? want : (1 << 20)));
  auto st = static_cast<cudaStream_t>(stream);
  int rc = 1;
  switch (head_size) {
    case 32: rc = va_host::launch_pdl(kv_quant_write_kernel<32>, grid, kThreads, st, a); break;
    case 64: rc = va_host::launch_pdl(kv_quant_write_kernel<64>, grid, kThreads, st, a); break;
    case 96: rc = va_host::launch_pdl(kv_quant_write_kernel<96>, grid, kThreads, st, a); break;
    case 128: rc = va_host::launch_pdl(kv_quant_write_kernel<128>, grid, kThreads, st, a); break;
  }
  return rc ? VA_ERR_LAUNCH : va_host::launch_status();
}

extern "C" int va_kv_dequant_blocks(const void *src_k, const void *src_v, const void *k_scale,
                                    const void *v_scale, void *dst_k, void *dst_v,
                                    const int32_t *block_table, const int32_t *dst_block_table,
                                    const int32_t *seq_lens, int64_t num_seqs,
                                    int64_t max_blocks_per_seq, int num_kv_heads, int head_size,
                                    int block_size, int64_t src_num_blocks,
                                    int64_t dst_num_blocks, int64_t src_s_block,
                                    int64_t src_s_head, int64_t src_s_token, int64_t sc_block,
                                    int64_t sc_head, int64_t sc_token, int64_t dst_s_block,
                                    int64_t dst_s_head, int64_t dst_s_token, int32_t *err_flag,
                                    void *stream) {
  if (num_seqs < 0 || max_blocks_per_seq < 0 || src_num_blocks < 0 || dst_num_blocks < 0 ||
      num_kv_heads <= 0 || block_size <= 0)
    return VA_ERR_INVALID_ARG;
  if (num_seqs == 0 || max_blocks_per_seq == 0) return VA_OK;
  if (!src_k || !src_v || !k_scale || !v_scale || !dst_k || !dst_v || !block_table || !seq_lens)
    return VA_ERR_INVALID_ARG;
  if (!head_size_ok(head_size)) return VA_ERR_UNSUPPORTED;
  // one block's pieces are counted in 32 bits
  if ((int64_t)num_kv_heads * block_size > (1 << 24)) return VA_ERR_UNSUPPORTED;
  if (num_seqs > INT32_MAX || max_blocks_per_seq > INT32_MAX) return VA_ERR_UNSUPPORTED;
  if (!va_host::aligned16(src_k) || !va_host::aligned16(src_v) || !va_host::aligned16(dst_k) ||
      !va_host::aligned16(dst_v) || !mult(src_s_block, 16) || !mult(src_s_head, 16) ||
      !mult(src_s_token, 16) || !mult(dst_s_block, 8) || !mult(dst_s_head, 8) ||
      !mult(dst_s_token, 8))
    return VA_ERR_INVALID_ARG;
  QReadArgs a{};
  a.kc = static_cast<const uint8_t *>(src_k);
  a.vc = static_cast<const uint8_t *>(src_v);
  a.ks = static_cast<const uint8_t *>(k_scale);
  a.vs = static_cast<const uint8_t *>(v_scale);
  a.dk = static_cast<__half *>(dst_k);
  a.dv = static_cast<__half *>(dst_v);
  a.bt = block_table;
  a.dbt = dst_block_table;
  a.sl = seq_lens;
  a.head_minor = src_s_head < src_s_token ? 1 : 0;
  a.inner = win::fast_div(a.head_minor ? num_kv_heads : block_size);
  a.rows_blk = win::fast_div(num_kv_heads * block_size);
  a.bs = block_size;
  a.num_seqs = num_seqs;
  a.max_blocks = max_blocks_per_seq;
  a.src_nb = src_num_blocks;
  a.dst_nb = dst_num_blocks;
  a.s_block = src_s_block; a.s_head = src_s_head; a.s_token = src_s_token;
  a.c_block = sc_block; a.c_head = sc_head; a.c_token = sc_token;
  a.d_block = dst_s_block; a.d_head = dst_s_head; a.d_token = dst_s_token;
  a.err = err_flag;
  // a unit is at least one step of the CTA; blocks larger than that are cut into parts while
  // the units are few (up to 4 for every CTA that the GPU holds at once)
  const int64_t pieces = (int64_t)num_kv_heads * block_size * (head_size / 16);
  const int64_t bpu = kThreads / pieces;
  a.bpu = (int)(bpu < 1 ? 1 : bpu);
  a.units_per_seq = (max_blocks_per_seq + a.bpu - 1) / a.bpu;
  const int64_t room = 4 * 8 * (int64_t)va_host::sm_count();
  a.parts = 1;
  while (a.parts * 2 * kThreads <= pieces && num_seqs * a.units_per_seq * a.parts * 2 <= room)
    a.parts *= 2;
  a.units_per_seq *= a.parts;
  const int64_t units = num_seqs * a.units_per_seq;
  const dim3 grid((unsigned)(units < (1 << 20) ? units : (1 << 20)));
  auto st = static_cast<cudaStream_t>(stream);
  int rc = 1;
  switch (head_size) {
    case 32: rc = va_host::launch_pdl(kv_dequant_kernel<32>, grid, kThreads, st, a); break;
    case 64: rc = va_host::launch_pdl(kv_dequant_kernel<64>, grid, kThreads, st, a); break;
    case 96: rc = va_host::launch_pdl(kv_dequant_kernel<96>, grid, kThreads, st, a); break;
    case 128: rc = va_host::launch_pdl(kv_dequant_kernel<128>, grid, kThreads, st, a); break;
  }
  return rc ? VA_ERR_LAUNCH : va_host::launch_status();
}

// Shared rules of the windowed attention kernels (window_decode.cu, window_prefill.cu).
//
// A query at position p sees the keys j <= p with p - j < window (window <= 0: all of
// them) or j < sinks.  The keys it reads are therefore one run [lo, p] with
// lo = max(0, p - window + 1), and the first min(sinks, lo) keys before it.  Both
// kernels walk that as a list of key tiles: the tiles that hold the sinks, then the
// tiles of the run that are not among them.  Blocks that hold no visible key are never
// read, so their block-table entries may hold anything (a freed block, -1).
#pragma once

#include <atomic>

#include "kv_q8.cuh"

namespace win {

// The tiles of `size` keys that hold the keys visible to at least one query position
// in [first, last] (0 <= first <= last).
struct Tiles {
  int sinks;  // tiles 0..sinks-1 hold the sinks before the run
  int start;  // first tile of the run
  int count;  // tiles in all
};
VA_DEVINL int run_start(int first, int window) {
  return window > 0 && first >= window ? first - window + 1 : 0;
}
VA_DEVINL Tiles key_tiles(int first, int last, int window, int sinks, int size) {
  const int lo = run_start(first, window);
  Tiles t;
  t.sinks = (min(sinks, lo) + size - 1) / size;
  t.start = max(t.sinks, lo / size);
  t.count = t.sinks + last / size + 1 - t.start;
  return t;
}
VA_DEVINL int tile_at(const Tiles &t, int i) { return i < t.sinks ? i : t.start + i - t.sinks; }

// Division of keys (0 <= n < 2^31) by a block size that is only known at launch, as one
// multiplication by m = ceil(2^(32 + sh) / d), where 2^sh < d <= 2^(sh + 1).
//   * 2^sh < d, so m is below 2^32 and fits its field.
//   * m d - 2^(32 + sh) < d, so n m / 2^(32 + sh) exceeds n / d by less than n / 2^(32 + sh).
//     That is less than 1 / d, since n d < 2^31 2^(sh + 1): the floor is n / d's.
struct FastDiv {
  uint32_t d, m, sh;
  VA_DEVINL int div(int n) const {
    if (d == 1) return n;
    return (int)(__umulhi((uint32_t)n, m) >> sh);
  }
  VA_DEVINL int mod(int n) const { return n - div(n) * (int)d; }
};
inline FastDiv fast_div(int d) {
  FastDiv f{};
  f.d = (uint32_t)d;
  if (d > 1) {
    uint32_t sh = 0;  // ceil(log2 d) - 1
    while ((uint64_t(2) << sh) < (uint64_t)d) ++sh;
    f.sh = sh;
    f.m = (uint32_t)(((uint64_t(1) << (32 + sh)) + d - 1) / d);
  }
  return f;
}

// Asynchronous copy of V bytes, or V zero bytes where `on` is false (the source is not
// read then).
template <int V>
VA_DEVINL void cp_async_zfill(uint32_t dst, const void *src, bool on) {
  const uint32_t n = on ? V : 0;
  if constexpr (V == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(V),
                 "r"(n)
                 : "memory");
}
template <int V>
VA_DEVINL void cp_async(uint32_t dst, const void *src) {
  if constexpr (V == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(V)
                 : "memory");
}
VA_DEVINL void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
VA_DEVINL void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Strides and bounds that every windowed entry point checks the same way: cache rows and
// query/output rows start on 16-byte boundaries.
inline bool strides_ok(int kv_q8, int64_t s_block, int64_t s_head, int64_t s_token) {
  const int64_t m = kv_q8 ? 16 : 8;
  return s_block % m == 0 && s_head % m == 0 && s_token % m == 0;
}
inline bool rows_ok(const void *p, int64_t s_token, int64_t s_head) {
  return va_host::aligned16(p) && s_token % 8 == 0 && s_head % 8 == 0;
}
inline bool head_size_ok(int D) { return D == 32 || D == 64 || D == 96 || D == 128; }
// Positions stay below INT32_MAX / 2, so a window past that is none.
inline int window_of(int window) { return window > 0 && window < INT32_MAX / 2 ? window : 0; }
inline int sinks_of(int sinks) { return sinks < INT32_MAX / 2 ? sinks : INT32_MAX / 2; }
// Opts a kernel in to `bytes` of dynamic shared memory, once per device (bit d of `done`;
// two threads setting it at once is harmless).
template <typename K>
bool allow_smem(K kernel, int bytes, std::atomic<uint64_t> &done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
      cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_release);
  return true;
}
inline bool scale_ok(float s) { return s > 0.f && s <= 3.402823466e38f; }

}  // namespace win

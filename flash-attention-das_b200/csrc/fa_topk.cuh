// Choice of the k largest of a row's values by one CTA, ties to the lowest index: the border value by a radix search
// over order-preserving integer keys (one histogram of 8 bits of the key per pass), then the chosen indices in
// ascending order.  Integer counts only, so the result does not depend on the order in which threads run.
#pragma once

#include "fa_common.cuh"

namespace fa {

// Keys that compare as the values do: -0 equals +0 and every NaN is above +inf.  ~0 is above every value's key.
__device__ __forceinline__ uint32_t order_key(float x) {
  uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) u = 0x7fc00000u;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double x) {
  uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
  if ((u & 0x7fffffffffffffffull) > 0x7ff0000000000000ull) u = 0x7ff8000000000000ull;
  if (u == 0x8000000000000000ull) u = 0ull;
  return (u & 0x8000000000000000ull) ? ~u : (u | 0x8000000000000000ull);
}

struct TopkShared {
  int hist[256];
  int bin, above;
  int warp_total[32];
};

// Border of the `want` largest of key(0) .. key(n - 1), 1 <= want <= n: all keys above the returned one belong to them,
// and the first `take_equal` (by index) of those equal to it.
template <int THREADS, class Key, class KeyAt>
__device__ __forceinline__ Key topk_border(int n, int want, KeyAt key, TopkShared& sh, int& take_equal) {
  const int tid = threadIdx.x, lane = tid & 31;
  Key prefix = 0, mask = 0;
  for (int shift = static_cast<int>(sizeof(Key)) * 8 - 8; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) sh.hist[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += THREADS) {
      const int i = i0 + tid;
      int digit = 256;
      if (i < n) {
        const Key x = key(i);
        if ((x & mask) == prefix) digit = static_cast<int>((x >> shift) & 255);
      }
      // values of one row share their leading bits: count equal digits of a warp with one atomic
      const uint32_t peers = __match_any_sync(0xffffffffu, digit);
      if (digit < 256 && lane == __ffs(peers) - 1) atomicAdd(&sh.hist[digit], __popc(peers));
    }
    __syncthreads();
    if (tid < 32) {   // lane l looks at digits 255 - 8 l .. 248 - 8 l
      int own[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) { own[j] = sh.hist[255 - 8 * lane - j]; sum += own[j]; }
      int upto = sum;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, upto, s);
        if (lane >= s) upto += t;
      }
      int above = upto - sum;
      if (above < want && want <= upto) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (above < want && want <= above + own[j]) { sh.bin = 255 - 8 * lane - j; sh.above = above; }
          above += own[j];
        }
      }
    }
    __syncthreads();
    prefix |= static_cast<Key>(sh.bin) << shift;
    mask |= static_cast<Key>(255) << shift;
    want -= sh.above;
    __syncthreads();
  }
  take_equal = want;
  return prefix;
}

// Calls emit(position, i) for the chosen indices i in ascending order (position 0, 1, ..) and rest(i) for the others.
// emit's reads of a chunk's values are the caller's business: `chunk_sync` barriers separate the chunks.
template <int THREADS, class Key, class KeyAt, class Emit>
__device__ __forceinline__ void topk_emit(int n, Key border, int take_equal, KeyAt key, TopkShared& sh, Emit emit) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base_gt = 0, base_eq = 0;
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + tid;
    bool gt = false, eq = false;
    if (i < n) {
      const Key x = key(i);
      gt = x > border;
      eq = x == border;
    }
    const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) sh.warp_total[warp] = __popc(bg) | (__popc(be) << 16);
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      const int t = sh.warp_total[w];
      if (w < warp) before += t;
      total += t;
    }
    const uint32_t below = (1u << lane) - 1u;
    const int n_gt = base_gt + (before & 0xffff) + __popc(bg & below);
    const int n_eq = base_eq + (before >> 16) + __popc(be & below);
    const bool chosen = gt || (eq && n_eq < take_equal);
    emit(chosen, n_gt + min(n_eq, take_equal), i);
    base_gt += total & 0xffff;
    base_eq += total >> 16;
    __syncthreads();
  }
}

}  // namespace fa

// Choice of the k largest of a row's values by one CTA, ties to the lowest index: the border value by a histogram search
// over order-preserving integer keys, then the chosen indices in ascending order.  Integer counts only, so the result
// does not depend on the order in which threads run.
#pragma once

#include "fa_common.cuh"

namespace fa {

// Keys that compare as the values do: -0 equals +0 and every NaN is above +inf.  ~0 is above every value's key, 0 below.
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

// The value of a key (of ~0: a NaN).
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

constexpr int kTopkBins = 1024, kTopkList = 2048;
struct TopkShared {
  int hist[kTopkBins];
  uint32_t list[kTopkList];
  int warp_total[32];
  uint32_t lo, hi;
  int sure, bin, above, in_bin, listed;
};

// Sum of x over the threads before this one; `total`: over all.
template <int THREADS>
__device__ __forceinline__ int block_exclusive(int x, TopkShared& sh, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = x;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, upto, s);
    if (lane >= s) upto += t;
  }
  __syncthreads();   // the totals of the call before have been read
  if (lane == 31) sh.warp_total[warp] = upto;
  __syncthreads();
  int w = lane < THREADS / 32 ? sh.warp_total[lane] : 0;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, w, s);
    if (lane >= s) w += t;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return (warp > 0 ? before : 0) + upto - x;
}

// Border of the `want` largest of the CTA's keys, 1 <= want <= their number: all keys above the returned one belong to
// them, and the first `take_equal` (by index) of those equal to it.  each(f) calls f(key) for the thread's share of the
// keys (0: no key; ~0: always taken).
//
// Every pass counts the keys between two bounds in kTopkBins equal steps and goes on in the step that holds the border, or
// ends when that step's keys are all wanted; once a step's keys fit a short list, the passes that follow read that.
// sure < 0: the first bounds are the smallest and largest key, so a row whose values share their leading bits costs no pass
// for them (but a look at every key first).  sure >= 0: the number of keys that are always taken; the first steps are half a
// power of two of a 32-bit value wide.
template <int THREADS, class Each>
__device__ __forceinline__ uint32_t topk_border(int want, int sure, Each each, TopkShared& sh, int& take_equal) {
  constexpr int kPer = kTopkBins / THREADS;
  static_assert(kPer * THREADS == kTopkBins, "whole bins per thread");
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t lo = 1u, hi = ~0u - 1u;
  if (tid == 0) { sh.lo = ~0u; sh.hi = 0u; sh.sure = 0; sh.bin = 0; sh.above = 0; sh.in_bin = 0; sh.listed = 0; }
  if (sure < 0) {
    lo = ~0u; hi = 0u;
    int count = 0;
    each([&](uint32_t k) {
      if (k == ~0u) ++count;
      else if (k != 0u) { lo = min(lo, k); hi = max(hi, k); }
    });
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0) {
      atomicMin(&sh.lo, lo);
      atomicMax(&sh.hi, hi);
      atomicAdd(&sh.sure, count);
    }
    __syncthreads();
    lo = sh.lo; hi = sh.hi;
    sure = sh.sure;
  }
  if (want <= sure) {
    take_equal = want;
    return ~0u;
  }
  want -= sure;
  bool listed = false;
  for (int pass = 0; pass < 5; ++pass) {   // 32 bits, ten at a time: four at most (values that change meanwhile end it too)
    const uint32_t span = hi - lo;
    const int shift = max(0, 32 - __clz(span) - 10);   // span >> shift < kTopkBins
#pragma unroll
    for (int j = 0; j < kPer; ++j) sh.hist[tid + j * THREADS] = 0;
    __syncthreads();
    auto count = [&](uint32_t k) {   // 0 and ~0 lie outside: 0 < lo, hi < ~0
      if (k - lo <= span) atomicAdd(&sh.hist[(k - lo) >> shift], 1);
    };
    if (listed) {
      for (int i = tid; i < sh.listed; i += THREADS) count(sh.list[i]);
    } else {
      each(count);
    }
    __syncthreads();
    int own[kPer], sum = 0, total;
#pragma unroll
    for (int j = 0; j < kPer; ++j) { own[j] = sh.hist[kTopkBins - 1 - (tid * kPer + j)]; sum += own[j]; }
    int above = block_exclusive<THREADS>(sum, sh, total);
    if (above < want && want <= above + sum) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (above < want && want <= above + own[j]) { sh.bin = kTopkBins - 1 - (tid * kPer + j); sh.above = above; sh.in_bin = own[j]; }
        above += own[j];
      }
    }
    __syncthreads();
    want -= sh.above;
    lo += static_cast<uint32_t>(sh.bin) << shift;
    hi = min(hi, lo + ((1u << shift) - 1u));
    if (sh.in_bin == want) {   // every key of the step (lo > 0: a key is not 0)
      take_equal = 0;
      return lo - 1u;
    }
    if (shift == 0) break;
    if (!listed && sh.in_bin <= kTopkList) {
      const uint32_t range = hi - lo;
      each([&](uint32_t k) {
        if (k - lo <= range) {
          const int at = atomicAdd(&sh.listed, 1);
          if (at < kTopkList) sh.list[at] = k;
        }
      });
      listed = true;
      __syncthreads();
    }
  }
  take_equal = want;
  return lo;
}

// Running numbers of the chosen.
struct TopkCount { int gt = 0, eq = 0; };

// The chosen among the next THREADS * V keys, V of them in a row per thread: emit(j, position) for the thread's chosen key j.
// All threads call it.
template <int THREADS, int V, class Emit>
__device__ __forceinline__ void topk_place(const uint32_t (&k)[V], uint32_t border, int take_equal, TopkCount& base, TopkShared& sh, Emit emit) {
  static_assert(THREADS * V <= 32768, "both counts fit a half word");
  int mine = 0;
  uint32_t largest = k[0];
#pragma unroll
  for (int j = 1; j < V; ++j) largest = max(largest, k[j]);
  if (largest >= border) {
#pragma unroll
    for (int j = 0; j < V; ++j) mine += (k[j] > border ? 1 : 0) | (k[j] == border && border != 0u ? 0x10000 : 0);
  }
  int total;
  const int before = block_exclusive<THREADS>(mine, sh, total);
  int n_gt = base.gt + (before & 0xffff), n_eq = base.eq + (before >> 16);
  if (mine != 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool gt = k[j] > border, eq = k[j] == border && border != 0u;
      if (gt || (eq && n_eq < take_equal)) emit(j, n_gt + min(n_eq, take_equal));
      n_gt += gt ? 1 : 0;
      n_eq += eq ? 1 : 0;
    }
  }
  base.gt += total & 0xffff;
  base.eq += total >> 16;
}

// The same border search over 64-bit keys, eight bits at a time: the rare rows whose choice 32 bits do not settle.
// each(f) calls f(key, valid) the same number of times in every thread of a warp.
template <int THREADS, class Each>
__device__ __noinline__ uint64_t topk_border64(int want, Each each, TopkShared& sh, int& take_equal) {
  const int tid = threadIdx.x, lane = tid & 31;
  uint64_t prefix = 0, mask = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) sh.hist[i] = 0;
    __syncthreads();
    each([&](uint64_t x, bool valid) {
      if (valid && (x & mask) == prefix) atomicAdd(&sh.hist[(x >> shift) & 255], 1);
    });
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
    prefix |= static_cast<uint64_t>(sh.bin) << shift;
    mask |= 255ull << shift;
    want -= sh.above;
    __syncthreads();
  }
  take_equal = want;
  return prefix;
}

}  // namespace fa

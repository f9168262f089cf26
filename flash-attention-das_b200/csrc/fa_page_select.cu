// Bounds of a paged cache's keys, and the choice of pages by them.
//
// Bounds.  lo[c] and hi[c] are the smallest and largest value of channel c among a page's keys, so for every key k of the
// page q . k = sum_c q_c k_c <= sum_c max(q_c lo_c, q_c hi_c): a bound on the score that costs one row pair per page
// instead of the page.  One warp per (page, kv head): 16-byte pieces of the rows, several rows in flight, packed 16-bit
// minimum and maximum (exact: the bounds are values of the cache).  HBM-bound for a whole prompt, a few microseconds of
// latency for the pages of one decode step.
//
// Choice.  One warp per page scores it in 64 bits (the choice has a border, and a sum in 32 bits could fall on its other
// side), then one CTA per (sequence, kv head) finds the border and writes the list.
#include "fa_topk.cuh"
#include "fa_kernels.h"

namespace fa {
namespace {

constexpr int kBoundsWarps = 4;
constexpr int kSelectThreads = 512;

template <int DT> struct Pair16;   // two 16-bit values
template <> struct Pair16<FA_B200_BF16> {
  using T = __nv_bfloat162;
  static __device__ __forceinline__ float2 to_float(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<T*>(&v)); }
};
template <> struct Pair16<FA_B200_F16> {
  using T = __half2;
  static __device__ __forceinline__ float2 to_float(uint32_t v) { return __half22float2(*reinterpret_cast<T*>(&v)); }
};
template <int DT> __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  using T = typename Pair16<DT>::T;
  T r = __hmin2_nan(*reinterpret_cast<T*>(&a), *reinterpret_cast<T*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
template <int DT> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  using T = typename Pair16<DT>::T;
  T r = __hmax2_nan(*reinterpret_cast<T*>(&a), *reinterpret_cast<T*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}

// DT: cache type; OT: type of the bounds (= DT for 16-bit caches).  A lane owns 8 channels of every row its lane group
// reads: 16 bytes of a 16-bit row, 8 of an fp8 row, whose values are compared as f16 (e4m3 and e5m2 values are f16 and
// bf16 values).
template <int DT, int OT>
__global__ void __launch_bounds__(kBoundsWarps * 32) page_bounds_kernel(const PageBoundsParams p) {
  constexpr bool kFp8 = DT == FA_B200_E4M3 || DT == FA_B200_E5M2;
  constexpr int CT = kFp8 ? FA_B200_F16 : DT;   // type of the comparisons
  constexpr int es = kFp8 ? 1 : 2;
  constexpr int U = 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kBoundsWarps + warp;   // (sequence, slot, head), heads fastest
  const int64_t items = static_cast<int64_t>(p.b) * p.slots * p.h_k;
  if (item >= items) return;
  const int hk = static_cast<int>(item % p.h_k);
  const int64_t rest = item / p.h_k;
  const int slot = static_cast<int>(rest % p.slots), bi = static_cast<int>(rest / p.slots);
  int len = p.seqlens[bi];
  const int64_t most = static_cast<int64_t>(p.max_blocks) * p.page_size;
  if (len > most) {
    len = static_cast<int>(most);
    if (slot == 0 && hk == 0 && lane == 0) atomicOr(p.status, kRangeBit);
  }
  const int first = p.new_tokens > 0 ? max(0, len - p.new_tokens) / p.page_size : 0;
  const int index = first + slot;
  const int rows = min(p.page_size, len - index * p.page_size);
  if (len <= 0 || rows <= 0) return;
  const int page = p.block_table[bi * p.bt_stride + index];
  if (page < 0 || page >= p.num_blocks) {
    if (lane == 0) atomicOr(p.status, kRangeBit);
    return;
  }
  const int nv = p.d >> 3;                      // lanes of a row: 8, 16, 24 or 32
  const int groups = 32 / nv;                   // rows read side by side
  const int grp = lane / nv, vec = lane - grp * nv;
  const bool live = grp < groups;
  const uint8_t* base = static_cast<const uint8_t*>(p.k_cache) +
                        (page * p.k_blk + hk * p.k_h + vec * 8) * es;
  uint32_t lo[4], hi[4];
  bool any = false;
  for (int r0 = grp; r0 < rows && live; r0 += groups * U) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // a row past the end repeats one that is there: it changes no minimum
      const int r = r0 + u * groups < rows ? r0 + u * groups : r0;
      if constexpr (kFp8) {
        const uint2 w = *reinterpret_cast<const uint2*>(base + static_cast<int64_t>(r) * p.k_row);
        v[u] = make_uint4(cvt_fp8x2_to_f16x2<DT == FA_B200_E5M2>(w.x), cvt_fp8x2_to_f16x2<DT == FA_B200_E5M2>(w.x >> 16),
                          cvt_fp8x2_to_f16x2<DT == FA_B200_E5M2>(w.y), cvt_fp8x2_to_f16x2<DT == FA_B200_E5M2>(w.y >> 16));
      } else {
        v[u] = *reinterpret_cast<const uint4*>(base + static_cast<int64_t>(r) * p.k_row * 2);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo[j] = (any || u > 0) ? min2<CT>(lo[j], x[j]) : x[j];
        hi[j] = (any || u > 0) ? max2<CT>(hi[j], x[j]) : x[j];
      }
    }
    any = true;
  }
  // lane groups side by side: 4 of 8 lanes or 2 of 16; a group without a row takes its partner's bounds
#pragma unroll
  for (int s = 8; s < 32; s <<= 1) {
    if (s < nv || groups * nv <= s) continue;
    const bool other = __shfl_xor_sync(0xffffffffu, any ? 1 : 0, s) != 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t l2 = __shfl_xor_sync(0xffffffffu, lo[j], s), h2 = __shfl_xor_sync(0xffffffffu, hi[j], s);
      if (other) {
        lo[j] = any ? min2<CT>(lo[j], l2) : l2;
        hi[j] = any ? max2<CT>(hi[j], h2) : h2;
      }
    }
    any = any || other;
  }
  if (!live || grp != 0) return;
  if constexpr (CT != OT) {   // f16 comparisons of fp8 values, bf16 bounds: every fp8 value is a bf16 value
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 l = Pair16<CT>::to_float(lo[j]), h = Pair16<CT>::to_float(hi[j]);
      lo[j] = pack_bf16(l.x, l.y);
      hi[j] = pack_bf16(h.x, h.y);
    }
  }
  uint16_t* out = static_cast<uint16_t*>(p.bounds) + (static_cast<int64_t>(page) * p.h_k + hk) * 2 * p.d + vec * 8;
  *reinterpret_cast<uint4*>(out) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  *reinterpret_cast<uint4*>(out + p.d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
}

// Pages of a sequence, and the first of those that hold its last sq tokens.
struct SeqPages { int len, pages, open; };
__device__ __forceinline__ SeqPages seq_pages(const PageSelectParams& p, int bi, bool report) {
  SeqPages s;
  s.len = max(p.seqlens[bi], 0);
  const int64_t most = static_cast<int64_t>(p.max_blocks) * p.page_size;
  if (s.len > most) {
    s.len = static_cast<int>(most);
    if (report) atomicOr(p.status, kRangeBit);
  }
  s.pages = (s.len + p.page_size - 1) / p.page_size;
  s.open = max(0, s.len - p.sq) / p.page_size;
  return s;
}
__device__ __forceinline__ bool always_taken(const PageSelectParams& p, const SeqPages& s, int i) {
  return i < p.sink_pages || i >= s.pages - p.recent_pages || i >= s.open;
}

// Score of one page in 64 bits by one warp: every lane returns it.
template <int DT>
__device__ __forceinline__ double page_score(const PageSelectParams& p, int bi, int hk, int page, int lane) {
  const uint32_t* lo = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.bounds) +
                                                         (static_cast<int64_t>(page) * p.h_k + hk) * 2 * p.d);
  const uint32_t* hi = lo + p.d / 2;
  double best = -INFINITY;
  bool nan = false;
  for (int r = 0; r < p.sq * p.group; ++r) {
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + bi * p.q_b + (r / p.group) * p.q_r +
                        (static_cast<int64_t>(hk) * p.group + r % p.group) * p.q_h;
    double sum = 0.;
    for (int c = lane; c < p.d / 2; c += 32) {
      const float2 l = Pair16<DT>::to_float(lo[c]), h = Pair16<DT>::to_float(hi[c]);
      const float2 x = Pair16<DT>::to_float(*reinterpret_cast<const uint32_t*>(q + 2 * c));
      // max(x lo, x hi) is x hi for x >= 0 and x lo below; the products of 16-bit values are exact in 64 bits
      sum = fma(static_cast<double>(x.x), static_cast<double>(x.x < 0.f ? l.x : h.x), sum);
      sum = fma(static_cast<double>(x.y), static_cast<double>(x.y < 0.f ? l.y : h.y), sum);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    nan = nan || isnan(sum);
    best = sum > best ? sum : best;
  }
  return nan ? static_cast<double>(NAN) : best;
}

template <int DT>
__global__ void __launch_bounds__(128) page_score_kernel(const PageSelectParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x * 4 + warp, hk = blockIdx.y, bi = blockIdx.z;
  const SeqPages s = seq_pages(p, bi, i == 0 && hk == 0 && lane == 0);
  if (i >= s.pages || s.pages <= p.num_pages) return;
  if (always_taken(p, s, i)) return;
  const int page = p.block_table[bi * p.bt_stride + i];
  double score = -INFINITY;
  if (page >= 0 && page < p.num_blocks) score = page_score<DT>(p, bi, hk, page, lane);
  else if (lane == 0) atomicOr(p.status, kRangeBit);
  if (lane == 0)
    static_cast<double*>(p.workspace)[(static_cast<int64_t>(bi) * p.h_k + hk) * p.max_blocks + i] = score;
}

__global__ void __launch_bounds__(kSelectThreads) page_select_kernel(const PageSelectParams p) {
  __shared__ TopkShared sh;
  const int hk = blockIdx.x, bi = blockIdx.y, tid = threadIdx.x;
  const SeqPages s = seq_pages(p, bi, false);
  const int64_t pair = static_cast<int64_t>(bi) * p.h_k + hk;
  const double* score = static_cast<const double*>(p.workspace) + pair * p.max_blocks;
  const int32_t* bt = p.block_table + bi * p.bt_stride;
  int32_t* index = p.page_index + pair * p.num_pages;
  int32_t* table = p.page_table + pair * p.num_pages;
  const int chosen = min(s.pages, p.num_pages);
  if (s.pages <= p.num_pages) {
    for (int i = tid; i < chosen; i += kSelectThreads) { index[i] = i; table[i] = bt[i]; }
  } else {
    auto key = [&](int i) -> uint64_t { return always_taken(p, s, i) ? ~0ull : order_key(score[i]); };
    int take_equal;
    const uint64_t border = topk_border<kSelectThreads, uint64_t>(s.pages, chosen, key, sh, take_equal);
    topk_emit<kSelectThreads>(s.pages, border, take_equal, key, sh, [&](bool take, int at, int i) {
      if (take) { index[at] = i; table[at] = bt[i]; }
    });
  }
  for (int i = chosen + tid; i < p.num_pages; i += kSelectThreads) { index[i] = -1; table[i] = -1; }
  // the last page is always taken, and it is the only one that can be partly filled
  if (tid == 0) p.seqlens_out[pair] = chosen * p.page_size - (s.pages * p.page_size - s.len);
}

}  // namespace

cudaError_t launch_page_bounds(int dtype, int bounds_dtype, const PageBoundsParams& p, cudaStream_t stream) {
  const int64_t items = static_cast<int64_t>(p.b) * p.slots * p.h_k;
  const int64_t grid = (items + kBoundsWarps - 1) / kBoundsWarps;
  if (grid == 0) return cudaSuccess;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const dim3 g(static_cast<unsigned>(grid)), t(kBoundsWarps * 32);
  const bool bf = bounds_dtype == FA_B200_BF16;
  switch (dtype) {
    case FA_B200_BF16: page_bounds_kernel<FA_B200_BF16, FA_B200_BF16><<<g, t, 0, stream>>>(p); break;
    case FA_B200_F16: page_bounds_kernel<FA_B200_F16, FA_B200_F16><<<g, t, 0, stream>>>(p); break;
    case FA_B200_E4M3:
      if (bf) page_bounds_kernel<FA_B200_E4M3, FA_B200_BF16><<<g, t, 0, stream>>>(p);
      else page_bounds_kernel<FA_B200_E4M3, FA_B200_F16><<<g, t, 0, stream>>>(p);
      break;
    case FA_B200_E5M2:
      if (bf) page_bounds_kernel<FA_B200_E5M2, FA_B200_BF16><<<g, t, 0, stream>>>(p);
      else page_bounds_kernel<FA_B200_E5M2, FA_B200_F16><<<g, t, 0, stream>>>(p);
      break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

size_t page_select_workspace_bytes(int b, int h_k, int max_blocks) {
  return static_cast<size_t>(b) * h_k * max_blocks * sizeof(double);
}

cudaError_t launch_page_select(int dtype, const PageSelectParams& p, cudaStream_t stream) {
  const dim3 g((p.max_blocks + 3) / 4, p.h_k, p.b);
  if (g.x > 0 && p.max_blocks > p.num_pages) {   // otherwise every sequence keeps all its pages
    if (dtype == FA_B200_BF16) page_score_kernel<FA_B200_BF16><<<g, 128, 0, stream>>>(p);
    else page_score_kernel<FA_B200_F16><<<g, 128, 0, stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  page_select_kernel<<<dim3(p.h_k, p.b), kSelectThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fa

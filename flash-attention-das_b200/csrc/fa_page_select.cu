// Bounds of a paged cache's keys, and the choice of pages by them.
//
// Bounds.  lo[c] and hi[c] are the smallest and largest value of channel c among a page's keys, so for every key k of the
// page q . k = sum_c q_c k_c <= sum_c max(q_c lo_c, q_c hi_c): a bound on the score that costs one row pair per page
// instead of the page.  One warp per (page, kv head): 16-byte pieces of the rows, several rows in flight, packed 16-bit
// minimum and maximum (exact: the bounds are values of the cache).  HBM-bound for a whole prompt (8 x 32768 tokens, 8 kv
// heads, bf16, 0.55 GB: 82 us, the copy rate), 4 us of latency for the pages of one decode step.
//
// Choice.  A score kernel reads every page's bounds once and scores it in 32 bits, then one CTA per (sequence, kv head)
// finds the border, looks again, in 64 bits, at the pages that are too near to it for 32, and writes the list.
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

// A 16-bit value in 64 bits times 2^-896 (bf16) or 2^-1008 (f16): its bits moved to the top of a 64-bit word, subnormals
// included; infinities and NaN read wrong.
template <int DT> __device__ __forceinline__ double wide_bits(uint32_t low16) {
  const uint32_t h = ((low16 & 0x7fffu) << (DT == FA_B200_BF16 ? 13 : 10)) | ((low16 << 16) & 0x80000000u);
  return __hiloint2double(static_cast<int>(h), 0);
}
template <int DT> __device__ __forceinline__ double wide_unit() {   // the inverse factor
  return __longlong_as_double(static_cast<long long>(1023 + (DT == FA_B200_BF16 ? 896 : 1008)) << 52);
}
template <int DT> __device__ __forceinline__ double to_double(uint16_t v) {
  constexpr uint32_t kExp = DT == FA_B200_BF16 ? 0x7f80u : 0x7c00u;
  if ((v & kExp) == kExp) return static_cast<double>(Pair16<DT>::to_float(v).x);
  return wide_bits<DT>(v) * wide_unit<DT>();
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

// One query row's score of a page in 64 bits by one warp; every lane returns it.  The products of 16-bit values are exact;
// the sum rounds, in a fixed order: at most d / 32 fused multiply-adds and five additions per term, so a score is within
// 13 * 2^-53 (d = 256) of the sum of its products' magnitudes.  Pages with equal bounds have equal scores.
template <int DT>
__device__ __forceinline__ double row_score(const PageSelectParams& p, int bi, int hk, int page, int r, int lane) {
  const uint16_t* lo = static_cast<const uint16_t*>(p.bounds) + (static_cast<int64_t>(page) * p.h_k + hk) * 2 * p.d;
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + bi * p.q_b + (r / p.group) * p.q_r +
                      (static_cast<int64_t>(hk) * p.group + r % p.group) * p.q_h;
  double sum = 0.;
#pragma unroll 2
  for (int c = lane * 4; c < p.d; c += 128) {
    const uint2 x = *reinterpret_cast<const uint2*>(q + c), l = *reinterpret_cast<const uint2*>(lo + c),
                h = *reinterpret_cast<const uint2*>(lo + p.d + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int sh = 16 * (j & 1);
      const uint16_t xv = static_cast<uint16_t>((j < 2 ? x.x : x.y) >> sh);
      const uint16_t lv = static_cast<uint16_t>((j < 2 ? l.x : l.y) >> sh), hv = static_cast<uint16_t>((j < 2 ? h.x : h.y) >> sh);
      sum = fma(to_double<DT>(xv), to_double<DT>(xv > 0x8000u ? lv : hv), sum);   // -0 is not below 0
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  return sum;
}

// Scores in 32 bits, with a bound on their error.  max(q lo, q hi) = q- lo + q+ hi with q- = min(q, 0) and q+ = max(q, 0),
// so the scores of all rows are a product of 16 x 2d queries [q-, q+] with the pages' rows [lo, hi] as they are stored: register-level
// MMAs with 8 pages as columns, whose B fragments come straight from 16-byte pieces of the rows (the order of the channels
// within a k-step is free as long as both operands agree).  What is left is reading every bound once.
//
// Error: the products are exact and each of the 2d additions is at least a 32-bit one, in any order and rounding: at most
// 2^-23 of a partial sum, none of which is above sum |q_c| times the largest bound.  What may be flushed to zero is below
// 2^-126: a query value (times a bound, d of them), a bound (times its query value), each product and sum, and the terms of
// sum |q_c| itself.  The kernel writes the sum of all that per warp (and infinity where it nears the end of the 32-bit range or
// is no number); the choice below looks again in 64 bits at pages that are closer to the border.
//
// 32 sequences x 131072 tokens in pages of 64, 8 kv heads, 256 MB of bounds, bf16: 52 us (5.2 TB/s; a CTA's start, which is a
// chain of trips to memory, is what it is away from the copy rate), then 14 for the choice.  64-bit sums throughout took 148 us,
// 32-bit multiply-adds on the FMA pipe 84 (both bound by the instructions they issue); four heads side by side in a CTA, one
// warp each, or more stages with fewer CTAs per SM measured the same or slower.
constexpr int kScoreWarps = 4;
constexpr int kBatch = 8;          // pages of a warp at a time: the columns of one MMA tile
// Two batches in flight per warp while one is scored; one above d = 128, where a batch is as large as two and shared memory
// decides how many CTAs an SM holds.
__host__ __device__ constexpr int score_stages(int hd) { return hd <= 128 ? 3 : 2; }
__host__ __device__ constexpr int score_ctas(int hd) { return hd <= 128 ? 4 : hd == 192 ? 3 : 2; }   // resident on an SM
constexpr int kMaxBatches = 32;
// Query fragments: in registers up to d = 128 (64 of them), else in shared memory.
__host__ __device__ constexpr bool a_in_regs(int hd) { return hd <= 128; }
__host__ __device__ constexpr int score_smem(int hd) { return (a_in_regs(hd) ? 0 : hd / 8 * 512) + kScoreWarps * score_stages(hd) * kBatch * 4 * hd; }

// All ones in each half whose sign bit is set.
__device__ __forceinline__ uint32_t sign_halves(uint32_t v) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(r) : "r"(v));
  return r;
}

// The larger magnitude of each half, with some sign; a NaN stays.  One instruction.
template <int DT> __device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (DT == FA_B200_BF16) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// blockIdx: x kv head, y share of the pages, z sequence: the heads of a page, whose bounds lie side by side, are read at about
// the same time.
template <int DT, int HD>
__global__ void __launch_bounds__(kScoreWarps * 32) page_score_kernel(const PageSelectParams p) {
  constexpr int kScoreStages = score_stages(HD);
  constexpr int kPieces = HD / 16;                // 64-byte pieces of a page's row pair: half of them lo, half hi
  extern __shared__ uint4 sm_dyn[];
  uint4* sm_a = sm_dyn;                           // A fragments: [2 * piece + step][lane]
  __shared__ float sm_q1[16];
  __shared__ int sm_ids[kScoreWarps * kBatch * kMaxBatches];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, qd = lane & 3;
  // bounds on their way: [warp][stage][piece][lane], written and read by the same lane
  uint4* ring = sm_dyn + (a_in_regs(HD) ? 0 : 2 * kPieces * 32) + warp * (kScoreStages * kPieces * 32) + lane;
  const int hk = blockIdx.x, chunk = blockIdx.y, bi = blockIdx.z;
  const int rows = p.sq * p.group;
  griddep_wait();
  griddep_launch_dependents();
  const SeqPages s = seq_pages(p, bi, chunk == 0 && hk == 0 && threadIdx.x == 0);
  if (s.pages <= p.num_pages || chunk * kScoreWarps * kBatch * p.batches >= s.pages) return;
  const int32_t* bt = p.block_table + bi * p.bt_stride;
  const int first_batch = chunk * kScoreWarps * p.batches + warp;   // this warp's batches: every kScoreWarps-th
  // the CTA's page ids; -1: not scored.  Read ahead of everything else, so that no copy waits for one.
  const int cta_first = chunk * kScoreWarps * p.batches * kBatch;
  for (int i = threadIdx.x; i < kScoreWarps * kBatch * p.batches; i += kScoreWarps * 32) {
    int id = -1;
    if (cta_first + i < s.pages && !always_taken(p, s, cta_first + i)) {
      id = bt[cta_first + i];
      if (id < 0 || id >= p.num_blocks) { atomicOr(p.status, kRangeBit); id = -1; }
    }
    sm_ids[i] = id;
  }
  __syncthreads();
  const int* ids = sm_ids + warp * kBatch;   // of batch n: from n * kScoreWarps * kBatch
  auto issue = [&](int n) {
    const int page = ids[n * kScoreWarps * kBatch + g];
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.bounds) +
                                                      (static_cast<int64_t>(max(page, 0)) * p.h_k + hk) * 2 * HD) + qd;
    uint4* dst = ring + (n % kScoreStages) * kPieces * 32;
#pragma unroll
    for (int c = 0; c < kPieces; ++c)   // a page that is not scored reads as zeros
      cp_async16(smem_u32(dst + c * 32), src + 4 * c, page >= 0 ? 16 : 0);
  };
#pragma unroll
  for (int n = 0; n < kScoreStages - 1; ++n) {
    if (n < p.batches) issue(n);
    cp_async_commit();
  }
  // A fragments of [q-, q+]: piece c of a row covers channels 32 (c mod kPieces / 2) .. + 31, of which this lane's are
  // 8 qd .. + 7, four for each of two k-steps.  Rows past the last query are zero.
  auto q_row = [&](int r) {
    return static_cast<const uint16_t*>(p.q) + bi * p.q_b + (r / p.group) * p.q_r + (static_cast<int64_t>(hk) * p.group + r % p.group) * p.q_h;
  };
  // Both the q- of piece c and the q+ of piece c + kPieces / 2.
  const uint16_t* const q_g = q_row(g < rows ? g : 0) + qd * 8;
  const uint16_t* const q_g8 = q_row(g + 8 < rows ? g + 8 : 0) + qd * 8;
  auto fragments = [&](int c, uint4& n0, uint4& n1, uint4& p0, uint4& p1) {
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    const uint4 r0 = g < rows ? *reinterpret_cast<const uint4*>(q_g + c * 32) : z;
    const uint4 r1 = g + 8 < rows ? *reinterpret_cast<const uint4*>(q_g8 + c * 32) : z;
    const uint32_t v[8] = {r0.x, r1.x, r0.y, r1.y, r0.z, r1.z, r0.w, r1.w};
    uint32_t n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = v[i] & sign_halves(v[i]);
    n0 = make_uint4(n[0], n[1], n[2], n[3]);
    n1 = make_uint4(n[4], n[5], n[6], n[7]);
    p0 = make_uint4(v[0] ^ n[0], v[1] ^ n[1], v[2] ^ n[2], v[3] ^ n[3]);
    p1 = make_uint4(v[4] ^ n[4], v[5] ^ n[5], v[6] ^ n[6], v[7] ^ n[7]);
  };
  constexpr int kHalf = kPieces / 2;
  uint4 a[a_in_regs(HD) ? 2 * kPieces : 1];
  if constexpr (a_in_regs(HD)) {
#pragma unroll
    for (int c = 0; c < kHalf; ++c) fragments(c, a[2 * c], a[2 * c + 1], a[2 * (c + kHalf)], a[2 * (c + kHalf) + 1]);
  } else {
    for (int c = warp; c < kHalf; c += kScoreWarps)
      fragments(c, sm_a[(2 * c) * 32 + lane], sm_a[(2 * c + 1) * 32 + lane], sm_a[(2 * (c + kHalf)) * 32 + lane], sm_a[(2 * (c + kHalf) + 1) * 32 + lane]);
  }
  for (int r = warp; r < rows; r += kScoreWarps) {   // sum |q_c| of every row
    float sum = 0.f;
    for (int c = lane; c < HD / 2; c += 32) {
      const float2 x = Pair16<DT>::to_float(*reinterpret_cast<const uint32_t*>(q_row(r) + 2 * c));
      sum += fabsf(x.x) + fabsf(x.y);
    }
#pragma unroll
    for (int st = 16; st > 0; st >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, st);
    if (lane == 0) sm_q1[r] = sum;
  }
  __syncthreads();
  float q1 = 0.f;
  for (int r = 0; r < rows; ++r) q1 = sm_q1[r] > q1 || isnan(sm_q1[r]) ? sm_q1[r] : q1;   // a NaN stays
  const int64_t pair = static_cast<int64_t>(bi) * p.h_k + hk;
  float* out = p.scores + pair * p.max_blocks;
  uint32_t top = 0, top2 = 0;   // largest magnitudes, of either sign
  for (int n = 0; n < p.batches; ++n) {
    const int first = (first_batch + n * kScoreWarps) * kBatch;
    if (first >= s.pages) break;
    if (n + kScoreStages - 1 < p.batches) issue(n + kScoreStages - 1);
    cp_async_commit();
    cp_async_wait<kScoreStages - 1>();
    const uint4* stage = ring + (n % kScoreStages) * kPieces * 32;
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, acc2[4] = {0.f, 0.f, 0.f, 0.f};   // two chains
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const uint4 v = stage[c * 32];
      const uint4 a0 = a_in_regs(HD) ? a[a_in_regs(HD) ? 2 * c : 0] : sm_a[(2 * c) * 32 + lane];
      const uint4 a1 = a_in_regs(HD) ? a[a_in_regs(HD) ? 2 * c + 1 : 0] : sm_a[(2 * c + 1) * 32 + lane];
      const uint32_t f0[4] = {a0.x, a0.y, a0.z, a0.w}, f1[4] = {a1.x, a1.y, a1.z, a1.w};
      if constexpr (DT == FA_B200_BF16) {
        mma_bf16_16816(acc, f0, v.x, v.y);
        mma_bf16_16816(acc2, f1, v.z, v.w);
      } else {
        mma_f16_16816(acc, f0, v.x, v.y);
        mma_f16_16816(acc2, f1, v.z, v.w);
      }
      top = abs_max2<DT>(abs_max2<DT>(top, v.x), v.y);
      top2 = abs_max2<DT>(abs_max2<DT>(top2, v.z), v.w);
    }
    // the largest of the rows g and g + 8 over g; columns 2 qd and 2 qd + 1
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float v = fmaxf(g < rows ? acc[e] + acc2[e] : -INFINITY, g + 8 < rows ? acc[2 + e] + acc2[2 + e] : -INFINITY);
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
      const int slot = 2 * qd + e;
      if (g == 0 && first + slot < s.pages) out[first + slot] = ids[n * kScoreWarps * kBatch + slot] >= 0 ? v : -INFINITY;
    }
  }
  top = abs_max2<DT>(top, top2);
#pragma unroll
  for (int st = 16; st > 0; st >>= 1) top = abs_max2<DT>(top, __shfl_xor_sync(0xffffffffu, top, st));
  const float most = Pair16<DT>::to_float(max(top & 0x7fffu, (top >> 16) & 0x7fffu)).x;   // ordered by their bits; NaN on top
  const float reach = q1 * most, flushed = ((most + 4.f) * HD + q1) * 0x1p-125f;   // twice each
  if (lane == 0)   // not below 1e37: too large, or no number
    p.errors[pair * p.err_stride + chunk * kScoreWarps + warp] = reach < 1e37f ? reach * (1.1f * 2 * HD * 0x1p-23f) + flushed : INFINITY;
  cp_async_wait<0>();
}

constexpr int kNear = 128;   // pages at the border that are ranked in shared memory; more: by another search over all

// V keys in a row per thread; IN_REGS: the row's keys stay in registers (up to V * kSelectThreads pages), else they are read
// again for every pass.
template <int DT, int V, bool IN_REGS>
__global__ void __launch_bounds__(kSelectThreads) page_select_kernel(const PageSelectParams p) {
  __shared__ TopkShared sh;
  __shared__ uint32_t sm_err, sm_min, sm_max;
  __shared__ int sm_near, sm_sure, near_page[kNear];
  __shared__ uint64_t near_key[kNear];
  __shared__ bool near_taken[kNear];
  const int hk = blockIdx.x, bi = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  griddep_wait();
  griddep_launch_dependents();
  const SeqPages s = seq_pages(p, bi, false);
  const int64_t pair = static_cast<int64_t>(bi) * p.h_k + hk;
  const float* score = p.scores + pair * p.max_blocks;
  const int32_t* bt = p.block_table + bi * p.bt_stride;
  int32_t* index = p.page_index + pair * p.num_pages;
  int32_t* table = p.page_table + pair * p.num_pages;
  const int chosen = min(s.pages, p.num_pages);
  constexpr int kTile = V * kSelectThreads;
  // An id that is no page is listed as it is where its page is taken all the same; sparse attention leaves its keys out.
  auto list = [&](int at, int i, int32_t id) {
    index[at] = i;
    table[at] = id;
    if (id < 0 || id >= p.num_blocks) atomicOr(p.status, kRangeBit);
  };
  if (s.pages <= p.num_pages) {
    for (int i = tid; i < chosen; i += kSelectThreads) list(i, i, bt[i]);
  } else {
    if (tid == 0) { sm_min = ~0u; sm_max = 0u; sm_err = 0u; sm_near = 0; sm_sure = 0; }
    constexpr bool kIds = IN_REGS && V <= 4;   // the pages' ids too: looked up beside the scores, not after the choice
    uint32_t k[V];
    int32_t id[kIds ? V : 1];
    auto load = [&](int i0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = i0 + j;
        if (kIds) id[kIds ? j : 0] = i < s.pages ? __ldg(bt + i) : -1;
        k[j] = i >= s.pages ? 0u : (always_taken(p, s, i) ? ~0u : order_key(__ldg(score + i)));
      }
    };
    if (IN_REGS) load(tid * V);
    // errors are not negative: their bits order as they do, infinity on top
    const int nb = (s.pages + kScoreWarps * kBatch * p.batches - 1) / (kScoreWarps * kBatch * p.batches) * kScoreWarps;
    uint32_t e = 0;
    for (int i = tid; i < nb; i += kSelectThreads) e = max(e, __float_as_uint(p.errors[pair * p.err_stride + i]));
    auto each = [&](auto f) {
      for (int i0 = 0; i0 < s.pages; i0 += kTile) {
        if (!IN_REGS) load(i0 + tid * V);
#pragma unroll
        for (int j = 0; j < V; ++j) f(k[j], i0 + tid * V + j);
      }
    };
    int take_equal;
    uint32_t border = topk_border<kSelectThreads>(chosen, -1, [&](auto f) { each([&](uint32_t x, int) { f(x); }); }, sh, take_equal);
    // The lowest score taken and the highest one left: the 32-bit choice stands if they differ by more than both errors.
    uint32_t lowest = ~0u, highest = 0u;
    each([&](uint32_t x, int) {
      if (x > border) lowest = min(lowest, x);
      else highest = max(highest, x);
    });
    if (take_equal > 0) lowest = border;
    lowest = __reduce_min_sync(0xffffffffu, lowest);
    highest = __reduce_max_sync(0xffffffffu, highest);
    e = __reduce_max_sync(0xffffffffu, e);
    if (lane == 0) {
      atomicMin(&sm_min, lowest);
      atomicMax(&sm_max, highest);
      atomicMax(&sm_err, e);
    }
    __syncthreads();
    const float t = key_value(sm_min), left = key_value(sm_max), err2 = 2.f * __uint_as_float(sm_err);
    const bool clear = sm_min == ~0u || t - left > err2 * 1.0001f;   // only pages that are always taken, or a clear border
    // Else: pages nearer to the k-th score t than 2 err are compared in 64 bits; one above t + 2 err has fewer than k pages
    // that can be better, one below t - 2 err has at least k that are.
    const float lo = t - err2 * 1.0001f, hi = t + err2 * 1.0001f;
    const bool all = !(err2 < INFINITY);
    auto is_sure = [&](uint32_t x) { return x == ~0u || (x != 0u && key_value(x) > hi); };
    auto is_near = [&](uint32_t x) { return x != 0u && !is_sure(x) && (all || key_value(x) >= lo); };
    if (!clear) {
      each([&](uint32_t x, int i) {
        if (is_sure(x)) atomicAdd(&sm_sure, 1);
        if (is_near(x)) {
          const int at = atomicAdd(&sm_near, 1);
          if (at < kNear) near_page[at] = i;
        }
      });
      __syncthreads();
    }
    TopkCount base;
    if (clear || sm_near <= kNear) {
      if (!clear) {
        const int n_near = sm_near, want = chosen - sm_sure;
        if (tid < n_near) near_key[tid] = 0ull;   // below every score: stays where the table holds no page
        __syncthreads();
        const int rows = p.sq * p.group;
        for (int c = tid >> 5; c < n_near * rows; c += kSelectThreads / 32) {   // a warp per page and row
          const int id = bt[near_page[c / rows]];
          if (id < 0 || id >= p.num_blocks) continue;
          const double v = row_score<DT>(p, bi, hk, id, c % rows, lane);
          if (lane == 0) atomicMax(reinterpret_cast<unsigned long long*>(&near_key[c / rows]), order_key(v));
        }
        __syncthreads();
        if (tid < n_near) {   // fewer than `want` better ones, ties to the lower page
          int better = 0;
          for (int c = 0; c < n_near; ++c)
            better += (near_key[c] > near_key[tid] || (near_key[c] == near_key[tid] && near_page[c] < near_page[tid])) ? 1 : 0;
          near_taken[tid] = better < want;
        }
        __syncthreads();
      }
      for (int i0 = 0; i0 < s.pages; i0 += kTile) {
        if (!IN_REGS) load(i0 + tid * V);
        if (!clear) {   // what is settled: 2 taken, 1 left
#pragma unroll
          for (int j = 0; j < V; ++j) {
            bool take = is_sure(k[j]);
            if (is_near(k[j]))
              for (int c = 0; c < sm_near; ++c)
                if (near_page[c] == i0 + tid * V + j) take = near_taken[c];
            k[j] = take ? 2u : 1u;
          }
        }
        topk_place<kSelectThreads, V>(k, clear ? border : 1u, clear ? take_equal : 0, base, sh, [&](int j, int at) {
          const int i = i0 + tid * V + j;
          list(at, i, kIds ? id[kIds ? j : 0] : bt[i]);
        });
      }
    } else {
      // hundreds of pages at the border (equal bounds, infinities): every one's key in 64 bits, and another search
      uint64_t* wide = p.wide + pair * p.max_blocks;
      each([&](uint32_t x, int i) {
        if (i < s.pages) wide[i] = is_sure(x) ? ~0ull : (is_near(x) ? 1ull : 0ull);
      });
      __syncthreads();
      for (int i = tid >> 5; i < s.pages; i += kSelectThreads / 32) {
        const int id = bt[i];
        if (wide[i] != 1ull || id < 0 || id >= p.num_blocks) continue;
        uint64_t most = 0;
        for (int r = 0; r < p.sq * p.group; ++r) most = max(most, order_key(row_score<DT>(p, bi, hk, id, r, lane)));
        if (lane == 0) wide[i] = most;
      }
      __syncthreads();
      int take_equal64;
      const uint64_t border64 = topk_border64<kSelectThreads>(chosen, [&](auto f) {
        for (int i = tid; i < s.pages; i += kSelectThreads) f(wide[i], true);
      }, sh, take_equal64);
      int n_eq = 0;   // the equal ones are taken in ascending order
      for (int i0 = 0; i0 < s.pages; i0 += kSelectThreads) {
        const uint64_t x = i0 + tid < s.pages ? wide[i0 + tid] : 0ull;
        int total;
        const int eq = i0 + tid < s.pages && x == border64 ? 1 : 0;
        const int before = n_eq + block_exclusive<kSelectThreads>(eq, sh, total);
        n_eq += total;
        const uint32_t one[1] = {i0 + tid < s.pages && (x > border64 || (eq && before < take_equal64)) ? 2u : 1u};
        topk_place<kSelectThreads, 1>(one, 1u, 0, base, sh, [&](int, int at) { list(at, i0 + tid, bt[i0 + tid]); });
      }
    }
  }
  for (int i = chosen + tid; i < p.num_pages; i += kSelectThreads) { index[i] = -1; table[i] = -1; }
  // the last page is always taken, and it is the only one that can be partly filled
  if (tid == 0) p.seqlens_out[pair] = chosen * p.page_size - (s.pages * p.page_size - s.len);
}

template <class Kernel>
cudaError_t launch_dependent(Kernel kern, dim3 grid, int threads, size_t smem, bool dependent, cudaStream_t stream, const PageSelectParams& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int DT, int HD>
cudaError_t launch_scores(PageSelectParams& p, cudaStream_t stream) {
  // Batches of a warp: one while that leaves room on the GPU (two rounds of what is resident on 148 SMs), up to 32, which share
  // the start-up of a CTA (lengths, page ids and queries are dependent trips to memory).
  const int64_t ctas = static_cast<int64_t>((p.max_blocks + kScoreWarps * kBatch - 1) / (kScoreWarps * kBatch)) * p.h_k * p.b;
  p.batches = 1;
  while (p.batches < kMaxBatches && ctas / (2 * p.batches) >= 148 * 2 * score_ctas(HD)) p.batches *= 2;
  const int per_cta = kScoreWarps * kBatch * p.batches;
  const dim3 g(p.h_k, (p.max_blocks + per_cta - 1) / per_cta, p.b);
  const auto kern = page_score_kernel<DT, HD>;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, score_smem(HD));
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_done[dev] = true;
  }
  return launch_dependent(kern, g, kScoreWarps * 32, score_smem(HD), p.dependent_launch, stream, p);
}

template <int DT>
cudaError_t launch_select_t(PageSelectParams p, cudaStream_t stream) {
  if (p.max_blocks > p.num_pages) {   // otherwise every sequence keeps all its pages
    const cudaError_t e = p.d == 64    ? launch_scores<DT, 64>(p, stream)
                          : p.d == 128 ? launch_scores<DT, 128>(p, stream)
                          : p.d == 192 ? launch_scores<DT, 192>(p, stream)
                                       : launch_scores<DT, 256>(p, stream);
    if (e != cudaSuccess) return e;
  }
  const auto kern = p.max_blocks <= kSelectThreads       ? page_select_kernel<DT, 1, true>
                    : p.max_blocks <= 4 * kSelectThreads  ? page_select_kernel<DT, 4, true>
                    : p.max_blocks <= 16 * kSelectThreads ? page_select_kernel<DT, 16, true>
                                                          : page_select_kernel<DT, 8, false>;
  return launch_dependent(kern, dim3(p.h_k, p.b), kSelectThreads, 0, p.dependent_launch, stream, p);
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

// Workspace: 64-bit keys, scores, and an error per warp of the score kernel.
static int error_words(int max_blocks) { return (max_blocks + kScoreWarps * kBatch - 1) / (kScoreWarps * kBatch) * kScoreWarps; }
size_t page_select_workspace_bytes(int b, int h_k, int max_blocks) {
  const size_t pairs = static_cast<size_t>(b) * h_k;
  return pairs * (static_cast<size_t>(max_blocks) * 12 + static_cast<size_t>(error_words(max_blocks)) * 4);
}

cudaError_t launch_page_select(int dtype, const PageSelectParams& p_, cudaStream_t stream) {
  PageSelectParams p = p_;
  const size_t n = static_cast<size_t>(p.b) * p.h_k * p.max_blocks;
  p.wide = static_cast<uint64_t*>(p.workspace);
  p.scores = reinterpret_cast<float*>(p.wide + n);
  p.errors = p.scores + n;
  p.err_stride = error_words(p.max_blocks);
  return dtype == FA_B200_BF16 ? launch_select_t<FA_B200_BF16>(p, stream) : launch_select_t<FA_B200_F16>(p, stream);
}

}  // namespace fa

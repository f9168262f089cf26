// Eviction from a paged KV cache by accumulated attention weight: which keys stay (one CTA per sequence and kv head),
// then their rows move together.
//
// Order is kept: kept position i goes to position i, and kept_index[i] >= i.  In place, a CTA therefore walks its
// (sequence, kv head, K or V) in ascending pieces with a barrier between a piece's reads and its writes: the rows it
// writes (below the piece's end) are never read by a later piece (kept_index[j] >= j >= the piece's end).  Into new pages
// the pieces are independent.
#include "fa_topk.cuh"
#include "fa_kernels.h"

namespace fa {
namespace {

constexpr int kPickThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;     // 16-byte vectors in flight per thread

__device__ __forceinline__ int evict_len(const KvEvictParams& p, int bi, bool report) {
  int len = max(p.seqlens[bi], 0);
  const int64_t most = min(static_cast<int64_t>(p.max_blocks) * p.page_size, static_cast<int64_t>(p.capacity));
  if (len > most) {
    len = static_cast<int>(most);
    if (report) atomicOr(p.status, kRangeBit);
  }
  return len;
}

__global__ void __launch_bounds__(kPickThreads) evict_pick_kernel(const KvEvictParams p) {
  __shared__ TopkShared sh;
  const int hk = blockIdx.x, bi = blockIdx.y, tid = threadIdx.x;
  const int len = evict_len(p, bi, hk == 0 && tid == 0);
  const int kept = min(len, p.budget);
  const float* w = p.w_in + bi * p.win_b + hk * p.win_h;
  float* wo = p.w_out + bi * p.wout_b + hk * p.wout_h;
  int32_t* out = p.kept + (static_cast<int64_t>(bi) * p.h_k + hk) * p.budget;
  if (hk == 0 && tid == 0) p.seqlens_out[bi] = kept;
  if (len <= p.budget) {
    for (int i = tid; i < len; i += kPickThreads) {
      out[i] = i;
      if (wo != w) wo[i] = w[i];
    }
  } else {
    auto key = [&](int i) -> uint32_t { return (i < p.sink || i >= len - p.recent) ? ~0u : order_key(w[i]); };
    int take_equal;
    const uint32_t border = topk_border<kPickThreads, uint32_t>(len, kept, key, sh, take_equal);
    // the weights move with the keys, chunk by chunk: a chunk's weights are read before topk_emit's barrier inside the
    // chunk (key) and again here, and the positions written lie at or below the ones read
    topk_emit<kPickThreads>(len, border, take_equal, key, sh, [&](bool take, int at, int i) {
      const float x = take ? w[i] : 0.f;
      __syncthreads();   // every thread has read its weight
      if (take) { out[at] = i; wo[at] = x; }
    });
    __syncthreads();
    for (int i = kept + tid; i < len; i += kPickThreads) wo[i] = 0.f;
  }
  for (int i = kept + tid; i < p.budget; i += kPickThreads) out[i] = -1;
}

// blockIdx: x piece (one CTA walks all pieces in place), y kv head and K / V, z sequence.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const KvEvictParams p) {
  const int hk = blockIdx.y >> 1, bi = blockIdx.z, tid = threadIdx.x;
  const bool is_v = blockIdx.y & 1;
  const int len = evict_len(p, bi, false);
  const int kept = min(len, p.budget);
  const bool in_place = p.new_block_table == nullptr;
  if (in_place && len <= p.budget) return;
  const int32_t* index = p.kept + (static_cast<int64_t>(bi) * p.h_k + hk) * p.budget;
  const int32_t* src_bt = p.block_table + bi * p.bt_stride;
  const int32_t* dst_bt = in_place ? src_bt : p.new_block_table + bi * p.nbt_stride;
  const int dst_max = in_place ? p.max_blocks : p.new_max_blocks;
  uint8_t* pool = static_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + hk * (is_v ? p.v_h : p.k_h);
  const int64_t blk = is_v ? p.v_blk : p.k_blk, row = is_v ? p.v_row : p.k_row;
  const int nv = p.row_bytes >> 4;                                   // 16-byte vectors of a row
  const int rows_per_pass = kMoveThreads / nv;                       // rows read side by side
  const int piece = rows_per_pass * kMoveUnroll;
  const int r_in = tid / nv, vec = tid - r_in * nv;
  const bool live = r_in < rows_per_pass;
  for (int first = blockIdx.x * piece; first < kept; first += gridDim.x * piece) {
    uint4 v[kMoveUnroll];
    uint8_t* dst[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = first + u * rows_per_pass + r_in;
      dst[u] = nullptr;
      if (!live || i >= kept) continue;
      const int from = index[i];
      if (in_place && from == i) continue;   // already there
      const int sp = src_bt[from / p.page_size];
      const int ds = i / p.page_size;
      const int dp = ds < dst_max ? dst_bt[ds] : -1;
      if (sp < 0 || sp >= p.num_blocks || dp < 0 || dp >= p.num_blocks) {
        atomicOr(p.status, kRangeBit);
        continue;
      }
      v[u] = *reinterpret_cast<const uint4*>(pool + sp * blk + (from % p.page_size) * row + vec * 16);
      dst[u] = pool + dp * blk + (i % p.page_size) * row + vec * 16;
    }
    if (in_place) __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u)
      if (dst[u]) *reinterpret_cast<uint4*>(dst[u]) = v[u];
  }
}

}  // namespace

cudaError_t launch_kv_evict(const KvEvictParams& p, cudaStream_t stream) {
  evict_pick_kernel<<<dim3(p.h_k, p.b), kPickThreads, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int piece = kMoveThreads / (p.row_bytes >> 4) * kMoveUnroll;
  const int pieces = p.new_block_table ? (p.budget + piece - 1) / piece : 1;
  evict_move_kernel<<<dim3(pieces, p.h_k * 2, p.b), kMoveThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fa

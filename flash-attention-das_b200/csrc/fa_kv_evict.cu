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
constexpr int kPickSmemKeys = 48 * 1024;
constexpr int kMoveThreads = 256, kMoveMaxThreads = 1024;   // into new pages; in place, where one CTA does all
constexpr int kMoveVectors = 8;    // 16-byte vectors in flight per thread

__device__ __forceinline__ int evict_len(const KvEvictParams& p, int bi, bool report) {
  int len = max(p.seqlens[bi], 0);
  const int64_t most = min(static_cast<int64_t>(p.max_blocks) * p.page_size, static_cast<int64_t>(p.capacity));
  if (len > most) {
    len = static_cast<int>(most);
    if (report) atomicOr(p.status, kRangeBit);
  }
  return len;
}

// IN_SMEM: the row's keys stay in shared memory (up to kPickSmemKeys tokens; two CTAs per SM up to 16384), else they are made
// again from the weights for every pass.  Four keys in a row per thread at a time.
template <bool IN_SMEM>
__global__ void __launch_bounds__(kPickThreads, IN_SMEM ? 2 : 1) evict_pick_kernel(const KvEvictParams p) {
  __shared__ TopkShared sh;
  extern __shared__ uint4 sm_keys[];
  const int hk = blockIdx.x, bi = blockIdx.y, tid = threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
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
    const bool aligned = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
    const int inner_end = len - p.recent;
    auto make = [&](int i0) -> uint4 {   // keys i0 .. i0 + 3; 0: past the end
      float x[4];
      if (i0 + 4 <= len && aligned) {
        const float4 v = *reinterpret_cast<const float4*>(w + i0);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = i0 + j < len ? w[i0 + j] : 0.f;
      }
      uint32_t k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = __float_as_uint(x[j]);
      // weights as they should be (0 to infinity, no -0) between the sinks and the recent tokens: a key is its bits, sign set
      if (i0 >= p.sink && i0 + 4 <= inner_end && max(max(k[0], k[1]), max(k[2], k[3])) <= 0x7f800000u) {
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] |= 0x80000000u;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = i0 + j;
          k[j] = i >= len ? 0u : ((i < p.sink || i >= inner_end) ? ~0u : order_key(x[j]));
        }
      }
      return make_uint4(k[0], k[1], k[2], k[3]);
    };
    const int quads = (len + 3) >> 2;
    if (IN_SMEM) {   // a thread reads back what it wrote
#pragma unroll 4
      for (int q = tid; q < quads; q += kPickThreads) sm_keys[q] = make(4 * q);
    }
    auto quad = [&](int q) -> uint4 { return IN_SMEM ? sm_keys[q] : make(4 * q); };
    int take_equal;
    const uint32_t border = topk_border<kPickThreads>(kept, p.sink + p.recent, [&](auto f) {
      for (int q = tid; q < quads; q += kPickThreads) {
        const uint4 k = quad(q);
        f(k.x); f(k.y); f(k.z); f(k.w);
      }
    }, sh, take_equal);
    // the weights move with the keys, tile by tile: a tile's weights are read before topk_place's barriers, and the
    // positions written lie at or below the ones read
    TopkCount base;
    for (int q0 = 0; q0 < quads; q0 += kPickThreads) {
      const int q = q0 + tid;
      const uint4 v = q < quads ? quad(q) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t k[4] = {v.x, v.y, v.z, v.w};
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (max(max(k[0], k[1]), max(k[2], k[3])) >= border) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k[j] >= border && k[j] != 0u) x[j] = w[4 * q + j];
      }
      topk_place<kPickThreads, 4>(k, border, take_equal, base, sh, [&](int j, int at) {
        out[at] = 4 * q + j;
        wo[at] = x[j];
      });
    }
    __syncthreads();
    for (int i = kept + tid; i < len; i += kPickThreads) wo[i] = 0.f;
  }
  for (int i = kept + tid; i < p.budget; i += kPickThreads) out[i] = -1;
}

// Rows that a warp moves at a time: what kMoveVectors vectors per lane hold, and no more than it has lanes to look them up.
__host__ __device__ constexpr int move_rows(int row_bytes) {
  const int rows = 32 / (row_bytes >> 4) * kMoveVectors;
  return rows < 32 ? rows : 32;
}

// A warp moves move_rows rows at a time: a lane looks up where one of them comes from
// and goes to, then all lanes load kMoveVectors vectors each, rows side by side, and store them.
// blockIdx: x kv head and K / V (fastest: the heads of a token lie side by side, and their kept positions are near each
// other), y piece of the kept rows (one CTA walks all pieces in place), z sequence.
// 32 ragged sequences of up to 16384 tokens cut to 4096, 8 kv heads, bf16, 0.95 GB moved: 146 us (6.5 TB/s), after 26 us of
// picking; in place 137 (what is in its place already stays).  One sequence of 16384: 23 us with the choice, in place 44 (16 CTAs).  Picking is bound by the integer instructions of the SM that got the two longest rows; bounds of the keys for the
// first search step, and weights taken back from their keys instead of read again, measured no better.
__global__ void __launch_bounds__(kMoveMaxThreads) evict_move_kernel(const KvEvictParams p) {
  const int hk = blockIdx.x >> 1, bi = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  griddep_wait();
  griddep_launch_dependents();
  const bool is_v = blockIdx.x & 1;
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
  const int nv = p.row_bytes >> 4;                                   // 16-byte vectors of a row: 4 to 32
  const int side = 32 / nv;                                          // rows side by side
  const int rows = move_rows(p.row_bytes);                           // of a warp at a time
  const int r_in = lane / nv, vec = lane - r_in * nv;
  const int piece = rows * (blockDim.x >> 5);
  for (int first = blockIdx.y * piece; first < kept; first += gridDim.y * piece) {
    int64_t from = -1, to = -1;
    const int i = first + warp * rows + lane;
    if (lane < rows && i < kept) {
      const int at = len <= p.budget ? i : index[i];
      if (!(in_place && at == i)) {   // else it is there already
        const int sp = src_bt[at / p.page_size], ds = i / p.page_size;
        const int dp = ds < dst_max ? dst_bt[ds] : -1;
        if (sp < 0 || sp >= p.num_blocks || dp < 0 || dp >= p.num_blocks) {
          atomicOr(p.status, kRangeBit);
        } else {
          from = sp * blk + (at % p.page_size) * row;
          to = dp * blk + (i % p.page_size) * row;
        }
      }
    }
    uint4 v[kMoveVectors];
#pragma unroll
    for (int u = 0; u < kMoveVectors; ++u) {
      const int64_t s = __shfl_sync(0xffffffffu, from, (u * side + r_in) & 31);
      if (s >= 0 && r_in < side && u * side < rows) v[u] = *reinterpret_cast<const uint4*>(pool + s + vec * 16);
    }
    if (in_place) __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveVectors; ++u) {
      const int64_t d = __shfl_sync(0xffffffffu, to, (u * side + r_in) & 31);
      if (d >= 0 && r_in < side && u * side < rows) *reinterpret_cast<uint4*>(pool + d + vec * 16) = v[u];
    }
  }
}

}  // namespace

cudaError_t launch_kv_evict(const KvEvictParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.h_k, p.b);
  cfg.blockDim = dim3(kPickThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.dependent_launch ? 1 : 0;
  const int64_t most = min(static_cast<int64_t>(p.max_blocks) * p.page_size, static_cast<int64_t>(p.capacity));
  cudaError_t e;
  if (most <= kPickSmemKeys) {
    static bool attr_done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !attr_done[dev]) {
      e = cudaFuncSetAttribute(evict_pick_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPickSmemKeys * 4);
      if (e != cudaSuccess) return e;
      if (dev < 64) attr_done[dev] = true;
    }
    cfg.dynamicSmemBytes = static_cast<size_t>(most + 3) / 4 * 16;
    e = cudaLaunchKernelEx(&cfg, evict_pick_kernel<true>, p);
    cfg.dynamicSmemBytes = 0;
  } else {
    e = cudaLaunchKernelEx(&cfg, evict_pick_kernel<false>, p);
  }
  if (e != cudaSuccess) return e;
  const bool in_place = p.new_block_table == nullptr;
  const int threads = in_place ? kMoveMaxThreads : kMoveThreads;
  const int piece = move_rows(p.row_bytes) * (threads / 32);
  cfg.gridDim = dim3(p.h_k * 2, in_place ? 1 : (p.budget + piece - 1) / piece, p.b);
  cfg.blockDim = dim3(threads);
  return cudaLaunchKernelEx(&cfg, evict_move_kernel, p);
}

}  // namespace fa

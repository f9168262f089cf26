// The weight that every cached key receives: sums of softmax probabilities over query rows.
//
// After a decode call.  The decode kernel leaves its scaled scores (log2 units) behind, rows x tokens in fp32: 4 bytes
// per (query head, key) against 2 * d * element size bytes of K and V per (kv head, key), small enough to stay in L2.  Once the row's
// log-sum-exp is known this kernel reads them back: w[t] = decay w[t] + sum_r 2^(s_rt - lse_r), rows in a fixed order.
//
// Of a prompt.  Given every query's log-sum-exp the weight of key t is a plain sum over the queries, with no running
// maximum: a CTA owns 128 keys of one kv head, keeps their tile in shared memory as the A operand and walks the query
// tiles that see them, S^T = K Q^T in TMEM.  A TMEM lane is then a key, so a key's sum stays in one thread's register:
// no reduction between threads, no atomics, no second pass.  A query tile holds 128 / group tokens of all heads of the
// group (rows token-major), which fills it for short windows too and makes the causal mask a column bound per key.
//   warps 0-3  one thread per key: 2^(s - lse) and its sum
//   warp 4     TMA producer: the key tile once (through the block table), query tiles into a ring
//   warp 5     MMA issuer, two S^T buffers
// Bound by the exponentials: 128 x 128 of them per tile take 1024 cycles of an SM's MUFU unit, its tcgen05 product 256.
// Long prompts are cut into shares of the query tiles per key tile (every num_chunks-th tile), whose sums a small kernel
// adds in order.
#include "fa_prefill_common.cuh"

namespace fa {
namespace {

constexpr int kFinishThreads = 256;

__global__ void __launch_bounds__(kFinishThreads) weights_finish_kernel(const WeightsFinishParams p) {
  __shared__ float sm_lse[16];
  const int hk = blockIdx.y, bi = blockIdx.z;
  const int rows = p.sq * p.group;
  griddep_wait();
  griddep_launch_dependents();
  const int len = min(min(p.seqlens[bi], p.max_len), p.capacity);
  const int tok = blockIdx.x * kFinishThreads + threadIdx.x;
  if (static_cast<int>(blockIdx.x) * kFinishThreads >= len) return;
  if (threadIdx.x < rows) {   // row r is query token r / group, head r % group
    const int r = threadIdx.x;
    sm_lse[r] = p.lse[(static_cast<int64_t>(bi) * p.h + hk * p.group + r % p.group) * p.sq + r / p.group] * kLog2e;
  }
  __syncthreads();
  if (tok >= len) return;
  const float* s = p.scores + (static_cast<int64_t>(bi) * p.h_k + hk) * rows * p.score_stride + tok;
  const int full = min(p.seqlens[bi], p.max_len);
  float sum = 0.f;
  for (int r = 0; r < rows; ++r) {
    const int behind = p.sq - 1 - r / p.group;   // query tokens after this row's
    const bool seen = !(p.causal && tok >= full - behind) &&
                      !(p.window_left >= 0 && tok < full - behind - 1 - p.window_left);
    if (seen) sum += exp2f(s[r * p.score_stride] - sm_lse[r]);
  }
  const float before = p.w_in ? p.w_in[bi * p.win_b + hk * p.win_h + tok] * p.decay : 0.f;
  p.w_out[bi * p.wout_b + hk * p.wout_h + tok] = before + sum;
}

constexpr int kTwThreads = 192;
constexpr int kTwSlots = 2;
struct TwLayout { int q_off, lse_off, bar_off, misc_off, total; };
template <int DT, int HD>
__host__ __device__ constexpr TwLayout tw_layout() {
  TwLayout s{};
  s.q_off = TileTraits<DT, HD>::kTileBytes;
  s.lse_off = s.q_off + kTwSlots * TileTraits<DT, HD>::kTileBytes;
  s.bar_off = s.lse_off + 2 * 128 * 4;
  s.misc_off = s.bar_off + 8 * (1 + 2 * kTwSlots + 4);
  s.total = s.misc_off + 16;
  return s;
}

// Sum of 2^(scale s + neg_lse) over the columns [c_first, c_end) of one S^T row; MASK false: all 128 columns.  `release`
// runs once the row has been read from TMEM.
template <bool MASK, class Release>
__device__ __forceinline__ float tile_sum(uint32_t t_s, const float* neg_lse, float scale, int c_first, int c_end, Release release) {
  const uint64_t sc2 = pack_f32x2(scale, scale);
  uint64_t acc0 = 0ull, acc1 = 0ull;
#pragma unroll
  for (int ch = 0; ch < 4; ++ch) {
    uint32_t s[32];
    tmem_ld_32x32(t_s + ch * 32, s);
    tmem_wait_ld();
    if (ch == 3) release();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 l = *reinterpret_cast<const float4*>(neg_lse + ch * 32 + i);
      float x0, x1, x2, x3;
      unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), sc2, pack_f32x2(l.x, l.y)), x0, x1);
      unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), sc2, pack_f32x2(l.z, l.w)), x2, x3);
      x0 = fast_exp2(x0); x1 = fast_exp2(x1); x2 = fast_exp2(x2); x3 = fast_exp2(x3);
      if (MASK) {   // a column that holds no visible query may hold anything
        const int c = ch * 32 + i;
        x0 = (c >= c_first && c < c_end) ? x0 : 0.f;
        x1 = (c + 1 >= c_first && c + 1 < c_end) ? x1 : 0.f;
        x2 = (c + 2 >= c_first && c + 2 < c_end) ? x2 : 0.f;
        x3 = (c + 3 >= c_first && c + 3 < c_end) ? x3 : 0.f;
      }
      acc0 = add_f32x2(acc0, pack_f32x2(x0, x1));
      acc1 = add_f32x2(acc1, pack_f32x2(x2, x3));
    }
  }
  float a, b, c, d;
  unpack_f32x2(acc0, a, b);
  unpack_f32x2(acc1, c, d);
  return (a + b) + (c + d);
}

// A barrier that a copy in flight will still complete: waited for after an abort, with a limit, so that nothing writes
// into shared memory that the CTA has given back.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < (1 << 16) && !mbar_try_wait(bar, parity); ++i) {}
}

// blockIdx: x share of the query tiles and kv head, y key tile (causal: heaviest first), z sequence.
template <int DT, int HD>
__global__ void __launch_bounds__(kTwThreads, HD > 128 ? 1 : 2)
token_weights_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const TokenWeightsParams p) {
  using T = TileTraits<DT, HD>;
  constexpr TwLayout L = tw_layout<DT, HD>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sm_lse = reinterpret_cast<float*>(smem + L.lse_off);          // [2][128], minus lse in log2 units
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L.bar_off);
  uint64_t* q_full = k_full + 1;
  uint64_t* q_empty = q_full + kTwSlots;
  uint64_t* s_full = q_empty + kTwSlots;   // [2]
  uint64_t* s_empty = s_full + 2;          // [2]
  uint32_t* sm_tmem_base = reinterpret_cast<uint32_t*>(smem + L.misc_off);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L.misc_off + 4);
  const WaitCtx wctx{abort_flag, p.status};

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.x / p.num_chunks, chunk = blockIdx.x - hk * p.num_chunks;
  const int k0 = blockIdx.y * 128, bi = blockIdx.z;
  int len = p.seqlens[bi];
  if (len > p.max_len) {
    len = p.max_len;
    if (threadIdx.x == 0) atomicOr(p.status, kRangeBit);
  }
  if (k0 >= len) return;
  const int q0 = p.cu_q[bi];
  int n = p.cu_q[bi + 1] - q0;
  if (n < 0 || q0 < 0 || static_cast<int64_t>(q0) + n > p.total_q) {
    n = 0;
    if (threadIdx.x == 0) atomicOr(p.status, kRangeBit);
  }
  const int shift = len - n;                                            // query i sits at position shift + i
  const int tt = p.tile_tokens;
  const int first = (p.causal && k0 > shift) ? (k0 - shift) / tt : 0;   // first query tile that sees a key of this tile
  const int tiles = (n + tt - 1) / tt;
  const int steps = tiles - first > chunk ? (tiles - first - chunk + p.num_chunks - 1) / p.num_chunks : 0;
  const int key = k0 + threadIdx.x;                                     // warps 0-3
  float sum = 0.f, comp = 0.f;
  bool ok = true;

  if (steps > 0) {
    if (threadIdx.x == 128) {
      *abort_flag = 0;
      mbar_init(smem_u32(k_full), 1);
      for (int i = 0; i < kTwSlots; ++i) {
        mbar_init(smem_u32(&q_full[i]), 1);
        mbar_init(smem_u32(&q_empty[i]), 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_u32(&s_full[i]), 1);
        mbar_init(smem_u32(&s_empty[i]), 128);
      }
      mbar_fence_init();
      tma_prefetch_desc(&tmap_q);
      tma_prefetch_desc(&tmap_k);
    }
    if (warp == 5) {
      tmem_alloc(smem_u32(sm_tmem_base), 256);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *sm_tmem_base;
    const uint32_t k_smem = smem_u32(smem), q_smem = smem_u32(smem + L.q_off);
    if (warp == 4) {
      if (lane == 0) {
        const int nbox = min(128 / p.box_rows, (len - k0 + p.box_rows - 1) / p.box_rows);
        mbar_expect_tx(smem_u32(k_full), static_cast<uint32_t>(nbox) * p.box_rows * 128u * T::kHalves);
        const int32_t* bt = p.block_table + bi * p.bt_stride;
        for (int i = 0; i < nbox; ++i) {
          const int tok = k0 + i * p.box_rows;
          const int page = bt[tok / p.page_size], row = tok % p.page_size;
          for (int hf = 0; hf < T::kHalves; ++hf)
            tma_load_4d(k_smem + hf * T::kHalfBytes + i * p.box_rows * 128, &tmap_k, smem_u32(k_full), hf * 64, hk, row, page);
        }
        const uint32_t q_bytes = static_cast<uint32_t>(tt) * p.group * 128u * T::kHalves;
        int j = 0;
        for (; j < steps; ++j) {
          const int slot = j % kTwSlots;
          if (!mbar_wait(smem_u32(&q_empty[slot]), ((j / kTwSlots) & 1) ^ 1u, wctx)) break;
          const uint32_t bar = smem_u32(&q_full[slot]);
          mbar_expect_tx(bar, q_bytes);
          const int tok = q0 + (first + chunk + j * p.num_chunks) * tt;
          for (int hf = 0; hf < T::kHalves; ++hf)
            tma_load_4d(q_smem + slot * T::kTileBytes + hf * T::kHalfBytes, &tmap_q, bar, hf * 64, hk * p.group, tok, 0);
        }
        if (j < steps) {   // gave up: the loads issued last may still be on their way
          drain(smem_u32(k_full), 0);
          for (int i = max(0, j - kTwSlots); i < j; ++i) drain(smem_u32(&q_full[i % kTwSlots]), (i / kTwSlots) & 1);
        }
      }
    } else if (warp == 5) {
      if (lane == 0) {
        bool go = mbar_wait(smem_u32(k_full), 0, wctx);
        int j = 0;
        for (; go && j < steps; ++j) {
          const int slot = j % kTwSlots, buf = j & 1;
          if (!mbar_wait(smem_u32(&q_full[slot]), (j / kTwSlots) & 1, wctx)) break;
          if (!mbar_wait(smem_u32(&s_empty[buf]), ((j >> 1) & 1) ^ 1u, wctx)) break;
          tc_fence_after();
          issue_qk<DT, HD>(k_smem, q_smem + slot * T::kTileBytes, tmem_base + buf * 128);   // rows: keys, columns: queries
          tc_commit(smem_u32(&q_empty[slot]));
          tc_commit(smem_u32(&s_full[buf]));
        }
        if (j < steps)     // gave up: products in flight end before TMEM is freed
          for (int i = max(0, j - 2); i < j; ++i) drain(smem_u32(&s_full[i & 1]), (i >> 1) & 1);
      }
      __syncwarp();
    } else {
      // this thread's column of every tile: token t_in of the tile, head h_in of the group
      const int t_in = threadIdx.x / p.group, h_in = threadIdx.x - t_in * p.group;
      const float* lse = p.lse + (static_cast<int64_t>(hk) * p.group + h_in) * p.lse_h + q0;
      const uint32_t t_s = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
      auto fetch = [&](int j) -> float {
        const int tok = (first + chunk + j * p.num_chunks) * tt + t_in;
        return (t_in < tt && tok < n) ? -__ldg(lse + tok) * kLog2e : -INFINITY;
      };
      float next = fetch(0);
      for (int j = 0; j < steps; ++j) {
        const int buf = j & 1;
        sm_lse[buf * 128 + threadIdx.x] = next;
        if (j + 1 < steps) next = fetch(j + 1);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        // after a wait that gave up the warps still meet at the barrier above, step by step
        ok = __all_sync(0xffffffffu, ok && mbar_wait(smem_u32(&s_full[buf]), (j >> 1) & 1, wctx));
        if (!ok) continue;
        tc_fence_after();
        const int tile0 = (first + chunk + j * p.num_chunks) * tt;
        const int c_first = p.causal ? max(0, min(key - shift - tile0, tt)) * p.group : 0;
        const int c_end = min(tt, n - tile0) * p.group;
        auto release = [&] {
          tc_fence_before();
          mbar_arrive(smem_u32(&s_empty[buf]));
        };
        const bool mask = c_end < 128 || (p.causal && k0 + warp * 32 + 31 - shift - tile0 > 0);   // the warp's last key
        const float part = mask ? tile_sum<true>(t_s + buf * 128, sm_lse + buf * 128, p.scale_log2, c_first, c_end, release)
                                : tile_sum<false>(t_s + buf * 128, sm_lse + buf * 128, p.scale_log2, 0, 128, release);
        // up to tens of thousands of queries: the total carries its rounding errors along
        const float total = __fadd_rn(sum, part);
        const float big = fmaxf(sum, part), small = fminf(sum, part);
        comp = __fadd_rn(comp, __fsub_rn(small, __fsub_rn(total, big)));
        sum = total;
      }
      __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
      tc_fence_after();
      tmem_dealloc(tmem_base, 256);
    }
  }
  if (warp < 4 && ok && key < len) {
    sum += comp;
    if (p.num_chunks > 1) {
      p.partial[((static_cast<int64_t>(chunk) * p.b + bi) * p.h_k + hk) * p.partial_stride + key] = sum;
    } else if (key < p.capacity) {
      const float before = p.w_in ? p.w_in[bi * p.win_b + hk * p.win_h + key] * p.decay : 0.f;
      p.w_out[bi * p.wout_b + hk * p.wout_h + key] = before + sum;
    }
  }
}

__global__ void __launch_bounds__(256) token_weights_join_kernel(const TokenWeightsParams p) {
  const int hk = blockIdx.y, bi = blockIdx.z, key = blockIdx.x * 256 + threadIdx.x;
  if (key >= min(min(p.seqlens[bi], p.max_len), p.capacity)) return;
  float sum = 0.f;
  for (int c = 0; c < p.num_chunks; ++c)
    sum += p.partial[((static_cast<int64_t>(c) * p.b + bi) * p.h_k + hk) * p.partial_stride + key];
  const float before = p.w_in ? p.w_in[bi * p.win_b + hk * p.win_h + key] * p.decay : 0.f;
  p.w_out[bi * p.wout_b + hk * p.wout_h + key] = before + sum;
}

template <int DT, int HD>
cudaError_t launch_tw(const CUtensorMap& tq, const CUtensorMap& tk, const TokenWeightsParams& p, cudaStream_t stream) {
  auto kern = token_weights_kernel<DT, HD>;
  const size_t smem = 1024 + tw_layout<DT, HD>().total;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_done[dev] = true;
  }
  kern<<<dim3(p.h_k * p.num_chunks, (p.max_len + 127) / 128, p.b), kTwThreads, smem, stream>>>(tq, tk, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_weights_finish(const WeightsFinishParams& p, cudaStream_t stream) {
  const int most = p.max_len < p.capacity ? p.max_len : p.capacity;
  if (most <= 0) return cudaSuccess;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((most + kFinishThreads - 1) / kFinishThreads, p.h_k, p.b);
  cfg.blockDim = dim3(kFinishThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.dependent_launch ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, weights_finish_kernel, p);
}

cudaError_t launch_token_weights(int dtype, const CUtensorMap& tq, const CUtensorMap& tk, const TokenWeightsParams& p,
                                 cudaStream_t stream) {
  const bool bf = dtype == FA_B200_BF16;
  cudaError_t e = cudaErrorInvalidValue;
  switch (p.d) {
    case 64: e = bf ? launch_tw<FA_B200_BF16, 64>(tq, tk, p, stream) : launch_tw<FA_B200_F16, 64>(tq, tk, p, stream); break;
    case 128: e = bf ? launch_tw<FA_B200_BF16, 128>(tq, tk, p, stream) : launch_tw<FA_B200_F16, 128>(tq, tk, p, stream); break;
    case 192: e = bf ? launch_tw<FA_B200_BF16, 192>(tq, tk, p, stream) : launch_tw<FA_B200_F16, 192>(tq, tk, p, stream); break;
    case 256: e = bf ? launch_tw<FA_B200_BF16, 256>(tq, tk, p, stream) : launch_tw<FA_B200_F16, 256>(tq, tk, p, stream); break;
  }
  if (e != cudaSuccess || p.num_chunks == 1) return e;
  const int most = p.max_len < p.capacity ? p.max_len : p.capacity;
  if (most <= 0) return cudaSuccess;
  token_weights_join_kernel<<<dim3((most + 255) / 256, p.h_k, p.b), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fa

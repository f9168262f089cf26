// The weight that every key of a decode call received, from the scores that the decode kernel left behind (log2 units,
// rows x tokens in fp32: 4 bytes per (query head, key) against 2 * d * element size of K and V per (kv head, key), which
// stays in L2 mostly, the pools' tiles being loaded to leave it first) and the rows' log-sum-exp:
// w[t] = decay w[t] + sum_r 2^(s_rt - lse_r), rows in a fixed order.  Bound by reading the scores: 16 ragged sequences of up to
// 32768 tokens, 184 us, of which the decode kernel takes 165 to 170 and this, with the merge of the partials, the rest (5 us more
// where the tiles of K and V compete with the scores for L2, 2 more where every row looks for its query token).
#pragma once

#include "fa_common.cuh"
#include "fa_kernels.h"

namespace fa {

constexpr int kFinishThreads = 128;
constexpr int kFinishTokens = 4 * kFinishThreads;   // of a CTA: four in a row per thread

// Of each row of the group: log-sum-exp, and the keys lo .. hi - 1 that it sees.
struct FinishRows { float lse[16]; int lo[16], hi[16]; };

// Log-sum-exp of the group's rows in log2 units: the merged one of an unsplit call, else from the partials
// (the sink as one more term); +inf: the row has no key.  All threads; the caller synchronises.
__device__ __forceinline__ void finish_lse(const WeightsFinishParams& p, int bi, int hk, int len, FinishRows& sh) {
  const int rows = p.sq * p.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < rows; r += kFinishThreads / 32) {   // row r is query token r / group, head r % group
    const int head = hk * p.group + r % p.group;
    const int64_t at = (static_cast<int64_t>(bi) * p.h + head) * p.sq + r / p.group;
    float l2;
    if (p.lse_partial == nullptr) {
      l2 = p.lse[at] * kLog2e;
    } else {
      const int n = min(p.num_parts, (len + p.partition_tokens - 1) / p.partition_tokens);
      float mx = -INFINITY;
      for (int i = lane; i < n; i += 32) {
        const float l = p.lse_partial[i * p.lse_part_stride + at];
        mx = fmaxf(mx, l == INFINITY ? -INFINITY : l);
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
      float sum = 0.f;
      for (int i = lane; i < n && mx != -INFINITY; i += 32) {
        const float l = p.lse_partial[i * p.lse_part_stride + at];
        sum += l == INFINITY ? 0.f : exp2f((l - mx) * kLog2e);
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      float m2 = mx * kLog2e;
      if (p.s_aux) {
        const float sink = load_sink_log2(p.s_aux, p.s_aux_dtype, head), m = fmaxf(m2, sink);
        sum = (m2 == -INFINITY ? 0.f : sum * exp2f(m2 - m)) + exp2f(sink - m);
        m2 = m;
      }
      l2 = sum > 0.f ? m2 + log2f(sum) : INFINITY;
      if (isnan(mx) || isnan(sum)) l2 = NAN;
    }
    if (lane == 0) {
      const int behind = p.sq - 1 - r / p.group;   // query tokens after this row's
      sh.lse[r] = l2;
      sh.hi[r] = p.causal ? len - behind : len;
      sh.lo[r] = p.window_left >= 0 ? len - behind - 1 - p.window_left : 0;
    }
  }
}

// Chunks first * loops .. of kFinishTokens tokens of one (sequence, kv head).  sh: shared memory.
__device__ __forceinline__ void finish_tokens(const WeightsFinishParams& p, int first, int hk, int bi, FinishRows& sh) {
  const int rows = p.sq * p.group;
  const int full = min(p.seqlens[bi], p.max_len), len = min(full, p.capacity);
  int tok = first * p.loops * kFinishTokens;
  if (tok >= len) return;
  tok += 4 * threadIdx.x;
  const float* in = p.w_in ? p.w_in + bi * p.win_b + hk * p.win_h : nullptr;
  float* out = p.w_out + bi * p.wout_b + hk * p.wout_h;
  const float* s = p.scores + (static_cast<int64_t>(bi) * p.h_k + hk) * rows * p.score_stride;
  const bool in16 = (reinterpret_cast<uintptr_t>(in) & 15) == 0, out16 = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const bool all = p.window_left < 0 && (p.sq == 1 || !p.causal);   // every row sees every key
  bool first_pass = true;
  for (int l = 0; l < p.loops; ++l, tok += kFinishTokens) {
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    if (in && tok < len) {   // on its way while the rows' log-sum-exps are looked up
      if (tok + 4 <= len && in16) {
        const float4 v = *reinterpret_cast<const float4*>(in + tok);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (tok + e < len) w[e] = in[tok + e];
      }
    }
    if (first_pass) {
      finish_lse(p, bi, hk, full, sh);
      __syncthreads();
      first_pass = false;
    }
    if (tok >= len) return;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const float* row = s + tok;   // rows are padded to whole tiles
    if (all) {
#pragma unroll 4
      for (int r = 0; r < rows; ++r, row += p.score_stride) {
        const float4 v = *reinterpret_cast<const float4*>(row);
        const float lse = sh.lse[r];
        sum[0] += exp2f(v.x - lse);
        sum[1] += exp2f(v.y - lse);
        sum[2] += exp2f(v.z - lse);
        sum[3] += exp2f(v.w - lse);
      }
    } else {
#pragma unroll 4
      for (int r = 0; r < rows; ++r, row += p.score_stride) {
        const float4 v = *reinterpret_cast<const float4*>(row);
        const float lse = sh.lse[r];
        const int lo = sh.lo[r], hi = sh.hi[r];
        const float x[4] = {exp2f(v.x - lse), exp2f(v.y - lse), exp2f(v.z - lse), exp2f(v.w - lse)};
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += (tok + e < hi && tok + e >= lo) ? x[e] : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = w[e] * p.decay + sum[e];
    if (tok + 4 <= len && out16) {
      *reinterpret_cast<float4*>(out + tok) = make_float4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (tok + e < len) out[tok + e] = w[e];
    }
  }
}

}  // namespace fa

// The weight that every cached key receives: sums of softmax probabilities over query rows.  After a decode call:
// fa_weights_finish.cuh.
//
// Of a prompt.  Given every query's log-sum-exp the weight of key t is a plain sum over the queries, with no running
// maximum: a CTA takes 128 keys of one kv head (256 above d = 128) as the A operand and walks the query tiles that see them,
// S^T = K Q^T in TMEM.  A TMEM lane is then a key, so a key's sum stays in a thread's registers: no atomics, no second pass.
// A query tile holds 128 / group tokens of all heads of the group (rows token-major), which fills it for short windows too
// and makes the causal mask a column bound per key.
//   warps 0-7  2^(s - lse) and its sum, one thread per key: two sets of four warps that take turns at the tiles (above
//              d = 128: one set for each 128 keys)
//   warp 8     TMA producer: key tiles (through the block table) and query tiles into a pool of tile buffers
//   warp 9     MMA issuer, an S^T buffer per set (two above d = 128)
// Two persistent CTAs per SM (one above d = 128) walk the items (key tiles, kv head, share of the query tiles) of the batch,
// so that the loads and the first product of an item run during the sums of the one before.  Long prompts: items go back and
// forth over the CTAs, heaviest first under a causal mask, and a key tile's query tiles are cut into shares (every
// num_chunks-th tile), whose sums a small kernel adds in order.  Short windows (one query tile per sequence): a CTA takes
// consecutive key tiles of one kv head and keeps the query tile, which leaves the keys as the only traffic; the CTAs of a
// token's kv heads, whose rows lie side by side in memory, walk the same tiles.
//
// What a role's threads do from item to item is bound by instruction latency (a dozen cycles each beside 16 busy warps): the
// walk over key tiles has no division, which took short windows from 37 to 34 us (bursts, keys partly in L2).
//
// Bound by latency beside the exponentials: 128 x 128 of them per tile take 1024 cycles of an SM's MUFU unit; the tcgen05 product
// takes 512, as long as its two operands take out of shared memory.  One prompt of 8192 tokens (32 heads, 8 kv heads, d = 128,
// causal): 416 us in a series of calls (1.84 GHz under the power cap), 387 in a burst at 1.965 GHz, 59 % of what the MUFU units
// could do; counters: MUFU pipe 67 % active, tensor pipe 33 %, issue slots 46 %, stalls on fixed latencies, on TMEM and
// log-sum-exp loads and on shared memory.  Measured in bursts, against 404 us then: a CTA per key tile 424 us, one CTA per SM with 256 keys 536, eight warps per SM 436, two warps per row with half of the
// columns each 408.  Exponentials on the FMA pipe (a degree-5 polynomial) cost more issue slots than the MUFU time they save: one
// group of columns in eight 416 us against 404.  A quarter of the columns for four rows per thread (16x256b loads) halves the
// shared-memory reads of the log-sum-exps and measured 399 against 404, but the registers that it takes cost short windows 50 us
// against 43.  The issuing threads' fixed walk through the buffers then took 404 to 387.  32 queries against 4 x 16384 keys (134 MB
// of keys): 39 us with keys that L2 does not hold; a CTA per key tile 78.
#include "fa_prefill_common.cuh"

namespace fa {
namespace {

// 128-key halves of a CTA: two CTAs per SM with one up to d = 128, one CTA with two above (shared memory).  Eight warps take
// the sums either way: with one half, two sets of four warps take turns at the tiles, all columns of a tile each, and their sums
// meet at the item's end (16 warps per SM keep the MUFU unit busier than 8 do).
__host__ __device__ constexpr int tw_halves(int hd) { return hd > 128 ? 2 : 1; }
constexpr int kTwThreads = 320;
constexpr int kTwMaxTiles = 4;
// Tile buffers for keys and queries.
__host__ __device__ constexpr int tw_tiles(int hd) { return hd == 192 ? 4 : 3; }
struct TwLayout { int lse_off, bar_off, misc_off, total; };
template <int DT, int HD>
__host__ __device__ constexpr TwLayout tw_layout() {
  TwLayout s{};
  s.lse_off = tw_tiles(HD) * TileTraits<DT, HD>::kTileBytes;
  s.bar_off = s.lse_off + 8 * 2 * 128 * 4 + 2 * 128 * 4;
  s.misc_off = s.bar_off + 8 * (2 * kTwMaxTiles + 8);
  s.total = s.misc_off + 16;
  return s;
}

// Sum of 2^(scale s + neg_lse) over the columns [c_first, c_end) of an S^T row; MASK false: all 128 columns.  `release` runs
// once the row has been read from TMEM.
template <bool MASK, class Release>
__device__ __forceinline__ float tile_sum(uint32_t t_s, const float* neg_lse, float scale, int c_first, int c_end, Release release) {
  const uint64_t sc2 = pack_f32x2(scale, scale);
  uint64_t acc0 = 0ull, acc1 = 0ull;
#pragma unroll 1
  for (int ch = 0; ch < 4; ++ch) {   // a loop, for the instruction cache
    uint32_t v[32];
    tmem_ld_32x32(t_s + ch * 32, v);
    tmem_wait_ld();
    if (ch == 3) release();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 l = *reinterpret_cast<const float4*>(neg_lse + ch * 32 + i);
      float x0, x1, x2, x3;
      unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), sc2, pack_f32x2(l.x, l.y)), x0, x1);
      unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), sc2, pack_f32x2(l.z, l.w)), x2, x3);
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

// A barrier that a copy or product in flight will still complete: waited for, with a limit, by the thread that issued it before
// the CTA ends, so that nothing writes into memory that the CTA has given back, also where another warp has given up on a wait.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < (1 << 16) && !mbar_try_wait(bar, parity); ++i) {}
}

__device__ __forceinline__ bool page_ok(const TokenWeightsParams& p, int32_t id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_blocks); }

// The sequence's tokens and queries as every role of the kernel sees them.
struct TwSeq { int len, q0, n, tiles; };
__device__ __forceinline__ TwSeq tw_seq(const TokenWeightsParams& p, int b) {
  TwSeq s;
  s.len = min(max(p.seqlens[b], 0), p.max_len);
  s.q0 = p.cu_q[b];
  s.n = p.cu_q[b + 1] - s.q0;
  if (s.n < 0 || s.n > p.max_q || s.q0 < 0 || static_cast<int64_t>(s.q0) + s.n > p.total_q) s.n = 0;   // reported by tw_report
  s.tiles = (s.n + p.tile_tokens - 1) / p.tile_tokens;
  return s;
}

// One CTA's walk over its items and their query tiles.  KEYS: keys of an item.
template <int KEYS>
struct TwWalk {
  int item, end, round;          // this item, the share's end (resident) or the batch's, rounds of the grid
  int b, base, here;             // sequence, its first item, its number of items
  int key_tiles;
  TwSeq s;
  int hk, chunk, k0, first, steps, j;
  __device__ __forceinline__ void enter(const TokenWeightsParams& p, int sequence) {
    b = sequence;
    s = tw_seq(p, b);
    key_tiles = (s.len + KEYS - 1) / KEYS;
    here = p.resident ? key_tiles : key_tiles * p.h_k * p.num_chunks;
  }
  // Moves to the next query tile, or the next item (steps may be 0: no query sees its keys).  false: done.
  __device__ __forceinline__ bool next(const TokenWeightsParams& p) { return ++j < steps || next_item(p); }
  __device__ __forceinline__ bool next_item(const TokenWeightsParams& p) {
    if (p.resident) {              // the next key tile, one step or none: no division, a single thread waits for each of them
      if (++item >= end) return false;
      k0 += KEYS;
      while (item >= base + here) {
        base += here;
        enter(p, b + 1);
        k0 = (item - base) * KEYS;
      }
      steps = s.tiles > 0 && !(p.causal && k0 - (s.len - s.n) >= p.tile_tokens) ? 1 : 0;
      j = 0;
      return true;
    }
    // back and forth, so that no CTA has the heavier item of every round
    const int g = gridDim.x;
    item = round * g + ((round & 1) ? g - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
    ++round;
    if (item >= end) return false;
    while (item >= base + here) {
      base += here;
      enter(p, b + 1);
    }
    // key tiles outermost: heaviest first under a causal mask
    int i = item - base;
    const int per = p.h_k * p.num_chunks;
    const int kt = i / per;
    i -= kt * per;
    hk = p.num_chunks > 1 ? i / p.num_chunks : i;
    chunk = i - hk * p.num_chunks;
    k0 = kt * KEYS;
    const int shift = s.len - s.n;                                   // query i sits at position shift + i
    first = ((p.causal && k0 > shift) ? (k0 - shift) / p.tile_tokens : 0) + chunk;
    steps = max(s.tiles - first, 0);
    if (p.num_chunks > 1) steps = (steps + p.num_chunks - 1) / p.num_chunks;
    j = 0;
    return true;
  }
  __device__ __forceinline__ bool begin(const TokenWeightsParams& p, int total) {
    if (p.resident) {              // a contiguous share of the key tiles, of one kv head
      const int64_t g = gridDim.y;
      item = static_cast<int>(total * static_cast<int64_t>(blockIdx.y) / g) - 1;
      end = static_cast<int>(total * static_cast<int64_t>(blockIdx.y + 1) / g);
      k0 = static_cast<int>(static_cast<uint32_t>(item) * KEYS);   // set anew in the item's sequence, unless that is the first
      hk = blockIdx.x;
      chunk = 0;
      first = 0;
    } else {
      round = 0;
      end = total;
    }
    base = 0; steps = 0; j = 0;
    enter(p, 0);
    return next_item(p);
  }
  __device__ __forceinline__ int tile_token(const TokenWeightsParams& p) const { return (first + j * p.num_chunks) * p.tile_tokens; }
  // Whether the second 128 keys exist, and whether a query of this tile sees one of them.
  __device__ __forceinline__ bool second() const { return KEYS > 128 && k0 + 128 < s.len; }
  __device__ __forceinline__ bool active(const TokenWeightsParams& p, int half) const {
    if (steps == 0) return false;
    if (half == 0) return true;
    return second() && (!p.causal || tile_token(p) + p.tile_tokens > k0 + 128 - (s.len - s.n));
  }
};

// Tile buffers as producer and MMA issuer both go through them: a load takes the buffer whose last use lies furthest back
// (keys are used until their item's last step, a resident query tile until the kv head changes).
template <int N>
struct TwBuffers {
  int last[N], loads[N];
  __device__ __forceinline__ TwBuffers() {
#pragma unroll
    for (int i = 0; i < N; ++i) { last[i] = -1; loads[i] = 0; }
  }
  __device__ __forceinline__ int take(int until) {
    int s = 0, least = last[0];
#pragma unroll
    for (int i = 1; i < N; ++i)
      if (last[i] < least) { s = i; least = last[i]; }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i == s) { last[i] = until; ++loads[i]; }
    return s;
  }
  __device__ __forceinline__ int count(int s) const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n = i == s ? loads[i] : n;
    return n;
  }
  __device__ __forceinline__ void ends(int s, int at) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i == s) last[i] = at;
  }
};

template <int DT, int HD>
__global__ void __launch_bounds__(kTwThreads, HD > 128 ? 1 : 2)
token_weights_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const TokenWeightsParams p) {
  using T = TileTraits<DT, HD>;
  constexpr TwLayout L = tw_layout<DT, HD>();
  constexpr int kTiles = tw_tiles(HD), kHalvesOfKeys = tw_halves(HD), kProducer = 8, kMma = 9;
  constexpr bool kTurns = kHalvesOfKeys == 1;     // two sets of four warps take turns at the tiles of one set of keys
  constexpr int kCols = 256 * kHalvesOfKeys;   // TMEM
  constexpr int kForever = 0x7fffffff;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bar_off);   // [kTiles]
  uint64_t* empty = full + kTwMaxTiles;                             // [kTiles]
  uint64_t* s_full = empty + kTwMaxTiles;                           // [2 halves][2]
  uint64_t* s_empty = s_full + 4;                                   // [2 halves][2]
  uint32_t* sm_tmem_base = reinterpret_cast<uint32_t*>(smem + L.misc_off);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L.misc_off + 4);
  int* sm_total = reinterpret_cast<int*>(smem + L.misc_off + 8);
  // Not 0: the producer has met an id that is no page.  Its keys are loaded as zeros, and whoever writes sums from then on looks
  // its key's id up and writes no sum for such a key.
  volatile int* sm_bad = reinterpret_cast<volatile int*>(smem + L.misc_off + 12);
  const WaitCtx wctx{abort_flag, p.status};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  griddep_wait();
  griddep_launch_dependents();
  if (threadIdx.x == 32 * kProducer) {
    *abort_flag = 0;
    *sm_bad = 0;
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&s_empty[i]), 128);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
  }
  if (warp == kMma) {
    tmem_alloc(smem_u32(sm_tmem_base), kCols);
    tmem_relinquish();
  }
  if (warp == 0) {   // number of items of the batch; what is wrong with the lengths on the device is reported once
    int total = 0;
    for (int b = lane; b < p.b; b += 32) {
      const TwSeq s = tw_seq(p, b);
      total += (s.len + 128 * kHalvesOfKeys - 1) / (128 * kHalvesOfKeys) * (p.resident ? 1 : p.h_k * p.num_chunks);
      const int n = p.cu_q[b + 1] - p.cu_q[b];
      if (blockIdx.x == 0 && blockIdx.y == 0 && (p.seqlens[b] > p.max_len || n != s.n)) atomicOr(p.status, kRangeBit);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    if (lane == 0) *sm_total = total;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *sm_tmem_base;
  const int total = *sm_total;
  const uint32_t tiles_smem = smem_u32(smem);
  auto report_page = [&] {
    *sm_bad = 1;
    atomicOr(p.status, kRangeBit);
  };

  // Up to d = 128 (kTurns) the three tile buffers go round by rule: an item's keys take the buffer that has been out of use
  // longest, its query tiles alternate between the other two; resident: the keys alternate between 0 and 1, the query tile
  // stays in 2.  `loaded` has the parity of every buffer's number of loads.
  if (kTurns && warp == kProducer) {
    if (lane == 0) {
      TwWalk<128> w{};
      int t = 0, q_key = -1, k = 0, q0 = 1, q1 = 2;
      const int tile_boxes = 128 / p.box_rows;
      int after_k0 = -1, after_b = -1, index = 0, row = 0;   // the key tile behind the last one: its first page and the row in it
      uint32_t loaded = 0, used = 0;
      const uint32_t q_bytes = static_cast<uint32_t>(p.tile_tokens) * p.group * 128u * T::kHalves;
      bool ok = true;
      auto reserve = [&](int slot) {
        if ((used >> slot) & 1u) ok = ok && mbar_wait(smem_u32(&empty[slot]), ((loaded >> slot) & 1u) ^ 1u, wctx);
        if (!ok) return;
        loaded ^= 1u << slot;
        used |= 1u << slot;
      };
      for (bool more = w.begin(p, total); more && ok; more = w.next_item(p)) {
        if (w.steps == 0) continue;
        if (p.resident) k = t & 1;
        {
          // the page ids are looked up before the wait for a buffer
          const int nbox = w.s.len - w.k0 >= 128 ? tile_boxes : (w.s.len - w.k0 + p.box_rows - 1) / p.box_rows;
          const int32_t* bt = p.block_table + w.b * p.bt_stride;
          if (w.k0 != after_k0 || w.b != after_b) {
            index = w.k0 / p.page_size;
            row = w.k0 - index * p.page_size;
          }
          int page[8], at[8];
          bool pages_ok = true;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i >= nbox) break;
            page[i] = __ldg(bt + index);
            pages_ok = pages_ok && page_ok(p, page[i]);
            at[i] = row;
            row += p.box_rows;      // boxes divide pages
            if (row >= p.page_size) { row = 0; ++index; }
          }
          after_k0 = w.k0 + 128;
          after_b = w.b;
          reserve(k);
          if (!ok) break;
          if (!pages_ok) report_page();
          const uint32_t bar = smem_u32(&full[k]);
          mbar_expect_tx(bar, static_cast<uint32_t>(nbox) * p.box_rows * 128u * T::kHalves);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i >= nbox) break;
#pragma unroll
            for (int hf = 0; hf < T::kHalves; ++hf)
              tma_load_4d(tiles_smem + k * T::kTileBytes + hf * T::kHalfBytes + i * p.box_rows * 128, &tmap_k, bar, hf * 64, w.hk, at[i], page[i]);
          }
        }
        const int key = w.b * p.h_k + w.hk;
        int tok = w.s.q0 + w.first * p.tile_tokens;
        for (int j = 0; j < w.steps && ok; ++j, tok += p.num_chunks * p.tile_tokens) {
          if (p.resident && key == q_key) continue;
          const int slot = p.resident ? 2 : ((j & 1) ? q1 : q0);
          reserve(slot);
          if (!ok) break;
          const uint32_t bar = smem_u32(&full[slot]);
          mbar_expect_tx(bar, q_bytes);
#pragma unroll
          for (int hf = 0; hf < T::kHalves; ++hf)
            tma_load_4d(tiles_smem + slot * T::kTileBytes + hf * T::kHalfBytes, &tmap_q, bar, hf * 64, w.hk * p.group, tok, 0);
        }
        q_key = key;
        t += w.steps;
        const int last = (w.steps & 1) ? q0 : q1, other = (w.steps & 1) ? q1 : q0, old_k = k;
        k = other; q0 = old_k; q1 = last;
      }
      for (int i = 0; i < 3; ++i)   // the loads issued last, whoever gives up on them meanwhile
        if ((used >> i) & 1u) drain(smem_u32(&full[i]), ((loaded >> i) & 1u) ^ 1u);
    }
  } else if (kTurns && warp == kMma) {
    if (lane == 0) {
      TwWalk<128> w{};
      int t = 0, q_key = -1, k = 0, q0 = 1, q1 = 2;
      uint32_t loaded = 0;
      bool ok = true;
      auto landed = [&](int slot) {   // the next load of a buffer
        loaded ^= 1u << slot;
        ok = ok && mbar_wait(smem_u32(&full[slot]), ((loaded >> slot) & 1u) ^ 1u, wctx);
      };
      for (bool more = w.begin(p, total); more && ok; more = w.next_item(p)) {
        if (w.steps == 0) continue;
        const int key = w.b * p.h_k + w.hk;
        if (p.resident) {
          k = t & 1;
          if (key != q_key) {
            if (q_key >= 0) tc_commit(smem_u32(&empty[2]));   // the products that read the old query tile have been issued
            landed(2);
          }
        }
        q_key = key;
        landed(k);
        for (int j = 0; j < w.steps && ok; ++j, ++t) {
          const int slot = p.resident ? 2 : ((j & 1) ? q1 : q0), buf = t & 1;
          if (!p.resident) landed(slot);
          ok = ok && mbar_wait(smem_u32(&s_empty[buf]), ((t >> 1) & 1) ^ 1u, wctx);
          if (!ok) break;
          tc_fence_after();
          issue_qk<DT, HD>(tiles_smem + k * T::kTileBytes, tiles_smem + slot * T::kTileBytes, tmem_base + buf * 128);
          tc_commit(smem_u32(&s_full[buf]));
          if (!p.resident) tc_commit(smem_u32(&empty[slot]));
        }
        if (!ok) break;
        tc_commit(smem_u32(&empty[k]));
        const int last = (w.steps & 1) ? q0 : q1, other = (w.steps & 1) ? q1 : q0, old_k = k;
        k = other; q0 = old_k; q1 = last;
      }
      for (int i = max(0, t - 2); i < t; ++i) drain(smem_u32(&s_full[i & 1]), (i >> 1) & 1);
    }
    __syncwarp();
  } else if (warp == kProducer) {
    if (lane == 0) {
      TwWalk<128 * kHalvesOfKeys> w{};
      TwBuffers<kTiles> buf;
      int t = 0, q_key = -1, q_slot = 0;     // step; (sequence, kv head) of the resident query tile
      const uint32_t q_bytes = static_cast<uint32_t>(p.tile_tokens) * p.group * 128u * T::kHalves;
      bool ok = true;
      auto reserve = [&](int until) -> int {
        const int slot = buf.take(until), n = buf.count(slot);
        if (n > 1 && !mbar_wait(smem_u32(&empty[slot]), n & 1, wctx)) ok = false;
        return slot;
      };
      auto load_keys = [&](int k0) {
        const int slot = reserve(t + w.steps - 1);
        if (!ok) return;
        const uint32_t bar = smem_u32(&full[slot]);
        const int nbox = min(128 / p.box_rows, (w.s.len - k0 + p.box_rows - 1) / p.box_rows);
        const int32_t* bt = p.block_table + w.b * p.bt_stride;
        for (int i = 0; i < nbox; ++i)
          if (!page_ok(p, __ldg(bt + (k0 + i * p.box_rows) / p.page_size))) report_page();
        mbar_expect_tx(bar, static_cast<uint32_t>(nbox) * p.box_rows * 128u * T::kHalves);
        for (int i = 0; i < nbox; ++i) {
          const int tok = k0 + i * p.box_rows;
          const int page = bt[tok / p.page_size], row = tok % p.page_size;
          for (int hf = 0; hf < T::kHalves; ++hf)
            tma_load_4d(tiles_smem + slot * T::kTileBytes + hf * T::kHalfBytes + i * p.box_rows * 128, &tmap_k, bar, hf * 64, w.hk, row, page);
        }
      };
      for (bool more = w.begin(p, total); more; more = w.next(p)) {
        if (w.steps == 0) continue;
        const int key = w.b * p.h_k + w.hk;
        const bool load_q = !p.resident || key != q_key;
        if (p.resident && load_q && q_key >= 0) buf.ends(q_slot, t - 1);
        if (w.j == 0) {
          load_keys(w.k0);
          if (ok && w.second()) load_keys(w.k0 + 128);
        }
        if (ok && load_q) {
          q_key = key;
          q_slot = reserve(p.resident ? kForever : t);
          if (ok) {
            const uint32_t bar = smem_u32(&full[q_slot]);
            mbar_expect_tx(bar, q_bytes);
            for (int hf = 0; hf < T::kHalves; ++hf)
              tma_load_4d(tiles_smem + q_slot * T::kTileBytes + hf * T::kHalfBytes, &tmap_q, bar, hf * 64, w.hk * p.group,
                          w.s.q0 + w.tile_token(p), 0);
          }
        }
        if (!ok) break;
        ++t;
      }
      for (int i = 0; i < kTiles; ++i)   // the loads issued last (one reserved and, after a wait given up, not issued just runs out)
        if (buf.count(i) > 0) drain(smem_u32(&full[i]), (buf.count(i) - 1) & 1);
    }
  } else if (warp == kMma) {
    if (lane == 0) {
      TwWalk<128 * kHalvesOfKeys> w{};
      TwBuffers<kTiles> buf;
      int t = 0, q_key = -1, k_slot[2] = {0, 0}, q_slot = 0, n_half[2] = {0, 0};
      bool ok = true, two = false, seen = false;   // seen: the second keys of this item have landed (a step has used them)
      bool more = w.begin(p, total);
      while (more && w.steps == 0) more = w.next(p);
      while (more && ok) {
        const int key = w.b * p.h_k + w.hk;
        const bool load_q = !p.resident || key != q_key;
        if (p.resident && load_q && q_key >= 0) buf.ends(q_slot, t - 1);
        if (w.j == 0) {
          two = w.second();
          seen = false;
          k_slot[0] = buf.take(t + w.steps - 1);
          if (two) k_slot[1] = buf.take(t + w.steps - 1);
        }
        if (load_q) {
          q_key = key;
          q_slot = buf.take(p.resident ? kForever : t);
        }
        ok = mbar_wait(smem_u32(&full[q_slot]), (buf.count(q_slot) - 1) & 1, wctx);
#pragma unroll
        for (int half = 0; half < kHalvesOfKeys; ++half) {
          if (!ok || !w.active(p, half)) continue;
          const int n = n_half[half]++, sb = 2 * half + (n & 1);
          ok = mbar_wait(smem_u32(&full[k_slot[half]]), (buf.count(k_slot[half]) - 1) & 1, wctx) &&
               mbar_wait(smem_u32(&s_empty[sb]), ((n >> 1) & 1) ^ 1u, wctx);
          if (!ok) { --n_half[half]; break; }
          tc_fence_after();
          issue_qk<DT, HD>(tiles_smem + k_slot[half] * T::kTileBytes, tiles_smem + q_slot * T::kTileBytes, tmem_base + sb * 128);
          tc_commit(smem_u32(&s_full[sb]));
          if (half == 1) seen = true;
        }
        const bool k_done = w.j == w.steps - 1;
        // A share of the query tiles may hold none that sees the second keys.  Their load is waited for all the same before the
        // buffer goes back: the producer must not arm its barrier again, nor the CTA end, while the bytes are on their way.
        if (ok && k_done && two && !seen) ok = mbar_wait(smem_u32(&full[k_slot[1]]), (buf.count(k_slot[1]) - 1) & 1, wctx);
        if (!ok) break;
        do { more = w.next(p); } while (more && w.steps == 0);
        if (k_done) {
          tc_commit(smem_u32(&empty[k_slot[0]]));
          if (two) tc_commit(smem_u32(&empty[k_slot[1]]));
        }
        if (!p.resident || !more || w.b * p.h_k + w.hk != q_key) tc_commit(smem_u32(&empty[q_slot]));
        ++t;
      }
      for (int half = 0; half < kHalvesOfKeys; ++half)
        for (int i = max(0, n_half[half] - 2); i < n_half[half]; ++i) drain(smem_u32(&s_full[2 * half + (i & 1)]), (i >> 1) & 1);
    }
    __syncwarp();
  } else {
    // Key half * 128 + row of the item's.  kTurns: set 0 takes the even steps of the CTA's walk and set 1 the odd ones (each
    // has one S^T buffer), so that one set's exponentials fill the other's waits; the sums meet at the item's end.  Items of
    // one step (resident) belong to one set.
    const int set = warp >> 2, half = kTurns ? 0 : set, row = threadIdx.x & 127;
    // this lane's four columns, whose log-sum-exp it fetches for the warp: token and head
    int t_in[4];
    int64_t h_off[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = lane * 4 + e;
      t_in[e] = c / p.group;
      h_off[e] = static_cast<int64_t>(c - t_in[e] * p.group) * p.lse_h + t_in[e];
    }
    float* sm_lse = reinterpret_cast<float*>(smem + L.lse_off) + warp * 256;   // this warp's own: [2][128]
    float* sm_sum = reinterpret_cast<float*>(smem + L.lse_off) + 8 * 256;      // [2][128]: sums of set 1
    const uint32_t t_s = tmem_base + half * 256 + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    TwWalk<128 * kHalvesOfKeys> w{};
    int t = 0, q_key = -1, items = 0, stage = 0;   // t: the CTA's steps before this item (kTurns), or this half's
    bool ok = true;
    float next[4];       // log-sum-exp of the lane's columns in the tile to come; +inf: no query
    const float* lse = nullptr;
    auto fetch = [&](int tok0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        next[e] = (t_in[e] < p.tile_tokens && tok0 + t_in[e] < w.s.n) ? __ldg(lse + h_off[e] + tok0) : INFINITY;
    };
    const int tile_step = p.num_chunks * p.tile_tokens * (kTurns ? 2 : 1);
    for (bool more = w.begin(p, total); more; more = w.next_item(p)) {   // after an abort the sets still meet, item by item
      const int key = w.k0 + half * 128 + row;
      float sum = 0.f, comp = 0.f;
      int j = 0;   // first step of this set or half
      if (kTurns) {
        j = (set ^ t) & 1;
        if (p.resident && (w.steps > 0 ? j : set) != 0) {   // the other set's item
          t += w.steps;
          continue;
        }
      } else if (half > 0) {   // steps whose last query sees the half's first key
        if (!w.second()) continue;
        if (p.causal)
          while (j < w.steps && w.first * p.tile_tokens + j * tile_step + p.tile_tokens <= w.k0 + 128 - (w.s.len - w.s.n)) ++j;
      }
      // what the sum is added to, on its way during the steps
      const bool writes = !kTurns || p.resident || set == 0;
      const bool adds = p.w_in && p.num_chunks == 1 && writes && key < w.s.len && key < p.capacity;
      float before = 0.f;   // no use of it up here: a load that is on its way
      if (adds) asm volatile("ld.global.f32 %0, [%1];" : "=f"(before) : "l"(p.w_in + w.b * p.win_b + w.hk * p.win_h + key));
      int tile0 = (w.first + j * p.num_chunks) * p.tile_tokens;
      if (j < w.steps && (!p.resident || w.b * p.h_k + w.hk != q_key)) {
        q_key = w.b * p.h_k + w.hk;
        lse = p.lse + static_cast<int64_t>(w.hk) * p.group * p.lse_h + w.s.q0;
        fetch(tile0);
      }
      int ahead = key - (w.s.len - w.s.n) - tile0;   // this key's position relative to the tile's first query
      for (; j < w.steps && ok; j += kTurns ? 2 : 1, tile0 += tile_step, ahead -= tile_step) {
        const int step = kTurns ? t + j : t, buf = step & 1;
        stage ^= 128;
        float4 neg;
        neg.x = -next[0] * kLog2e; neg.y = -next[1] * kLog2e; neg.z = -next[2] * kLog2e; neg.w = -next[3] * kLog2e;
        *reinterpret_cast<float4*>(sm_lse + stage + lane * 4) = neg;
        if (j + (kTurns ? 2 : 1) < w.steps) fetch(tile0 + tile_step);
        const int c_end = min(p.tile_tokens, w.s.n - tile0) * p.group;
        const int c_first = p.causal ? max(0, min(ahead, p.tile_tokens)) * p.group : 0;
        const bool mask = c_end < 128 || __any_sync(0xffffffffu, c_first > 0);
        __syncwarp();
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[2 * half + buf]), (step >> 1) & 1, wctx));
        if (!ok) break;
        tc_fence_after();
        auto release = [&] {
          tc_fence_before();
          mbar_arrive(smem_u32(&s_empty[2 * half + buf]));
        };
        const float part = mask ? tile_sum<true>(t_s + buf * 128, sm_lse + stage, p.scale_log2, c_first, c_end, release)
                                : tile_sum<false>(t_s + buf * 128, sm_lse + stage, p.scale_log2, 0, 128, release);
        // up to tens of thousands of queries: the total carries its rounding errors along
        const float now = __fadd_rn(sum, part);
        const float big = fmaxf(sum, part), small = fminf(sum, part);
        comp = __fadd_rn(comp, __fsub_rn(small, __fsub_rn(now, big)));
        sum = now;
        if (!kTurns) ++t;
      }
      if (kTurns) t += w.steps;
      sum += comp;
      if (kTurns && !p.resident) {   // two buffers, so one meeting per item
        float* s = sm_sum + (items++ & 1) * 128;
        if (set == 1) s[row] = sum;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
        if (set == 1) continue;
        sum += s[row];
      }
      if (ok && key < w.s.len) {
        // set ahead of the load of the keys, whose product this warp has waited for, or the one that it has just met
        if (*sm_bad != 0 && !page_ok(p, __ldg(p.block_table + w.b * p.bt_stride + key / p.page_size))) sum = 0.f;
        if (p.num_chunks > 1)
          p.partial[((static_cast<int64_t>(w.chunk) * p.b + w.b) * p.h_k + w.hk) * p.partial_stride + key] = sum;
        else if (key < p.capacity)
          p.w_out[w.b * p.wout_b + w.hk * p.wout_h + key] = fmaf(before, p.decay, sum);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kCols);
  }
}

__global__ void __launch_bounds__(256) token_weights_join_kernel(const TokenWeightsParams p) {
  const int hk = blockIdx.y, bi = blockIdx.z, key = blockIdx.x * 256 + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
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
  const int64_t tiles = static_cast<int64_t>((p.max_len + p.item_keys - 1) / p.item_keys) * p.b;   // of keys
  const int64_t slots = 148 * (HD > 128 ? 1 : 2);
  cudaLaunchConfig_t cfg{};
  if (p.resident) {
    const int64_t shares = max(min(slots / p.h_k, tiles), int64_t{1});
    cfg.gridDim = dim3(static_cast<unsigned>(p.h_k), static_cast<unsigned>(shares));
  } else {
    cfg.gridDim = dim3(static_cast<unsigned>(min(tiles * p.h_k * p.num_chunks, slots)));
  }
  cfg.blockDim = dim3(kTwThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.dependent_launch ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, tq, tk, p);
}

}  // namespace

int token_weights_item_keys(int d) { return 128 * tw_halves(d); }

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
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((most + 255) / 256, p.h_k, p.b);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.dependent_launch ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, token_weights_join_kernel, p);
}

}  // namespace fa

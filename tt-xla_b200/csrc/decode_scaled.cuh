// Paged GQA decode attention over an 8-bit KV cache with one fp32 scale for each page and KV head
// (what paged_write_kernel writes), int8 or e4m3, head_size 64 or 128.
//
//   s_j = (q . c_j) * scale * ks(page of j)        c: codes, ks / vs: the page's K / V scale
//   out = sum_j 2^(s_j - m) vs(page of j) c'_j / sum_j 2^(s_j - m)
//
// HBM-bound: a key and value cost 2 * head_size bytes and are read once.  As in the bf16 kernel a
// CTA works on one KV head of one user at a time, a producer warp keeps a ring of tiles full with
// TMA, and four warps take a quarter of a tile each.  What differs:
//   * the launch is one CTA per resident slot and the tiles of all (user, KV head) pairs, end to
//     end, are dealt to them in equal shares: no wave is partly filled and ragged contexts balance.
//     A share covers the end of one pair, whole pairs and the start of another; the ring runs on
//     across them.  A pair that several CTAs share is merged by the one that finishes last;
//   * the products are transposed: S^T = K Q^T and O^T = V^T P^T, tokens resp. head elements in
//     the 16 rows of m16n8k16 and the query heads in its 8 columns.  Up to 8 query heads per KV
//     head then fill an MMA (otherwise half of the 16 rows would be padding), and the
//     accumulators of 128 x 8 outputs are 32 registers;
//   * codes become f16 in registers, exactly.  A 16-bit `ldmatrix` hands a thread four consecutive
//     bytes b0..b3 of a token (K), or 2 elements of 2 tokens (V, transposed).  Bytes 0 and 2 of a
//     word make one f16 pair and bytes 1 and 3 the other: for int8 that is two LOP3 (code + 1152
//     as f16 bits) and two subtractions per word and no byte shuffles.  The resulting order of
//     the contraction index (K) is matched by the order the Q fragments are loaded in, and that of
//     the head elements (V) is undone at the store;
//   * the K scale multiplies S in fp32.  The V scale goes into the exponent of the weights,
//     P' = 2^((s - m) + log2 vs - r), with a maximum r of its own (relative to m, so that scores of
//     any size leave the scale its bits): the f16 weights are then at most 2^8 whatever the scales
//     are, and a page's values keep 11 bits next to pages whose scale is far larger but whose
//     weight is small.  Weights below 2^-14 of the largest a warp has seen lose bits, up to 2^-25 of
//     it each: 2^-12 of the mean |v| over 8192 keys, a sixteenth of the result's own rounding.  The row
//     sum uses 2^(s - m), in fp32, unrounded;
//   * a tile is 128 tokens, 32 per warp in two halves of 16 that share one page (and its scales),
//     one vote and one set of waits: with 8-bit keys the issue slots and the length of the chain
//     load - widen - MMA - softmax - MMA bound a warp, not the bytes;
//   * the maxima are raised only when a score passes them by more than 2^8 (one vote per 32
//     tokens instead of six shuffles); until then weights may be up to 2^8, which f16 and the
//     fp32 sums hold without loss;
//   * q is scaled by a power of two per head to at most 1 before it is rounded to f16.
// Measured (head_size 128, 8 KV heads): 32 users of 32768 tokens 350 us, 6.1 TB/s, 0.94 of the
// measured copy rate; 64 users of 1024 to 8192 tokens 110 us, 5.4 TB/s (138 us with
// 16 query heads per KV head, whose fragments take more registers than there are); one user of 32768
// tokens 26 us, of which the stream is 10: the rest is launch, first loads and the merge.
#pragma once
#include <cfloat>

#include "decode_fp8.cuh"
#include "paged_write.cuh"

namespace b200attn {

struct DecodeScaledParams {
  DecodeParams d;            // num_splits == 0: equal shares; part_o / part_ml: [slot][G] rows
  const float* k_scale;      // [num_blocks, num_kv_heads]
  const float* v_scale;
  int num_pairs;             // users * KV heads
  int whole_pairs;           // equal shares rounded to pairs (more pairs than arrival counters)
};

constexpr int kDsTile = 128;           // tokens per pipeline stage
constexpr int kDsWarpTokens = 32;      // of them per consumer warp

template <int HD, int BS, int NG, int STAGES>
struct DecodeScaledSmem {
  static constexpr int kPages = kDsTile / BS;
  static constexpr int kBoxBytes = BS * HD;                    // one page of one head
  static constexpr int kTensorBytes = kPages * kBoxBytes;      // K (or V) of one tile
  static constexpr int kStageBytes = 2 * kTensorBytes;
  static constexpr int kRingBytes = STAGES * kStageBytes;
  static constexpr int kScaleBytes = STAGES * kPages * 8;      // (K scale, log2 of the V scale)
  static constexpr int kBarrierBytes = 2 * STAGES * 8 + 16;
  static constexpr int kRow = HD + 4;                          // padded: fewer bank conflicts
  // merge of the warps, two at a time: rows of 8 NG heads and their (max, scale max, sum)
  static constexpr int kMergeBytes = 2 * 8 * NG * (kRow + 4) * 4;
  static constexpr int kMergeOff = kRingBytes + kScaleBytes + kBarrierBytes;
  static constexpr int kPlanOff = kMergeOff + kMergeBytes;     // the CTA's share; block scan
  static constexpr int kTotalBytes = kPlanOff + 128 + 1024;
  static_assert(kMergeOff % 16 == 0 && kPlanOff % 16 == 0, "vector access");
  static_assert((8 * NG * (32 + 2) + 1) * 4 <= kMergeBytes, "the merge of partials fits");
};

// Four codes in a word -> f16 pairs (bytes 0, 2) and (bytes 1, 3), exact.
template <int FMT>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& even, uint32_t& odd) {
  if (FMT == kPageInt8) {
    // 0x6400 | (code ^ 0x80) is 1024 + (code + 128) in f16
    uint32_t e, o;
    asm("lop3.b32 %0, %1, 0x00ff00ff, 0x64806480, 0x6a;" : "=r"(e) : "r"(w));   // (w & m) ^ k
    asm("lop3.b32 %0, %1, 0x00ff00ff, 0x64806480, 0x6a;" : "=r"(o) : "r"(w >> 8));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(even) : "r"(e), "r"(0x64806480u));    // - 1152
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(odd) : "r"(o), "r"(0x64806480u));
  } else {
    const uint32_t p = byte_perm(w, 0x3120u);
    even = e4m3x2_to_f16x2(p);
    odd = e4m3x2_to_f16x2(p >> 16);
  }
}

// 8x8 matrix of 16-bit values held as rows (thread 4 r + j: row r, columns 2 j, 2 j + 1),
// transposed across the warp.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

constexpr float kScoreSlack = 8.f;   // log2 units a score may pass the running maximum by

// A run of tiles of one (user, KV head) pair that one CTA works on.
struct DsSegment {
  int user, kvh, ctx, lo;    // keys lo .. ctx - 1 are attended
  int t_begin, t_end;        // tiles
  int n_tiles;               // of the pair in all
  int64_t pair_pos;          // where the pair's tiles start among all pairs' tiles
};

// First attended key and tiles of a pair.  A position behind the end of the page table is reported
// and the keys up to that end are attended.
template <int BS>
__device__ __forceinline__ int ds_pair_tiles(const DecodeParams& p, int user, int kvh, int* ctx_out,
                                             int* lo_out) {
  int pos = decode_cur_pos(p, user, kvh);
  const int64_t most = static_cast<int64_t>(p.page_table_width) * BS - 1;
  if (pos > most) {
    atomicExch(p.err_word, kDevBadIndex);
    pos = static_cast<int>(most);
  }
  const int ctx = pos + 1;             // the host keeps width * block_size below 2^31 - kDsTile
  const int lo = (p.window > 0 && ctx > p.window) ? ctx - p.window : 0;
  *ctx_out = ctx;
  *lo_out = lo;
  return ctx > 0 ? (ctx + kDsTile - 1) / kDsTile - lo / kDsTile : 0;
}

// The CTA's share of the work, walked segment by segment by every warp for itself.
struct DsShare {
  int64_t pos, end;          // tiles [pos, end) of all pairs' tiles
  int pair, offset;          // the pair that pos lies in, and the tile within it
  int shares;                // CTAs that have a share
  int64_t each, extra;       // tiles per share; the first `extra` shares have one more

  // `total` tiles in n equal shares (64-bit divisions take a microsecond: only where they must)
  __device__ __forceinline__ void divide(int64_t total, int n) {
    shares = n;
    if (n == 0) {
      each = extra = 0;
      return;
    }
    each = (total >> 32) == 0 ? static_cast<uint32_t>(total) / static_cast<uint32_t>(n) : total / n;
    extra = total - each * n;
  }
  __device__ __forceinline__ int64_t start_of(int c) const {
    return each * c + min(static_cast<int64_t>(c), extra);
  }
  // The share that tile x lies in.
  __device__ __forceinline__ int share_of(int64_t x) const {
    const int64_t longer = extra * (each + 1);      // tiles in the longer shares
    const int64_t rest = x < longer ? x : x - longer;
    const int64_t by = x < longer ? each + 1 : each;
    const int64_t c = ((rest | by) >> 32) == 0
                          ? static_cast<uint32_t>(rest) / static_cast<uint32_t>(by) : rest / by;
    return static_cast<int>(x < longer ? c : extra + c);
  }

  // Next segment; false at the end of the share.  Empty pairs are passed over.
  template <int BS>
  __device__ __forceinline__ bool next(const DecodeScaledParams& sp, DsSegment& s) {
    const DecodeParams& p = sp.d;
    while (pos < end && pair < sp.num_pairs) {
      s.user = pair / p.num_kv_heads;
      s.kvh = pair - s.user * p.num_kv_heads;
      s.n_tiles = ds_pair_tiles<BS>(p, s.user, s.kvh, &s.ctx, &s.lo);
      const int first = offset, left = s.n_tiles - first;
      if (sp.whole_pairs && first > 0) {       // the pair belongs to the share it starts in
        pos += left;
        ++pair;
        offset = 0;
        continue;
      }
      const int n = sp.whole_pairs ? left : static_cast<int>(min(static_cast<int64_t>(left), end - pos));
      s.pair_pos = pos - first;
      s.t_begin = s.lo / kDsTile + first;
      s.t_end = s.t_begin + n;
      pos += n;
      offset = 0;
      ++pair;
      if (n > 0) return true;
    }
    return false;
  }
};

// Where the partials of a shared pair lie: the i-th in slot first (i = 0) or base + i * step.
struct DsSlots {
  int64_t first, base;
  int step, count;
  __device__ __forceinline__ int64_t operator()(int i) const { return i == 0 ? first : base + i * step; }
};

// End of a segment that is not its pair's only one: the partial rows are in global memory, written
// by warp 0.  Whoever of the pair's CTAs arrives last (a ticket) finds all of them published and
// merges them; nobody waits.  The merge is one CTA reading count * G * head_size floats and its time
// is their latency: every thread keeps several 16-byte loads in flight for each of the vectors it
// owns.  Called by the consumer threads; `scratch` is shared memory of kMergeBytes.
template <int HD, int NG>
__device__ __forceinline__ void ds_finish(const DecodeParams& p, int user, int kvh,
                                          const DsSlots& slots, float* scratch, int tid) {
  constexpr int kThreads = kDecConsumerWarps * 32;
  constexpr int kChunk = 32;               // partials whose weights are held at once
  constexpr int kVec = HD / 4;
  constexpr int kItems = 8 * NG * kVec / kThreads;       // vectors per thread
  constexpr int kBatch = kItems > 2 ? 4 : 8;             // loads in flight for each
  const int G = p.group, count = slots.count;
  float* weight = scratch;                 // [8 NG][kChunk]
  float* row_m = weight + 8 * NG * kChunk;               // [8 NG] merged max
  float* row_l = row_m + 8 * NG;                         // [8 NG] merged sum
  volatile int* last_flag = reinterpret_cast<volatile int*>(row_l + 8 * NG);
  unsigned int* ticket = p.tickets + static_cast<int64_t>(user) * p.num_kv_heads + kvh;

  if (tid < 32) {
    __threadfence();                       // this lane's partial stores, device-wide
    __syncwarp();
    if (tid == 0) {
      *last_flag = atomicAdd(ticket, 1u) == static_cast<unsigned int>(count - 1);
      __threadfence();
    }
  }
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
  if (!*last_flag) return;
  if (tid == 0) *ticket = 0u;              // leave the counter as the next launch expects it

  const int warp = tid >> 5, lane = tid & 31;
  for (int r = warp; r < G; r += kDecConsumerWarps) {
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < count; i += 32) m = fmaxf(m, __ldcg(p.part_ml + slots(i) * G + r).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    for (int i = lane; i < count; i += 32) {
      const float2 v = __ldcg(p.part_ml + slots(i) * G + r);
      l += (v.x == -INFINITY ? 0.f : fast_exp2(v.x - m)) * v.y;   // -inf: attended nothing
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {
      row_m[r] = m;
      row_l[r] = l;
    }
  }
  float acc[kItems][4];
#pragma unroll
  for (int k = 0; k < kItems; ++k) acc[k][0] = acc[k][1] = acc[k][2] = acc[k][3] = 0.f;
  for (int s0 = 0; s0 < count; s0 += kChunk) {
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    for (int i = tid; i < 8 * NG * kChunk; i += kThreads) {
      const int r = i / kChunk, j = s0 + i % kChunk;
      float w = 0.f;                       // also for a partial that attended nothing
      if (r < G && j < count) {
        const float m = __ldcg(p.part_ml + slots(j) * G + r).x;
        if (m != -INFINITY) w = fast_exp2(m - row_m[r]);
      }
      weight[i] = w;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    const int n = min(kChunk, count - s0);
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += kBatch) {
      float4 x[kItems][kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int64_t row = slots(s0 + min(j0 + j, n - 1)) * G;
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
          const int i = tid + k * kThreads, r = min(i / kVec, G - 1), d = (i % kVec) * 4;
          x[k][j] = __ldcg(reinterpret_cast<const float4*>(p.part_o + (row + r) * HD + d));
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
          const int r = min((tid + k * kThreads) / kVec, G - 1);
          const float w = j0 + j < n ? weight[r * kChunk + j0 + j] : 0.f;
          if (w != 0.f) {                  // what a zero weight stands for may be no row at all
            acc[k][0] += w * x[k][j].x;
            acc[k][1] += w * x[k][j].y;
            acc[k][2] += w * x[k][j].z;
            acc[k][3] += w * x[k][j].w;
          }
        }
    }
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int i = tid + k * kThreads, r = i / kVec, d = (i % kVec) * 4;
    if (r >= G) break;
    float m = row_m[r], l = row_l[r];
    const int head = kvh * G + r;
    float by = p.sinks ? apply_sink(m, l, p.sinks[head] * 1.4426950408889634f) : 1.f;
    by = l > 0.f || l != l ? by / l : 0.f;
    uint2 y;
    y.x = pack_bf16x2(acc[k][0] * by, acc[k][1] * by);
    y.y = pack_bf16x2(acc[k][2] * by, acc[k][3] * by);
    *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(user) * p.out_row_stride + head * HD + d) = y;
  }
}

template <int HD, int BS, int FMT, int NG, int STAGES>
__global__ void __launch_bounds__(kDecThreads, 2)
paged_decode_scaled_kernel(const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const DecodeScaledParams sp) {
  using L = DecodeScaledSmem<HD, BS, NG, STAGES>;
  const DecodeParams& p = sp.d;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float2* scales = reinterpret_cast<float2*>(ring + L::kRingBytes);       // [STAGES][kPages]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(ring + L::kRingBytes + L::kScaleBytes);
  uint64_t* empty_bar = full_bar + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty_bar + STAGES);
  int64_t* plan = reinterpret_cast<int64_t*>(ring + L::kPlanOff);   // [0..4] warp sums, [5] total
  int* plan_at = reinterpret_cast<int*>(plan + 6);                  // pair and offset of the start

  // A CTA of this launch just gave up on a wait: do not repeat the timeout per CTA.
  if (timeout_drain_window(p.err_word)) return;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int G = p.group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], kDecConsumerWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  // ---- this CTA's share of the tiles
  DsShare share;
  int any_empty;             // some pair has no context (its rows are zeros)
  if (p.num_splits > 0) {
    // every pair cut into num_splits (or as many as it has tiles): one segment
    share.pair = blockIdx.x / p.num_splits;
    const int split = blockIdx.x - share.pair * p.num_splits;
    int ctx, lo;
    const int user = share.pair / p.num_kv_heads;
    const int n = ds_pair_tiles<BS>(p, user, share.pair - user * p.num_kv_heads, &ctx, &lo);
    share.divide(n, min(p.num_splits, n));
    share.pos = split < share.shares ? share.start_of(split) : 0;
    share.end = split < share.shares ? share.start_of(split + 1) : 0;
    share.offset = static_cast<int>(share.pos);
    any_empty = n == 0;
  } else {
    // all pairs' tiles in equal shares: a prefix sum over the pairs finds the start of this one
    const int per = (sp.num_pairs + kDecThreads - 1) / kDecThreads;
    const int first = min(sp.num_pairs, static_cast<int>(threadIdx.x) * per);
    const int last = min(sp.num_pairs, first + per);
    int64_t mine = 0;
    int ctx, lo, empty = 0;
    for (int q = first; q < last; ++q) {
      const int n = ds_pair_tiles<BS>(p, q / p.num_kv_heads, q % p.num_kv_heads, &ctx, &lo);
      mine += n;
      empty |= n == 0;
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) plan[warp] = incl;
    any_empty = __syncthreads_or(empty);
    int64_t before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kDecThreads / 32; ++w) {
      if (w < warp) before += plan[w];
      total += plan[w];
    }
    share.divide(total, static_cast<int>(min(static_cast<int64_t>(gridDim.x), total)));
    const int c = blockIdx.x;
    const bool has = c < share.shares;
    share.pos = has ? share.start_of(c) : 0;
    share.end = has ? share.start_of(c + 1) : 0;
    if (has && share.pos >= before && share.pos < before + mine) {
      int q = first;
      for (; q < last; ++q) {
        const int n = ds_pair_tiles<BS>(p, q / p.num_kv_heads, q % p.num_kv_heads, &ctx, &lo);
        if (share.pos < before + n) break;
        before += n;
      }
      plan_at[0] = q;
      plan_at[1] = static_cast<int>(share.pos - before);
    }
    __syncthreads();
    share.pair = plan_at[0];
    share.offset = plan_at[1];
  }
  // rows of pairs without context are zeros
  if (any_empty) {
    const int step = p.num_splits > 0 ? sp.num_pairs : static_cast<int>(gridDim.x);
    int q = p.num_splits > 0 ? (blockIdx.x % p.num_splits == 0 ? blockIdx.x / p.num_splits
                                                               : sp.num_pairs)
                             : blockIdx.x;
    for (; q < sp.num_pairs; q += step) {
      int ctx, lo;
      const int user = q / p.num_kv_heads, kvh = q - user * p.num_kv_heads;
      if (ds_pair_tiles<BS>(p, user, kvh, &ctx, &lo) > 0) continue;
      for (int i = threadIdx.x; i < G * HD; i += kDecThreads)
        p.out[static_cast<int64_t>(user) * p.out_row_stride + kvh * G * HD + i] = __float2bfloat16(0.f);
    }
  }
  __syncthreads();
  if (share.pos >= share.end) return;
  DsSegment seg;

  if (warp == kDecConsumerWarps) {
    // ------------------------------------------------------------------ producer warp
    if (lane == 0) {
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
    }
    const uint64_t policy = l2_policy_evict_first();
    // Each lane keeps the id and the scales of one page of a 32-page window; the next window is
    // fetched early, so only the first tiles of a segment wait for a page's scales.
    struct Window {
      int id;
      float ks, vs;     // K scale, log2 of the V scale
    };
    uint32_t it = 0;    // tiles since the start of the share
    while (share.next<BS>(sp, seg)) {
      const int kvh = seg.kvh;
      const int n_pages = (seg.ctx + BS - 1) / BS;
      const int32_t* pt = decode_page_row(p, seg.user, kvh);
      auto fetch = [&](int base) {
        Window w;
        const int idx = min(min(base + lane, n_pages - 1), p.page_table_width - 1);
        w.id = pt[idx];
        const bool ok = w.id >= 0 && w.id < p.num_blocks;
        const int64_t at = ok ? static_cast<int64_t>(w.id) * p.num_kv_heads + kvh : kvh;
        // what is no scale (negative, infinite) is read as NaN, as prefill does
        const float ks = __ldg(sp.k_scale + at), vs = __ldg(sp.v_scale + at);
        w.ks = ks >= 0.f && ks < INFINITY ? ks : NAN;
        w.vs = vs >= 0.f && vs < INFINITY ? __log2f(vs) : NAN;
        return w;
      };
      int win_base = seg.t_begin * L::kPages;
      Window cur = fetch(win_base), nxt = fetch(win_base + 32);
      // the loads of a tile's pages, not of those past the context (the stage's barrier takes their
      // bytes before it is armed ...)
      auto pages_of = [&](int t) { return min(L::kPages, n_pages - t * L::kPages); };
      auto load_tile = [&](int t, int stage) {
        const int live = pages_of(t);
        uint8_t* kdst = ring + stage * L::kStageBytes;
        uint8_t* vdst = kdst + L::kTensorBytes;
        if (t * L::kPages - win_base >= 32) {     // windows start at a tile and hold whole tiles
          win_base += 32;
          cur = nxt;
          nxt = fetch(win_base + 32);
        }
#pragma unroll
        for (int pg = 0; pg < L::kPages; ++pg) {
          if (pg >= live) break;
          const int page_idx = t * L::kPages + pg;
          int64_t blk = __shfl_sync(0xffffffffu, cur.id, page_idx - win_base);
          if (blk < 0 || blk >= p.num_blocks) {
            if (lane == 0) atomicExch(p.err_word, kDevBadIndex);
            blk = 0;
          }
          if (lane == 0) {
            const int32_t y = static_cast<int32_t>((blk * p.num_kv_heads + kvh) * (BS * HD / 128));
            tma_load_2d(kdst + pg * L::kBoxBytes, &tm_k, &full_bar[stage], 0, y, policy);
            tma_load_2d(vdst + pg * L::kBoxBytes, &tm_v, &full_bar[stage], 0, y, policy);
          }
        }
      };
      // (... here) and its scales
      auto arm_tile = [&](int t, int stage) {
        const int live = pages_of(t);
#pragma unroll
        for (int pg = 0; pg < L::kPages; ++pg) {
          if (pg >= live) break;
          const int page_idx = t * L::kPages + pg;
          const float ks = __shfl_sync(0xffffffffu, cur.ks, page_idx - win_base);
          const float vs = __shfl_sync(0xffffffffu, cur.vs, page_idx - win_base);
          if (lane == 0) scales[stage * L::kPages + pg] = make_float2(ks, vs);
        }
        if (lane == 0) mbar_arrive_expect_tx(&full_bar[stage], live * 2 * L::kBoxBytes);
      };
      static_assert(32 % L::kPages == 0, "a window holds whole tiles");
      static_assert(STAGES * L::kPages <= 32, "the first fill stays in one window");
      int t = seg.t_begin;
      if (it == 0) {
        // first fill: all loads go out before anything waits for a scale
        const int first = min(seg.t_end, t + STAGES);
        for (int j = t; j < first; ++j) load_tile(j, j - t);
        for (int j = t; j < first; ++j) arm_tile(j, j - t);
        it = first - t;
        t = first;
      }
      for (; t < seg.t_end; ++t, ++it) {
        const int stage = it % STAGES;
        mbar_wait(&empty_bar[stage], ((it / STAGES) & 1) ^ 1, abort_flag, p.err_word);
        load_tile(t, stage);
        arm_tile(t, stage);
      }
    }
    return;  // consumers wait on every full barrier, so no copy is in flight at kernel end
  }

  // -------------------------------------------------------------------- consumer warps
  const int g = lane >> 2;
  const int tq = lane & 3;
  static_assert(kDecConsumerWarps * kDsWarpTokens == kDsTile && BS % kDsWarpTokens == 0, "");

  // Per-lane ldmatrix addressing inside a tile: token t's head_size bytes start at t * HD; 128-byte
  // rows, 16-byte chunks XOR-swizzled with the row's low three bits (the two halves of a warp's
  // tokens are a multiple of 8 rows apart: same swizzle).  Matrix lane / 8: token half of the 16
  // (bit 0) and chunk of a pair (bit 1), for K and for V.
  const int lm = lane >> 3, lr = lane & 7;
  const int tok = warp * kDsWarpTokens + (lm & 1) * 8 + lr;
  const uint32_t row = static_cast<uint32_t>(tok * HD) >> 7;
  const uint32_t chunk0 = ((static_cast<uint32_t>(tok * HD) & 127u) >> 4) + (lm >> 1);
  uint32_t at[HD / 32];
#pragma unroll
  for (int cp = 0; cp < HD / 32; ++cp) at[cp] = (row << 7) + (((chunk0 + 2 * cp) ^ (row & 7)) << 4);
  constexpr uint32_t kHalf = 16 * HD;      // bytes from a warp's first 16 tokens to its second

  float* mo = reinterpret_cast<float*>(ring + L::kMergeOff);       // [2][8 NG heads][kRow]
  float4* ms = reinterpret_cast<float4*>(mo + 2 * 8 * NG * L::kRow);   // [2][8 NG] m, r, l
  uint32_t it = 0;                  // tiles since the start of the share
  int segments = 0;
  while (share.next<BS>(sp, seg)) {
  // Q fragments (B operand, columns = query heads 8 ng + g; heads >= G are zero).  Within the
  // 16 elements of k-step ks the thread holds 4tq .. 4tq+3; slots {2tq, 2tq+1} take elements 0
  // and 2 of these, slots {2tq+8, 2tq+9} elements 1 and 3: the order codes_to_f16 gives.
  uint32_t qf[NG][HD / 16][2];
  float qs[NG][2];     // scale * log2(e) * 2^e of query heads 8 ng + 2 tq, + 1 (the S columns)
#pragma unroll
  for (int ng = 0; ng < NG; ++ng) {
    const int head = ng * 8 + g;
    uint2 raw[HD / 16];
    uint32_t top = 0;
    const __nv_bfloat16* qrow = p.q + static_cast<int64_t>(seg.user) * p.q_row_stride +
                                (static_cast<int64_t>(seg.kvh) * G + head) * HD;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      raw[ks] = head < G ? *reinterpret_cast<const uint2*>(qrow + ks * 16 + tq * 4)
                         : make_uint2(0u, 0u);
      top = __vmaxu2(top, __vmaxu2(raw[ks].x & 0x7fff7fffu, raw[ks].y & 0x7fff7fffu));
    }
    top = max(top & 0xffffu, top >> 16);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^-(e+1), e the exponent of the head's largest |q| (bf16 bits 7..14, bias 127), so that
    // |q| < 1; left alone for zero, subnormal and non-finite heads
    const int e = static_cast<int>(top >> 7);
    const bool norm = e >= 2 && e < 253;
    const float down = norm ? __uint_as_float(static_cast<uint32_t>(253 - e) << 23) : 1.f;
    const float up = norm ? __uint_as_float(static_cast<uint32_t>(e + 1) << 23) : 1.f;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      const float q0 = __uint_as_float(raw[ks].x << 16) * down;
      const float q1 = __uint_as_float(raw[ks].x & 0xffff0000u) * down;
      const float q2 = __uint_as_float(raw[ks].y << 16) * down;
      const float q3 = __uint_as_float(raw[ks].y & 0xffff0000u) * down;
      qf[ng][ks][0] = pack_f16x2(q0, q2);
      qf[ng][ks][1] = pack_f16x2(q1, q3);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)     // head 8 ng + 2 tq + j sits with lanes 4 (2 tq + j) ..
      qs[ng][j] = p.scale_log2 * __shfl_sync(0xffffffffu, up, (2 * tq + j) * 4);
  }

  // o[ng][c][0..1]: element 16 c + 2 g, [2..3]: 16 c + 2 g + 1, of query heads 8 ng + 2 tq, + 1
  float o[NG][HD / 16][4];
  float m[NG][2], r[NG][2], l[NG][2];   // max of s, max of s - m + log2 vs, sum (this lane's share)
#pragma unroll
  for (int ng = 0; ng < NG; ++ng) {
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) o[ng][c][0] = o[ng][c][1] = o[ng][c][2] = o[ng][c][3] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[ng][j] = r[ng][j] = -FLT_MAX;
      l[ng][j] = 0.f;
    }
  }

  for (int t = seg.t_begin; t < seg.t_end; ++t, ++it) {
    const int stage = it % STAGES;
    mbar_wait(&full_bar[stage], (it / STAGES) & 1, abort_flag, p.err_word);
    const uint32_t kbase = smem_u32(ring + stage * L::kStageBytes);
    const uint32_t vbase = kbase + L::kTensorBytes;
    const int ctx = seg.ctx, lo = seg.lo;
    const int tok0 = t * kDsTile + warp * kDsWarpTokens;   // first token of this warp's slice

    if (tok0 < ctx && tok0 + kDsWarpTokens > lo) {  // at least one of this warp's keys is attended
      const bool tail = (tok0 + kDsWarpTokens > ctx) || (tok0 < lo);
      if (tail && FMT != kPageInt8) {
        // Rows past the context, and rows a window has left behind, may hold NaN codes: zero them,
        // 0 * NaN would reach the sums.
        for (int i = lane; i < kDsWarpTokens * (HD / 16); i += 32) {
          const int r = warp * kDsWarpTokens + i / (HD / 16), c = i % (HD / 16);
          if (t * kDsTile + r >= ctx || t * kDsTile + r < lo) {
            const uint32_t b = static_cast<uint32_t>(r * HD + c * 16);
            const uint32_t a = vbase + (b & ~127u) + ((((b >> 4) & 7u) ^ ((b >> 7) & 7u)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0) : "memory");
          }
        }
        fence_proxy_async_smem();  // the next TMA write to this stage follows generic writes
        __syncwarp();
      }
      const float2 sc = scales[stage * L::kPages + (warp * kDsWarpTokens) / BS];   // one page

      // ---- S^T = K Q^T: rows = 16 tokens, columns = query heads
      float s[2][NG][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int ng = 0; ng < NG; ++ng)
          s[u][ng][0] = s[u][ng][1] = s[u][ng][2] = s[u][ng][3] = 0.f;
#pragma unroll
      for (int cp = 0; cp < HD / 32; ++cp)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t b[4];
          ldmatrix_x4(b, kbase + at[cp] + u * kHalf);
          // b[0]: tokens 0-7, b[1]: tokens 8-15 of chunk 2cp; b[2], b[3]: of chunk 2cp+1
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a[4];
            codes_to_f16<FMT>(b[2 * h], a[0], a[2]);
            codes_to_f16<FMT>(b[2 * h + 1], a[1], a[3]);
#pragma unroll
            for (int ng = 0; ng < NG; ++ng)
              mma_f16_16816(s[u][ng], a, qf[ng][2 * cp + h][0], qf[ng][2 * cp + h][1]);
          }
        }

      // ---- scores in log2 units; s[u][ng][i]: token 16 u + g + 8 (i / 2), head 8 ng + 2 tq + i % 2
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) {
        const float f[2] = {qs[ng][0] * sc.x, qs[ng][1] * sc.x};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][ng][i] *= f[i & 1];
      }
      if (tail) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = tok0 + u * 16 + g + (i >> 1) * 8;
            if (j >= ctx || j < lo)
#pragma unroll
              for (int ng = 0; ng < NG; ++ng) s[u][ng][i] = -INFINITY;
          }
      }
      // the exponents' largest: d = s - m of the sum, d + log2 vs - r of the weights
      bool over = false;
#pragma unroll
      for (int ng = 0; ng < NG; ++ng)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float d = fmaxf(fmaxf(s[0][ng][j], s[0][ng][j + 2]),
                                fmaxf(s[1][ng][j], s[1][ng][j + 2])) - m[ng][j];
          over |= d > kScoreSlack || d + sc.y > r[ng][j] + kScoreSlack;
        }
      if (__any_sync(0xffffffffu, over)) {      // raise the maxima
#pragma unroll
        for (int ng = 0; ng < NG; ++ng) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = fmaxf(fmaxf(s[0][ng][j], s[0][ng][j + 2]),
                             fmaxf(s[1][ng][j], s[1][ng][j + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = fmaxf(m[ng][j], mx), by = mn - m[ng][j];
            // r seen from the new m; kept finite, so that pages of zero values alone leave it so
            const float was = fmaxf(r[ng][j] - by, -FLT_MAX);
            const float rn = fmaxf(was, (mx - mn) + sc.y);
            l[ng][j] *= fast_exp2(-by);
            const float f = fast_exp2(was - rn);
            m[ng][j] = mn;
            r[ng][j] = rn;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
              o[ng][c][j] *= f;
              o[ng][c][j + 2] *= f;
            }
          }
        }
      }
      // ---- P'^T as B operand: transposed 8x8 blocks, k = tokens, columns = heads
      uint32_t pb[2][NG][2];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) {
        const float add[2] = {sc.y - r[ng][0], sc.y - r[ng][1]};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float d = s[u][ng][i] - m[ng][i & 1];
            l[ng][i & 1] += fast_exp2(d);
            w[i] = fast_exp2(d + add[i & 1]);
          }
          pb[u][ng][0] = transpose_8x8(pack_f16x2(w[0], w[1]));
          pb[u][ng][1] = transpose_8x8(pack_f16x2(w[2], w[3]));
        }
      }

      // ---- O^T += V^T P'^T: rows = the 16 head elements of a chunk (even ones, then odd ones)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int cp = 0; cp < HD / 32; ++cp) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, vbase + at[cp] + u * kHalf);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a[4];
            codes_to_f16<FMT>(b[2 * h], a[0], a[1]);
            codes_to_f16<FMT>(b[2 * h + 1], a[2], a[3]);
#pragma unroll
            for (int ng = 0; ng < NG; ++ng)
              mma_f16_16816(o[ng][2 * cp + h], a, pb[u][ng][0], pb[u][ng][1]);
          }
        }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty_bar[stage]);
  }

  // -------------------------------------------------------------------- merge the 4 warps
#pragma unroll
  for (int ng = 0; ng < NG; ++ng)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[ng][j] += __shfl_xor_sync(0xffffffffu, l[ng][j], 4);
      l[ng][j] += __shfl_xor_sync(0xffffffffu, l[ng][j], 8);
      l[ng][j] += __shfl_xor_sync(0xffffffffu, l[ng][j], 16);
    }
  // Warps 2 and 3 hand their rows to warps 0 and 1, then warp 1 to warp 0 (the ring is busy with
  // the next segment's tiles, so the rows of two warps are what there is room for).
  auto heads_do = [&](int from, auto f) {
#pragma unroll
    for (int ng = 0; ng < NG; ++ng)
#pragma unroll
      for (int j = 0; j < 2; ++j) f(from * 8 * NG + ng * 8 + 2 * tq + j, ng, j);
  };
#pragma unroll 1
  for (int half = kDecConsumerWarps / 2; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) {
      heads_do(warp - half, [&](int head, int ng, int j) {
#pragma unroll
        for (int c = 0; c < HD / 16; ++c)
          *reinterpret_cast<float2*>(mo + head * L::kRow + c * 16 + 2 * g) =
              make_float2(o[ng][c][j], o[ng][c][j + 2]);
        if (g == 0) ms[head] = make_float4(m[ng][j], r[ng][j], l[ng][j], 0.f);
      });
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kDecConsumerWarps * 32) : "memory");
    if (warp < half) {
      heads_do(warp, [&](int head, int ng, int j) {
        const float4 other = ms[head];
        // a warp that attended no key has m = -FLT_MAX and a zero sum: factor 0 (or 1 when both)
        const float mn = fmaxf(m[ng][j], other.x);
        const float fa = fast_exp2(m[ng][j] - mn), fb = fast_exp2(other.x - mn);
        const float ra = fmaxf(r[ng][j] + (m[ng][j] - mn), -FLT_MAX);
        const float rb = fmaxf(other.y + (other.x - mn), -FLT_MAX);
        const float rn = fmaxf(ra, rb);
        const float ga = fast_exp2(ra - rn), gb = fast_exp2(rb - rn);
        m[ng][j] = mn;
        r[ng][j] = rn;
        l[ng][j] = l[ng][j] * fa + other.z * fb;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
          const float2 x = *reinterpret_cast<const float2*>(mo + head * L::kRow + c * 16 + 2 * g);
          o[ng][c][j] = o[ng][c][j] * ga + x.x * gb;
          o[ng][c][j + 2] = o[ng][c][j + 2] * ga + x.y * gb;
        }
      });
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kDecConsumerWarps * 32) : "memory");
  }
  // warp 0 holds the segment's rows: 2^r gives the V scales back
  const bool whole = seg.t_end - seg.t_begin == seg.n_tiles;
  const int64_t my_slot = p.num_splits > 0 ? blockIdx.x
                                           : 2 * static_cast<int64_t>(blockIdx.x) + (segments > 0);
  ++segments;
  if (warp == 0) {
    heads_do(0, [&](int, int ng, int j) {
      const int h = ng * 8 + 2 * tq + j;
      if (h >= G) return;
      float mm = m[ng][j], ll = l[ng][j], by = exp2f(r[ng][j]);
      if (r[ng][j] == -FLT_MAX) by = ll != ll ? NAN : 0.f;      // nothing but zero values
      if (whole) {
        const int head = seg.kvh * G + h;
        if (p.sinks) by *= apply_sink(mm, ll, p.sinks[head] * 1.4426950408889634f);
        by = ll > 0.f || ll != ll ? by / ll : 0.f;
        __nv_bfloat16* dst = p.out + static_cast<int64_t>(seg.user) * p.out_row_stride + head * HD;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c)
          *reinterpret_cast<uint32_t*>(dst + c * 16 + 2 * g) =
              pack_bf16x2(o[ng][c][j] * by, o[ng][c][j + 2] * by);
      } else {
        float* dst = p.part_o + (my_slot * G + h) * HD;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c)
          *reinterpret_cast<float2*>(dst + c * 16 + 2 * g) =
              make_float2(o[ng][c][j] * by, o[ng][c][j + 2] * by);
        if (g == 0)
          p.part_ml[my_slot * G + h] = make_float2(mm == -FLT_MAX && ll == 0.f ? -INFINITY : mm, ll);
      }
    });
  }
  if (!whole) {
    DsSlots slots;
    if (p.num_splits > 0) {
      const int64_t pair = static_cast<int64_t>(seg.user) * p.num_kv_heads + seg.kvh;
      slots = DsSlots{pair * p.num_splits, pair * p.num_splits, 1, share.shares};
    } else {
      // a share's first segment has slot 2 c, its last 2 c + 1
      const int c0 = share.share_of(seg.pair_pos);
      const int c1 = share.share_of(seg.pair_pos + seg.n_tiles - 1);
      const bool inside = share.start_of(c0) < seg.pair_pos;
      slots = DsSlots{2 * static_cast<int64_t>(c0) + (inside ? 1 : 0), 2 * static_cast<int64_t>(c0),
                      2, c1 - c0 + 1};
    }
    ds_finish<HD, NG>(p, seg.user, seg.kvh, slots, reinterpret_cast<float*>(mo), threadIdx.x);
    asm volatile("bar.sync 1, %0;" ::"n"(kDecConsumerWarps * 32) : "memory");   // mo is free again
  }
  }
}

}  // namespace b200attn

// Paged GQA decode attention over an 8-bit KV cache with one fp32 scale for each page and KV head
// (what paged_write_kernel writes), int8 or e4m3, head_size 64 or 128.
//
//   s_j = (q . c_j) * scale * ks(page of j)        c: codes, ks / vs: the page's K / V scale
//   out = sum_j 2^(s_j - m) vs(page of j) c'_j / sum_j 2^(s_j - m)
//
// HBM-bound: a key and value cost 2 * head_size bytes and are read once.  As in the bf16 kernel a
// CTA owns one KV head of one user (and a slice of the context), a producer warp keeps a ring of
// tiles full with TMA, and four warps take a quarter of a tile each.  What differs:
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
//     weight is small.  The row sum uses 2^(s - m), in fp32, unrounded;
//   * a tile is 128 tokens, 32 per warp in two halves of 16 that share one page (and its scales),
//     one vote and one set of waits: with 8-bit keys the issue slots and the length of the chain
//     load - widen - MMA - softmax - MMA bound a warp, not the bytes;
//   * the maxima are raised only when a score passes them by more than 2^8 (one vote per 32
//     tokens instead of six shuffles); until then weights may be up to 2^8, which f16 and the
//     fp32 sums hold without loss;
//   * q is scaled by a power of two per head to at most 1 before it is rounded to f16.
#pragma once
#include <cfloat>

#include "decode_fp8.cuh"
#include "paged_write.cuh"

namespace b200attn {

struct DecodeScaledParams {
  DecodeParams d;
  const float* k_scale;      // [num_blocks, num_kv_heads]
  const float* v_scale;
};

constexpr int kDsTile = 128;           // tokens per pipeline stage
constexpr int kDsWarpTokens = 32;      // of them per consumer warp

template <int HD, int BS, int STAGES>
struct DecodeScaledSmem {
  static constexpr int kPages = kDsTile / BS;
  static constexpr int kBoxBytes = BS * HD;                    // one page of one head
  static constexpr int kTensorBytes = kPages * kBoxBytes;      // K (or V) of one tile
  static constexpr int kStageBytes = 2 * kTensorBytes;
  static constexpr int kRingBytes = STAGES * kStageBytes;
  static constexpr int kScaleBytes = STAGES * kPages * 8;      // (K scale, log2 of the V scale)
  static constexpr int kBarrierBytes = 2 * STAGES * 8 + 16;
  static constexpr int kTotalBytes = kRingBytes + kScaleBytes + kBarrierBytes + 1024;
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

// decode_split_finish for this kernel: the same protocol (the split that arrives last merges), with
// the partial rows read as 16-byte vectors, eight splits in flight per thread: the merge is one CTA
// reading splits * G * head_size floats, and its time is their latency.
template <int HD>
__device__ __forceinline__ void decode_scaled_finish(const DecodeParams& p, int user, int kvh,
                                                     float* scratch, int tid) {
  constexpr int kThreads = kDecConsumerWarps * 32;
  const int S = p.num_splits, G = p.group;
  float* fac = scratch;                    // [G][S] running max of a split, then its merge factor
  float* row_m = scratch + 16 * S;         // [G] merged max
  float* row_l = row_m + 16;               // [G] merged sum
  volatile int* last_flag = reinterpret_cast<volatile int*>(row_l + 16);
  unsigned int* ticket = p.tickets + static_cast<int64_t>(user) * p.num_kv_heads + kvh;

  __threadfence();                         // this thread's partial stores, device-wide
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
  if (tid == 0) *last_flag = atomicAdd(ticket, 1u) == static_cast<unsigned int>(S - 1);
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
  if (!*last_flag) return;
  __threadfence();
  if (tid == 0) *ticket = 0u;              // leave the counter as the next launch expects it

  const int64_t row0 = (static_cast<int64_t>(user) * p.num_q_heads + kvh * G) * S;
  const int warp = tid >> 5, lane = tid & 31;
  for (int r = warp; r < G; r += kDecConsumerWarps) {
    const float2* ml = p.part_ml + row0 + static_cast<int64_t>(r) * S;
    float m = -INFINITY, l = 0.f;
    // two passes over at most kDecMaxSplits pairs: they stay in registers
    float2 v[kDecMaxSplits / 32];
#pragma unroll
    for (int i = 0; i < kDecMaxSplits / 32; ++i) {
      v[i] = i * 32 + lane < S ? __ldcg(ml + i * 32 + lane) : make_float2(-INFINITY, 0.f);
      m = fmaxf(m, v[i].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int i = 0; i < kDecMaxSplits / 32; ++i) {
      const float f = v[i].x == -INFINITY ? 0.f : fast_exp2(v[i].x - m);   // empty splits: -inf
      l += f * v[i].y;
      if (i * 32 + lane < S) fac[r * S + i * 32 + lane] = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {
      row_m[r] = m;
      row_l[r] = l;
    }
  }
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
  constexpr int kVec = HD / 4;
  for (int i = tid; i < G * kVec; i += kThreads) {
    const int r = i / kVec, d = (i - r * kVec) * 4;
    const float* src = p.part_o + (row0 + static_cast<int64_t>(r) * S) * HD + d;
    float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
    for (int s0 = 0; s0 < S; s0 += 8) {
      float4 x[8];
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // an empty split published no rows: its memory must not be read into the sum
        f[j] = s0 + j < S ? fac[r * S + s0 + j] : 0.f;
        x[j] = f[j] != 0.f ? __ldcg(reinterpret_cast<const float4*>(
                                 src + static_cast<int64_t>(s0 + j) * HD))
                           : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a0 += f[j] * x[j].x;
        a1 += f[j] * x[j].y;
        a2 += f[j] * x[j].z;
        a3 += f[j] * x[j].w;
      }
    }
    float m = row_m[r], l = row_l[r];
    const int head = kvh * G + r;
    float by = p.sinks ? apply_sink(m, l, p.sinks[head] * 1.4426950408889634f) : 1.f;
    by = l > 0.f || l != l ? by / l : 0.f;
    uint2 y;
    y.x = pack_bf16x2(a0 * by, a1 * by);
    y.y = pack_bf16x2(a2 * by, a3 * by);
    *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(user) * p.out_row_stride + head * HD + d) = y;
  }
}

template <int HD, int BS, int FMT, int NG, int STAGES>
__global__ void __launch_bounds__(kDecThreads)
paged_decode_scaled_kernel(const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const DecodeScaledParams sp) {
  using L = DecodeScaledSmem<HD, BS, STAGES>;
  const DecodeParams& p = sp.d;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float2* scales = reinterpret_cast<float2*>(ring + L::kRingBytes);       // [STAGES][kPages]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(ring + L::kRingBytes + L::kScaleBytes);
  uint64_t* empty_bar = full_bar + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty_bar + STAGES);

  // A CTA of this launch just gave up on a wait: do not repeat the timeout per CTA.
  if (timeout_drain_window(p.err_word)) return;

  const int split = blockIdx.x;
  const int kvh = blockIdx.y;
  const int user = blockIdx.z;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  const int ctx = decode_cur_pos(p, user, kvh) + 1;  // keys 0 .. cur_pos
  const int lo = (p.window > 0 && ctx > p.window) ? ctx - p.window : 0;   // first key attended
  const int n_tiles = ctx > 0 ? (ctx + kDsTile - 1) / kDsTile : 0;
  const int t_lo = lo / kDsTile;
  const int tiles_per_split = (n_tiles - t_lo + p.num_splits - 1) / p.num_splits;
  const int t_begin = t_lo + split * tiles_per_split;
  const int t_end = min(n_tiles, t_begin + tiles_per_split);
  const int G = p.group;

  if (t_begin >= t_end) {
    // Nothing for this split: publish an empty partial (or zeros when it is the only split).
    if (p.num_splits > 1) {
      if (threadIdx.x < G) {
        const int64_t row = (static_cast<int64_t>(user) * p.num_q_heads + kvh * G + threadIdx.x) *
                                p.num_splits + split;
        p.part_ml[row] = make_float2(-INFINITY, 0.f);
      }
      if (p.tickets && threadIdx.x < kDecConsumerWarps * 32)
        decode_scaled_finish<HD>(p, user, kvh, reinterpret_cast<float*>(ring), threadIdx.x);
    } else {
      for (int i = threadIdx.x; i < G * HD; i += blockDim.x) {
        const int r = i / HD, d = i - r * HD;
        p.out[static_cast<int64_t>(user) * p.out_row_stride + (kvh * G + r) * HD + d] =
            __float2bfloat16(0.f);
      }
    }
    return;
  }

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], kDecConsumerWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();

  if (warp == kDecConsumerWarps) {
    // ------------------------------------------------------------------ producer warp
    if (lane == 0) {
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
    }
    const uint64_t policy = l2_policy_evict_first();
    const int n_pages = (ctx + BS - 1) / BS;
    const int32_t* pt = decode_page_row(p, user, kvh);
    // Each lane keeps the id and the scales of one page of a 32-page window; the next window is
    // fetched early, so only the first tiles wait for a page's scales.
    struct Window {
      int id;
      float ks, vs;     // K scale, log2 of the V scale
    };
    auto fetch = [&](int base) {
      Window w;
      const int idx = min(min(base + lane, n_pages - 1), p.page_table_width - 1);
      w.id = pt[idx];
      const bool ok = w.id >= 0 && w.id < p.num_blocks;
      const int64_t at = ok ? static_cast<int64_t>(w.id) * p.num_kv_heads + kvh : kvh;
      w.ks = __ldg(sp.k_scale + at);
      w.vs = __log2f(__ldg(sp.v_scale + at));
      return w;
    };
    int win_base = t_begin * L::kPages;
    Window cur = fetch(win_base), nxt = fetch(win_base + 32);
    auto advance = [&](int page_idx) {
      if (page_idx - win_base >= 32) {
        win_base += 32;
        cur = nxt;
        nxt = fetch(win_base + 32);
      }
    };
    // the loads of a tile's pages, not of those past the context (the stage's barrier takes their
    // bytes before it is armed ...)
    auto pages_of = [&](int t) { return min(L::kPages, n_pages - t * L::kPages); };
    auto load_tile = [&](int t, int stage) {
      const int live = pages_of(t);
      uint8_t* kdst = ring + stage * L::kStageBytes;
      uint8_t* vdst = kdst + L::kTensorBytes;
#pragma unroll
      for (int pg = 0; pg < L::kPages; ++pg) {
        if (pg >= live) break;
        const int page_idx = t * L::kPages + pg;
        advance(page_idx);
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
    // First fill: all loads go out before anything waits for a scale (all of these pages are in
    // the first window).
    static_assert(STAGES * L::kPages <= 32, "the first fill stays in one window");
    const int first = min(t_end, t_begin + STAGES);
    for (int t = t_begin; t < first; ++t) load_tile(t, t - t_begin);
    for (int t = t_begin; t < first; ++t) arm_tile(t, t - t_begin);
    for (int t = first; t < t_end; ++t) {
      const int it = t - t_begin;
      const int stage = it % STAGES;
      mbar_wait(&empty_bar[stage], ((it / STAGES) & 1) ^ 1, abort_flag, p.err_word);
      load_tile(t, stage);
      arm_tile(t, stage);
    }
    return;  // consumers wait on every full barrier, so no copy is in flight at kernel end
  }

  // -------------------------------------------------------------------- consumer warps
  const int g = lane >> 2;
  const int tq = lane & 3;
  static_assert(kDecConsumerWarps * kDsWarpTokens == kDsTile && BS % kDsWarpTokens == 0, "");

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
    const __nv_bfloat16* qrow = p.q + static_cast<int64_t>(user) * p.q_row_stride +
                                (static_cast<int64_t>(kvh) * G + head) * HD;
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

  for (int t = t_begin; t < t_end; ++t) {
    const int it = t - t_begin;
    const int stage = it % STAGES;
    mbar_wait(&full_bar[stage], (it / STAGES) & 1, abort_flag, p.err_word);
    const uint32_t kbase = smem_u32(ring + stage * L::kStageBytes);
    const uint32_t vbase = kbase + L::kTensorBytes;
    const int tok0 = t * kDsTile + warp * kDsWarpTokens;   // first token of this warp's slice

    if (tok0 < ctx && tok0 + kDsWarpTokens > lo) {  // at least one of this warp's keys is attended
      const bool tail = (tok0 + kDsWarpTokens > ctx) || (tok0 < lo);
      if (tail && FMT != kPageInt8) {
        // Rows past the context may hold NaN codes: zero them, 0 * NaN would reach the sums.
        for (int i = lane; i < kDsWarpTokens * (HD / 16); i += 32) {
          const int r = warp * kDsWarpTokens + i / (HD / 16), c = i % (HD / 16);
          if (t * kDsTile + r >= ctx) {
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
  // All consumer warps are past their last full-barrier wait: the ring is free to reuse.
  asm volatile("bar.sync 1, %0;" ::"n"(kDecConsumerWarps * 32));
  constexpr int kRow = HD + 4;                                      // padded: fewer bank conflicts
  float* so = reinterpret_cast<float*>(ring);                       // [4 warps][8 NG heads][kRow]
  float* sm = so + kDecConsumerWarps * 8 * NG * kRow;               // [4][8 NG] max of s
  float* sr = sm + kDecConsumerWarps * 8 * NG;                      // [4][8 NG] max of s - m + log2 vs
  float* sl = sr + kDecConsumerWarps * 8 * NG;                      // [4][8 NG] sum
  static_assert(kDecConsumerWarps * 8 * NG * (kRow + 3) * 4 <= L::kRingBytes, "merge scratch fits");
  static_assert((16 * kDecMaxSplits + 40) * 4 <= L::kRingBytes, "split merge scratch fits");
#pragma unroll
  for (int ng = 0; ng < NG; ++ng)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int head = warp * 8 * NG + ng * 8 + 2 * tq + j;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c)
        *reinterpret_cast<float2*>(so + head * kRow + c * 16 + 2 * g) =
            make_float2(o[ng][c][j], o[ng][c][j + 2]);
      if (g == 0) {
        sm[head] = m[ng][j];
        sr[head] = r[ng][j];
        sl[head] = l[ng][j];
      }
    }
  asm volatile("bar.sync 1, %0;" ::"n"(kDecConsumerWarps * 32));

  for (int i = threadIdx.x; i < G * HD; i += kDecConsumerWarps * 32) {
    const int r = i / HD, d = i - r * HD;
    float mm = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < kDecConsumerWarps; ++w) mm = fmaxf(mm, sm[w * 8 * NG + r]);
    float acc = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kDecConsumerWarps; ++w) {
      const int at = w * 8 * NG + r;
      if (sm[at] == -FLT_MAX && sl[at] == 0.f) continue;   // no key of this warp was attended
      ll += fast_exp2(sm[at] - mm) * sl[at];
      acc += exp2f((sm[at] - mm) + sr[at]) * so[at * kRow + d];   // 2^r gives the V scales back
    }
    const int head = kvh * G + r;
    if (p.num_splits == 1) {
      if (p.sinks) acc *= apply_sink(mm, ll, p.sinks[head] * 1.4426950408889634f);
      p.out[static_cast<int64_t>(user) * p.out_row_stride + head * HD + d] =
          __float2bfloat16(ll > 0.f || ll != ll ? acc / ll : 0.f);
    } else {
      const int64_t prow =
          (static_cast<int64_t>(user) * p.num_q_heads + head) * p.num_splits + split;
      p.part_o[prow * HD + d] = acc;
      if (d == 0) p.part_ml[prow] = make_float2(mm == -FLT_MAX && ll == 0.f ? -INFINITY : mm, ll);
    }
  }
  if (p.num_splits > 1 && p.tickets)
    decode_scaled_finish<HD>(p, user, kvh, reinterpret_cast<float*>(ring), threadIdx.x);
}

}  // namespace b200attn

// Norms of queries and keys for each head and the position rotation in one pass, with the
// slot-mapping cache write of the rotated key and of the value.
//
//   x' = x * rsqrt(mean_d x_d^2 + eps) * w_d        per head, w shared by the heads
//   (a, b) -> (a cos f - b sin f, b cos f + a sin f), f = position * inv_freq_i
// with (a, b) = (x'_i, x'_{i + r/2}) (NeoX) or (x'_{2i}, x'_{2i+1}) (interleaved), i < r/2.
//
// Everything is held in fp32 and rounded to bf16 once, at the store.  The angle is formed in
// fp64 and reduced to a fraction of a turn before it is narrowed: at position 10^6 an fp32
// product would be off by up to 0.03 rad.
//
// HBM-bound: each row is read once and written once.  One CTA per token; a head is held by
// HD / 8 neighbouring lanes (eight elements each, in one or two accesses), so the sum of squares is a
// few shuffles and the rotation partner is in the same thread or warp: no shared memory but the
// token's cos / sin row.
#pragma once
#include "kv_scatter.cuh"

namespace b200attn {

struct QkNormRopeParams {
  const __nv_bfloat16* q;
  int64_t q_stride;       // elements between token rows
  const __nv_bfloat16* k;
  int64_t k_stride;
  const __nv_bfloat16* v;
  int64_t v_stride;
  __nv_bfloat16* q_out;
  int64_t q_out_stride;
  __nv_bfloat16* k_out;
  int64_t k_out_stride;
  const void* q_weight;   // [head_size] bf16 or fp32
  const void* k_weight;
  int weight_f32;
  float eps;
  const int64_t* positions;
  const float* inv_freq;  // [rotary_dim / 2]
  int rotary_dim;
  int neox;
  uint8_t* k_cache;
  uint8_t* v_cache;
  int cache_fp8;
  const int64_t* slot_mapping;   // NULL: no cache write
  int num_q_heads;
  int num_kv_heads;
  int log2_block_size;
  int64_t num_blocks;
  int* err_word;
};

__device__ __forceinline__ void unpack_bf16x8_f32x2(const uint4 v, uint64_t (&x)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = pack_f32x2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}

constexpr int kNrThreads = 256;
constexpr int kNrPrefetch = 3;   // head slices a thread loads before it needs the cos / sin row

// How a head lies in its HD / 8 lanes (lane li of the head) and where a rotation partner is:
//   kNrSplit      NeoX, whole head rotated: elements 4 li .. + 3 and HD/2 + 4 li .. + 3, two 8-byte
//                 accesses; both halves of a pair are in one thread
//   kNrShuffle    NeoX, part of the head rotated: elements 8 li .. + 7; the partner is a lane away
//   kNrAdjacent   interleaved: elements 8 li .. + 7, pairs of neighbours
// 8192 tokens of 32 + 8 + 8 heads of 128, cache written: kNrSplit 48 us, kNrAdjacent 51 us,
// kNrShuffle 57 us (its four 64-bit shuffles per thread and head; kNrSplit would need the rotated
// part to be the whole head).  Floor 33 us (218 MB at the measured copy rate); what is left is
// instructions (packed fp32 took it from 54 us; value heads, which only go to the cache, pass through
// the norm too) and the cos / sin row that a CTA waits for once.
enum NrLayout : int { kNrSplit = 0, kNrShuffle = 1, kNrAdjacent = 2 };

template <int HD, int LAYOUT>
__global__ void __launch_bounds__(kNrThreads, 4) qk_norm_rope_kernel(const QkNormRopeParams p) {
  constexpr int kLanes = HD / 8;                    // lanes per head
  constexpr int kHeadsPerPass = kNrThreads / kLanes;
  constexpr int kAngles = LAYOUT == kNrShuffle ? 8 : 4;      // that a thread needs
  __shared__ float4 cs4[HD / 8];
  __shared__ float4 sn4[HD / 8];
  const int64_t t = blockIdx.x;
  const int half = p.rotary_dim / 2;
  const int li = threadIdx.x % kLanes;
  const int h0 = threadIdx.x / kLanes;
  const int nqk = p.num_q_heads + p.num_kv_heads;
  const int all = nqk + (p.slot_mapping ? p.num_kv_heads : 0);   // q, k and (to be written) v heads
  // this token's rows, at this thread's first element of head 0 (k and v seen from their place in
  // the order q, k, v, so that a head's offset is its index times HD for all three)
  constexpr int kEl = LAYOUT == kNrSplit ? 4 : 8;
  const __nv_bfloat16* q_in = p.q + t * p.q_stride + li * kEl;
  const __nv_bfloat16* k_in = p.k + t * p.k_stride + li * kEl - p.num_q_heads * HD;
  const __nv_bfloat16* v_in = p.v + t * p.v_stride + li * kEl - nqk * HD;
  __nv_bfloat16* q_to = p.q_out + t * p.q_out_stride + li * kEl;
  __nv_bfloat16* k_to = p.k_out + t * p.k_out_stride + li * kEl - p.num_q_heads * HD;

  auto load = [&](int head) -> uint4 {
    const __nv_bfloat16* src = (head < p.num_q_heads ? q_in : head < nqk ? k_in : v_in) + head * HD;
    if (LAYOUT == kNrSplit) {
      const uint2 a = *reinterpret_cast<const uint2*>(src);
      const uint2 b = *reinterpret_cast<const uint2*>(src + HD / 2);
      return make_uint4(a.x, a.y, b.x, b.y);
    }
    return *reinterpret_cast<const uint4*>(src);
  };
  auto store = [&](__nv_bfloat16* dst, const uint4 y) {
    if (LAYOUT == kNrSplit) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(y.x, y.y);
      *reinterpret_cast<uint2*>(dst + HD / 2) = make_uint2(y.z, y.w);
    } else {
      *reinterpret_cast<uint4*>(dst) = y;
    }
  };
  uint4 pre[kNrPrefetch];
#pragma unroll
  for (int i = 0; i < kNrPrefetch; ++i) {
    const int head = h0 + i * kHeadsPerPass;
    pre[i] = head < all ? load(head) : make_uint4(0u, 0u, 0u, 0u);
  }

  if (threadIdx.x < half) {
    const double turns = static_cast<double>(p.positions[t]) *
                         static_cast<double>(p.inv_freq[threadIdx.x]) * 0.15915494309189535;
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    reinterpret_cast<float*>(sn4)[threadIdx.x] = s;
    reinterpret_cast<float*>(cs4)[threadIdx.x] = c;
  }
  // element offset of KV head 0's row of this token's slot in the caches; negative: not written
  int64_t cache_row = -1;
  if (p.slot_mapping) {
    const int64_t slot = p.slot_mapping[t];
    if (slot >= 0) {
      const int64_t blk = slot >> p.log2_block_size;
      if (blk >= p.num_blocks) {
        if (threadIdx.x == 0) atomicExch(p.err_word, kDevBadIndex);
      } else {
        const int64_t off = slot & ((1 << p.log2_block_size) - 1);
        cache_row = (((blk * p.num_kv_heads) << p.log2_block_size) + off) * HD + li * kEl;
      }
    }
  }
  auto store_cache = [&](uint8_t* cache, int h, const uint4 y) {
    const int64_t at = cache_row + (static_cast<int64_t>(h * HD) << p.log2_block_size);
    if (!p.cache_fp8) {
      store(reinterpret_cast<__nv_bfloat16*>(cache) + at, y);
      return;
    }
    const uint2 c = bf16x8_to_e4m3x8(y);
    if (LAYOUT == kNrSplit) {
      *reinterpret_cast<uint32_t*>(cache + at) = c.x;
      *reinterpret_cast<uint32_t*>(cache + at + HD / 2) = c.y;
    } else {
      *reinterpret_cast<uint2*>(cache + at) = c;
    }
  };
  __syncthreads();

  // This thread's part in the rotation: which angles, and (kNrShuffle) which lane is the partner:
  // lanes [0, r/16) of a head hold the a's, [r/16, r/8) the b's.
  const int pair_lanes = half / 8;
  const bool rotates = LAYOUT == kNrSplit || li < 2 * pair_lanes;
  const bool second = LAYOUT == kNrShuffle && li >= pair_lanes;
  const int lane = threadIdx.x & 31;
  const int partner = rotates ? (second ? lane - pair_lanes : lane + pair_lanes) : lane;
  float c[kAngles], s[kAngles];
#pragma unroll
  for (int i = 0; i < kAngles; i += 4) {
    float4 cv = make_float4(1.f, 1.f, 1.f, 1.f), sv = make_float4(0.f, 0.f, 0.f, 0.f);
    if (rotates) {
      const int v = LAYOUT == kNrShuffle ? (second ? li - pair_lanes : li) * 2 + i / 4 : li;
      cv = cs4[v];
      sv = sn4[v];
    }
    c[i] = cv.x, c[i + 1] = cv.y, c[i + 2] = cv.z, c[i + 3] = cv.w;
    s[i] = sv.x, s[i + 1] = sv.y, s[i + 2] = sv.z, s[i + 3] = sv.w;
  }
  // Two values a register pair and instruction (packed fp32): w2[i] are elements 2 i, 2 i + 1.
  uint64_t w2[4];
  bool have_k = false;
  auto load_weight = [&](const void* weight) {
    if (p.weight_f32) {
      const float* f = static_cast<const float*>(weight) + li * kEl;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(
            f + (i == 0 ? 0 : LAYOUT == kNrSplit ? HD / 2 : 4)));
        w2[2 * i] = pack_f32x2(v.x, v.y);
        w2[2 * i + 1] = pack_f32x2(v.z, v.w);
      }
    } else {
      const __nv_bfloat16* f = static_cast<const __nv_bfloat16*>(weight) + li * kEl;
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(f));
      const uint2 b = __ldg(reinterpret_cast<const uint2*>(f + (LAYOUT == kNrSplit ? HD / 2 : 4)));
      unpack_bf16x8_f32x2(make_uint4(a.x, a.y, b.x, b.y), w2);
    }
  };
  load_weight(p.q_weight);
  uint64_t c2[kAngles / 2], s2[kAngles / 2], n2[kAngles / 2];      // cos, sin, - sin
#pragma unroll
  for (int i = 0; i < kAngles / 2; ++i) {
    c2[i] = pack_f32x2(c[2 * i], c[2 * i + 1]);
    s2[i] = pack_f32x2(s[2 * i], s[2 * i + 1]);
    n2[i] = pack_f32x2(-s[2 * i], -s[2 * i + 1]);
  }

  auto process = [&](int head, uint4 raw) {   // every lane of the warp comes here
    if (head >= nqk && head < all && cache_row >= 0) store_cache(p.v_cache, head - nqk, raw);
    const bool is_k = head >= p.num_q_heads;
    if (is_k && !have_k) {                    // heads come in ascending order: q, then k
      load_weight(p.k_weight);
      have_k = true;
    }
    uint64_t x[4];
    unpack_bf16x8_f32x2(raw, x);
    uint64_t sq = mul_f32x2(x[0], x[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) sq = fma_f32x2(x[i], x[i], sq);
    float ss, ss1;
    unpack_f32x2(sq, ss, ss1);
    ss += ss1;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * (1.f / HD) + p.eps);
    const uint64_t r2 = pack_f32x2(r, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = mul_f32x2(mul_f32x2(x[i], r2), w2[i]);
    if (LAYOUT == kNrSplit) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint64_t a = x[i], b = x[i + 2];
        x[i] = fma_f32x2(a, c2[i], mul_f32x2(b, n2[i]));
        x[i + 2] = fma_f32x2(b, c2[i], mul_f32x2(a, s2[i]));
      }
    } else if (LAYOUT == kNrShuffle) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t other = __shfl_sync(0xffffffffu, x[i], partner);
        if (rotates) x[i] = fma_f32x2(x[i], c2[i], mul_f32x2(other, second ? s2[i] : n2[i]));
      }
    } else if (rotates) {
      const uint64_t* cp = c2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b, c0, c1, s0, s1;
        unpack_f32x2(x[i], a, b);
        unpack_f32x2(cp[i / 2], c0, c1);
        unpack_f32x2(s2[i / 2], s0, s1);
        const float cc = i & 1 ? c1 : c0, sn = i & 1 ? s1 : s0;
        x[i] = pack_f32x2(a * cc - b * sn, b * cc + a * sn);
      }
    }
    if (head >= nqk) return;
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      unpack_f32x2(x[i], a, b);
      y[i] = pack_bf16x2(a, b);
    }
    const uint4 yy = make_uint4(y[0], y[1], y[2], y[3]);
    if (!is_k) {
      store(q_to + head * HD, yy);
      return;
    }
    store(k_to + head * HD, yy);
    if (cache_row >= 0) store_cache(p.k_cache, head - p.num_q_heads, yy);
  };

  // the bound is rounded up to whole warps: all lanes of a warp take the shuffles together
  const int first_of_warp = (threadIdx.x & ~31) / kLanes;
#pragma unroll
  for (int i = 0; i < kNrPrefetch; ++i)
    if (first_of_warp + i * kHeadsPerPass < all) process(h0 + i * kHeadsPerPass, pre[i]);
  for (int b = kNrPrefetch * kHeadsPerPass; first_of_warp + b < all; b += kHeadsPerPass) {
    const int head = h0 + b;
    process(head, head < all ? load(head) : make_uint4(0u, 0u, 0u, 0u));
  }
}

}  // namespace b200attn

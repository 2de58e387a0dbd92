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
// HD / 8 neighbouring lanes (16 bytes each), so the sum of squares is a few shuffles and the
// rotation partner is a lane of the same warp: no shared memory but the token's cos / sin row.
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
  int block_size;
  int64_t num_blocks;
  int* err_word;
};

__device__ __forceinline__ void unpack_bf16x8(const uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

constexpr int kNrThreads = 256;
constexpr int kNrPrefetch = 3;   // head slices a thread loads before it needs the cos / sin row

template <int HD>
__global__ void __launch_bounds__(kNrThreads) qk_norm_rope_kernel(const QkNormRopeParams p) {
  constexpr int kLanes = HD / 8;                    // lanes per head
  constexpr int kHeadsPerPass = kNrThreads / kLanes;
  __shared__ float cs[HD / 2];
  __shared__ float sn[HD / 2];
  const int64_t t = blockIdx.x;
  const int half = p.rotary_dim / 2;
  const int li = threadIdx.x % kLanes;              // this lane's 8 elements: 8 li .. 8 li + 7
  const int h0 = threadIdx.x / kLanes;

  int64_t blk = -1;
  int off = 0;
  if (p.slot_mapping) {
    const int64_t slot = p.slot_mapping[t];
    if (slot >= 0) {
      blk = slot / p.block_size;
      off = static_cast<int>(slot - blk * p.block_size);
      if (blk >= p.num_blocks) {
        if (threadIdx.x == 0) atomicExch(p.err_word, kDevBadIndex);
        blk = -1;
      }
    }
  }
  const int nqk = p.num_q_heads + p.num_kv_heads;
  const int heads = nqk + (blk >= 0 ? p.num_kv_heads : 0);   // q, k and (when written) v heads

  auto load = [&](int head) -> uint4 {
    const __nv_bfloat16* src;
    if (head < p.num_q_heads)
      src = p.q + t * p.q_stride + static_cast<int64_t>(head) * HD;
    else if (head < nqk)
      src = p.k + t * p.k_stride + static_cast<int64_t>(head - p.num_q_heads) * HD;
    else
      src = p.v + t * p.v_stride + static_cast<int64_t>(head - nqk) * HD;
    return *reinterpret_cast<const uint4*>(src + li * 8);
  };
  uint4 pre[kNrPrefetch];
#pragma unroll
  for (int i = 0; i < kNrPrefetch; ++i) {
    const int head = h0 + i * kHeadsPerPass;
    pre[i] = head < heads ? load(head) : make_uint4(0u, 0u, 0u, 0u);
  }
  float wq[8], wk[8];
  if (p.weight_f32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wq[i] = static_cast<const float*>(p.q_weight)[li * 8 + i];
      wk[i] = static_cast<const float*>(p.k_weight)[li * 8 + i];
    }
  } else {
    unpack_bf16x8(*(static_cast<const uint4*>(p.q_weight) + li), wq);
    unpack_bf16x8(*(static_cast<const uint4*>(p.k_weight) + li), wk);
  }
  if (threadIdx.x < half) {
    const double turns = static_cast<double>(p.positions[t]) *
                         static_cast<double>(p.inv_freq[threadIdx.x]) * 0.15915494309189535;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn[threadIdx.x], &cs[threadIdx.x]);
  }
  __syncthreads();

  // This lane's part in the rotation.  NeoX: lanes [0, r/16) hold the a's, [r/16, r/8) the b's.
  const int pair_lanes = half / 8;
  const bool rotates = li < 2 * pair_lanes;
  const bool second = p.neox && li >= pair_lanes;
  const int lane = threadIdx.x & 31;
  const int partner = rotates && p.neox ? (second ? lane - pair_lanes : lane + pair_lanes) : lane;
  // angle index of element 0: NeoX 8 (li mod r/16), interleaved 4 li
  const int a0 = rotates ? (p.neox ? (second ? li - pair_lanes : li) * 8 : li * 4) : 0;

  auto process = [&](int head, uint4 raw) {   // every lane of the warp comes here
    if (head >= nqk) {
      if (head < heads) {
        const int64_t dst =
            ((blk * p.num_kv_heads + (head - nqk)) * p.block_size + off) * kLanes + li;
        if (p.cache_fp8)
          reinterpret_cast<uint2*>(p.v_cache)[dst] = bf16x8_to_e4m3x8(raw);
        else
          reinterpret_cast<uint4*>(p.v_cache)[dst] = raw;
      }
    }
    float x[8];
    unpack_bf16x8(raw, x);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * (1.f / HD) + p.eps);
    const bool is_k = head >= p.num_q_heads;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (is_k ? wk[i] : wq[i]);
    if (p.neox) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float other = __shfl_sync(0xffffffffu, x[i], partner);
        if (rotates) {
          const float c = cs[a0 + i], s = sn[a0 + i];
          x[i] = second ? x[i] * c + other * s : x[i] * c - other * s;
        }
      }
    } else if (rotates) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float c = cs[a0 + i], s = sn[a0 + i];
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = a * c - b * s;
        x[2 * i + 1] = b * c + a * s;
      }
    }
    if (head >= nqk) return;
    const uint4 y = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                               pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    if (!is_k) {
      *reinterpret_cast<uint4*>(p.q_out + t * p.q_out_stride + static_cast<int64_t>(head) * HD +
                                li * 8) = y;
      return;
    }
    const int h = head - p.num_q_heads;
    *reinterpret_cast<uint4*>(p.k_out + t * p.k_out_stride + static_cast<int64_t>(h) * HD +
                              li * 8) = y;
    if (blk >= 0) {
      const int64_t dst = ((blk * p.num_kv_heads + h) * p.block_size + off) * kLanes + li;
      if (p.cache_fp8)
        reinterpret_cast<uint2*>(p.k_cache)[dst] = bf16x8_to_e4m3x8(y);
      else
        reinterpret_cast<uint4*>(p.k_cache)[dst] = y;
    }
  };

  // the bound is rounded up to whole warps: all lanes of a warp take the shuffles together
  const int first_of_warp = (threadIdx.x & ~31) / kLanes;
#pragma unroll
  for (int i = 0; i < kNrPrefetch; ++i)
    if (first_of_warp + i * kHeadsPerPass < heads) process(h0 + i * kHeadsPerPass, pre[i]);
  for (int b = kNrPrefetch * kHeadsPerPass; first_of_warp + b < heads; b += kHeadsPerPass) {
    const int head = h0 + b;
    process(head, head < heads ? load(head) : make_uint4(0u, 0u, 0u, 0u));
  }
}

}  // namespace b200attn

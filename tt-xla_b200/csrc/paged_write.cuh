// Varlen KV-cache write that keeps what belongs to a whole page: the scale of an 8-bit page and
// the key bounds that page selection reads.
//
// Sequence s's new tokens (rows cu_q[s] .. cu_q[s+1] of key / value) go to positions q_start[s],
// q_start[s] + 1, ... through its page-table row.  A page and KV head is one unit of work with one
// owner CTA, so nothing is accumulated with atomics and a result does not depend on any order.
//
// Scale of a page and head (K and V apart), x the new rows, need = max|x| * (1 / qmax) in fp32
// (qmax 127 or 448, its reciprocal rounded to fp32):
//   * a page whose first row is written starts afresh: scale = need;
//   * a page that goes on keeps its scale while need <= scale, else the scale grows by the
//     smallest power of two that is enough, 2^n, and the rows that stay (those before the first new
//     one; what lies behind the new rows is dead) are re-rounded to code * 2^-n.  Power-of-two steps
//     make that exact for e4m3 (but for its subnormals), and for int8 bound what all re-roundings of
//     a page together can cost by one step of the final scale, however often a page grows (steps s,
//     s/2, s/4, ... add up to less than s);
//   * a NaN or an infinity cannot be held: the scale becomes NaN, so everything read through the
//     page is NaN until it is started afresh, and the codes are 0.
// code = round(x / scale), ties to even, of the 32-bit quotient, so the codes are reproducible.
//
// Key bounds of a page and head: the least and the greatest key of each channel, merged with what
// is there unless the page starts afresh (NaN keys make the channel's bounds NaN).
//
// Memory-bound: 2 bytes read and 1 written per element.  Grid (page of the batch, KV head, K / V),
// 128 threads that hold a page's rows of one head in registers (16 elements each per pass), so the
// rows are read once for both the maximum and the codes.
// Measured: 8192 tokens of 8 heads of 128 (50 MB) 15.7 us in int8 (16.7 with bounds), 16.9 us in e4m3
// (3.2 / 3.0 TB/s: nearly two rounds of CTAs, each a chain of offsets, rows, maximum and codes during
// which nothing of another page is loaded); in bf16 with bounds (68 MB) 14.2 us; one token for each
// of 64 sequences 5.1 us in int8, 4.1 in bf16, launch and the same chain.
#pragma once
#include "kv_scatter.cuh"

namespace b200attn {

enum PageFormat : int { kPageBf16 = 0, kPageE4m3 = 1, kPageInt8 = 2 };

struct PagedWriteParams {
  uint8_t* cache[2];            // K, V
  const __nv_bfloat16* src[2];  // key, value rows
  int64_t src_stride[2];        // elements between token rows
  float* scale[2];              // [num_blocks, num_kv_heads] (8-bit formats)
  __nv_bfloat16* bounds;        // [num_blocks, num_kv_heads, 2, head_size] or NULL
  const int32_t* page_table;
  int64_t page_table_stride;
  int page_table_width;
  const int32_t* cu_q;          // [num_seqs + 1], NULL: one token per sequence
  const int32_t* q_len;         // [num_seqs] tokens to write of each sequence, NULL: all
  const int32_t* q_start;       // [num_seqs]; negative: the sequence is skipped
  int num_seqs;
  int total_tokens;
  int num_kv_heads;
  int64_t num_blocks;
  int* err_word;
};

// Item space over cu_q: sequence s owns items [base(s), base(s + 1)) with
// base(s) = cu_q[s] / BS + 2 s, which leaves room for the pages of any start offset.
template <int BS>
__device__ __forceinline__ int64_t write_item_base(const PagedWriteParams& p, int s) {
  const int c = p.cu_q[s];
  return static_cast<int64_t>(c > 0 ? c / BS : 0) + 2 * static_cast<int64_t>(s);
}

// The sequence that owns `item`, found by the 32 lanes of a warp together.
template <int BS>
__device__ __forceinline__ int write_item_seq(const PagedWriteParams& p, int64_t item, int lane) {
  int lo = 0, n = p.num_seqs;     // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int s = lo + lane * step;
    const bool le = lane * step < n && write_item_base<BS>(p, s) <= item;
    const int k = __popc(__ballot_sync(0xffffffffu, le));
    if (k == 0) return lo;        // lengths out of order: the caller's range checks catch it
    lo += (k - 1) * step;
    n = min(step, n - (k - 1) * step);
  }
  return lo;
}

__device__ __forceinline__ uint32_t int8x4(float a, float b, float c, float d) {
  auto code = [](float x) {       // NaN -> 0
    return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(x)))) & 0xffu;
  };
  return code(a) | (code(b) << 8) | (code(c) << 16) | (code(d) << 24);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
template <int FMT>
__device__ __forceinline__ uint32_t codes_x4(float a, float b, float c, float d) {
  return FMT == kPageInt8 ? int8x4(a, b, c, d) : e4m3x4(a, b, c, d);
}
// int8 codes of x[0..3] / scale from the products with r = 1 / scale.  A product differs from the
// quotient by less than 3 units in the last place (127 * 3 * 2^-24 < 1e-4), which decides nothing
// unless it lies that close to the middle between two whole numbers: `near` is set then (and for
// NaN), and the caller divides.  Adding 1.5 * 2^23 rounds to a whole number, ties to even, and
// leaves it in the low bits.
__device__ __forceinline__ uint32_t int8x4_by_product(const float (&x)[4], float r, bool& near) {
  constexpr float kMagic = 12582912.f;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = x[i] * r, u = t + kMagic;
    near |= !(fabsf(t - (u - kMagic)) < 0.4999f);
    w[i] = __float_as_uint(u);
  }
  return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}

// four codes -> four floats, exact
template <int FMT>
__device__ __forceinline__ void codes_to_f32(uint32_t w, float (&x)[4]) {
  if (FMT == kPageInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = static_cast<float>(static_cast<int8_t>((w >> (8 * i)) & 0xffu));
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t h;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;"
          : "=r"(h)
          : "h"(static_cast<uint16_t>(w >> (16 * i))));
      asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
          "cvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
          : "=f"(x[2 * i]), "=f"(x[2 * i + 1])
          : "r"(h));
    }
  }
}

// smallest n >= 0 with scale * 2^n >= need (scale, need > 0 and finite)
__device__ __forceinline__ int scale_steps(float scale, float need) {
  int es, en;
  const float ms = frexpf(scale, &es), mn = frexpf(need, &en);
  const int n = en - es + (mn > ms ? 1 : 0);
  return n > 0 ? n : 0;
}

constexpr int kPwThreads = 128;

template <int HD, int BS, int FMT>
__global__ void __launch_bounds__(kPwThreads, 8) paged_write_kernel(const PagedWriteParams p) {
  constexpr int kLanes = HD / 16;                       // threads per row
  constexpr int kRowsPerPass = kPwThreads / kLanes;
  constexpr int kPasses = (BS + kRowsPerPass - 1) / kRowsPerPass;
  __shared__ uint32_t warp_max[kPwThreads / 32];
  __shared__ uint32_t red[2][kPwThreads / 32][HD / 2];  // bounds, two channels a word
  const int h = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which page of which sequence
  int s, tok0, page_of_chunk;
  int64_t len;
  if (p.cu_q) {
    s = write_item_seq<BS>(p, blockIdx.x, lane);
    tok0 = p.cu_q[s];
    const int end = p.cu_q[s + 1];
    if (tok0 < 0 || end < tok0 || end > p.total_tokens) {
      if (threadIdx.x == 0) atomicExch(p.err_word, kDevBadIndex);
      return;
    }
    len = end - tok0;
    page_of_chunk = static_cast<int>(blockIdx.x - write_item_base<BS>(p, s));
  } else {
    s = blockIdx.x;
    tok0 = s;
    len = 1;
    page_of_chunk = 0;
  }
  const int start = p.q_start[s];
  if (p.q_len) len = min(len, static_cast<int64_t>(p.q_len[s]));
  if (start < 0 || len <= 0 || page_of_chunk < 0) return;
  const int64_t col = start / BS + static_cast<int64_t>(page_of_chunk);
  const int64_t lo = max(static_cast<int64_t>(start), col * BS);
  const int64_t hi = min(static_cast<int64_t>(start) + len, (col + 1) * BS);
  if (lo >= hi) return;
  const int r0 = static_cast<int>(lo - col * BS);       // first new row of the page
  const int n = static_cast<int>(hi - lo);
  const bool fresh = r0 == 0;

  // ---- the new rows: their loads go out before the page id is known
  const int c = threadIdx.x % kLanes, r = threadIdx.x / kLanes;
  const int64_t stride = is_v ? p.src_stride[1] : p.src_stride[0];
  const __nv_bfloat16* src = (is_v ? p.src[1] : p.src[0]) + (tok0 + (lo - start)) * stride +
                             static_cast<int64_t>(h) * HD + c * 16;
  uint4 x[kPasses][2];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int row = i * kRowsPerPass + r;
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    if (row < n) {
      const uint4* at = reinterpret_cast<const uint4*>(src + row * stride);
      x[i][0] = __ldg(at);
      x[i][1] = __ldg(at + 1);
    }
  }
  int64_t blk = -1;
  if (col < p.page_table_width)
    blk = p.page_table[static_cast<int64_t>(s) * p.page_table_stride + col];
  if (blk < 0 || blk >= p.num_blocks) {
    if (threadIdx.x == 0) atomicExch(p.err_word, kDevBadIndex);
    return;
  }
  const int64_t page = blk * p.num_kv_heads + h;
  float* scale_ptr = nullptr;
  float old = 0.f;
  if (FMT != kPageBf16) {
    scale_ptr = (is_v ? p.scale[1] : p.scale[0]) + page;
    if (!fresh) old = *scale_ptr;
  }

  // ---- key bounds
  if (p.bounds && !is_v) {
    uint32_t mn[8], mx[8];        // channels 16 c + 2 j, + 1
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mn[j] = 0x7f807f80u;        // +inf
      mx[j] = 0xff80ff80u;        // -inf
    }
    auto lo2 = [](uint32_t a, uint32_t b) {
      uint32_t o;
      asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(o) : "r"(a), "r"(b));
      return o;
    };
    auto hi2 = [](uint32_t a, uint32_t b) {
      uint32_t o;
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o) : "r"(a), "r"(b));
      return o;
    };
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      if (i * kRowsPerPass + r < n) {
        const uint32_t w[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w,
                               x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          mn[j] = lo2(mn[j], w[j]);
          mx[j] = hi2(mx[j], w[j]);
        }
      }
    }
#pragma unroll
    for (int o = 16; o >= kLanes; o >>= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        mn[j] = lo2(mn[j], __shfl_xor_sync(0xffffffffu, mn[j], o));
        mx[j] = hi2(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
      }
    if (lane < kLanes)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        red[0][warp][c * 8 + j] = mn[j];
        red[1][warp][c * 8 + j] = mx[j];
      }
    __syncthreads();
    uint32_t* b = reinterpret_cast<uint32_t*>(p.bounds + page * 2 * HD);
    for (int i = threadIdx.x; i < HD; i += kPwThreads) {     // HD / 2 words of each kind
      const bool top = i >= HD / 2;
      const int j = top ? i - HD / 2 : i;
      uint32_t v = red[top][0][j];
#pragma unroll
      for (int w = 1; w < kPwThreads / 32; ++w)
        v = top ? hi2(v, red[1][w][j]) : lo2(v, red[0][w][j]);
      if (!fresh) v = top ? hi2(v, b[i]) : lo2(v, b[i]);
      b[i] = v;
    }
  }

  uint8_t* out = is_v ? p.cache[1] : p.cache[0];
  if (FMT == kPageBf16) {
    uint4* dst = reinterpret_cast<uint4*>(out) + (page * BS + r0) * (HD / 8) + c * 2;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = i * kRowsPerPass + r;
      if (row < n) {
        dst[row * (HD / 8)] = x[i][0];
        dst[row * (HD / 8) + 1] = x[i][1];
      }
    }
    return;
  }

  // ---- the scale
  uint32_t top = 0;               // largest |bf16| pattern; 0x7f80 and above: not finite
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const uint32_t w[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w,
                           x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) top = __vmaxu2(top, w[j] & 0x7fff7fffu);
  }
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) warp_max[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPwThreads / 32; ++w) top = max(top, warp_max[w]);
  constexpr float kQmax = FMT == kPageInt8 ? 127.f : 448.f;
  const float need = __fmul_rn(__uint_as_float(top << 16), 1.f / kQmax);
  float now = need, shrink = 1.f;
  if (!fresh) {
    if (!(old >= 0.f) || old == INFINITY) {
      now = NAN;
    } else if (old > 0.f) {
      now = old;
      if (need > old && top < 0x7f80u) {
        const int steps = scale_steps(old, need);
        now = ldexpf(old, steps);
        shrink = ldexpf(1.f, -steps);
      }
    }
  }
  if (top >= 0x7f80u) now = NAN;
  // every thread has the old scale in a register by now (the barrier above)
  if (threadIdx.x == 0) *scale_ptr = now;

  // ---- codes: the rows that stay, re-rounded when the scale grew, then the new rows
  uint4* base = reinterpret_cast<uint4*>(out) + page * BS * kLanes;
  if (shrink != 1.f) {
    for (int i = threadIdx.x; i < r0 * kLanes; i += kPwThreads) {
      const uint4 v = base[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[4];
        codes_to_f32<FMT>(w[j], f);
        o[j] = codes_x4<FMT>(f[0] * shrink, f[1] * shrink, f[2] * shrink, f[3] * shrink);
      }
      base[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
  const bool live = now > 0.f;    // false for a zero and for a NaN scale: all codes are 0
  // int8 by products (15.6 us instead of 19.5 for 8192 tokens of 8 heads of 128); e4m3, whose
  // middles take more to recognise, by division (16.7 us, 24 by products)
  const bool by_product = FMT == kPageInt8 && now > 1e-30f && now < 1e30f;
  const float rec = by_product ? 1.f / now : 0.f;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int row = i * kRowsPerPass + r;
    if (row < n) {
      uint32_t o[4] = {0u, 0u, 0u, 0u};
      const uint32_t w[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w,
                             x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
      if (live) {
        bool divide = !by_product;
        if (by_product) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float f[4] = {
                __uint_as_float(w[2 * j] << 16), __uint_as_float(w[2 * j] & 0xffff0000u),
                __uint_as_float(w[2 * j + 1] << 16), __uint_as_float(w[2 * j + 1] & 0xffff0000u)};
            o[j] = int8x4_by_product(f, rec, divide);
          }
        }
        if (divide) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = codes_x4<FMT>(
                __fdiv_rn(__uint_as_float(w[2 * j] << 16), now),
                __fdiv_rn(__uint_as_float(w[2 * j] & 0xffff0000u), now),
                __fdiv_rn(__uint_as_float(w[2 * j + 1] << 16), now),
                __fdiv_rn(__uint_as_float(w[2 * j + 1] & 0xffff0000u), now));
        }
      }
      base[(r0 + row) * kLanes + c] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// ------------------------------------------------------------------------------------------
// Widening of the pages a prefill batch reads from a block-scaled cache into a bf16 page pool
// (the pool layout of dequant_pages_kernel).
//
// A code has at most 7 significant bits, so code * 2^e is exact in bf16; code * scale is not, and
// its rounding would be as large as the one of the result.  The pool therefore holds code * 2^e
// with scale = f * 2^e, 1 <= f < 2, and the attention kernel applies the factors f in fp32:
// `factors` gets (f of K, log2 f of V) for each page and head of the pool.  A zero scale gives zeros
// and f = 1.  A page whose K or V scale is NaN (or no scale at all: negative, infinite), or whose id
// is out of range (reported), gets NaN keys and zero values: rows that attend it come out as NaN,
// rows for which it is masked do not.  Memory-bound: 1 byte read and 2 written per element (2 x 4608 tokens of 8 heads of 128,
// 55 MB: 15 us).
struct DequantScaledParams {
  const uint8_t* src[2];
  __nv_bfloat16* dst[2];
  const float* scale[2];
  float2* factors;            // [num_seqs * page_table_width, num_kv_heads]
  const int32_t* page_table;
  int64_t page_table_stride;
  int page_table_width;
  const int32_t* cu_q;
  const int32_t* q_start;
  int max_context_len;        // > 0: a longer context is reported
  int num_kv_heads;
  int64_t num_blocks;
  int* err_word;
};

// scale -> f in [1, 2) and 2^e in two factors (2^e alone may be subnormal)
struct SplitScale {
  float f, p0, p1;
};
__device__ __forceinline__ SplitScale split_scale(float s) {
  SplitScale r{1.f, 0.f, 0.f};
  if (s > 0.f) {
    int e;
    r.f = 2.f * frexpf(s, &e);
    const int half = (e - 1) / 2;
    r.p0 = ldexpf(1.f, half);
    r.p1 = ldexpf(1.f, e - 1 - half);
  }
  return r;
}

// grid (page slot * KV head, sequence, K / V)
template <int HD, int BS, int FMT>
__global__ void __launch_bounds__(128) dequant_scaled_kernel(const DequantScaledParams p) {
  constexpr int kVecs = BS * HD / 16;              // 16 codes each
  const int slot = blockIdx.x / p.num_kv_heads, h = blockIdx.x - slot * p.num_kv_heads;
  const int seq = blockIdx.y, z = blockIdx.z;
  const int len = p.cu_q[seq + 1] - p.cu_q[seq];
  const int64_t ctx = static_cast<int64_t>(p.q_start ? p.q_start[seq] : 0) + len;
  if (blockIdx.x == 0 && z == 0 && threadIdx.x == 0 && p.max_context_len > 0 && len > 0 &&
      ctx > p.max_context_len)
    atomicExch(p.err_word, kDevBadIndex);
  if (len <= 0 || slot >= (ctx + BS - 1) / BS) return;
  const int64_t blk = p.page_table[static_cast<int64_t>(seq) * p.page_table_stride + slot];
  const int64_t dst_page =
      (static_cast<int64_t>(seq) * p.page_table_width + slot) * p.num_kv_heads + h;
  const bool ok = blk >= 0 && blk < p.num_blocks;
  if (!ok && threadIdx.x == 0) atomicExch(p.err_word, kDevBadIndex);
  const int64_t src_page = (ok ? blk : 0) * p.num_kv_heads + h;
  const float ks = __ldg(p.scale[0] + src_page), vs = __ldg(p.scale[1] + src_page);
  const bool live = ok && ks >= 0.f && ks < INFINITY && vs >= 0.f && vs < INFINITY;
  const SplitScale sp = split_scale(z ? vs : ks);
  if (threadIdx.x == 0 && z == 0)
    p.factors[dst_page] = live ? make_float2(sp.f, log2f(split_scale(vs).f)) : make_float2(1.f, 0.f);
  const uint4* src = reinterpret_cast<const uint4*>(z ? p.src[1] : p.src[0]) + src_page * kVecs;
  uint4* dst = reinterpret_cast<uint4*>(z ? p.dst[1] : p.dst[0]) + dst_page * kVecs * 2;
  constexpr int kUnroll = kVecs / 128;
  static_assert(kVecs % 128 == 0, "whole passes");
  uint4 in[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) in[u] = __ldg(src + u * 128 + threadIdx.x);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int i = u * 128 + threadIdx.x;
    const uint32_t w[4] = {in[u].x, in[u].y, in[u].z, in[u].w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[4];
      codes_to_f32<FMT>(w[j], f);
      o[2 * j] = pack_bf16x2(f[0] * sp.p0 * sp.p1, f[1] * sp.p0 * sp.p1);
      o[2 * j + 1] = pack_bf16x2(f[2] * sp.p0 * sp.p1, f[3] * sp.p0 * sp.p1);
      if (!live) o[2 * j] = o[2 * j + 1] = z ? 0u : 0x7fc07fc0u;
    }
    dst[2 * i] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[2 * i + 1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

}  // namespace b200attn

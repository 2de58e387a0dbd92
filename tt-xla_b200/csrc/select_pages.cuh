// Page selection for block-sparse decode attention: which pages of its context a (user, KV head)
// attends to, by a cheap score from the pages' key bounds.
//
//   score[p] = max over the G query heads of  sum_d min(q_d, 0) kmin[p, d] + max(q_d, 0) kmax[p, d]
// is the largest logit (before the softmax scale) that any key of page p can have.  The first
// `keep_first` and the last `keep_last` pages are always taken, the rest of the `num_pages` by
// score; equal scores go to the lower page.  A score that is not a number ranks first.
//
// Scoring is memory-bound: 4 * head_size bytes of bounds per page and KV head.  16 pages x 8 query
// heads x 16 channels are one m16n8k16 MMA (rows = pages), fed from global memory by 16-byte loads:
// the channel order within the contraction is free as long as q is loaded in the same order, so no
// shared memory and no shuffles are needed.
//
// The choice is the one the exact scores make.  bf16 products are exact in fp32 and the fp32 sum of
// 2 * head_size of them is off by at most 4 * head_size * 2^-23 times the sum of their magnitudes
// (a second MMA with |q| and |bounds|): 2 * head_size terms and head_size / 8 accumulators are
// added, each addition truncating at worst, and the factor covers that almost twice.  Only pages
// whose fp32 score is within twice that of the border can be on the wrong side of it: these few
// are summed again in fp64, and the border is drawn among them.
//
// One launch: the CTAs of a (user, KV head) each score a slice of the pages; the one that arrives
// last (a ticket in the workspace) makes the choice.
#pragma once
#include "kv_scatter.cuh"

namespace b200attn {

struct SelectPagesParams {
  const __nv_bfloat16* q;
  int64_t q_row_stride;
  const __nv_bfloat16* bounds;   // [num_blocks, nkv, 2, hd]
  const int32_t* page_table;
  int64_t page_table_stride;
  int page_table_width;
  const int32_t* cur_pos;        // [users]
  int32_t* out_table;            // [users, nkv, num_pages]
  int32_t* out_pos;              // [users, nkv]
  int num_q_heads;
  int num_kv_heads;
  int group;
  int64_t num_blocks;
  int num_pages;
  int keep_first;
  int keep_last;
  int max_pages;                 // page-table width: row length of the scratch
  int slice;                     // pages per CTA, a multiple of 16
  unsigned int* tickets;         // [users, nkv], zero between launches
  float2* score;                 // [users, nkv, max_pages]  (score, its possible error)
  unsigned long long* exact;     // [users, nkv, max_pages]  ordered fp64 score / mark
  int* err_word;
};

__device__ __forceinline__ uint32_t ordered_key(float x) {      // larger float, larger key
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long ordered_key(double x) {
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(x == 0.0 ? 0.0 : x));
  return b >> 63 ? ~b : b | (1ull << 63);
}

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;

struct SelectShared {
  unsigned int hist[256];
  unsigned int warp_sum[kSelWarps];
  float warp_err[kSelWarps];
  unsigned int digit, left, count_sure, count_near;
  int last;
};

// The k-th largest (k >= 1) of the keys key(i), i in [0, n) with use(i); at least k of them are
// used.  Eight bits a pass from the top; all threads return the key.  `left` returns how many of
// the keys equal to it belong to the k largest.
template <typename Key, typename Use, typename Get>
__device__ Key kth_largest(SelectShared& sh, int n, unsigned int k, Use use, Get get,
                           unsigned int* left) {
  Key prefix = 0, mask = 0;
  for (int shift = static_cast<int>(sizeof(Key)) * 8 - 8; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kSelThreads) sh.hist[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSelThreads) {
      if (!use(i)) continue;
      const Key v = get(i);
      if ((v & mask) == prefix) atomicAdd(&sh.hist[(v >> shift) & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      // lane l owns digits 255 - 8 l .. 248 - 8 l, from the top
      unsigned int h[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[j] = sh.hist[255 - 8 * static_cast<int>(threadIdx.x) - j];
        sum += h[j];
      }
      unsigned int above = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned int up = __shfl_up_sync(0xffffffffu, above, o);
        if (static_cast<int>(threadIdx.x) >= o) above += up;
      }
      above -= sum;
      if (above < k && k <= above + sum) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (above < k && k <= above + h[j]) {
            sh.digit = 255 - 8 * threadIdx.x - j;
            sh.left = k - above;
          }
          above += h[j];
        }
      }
    }
    __syncthreads();
    prefix |= static_cast<Key>(sh.digit) << shift;
    mask |= static_cast<Key>(255) << shift;
    k = sh.left;
    __syncthreads();
  }
  *left = k;
  return prefix;
}

// Exclusive position of each set flag in thread order, and the number of flags (all threads call).
__device__ __forceinline__ unsigned int block_rank(SelectShared& sh, bool flag, unsigned int* total) {
  const unsigned int b = __ballot_sync(0xffffffffu, flag);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sh.warp_sum[warp] = __popc(b);
  __syncthreads();
  unsigned int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    const unsigned int c = sh.warp_sum[w];
    before += w < warp ? c : 0u;
    all += c;
  }
  __syncthreads();
  *total = all;
  return before + __popc(b & ((1u << lane) - 1u));
}

// fp64 score of one page, by a warp.
template <int HD>
__device__ double exact_page_score(const SelectPagesParams& p, int user, int kvh, int64_t blk,
                                   int lane) {
  const __nv_bfloat16* b = p.bounds + (blk * p.num_kv_heads + kvh) * 2 * HD;
  double best = -INFINITY;
  for (int g = 0; g < p.group; ++g) {
    const __nv_bfloat16* q = p.q + static_cast<int64_t>(user) * p.q_row_stride +
                             (static_cast<int64_t>(kvh) * p.group + g) * HD;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int d = i * 32 + lane;
      const float x = __bfloat162float(q[d]);
      const float lo = __bfloat162float(b[d]), hi = __bfloat162float(b[HD + d]);
      // the products have 16 significant bits: exact in fp64, like the sums of such a range
      const double neg = x > 0.f ? 0.0 : x, pos = x < 0.f ? 0.0 : x;   // a NaN stays in both
      sum += neg * lo + pos * hi;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sum != sum) sum = INFINITY;
    best = sum > best ? sum : best;
  }
  return best;
}

template <int HD, int BS, int NG>
__global__ void __launch_bounds__(kSelThreads) select_pages_kernel(const SelectPagesParams p) {
  __shared__ SelectShared sh;
  const int kvh = blockIdx.y, user = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pos = p.cur_pos[user];
  const int64_t uh = static_cast<int64_t>(user) * p.num_kv_heads + kvh;
  int32_t* table = p.out_table + uh * p.num_pages;
  const int32_t* pt = p.page_table + static_cast<int64_t>(user) * p.page_table_stride;
  int n = pos < 0 ? 0 : pos / BS + 1;
  n = min(n, p.max_pages);
  // position within the last page: a context longer than the table ends with the table
  const int in_page = pos < 0 ? 0 : (pos / BS + 1 > n ? BS - 1 : pos % BS);

  if (n <= p.num_pages) {            // everything is taken
    if (blockIdx.x != 0) return;
    for (int i = threadIdx.x; i < p.num_pages; i += kSelThreads) table[i] = i < n ? pt[i] : 0;
    if (threadIdx.x == 0) p.out_pos[uh] = n == 0 ? -1 : (n - 1) * BS + in_page;
    return;
  }

  // ---------------------------------------------------------------- scores of this CTA's slices
  const int num_slices = (n + p.slice - 1) / p.slice;
  const int arrivals = min(num_slices, static_cast<int>(gridDim.x));
  if (static_cast<int>(blockIdx.x) >= num_slices) return;   // beyond the context: takes no ticket
  float2* score = p.score + uh * p.max_pages;
  const int g = lane >> 2, tq = lane & 3;
  {
    // Q fragments (B operand: columns = query heads 8 ng + g): positive and negative part.  The
    // thread's 8 elements 32 j + 8 tq .. + 7 of a 32-channel step serve two k-steps of four.
    uint32_t qp[NG][HD / 16][2], qn[NG][HD / 16][2];
#pragma unroll
    for (int ng = 0; ng < NG; ++ng) {
      const int head = ng * 8 + g;
      const __nv_bfloat16* q = p.q + static_cast<int64_t>(user) * p.q_row_stride +
                               (static_cast<int64_t>(kvh) * p.group + head) * HD;
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) {
        const uint4 v = head < p.group ? *reinterpret_cast<const uint4*>(q + j * 32 + tq * 8)
                                       : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t a, b;
          asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(w[e]), "r"(0u));
          asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(w[e]), "r"(0u));
          qp[ng][2 * j + (e >> 1)][e & 1] = a;
          qn[ng][2 * j + (e >> 1)][e & 1] = b;
        }
      }
    }
    // a slice's 16-page groups go to the warps in turn; then this CTA's next slice
    int slice = blockIdx.x;
    for (int p0 = slice * p.slice + warp * 16;; p0 += kSelWarps * 16) {
      int end = min(n, (slice + 1) * p.slice);
      while (p0 >= end) {
        slice += gridDim.x;
        if (slice >= num_slices) break;
        p0 = slice * p.slice + warp * 16;
        end = min(n, (slice + 1) * p.slice);
      }
      if (slice >= num_slices) break;
      const int rows[2] = {p0 + g, p0 + g + 8};
      const uint4* src[2];
      bool ok[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int64_t blk = rows[r] < end ? pt[rows[r]] : -1;
        ok[r] = blk >= 0 && blk < p.num_blocks;
        if (!ok[r] && rows[r] < end && tq == 0) atomicExch(p.err_word, kDevBadIndex);
        src[r] = reinterpret_cast<const uint4*>(
                     p.bounds + ((ok[r] ? blk : 0) * p.num_kv_heads + kvh) * 2 * HD) + tq;
      }
      uint4 b[2][2][HD / 32];        // [row][min / max][32-channel step]
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < HD / 32; ++j)
            b[r][k][j] = ok[r] ? __ldg(src[r] + k * (HD / 8) + j * 4) : make_uint4(0u, 0u, 0u, 0u);
      float s[NG][4], a[NG][4];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[ng][i] = a[ng][i] = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const uint32_t w0[4] = {b[0][k][j].x, b[0][k][j].y, b[0][k][j].z, b[0][k][j].w};
          const uint32_t w1[4] = {b[1][k][j].x, b[1][k][j].y, b[1][k][j].z, b[1][k][j].w};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t f[4] = {w0[2 * e], w1[2 * e], w0[2 * e + 1], w1[2 * e + 1]};
            const uint32_t m[4] = {f[0] & 0x7fff7fffu, f[1] & 0x7fff7fffu, f[2] & 0x7fff7fffu,
                                   f[3] & 0x7fff7fffu};
#pragma unroll
            for (int ng = 0; ng < NG; ++ng) {
              const uint32_t* qq = k ? qp[ng][2 * j + e] : qn[ng][2 * j + e];
              mma_bf16_16816(s[ng], f, qq[0], qq[1]);
              mma_bf16_16816(a[ng], m, qq[0] & 0x7fff7fffu, qq[1] & 0x7fff7fffu);
            }
          }
        }
      // columns 8 ng + 2 tq, + 1; rows g (i < 2) and g + 8
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float best = -INFINITY, mag = 0.f;
#pragma unroll
        for (int ng = 0; ng < NG; ++ng)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (ng * 8 + 2 * tq + i < p.group) {
              const float v = s[ng][2 * r + i], w = a[ng][2 * r + i];
              best = fmaxf(best, v != v ? INFINITY : v);
              mag = fmaxf(mag, w != w ? INFINITY : w);
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
          mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, o));
        }
        if (tq == 0 && rows[r] < end)
          score[rows[r]] = ok[r] ? make_float2(best, mag * (4.f * HD / 8388608.f))
                                 : make_float2(-INFINITY, 0.f);
      }
    }
  }

  // ---------------------------------------------------------------- the last CTA chooses
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0)
    sh.last = atomicAdd(p.tickets + uh, 1u) == static_cast<unsigned int>(arrivals - 1);
  __syncthreads();
  if (!sh.last) return;
  __threadfence();
  if (threadIdx.x == 0) {
    p.tickets[uh] = 0u;              // leave the counter as the next launch expects it
    sh.count_sure = sh.count_near = 0u;
  }
  const int e0 = p.keep_first, m = n - p.keep_last - p.keep_first;   // candidates e0 .. e0 + m - 1
  const unsigned int want = static_cast<unsigned int>(p.num_pages - p.keep_first - p.keep_last);
  unsigned long long* exact = p.exact + uh * p.max_pages;
  const float2* sc = score + e0;
  constexpr unsigned long long kPicked = ~0ull;

  float border = INFINITY, width = 0.f;
  bool take_all_near = true;
  __syncthreads();
  if (want > 0) {
    float err = 0.f;
    for (int i = threadIdx.x; i < m; i += kSelThreads) err = fmaxf(err, __ldcg(sc + i).y);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) err = fmaxf(err, __shfl_xor_sync(0xffffffffu, err, o));
    if (lane == 0) sh.warp_err[warp] = err;
    unsigned int left;
    const uint32_t key = kth_largest<uint32_t>(
        sh, m, want, [](int) { return true; },
        [&](int i) { return ordered_key(__ldcg(sc + i).x); }, &left);
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) err = fmaxf(err, sh.warp_err[w]);
    border = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    // both the page's and the border's score may be off by err; the difference is rounded once
    width = 2.f * err * 1.000001f;
    // above: surely among the `want` best; near: may be on either side
    unsigned int sure = 0, near = 0;
    for (int i = threadIdx.x; i < m; i += kSelThreads) {
      const float s = __ldcg(sc + i).x;
      const bool is_near = s == border || fabsf(s - border) <= width;
      sure += !is_near && s > border;
      near += is_near;
    }
    sure = __reduce_add_sync(0xffffffffu, sure);
    near = __reduce_add_sync(0xffffffffu, near);
    if (lane == 0) {
      atomicAdd(&sh.count_sure, sure);
      atomicAdd(&sh.count_near, near);
    }
    __syncthreads();
    const unsigned int open = want - sh.count_sure;      // places for the near ones
    take_all_near = open == sh.count_near;
    if (!take_all_near) {
      auto is_near = [&](int i) {
        const float s = __ldcg(sc + i).x;
        return s == border || fabsf(s - border) <= width;
      };
      for (int i = warp; i < m; i += kSelWarps) {
        if (!is_near(i)) continue;                       // uniform in the warp
        const int64_t blk = pt[e0 + i];
        const bool ok = blk >= 0 && blk < p.num_blocks;
        const double v = ok ? exact_page_score<HD>(p, user, kvh, blk, lane) : -INFINITY;
        if (lane == 0) exact[e0 + i] = ordered_key(v);
      }
      __syncthreads();
      unsigned int ties;
      const unsigned long long at = kth_largest<unsigned long long>(
          sh, m, open, is_near, [&](int i) { return exact[e0 + i]; }, &ties);
      // mark the chosen ones; of the keys equal to the border's the first `ties`
      unsigned int before = 0;
      for (int i0 = 0; i0 < m; i0 += kSelThreads) {
        const int i = i0 + threadIdx.x;
        const bool here = i < m && is_near(i);
        const unsigned long long v = here ? exact[e0 + i] : 0ull;
        unsigned int total;
        const unsigned int rank = before + block_rank(sh, here && v == at, &total);
        before += total;
        if (here) exact[e0 + i] = v > at || (v == at && rank < ties) ? kPicked : 0ull;
      }
      __syncthreads();
    }
  }

  // ---------------------------------------------------------------- the list, in page order
  unsigned int filled = 0;
  for (int i0 = 0; i0 < n; i0 += kSelThreads) {
    const int i = i0 + threadIdx.x;
    bool take = i < e0 || (i >= n - p.keep_last && i < n);
    if (i >= e0 && i < e0 + m && want > 0) {
      const float s = __ldcg(score + i).x;
      const bool is_near = s == border || fabsf(s - border) <= width;
      take = is_near ? take_all_near || exact[i] == kPicked : s > border;
    }
    unsigned int total;
    const unsigned int at = filled + block_rank(sh, take, &total);
    if (take && at < static_cast<unsigned int>(p.num_pages)) table[at] = pt[i];
    filled += total;
  }
  if (threadIdx.x == 0) p.out_pos[uh] = (p.num_pages - 1) * BS + in_page;
}

}  // namespace b200attn

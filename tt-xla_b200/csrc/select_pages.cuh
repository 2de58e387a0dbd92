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
// added, each addition truncating at worst, and the factor covers that almost twice.  Below the
// normal range a product or an addition may lose all of itself, less than FLT_MIN each: 4 * head_size
// times that is added, which no score of an ordinary size notices.  Only pages
// whose fp32 score is within twice that of the border can be on the wrong side of it: these few
// are summed again in fp64, and the border is drawn among them.
//
// One launch: one CTA per (user, KV head) when these fill the machine, else several that each score
// a slice of the pages; the one that arrives last (a ticket in the workspace) makes the choice.
// Choosing is a chain of block-wide counts, so it is a bisection that starts at the highest bit in
// which the scores differ and ends as soon as the count is right.
// Measured: 64 of up to 512 pages for 32 users x 8 KV heads of 128 (67 MB of bounds) 29 us, of which
// scoring takes 20 (3.4 TB/s: 512-byte pieces, one round of CTAs) and choosing 9; 62 with a radix
// choice in global memory, 33 before the next group's bounds were loaded ahead.
#pragma once
#include <cfloat>

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
constexpr int kSelShared = 4096;     // pages whose scores stay in shared memory

struct SelectShared {
  float2 score[kSelShared];
  unsigned int part[2][kSelWarps];   // a block sum, double-buffered: one barrier each
  float warp_err[kSelWarps];
  unsigned int warp_lo[kSelWarps], warp_hi[kSelWarps];
  unsigned int near_list[32];
  unsigned long long near_key[32];
  unsigned int near_count;
  int last;
};

// Sum over the block, the same for all threads; `turn` alternates the buffer.
__device__ __forceinline__ unsigned int block_sum(SelectShared& sh, unsigned int v, unsigned int& turn) {
  v = __reduce_add_sync(0xffffffffu, v);
  unsigned int* part = sh.part[turn & 1];
  ++turn;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned int sum = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) sum += part[w];
  return sum;
}

// The k-th largest (k >= 1, at least k keys) of the keys get(i), i in [0, n) with use(i), by
// bisection from `top` (the highest bit the keys differ in; the bits above are `prefix`).  The
// barrier per step is what a step costs, so it ends as soon as exactly k keys are at least as large
// as the candidate: `border` is then such a candidate, not a key.
template <typename Key, typename Use, typename Get>
__device__ Key kth_border(SelectShared& sh, int n, unsigned int k, Key prefix, int top, Use use,
                          Get get, unsigned int& turn) {
  for (int bit = top; bit >= 0; --bit) {
    const Key cand = prefix | (static_cast<Key>(1) << bit);
    unsigned int c = 0;
    for (int i = threadIdx.x; i < n; i += kSelThreads) c += use(i) && get(i) >= cand;
    c = block_sum(sh, c, turn);
    if (c >= k) prefix = cand;
    if (c == k) break;
  }
  return prefix;
}

// Exclusive position of each set flag in thread order, and the number of flags (all threads call).
__device__ __forceinline__ unsigned int block_rank(SelectShared& sh, bool flag, unsigned int* total,
                                                   unsigned int& turn) {
  const unsigned int b = __ballot_sync(0xffffffffu, flag);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned int* part = sh.part[turn & 1];
  ++turn;
  if (lane == 0) part[warp] = __popc(b);
  __syncthreads();
  unsigned int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    const unsigned int c = part[w];
    before += w < warp ? c : 0u;
    all += c;
  }
  *total = all;
  return before + __popc(b & ((1u << lane) - 1u));
}

// fp64 score of one page, by a warp.
template <int HD>
__device__ double exact_page_score(const SelectPagesParams& p, int user, int kvh, int64_t blk,
                                   int lane) {
  const __nv_bfloat16* b = p.bounds + (blk * p.num_kv_heads + kvh) * 2 * HD;
  const __nv_bfloat16* q = p.q + static_cast<int64_t>(user) * p.q_row_stride +
                           static_cast<int64_t>(kvh) * p.group * HD;
  constexpr int kPer = HD / 32;            // channels per lane
  float lo[kPer], hi[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    lo[i] = __bfloat162float(b[i * 32 + lane]);
    hi[i] = __bfloat162float(b[HD + i * 32 + lane]);
  }
  double best = -INFINITY;
  for (int g0 = 0; g0 < p.group; g0 += 4) {
    float x[4][kPer];                      // four heads' loads in flight
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        x[g][i] = __bfloat162float(q[min(g0 + g, p.group - 1) * HD + i * 32 + lane]);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        // the products have 16 significant bits: exact in fp64, like the sums of such a range
        const double neg = x[g][i] > 0.f ? 0.0 : x[g][i];     // a NaN stays in both
        const double pos = x[g][i] < 0.f ? 0.0 : x[g][i];
        sum += neg * lo[i] + pos * hi[i];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (sum != sum) sum = INFINITY;
      best = sum > best ? sum : best;
    }
  }
  return best;
}

template <int HD, int BS, int NG>
__global__ void __launch_bounds__(kSelThreads, NG == 1 ? 2 : 1) select_pages_kernel(const SelectPagesParams p) {
  __shared__ SelectShared sh;
  const int kvh = blockIdx.y, user = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pos = p.cur_pos[user];
  const int64_t uh = static_cast<int64_t>(user) * p.num_kv_heads + kvh;
  int32_t* table = p.out_table + uh * p.num_pages;
  const int32_t* pt = p.page_table + static_cast<int64_t>(user) * p.page_table_stride;
  // a position behind the table is reported; the choice is then the one at the table's last key
  const bool behind = pos >= 0 && pos / BS >= p.max_pages;
  if (behind && blockIdx.x == 0 && threadIdx.x == 0) atomicExch(p.err_word, kDevBadIndex);
  const int n = pos < 0 ? 0 : behind ? p.max_pages : pos / BS + 1;
  const int in_page = pos < 0 ? 0 : behind ? BS - 1 : pos % BS;    // of the newest key

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
  // One CTA for all pages keeps the scores to itself; else they go through global memory.
  const bool shared_scores = n <= kSelShared;
  float2* score = p.score + uh * p.max_pages;
  float2* put = arrivals == 1 && shared_scores ? sh.score : score;
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
    // A slice's 16-page groups go to the warps in turn; then this CTA's next slice.  The bounds of
    // the next group are loaded half by half (minima, maxima) as the halves of this one are used,
    // and its page ids before that, so loads are always in flight.
    int slice = blockIdx.x, p0 = slice * p.slice + warp * 16;
    auto settle = [&]() {                 // the next group at or behind p0; false when there is none
      for (;;) {
        if (slice >= num_slices) return false;
        if (p0 < min(n, (slice + 1) * p.slice)) return true;
        slice += gridDim.x;
        p0 = slice * p.slice + warp * 16;
      }
    };
    struct Group {
      int row[2];                         // pages p0 + g, p0 + g + 8; -1: none
      int64_t blk[2];                     // -1: none, or out of range
    };
    auto find = [&](Group& gr) {
      const bool any = settle();
      const int end = any ? min(n, (slice + 1) * p.slice) : 0;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int at = p0 + g + 8 * r;
        gr.row[r] = any && at < end ? at : -1;
        gr.blk[r] = gr.row[r] >= 0 ? pt[at] : -1;
      }
      p0 += kSelWarps * 16;
      return any;
    };
    auto check = [&](Group& gr) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (gr.blk[r] < 0 || gr.blk[r] >= p.num_blocks) {
          if (gr.row[r] >= 0 && tq == 0) atomicExch(p.err_word, kDevBadIndex);
          gr.blk[r] = -1;
        }
      }
    };
    uint4 b[2][2][HD / 32];               // [min / max][row][32-channel step]
    auto load_half = [&](const Group& gr, int k) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint4* src = reinterpret_cast<const uint4*>(
                               p.bounds + ((gr.blk[r] < 0 ? 0 : gr.blk[r]) * p.num_kv_heads + kvh) * 2 * HD) +
                           k * (HD / 8) + tq;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j)
          b[k][r][j] = gr.blk[r] >= 0 ? __ldg(src + j * 4) : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    Group cur;
    bool more = find(cur);
    check(cur);
    load_half(cur, 0);
    load_half(cur, 1);
    while (more) {
      Group nxt;
      const bool next_more = find(nxt);
      float s[NG][4], a[NG][4];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[ng][i] = a[ng][i] = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const uint4 r0 = b[k][0][j], r1 = b[k][1][j];
          const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w};
          const uint32_t w1[4] = {r1.x, r1.y, r1.z, r1.w};
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
        if (next_more) {
          if (k == 0) check(nxt);
          load_half(nxt, k);
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
        if (tq == 0 && cur.row[r] >= 0)
          put[cur.row[r]] = cur.blk[r] >= 0
                                ? make_float2(best, mag * (4.f * HD / 8388608.f) + 4.f * HD * FLT_MIN)
                                            : make_float2(-INFINITY, 0.f);
      }
      cur = nxt;
      more = next_more;
    }
  }

  // ---------------------------------------------------------------- the last CTA chooses
  if (arrivals > 1) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0)
      sh.last = atomicAdd(p.tickets + uh, 1u) == static_cast<unsigned int>(arrivals - 1);
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    if (threadIdx.x == 0) p.tickets[uh] = 0u;    // leave the counter as the next launch expects it
    if (shared_scores)
      for (int i = threadIdx.x; i < n; i += kSelThreads) sh.score[i] = __ldcg(score + i);
  }
  const int e0 = p.keep_first, m = n - p.keep_last - p.keep_first;   // candidates e0 .. e0 + m - 1
  const unsigned int want = static_cast<unsigned int>(p.num_pages - p.keep_first - p.keep_last);
  unsigned long long* exact = p.exact + uh * p.max_pages;
  auto score_of = [&](int page) { return shared_scores ? sh.score[page] : __ldcg(score + page); };
  constexpr unsigned long long kPicked = ~0ull;
  unsigned int turn = 0;

  float border = INFINITY, width = 0.f;
  bool take_all_near = true;
  if (threadIdx.x == 0) sh.near_count = 0u;
  __syncthreads();
  if (want > 0) {
    float err = 0.f;
    unsigned int lo = ~0u, hi = 0u;
    for (int i = threadIdx.x; i < m; i += kSelThreads) {
      const float2 v = score_of(e0 + i);
      err = fmaxf(err, v.y);
      const uint32_t key = ordered_key(v.x);
      lo = min(lo, key);
      hi = max(hi, key);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) err = fmaxf(err, __shfl_xor_sync(0xffffffffu, err, o));
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      sh.warp_err[warp] = err;
      sh.warp_lo[warp] = lo;
      sh.warp_hi[warp] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
      err = fmaxf(err, sh.warp_err[w]);
      lo = min(lo, sh.warp_lo[w]);
      hi = max(hi, sh.warp_hi[w]);
    }
    // the keys share the bits above the highest one in which the least and the greatest differ
    const int top = lo == hi ? -1 : 31 - __clz(lo ^ hi);
    const uint32_t prefix = lo == hi ? lo : top == 31 ? 0u : lo & ~((2u << top) - 1u);
    const uint32_t at = kth_border<uint32_t>(
        sh, m, want, prefix, top, [](int) { return true; },
        [&](int i) { return ordered_key(score_of(e0 + i).x); }, turn);
    // the border score: the least of the keys that are >= `at`
    uint32_t least = ~0u;
    for (int i = threadIdx.x; i < m; i += kSelThreads) {
      const uint32_t key = ordered_key(score_of(e0 + i).x);
      if (key >= at) least = min(least, key);
    }
    least = __reduce_min_sync(0xffffffffu, least);
    __syncthreads();
    if (lane == 0) sh.warp_lo[warp] = least;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) least = min(least, sh.warp_lo[w]);
    border = __uint_as_float(least & 0x80000000u ? least & 0x7fffffffu : ~least);
    // both the page's and the border's score may be off by err; the difference is rounded once
    width = 2.f * err * 1.000001f;
    // above: surely among the `want` best; near: may be on either side
    auto is_near = [&](int i) {
      const float s = score_of(e0 + i).x;
      return s == border || fabsf(s - border) <= width;
    };
    unsigned int counts = 0, near_mine = 0;              // sure ones; near ones
    for (int i = threadIdx.x; i < m; i += kSelThreads) {
      const bool n_i = is_near(i);
      near_mine += n_i;
      counts += !n_i && score_of(e0 + i).x > border;
      if (n_i) {
        const unsigned int slot = atomicAdd(&sh.near_count, 1u);
        if (slot < 32u) sh.near_list[slot] = static_cast<unsigned int>(i);
      }
    }
    const unsigned int sure = block_sum(sh, counts, turn);
    const unsigned int near = block_sum(sh, near_mine, turn);
    const unsigned int open = want - sure;               // places for the near ones
    take_all_near = open == near;
    if (!take_all_near && near <= 32u) {
      // a handful: exact scores, and each one's rank among them
      for (unsigned int j = warp; j < near; j += kSelWarps) {
        const int i = static_cast<int>(sh.near_list[j]);
        const int64_t blk = pt[e0 + i];
        const bool ok = blk >= 0 && blk < p.num_blocks;
        const double v = ok ? exact_page_score<HD>(p, user, kvh, blk, lane) : -INFINITY;
        if (lane == 0) sh.near_key[j] = ordered_key(v);
      }
      __syncthreads();
      if (threadIdx.x < near) {
        const unsigned long long key = sh.near_key[threadIdx.x];
        const unsigned int mine = sh.near_list[threadIdx.x];
        unsigned int rank = 0;
        for (unsigned int j = 0; j < near; ++j)
          rank += sh.near_key[j] > key || (sh.near_key[j] == key && sh.near_list[j] < mine);
        exact[e0 + mine] = rank < open ? kPicked : 0ull;
      }
      __syncthreads();
    } else if (!take_all_near) {
      // many (equal pages): the same choice by bisection on the exact scores
      for (int i = warp; i < m; i += kSelWarps) {
        if (!is_near(i)) continue;                       // uniform in the warp
        const int64_t blk = pt[e0 + i];
        const bool ok = blk >= 0 && blk < p.num_blocks;
        const double v = ok ? exact_page_score<HD>(p, user, kvh, blk, lane) : -INFINITY;
        if (lane == 0) exact[e0 + i] = ordered_key(v);
      }
      __syncthreads();
      const unsigned long long edge = kth_border<unsigned long long>(
          sh, m, open, 0ull, 63, is_near, [&](int i) { return exact[e0 + i]; }, turn);
      unsigned int above = 0;
      for (int i = threadIdx.x; i < m; i += kSelThreads) above += is_near(i) && exact[e0 + i] > edge;
      above = block_sum(sh, above, turn);
      // mark the chosen ones: all above the edge, and of those on it the first `open - above`
      unsigned int before = 0;
      for (int i0 = 0; i0 < m; i0 += kSelThreads) {
        const int i = i0 + threadIdx.x;
        const bool here = i < m && is_near(i);
        const unsigned long long v = here ? exact[e0 + i] : 0ull;
        unsigned int total;
        const unsigned int rank = before + block_rank(sh, here && v == edge, &total, turn);
        before += total;
        if (here) exact[e0 + i] = v > edge || (v == edge && rank + above < open) ? kPicked : 0ull;
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
      const float s = score_of(i).x;
      const bool is_near = s == border || fabsf(s - border) <= width;
      take = is_near ? take_all_near || exact[i] == kPicked : s > border;
    }
    const int32_t id = i < n ? pt[i] : 0;
    unsigned int total;
    const unsigned int at = filled + block_rank(sh, take, &total, turn);
    if (take && at < static_cast<unsigned int>(p.num_pages)) table[at] = id;
    filled += total;
  }
  if (threadIdx.x == 0) p.out_pos[uh] = (p.num_pages - 1) * BS + in_page;
}

}  // namespace b200attn

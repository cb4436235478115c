// kvquant_decode_sm100.cu -- decode attention (query length 1) over the
// quantised paged KV cache (format: kvquant.cuh), and the selection of pages
// by a cheap score.
//
//   score_select_kernel             the top_k pages of every (sequence, KV head);
//   scores_kernel, select_kernel    the same in two steps for long tables
//   decode_kernel                   attention over all or the selected pages
//   combine_kernel                  LSE-weighted merge of what several warps shared
#include <type_traits>

#include "kvquant.cuh"
#include "b2a_host.h"

namespace b2a {
namespace kvq {

constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;
// Exponentials are of scores less their maximum less kDown: values next to the
// type's largest can be summed over 2^kDown tokens, or merged from as many warps,
// before their sum is divided by that of the exponentials.  What that costs lies
// below bf16's smallest normal number.
constexpr float kDown = 16.f, kUp = 65536.f;
constexpr uint64_t kDrainNs = 100000000ull;  // 0.1 s

// The length of sequence b as the block table can hold it.
__device__ __forceinline__ int table_len(const int32_t* kv_lens, int b, int page_size,
                                         int max_pages, bool flag) {
  const int len = kv_lens[b];
  const long long cap = (long long)max_pages * page_size;
  if (len < 0 || len > cap) {
    if (flag) atomicOr(&g_error_flags, 2u);
    return len < 0 ? 0 : (int)cap;
  }
  return len;
}

// ---------------------------------------------------------------- page scores
// An fp32 score as an unsigned key of the same order (-0 counts as +0).
__device__ __forceinline__ uint32_t order_key(float s) {
  const uint32_t u = __float_as_uint(s + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// score(page) = max over the group's heads of (dot * q_scale) * page_scale,
// dot = sum_d max(q8 * min8, q8 * max8): an upper bound of q.k over the page's
// keys, up to the roundings to 8 bits.  dot is a whole number below 2^24 and
// the two products are rounded one by one, so the scores are the same to the
// bit however the work is split.
//   8 lanes hold a page's bounds with 16 bytes each (8 at D = 64), and every
// lane the same channels of up to GP query heads in registers.  The GP sums over
// 8 lanes are reduced together, halving the heads a lane carries at each step.
constexpr int kScoreWarps = 8;
constexpr int kScorePages = 32 * kScoreWarps;  // pages per round of a CTA, 32 a warp
struct ScoreArgs {
  const void* q;
  long long q_b, q_h;  // element strides
  const int8_t* index;
  const float* index_scale;
  const int32_t* block_table;
  const int32_t* kv_lens;
  int G, Hkv, page_size, max_pages, num_pages;
};

// The keys of pages [first, last) of (b, hkv), by a CTA of kScoreWarps warps; page
// p's goes to keys[p].
template <int D, int GP, bool BF16>
__device__ __forceinline__ void score_pages(const ScoreArgs& a, int b, int hkv, int first,
                                            int last, uint32_t* keys) {
  using T1 = typename Elem<BF16>::T;
  constexpr int W = D / 32;  // words of 4 channels per lane
  __shared__ __align__(16) int s_q[2][GP][D / 4];  // max(q8, 0), min(q8, 0)
  __shared__ float s_scale[GP];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.G;
  // this warp's next 32 pages, one a lane
  auto lookup = [&](int p0) {
    int page = p0 + lane < last ? a.block_table[(size_t)b * a.max_pages + p0 + lane] : 0;
    if (page < 0 || page >= a.num_pages) {
      atomicOr(&g_error_flags, 2u);  // page number out of range: page 0's bounds instead
      page = 0;
    }
    return page;
  };
  int mine = lookup(first + warp * 32);
  const int sub = lane & 7;
  // NB page quadruples are in flight at a time, the first before the query is
  // rounded; a slot is loaded again as soon as it is used.
  constexpr int NB = GP == 8 && D == 128 ? 2 : 4;  // as many as registers hold
  int lo[NB][W], hi[NB][W];
  float ps[NB];
  auto load = [&](int k, int pages, int it) {  // quadruple `it` of a warp's 32 pages into slot k
    const int page = __shfl_sync(0xffffffffu, pages, 4 * it + (lane >> 3));
    const size_t row = (size_t)page * a.Hkv + hkv;
    ps[k] = a.index_scale[row];
    const int8_t* at = a.index + row * 2 * D;
    if constexpr (W == 4) {
      *reinterpret_cast<int4*>(lo[k]) = reinterpret_cast<const int4*>(at)[sub];
      *reinterpret_cast<int4*>(hi[k]) = reinterpret_cast<const int4*>(at + D)[sub];
    } else {
      *reinterpret_cast<int2*>(lo[k]) = reinterpret_cast<const int2*>(at)[sub];
      *reinterpret_cast<int2*>(hi[k]) = reinterpret_cast<const int2*>(at + D)[sub];
    }
  };
#pragma unroll
  for (int k = 0; k < NB; ++k) load(k, mine, k);
  if (warp < GP) {  // a warp a head; heads past the group's are zeros
    const int g = warp;
    float v[D / 32], top = 0.f;
    bool ok = true;
    const T1* qp =
        static_cast<const T1*>(a.q) + b * a.q_b + (long long)(hkv * G + min(g, G - 1)) * a.q_h;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      v[i] = (float)qp[lane + 32 * i];
      ok = ok && finite(v[i]);
      top = fmaxf(top, fabsf(v[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float scale = __all_sync(0xffffffffu, ok) ? scale127(top) : __int_as_float(0x7fc00000);
    const float inv = __frcp_rn(scale);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int c = g < G ? code127(v[i], scale, inv) : 0;
      reinterpret_cast<int8_t*>(s_q[0][g])[lane + 32 * i] = (int8_t)max(c, 0);
      reinterpret_cast<int8_t*>(s_q[1][g])[lane + 32 * i] = (int8_t)min(c, 0);
    }
    if (lane == 0) s_scale[g] = scale;
  }
  __syncthreads();
  int qp[GP][W], qn[GP][W];
#pragma unroll
  for (int g = 0; g < GP; ++g)
#pragma unroll
    for (int i = 0; i < W; ++i) {
      qp[g][i] = s_q[0][g][sub * W + i];
      qn[g][i] = s_q[1][g][sub * W + i];
    }
  // after the reduction lane `sub` holds head sub % GP (heads past G: -inf)
  const int head = sub & (GP - 1);
  const float qs = s_scale[head];
  const bool real = head < G;
  for (int p0 = first + warp * 32; p0 < last; p0 += kScorePages) {
    const int next = p0 + kScorePages < last ? lookup(p0 + kScorePages) : 0;
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int p = p0 + 4 * it + (lane >> 3), k = it % NB;
      int dot[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        dot[g] = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          dot[g] = __dp4a(hi[k][i], qp[g][i], dot[g]);
          dot[g] = __dp4a(lo[k][i], qn[g][i], dot[g]);
        }
      }
      const float page_scale = ps[k];
      if (it + NB < 8) load(k, mine, it + NB);
      else if (p0 + kScorePages < last) load(k, next, it + NB - 8);
      // lanes that differ in bit x keep the heads whose number agrees with theirs
#pragma unroll
      for (int x = 4, h = GP; x > 0; x >>= 1) {
        if (h > x) {  // h == 2 x: hand over half the heads
#pragma unroll
          for (int g = 0; g < GP / 2; ++g)
            if (g < h / 2) {
              const int keep = sub & x ? dot[g + h / 2] : dot[g];
              const int give = sub & x ? dot[g] : dot[g + h / 2];
              dot[g] = keep + __shfl_xor_sync(0xffffffffu, give, x);
            }
          h /= 2;
        } else {  // fewer heads than lanes: a plain sum
#pragma unroll
          for (int g = 0; g < GP; ++g)
            if (g < h) dot[g] += __shfl_xor_sync(0xffffffffu, dot[g], x);
        }
      }
      float best = real ? __fmul_rn(__fmul_rn((float)dot[0], qs), page_scale) : -INFINITY;
      if (isnan(best)) best = INFINITY;  // a page or query that is not finite is not hidden
#pragma unroll
      for (int x = 1; x < GP; x <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, x));
      if (sub == 0 && p < last) keys[p] = order_key(best);
    }
    mine = next;
  }
}

template <int D, int GP, bool BF16>
__global__ void __launch_bounds__(32 * kScoreWarps, 2)
    scores_kernel(const ScoreArgs a, uint32_t* __restrict__ keys, int top_k) {
  const int b = blockIdx.z, hkv = blockIdx.y;
  pdl_trigger();
  pdl_wait();
  const int len = table_len(a.kv_lens, b, a.page_size, a.max_pages,
                            blockIdx.x == 0 && hkv == 0 && threadIdx.x == 0);
  const int count = (int)(((long long)len + a.page_size - 1) / a.page_size);
  const int first = blockIdx.x * kScorePages;
  if (first >= count || count <= top_k) return;  // all pages are taken: no score needed
  score_pages<D, GP, BF16>(a, b, hkv, first, min(count, first + kScorePages),
                           keys + ((size_t)b * a.Hkv + hkv) * a.max_pages);
}

// The top_k pages, ties to the lowest page, in ascending order.  The last page
// counts as +infinity: it and the top_k - 1 best of the others, unless top_k of
// those are infinite themselves.  One CTA per (sequence, KV head); up to KPT
// keys a thread stay in registers, more are read again at each pass.  The
// smallest key that is taken is found 8 bits at a time below the bits that all
// keys share: a pass counts the keys that agree so far by their next 8 bits, in
// shared memory, and one warp finds the digit.  (One bit a pass, by compares and
// a block-wide sum: 32 us with the scores for 8192 pages.)
template <int THREADS, int KPT>
__device__ __forceinline__ void select_top(const uint32_t* kp, int all, int32_t* out, int top_k) {
  constexpr int NW = THREADS / 32;
  __shared__ int2 s_cnt[NW];
  __shared__ uint32_t s_at[KPT][NW];
  __shared__ __align__(16) int s_hist[256];
  __shared__ int4 s_digit;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (all <= top_k) {
    for (int i = threadIdx.x; i < top_k; i += THREADS) out[i] = i < all ? i : -1;
    return;
  }
  const int count = all - 1;  // without the last page
  int want = top_k - 1;
  const bool held = count <= KPT * THREADS;
  const int rounds = (count + THREADS - 1) / THREADS;
  uint32_t key[KPT];
  uint32_t top = 0, low = 0xffffffffu;
  auto each = [&](auto f) {  // every key of this thread
    if (held) {
#pragma unroll
      for (int c = 0; c < KPT; ++c) {
        if (c >= rounds) break;
        if (c * THREADS + (int)threadIdx.x < count) f(key[c]);
      }
    } else {
      for (int i = threadIdx.x; i < count; i += THREADS) f(kp[i]);
    }
  };
  if (held) {
#pragma unroll
    for (int c = 0; c < KPT; ++c) {
      const int i = c * THREADS + threadIdx.x;
      key[c] = i < count ? kp[i] : 0u;
    }
  }
  each([&](uint32_t k) {
    top = max(top, k);
    low = min(low, k);
  });
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  if (lane == 0) s_cnt[warp] = make_int2((int)top, (int)low);
  __syncthreads();
  {
    const int2 v = s_cnt[lane < NW ? lane : 0];
    top = __reduce_max_sync(0xffffffffu, (uint32_t)v.x);
    low = __reduce_min_sync(0xffffffffu, (uint32_t)v.y);
  }
  const uint32_t infinite = order_key(INFINITY);
  int inf_keys = 0;
  if (top >= infinite) {  // the same in every thread
    each([&](uint32_t k) { inf_keys += k >= infinite; });
    inf_keys = __reduce_add_sync(0xffffffffu, inf_keys);
    __syncthreads();
    if (lane == 0) s_cnt[warp].x = inf_keys;
    __syncthreads();
    inf_keys = __reduce_add_sync(0xffffffffu, lane < NW ? s_cnt[lane].x : 0);
  }
  if (inf_keys >= top_k) want = top_k;
  else if (threadIdx.x == 0) out[want] = count;
  if (want == 0) return;
  // t: the want-th largest key; ties: how many keys equal to it are taken
  int ties = want, hi = 32 - __clz(top ^ low);  // bits above hi are settled
  uint32_t t = hi == 32 ? 0u : top >> hi << hi;
  while (hi > 0) {
    const int bits = min(8, hi), lo = hi - bits;
    for (int i = threadIdx.x; i < 256; i += THREADS) s_hist[i] = 0;
    __syncthreads();
    each([&](uint32_t k) {
      if (((k ^ t) >> (hi - 1) >> 1) == 0) atomicAdd(&s_hist[(k >> lo) & ((1u << bits) - 1)], 1);
    });
    __syncthreads();
    if (warp == 0) {  // lane l: digits 8 l .. 8 l + 7; sums from the top
      int n[8], sum = 0;
#pragma unroll
      for (int d = 7; d >= 0; --d) n[d] = sum += s_hist[8 * lane + d];
      int above = sum;  // keys of this lane's digits and all higher lanes'
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int y = __shfl_down_sync(0xffffffffu, above, x);
        if (lane + x < 32) above += y;
      }
      above -= sum;  // of higher lanes alone
      if (above < ties && above + sum >= ties) {  // one lane
        int d = 7;
#pragma unroll
        for (int e = 7; e > 0; --e)
          if (above + n[e] < ties) d = e - 1;
        int over = above;  // keys with a higher digit
#pragma unroll
        for (int e = 1; e < 8; ++e)
          if (e == d + 1) over += n[e];
        int upto = 0;  // and with this one
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e == d) upto = above + n[e];
        s_digit = make_int4(8 * lane + d, over, upto, 0);
      }
    }
    __syncthreads();
    const int4 found = s_digit;
    t |= (uint32_t)found.x << lo;
    if (found.z == ties) {  // the digit's keys are all taken: no further digit matters
      --t;
      ties = 0;
      break;
    }
    ties -= found.y;
    hi = lo;
  }
  if (held) {
    // above (low 16 bits) and equal of each warp's 32 pages, in page order
#pragma unroll
    for (int c = 0; c < KPT; ++c) {
      if (c >= rounds) break;
      const bool in = c * THREADS + (int)threadIdx.x < count;
      const int gt = __popc(__ballot_sync(0xffffffffu, in && key[c] > t));
      const int eq = __popc(__ballot_sync(0xffffffffu, in && key[c] == t));
      if (lane == 0) s_at[c][warp] = gt | eq << 16;
    }
    __syncthreads();
    if (warp == 0) {  // their exclusive prefix sums
      uint32_t base = 0;
      uint32_t* at = &s_at[0][0];
      const int entries = rounds * NW;
      for (int k = 0; k < entries; k += 32) {
        const uint32_t v = k + lane < entries ? at[k + lane] : 0u;
        uint32_t inc = v;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, inc, x);
          if (lane >= x) inc += y;
        }
        if (k + lane < entries) at[k + lane] = base + inc - v;
        base += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < KPT; ++c) {
      if (c >= rounds) break;
      const int i = c * THREADS + threadIdx.x;
      const bool gt = i < count && key[c] > t, eq = i < count && key[c] == t;
      const unsigned below = (1u << lane) - 1;
      const int gt_at = __popc(__ballot_sync(0xffffffffu, gt) & below) + (s_at[c][warp] & 0xffffu);
      const int eq_at = __popc(__ballot_sync(0xffffffffu, eq) & below) + (s_at[c][warp] >> 16);
      if (gt || (eq && eq_at < ties)) out[gt_at + min(eq_at, ties)] = i;
    }
    return;
  }
  int base = 0, seen = 0;  // written, and equal keys met, so far
  for (int i0 = 0; i0 < count; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    const uint32_t k = i < count ? kp[i] : 0u;
    const bool eq = i < count && k == t, gt = i < count && k > t;
    const unsigned meq = __ballot_sync(0xffffffffu, eq), mgt = __ballot_sync(0xffffffffu, gt);
    const unsigned below = (1u << lane) - 1;
    __syncthreads();
    if (lane == 0) s_cnt[warp] = make_int2(__popc(mgt), __popc(meq));
    __syncthreads();
    int gt_at = __popc(mgt & below), eq_at = __popc(meq & below), gt_all = 0, eq_all = 0;
    for (int w = 0; w < NW; ++w) {
      const int2 v = s_cnt[w];
      if (w < warp) gt_at += v.x, eq_at += v.y;
      gt_all += v.x, eq_all += v.y;
    }
    if (gt || (eq && seen + eq_at < ties)) out[base + gt_at + min(eq_at, ties - seen)] = i;
    base += gt_all + min(eq_all, ties - seen);
    seen = min(seen + eq_all, ties);
  }
}

template <int THREADS, int KPT>
__global__ void __launch_bounds__(THREADS)
    select_kernel(const uint32_t* keys, const int32_t* kv_lens,
                  int32_t* __restrict__ pages, int Hkv, int page_size, int max_pages, int top_k) {
  const int hkv = blockIdx.x, b = blockIdx.y;
  pdl_trigger();
  pdl_wait();
  const int len = table_len(kv_lens, b, page_size, max_pages, false);
  const size_t tile = (size_t)b * Hkv + hkv;
  select_top<THREADS, KPT>(keys + tile * max_pages,
                           (int)(((long long)len + page_size - 1) / page_size),
                           pages + tile * top_k, top_k);
}

// Scores and selection of tables of up to kFusedPages pages in one CTA, the keys
// in shared memory: one launch, no trip through memory and the query rounded once.
// The table's width decides, which the host knows; the lengths lie on the device.
// Measured at D = 128, 4 heads a group, us in one CTA / in two steps:
//   pages     100        300         1000        2048        4096        8192
//   256 sets  7.1/16.3   10.2/19.7   17.9/26.5   35.8/46.8   64.7/85.4   -
//   64 sets   -          8.6/10.6    13.5/11.3   21.3/14.8   39.7/24.5   88.0/44.5
//   8 sets    -          8.4/8.6     12.7/8.6    20.4/9.7    36.9/11.6   67.5/13.7
// (a set is a (sequence, KV head); past 2048 with the bound moved).  One CTA a set
// fills the GPU where sets are many and is a long walk where they are few; 2048 caps
// what that walk costs at 11 us.
template <int D, int GP, bool BF16>
__global__ void __launch_bounds__(32 * kScoreWarps, 2)
    score_select_kernel(const ScoreArgs a, int32_t* __restrict__ pages, int top_k) {
  __shared__ uint32_t s_keys[kFusedPages];
  const int hkv = blockIdx.x, b = blockIdx.y;
  pdl_trigger();
  pdl_wait();
  const int len = table_len(a.kv_lens, b, a.page_size, a.max_pages, hkv == 0 && threadIdx.x == 0);
  const int count = (int)(((long long)len + a.page_size - 1) / a.page_size);
  if (count > top_k) {
    score_pages<D, GP, BF16>(a, b, hkv, 0, count, s_keys);
    __syncthreads();
  }
  select_top<32 * kScoreWarps, kFusedPages / (32 * kScoreWarps)>(
      s_keys, count, pages + ((size_t)b * a.Hkv + hkv) * top_k, top_k);
}

// ------------------------------------------------------------------- attention
// The work is a list of 64-token steps: all steps of KV head 0 of sequence 0,
// of its head 1, ..., of sequence 1, ...  Every warp takes an equal run of it,
// whatever the lengths, and works alone: it fills its own ring of stages with
// bulk copies (one a page: a block is contiguous), keeps its own online softmax
// and never waits for another warp.  A (sequence, KV head) that lies in one
// run is finished by its warp; the partials of one that is cut are merged by
// combine_kernel.
//
// Both products run on the tensor cores on the raw codes, and the (scale, min)
// pairs are applied outside them in fp32:
//   S[tok, h] = sum_g kscale[tok, g] (code . q)_g + kmin[tok, g] qsum[h, g]
//   O[h, d]   = sum_tok (p vscale[tok, g]) (code[tok, d] - mid)
//             + sum_tok p (vmin[tok, g] + mid vscale[tok, g])
// so K is used exactly and p*vscale is the only value rounded to 16 bits.  mid, 8
// or 128, centres the codes: the sums of the rounded p*vscale over a step come
// from a matrix instruction on ones, and their products with mid are taken off the
// accumulators step by step.  Without it O is a small difference of two large sums,
// which costs the accumulators' last bits and weighs each rounding of p*vscale with
// a code of 0..15 instead of -8..7.  It takes 5% of the time, and the error of fp16
// outputs over 16640 tokens falls from 8.3e-4 to 2.8e-4 (2.1e-4 is the rounding of
// the result alone).
//   Codes are not converted: a code c in the low mantissa bits of an fp16 with
// zero exponent IS the subnormal c * 2^-24, which the tensor cores multiply
// exactly, so unpacking is one mask a pair (and a shift every second one).  Codes
// masked where they lie are 4, 16 or 64 c * 2^-24; the factor is taken out of q
// (K), or of the finished channel (V, whose odd channels sum whole bytes 16 c' + c
// and lose the even neighbour's sum at the end: 4 us less below).  Where in the
// mantissa a code lies matters to K's sums, whose last bits go by their operands'
// exponents, a subnormal's being 2^-14: with K's codes at bits 2-5 and 6-9, not 0-3
// and 4-7, lse of fp16 caches is off by 0.6e-7 of its size instead of 4e-7 (fp32
// products: 0.4e-7), for another shift, 4 us below.  Both cache dtypes use fp16
// operands: each group of a query head is brought to [2^12, 2^13) by a power of two
// (over 64, a channel is off by 2^-25 of the group's largest at most; the groups'
// sums meet in fp32), and p*vscale by a running factor of its own for each head and
// group, which at the last change brought the step's largest product to [2^7, 2^8).
// That goes by the products, so a token whose values are large but that has no weight
// takes no bits from the others, and the factor grows as the maximum does, so what is
// left of early tokens takes none from later ones.  A product within 2^-21 of the
// largest keeps fp16's 11 bits, one below is off by 2^-32 of the largest at most; V's
// codes lie at bits 0-3, and a sum of 16 tokens is off by some 2^-14 of its largest
// product besides.
//   Products are bounded by their value steps as long as that will do, and looked at
// one by one where it will not (heavy tokens of small values beside large ones without
// weight: in every step, 12% of the time; elsewhere in the first).
//
// The token dimension is M of both products (A = K codes [tok, d], and A =
// V codes transposed [d, tok]) and the heads are N = 8, so no row of the
// matrix instructions is wasted for groups of 8 and P needs only an 8x8
// transpose (movmatrix) between them.  Contraction and output channels are
// dealt to lanes so that a lane's operand is a run of codes as they lie in
// memory.
//   HALF (groups of up to 4 heads): the four spare columns hold the same heads
// again; in S a lane takes the one or the other token row of its column, in O
// they take the second half of the tokens.  A lane then keeps one token row
// instead of two, and the scores, exponentials and products with the scales are
// done once each instead of half of them for columns that nobody reads.
//
// What bounds it: at 4 bits and D = 128 a 16-token slab of one KV head is 2304
// bytes and about 250 instructions, 84 of them the unpacking.  12 warps an SM fit
// (two 9 KB stages a warp fill shared memory, O and the operands the registers),
// three a scheduler, and those issue in half of the cycles: their own dependences and
// latencies are the limit, not HBM nor one unit (ALU 50%, tensor 28%).  64 ragged
// sequences of 8 KV heads, 1285 MB of blocks, take 240 us in short runs, 5.4 TB/s
// (6.45 TB/s is the measured copy), and 276 us in a long run, where the power limit
// takes the clock from 1.97 to about 1.7 GHz.  At 8 bits, with twice the bytes an
// instruction, 32 sequences of 16384 tokens, 1141 MB, take 189 us, 6.0 TB/s.  Warps
// alone on their scheduler take 2.4 us a step and three together 3.1 each.  32-token
// steps with 16 warps an SM were slower (257 us where 64-token ones took 221: what a
// step costs besides its tokens), so were K and V in separate halves of a stage (273
// us: several small copies a page where one does).
template <int D, int BITS>
struct DecCfg {
  static constexpr int kStep = 64;  // tokens per step
  static constexpr int kRow = row_bytes(D, BITS);
  static constexpr int kNG = D / kGroup;
  static constexpr int kStage = kStep * (2 * kRow + 2 * kNG * 4);
  // Two stages of 4.6 to 17 KB a warp: three CTAs of 76 or 71 KB fit an SM, four
  // of 39.
  static constexpr int kWarps = (D == 128 && BITS == 8) ? 2 : 4;
  static constexpr int kStages = 2;
  static constexpr int kCtas = (D == 64 && BITS == 4) ? 4 : 3;  // per SM
  static constexpr int kRing = kStages * kStage;
  static constexpr int kOffBar = kWarps * kRing;
  static constexpr int kOffValid = kOffBar + kWarps * kStages * 8;    // [warp][stage] int4
  static constexpr int kOffAbort = kOffValid + kWarps * kStages * 16;  // [warp] int
  static constexpr int kOffQuery = (kOffAbort + kWarps * 4 + 15) / 16 * 16;  // [warp][4][8] float
  static constexpr int kOffLag = kOffQuery + kWarps * 128;  // [thread] float2
  static constexpr int kSmem = kOffLag + kWarps * 256;
};

// D[16x8] += A[16x16] B[16x8], fp16 operands, fp32 accumulators
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// D[16x8] = A[16x16] B[16x8]
__device__ __forceinline__ void mma16816_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// The four 4-bit codes at bits 4j of each 16-bit half of x as pairs of fp16
// subnormals and small values: r[0], r[2] hold 4 c * 2^-24, r[1], r[3] 64 c * 2^-24.
__device__ __forceinline__ void unpack4(uint32_t x, uint32_t* r) {
  const uint32_t y = x << 2;
  r[0] = y & 0x003c003cu;
  r[1] = y & 0x03c003c0u;
  x >>= 6;
  r[2] = x & 0x003c003cu;
  r[3] = x & 0x03c003c0u;
}
// For V: r[0], r[2] hold c * 2^-24 and r[1], r[3] the whole byte, (16 c' + c) * 2^-24,
// two operations less; the finished channel of c' is freed of c's.
__device__ __forceinline__ void unpack4_bytes(uint32_t x, uint32_t* r) {
  r[0] = x & 0x000f000fu;
  r[1] = x & 0x00ff00ffu;
  r[3] = __byte_perm(x, 0, 0x4341);
  r[2] = r[3] & 0x000f000fu;
}
// two neighbours of an array as a pair, for the two-wide fp32 instructions
__device__ __forceinline__ float2& pair(float* x) { return *reinterpret_cast<float2*>(x); }
// the power of two in x > 0
__device__ __forceinline__ float pow2_of(float x) {
  return __uint_as_float(__float_as_uint(x) & 0x7f800000u);
}
// 2^e as fp32, e clamped to the normal range
__device__ __forceinline__ float pow2i(int e) {
  return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23);
}

// The steps of sequence b.
__device__ __forceinline__ int seq_steps(int len, int n_list, int page_shift) {
  if (len == 0) return 0;
  const long long tokens = n_list > 0 ? (long long)n_list << page_shift : len;
  return (int)((tokens + 63) >> 6);
}

template <int D, int BITS, bool BF16, bool HALF>
__global__ void __launch_bounds__(32 * DecCfg<D, BITS>::kWarps, DecCfg<D, BITS>::kCtas)
    decode_kernel(const void* q, long long q_b, long long q_h,
                  const uint8_t* data, const int32_t* block_table,
                  const int32_t* kv_lens, const int32_t* pages,
                  int n_list, float* __restrict__ o_part, float* __restrict__ l_part,
                  int* __restrict__ meta, void* __restrict__ out, float* __restrict__ lse, int B,
                  int G, int Hkv, int workers, int by_tile, int page_shift, int max_pages,
                  int num_pages, float scale_log2) {
  using C = DecCfg<D, BITS>;
  using T1 = typename Elem<BF16>::T;
  using T2 = typename Elem<BF16>::T2;
  constexpr int ROW = C::kRow, NG = C::kNG, S = C::kStages, STEP = C::kStep;
  constexpr int SL = STEP / 16;         // 16-token slabs per step
  constexpr int R = HALF ? 1 : 2;       // token rows of a slab per lane
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int worker = blockIdx.x * C::kWarps + warp;
  pdl_trigger();
  if (worker >= workers) return;
  pdl_wait();
  const int page_size = 1 << page_shift;
  const long long cap = (long long)max_pages << page_shift;
  auto length = [&](int b) {  // as the block table can hold it
    const int len = kv_lens[b];
    return len < 0 ? 0 : len > cap ? (int)cap : len;
  };
  auto steps_of = [&](int b) { return b < B ? seq_steps(length(b), n_list, page_shift) : 0; };
  if (worker == 0)
    for (int k = lane; k < B; k += 32)
      if (kv_lens[k] < 0 || kv_lens[k] > cap) atomicOr(&g_error_flags, 2u);

  // ------------------------------------------------------------ this warp's run
  // Every warp adds up all lengths and finds its place among them, with loads in
  // flight together: one chunk of 32 after the other, 2048 sequences took 18 us.
  long long total = 0;
  for (int b0 = 0; b0 < B; b0 += 256) {
    int s[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) s[u] = steps_of(b0 + 32 * u + lane);
#pragma unroll
    for (int u = 0; u < 8; ++u) total += s[u];
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
  total *= Hkv;
  const long long per = (total + workers - 1) / workers;
  const long long u0 = worker * per;
  const int n = (int)max(0ll, min(per, total - u0));  // steps
  // the answer of empty sequences, dealt over the warps
  for (int k = worker; k < B; k += workers)
    if (length(k) == 0) {
      for (int x = lane; x < Hkv * G * D; x += 32)
        static_cast<T1*>(out)[(size_t)k * Hkv * G * D + x] = Elem<BF16>::from(0.f);
      for (int x = lane; x < Hkv * G && lse != nullptr; x += 32)
        lse[(size_t)k * Hkv * G + x] = -INFINITY;
    }
  if (!by_tile && lane == 0) meta[2 * worker] = -1;
  if (n == 0) return;
  // its first (sequence, head, step)
  int b = 0, hkv = 0, i = 0, nst = 1;
  {
    long long base = 0;  // steps of a head of the sequences before the chunk
    bool found = false;
    for (int b0 = 0; !found; b0 += 128) {  // ends: u0 < total
      int s[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] = steps_of(b0 + 32 * u + lane);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const long long after = base + __reduce_add_sync(0xffffffffu, (unsigned)s[u]);
        if (!found && after * Hkv > u0) {
          found = true;
          int inc = s[u];
#pragma unroll
          for (int x = 1; x < 32; x <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, x);
            if (lane >= x) inc += y;
          }
          const int src = __ffs(__ballot_sync(0xffffffffu, (base + inc) * Hkv > u0)) - 1;
          nst = __shfl_sync(0xffffffffu, s[u], src);
          const long long rem = u0 - (base + __shfl_sync(0xffffffffu, inc, src) - nst) * Hkv;
          b = b0 + 32 * u + src;
          hkv = (int)(rem / nst);
          i = (int)(rem % nst);
        }
        base = after;
      }
      found = found || b0 >= B;  // only where the lengths change under the kernel
    }
    if (b >= B) return;
  }

  // ---------------------------------------------------------------- the ring
  const int np_shift = 6 - page_shift;  // log2 of the blocks per stage: 1, 2 or 4
  const uint32_t blk = (uint32_t)block_bytes(D, 1, BITS) << page_shift;
  uint8_t* ring = smem + warp * C::kRing;
  const uint32_t ring0 = smem_u32(ring), bar0 = smem_u32(smem + C::kOffBar) + warp * S * 8;
  int* s_valid = reinterpret_cast<int*>(smem + C::kOffValid) + warp * S * 4;  // tokens per slab
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffAbort) + warp;
  if (lane < S) mbar_init(bar0 + 8 * lane, 1u);
  if (lane == 0) *abort_flag = 0;
  fence_mbar_init();
  __syncwarp();

  // Page numbers are looked up 32 blocks at a time, one a lane, and one window
  // ahead, so that the dependent loads are off the loop's path.  (cb, ch) is the
  // (sequence, head) of the window's first step, cf its first step counted in
  // this run, cn its number of steps.
  int cb = b, ch = hkv, cf = -i, cn = nst;
  auto lookup = [&](int k, int& row, int& valid) {  // this run's block k
    row = 0;
    valid = 0;
    const int j = k >> np_shift;
    int lb = cb, lh = ch, lf = cf, ln = cn;
    if (j < n) {
      while (j - lf >= ln) {  // it ends: j < n lies in some sequence
        lf += ln;
        if (++lh == Hkv) {
          lh = 0;
          do ln = ++lb < B ? steps_of(lb) : n + 1;
          while (ln == 0);
        }
      }
      int lp = ((j - lf) << np_shift) + (k & ((1 << np_shift) - 1));
      if (lb >= B) lp = -1;  // only where the lengths change under the kernel
      else if (n_list > 0)
        lp = lp < n_list ? pages[((size_t)lb * Hkv + lh) * n_list + lp] : -1;
      if (lp >= 0 && lp < max_pages) {
        valid = min(max(length(lb) - (lp << page_shift), 0), page_size);
        if (valid > 0) {
          int page = block_table[(size_t)lb * max_pages + lp];
          if (page < 0 || page >= num_pages) {
            atomicOr(&g_error_flags, 2u);  // page number out of range: read page 0 instead
            page = 0;
          }
          row = page * Hkv + lh;
        }
      }
    }
    __syncwarp();
    // where the next window starts from (unused if the run ends before)
    cb = __shfl_sync(0xffffffffu, lb, 31);
    ch = __shfl_sync(0xffffffffu, lh, 31);
    cf = __shfl_sync(0xffffffffu, lf, 31);
    cn = __shfl_sync(0xffffffffu, ln, 31);
  };
  int row0, valid0, row1 = 0, valid1 = 0;
  lookup(lane, row0, valid0);
  if ((n << np_shift) > 32) lookup(32 + lane, row1, valid1);
  unsigned full = 0;  // bit st: every token of stage st is valid
  auto issue = [&](int j, int st) {  // copy step j's blocks into stage st, one a lane
    const int k = j << np_shift;
    if ((k & 31) == 0 && k > 0) {
      row0 = row1;
      valid0 = valid1;
      if ((n << np_shift) > k + 32) lookup(k + 32 + lane, row1, valid1);
    }
    const int row = __shfl_sync(0xffffffffu, row0, (k + lane) & 31);
    const int valid = __shfl_sync(0xffffffffu, valid0, (k + lane) & 31);
    const bool mine = (lane >> np_shift) == 0;
    const bool copy = mine && valid > 0;
    uint32_t bytes = C::kStage;
    if (__all_sync(0xffffffffu, !mine || valid == page_size)) {
      full |= 1u << st;
    } else {
      full &= ~(1u << st);
      bytes = __popc(__ballot_sync(0xffffffffu, copy)) * blk;
      // slab `lane` (< 4) lies in block lane / (page / 16)
      const int slab = __shfl_sync(0xffffffffu, valid0, (k + (lane >> (page_shift - 4))) & 31) -
                       16 * (lane & ((1 << (page_shift - 4)) - 1));
      if (lane < 4) s_valid[4 * st + lane] = min(max(slab, 0), 16);
    }
    const uint32_t bar = bar0 + 8 * st;
    if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
    __syncwarp();
    if (copy)
      bulk_load(ring0 + st * C::kStage + lane * blk, data + (size_t)(uint32_t)row * blk, blk, bar);
  };
  for (int j = 0; j < min(n, S); ++j) issue(j, j);

  // ------------------------------------------------------------------ queries
  // B fragments of S: lane (g, t) holds its head's channels 64*grp + 16 t +
  // 0..15 in the order in which a K row's codes unpack, over 4 or 64 as those are
  // 4 c or 64 c.  Column g is head g, in HALF head g & 3.
  const int half = t >> 1;                      // HALF: this lane's token row, g or g + 8
  const int head0 = HALF ? 2 * (t & 1) : 2 * t;  // its heads: head0, head0 + 1
  uint32_t qb[NG * 4][2];
  // Of columns 2t and 2t + 1, in shared memory: sums of the groups' channels, the
  // factor from the second group's units of S to the first's, and what a score in
  // these units is in log2.
  float* s_q = reinterpret_cast<float*>(smem + C::kOffQuery) + warp * 32;
  auto load_q = [&]() {
    const int hq = HALF ? g & 3 : g;
    const T1* qp = static_cast<const T1*>(q) + b * q_b + (long long)(hkv * G + hq) * q_h + 16 * t;
    float f[NG][16];
    int shift[NG];  // to [2^12, 2^13)
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      float top = 0.f;
      uint32_t u[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
      if (hq < G) {
        *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(qp + gr * 64);
        *reinterpret_cast<uint4*>(u + 4) = *reinterpret_cast<const uint4*>(qp + gr * 64 + 8);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 v = param<BF16>(u[j]);
        f[gr][2 * j] = v.x;
        f[gr][2 * j + 1] = v.y;
        top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      shift[gr] = min(139 - (int)(__float_as_uint(top) >> 23), 127);
    }
    float fac = 1.f;
    if constexpr (NG == 2) {  // units at most 2^30 apart: sums of both stay in fp32's range
      const int least = min(shift[0], shift[1]);
      shift[0] = min(shift[0], least + 30);
      shift[1] = min(shift[1], least + 30);
      fac = pow2i(shift[0] - shift[1]);
    }
    __syncwarp();  // every lane is done with the last head's
    float* mine = s_q + (g >> 1) * 8 + (g & 1);  // column g's, written by one of its lanes
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      const float mul = pow2i(shift[gr]);
      float sum = 0.f;  // of a column's channels
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        f[gr][j] *= mul;
        sum += f[gr][j];
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= pow2i(-24);  // the codes' factor
      if (t == 0) mine[2 * gr] = sum;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (BITS == 4) {
          const float* x = &f[gr][8 * (k / 2) + 2 * (k & 1)];
          qb[gr * 4 + k][0] = pack2_u32<false>(x[0] * 0.25f, x[4] * 0.25f);
          qb[gr * 4 + k][1] = pack2_u32<false>(x[1] * 0.015625f, x[5] * 0.015625f);
        } else {
          const float* x = &f[gr][4 * k];
          qb[gr * 4 + k][0] = pack2_u32<false>(x[0], x[1]);
          qb[gr * 4 + k][1] = pack2_u32<false>(x[2], x[3]);
        }
      }
    }
    const int e = 24 - max(shift[0], -126);  // up to 140: in two steps
    // not 0: a masked score is -inf, whose product with it stays -inf
    const float s2 = fmaxf(scale_log2 * pow2i(e / 2) * pow2i(e - e / 2), 1.401298464e-45f);
    if (t == 0) {
      if (NG == 2) mine[4] = fac;
      mine[6] = s2;
    }
    __syncwarp();
  };

  // --------------------------------------------------------------------- state
  alignas(16) float o[NG][4][4];  // [group][tile][(d even, column 2t), (even, 2t+1), (odd, 2t), (odd, 2t+1)]
  alignas(8) float omin[NG][2];  // sum of p * (vmin + mid * vscale) over this lane's tokens
  float m[2], l[2];  // the largest score, in the units of S, and the sum of p
  // p * vscale of a head's group is multiplied by vmul before it is rounded; o holds
  // sums of such products.  A power of two, for the product of a head's largest score is
  // then its step, which is not rounded (with any other factor the error of fp16 outputs
  // over 16000 tokens is 2.96e-4, so 2.75e-4); lag is what vmul is behind the growth of
  // the maximum, 1 to 2.  Steps are 0 or 2^-100 and more.
  alignas(8) float vmul[NG][2];
  float2* s_lag = reinterpret_cast<float2*>(smem + C::kOffLag) + threadIdx.x;
  constexpr float kMaxMul = 4.253529586511731e37f;  // 2^125
  constexpr float kMaxProduct = 32768.f;            // fp16 ends at 65504
  constexpr float kMaxStep = kMaxProduct * kUp;     // p is at most 1 / kUp
  auto reset = [&]() {
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
    *s_lag = make_float2(1.f, 1.f);
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      omin[gr][0] = omin[gr][1] = 0.f;
      vmul[gr][0] = vmul[gr][1] = 1.f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[gr][k][e] = 0.f;
    }
  };
  // Slab s of a stage: codes at (s >> 1) * code_hi + (s & 1) * code_lo, params
  // likewise; 16-token pages put each slab in a block of its own.
  const uint32_t code_lo = page_shift == 4 ? blk : 16 * ROW;
  const uint32_t code_hi = page_shift == 6 ? 32 * ROW : page_shift == 5 ? blk : 2 * blk;
  const uint32_t par_lo = page_shift == 4 ? blk : 16 * NG * 4;
  const uint32_t par_hi = page_shift == 6 ? 32 * NG * 4 : page_shift == 5 ? blk : 2 * blk;
  const uint32_t v_off = ROW << page_shift, vp_off = (NG * 4) << page_shift;
  // -mid as the accumulators hold codes: times 2^-24, odd channels at 4 bits as bytes
  constexpr float kMid = BITS == 4 ? 8.f : 128.f;
  constexpr float kMidEven = -kMid / 16777216.f, kMidOdd = BITS == 4 ? 17.f * kMidEven : kMidEven;
  constexpr uint32_t kOnes = 0x3c003c00u;
  const int tok = (g >> 1) + (g & 1) * 4;  // S row g is token `tok` of the slab, row g+8 8 later
  const int vtok = HALF ? tok + 8 * half : tok;  // the first token whose p this lane holds

  // The scores of a step; nvs: tokens of each slab.  FULL: all of them, known by the
  // caller, which leaves one run of straight code whose slabs overlap.
  alignas(16) float s[SL][R][2];
  uint32_t vpar[SL][R][NG];  // (scale, min) of V of this lane's rows
  auto scores = [&](auto all, const uint8_t* stage, const int4 nvs) {
    constexpr bool FULL = decltype(all)::value;
    const int nv[4] = {nvs.x, nvs.y, nvs.z, nvs.w};

    const float4 qa = *reinterpret_cast<const float4*>(s_q + 8 * t);
    const float2 qsum[2] = {make_float2(qa.x, qa.y), make_float2(qa.z, qa.w)};
    const float2 qfac = *reinterpret_cast<const float2*>(s_q + 8 * t + 4);

    // ---- S = K q^T
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) {
      if (!FULL && nv[sl] == 0) {  // the same in every lane
#pragma unroll
        for (int r = 0; r < R; ++r) {
          s[sl][r][0] = s[sl][r][1] = -INFINITY;
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) vpar[sl][r][gr] = 0u;
        }
        continue;
      }
      const uint8_t* kc = stage + (sl >> 1) * code_hi + (sl & 1) * code_lo + tok * ROW;
      const uint8_t* pp = stage + 2 * v_off + (sl >> 1) * par_hi + (sl & 1) * par_lo;
      uint32_t kpar[R][NG];  // of this lane's rows
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint8_t* kp = pp + (vtok + 8 * r) * NG * 4;
        if constexpr (NG == 2) {
          *reinterpret_cast<uint2*>(kpar[r]) = *reinterpret_cast<const uint2*>(kp);
          *reinterpret_cast<uint2*>(vpar[sl][r]) = *reinterpret_cast<const uint2*>(kp + vp_off);
        } else {
          kpar[r][0] = *reinterpret_cast<const uint32_t*>(kp);
          vpar[sl][r][0] = *reinterpret_cast<const uint32_t*>(kp + vp_off);
        }
      }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        alignas(8) float acc[4];  // (row g, column 2t), (g, 2t+1), (g+8, 2t), (g+8, 2t+1)
        if constexpr (BITS == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(kc + gr * 32 + t * 8);
          const uint2 y = *reinterpret_cast<const uint2*>(kc + 8 * ROW + gr * 32 + t * 8);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t a[4], z[4];
            unpack4(w ? x.y : x.x, a);
            unpack4(w ? y.y : y.x, z);
            if (w == 0) mma16816_first(acc, a[0], z[0], a[1], z[1], qb[gr * 4][0], qb[gr * 4][1]);
            else mma16816(acc, a[0], z[0], a[1], z[1], qb[gr * 4 + 2][0], qb[gr * 4 + 2][1]);
            mma16816(acc, a[2], z[2], a[3], z[3], qb[gr * 4 + 2 * w + 1][0],
                     qb[gr * 4 + 2 * w + 1][1]);
          }
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(kc + gr * 64 + t * 16);
          const uint4 y = *reinterpret_cast<const uint4*>(kc + 8 * ROW + gr * 64 + t * 16);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = __byte_perm(xs[w], 0, 0x4140), a1 = __byte_perm(ys[w], 0, 0x4140);
            const uint32_t a2 = __byte_perm(xs[w], 0, 0x4342), a3 = __byte_perm(ys[w], 0, 0x4342);
            if (w == 0) mma16816_first(acc, a0, a1, a2, a3, qb[gr * 4][0], qb[gr * 4][1]);
            else mma16816(acc, a0, a1, a2, a3, qb[gr * 4 + w][0], qb[gr * 4 + w][1]);
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float2 pr = param<BF16>(kpar[r][gr]);
          const float2 a = HALF ? (half ? pair(acc + 2) : pair(acc)) : pair(acc + 2 * r);
          const float2 x = ffma2(make_float2(pr.x, pr.x), a,
                                 fmul2(make_float2(pr.y, pr.y), qsum[gr]));
          pair(s[sl][r]) = gr == 0 ? x : ffma2(x, qfac, pair(s[sl][r]));
        }
      }
      // tokens past the end: whatever their slots hold is dropped here
      if (!FULL && nv[sl] < 16) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (vtok + 8 * r >= nv[sl]) {
            s[sl][r][0] = s[sl][r][1] = -INFINITY;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) vpar[sl][r][gr] = 0u;
          }
      }
    }
  };
  // One step.  What follows the scores is there once, for partial steps too, whose
  // tokens past the end weigh nothing: twice the code costs sequences of a few steps
  // more in instruction fetches (2048 of 100 to 200 tokens: 201 us, so 181).
  auto step = [&](const uint8_t* stage, bool whole, const int4 nvs) {
    if (whole) scores(std::true_type{}, stage, nvs);
    else scores(std::false_type{}, stage, nvs);
    const float2 sl2 = *reinterpret_cast<const float2*>(s_q + 8 * t + 6);

    // ---- online softmax, per head over the step's tokens
    float alpha[2], nmu[2];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = s[0][0][h];
#pragma unroll
      for (int k = 1; k < SL * R; ++k) mx = fmaxf(mx, s[k / R][k % R][h]);
#pragma unroll
      for (int x = HALF ? 2 : 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[h], mx);
      const float mu = mn == -INFINITY ? 0.f : mn;
      alpha[h] = ex2_mufu((m[h] - mu) * (h ? sl2.y : sl2.x));
      moved = moved || mn != m[h];
      m[h] = mn;
      nmu[h] = -mu;
    }
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < SL * R; ++k) {
      float2& x = pair(s[k / R][k % R]);
      // The difference first: the largest score's is 0 whatever its size.  (s * sl2 - m in
      // one instruction leaves what a maximum in log2 units lost in rounding: past 2^31 p
      // of all tokens is 0 or infinite.)
      x = ffma2(fadd2(x, make_float2(nmu[0], nmu[1])), sl2, make_float2(-kDown, -kDown));
      x.x = ex2_mufu(x.x);
      x.y = ex2_mufu(x.y);
      sum = fadd2(sum, x);
    }
    l[0] = fmaf(l[0], alpha[0], sum.x);
    l[1] = fmaf(l[1], alpha[1], sum.y);
    // Where a maximum rises, vmul grows by what p of the tokens so far shrink by, and o
    // takes what of that is no power of two.  Products are bounded by their steps alone
    // as long as that will do.
    float vbig[NG];  // largest value step of this lane's tokens
    bool look = moved;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      T2 big = *reinterpret_cast<T2*>(&vpar[0][0][gr]);
#pragma unroll
      for (int k = 1; k < SL * R; ++k)
        big = __hmax2(big, *reinterpret_cast<T2*>(&vpar[k / R][k % R][gr]));
      vbig[gr] = Elem<BF16>::unpack(big).x;
      look = look || vbig[gr] * fmaxf(vmul[gr][0], vmul[gr][1]) >= kMaxStep;
    }
    if (__any_sync(0xffffffffu, look)) {
      bool over = false;
      const float2 lag2 = *s_lag;
      float lag[2] = {lag2.x, lag2.y};
      float was[NG][2];
      alignas(8) float f[NG][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float grow = lag[h] * __fdividef(1.f, alpha[h]);  // infinite at a head's first token
        const float up = pow2_of(grow);
        lag[h] = __uint_as_float((__float_as_uint(grow) & 0x7fffffu) | 0x3f800000u);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          omin[gr][h] *= alpha[h];
          f[gr][h] = alpha[h] * up;
          was[gr][h] = vmul[gr][h];
          vmul[gr][h] *= up;
          over = over || vmul[gr][h] > kMaxMul || vbig[gr] * vmul[gr][h] >= kMaxStep;
        }
      }
      *s_lag = make_float2(lag[0], lag[1]);
      if (__any_sync(0xffffffffu, over)) {
        // The products themselves (bf16 has their range and bits enough): where one is
        // too large for vmul, the step's largest goes to [2^7, 2^8).
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          uint32_t top2 = 0u;  // of both heads, in bf16
          auto larger = [&](uint32_t w) {
            const __nv_bfloat162 y = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&top2),
                                             *reinterpret_cast<__nv_bfloat162*>(&w));
            top2 = *reinterpret_cast<const uint32_t*>(&y);
          };
#pragma unroll
          for (int k = 0; k < SL * R; ++k) {
            const float vs = param<BF16>(vpar[k / R][k % R][gr]).x;
            larger(pack2_u32<true>(s[k / R][k % R][0] * vs, s[k / R][k % R][1] * vs));
          }
#pragma unroll
          for (int x = HALF ? 2 : 4; x < 32; x <<= 1) larger(__shfl_xor_sync(0xffffffffu, top2, x));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float top = __uint_as_float(h ? top2 & 0xffff0000u : top2 << 16);
            if (!(vmul[gr][h] <= kMaxMul && top * vmul[gr][h] < kMaxProduct)) {
              const int fit = max(min(261 - (int)(__float_as_uint(top) >> 23), 252), 1);  // biased
              f[gr][h] = alpha[h] * pow2i(fit - (int)(__float_as_uint(was[gr][h]) >> 23));
              vmul[gr][h] = __uint_as_float((uint32_t)fit << 23);
            }
          }
        }
      }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          for (int e = 0; e < 4; e += 2)
            pair(&o[gr][k][e]) = fmul2(pair(&o[gr][k][e]), pair(f[gr]));
    }

    // ---- O += V^T P
    alignas(16) float psum[NG][4];  // sums of the rounded p * vscale over the step
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) psum[gr][0] = psum[gr][1] = psum[gr][2] = psum[gr][3] = 0.f;
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) {
      const uint8_t* vc =
          stage + v_off + (sl >> 1) * code_hi + (sl & 1) * code_lo + g * BITS + t * ROW;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        uint32_t pb[2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float2 pr = param<BF16>(vpar[sl][r][gr]);
          const float vmid = fmaf(pr.x, kMid, pr.y);
          omin[gr][0] = fmaf(s[sl][r][0], vmid, omin[gr][0]);
          omin[gr][1] = fmaf(s[sl][r][1], vmid, omin[gr][1]);
          // vmul last: vscale * vmul may pass fp32 where p is next to nothing
          const float2 w = fmul2(make_float2(s[sl][r][0] * pr.x, s[sl][r][1] * pr.x), pair(vmul[gr]));
          pb[r] = movmatrix_trans(pack2_u32<false>(w.x, w.y));
        }
        if constexpr (HALF) {  // columns 0-3: tokens 0-7 of the slab, columns 4-7: tokens 8-15
          pb[1] = g >= 4 ? pb[0] : 0u;
          pb[0] = g >= 4 ? 0u : pb[0];
        }
        mma16816(psum[gr], kOnes, kOnes, kOnes, kOnes, pb[0], pb[1]);
        if constexpr (BITS == 4) {
          const uint32_t wa = *reinterpret_cast<const uint32_t*>(vc + gr * 32);
          const uint32_t wb = *reinterpret_cast<const uint32_t*>(vc + gr * 32 + 4 * ROW);
          const uint32_t wc = *reinterpret_cast<const uint32_t*>(vc + gr * 32 + 8 * ROW);
          const uint32_t wd = *reinterpret_cast<const uint32_t*>(vc + gr * 32 + 12 * ROW);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // channels 8g + 4*hf + 0..3
            uint32_t a[4], z[4];
            unpack4_bytes(__byte_perm(wa, wb, hf ? 0x7632 : 0x5410), a);
            unpack4_bytes(__byte_perm(wc, wd, hf ? 0x7632 : 0x5410), z);
            mma16816(o[gr][2 * hf], a[0], a[1], z[0], z[1], pb[0], pb[1]);
            mma16816(o[gr][2 * hf + 1], a[2], a[3], z[2], z[3], pb[0], pb[1]);
          }
        } else {
          const uint2 wa = *reinterpret_cast<const uint2*>(vc + gr * 64);
          const uint2 wb = *reinterpret_cast<const uint2*>(vc + gr * 64 + 4 * ROW);
          const uint2 wc = *reinterpret_cast<const uint2*>(vc + gr * 64 + 8 * ROW);
          const uint2 wd = *reinterpret_cast<const uint2*>(vc + gr * 64 + 12 * ROW);
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // channels 8g + 2k, 2k+1
            const uint32_t xa = k < 2 ? wa.x : wa.y, xb = k < 2 ? wb.x : wb.y;
            const uint32_t xc = k < 2 ? wc.x : wc.y, xd = k < 2 ? wd.x : wd.y;
            const uint32_t s0 = k & 1 ? 0x6622 : 0x4400, s1 = k & 1 ? 0x7733 : 0x5511;
            mma16816(o[gr][k], __byte_perm(xa, xb, s0) & 0x00ff00ffu,
                     __byte_perm(xa, xb, s1) & 0x00ff00ffu, __byte_perm(xc, xd, s0) & 0x00ff00ffu,
                     __byte_perm(xc, xd, s1) & 0x00ff00ffu, pb[0], pb[1]);
          }
        }
      }
    }
#pragma unroll
    for (int gr = 0; gr < NG; ++gr)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        for (int e = 0; e < 4; e += 2)
          pair(&o[gr][k][e]) = ffma2(pair(psum[gr]), e ? make_float2(kMidOdd, kMidOdd)
                                                       : make_float2(kMidEven, kMidEven),
                                     pair(&o[gr][k][e]));
  };

  // Write out what was gathered for (b, hkv): the answer where this warp had all
  // of it, else a partial (o normalised, natural log l).
  auto flush = [&](bool first, bool last, int next) {  // next: the step after, in this run
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int x = HALF ? 2 : 4; x < 32; x <<= 1) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
          omin[gr][h] += __shfl_xor_sync(0xffffffffu, omin[gr][h], x);
      }
    }
    constexpr float kEven = 16777216.f;  // 2^24: the codes' factor
    constexpr float kOdd = BITS == 4 ? 1048576.f : kEven;  // odd channels were 16 c
    const bool whole = first && last;
    const int tile = b * Hkv + hkv;
    const size_t seg = (size_t)worker + tile;  // either grows along the list: no two alike
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int head = head0 + h;
      const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
      const float ll = l[h] == 0.f ? -INFINITY : m[h] * s_q[8 * t + 6 + h] * kLn2 + logf(l[h] * kUp);
      const size_t orow = whole ? (size_t)b * Hkv * G + hkv * G + head : seg * G + head;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        const float unit = __fdividef(1.f, vmul[gr][h]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x = o[gr][k][h], y = o[gr][k][2 + h];
          if constexpr (HALF) {  // the other tokens' half
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            y += __shfl_xor_sync(0xffffffffu, y, 2);
          }
          if constexpr (BITS == 4) y -= x;  // bytes 16 c' + c: what is left is 16 c'
          x = fmaf(x * kEven, unit, omin[gr][h]) * inv;
          y = fmaf(y * kOdd, unit, omin[gr][h]) * inv;
          const size_t at = orow * D + gr * 64 + 8 * g + 2 * k;
          if (head < G && (!HALF || (k >> 1) == half)) {
            if (whole) *reinterpret_cast<uint32_t*>(static_cast<T1*>(out) + at) = pack2_u32<BF16>(x, y);
            else *reinterpret_cast<float2*>(o_part + at) = make_float2(x, y);
          }
        }
      }
      if (g == 0 && head < G && (!HALF || half == 0)) {
        if (!whole) l_part[orow] = ll;
        else if (lse != nullptr) lse[orow] = ll;
      }
    }
    if (lane == 0) {  // which workers hold partials of this (sequence, KV head)
      if (by_tile) {
        if (first) meta[2 * tile] = whole ? -1 : worker;
        if (last) meta[2 * tile + 1] = worker;
      } else if (!whole) {
        if (first) meta[2 * worker] = tile;
        if (last) meta[2 * ((u0 + next - nst) / per) + 1] = worker;  // at the worker it began in
      }
    }
  };

  // ---------------------------------------------------------------------- loop
  load_q();
  reset();
  int i0 = i;  // the step at which this warp entered (b, hkv)
  bool ok = true;
  int st = 0;
  uint32_t phase = 0;
  for (int j = 0; j < n; ++j) {
    // one answer for the warp: a copy that lands between two lanes' last looks must
    // not leave it divided before its shuffles
    ok = __all_sync(0xffffffffu, ok && mbar_wait(bar0 + 8 * st, phase, abort_flag));
    if (ok) {
      const uint8_t* stage = ring + st * C::kStage;
      const bool whole = full >> st & 1u;
      const int4 v = *reinterpret_cast<const int4*>(s_valid + 4 * st);
      step(stage, whole, v);
      __syncwarp();  // every lane has read the stage
      if (j + S < n) issue(j + S, st);
      if (++st == S) {
        st = 0;
        phase ^= 1u;
      }
    }
    if (++i == nst || j == n - 1) {
      flush(i0 == 0, i == nst, j + 1);
      if (j < n - 1) {  // the next (sequence, KV head) with a step
        i = i0 = 0;
        if (++hkv == Hkv) {
          hkv = 0;
          do nst = ++b < B ? steps_of(b) : 1;
          while (nst == 0);
          if (b >= B) break;  // only where the lengths change under the kernel
        }
        load_q();
        reset();
      }
    }
  }
  if (!ok) {
    // A copy never arrived.  Give the ones still in flight a bounded time to
    // land before this block's shared memory goes to another.
    for (int k = 0; k < S; ++k) {
      volatile int never = 0;
      mbar_wait_limit(bar0 + 8 * k, 0, &never, kDrainNs);
      mbar_wait_limit(bar0 + 8 * k, 1, &never, kDrainNs);
    }
  }
}

// One CTA of NW warps per query head of a (sequence, KV head) that was cut: the
// CTAs go by (sequence, KV head), or, where those are many, by the worker in whose
// run a cut one began, which are no more than the workers (1024 sequences of 512
// tokens, 8 KV heads: 170 us by (sequence, KV head), 151 by worker).  A partial
// whose l is -inf has no token; a NaN goes through to O and L.  Rows are read as 16
// bytes a lane, eight in flight a warp, the first eight before their weights are
// known: two loads' latencies in a row, and not one per partial.
constexpr int kChunk = 512;  // weights held at a time
template <int D, int NW, bool BF16>
__global__ void __launch_bounds__(32 * NW)
    combine_kernel(const float* o_part, const float* l_part,
                   const int* meta, const int32_t* kv_lens,
                   void* __restrict__ out, float* __restrict__ lse, int G, int Hkv, int by_tile) {
  using T1 = typename Elem<BF16>::T;
  constexpr int LPR = D / 4, RPW = 32 / LPR;  // lanes per row, rows per warp
  constexpr int STEP = NW * RPW;              // rows per round of the CTA
  __shared__ float s_w[kChunk], s_red[2][NW];
  __shared__ float4 s_acc[STEP][LPR];
  const int at = blockIdx.x / G, h = blockIdx.x % G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  const int2 m = reinterpret_cast<const int2*>(meta)[at];
  if (by_tile && kv_lens[at / Hkv] <= 0) return;  // no steps: meta was not written
  if (m.x < 0) return;  // one warp had all of it, or none was cut
  const int tile = by_tile ? at : m.x, first = by_tile ? m.x : at;
  const int S = m.y - first + 1;
  const size_t row = (size_t)tile * G + h, seg0 = (size_t)first + tile;
  const float* lp = l_part + seg0 * G + h;  // partial s at s * G
  const float4* op = reinterpret_cast<const float4*>(o_part + (seg0 * G + h) * D);
  const int sub = warp * RPW + lane / LPR, c = lane % LPR;
  float4 v[8];
  auto load = [&](int s0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = s0 + k * STEP;
      v[k] = s < S ? op[(size_t)s * G * LPR + c] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  load(sub);
  float M = -INFINITY;
  for (int s = threadIdx.x; s < S; s += 32 * NW) M = fmaxf(M, lp[(size_t)s * G]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  if (lane == 0) s_red[0][warp] = M;
  __syncthreads();
  M = s_red[0][0];
#pragma unroll
  for (int w = 1; w < NW; ++w) M = fmaxf(M, s_red[0][w]);
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  static_assert(kChunk % (8 * STEP) == 0, "a batch of rows lies in one chunk");
  for (int c0 = 0; c0 < S; c0 += kChunk) {
    const int cn = min(kChunk, S - c0);
    if (c0 > 0) __syncthreads();  // the previous chunk's weights are used
    for (int s = threadIdx.x; s < cn; s += 32 * NW) {
      const float x = lp[(size_t)(c0 + s) * G];
      const float w = x == -INFINITY ? 0.f : expf(x - M) * (1.f / kUp);
      s_w[s] = w;
      L += w;
    }
    __syncthreads();
    for (int s0 = sub; s0 < cn; s0 += 8 * STEP) {
      if (c0 + s0 != sub) load(c0 + s0);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int s = s0 + k * STEP;
        const float w = s < cn ? s_w[s] : 0.f;
        acc.x = fmaf(w, v[k].x, acc.x);
        acc.y = fmaf(w, v[k].y, acc.y);
        acc.z = fmaf(w, v[k].z, acc.z);
        acc.w = fmaf(w, v[k].w, acc.w);
      }
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
  if (lane == 0) s_red[1][warp] = L;
  s_acc[sub][c] = acc;
  __syncthreads();
  L = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) L += s_red[1][w];
  if (threadIdx.x < D) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < STEP; ++k) a += reinterpret_cast<const float*>(s_acc[k])[threadIdx.x];
    static_cast<T1*>(out)[row * D + threadIdx.x] = Elem<BF16>::from(L == 0.f ? 0.f : a / L);
  }
  if (threadIdx.x == 0 && lse != nullptr) lse[row] = L == 0.f ? -INFINITY : M + logf(L * kUp);
}

}  // namespace kvq

B2A_DEFINE_ERROR_READER(kvquant_decode)

int kvq_select_dispatch(const void* q, int64_t q_b, int64_t q_h, const int8_t* index,
                        const float* index_scale, const int32_t* block_table,
                        const int32_t* kv_lens, uint32_t* keys, int32_t* pages, int B, int H,
                        int Hkv, int D, int page_size, int max_pages, int num_pages, int top_k,
                        int dtype, cudaStream_t stream) {
  using namespace kvq;
  const int G = H / Hkv;
  const ScoreArgs a{q,       q_b, q_h, index,     index_scale, block_table,
                    kv_lens, G,   Hkv, page_size, max_pages,   num_pages};
  const bool bf = dtype == B2A_BF16;
  const dim3 tiles((unsigned)Hkv, (unsigned)B);
  cudaError_t e;
#define B2A_KVQ_SCORES(KERNEL, GO)                                                      \
  if (D == 64 && G <= 4) e = bf ? GO((KERNEL<64, 4, true>)) : GO((KERNEL<64, 4, false>)); \
  else if (D == 64) e = bf ? GO((KERNEL<64, 8, true>)) : GO((KERNEL<64, 8, false>));      \
  else if (G <= 4) e = bf ? GO((KERNEL<128, 4, true>)) : GO((KERNEL<128, 4, false>));     \
  else e = bf ? GO((KERNEL<128, 8, true>)) : GO((KERNEL<128, 8, false>));
  if (max_pages <= kFusedPages) {
    auto go = [&](auto kern) {
      return launch_pdl(kern, tiles, 32 * kScoreWarps, 0, stream, a, pages, top_k);
    };
    B2A_KVQ_SCORES(score_select_kernel, go)
    if (e != cudaSuccess) return set_cuda_error(e, "page selection kernel launch");
    return B2A_OK;
  }
  const dim3 grid((unsigned)((max_pages + kScorePages - 1) / kScorePages), (unsigned)Hkv,
                  (unsigned)B);
  auto go = [&](auto kern) {
    return launch_pdl(kern, grid, 32 * kScoreWarps, 0, stream, a, keys, top_k);
  };
  B2A_KVQ_SCORES(scores_kernel, go)
#undef B2A_KVQ_SCORES
  if (e != cudaSuccess) return set_cuda_error(e, "page score kernel launch");
  e = launch_pdl(select_kernel<1024, 16>, tiles, 1024, 0, stream, keys, kv_lens, pages, Hkv,
                 page_size, max_pages, top_k);
  if (e != cudaSuccess) return set_cuda_error(e, "page selection kernel launch");
  return B2A_OK;
}

int64_t kvq_select_keys_words(int B, int Hkv, int max_pages) {
  return max_pages <= kvq::kFusedPages ? 0 : (int64_t)B * Hkv * max_pages;
}

// Warps that the GPU (148 SMs) runs at a time; no more than there can be steps.
template <int D, int BITS>
constexpr long long resident_warps() {
  return 148ll * kvq::DecCfg<D, BITS>::kCtas * kvq::DecCfg<D, BITS>::kWarps;
}
int kvq_decode_workers(int B, int Hkv, int D, int bits, long long max_tokens) {
  const long long resident = D == 64 ? (bits == 4 ? resident_warps<64, 4>() : resident_warps<64, 8>())
                                     : (bits == 4 ? resident_warps<128, 4>() : resident_warps<128, 8>());
  const long long steps = (long long)B * Hkv * ((max_tokens + 63) / 64);
  return (int)(steps < resident ? steps : resident);
}

// Partials: a worker's share of a (sequence, KV head) has number worker + tile.
// [worker + tile][G][D] o, [worker + tile][G] l, then pairs of ints: per tile its
// first and last worker, or per worker the tile that began in it and was cut and
// that tile's last worker.
int64_t kvq_decode_workspace_floats(int B, int H, int Hkv, int D, int workers) {
  const int64_t tiles = (int64_t)B * Hkv;
  return (workers + tiles) * (H / Hkv) * (D + 1) + 2 * (workers > tiles ? workers : tiles) + 1;
}

template <int D, int BITS, bool BF16, bool HALF>
static int launch_kvq_decode(const void* q, int64_t q_b, int64_t q_h, const uint8_t* data,
                             const int32_t* block_table, const int32_t* kv_lens,
                             const int32_t* pages, int n_list, float* ws, void* o, float* lse,
                             int B, int G, int Hkv, int workers, int page_shift, int max_pages,
                             int num_pages, float scale, cudaStream_t stream) {
  using namespace kvq;
  using C = DecCfg<D, BITS>;
  auto kern = decode_kernel<D, BITS, BF16, HALF>;
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return set_error(B2A_ERR_CUDA, "cudaGetDevice failed");
  if (!attr_done[dev]) {
    cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return set_cuda_error(e, "cudaFuncSetAttribute(quantised decode)");
    attr_done[dev] = true;
  }
  const int64_t segs = (int64_t)workers + (int64_t)B * Hkv;
  float* l_part = ws + segs * G * D;
  int* meta = reinterpret_cast<int*>(l_part + (segs * G + 1) / 2 * 2);  // pairs of ints
  const int64_t tiles = (int64_t)B * Hkv;
  const int by_tile = tiles <= workers;
  cudaError_t e = launch_pdl(kern, dim3((workers + C::kWarps - 1) / C::kWarps), 32 * C::kWarps,
                             C::kSmem, stream, q, q_b, q_h, data, block_table, kv_lens, pages,
                             n_list, ws, l_part, meta, o, lse, B, G, Hkv, workers, by_tile,
                             page_shift, max_pages, num_pages, scale * kLog2e);
  if (e != cudaSuccess) return set_cuda_error(e, "quantised decode kernel launch");
  // Few (sequence, KV head)s have many partials each: more warps for each.  Decode
  // and merge of 131072 tokens in all, 8 KV heads, us with 16 warps / with 4, by workers
  // per (sequence, KV head): 222 46.8/48.8, 111 45.3/46.9, 56 45.5/47.8, 37 45.9/48.2,
  // 28 45.7/46.6, 19 48.8/46.8, 14 49.0/46.1, 7 53.4/46.1.
  if (workers > 32 * tiles)
    e = launch_pdl(combine_kernel<D, 16, BF16>, dim3((unsigned)(tiles * G)), 512, 0, stream, ws,
                   l_part, meta, kv_lens, o, lse, G, Hkv, by_tile);
  else
    e = launch_pdl(combine_kernel<D, 4, BF16>,
                   dim3((unsigned)((by_tile ? tiles : (int64_t)workers) * G)), 128, 0, stream, ws,
                   l_part, meta, kv_lens, o, lse, G, Hkv, by_tile);
  if (e != cudaSuccess) return set_cuda_error(e, "quantised decode combine launch");
  return B2A_OK;
}

int kvq_decode_dispatch(const void* q, int64_t q_b, int64_t q_h, const void* data,
                        const int32_t* block_table, const int32_t* kv_lens, const int32_t* pages,
                        int n_list, float* workspace, void* o, float* lse, int B, int H, int Hkv,
                        int D, int page_size, int max_pages, int num_pages, int workers, int bits,
                        int dtype, float scale, cudaStream_t stream) {
  const int shift = page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
  const int G = H / Hkv;
  auto go = [&](auto fn) {
    return fn(q, q_b, q_h, static_cast<const uint8_t*>(data), block_table, kv_lens, pages,
              pages != nullptr ? n_list : 0, workspace, o, lse, B, G, Hkv, workers, shift,
              max_pages, num_pages, scale, stream);
  };
  const bool bf = dtype == B2A_BF16;
#define B2A_KVQ(DD, BB)                                                                      \
  if (D == DD && bits == BB)                                                                 \
    return G <= 4 ? (bf ? go(launch_kvq_decode<DD, BB, true, true>)                          \
                        : go(launch_kvq_decode<DD, BB, false, true>))                        \
                  : (bf ? go(launch_kvq_decode<DD, BB, true, false>)                         \
                        : go(launch_kvq_decode<DD, BB, false, false>));
  B2A_KVQ(64, 4)
  B2A_KVQ(64, 8)
  B2A_KVQ(128, 4)
  B2A_KVQ(128, 8)
#undef B2A_KVQ
  return set_error(B2A_ERR_UNSUPPORTED, "quantised decode: unsupported (D, bits)");
}

}  // namespace b2a

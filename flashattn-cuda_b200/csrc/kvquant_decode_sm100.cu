// kvquant_decode_sm100.cu -- decode attention (query length 1) over the
// quantised paged KV cache (format: kvquant.cuh), and the selection of pages
// by a cheap score.
//
//   scores_kernel / select_kernel   the top_k pages of every (sequence, KV head)
//   decode_kernel                   split-KV partials over all or the selected pages
//   combine_kernel                  LSE-weighted merge of the splits
#include <type_traits>

#include "kvquant.cuh"
#include "b2a_host.h"

namespace b2a {
namespace kvq {

constexpr int kMaxG = 8;  // query heads of one KV head
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;
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
// bit however the work is split.  8 lanes hold a page's bounds, 4 pages a warp.
template <int D, bool BF16>
__global__ void __launch_bounds__(128)
    scores_kernel(const void* __restrict__ q, long long q_b, long long q_h,
                  const int8_t* __restrict__ index, const float* __restrict__ index_scale,
                  const int32_t* __restrict__ block_table, const int32_t* __restrict__ kv_lens,
                  uint32_t* __restrict__ keys, int G, int Hkv, int page_size, int max_pages,
                  int num_pages) {
  using T1 = typename Elem<BF16>::T;
  __shared__ __align__(16) int8_t s_pos[kMaxG][D];  // max(q8, 0)
  __shared__ __align__(16) int8_t s_neg[kMaxG][D];  // min(q8, 0)
  __shared__ float s_scale[kMaxG];
  const int b = blockIdx.z, hkv = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = table_len(kv_lens, b, page_size, max_pages,
                            blockIdx.x == 0 && hkv == 0 && threadIdx.x == 0);
  const int count = (int)(((long long)len + page_size - 1) / page_size);
  if ((int)(blockIdx.x * 128) >= count) return;
  for (int g = warp; g < G; g += 4) {
    const T1* qp = static_cast<const T1*>(q) + b * q_b + (hkv * G + g) * q_h;
    float v[D / 32], top = 0.f;
    bool ok = true;
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
      const int c = code127(v[i], scale, inv);
      s_pos[g][lane + 32 * i] = (int8_t)max(c, 0);
      s_neg[g][lane + 32 * i] = (int8_t)min(c, 0);
    }
    if (lane == 0) s_scale[g] = scale;
  }
  __syncthreads();
  constexpr int W = D / 32;  // 4-byte words per lane of a row's D bytes
  const int sub = lane & 7;
  // 128 pages per CTA
  for (int p = blockIdx.x * 128 + warp * 4 + (lane >> 3); p < min(count, (int)(blockIdx.x + 1) * 128);
       p += 16) {
    const unsigned mask = 0xffu << (lane & 24);  // the page's 8 lanes
    int page = block_table[(size_t)b * max_pages + p];
    if (page < 0 || page >= num_pages) {
      if (sub == 0) atomicOr(&g_error_flags, 2u);
      page = 0;
    }
    const size_t row = (size_t)page * Hkv + hkv;
    const int* lo = reinterpret_cast<const int*>(index + row * 2 * D) + sub * W;
    const int* hi = reinterpret_cast<const int*>(index + row * 2 * D + D) + sub * W;
    const float ps = index_scale[row];
    float best = -INFINITY;
    for (int g = 0; g < G; ++g) {
      int dot = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        dot = __dp4a(hi[i], reinterpret_cast<const int*>(s_pos[g])[sub * W + i], dot);
        dot = __dp4a(lo[i], reinterpret_cast<const int*>(s_neg[g])[sub * W + i], dot);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) dot += __shfl_xor_sync(mask, dot, o);
      float s = __fmul_rn(__fmul_rn((float)dot, s_scale[g]), ps);
      if (isnan(s)) s = INFINITY;  // a page or query that is not finite is not hidden
      best = fmaxf(best, s);
    }
    if (p == count - 1) best = INFINITY;  // the page being filled
    if (sub == 0) keys[((size_t)b * Hkv + hkv) * max_pages + p] = order_key(best);
  }
}

// The top_k of `count` keys, ties to the lowest page, in ascending order.
constexpr int kSelThreads = 256;
__global__ void __launch_bounds__(kSelThreads)
    select_kernel(const uint32_t* __restrict__ keys, const int32_t* __restrict__ kv_lens,
                  int32_t* __restrict__ pages, int Hkv, int page_size, int max_pages, int top_k) {
  __shared__ int s_cnt[kSelThreads / 32][2];
  const int hkv = blockIdx.x, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = table_len(kv_lens, b, page_size, max_pages, false);
  const int count = (int)(((long long)len + page_size - 1) / page_size);
  const uint32_t* kp = keys + ((size_t)b * Hkv + hkv) * max_pages;
  int32_t* out = pages + ((size_t)b * Hkv + hkv) * top_k;
  if (count <= top_k) {
    for (int i = threadIdx.x; i < top_k; i += kSelThreads) out[i] = i < count ? i : -1;
    return;
  }
  auto total = [&](int n) {  // sum over the block
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if (lane == 0) s_cnt[warp][0] = n;
    __syncthreads();
    int t = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) t += s_cnt[w][0];
    return t;
  };
  // the top_k-th largest key, bit by bit: the largest t with top_k keys >= t
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = t | (1u << bit);
    int n = 0;
    for (int i = threadIdx.x; i < count; i += kSelThreads) n += kp[i] >= cand;
    if (total(n) >= top_k) t = cand;
  }
  int n = 0;
  for (int i = threadIdx.x; i < count; i += kSelThreads) n += kp[i] > t;
  int ties = top_k - total(n);  // how many keys equal to t are taken, lowest pages first
  int base = 0, seen = 0;       // written, and equal keys met, so far
  for (int i0 = 0; i0 < count; i0 += kSelThreads) {
    const int i = i0 + threadIdx.x;
    const uint32_t k = i < count ? kp[i] : 0u;
    const bool eq = i < count && k == t, gt = i < count && k > t;
    const unsigned meq = __ballot_sync(0xffffffffu, eq), mgt = __ballot_sync(0xffffffffu, gt);
    __syncthreads();
    if (lane == 0) {
      s_cnt[warp][0] = __popc(mgt);
      s_cnt[warp][1] = __popc(meq);
    }
    __syncthreads();
    int gt_before = __popc(mgt & ((1u << lane) - 1)), eq_before = __popc(meq & ((1u << lane) - 1));
    int gt_all = 0, eq_all = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) {
      if (w < warp) gt_before += s_cnt[w][0], eq_before += s_cnt[w][1];
      gt_all += s_cnt[w][0], eq_all += s_cnt[w][1];
    }
    if (gt || (eq && seen + eq_before < ties))
      out[base + gt_before + min(eq_before, ties - seen)] = i;
    base += gt_all + min(eq_all, ties - seen);
    seen = min(seen + eq_all, ties);
  }
}

// ------------------------------------------------------------------- attention
// One CTA per (split, KV head, sequence).  Its warps take the split's 64-token
// steps in turn and work alone: each has its own ring of stages that its lanes
// fill with bulk copies (one copy a page: a block is contiguous), its own
// online softmax and its own accumulators, so the loop has no barrier between
// warps; they merge once at the end.
//
// Both products run on the tensor cores on the raw codes, and the (scale, min)
// pairs are applied outside them in fp32:
//   S[tok, h] = sum_g kscale[tok, g] (code . q)_g + kmin[tok, g] qsum[h, g]
//   O[h, d]   = sum_tok (p vscale[tok, g]) code[tok, d] + sum_tok p vmin[tok, g]
// so K is used exactly and p*vscale is the only value rounded to 16 bits.
//   Codes are not converted: a code c in the low mantissa bits of an fp16 with
// zero exponent IS the subnormal c * 2^-24, which the tensor cores multiply
// exactly, so unpacking is one mask a pair (and a shift by 8 every second one).
// Codes masked in place at bits 4-7 are 16 c * 2^-24; the 16 is taken out of q
// (K) or of the finished channel (V).  Both cache dtypes use fp16 operands: a
// query head is brought to [2^12, 2^13) by a power of two, and p*vscale to at
// most 2 by a running one, so neither overflows nor loses bits that matter.
//
// The token dimension is M of both products (A = K codes [tok, d], and A =
// V codes transposed [d, tok]) and the heads are N = 8, so no row of the
// matrix instructions is wasted for groups of 8 and P needs only an 8x8
// transpose (movmatrix) between them.  Contraction and output channels are
// dealt to lanes so that a lane's operand is a run of codes as they lie in
// memory.
template <int D, int BITS>
struct DecCfg {
  static constexpr int kStep = 64;  // tokens per step
  static constexpr int kRow = row_bytes(D, BITS);
  static constexpr int kNG = D / kGroup;
  static constexpr int kStage = kStep * (2 * kRow + 2 * kNG * 4);
  // Two stages of 9 or 17 KB a warp; three CTAs of 74 or 70 KB fit an SM.
  static constexpr int kWarps = (D == 128 && BITS == 8) ? 2 : 4;
  static constexpr int kStages = 2;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kPad = D + 4;  // merge row, padded against bank conflicts
  static constexpr int kMerge = kWarps * (8 * kPad + 16) * 4;
  static constexpr int kOffBar = kRing > kMerge ? kRing : kMerge;
  static constexpr int kOffValid = kOffBar + kWarps * kStages * 8;  // [warp][stage] int4
  static constexpr int kOffAbort = kOffValid + kWarps * kStages * 16;
  static constexpr int kSmem = kOffAbort + 16;
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
// subnormals: r[0], r[2] hold c * 2^-24, r[1], r[3] hold 16 c * 2^-24.
__device__ __forceinline__ void unpack4(uint32_t x, uint32_t* r) {
  r[0] = x & 0x000f000fu;
  r[1] = x & 0x00f000f0u;
  x >>= 8;
  r[2] = x & 0x000f000fu;
  r[3] = x & 0x00f000f0u;
}
// 2^e as fp32, e clamped to the normal range
__device__ __forceinline__ float pow2i(int e) {
  return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23);
}

template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(32 * DecCfg<D, BITS>::kWarps, 3)
    decode_kernel(const void* __restrict__ q, long long q_b, long long q_h,
                  const uint8_t* __restrict__ data, const int32_t* __restrict__ block_table,
                  const int32_t* __restrict__ kv_lens, const int32_t* __restrict__ pages,
                  int n_list, float* __restrict__ o_part, float* __restrict__ l_part,
                  void* __restrict__ out, float* __restrict__ lse, int G, int Hkv, int splits,
                  int tps, int page_shift, int max_pages, int num_pages, float scale_log2) {
  using C = DecCfg<D, BITS>;
  using T1 = typename Elem<BF16>::T;
  using T2 = typename Elem<BF16>::T2;
  constexpr int ROW = C::kRow, NG = C::kNG, S = C::kStages, STEP = C::kStep, W = C::kWarps;
  constexpr int SL = STEP / 16;  // 16-token slabs per step
  extern __shared__ __align__(128) uint8_t smem[];
  const int split = blockIdx.x, hkv = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int H = Hkv * G;
  const int page_size = 1 << page_shift;
  const int len = table_len(kv_lens, b, page_size, max_pages,
                            split == 0 && hkv == 0 && threadIdx.x == 0);
  const int span = pages != nullptr ? n_list << page_shift : len;
  const int t_begin = split * tps, t_end = min(span, t_begin + tps);
  const size_t row0 = (size_t)b * H + hkv * G;  // first query head
  if (t_begin >= t_end) {  // no token: an empty partial, or the whole answer
    for (int i = threadIdx.x; i < G; i += 32 * W) {
      if (splits > 1) l_part[(row0 + i) * splits + split] = -INFINITY;
      else if (lse != nullptr) lse[row0 + i] = -INFINITY;
    }
    if (splits == 1)
      for (int i = threadIdx.x; i < G * D; i += 32 * W)
        static_cast<T1*>(out)[row0 * D + i] = Elem<BF16>::from(0.f);
    return;
  }

  // ---------------------------------------------------------------- the ring
  const int np_shift = 6 - page_shift;  // log2 of the blocks per stage: 1, 2 or 4
  const uint32_t blk = (uint32_t)block_bytes(D, 1, BITS) << page_shift;
  uint8_t* ring = smem + warp * S * C::kStage;
  const uint32_t ring0 = smem_u32(ring), bar0 = smem_u32(smem + C::kOffBar) + warp * S * 8;
  int* s_valid = reinterpret_cast<int*>(smem + C::kOffValid) + warp * S * 4;  // tokens per slab
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffAbort);
  if (lane < S) mbar_init(bar0 + 8 * lane, 1u);
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_mbar_init();
  __syncthreads();
  const int steps = (t_end - t_begin + STEP - 1) / STEP;
  const int n = (steps - warp + W - 1) / W;  // this warp's steps
  const int32_t* list = pages == nullptr ? nullptr : pages + ((size_t)b * Hkv + hkv) * n_list;
  const int32_t* table = block_table + (size_t)b * max_pages;

  // Page numbers are looked up 32 blocks at a time, one a lane, and one window
  // ahead, so that the two dependent loads are off the loop's path.
  auto lookup = [&](int k, int& page, int& valid) {  // this warp's block k
    page = -1;
    valid = 0;
    const int i = k >> np_shift;
    if (i >= n) return;
    const int pos = t_begin + (warp + W * i) * STEP + ((k & ((1 << np_shift) - 1)) << page_shift);
    if (pos >= t_end) return;
    int lp = pos >> page_shift;
    if (list != nullptr) lp = list[lp];
    if (lp < 0 || lp >= max_pages) return;
    valid = min(max(len - (lp << page_shift), 0), page_size);
    if (valid == 0) return;
    page = table[lp];
    if (page < 0 || page >= num_pages) {
      atomicOr(&g_error_flags, 2u);  // page number out of range: read page 0 instead
      page = 0;
    }
  };
  int page0, valid0, page1, valid1;
  lookup(lane, page0, valid0);
  lookup(32 + lane, page1, valid1);
  auto issue = [&](int i, int st) {  // copy step i's blocks into stage st
    const int k = i << np_shift;
    if ((k & 31) == 0 && k > 0) {
      page0 = page1;
      valid0 = valid1;
      lookup(k + 32 + lane, page1, valid1);
    }
    const int page = __shfl_sync(0xffffffffu, page0, (k + lane) & 31);
    const int valid = __shfl_sync(0xffffffffu, valid0, (k + lane) & 31);
    // slab `lane` (< 4) lies in block lane / (page / 16)
    const int slab = __shfl_sync(0xffffffffu, valid0, (k + (lane >> (page_shift - 4))) & 31) -
                     16 * (lane & ((1 << (page_shift - 4)) - 1));
    const bool copy = lane < (1 << np_shift) && valid > 0;
    const int some = __popc(__ballot_sync(0xffffffffu, copy));
    if (lane < 4) s_valid[4 * st + lane] = min(max(slab, 0), 16);
    const uint32_t bar = bar0 + 8 * st;
    if (lane == 0) mbar_arrive_expect_tx(bar, some * blk);
    __syncwarp();
    if (copy)
      bulk_load(ring0 + st * C::kStage + lane * blk, data + ((size_t)page * Hkv + hkv) * blk, blk,
                bar);
  };
  for (int i = 0; i < min(n, S); ++i) issue(i, i);

  // ------------------------------------------------------------------ queries
  // B fragments of S: lane (g, t) holds head g's channels 64*grp + 16 t + 0..15
  // in the order in which a K row's codes unpack, over 16 where those are 16 c.
  uint32_t qb[NG * 4][2];
  float qsum[NG][2], sl2[2];  // of heads 2t, 2t+1
  {
    const T1* qp = static_cast<const T1*>(q) + b * q_b + (long long)(hkv * G + g) * q_h + 16 * t;
    float f[NG][16], top = 0.f;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      uint32_t u[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
      if (g < G) {
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
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int shift = 139 - (int)(__float_as_uint(top) >> 23);  // to [2^12, 2^13)
    const float mul = pow2i(shift);
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        f[gr][j] *= mul;
        sum += f[gr][j];
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= pow2i(-24);  // the codes' factor
      qsum[gr][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
      qsum[gr][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (BITS == 4) {
          const float* x = &f[gr][8 * (k / 2) + 2 * (k & 1)];
          qb[gr * 4 + k][0] = pack2_u32<false>(x[0], x[4]);
          qb[gr * 4 + k][1] = pack2_u32<false>(x[1] * 0.0625f, x[5] * 0.0625f);
        } else {
          const float* x = &f[gr][4 * k];
          qb[gr * 4 + k][0] = pack2_u32<false>(x[0], x[1]);
          qb[gr * 4 + k][1] = pack2_u32<false>(x[2], x[3]);
        }
      }
    }
    const int e = 24 - min(max(shift, -126), 127);
    const float s2 = scale_log2 * pow2i(e);  // what a score in these units is in log2
    sl2[0] = __shfl_sync(0xffffffffu, s2, 8 * t);
    sl2[1] = __shfl_sync(0xffffffffu, s2, 8 * t + 4);
  }

  // --------------------------------------------------------------------- loop
  float o[NG][4][4];  // [group][tile][(d even, head 2t), (even, 2t+1), (odd, 2t), (odd, 2t+1)]
  float omin[NG][2];  // sum of p * vmin over this lane's tokens
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  // value scales are multiplied by vmul = 2^(127 - vexp), vexp the biased
  // exponent of the largest so far
  int vexp = 1;
  float vmul = pow2i(126);
#pragma unroll
  for (int gr = 0; gr < NG; ++gr) {
    omin[gr][0] = omin[gr][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[gr][i][e] = 0.f;
  }
  // Slab s of a stage: codes at (s >> 1) * code_hi + (s & 1) * code_lo, params
  // likewise; 16-token pages put each slab in a block of its own.
  const uint32_t code_lo = page_shift == 4 ? blk : 16 * ROW;
  const uint32_t code_hi = page_shift == 6 ? 32 * ROW : page_shift == 5 ? blk : 2 * blk;
  const uint32_t par_lo = page_shift == 4 ? blk : 16 * NG * 4;
  const uint32_t par_hi = page_shift == 6 ? 32 * NG * 4 : page_shift == 5 ? blk : 2 * blk;
  const uint32_t v_off = ROW << page_shift, vp_off = (NG * 4) << page_shift;
  const int tok = (g >> 1) + (g & 1) * 4;  // S row g is token `tok` of the slab, row g+8 8 later

  // One step; nv: tokens of each slab.  FULL: all of them, known by the caller,
  // which leaves one run of straight code whose slabs overlap.
  auto step = [&](auto full, const uint8_t* stage, const int (&nv)[4]) {
    constexpr bool FULL = decltype(full)::value;

    // ---- S = K q^T
    float s[SL][4];
    uint32_t vpar[SL][2][NG];  // (scale, min) of V of rows g, g+8
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) {
      if (!FULL && nv[sl] == 0) {  // the same in every lane
        s[sl][0] = s[sl][1] = s[sl][2] = s[sl][3] = -INFINITY;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) vpar[sl][0][gr] = vpar[sl][1][gr] = 0u;
        continue;
      }
      const uint8_t* kc = stage + (sl >> 1) * code_hi + (sl & 1) * code_lo + tok * ROW;
      const uint8_t* kp =
          stage + 2 * v_off + (sl >> 1) * par_hi + (sl & 1) * par_lo + tok * NG * 4;
      uint32_t kpar[2][NG];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if constexpr (NG == 2) {
          *reinterpret_cast<uint2*>(kpar[r]) = *reinterpret_cast<const uint2*>(kp + r * 8 * NG * 4);
          *reinterpret_cast<uint2*>(vpar[sl][r]) =
              *reinterpret_cast<const uint2*>(kp + vp_off + r * 8 * NG * 4);
        } else {
          kpar[r][0] = *reinterpret_cast<const uint32_t*>(kp + r * 8 * NG * 4);
          vpar[sl][r][0] = *reinterpret_cast<const uint32_t*>(kp + vp_off + r * 8 * NG * 4);
        }
      }
      s[sl][0] = s[sl][1] = s[sl][2] = s[sl][3] = 0.f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        float acc[4];
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
        for (int r = 0; r < 2; ++r) {
          const float2 pr = param<BF16>(kpar[r][gr]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            s[sl][2 * r + h] =
                fmaf(pr.x, acc[2 * r + h], fmaf(pr.y, qsum[gr][h], s[sl][2 * r + h]));
        }
      }
      // tokens past the end: whatever their slots hold is dropped here
      if (!FULL && nv[sl] < 16) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (tok + 8 * r >= nv[sl]) {
            s[sl][2 * r] = s[sl][2 * r + 1] = -INFINITY;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) vpar[sl][r][gr] = 0u;
          }
      }
    }

    // ---- online softmax, per head over the step's tokens (rows: lanes of one t)
    float alpha[2];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = fmaxf(s[0][h], s[0][h + 2]);
#pragma unroll
      for (int sl = 1; sl < SL; ++sl) mx = fmax3(mx, s[sl][h], s[sl][h + 2]);
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[h], mx * sl2[h]);
      const float mu = mn == -INFINITY ? 0.f : mn;
      alpha[h] = ex2_mufu(m[h] - mu);
      moved = moved || alpha[h] != 1.f;
      m[h] = mn;
      float sum = 0.f;
#pragma unroll
      for (int sl = 0; sl < SL; ++sl)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float p = ex2_mufu(fmaf(s[sl][2 * r + h], sl2[h], -mu));
          s[sl][2 * r + h] = p;
          sum += p;
        }
      l[h] = l[h] * alpha[h] + sum;
    }
    T2 big = *reinterpret_cast<T2*>(&vpar[0][0][0]);  // largest value scale, in .x
#pragma unroll
    for (int sl = 0; sl < SL; ++sl)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) big = __hmax2(big, *reinterpret_cast<T2*>(&vpar[sl][r][gr]));
    const float vbig = Elem<BF16>::unpack(big).x;
    float f = 1.f;
    if (__any_sync(0xffffffffu, vbig * vmul >= 2.f)) {
      const int e = min((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(vbig)) >> 23), 253);
      f = pow2i(vexp - e);
      moved = true;
      vexp = e;
      vmul = pow2i(127 - e);
    }
    if (__any_sync(0xffffffffu, moved)) {
      const float ao[2] = {alpha[0] * f, alpha[1] * f};
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        omin[gr][0] *= alpha[0];
        omin[gr][1] *= alpha[1];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[gr][k][e] *= ao[e & 1];
      }
    }

    // ---- O += V^T P
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) {
      if (!FULL && nv[sl] == 0) continue;
      const uint8_t* vc =
          stage + v_off + (sl >> 1) * code_hi + (sl & 1) * code_lo + g * BITS + t * ROW;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        uint32_t pb[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 pr = param<BF16>(vpar[sl][r][gr]);
          const float w = pr.x * vmul;
          omin[gr][0] = fmaf(s[sl][2 * r], pr.y, omin[gr][0]);
          omin[gr][1] = fmaf(s[sl][2 * r + 1], pr.y, omin[gr][1]);
          pb[r] = movmatrix_trans(pack2_u32<false>(s[sl][2 * r] * w, s[sl][2 * r + 1] * w));
        }
        if constexpr (BITS == 4) {
          const uint32_t wa = *reinterpret_cast<const uint32_t*>(vc + gr * 32);
          const uint32_t wb = *reinterpret_cast<const uint32_t*>(vc + gr * 32 + 4 * ROW);
          const uint32_t wc = *reinterpret_cast<const uint32_t*>(vc + gr * 32 + 8 * ROW);
          const uint32_t wd = *reinterpret_cast<const uint32_t*>(vc + gr * 32 + 12 * ROW);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // channels 8g + 4*hf + 0..3
            uint32_t a[4], z[4];
            unpack4(__byte_perm(wa, wb, hf ? 0x7632 : 0x5410), a);
            unpack4(__byte_perm(wc, wd, hf ? 0x7632 : 0x5410), z);
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

  };

  bool ok = true;
  int st = 0;
  uint32_t phase = 0;
  for (int i = 0; i < n; ++i) {
    if (!mbar_wait(bar0 + 8 * st, phase, abort_flag)) {
      ok = false;
      break;
    }
    const uint8_t* stage = ring + st * C::kStage;
    const int4 nv4 = *reinterpret_cast<const int4*>(s_valid + 4 * st);
    const int nv[4] = {nv4.x, nv4.y, nv4.z, nv4.w};
    if (nv4.x + nv4.y + nv4.z + nv4.w == STEP) step(std::true_type{}, stage, nv);
    else step(std::false_type{}, stage, nv);
    __syncwarp();  // every lane has read the stage
    if (i + S < n) issue(i + S, st);
    if (++st == S) {
      st = 0;
      phase ^= 1u;
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

  // ---------------------------------------------------------------- merge warps
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) omin[gr][h] += __shfl_xor_sync(0xffffffffu, omin[gr][h], x);
    }
    if (!ok) l[h] = 0.f;
  }
  const float vscale = pow2i(vexp - 127);
  constexpr float kEven = 16777216.f;  // 2^24: the codes' factor
  constexpr float kOdd = BITS == 4 ? 1048576.f : kEven;  // odd channels were 16 c
  __syncthreads();  // the rings are drained: their memory holds the merge now
  constexpr int P = C::kPad;
  float* mo = reinterpret_cast<float*>(smem);  // [W][8][P]
  float* mm = mo + W * 8 * P;                  // [W][8] m, [W][8] l
  float* ml = mm + W * 8;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float* dst = mo + (warp * 8 + 2 * t + h) * P + 8 * g;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<float2*>(dst + gr * 64 + 2 * k) =
            make_float2(fmaf(o[gr][k][h] * kEven, vscale, omin[gr][h]),
                        fmaf(o[gr][k][2 + h] * kOdd, vscale, omin[gr][h]));
    if (g == 0) {
      mm[warp * 8 + 2 * t + h] = m[h];
      ml[warp * 8 + 2 * t + h] = l[h];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += 32 * W) {
    const int h = i / D, d = i % D;
    float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, mm[w * 8 + h]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float lw = ml[w * 8 + h];
      if (lw == 0.f) continue;  // no token
      const float x = ex2_mufu(mm[w * 8 + h] - M);
      L += lw * x;
      acc += mo[(w * 8 + h) * P + d] * x;
    }
    const float val = L == 0.f ? 0.f : acc / L;
    const float ll = L == 0.f ? -INFINITY : M * kLn2 + logf(L);
    const size_t row = row0 + h;
    if (splits > 1) {
      o_part[(row * splits + split) * D + d] = val;
      if (d == 0) l_part[row * splits + split] = ll;
    } else {
      static_cast<T1*>(out)[row * D + d] = Elem<BF16>::from(val);
      if (d == 0 && lse != nullptr) lse[row] = ll;
    }
  }
}

// One CTA of 4 warps per (sequence, query head).  A split whose l is -inf has
// no token and its o is not read; a NaN goes through to O and L.  The splits'
// weights are made first, one a thread; then each row of a split is read as
// 16 bytes a lane, with eight rows in flight a warp, so that a load's latency
// is paid a few times and not once per split.
constexpr int kChunk = 512;  // weights held at a time
template <int D, bool BF16>
__global__ void __launch_bounds__(128)
    combine_kernel(const float* __restrict__ o_part, const float* __restrict__ l_part,
                   void* __restrict__ out, float* __restrict__ lse, int S) {
  constexpr int LPR = D / 4, RPW = 32 / LPR;  // lanes per row, rows per warp
  __shared__ float s_w[kChunk], s_red[2][4];
  __shared__ float4 s_acc[4 * RPW][LPR];
  const size_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* lp = l_part + row * S;
  const float4* op = reinterpret_cast<const float4*>(o_part + row * S * D);
  float M = -INFINITY;
  for (int s = threadIdx.x; s < S; s += 128) M = fmaxf(M, lp[s]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  if (lane == 0) s_red[0][warp] = M;
  __syncthreads();
  M = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  const int sub = warp * RPW + lane / LPR, c = lane % LPR;
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c0 = 0; c0 < S; c0 += kChunk) {
    const int cn = min(kChunk, S - c0);
    __syncthreads();
    for (int s = threadIdx.x; s < cn; s += 128) {
      const float v = lp[c0 + s];
      const float w = v == -INFINITY ? 0.f : expf(v - M);
      s_w[s] = w;
      L += w;
    }
    __syncthreads();
    for (int s0 = sub; s0 < cn; s0 += 8 * 4 * RPW) {
      float4 v[8];
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int s = s0 + k * 4 * RPW;
        w[k] = s < cn ? s_w[s] : 0.f;
        // a weight of zero may stand for a row that was not written
        v[k] = w[k] != 0.f ? op[(size_t)(c0 + s) * LPR + c] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        acc.x = fmaf(w[k], v[k].x, acc.x);
        acc.y = fmaf(w[k], v[k].y, acc.y);
        acc.z = fmaf(w[k], v[k].z, acc.z);
        acc.w = fmaf(w[k], v[k].w, acc.w);
      }
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
  if (lane == 0) s_red[1][warp] = L;
  s_acc[sub][c] = acc;
  __syncthreads();
  L = s_red[1][0] + s_red[1][1] + s_red[1][2] + s_red[1][3];
  if (threadIdx.x < D) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 4 * RPW; ++k)
      a += reinterpret_cast<const float*>(s_acc[k])[threadIdx.x];
    static_cast<typename Elem<BF16>::T*>(out)[row * D + threadIdx.x] =
        Elem<BF16>::from(L == 0.f ? 0.f : a / L);
  }
  if (threadIdx.x == 0 && lse != nullptr) lse[row] = L == 0.f ? -INFINITY : M + logf(L);
}

}  // namespace kvq

B2A_DEFINE_ERROR_READER(kvquant_decode)

int kvq_select_dispatch(const void* q, int64_t q_b, int64_t q_h, const int8_t* index,
                        const float* index_scale, const int32_t* block_table,
                        const int32_t* kv_lens, uint32_t* keys, int32_t* pages, int B, int H,
                        int Hkv, int D, int page_size, int max_pages, int num_pages, int top_k,
                        int dtype, cudaStream_t stream) {
  using namespace kvq;
  dim3 grid((unsigned)((max_pages + 127) / 128), (unsigned)Hkv, (unsigned)B);
  auto go = [&](auto kern) {
    kern<<<grid, 128, 0, stream>>>(q, q_b, q_h, index, index_scale, block_table, kv_lens, keys,
                                   H / Hkv, Hkv, page_size, max_pages, num_pages);
  };
  const bool bf = dtype == B2A_BF16;
  if (D == 64) bf ? go(scores_kernel<64, true>) : go(scores_kernel<64, false>);
  else bf ? go(scores_kernel<128, true>) : go(scores_kernel<128, false>);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "page score kernel launch");
  select_kernel<<<dim3((unsigned)Hkv, (unsigned)B), kSelThreads, 0, stream>>>(
      keys, kv_lens, pages, Hkv, page_size, max_pages, top_k);
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "page selection kernel launch");
  return B2A_OK;
}

int kvq_decode_splits(int B, int Hkv, long long max_tokens) {
  const long long want = 148 * 4;
  long long s = (want + (long long)B * Hkv - 1) / ((long long)B * Hkv);
  const long long most = (max_tokens + 255) / 256;
  s = s < most ? s : most;
  const long long least = (max_tokens + 4095) / 4096;
  s = s > least ? s : least;
  return (int)(s < 1 ? 1 : s > 65535 ? 65535 : s);
}

template <int D, int BITS, bool BF16>
static int launch_kvq_decode(const void* q, int64_t q_b, int64_t q_h, const uint8_t* data,
                             const int32_t* block_table, const int32_t* kv_lens,
                             const int32_t* pages, int n_list, float* o_part, float* l_part,
                             void* o, float* lse, int B, int G, int Hkv, int splits, int tps,
                             int page_shift, int max_pages, int num_pages, float scale,
                             cudaStream_t stream) {
  using namespace kvq;
  auto kern = decode_kernel<D, BITS, BF16>;
  constexpr int smem = DecCfg<D, BITS>::kSmem;
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return set_error(B2A_ERR_CUDA, "cudaGetDevice failed");
  if (!attr_done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return set_cuda_error(e, "cudaFuncSetAttribute(quantised decode)");
    attr_done[dev] = true;
  }
  kern<<<dim3((unsigned)splits, (unsigned)Hkv, (unsigned)B), 32 * DecCfg<D, BITS>::kWarps, smem,
         stream>>>(
      q, q_b, q_h, data, block_table, kv_lens, pages, n_list, o_part, l_part, o, lse, G, Hkv,
      splits, tps, page_shift, max_pages, num_pages, scale * kLog2e);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "quantised decode kernel launch");
  if (splits > 1) {
    combine_kernel<D, BF16><<<B * G * Hkv, 128, 0, stream>>>(o_part, l_part, o, lse, splits);
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(e, "quantised decode combine launch");
  }
  return B2A_OK;
}

int kvq_decode_dispatch(const void* q, int64_t q_b, int64_t q_h, const void* data,
                        const int32_t* block_table, const int32_t* kv_lens, const int32_t* pages,
                        int n_list, float* o_part, float* l_part, void* o, float* lse, int B,
                        int H, int Hkv, int D, int page_size, int max_pages, int num_pages,
                        int splits, int bits, int dtype, float scale, cudaStream_t stream) {
  const long long span = (long long)(pages != nullptr ? n_list : max_pages) * page_size;
  // whole pages and whole 64-token pieces, so that no step straddles a split
  const int tps = (int)(((span + splits - 1) / splits + 63) / 64 * 64);
  const int shift = page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
  auto go = [&](auto fn) {
    return fn(q, q_b, q_h, static_cast<const uint8_t*>(data), block_table, kv_lens, pages, n_list,
              o_part, l_part, o, lse, B, H / Hkv, Hkv, splits, tps, shift, max_pages, num_pages,
              scale, stream);
  };
  const bool bf = dtype == B2A_BF16;
  if (D == 64 && bits == 4)
    return bf ? go(launch_kvq_decode<64, 4, true>) : go(launch_kvq_decode<64, 4, false>);
  if (D == 64) return bf ? go(launch_kvq_decode<64, 8, true>) : go(launch_kvq_decode<64, 8, false>);
  if (bits == 4)
    return bf ? go(launch_kvq_decode<128, 4, true>) : go(launch_kvq_decode<128, 4, false>);
  return bf ? go(launch_kvq_decode<128, 8, true>) : go(launch_kvq_decode<128, 8, false>);
}

}  // namespace b2a

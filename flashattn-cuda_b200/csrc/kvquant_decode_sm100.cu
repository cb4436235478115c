// kvquant_decode_sm100.cu -- decode attention (query length 1) over the
// quantised paged KV cache (format: kvquant.cuh), and the selection of pages
// by a cheap score.
//
//   scores_kernel / select_kernel   the top_k pages of every (sequence, KV head)
//   decode_kernel                   split-KV partials over all or the selected pages
//   combine_kernel                  LSE-weighted merge of the splits
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
// One CTA per (split, KV head, sequence).  Its four warps take the split's
// 32-token steps in turn and work alone: each has its own ring of stages that
// its lanes fill with bulk copies (a whole block per page, one copy), its own
// online softmax and its own accumulators, so the loop has no barrier between
// warps; they merge once at the end.
//
// Both products run on the tensor cores on the raw codes, which are exact in
// 16 bits; the (scale, min) pairs are applied outside them in fp32:
//   S[tok, h] = sum_g kscale[tok, g] (code . q)_g + kmin[tok, g] qsum[h, g]
//   O[h, d]   = sum_tok (p vscale[tok, g]) code[tok, d] + sum_tok p vmin[tok, g]
// so K is used exactly and each p*vscale is the only value rounded to 16 bits.
// In fp16 the scales are brought to at most 2 by a running power of two, so
// that p*vscale neither overflows nor sinks into subnormals.
//
// The token dimension is M of both products (A = K codes [tok, d], and A =
// V codes transposed [d, tok]) and the heads are N = 8, so no row of the
// matrix instructions is wasted for groups of 8 and P needs only an 8x8
// transpose (movmatrix) between them.  Contraction and output channels are
// dealt to lanes so that a lane's operand is a run of codes as they lie in
// memory: unpacking is mask, or-in an exponent, subtract.
template <int D, int BITS>
struct DecCfg {
  static constexpr int kStep = 32;  // tokens per step
  static constexpr int kRow = row_bytes(D, BITS);
  static constexpr int kNG = D / kGroup;
  static constexpr uint32_t kStage = kStep * (2 * kRow + 2 * kNG * 4);
  static constexpr int kStages = (D == 128 && BITS == 8) ? 2 : 3;
  static constexpr uint32_t kRing = 4 * kStages * kStage;
  static constexpr uint32_t kMerge = 4 * (8 * (D + 4) + 16) * 4;
  static constexpr uint32_t kBody = kRing > kMerge ? kRing : kMerge;
  static constexpr uint32_t kOffBar = kBody;
  static constexpr uint32_t kOffValid = kOffBar + 4 * kStages * 8;       // [warp][stage] int2
  static constexpr uint32_t kOffAbort = kOffValid + 4 * kStages * 8;
  static constexpr uint32_t kSmem = kOffAbort + 16;
};

// D[16x8] += A[16x16] B[16x8]
template <bool BF16>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// (a & b) | c
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t add2(uint32_t a, uint32_t b) {
  using T2 = typename Elem<BF16>::T2;
  T2 r = __hadd2(*reinterpret_cast<T2*>(&a), *reinterpret_cast<T2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
template <bool BF16>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  using T2 = typename Elem<BF16>::T2;
  T2 r = __hfma2(*reinterpret_cast<T2*>(&a), *reinterpret_cast<T2*>(&b), *reinterpret_cast<T2*>(&c));
  return *reinterpret_cast<uint32_t*>(&r);
}

// The four 4-bit codes at bits 4j of each 16-bit half of x, j = 0..3, as exact
// pairs (low half, high half).  A code is or-ed into the mantissa of a power of
// two (fp16: 1024 at bits 0-3, and 64 * 16 at bits 4-7; bf16, with 7 mantissa
// bits: 128 at bits 0-3), which is then subtracted.
template <bool BF16>
__device__ __forceinline__ void unpack4(uint32_t x, uint32_t* r) {
  if constexpr (BF16) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      r[j] = add2<true>(and_or(x >> (4 * j), 0x000f000fu, 0x43004300u), 0xc300c300u);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      r[j] = add2<false>(and_or(x, 0x000f000fu, 0x64006400u), 0xe400e400u);
      r[j + 1] = fma2<false>(and_or(x, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd400d400u);
      x >>= 8;
    }
  }
}
// The 8-bit codes of x = [c, *, c', *] as an exact pair.  fp16: 1024 + c.
// bf16 (8 significant bits): 16 (128 + high nibble) - 2176 + (128 + low nibble).
template <bool BF16>
__device__ __forceinline__ uint32_t unpack8(uint32_t x) {
  if constexpr (BF16) {
    const uint32_t lo = and_or(x, 0x000f000fu, 0x43004300u);
    const uint32_t hi = and_or(x >> 4, 0x000f000fu, 0x43004300u);
    return add2<true>(fma2<true>(hi, 0x41804180u, 0xc508c508u), lo);
  } else {
    return add2<false>(and_or(x, 0x00ff00ffu, 0x64006400u), 0xe400e400u);
  }
}

template <int NG, bool BF16>
__device__ __forceinline__ void load_params(const uint8_t* p, float2* out) {
  if constexpr (NG == 2) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    out[0] = param<BF16>(w.x);
    out[1] = param<BF16>(w.y);
  } else {
    out[0] = param<BF16>(*reinterpret_cast<const uint32_t*>(p));
  }
}

template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(128, (BITS == 8 && D == 128) ? 3 : 4)
    decode_kernel(const void* __restrict__ q, long long q_b, long long q_h,
                  const uint8_t* __restrict__ data, const int32_t* __restrict__ block_table,
                  const int32_t* __restrict__ kv_lens, const int32_t* __restrict__ pages,
                  int n_list, float* __restrict__ o_part, float* __restrict__ l_part,
                  void* __restrict__ out, float* __restrict__ lse, int G, int Hkv, int splits,
                  int tps, int page_shift, int max_pages, int num_pages, float scale_log2) {
  using C = DecCfg<D, BITS>;
  using T1 = typename Elem<BF16>::T;
  constexpr int ROW = C::kRow, NG = C::kNG, S = C::kStages, STEP = C::kStep;
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
    for (int i = threadIdx.x; i < G; i += 128) {
      if (splits > 1) l_part[(row0 + i) * splits + split] = -INFINITY;
      else if (lse != nullptr) lse[row0 + i] = -INFINITY;
    }
    if (splits == 1)
      for (int i = threadIdx.x; i < G * D; i += 128)
        static_cast<T1*>(out)[row0 * D + i] = Elem<BF16>::from(0.f);
    return;
  }

  // ---------------------------------------------------------------- the ring
  // A stage holds STEP tokens as blocks of pg = min(page, STEP) tokens.
  const int pg = min(page_size, STEP);
  const int np = STEP / pg;  // blocks per stage: 1 or 2
  uint8_t* ring = smem + warp * S * C::kStage;
  const uint32_t bar0 = smem_u32(smem + C::kOffBar) + warp * S * 8;
  int2* s_valid = reinterpret_cast<int2*>(smem + C::kOffValid) + warp * S;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffAbort);
  if (lane < S) mbar_init(bar0 + 8 * lane, 1u);
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_mbar_init();
  __syncthreads();
  const int steps = (t_end - t_begin + STEP - 1) / STEP;
  const int n = (steps - warp + 3) >> 2;  // this warp's steps
  const int32_t* list = pages == nullptr ? nullptr : pages + ((size_t)b * Hkv + hkv) * n_list;
  const int32_t* table = block_table + (size_t)b * max_pages;

  // Block `lane` (< np) of this warp's step i: its pool page (-1: nothing to
  // read) and tokens.
  auto lookup = [&](int i, int& page, int& valid) {
    page = -1;
    valid = 0;
    const int pos = t_begin + (warp + 4 * i) * STEP + lane * pg;
    if (i >= n || lane >= np || pos >= t_end) return;
    int lp = pos >> page_shift;
    if (list != nullptr) lp = list[lp];
    if (lp < 0 || lp >= max_pages) return;
    const int first = (lp << page_shift) + (pos & (page_size - 1));
    valid = min(max(len - first, 0), pg);
    if (valid == 0) return;
    page = table[lp];
    if (page < 0 || page >= num_pages) {
      atomicOr(&g_error_flags, 2u);  // page number out of range: read page 0 instead
      page = 0;
    }
  };
  auto issue = [&](int i, int page, int valid) {
    const int st = i % S;
    const uint32_t dst = smem_u32(ring + st * C::kStage), bar = bar0 + 8 * st;
    const int other = __shfl_sync(0xffffffffu, valid, 1);
    const unsigned some = __ballot_sync(0xffffffffu, valid > 0);
    const uint32_t blk = (uint32_t)(pg * (2 * ROW + 2 * NG * 4));
    if (lane == 0) {
      s_valid[st] = make_int2(valid, np == 2 ? other : 0);
      mbar_arrive_expect_tx(bar, __popc(some) * blk);
    }
    __syncwarp();
    const size_t bytes = (size_t)block_bytes(D, 1, BITS) << page_shift;
    if (page_size <= STEP) {
      if (valid > 0) bulk_load(dst + lane * blk, data + ((size_t)page * Hkv + hkv) * bytes, blk, bar);
    } else if (some) {  // a part of a page: its rows of the four pieces
      const int pool = __shfl_sync(0xffffffffu, page, 0);
      const int off = (t_begin + (warp + 4 * i) * STEP) & (page_size - 1);
      if (lane < 4) {
        const uint8_t* src = data + ((size_t)pool * Hkv + hkv) * bytes;
        const int side = lane & 1;
        if (lane < 2)
          bulk_load(dst + side * STEP * ROW, src + (side * page_size + off) * ROW, STEP * ROW, bar);
        else
          bulk_load(dst + 2 * STEP * ROW + side * STEP * NG * 4,
                    src + 2 * page_size * ROW + (side * page_size + off) * NG * 4, STEP * NG * 4,
                    bar);
      }
    }
  };
  int pageA, validA;
#pragma unroll 1
  for (int i = 0; i < S; ++i) {
    lookup(i, pageA, validA);
    if (i < n) issue(i, pageA, validA);
  }
  lookup(S, pageA, validA);  // the next step's, one step ahead

  // ------------------------------------------------------------------ queries
  // B fragments of S: lane (g, t) holds head g's channels 64*grp + 16 t + 0..15
  // in the order in which a K row's codes unpack.
  uint32_t qb[NG * 4][2];
  float qsum[NG][2];  // of heads 2t, 2t+1
  {
    const T1* qp = static_cast<const T1*>(q) + b * q_b + (long long)(hkv * G + g) * q_h + 16 * t;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      uint32_t u[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
      if (g < G) {
        *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(qp + gr * 64);
        *reinterpret_cast<uint4*>(u + 4) = *reinterpret_cast<const uint4*>(qp + gr * 64 + 8);
      }
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = param<BF16>(u[j]);
        sum += f.x + f.y;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qsum[gr][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
      qsum[gr][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (BITS == 4) {
          const uint32_t a = u[4 * (k / 2) + (k & 1)], z = u[4 * (k / 2) + (k & 1) + 2];
          qb[gr * 4 + k][0] = __byte_perm(a, z, 0x5410);
          qb[gr * 4 + k][1] = __byte_perm(a, z, 0x7632);
        } else {
          qb[gr * 4 + k][0] = u[2 * k];
          qb[gr * 4 + k][1] = u[2 * k + 1];
        }
      }
    }
  }

  // --------------------------------------------------------------------- loop
  float o[NG][4][4];    // [group][tile][(d even, head 2t), (even, 2t+1), (odd, 2t), (odd, 2t+1)]
  float omin[NG][2];    // sum of p * vmin over this lane's tokens
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int vexp = 0;         // fp16: biased exponent of the largest value scale so far
#pragma unroll
  for (int gr = 0; gr < NG; ++gr) {
    omin[gr][0] = omin[gr][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[gr][i][e] = 0.f;
  }
  // Offsets of 16-token slab s in a stage: pg = 16 puts each slab in a block of
  // its own, pg = 32 both in one.
  const uint32_t BLK16 = 16 * (2 * ROW + 2 * NG * 4);
  const uint32_t code_step = np == 2 ? BLK16 : 16 * ROW;
  const uint32_t par_step = np == 2 ? BLK16 : 16 * NG * 4;
  const uint32_t v_off = pg * ROW, kp_off = 2 * pg * ROW, vp_off = kp_off + pg * NG * 4;
  const int tok = (g >> 1) + (g & 1) * 4;  // S row g is token `tok` of the slab, row g+8 8 later

  bool ok = true;
  for (int i = 0; i < n; ++i) {
    const int st = i % S;
    if (!mbar_wait(bar0 + 8 * st, (i / S) & 1, abort_flag)) {
      ok = false;
      break;
    }
    const uint8_t* stage = ring + st * C::kStage;
    const int2 vd = s_valid[st];
    // tokens of each slab
    const int nv[2] = {np == 2 ? vd.x : min(vd.x, 16), np == 2 ? vd.y : max(vd.x - 16, 0)};

    // ---- S = K q^T
    float s[2][4];
    float2 vp[2][2][NG];  // (scale, min) of V of rows g, g+8
#pragma unroll
    for (int sl = 0; sl < 2; ++sl) {
      if (nv[sl] <= 0) {  // the same in every lane
        s[sl][0] = s[sl][1] = s[sl][2] = s[sl][3] = -INFINITY;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) vp[sl][0][gr] = vp[sl][1][gr] = make_float2(0.f, 0.f);
        continue;
      }
      const uint8_t* kc = stage + sl * code_step + tok * ROW;
      const uint8_t* kp = stage + kp_off + sl * par_step + tok * NG * 4;
      float2 par[2][NG];
      load_params<NG, BF16>(kp, par[0]);
      load_params<NG, BF16>(kp + 8 * NG * 4, par[1]);
      load_params<NG, BF16>(kp + (vp_off - kp_off), vp[sl][0]);
      load_params<NG, BF16>(kp + (vp_off - kp_off) + 8 * NG * 4, vp[sl][1]);
      s[sl][0] = s[sl][1] = s[sl][2] = s[sl][3] = 0.f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        if constexpr (BITS == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(kc + gr * 32 + t * 8);
          const uint2 y = *reinterpret_cast<const uint2*>(kc + 8 * ROW + gr * 32 + t * 8);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t a[4], z[4];
            unpack4<BF16>(w ? x.y : x.x, a);
            unpack4<BF16>(w ? y.y : y.x, z);
            mma16816<BF16>(acc, a[0], z[0], a[1], z[1], qb[gr * 4 + 2 * w][0], qb[gr * 4 + 2 * w][1]);
            mma16816<BF16>(acc, a[2], z[2], a[3], z[3], qb[gr * 4 + 2 * w + 1][0],
                           qb[gr * 4 + 2 * w + 1][1]);
          }
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(kc + gr * 64 + t * 16);
          const uint4 y = *reinterpret_cast<const uint4*>(kc + 8 * ROW + gr * 64 + t * 16);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int w = 0; w < 4; ++w)
            mma16816<BF16>(acc, unpack8<BF16>(__byte_perm(xs[w], 0, 0x4140)),
                           unpack8<BF16>(__byte_perm(ys[w], 0, 0x4140)),
                           unpack8<BF16>(__byte_perm(xs[w], 0, 0x4342)),
                           unpack8<BF16>(__byte_perm(ys[w], 0, 0x4342)), qb[gr * 4 + w][0],
                           qb[gr * 4 + w][1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 pr = par[e >> 1][gr];
          s[sl][e] = fmaf(pr.x, acc[e], fmaf(pr.y, qsum[gr][e & 1], s[sl][e]));
        }
      }
      // tokens past the end: whatever their slots hold is dropped here
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (tok + 8 * r >= nv[sl]) {
          s[sl][2 * r] = s[sl][2 * r + 1] = -INFINITY;
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) vp[sl][r][gr] = make_float2(0.f, 0.f);
        }
    }

    // ---- online softmax, per head over the step's tokens (rows: lanes of one t)
    float alpha[2];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = fmaxf(fmaxf(s[0][h], s[0][h + 2]), fmaxf(s[1][h], s[1][h + 2]));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[h], mx * scale_log2);
      const float mu = mn == -INFINITY ? 0.f : mn;
      alpha[h] = ex2_mufu(m[h] - mu);
      moved = moved || alpha[h] != 1.f;
      m[h] = mn;
      float sum = 0.f;
#pragma unroll
      for (int sl = 0; sl < 2; ++sl)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float p = ex2_mufu(fmaf(s[sl][2 * r + h], scale_log2, -mu));
          s[sl][2 * r + h] = p;
          sum += p;
        }
      l[h] = l[h] * alpha[h] + sum;
    }
    float ao[2] = {alpha[0], alpha[1]};  // of o, which also follows vexp
    float vmul = 1.f;
    if constexpr (!BF16) {
      float big = 0.f;
#pragma unroll
      for (int sl = 0; sl < 2; ++sl)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) big = fmaxf(big, vp[sl][r][gr].x);
      const int e = min((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(big)) >> 23), 253);
      if (e > vexp) {  // the same in every lane
        const float f = __uint_as_float((uint32_t)max(127 - (e - vexp), 0) << 23);
        ao[0] *= f;
        ao[1] *= f;
        moved = true;
        vexp = e;
      }
      vmul = __uint_as_float((uint32_t)(254 - vexp) << 23);
    }
    if (__any_sync(0xffffffffu, moved)) {
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
    for (int sl = 0; sl < 2; ++sl) {
      if (nv[sl] <= 0) continue;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        uint32_t pb[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 pr = vp[sl][r][gr];
          const float w = BF16 ? pr.x : pr.x * vmul;
          omin[gr][0] = fmaf(s[sl][2 * r], pr.y, omin[gr][0]);
          omin[gr][1] = fmaf(s[sl][2 * r + 1], pr.y, omin[gr][1]);
          pb[r] = movmatrix_trans(pack2_u32<BF16>(s[sl][2 * r] * w, s[sl][2 * r + 1] * w));
        }
        const uint8_t* vc = stage + v_off + sl * code_step + gr * 8 * BITS + g * BITS + t * ROW;
        if constexpr (BITS == 4) {
          const uint32_t wa = *reinterpret_cast<const uint32_t*>(vc);
          const uint32_t wb = *reinterpret_cast<const uint32_t*>(vc + 4 * ROW);
          const uint32_t wc = *reinterpret_cast<const uint32_t*>(vc + 8 * ROW);
          const uint32_t wd = *reinterpret_cast<const uint32_t*>(vc + 12 * ROW);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // channels 8g + 4*hf + 0..3
            uint32_t a[4], z[4];
            unpack4<BF16>(__byte_perm(wa, wb, hf ? 0x7632 : 0x5410), a);
            unpack4<BF16>(__byte_perm(wc, wd, hf ? 0x7632 : 0x5410), z);
            mma16816<BF16>(o[gr][2 * hf], a[0], a[1], z[0], z[1], pb[0], pb[1]);
            mma16816<BF16>(o[gr][2 * hf + 1], a[2], a[3], z[2], z[3], pb[0], pb[1]);
          }
        } else {
          const uint2 wa = *reinterpret_cast<const uint2*>(vc);
          const uint2 wb = *reinterpret_cast<const uint2*>(vc + 4 * ROW);
          const uint2 wc = *reinterpret_cast<const uint2*>(vc + 8 * ROW);
          const uint2 wd = *reinterpret_cast<const uint2*>(vc + 12 * ROW);
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // channels 8g + 2k, 2k+1
            const uint32_t xa = k < 2 ? wa.x : wa.y, xb = k < 2 ? wb.x : wb.y;
            const uint32_t xc = k < 2 ? wc.x : wc.y, xd = k < 2 ? wd.x : wd.y;
            const uint32_t s0 = k & 1 ? 0x6622 : 0x4400, s1 = k & 1 ? 0x7733 : 0x5511;
            mma16816<BF16>(o[gr][k], unpack8<BF16>(__byte_perm(xa, xb, s0)),
                           unpack8<BF16>(__byte_perm(xa, xb, s1)),
                           unpack8<BF16>(__byte_perm(xc, xd, s0)),
                           unpack8<BF16>(__byte_perm(xc, xd, s1)), pb[0], pb[1]);
          }
        }
      }
    }

    __syncwarp();  // every lane has read the stage
    if (i + S < n) issue(i + S, pageA, validA);
    lookup(i + S + 1, pageA, validA);
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
  const float vscale = BF16 ? 1.f : __uint_as_float((uint32_t)vexp << 23);
  __syncthreads();  // the rings are drained: their memory holds the merge now
  constexpr int P = D + 4;  // padded against bank conflicts
  float* mo = reinterpret_cast<float*>(smem);  // [4][8][P]
  float* mm = mo + 4 * 8 * P;                  // [4][8] m, [4][8] l
  float* ml = mm + 32;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float* dst = mo + (warp * 8 + 2 * t + h) * P + 8 * g;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<float2*>(dst + gr * 64 + 2 * k) =
            make_float2(fmaf(o[gr][k][h], vscale, omin[gr][h]),
                        fmaf(o[gr][k][2 + h], vscale, omin[gr][h]));
    if (g == 0) {
      mm[warp * 8 + 2 * t + h] = m[h];
      ml[warp * 8 + 2 * t + h] = l[h];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += 128) {
    const int h = i / D, d = i % D;
    float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, mm[w * 8 + h]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float lw = ml[w * 8 + h];
      if (lw == 0.f) continue;  // no token
      const float f = ex2_mufu(mm[w * 8 + h] - M);
      L += lw * f;
      acc += mo[(w * 8 + h) * P + d] * f;
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

// One CTA of D threads per (sequence, query head).  A split whose l is -inf has
// no token and its o is not read; a NaN goes through to O and L.
template <bool BF16>
__global__ void combine_kernel(const float* __restrict__ o_part, const float* __restrict__ l_part,
                               void* __restrict__ out, float* __restrict__ lse, int S, int D) {
  const size_t row = blockIdx.x;
  const int d = threadIdx.x;
  const float* lp = l_part + row * S;
  float M = -INFINITY;
  for (int s = 0; s < S; ++s) M = fmaxf(M, lp[s]);
  float L = 0.f, acc = 0.f;
  for (int s = 0; s < S; ++s) {
    if (lp[s] == -INFINITY) continue;
    const float w = expf(lp[s] - M);
    L += w;
    acc += w * o_part[(row * S + s) * D + d];
  }
  static_cast<typename Elem<BF16>::T*>(out)[row * D + d] =
      Elem<BF16>::from(L == 0.f ? 0.f : acc / L);
  if (d == 0 && lse != nullptr) lse[row] = L == 0.f ? -INFINITY : M + logf(L);
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
  constexpr int smem = (int)DecCfg<D, BITS>::kSmem;
  static bool attr_done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return set_error(B2A_ERR_CUDA, "cudaGetDevice failed");
  if (!attr_done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return set_cuda_error(e, "cudaFuncSetAttribute(quantised decode)");
    attr_done[dev] = true;
  }
  kern<<<dim3((unsigned)splits, (unsigned)Hkv, (unsigned)B), 128, smem, stream>>>(
      q, q_b, q_h, data, block_table, kv_lens, pages, n_list, o_part, l_part, o, lse, G, Hkv,
      splits, tps, page_shift, max_pages, num_pages, scale * kLog2e);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "quantised decode kernel launch");
  if (splits > 1) {
    combine_kernel<BF16><<<B * G * Hkv, D, 0, stream>>>(o_part, l_part, o, lse, splits, D);
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

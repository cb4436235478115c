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
// One CTA per (split, KV head, sequence); its four warps take the split's
// tokens in turn, each with its own online softmax, merged at the end.
template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(128)
    decode_kernel(const void* __restrict__ q, long long q_b, long long q_h,
                  const uint8_t* __restrict__ data, const int32_t* __restrict__ block_table,
                  const int32_t* __restrict__ kv_lens, const int32_t* __restrict__ pages,
                  int n_list, float* __restrict__ o_part, float* __restrict__ l_part,
                  void* __restrict__ out, float* __restrict__ lse, int G, int Hkv, int splits,
                  int tps, int page_size, int max_pages, int num_pages, float scale_log2) {
  using T1 = typename Elem<BF16>::T;
  constexpr int E = D / 32;  // channels per lane
  constexpr int ROW = row_bytes(D, BITS), NG = D / kGroup;
  __shared__ float s_o[4][kMaxG][D];
  __shared__ float s_m[4][kMaxG], s_l[4][kMaxG];
  const int split = blockIdx.x, hkv = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = Hkv * G;
  const int len = table_len(kv_lens, b, page_size, max_pages,
                            split == 0 && hkv == 0 && threadIdx.x == 0);
  const int span = pages != nullptr ? n_list * page_size : len;
  const int t0 = split * tps, t1 = min(span, t0 + tps);
  float qr[kMaxG][E], o[kMaxG][E], m[kMaxG], l[kMaxG];
#pragma unroll
  for (int g = 0; g < kMaxG; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[g][e] = 0.f;
      qr[g][e] = g < G ? (float)static_cast<const T1*>(q)[b * q_b + (hkv * G + g) * q_h + lane * E + e]
                       : 0.f;
    }
  }
  for (int t = t0 + warp; t < t1; t += 4) {
    int lp = t / page_size;
    const int slot = t % page_size;
    if (pages != nullptr) lp = pages[((size_t)b * Hkv + hkv) * n_list + lp];
    if (lp < 0 || lp >= max_pages || (long long)lp * page_size + slot >= len) continue;
    int page = block_table[(size_t)b * max_pages + lp];
    if (page < 0 || page >= num_pages) {
      if (lane == 0) atomicOr(&g_error_flags, 2u);
      page = 0;
    }
    const uint8_t* blk = data + ((size_t)page * Hkv + hkv) * block_bytes(D, page_size, BITS);
    float kv[2][E];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const uint8_t* row = blk + (size_t)(side * page_size + slot) * ROW;
      const float2 p = param<BF16>(reinterpret_cast<const uint32_t*>(
          blk + 2 * page_size * ROW)[(side * page_size + slot) * NG + lane * E / kGroup]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        const int c = BITS == 8 ? row[d] : (row[d / 2] >> (4 * (d & 1))) & 15;
        kv[side][e] = __fmaf_rn((float)c, p.x, p.y);
      }
    }
#pragma unroll
    for (int g = 0; g < kMaxG; ++g) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += qr[g][e] * kv[0][e];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= scale_log2;
      const float mn = fmaxf(m[g], s);
      const float a = exp2f(m[g] - mn), p = exp2f(s - mn);
      m[g] = mn;
      l[g] = l[g] * a + p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[g][e] = o[g][e] * a + p * kv[1][e];
    }
  }
#pragma unroll
  for (int g = 0; g < kMaxG; ++g) {
    s_m[warp][g] = m[g];
    s_l[warp][g] = l[g];
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][g][lane * E + e] = o[g][e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += 128) {
    const int g = i / D, d = i % D;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w][g]);
    for (int w = 0; w < 4; ++w) {
      if (s_l[w][g] == 0.f) continue;
      const float f = exp2f(s_m[w][g] - M);
      L += s_l[w][g] * f;
      acc += s_o[w][g][d] * f;
    }
    const float val = L == 0.f ? 0.f : acc / L;
    const float ll = L == 0.f ? -INFINITY : M * kLn2 + logf(L);
    const size_t row = (size_t)b * H + hkv * G + g;
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

int kvq_decode_dispatch(const void* q, int64_t q_b, int64_t q_h, const void* data,
                        const int32_t* block_table, const int32_t* kv_lens, const int32_t* pages,
                        int n_list, float* o_part, float* l_part, void* o, float* lse, int B,
                        int H, int Hkv, int D, int page_size, int max_pages, int num_pages,
                        int splits, int bits, int dtype, float scale, cudaStream_t stream) {
  using namespace kvq;
  const long long span = (long long)(pages != nullptr ? n_list : max_pages) * page_size;
  const int tps = (int)(((span + splits - 1) / splits + 63) / 64 * 64);
  dim3 grid((unsigned)splits, (unsigned)Hkv, (unsigned)B);
  auto go = [&](auto kern) {
    kern<<<grid, 128, 0, stream>>>(q, q_b, q_h, static_cast<const uint8_t*>(data), block_table,
                                   kv_lens, pages, n_list, o_part, l_part, o, lse, H / Hkv, Hkv,
                                   splits, tps, page_size, max_pages, num_pages, scale * kLog2e);
  };
  const bool bf = dtype == B2A_BF16;
  if (D == 64 && bits == 4) bf ? go(decode_kernel<64, 4, true>) : go(decode_kernel<64, 4, false>);
  else if (D == 64) bf ? go(decode_kernel<64, 8, true>) : go(decode_kernel<64, 8, false>);
  else if (bits == 4) bf ? go(decode_kernel<128, 4, true>) : go(decode_kernel<128, 4, false>);
  else bf ? go(decode_kernel<128, 8, true>) : go(decode_kernel<128, 8, false>);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "quantised decode kernel launch");
  if (splits > 1) {
    if (bf) combine_kernel<true><<<B * H, D, 0, stream>>>(o_part, l_part, o, lse, splits, D);
    else combine_kernel<false><<<B * H, D, 0, stream>>>(o_part, l_part, o, lse, splits, D);
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(e, "quantised decode combine launch");
  }
  return B2A_OK;
}

}  // namespace b2a

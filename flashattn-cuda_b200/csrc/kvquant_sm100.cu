// kvquant_sm100.cu -- writing and reading back the quantised paged KV cache
// (format: kvquant.cuh).
//
// append: tokens [B, Hkv, T, D] (any strides, rows contiguous) -> codes and
// params of the pages that the block table names, and, when the cache has an
// index, the page's channel bounds.  read: tokens of each sequence back to
// packed token-major [total, Hkv, D] rows, the layout forward_varlen takes.
//
// One warp owns one (sequence, page, KV head): the block it writes or reads is
// one contiguous piece, its param and index reductions stay inside the warp, and
// a page's index has one writer.  A row of D values is held by D/8 lanes with 16
// bytes each, so a group of 64 channels is 8 lanes and its extremes take three
// shuffles.
//
// Both are copies.  Measured at D = 128, 4 bits: reading 16 sequences of 512 to
// 16384 tokens of 8 KV heads back (709 MB read and written) 117 us, 94% of the
// measured copy rate; appending 4 x 8192 bf16 tokens (172 MB) 40 us, 67%, where
// the instructions, 247 for every two rows of K and of V, are the limit: they issue in
// 78% of the cycles, DRAM is active in 45% (41 us with one value an instruction and
// every code clamped; 8 x 8192 fp16 tokens at 8 bits with an index: 94 -> 88 us).
#include <type_traits>

#include "kvquant.cuh"
#include "b2a_host.h"

namespace b2a {
namespace kvq {

constexpr int kWarps = 4;  // warps per CTA where a sequence's units do not fit one CTA

struct NewRows {  // element strides of k_new / v_new [B, Hkv, T, D]
  long long b, h, t;
};

// A length after T more tokens: a negative one, whose tokens are dropped, stays, so
// that it does not turn into one that looks valid; nor does one pass 2^31 - 1.
__device__ __forceinline__ int advanced(int len, int T) {
  return len < 0 ? len : (int)min((long long)len + T, 0x7fffffffll);
}

template <int D, int BITS, bool BF16>
__global__ void append_kernel(const void* k_new, const void* v_new,
                              NewRows ks, NewRows vs, uint8_t* __restrict__ data,
                              int8_t* __restrict__ index, float* __restrict__ index_scale,
                              const int32_t* block_table, int32_t* kv_lens, int Hkv,
                              int T, int J, int page_shift, int max_pages, int num_pages,
                              int one_cta, int advance) {
  using T1 = typename Elem<BF16>::T;
  using T2 = typename Elem<BF16>::T2;
  constexpr int LPR = D / 8;             // lanes per row
  constexpr int RPI = 32 / LPR;          // rows per iteration
  constexpr int ROW = row_bytes(D, BITS);
  constexpr int NG = D / kGroup;
  const int b = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // a CTA holds pages of one KV head, or (one_cta) all of its sequence's units
  const int hkv = one_cta ? warp % Hkv : blockIdx.y;
  const int j = one_cta ? warp / Hkv : blockIdx.x * (blockDim.x >> 5) + warp;
  const int page_size = 1 << page_shift;
  pdl_trigger();
  pdl_wait();
  const int len = kv_lens[b];
  // With `advance` one CTA holds all units of its sequence: the length moves
  // only after every warp has read it.
  if (advance) {
    __syncthreads();
    if (threadIdx.x == 0) kv_lens[b] = advanced(len, T);
  }
  if (j >= J) return;
  if (len < 0) {
    if (lane == 0) atomicOr(&g_error_flags, 4u);
    return;
  }
  const long long pidx = (len >> page_shift) + (long long)j;  // 64 bits: len + T may pass 2^31
  const long long first = pidx << page_shift;
  const long long end = (long long)len + T;
  if (first >= end) return;
  const int page = pidx < max_pages ? block_table[(size_t)b * max_pages + pidx] : -1;
  if (page < 0 || page >= num_pages) {
    if (lane == 0) atomicOr(&g_error_flags, 4u);  // no page for these tokens: dropped
    return;
  }
  const int s0 = (int)max(0ll, len - first);              // slots [s0, s1) are written
  const int s1 = (int)min((long long)page_size, end - first);
  const long long t0 = first - len;                       // token of slot 0
  uint8_t* blk = data + ((size_t)page * Hkv + hkv) * block_bytes(D, page_size, BITS);
  const int r = lane / LPR, c = lane % LPR;               // row of the iteration, 8-channel chunk
  const int grp = c / 8;
  const T1* kp = static_cast<const T1*>(k_new) + b * ks.b + hkv * ks.h + 8 * c;
  const T1* vp = static_cast<const T1*>(v_new) + b * vs.b + hkv * vs.h + 8 * c;

  Vec8<BF16> mn, mx;  // index: channel bounds over this lane's rows
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mn.v[i] = Elem<BF16>::pack(INFINITY, INFINITY);
    mx.v[i] = Elem<BF16>::pack(-INFINITY, -INFINITY);
  }
  auto bound = [&](const Vec8<BF16>& y) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mn.v[i] = min2_nan<BF16>(mn.v[i], y.v[i]);
      mx.v[i] = max2_nan<BF16>(mx.v[i], y.v[i]);
    }
  };

  // (min, -max) of a row's group in one word; NaN wins every comparison
  auto extremes = [&](const Vec8<BF16>& x) {
    T2 lo = min2_nan<BF16>(min2_nan<BF16>(x.v[0], x.v[1]), min2_nan<BF16>(x.v[2], x.v[3]));
    T2 hi = max2_nan<BF16>(max2_nan<BF16>(x.v[0], x.v[1]), max2_nan<BF16>(x.v[2], x.v[3]));
    T2 m;
    m.x = __hmin_nan(lo.x, lo.y);
    m.y = __hneg(__hmax_nan(hi.x, hi.y));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      uint32_t w = *reinterpret_cast<uint32_t*>(&m);
      w = __shfl_xor_sync(0xffffffffu, w, o);
      m = min2_nan<BF16>(m, *reinterpret_cast<T2*>(&w));
    }
    return m;
  };
  uint32_t* params = reinterpret_cast<uint32_t*>(blk + 2 * page_size * ROW);
  // This lane's row of the next iteration; one behind the last keeps its values,
  // so that the shuffles stay whole.
  Vec8<BF16> next[2];
  {
    const long long t = t0 + (s0 + r < s1 ? s0 + r : s0);
    kp += t * ks.t;
    vp += t * vs.t;
    *reinterpret_cast<uint4*>(&next[0]) = *reinterpret_cast<const uint4*>(kp);
    *reinterpret_cast<uint4*>(&next[1]) = *reinterpret_cast<const uint4*>(vp);
  }
  const long long k_step = RPI * ks.t, v_step = RPI * vs.t;
  uint8_t* row = blk + (s0 + r) * ROW + c * (ROW / LPR);
  uint32_t* par = params + ((c & 4 ? page_size : 0) + s0 + r) * NG + grp;
  for (int s = s0 + r; s - r < s1; s += RPI) {
    const bool live = s < s1;
    const Vec8<BF16> x[2] = {next[0], next[1]};
    kp += k_step;
    vp += v_step;
    if (s + RPI < s1) {  // ahead of this row's arithmetic
      *reinterpret_cast<uint4*>(&next[0]) = *reinterpret_cast<const uint4*>(kp);
      *reinterpret_cast<uint4*>(&next[1]) = *reinterpret_cast<const uint4*>(vp);
    }
    // The steps of K and V are worked out side by side: K's by the lower four
    // lanes of a group, V's by the upper four.
    const T2 ext[2] = {extremes(x[0]), extremes(x[1])};
    const bool upper = c & 4;
    const float2 e = Elem<BF16>::unpack(upper ? ext[1] : ext[0]);
    float low = e.x, step;
    bool down = false;
    if (finite(e.x) && finite(e.y)) step = group_step<BF16, BITS>(e.x, -e.y, down);
    else low = step = __int_as_float(0x7fc00000);  // a NaN or infinity: the group reads as NaN
    const bool clamp = __any_sync(0xffffffffu, down);  // values next to the dtype's largest
    const float inv = step_inverse(step);
    const float other = __shfl_xor_sync(0xffffffffu, inv, 4);
    // lane 0 of a group writes K's pair, lane 4 V's
    if (live && (c & 3) == 0) *par = pack2_u32<BF16>(step, low);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const float iv = upper == (side == 1) ? inv : other;
      const float lo = Elem<BF16>::unpack(ext[side]).x;
      uint2 w = clamp ? encode8<BF16, BITS, true>(x[side], lo, iv)
                      : encode8<BF16, BITS, false>(x[side], lo, iv);
      if (iv == 0.f) w = make_uint2(0u, 0u);  // no step, or none that is a number
      if (live) {
        uint8_t* dst = row + (side ? page_size * ROW : 0);
        if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(dst) = w.x;
        else *reinterpret_cast<uint2*>(dst) = w;
      }
      if (side == 0 && index != nullptr) {
        const float k_step = __shfl_sync(0xffffffffu, step, lane & ~4);
        bound(decode8<BF16, BITS>(w, k_step, __shfl_sync(0xffffffffu, low, lane & ~4)));
      }
    }
    row += RPI * ROW;
    par += RPI * NG;
  }
  if (index == nullptr) return;
  // the keys already in the page
  for (int s = 0; s < s0; s += RPI) {
    const int slot = min(s + r, s0 - 1);
    const uint8_t* old = blk + (size_t)slot * ROW;
    uint2 w = make_uint2(0u, 0u);
    if constexpr (BITS == 4) w.x = reinterpret_cast<const uint32_t*>(old)[c];
    else w = reinterpret_cast<const uint2*>(old)[c];
    const float2 p = param<BF16>(
        reinterpret_cast<const uint32_t*>(blk + 2 * page_size * ROW)[slot * NG + grp]);
    bound(decode8<BF16, BITS>(w, p.x, p.y));
  }
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&mn.v[i]), o);
      mn.v[i] = min2_nan<BF16>(mn.v[i], *reinterpret_cast<T2*>(&w));
      w = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&mx.v[i]), o);
      mx.v[i] = max2_nan<BF16>(mx.v[i], *reinterpret_cast<T2*>(&w));
    }
  }
  float top = 0.f;
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = Elem<BF16>::unpack(mn.v[i]), z = Elem<BF16>::unpack(mx.v[i]);
    ok = ok && finite(a.x) && finite(a.y) && finite(z.x) && finite(z.y);
    top = fmaxf(top, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(z.x), fabsf(z.y))));
  }
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float scale = __all_sync(0xffffffffu, ok) ? scale127(top) : __int_as_float(0x7fc00000);
  const float inv = __frcp_rn(scale);
  if (lane < LPR) {
    uint32_t cn[2] = {0u, 0u}, cx[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = Elem<BF16>::unpack(mn.v[i]), z = Elem<BF16>::unpack(mx.v[i]);
      const int sh = 16 * (i & 1);
      cn[i / 2] |= ((code127(a.x, scale, inv) & 255u) | ((code127(a.y, scale, inv) & 255u) << 8)) << sh;
      cx[i / 2] |= ((code127(z.x, scale, inv) & 255u) | ((code127(z.y, scale, inv) & 255u) << 8)) << sh;
    }
    const size_t row = (size_t)page * Hkv + hkv;
    reinterpret_cast<uint2*>(index + row * 2 * D)[c] = make_uint2(cn[0], cn[1]);
    reinterpret_cast<uint2*>(index + row * 2 * D + D)[c] = make_uint2(cx[0], cx[1]);
    if (lane == 0) index_scale[row] = scale;
  }
}

__global__ void advance_kernel(int32_t* __restrict__ kv_lens, int B, int T) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < B) kv_lens[b] = advanced(kv_lens[b], T);
}

template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(32 * kWarps)
    read_kernel(const uint8_t* data, const int32_t* block_table,
                const int32_t* start, const int32_t* cu,
                void* __restrict__ k_out, void* __restrict__ v_out, int Hkv, int J, int page_shift,
                int max_pages, int num_pages, int total, int max_len) {
  using T1 = typename Elem<BF16>::T;
  constexpr int LPR = D / 8, RPI = 32 / LPR, ROW = row_bytes(D, BITS), NG = D / kGroup;
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 31;
  // neighbouring warps write neighbouring heads of the same tokens
  const int unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int hkv = unit % Hkv, j = unit / Hkv;
  const int page_size = 1 << page_shift;
  pdl_trigger();
  if (j >= J) return;
  pdl_wait();
  const int r0 = cu[b], r1 = cu[b + 1];
  const int from = start != nullptr ? start[b] : 0;
  if (r0 < 0 || r1 < r0 || r1 > total || r1 - r0 > max_len || from < 0) {
    if (lane == 0) atomicOr(&g_error_flags, 8u);  // bad cu_seqlens, start or max_len: not read
    return;
  }
  const long long end = (long long)from + (r1 - r0);
  const long long pidx = (from >> page_shift) + (long long)j;
  const long long first = pidx << page_shift;
  if (first >= end) return;
  int page = pidx < max_pages ? block_table[(size_t)b * max_pages + pidx] : -1;
  const bool have = page >= 0 && page < num_pages;
  if (!have) {
    if (lane == 0) atomicOr(&g_error_flags, 2u);  // no such page: its rows read as zero
    page = 0;
  }
  const int s0 = (int)max(0ll, from - first);
  const int s1 = (int)min((long long)page_size, end - first);
  const uint8_t* blk = data + ((size_t)page * Hkv + hkv) * block_bytes(D, page_size, BITS);
  const int r = lane / LPR, c = lane % LPR;
  // U rows of K and of V are in flight at a time: one at a time the loads' latency
  // bounds the copy (709 MB read and written: 157 us).  Rows outside [s0, s1) lie
  // in the same block: they are read and not written.
  constexpr int U = 4, STEP = RPI * U;  // divides every page size
  using Code = typename std::conditional<BITS == 4, uint32_t, uint2>::type;
  const int sb = s0 / STEP * STEP + r;
  const uint8_t* kc = blk + sb * ROW + c * sizeof(Code);
  const uint8_t* kp = blk + 2 * page_size * ROW + (sb * NG + c / 8) * 4;
  const uint32_t v_codes = page_size * ROW, v_params = page_size * NG * 4;
  const long long stride = (long long)RPI * Hkv * D;
  long long out = ((r0 + (first - from) + sb) * Hkv + hkv) * D + 8 * c;
  for (int s = sb; s - r < s1; s += STEP) {
    uint2 w[U][2];
    uint32_t p[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        *reinterpret_cast<Code*>(&w[u][side]) =
            *reinterpret_cast<const Code*>(kc + u * RPI * ROW + (side ? v_codes : 0u));
        p[u][side] = *reinterpret_cast<const uint32_t*>(kp + u * RPI * NG * 4 + (side ? v_params : 0u));
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = s + u * RPI;
      if (row >= s0 && row < s1) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const float2 f = param<BF16>(p[u][side]);
          Vec8<BF16> y = decode8<BF16, BITS>(w[u][side], f.x, f.y);
          if (!have) *reinterpret_cast<uint4*>(&y) = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(static_cast<T1*>(side == 0 ? k_out : v_out) + out) =
              *reinterpret_cast<uint4*>(&y);
        }
      }
      out += stride;
    }
    kc += STEP * ROW;
    kp += STEP * NG * 4;
  }
}

}  // namespace kvq

B2A_DEFINE_ERROR_READER(kvquant)

int kvq_append_dispatch(const void* k_new, const void* v_new, const int64_t* k_strides,
                        const int64_t* v_strides, void* data, int8_t* index, float* index_scale,
                        const int32_t* block_table, int32_t* kv_lens, int B, int Hkv, int T, int D,
                        int page_size, int max_pages, int num_pages, int bits, int dtype,
                        int advance, cudaStream_t stream) {
  using namespace kvq;
  const long long J = ((long long)T + page_size - 2) / page_size + 1;  // pages a run of T may touch
  const long long units = J * Hkv;
  // Few units (a decode step's token): one CTA per sequence, which can then
  // move the length itself.
  const bool one = units <= 16;
  const int warps = one ? (int)units : kWarps;
  const dim3 grid(one ? 1u : (unsigned)((J + kWarps - 1) / kWarps), one ? 1u : (unsigned)Hkv,
                  (unsigned)B);
  const int shift = page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
  const NewRows ks{k_strides[0], k_strides[1], k_strides[2]};
  const NewRows vs{v_strides[0], v_strides[1], v_strides[2]};
  auto go = [&](auto kern) {
    return launch_pdl(kern, grid, 32 * warps, 0, stream, k_new, v_new, ks, vs,
                      static_cast<uint8_t*>(data), index, index_scale, block_table, kv_lens, Hkv,
                      T, (int)J, shift, max_pages, num_pages, (int)one, (int)(advance && one));
  };
  const bool bf = dtype == B2A_BF16;
  cudaError_t e;
  if (D == 64 && bits == 4) e = bf ? go(append_kernel<64, 4, true>) : go(append_kernel<64, 4, false>);
  else if (D == 64) e = bf ? go(append_kernel<64, 8, true>) : go(append_kernel<64, 8, false>);
  else if (bits == 4) e = bf ? go(append_kernel<128, 4, true>) : go(append_kernel<128, 4, false>);
  else e = bf ? go(append_kernel<128, 8, true>) : go(append_kernel<128, 8, false>);
  if (e != cudaSuccess) return set_cuda_error(e, "quantised kv append launch");
  if (advance && !one) {
    e = launch_pdl(advance_kernel, dim3((B + 255) / 256), 256, 0, stream, kv_lens, B, T);
    if (e != cudaSuccess) return set_cuda_error(e, "kv length update launch");
  }
  return B2A_OK;
}

int kvq_read_dispatch(const void* data, const int32_t* block_table, const int32_t* start,
                      const int32_t* cu, void* k_out, void* v_out, int B, int Hkv, int D,
                      int page_size, int max_pages, int num_pages, int total, int max_len,
                      int bits, int dtype, cudaStream_t stream) {
  using namespace kvq;
  // No sequence has more rows than there are, however loose a bound max_len is.
  const long long longest = max_len < total ? max_len : total;
  const long long J = (longest + page_size - 2) / page_size + 1;
  if (J * Hkv > 0x7fffff00ll)  // a warp's unit is an int
    return set_error(B2A_ERR_INVALID_ARG, "total and max_len too large");
  const long long gx = (J * Hkv + kWarps - 1) / kWarps;
  const dim3 grid((unsigned)gx, (unsigned)B);
  const int shift = page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
  auto go = [&](auto kern) {
    return launch_pdl(kern, grid, 32 * kWarps, 0, stream, static_cast<const uint8_t*>(data),
                      block_table, start, cu, k_out, v_out, Hkv, (int)J, shift, max_pages,
                      num_pages, total, max_len);
  };
  const bool bf = dtype == B2A_BF16;
  cudaError_t e;
  if (D == 64 && bits == 4) e = bf ? go(read_kernel<64, 4, true>) : go(read_kernel<64, 4, false>);
  else if (D == 64) e = bf ? go(read_kernel<64, 8, true>) : go(read_kernel<64, 8, false>);
  else if (bits == 4) e = bf ? go(read_kernel<128, 4, true>) : go(read_kernel<128, 4, false>);
  else e = bf ? go(read_kernel<128, 8, true>) : go(read_kernel<128, 8, false>);
  if (e != cudaSuccess) return set_cuda_error(e, "quantised kv read launch");
  return B2A_OK;
}

}  // namespace b2a

// kvquant.cuh -- the format of the quantised paged KV cache, shared by its
// write / read-back kernels (kvquant_sm100.cu) and its attention
// (kvquant_decode_sm100.cu).
//
// The block of one (page, KV head) is one contiguous piece of memory,
//   [K codes | V codes | K params | V params],
// so that a bulk copy fetches everything attention needs of a page at once.
// Codes are token-major rows of D*bits/8 bytes, low nibble first at 4 bits.
// Params hold one (scale, min) pair in the cache's dtype per token and group
// of kGroup channels; a code c stands for scale*c + min.
#pragma once
#include "sm100_ptx.cuh"

namespace b2a {
namespace kvq {

constexpr int kFusedPages = 2048;  // tables up to this width are selected from in one launch
constexpr int kGroup = 64;  // channels sharing one (scale, min): 4.5 / 8.5 bits an element
// Steps below this are stored as 0 (the group reads back as its min), so that
// the reciprocal of a step is always a finite fp32.
constexpr float kTinyStep = 7.8886090522101181e-31f;  // 2^-100

__host__ __device__ constexpr int row_bytes(int D, int bits) { return D * bits / 8; }
__host__ __device__ constexpr int block_bytes(int D, int page, int bits) {
  return 2 * page * (row_bytes(D, bits) + D / kGroup * 4);
}

// Programmatic dependent launch: a kernel lets the next one on its stream start
// as soon as all its own blocks run (pdl_trigger), and a kernel that was started
// so waits for the one before it, and its memory, before it touches any
// (pdl_wait).  Only the launch itself overlaps; after a foreign kernel both do
// nothing.  A kernel may thus be alive while the one before writes what it will
// read: no pointer that it reads through is both const and __restrict__, which would
// promise memory that nobody writes while the kernel lives, and let loads of it
// pass the wait.
__device__ __forceinline__ void pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
inline cudaError_t launch_pdl(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem,
                              cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

// 8 consecutive values of a row as four packed pairs.
template <bool BF16>
struct Vec8 {
  typename Elem<BF16>::T2 v[4];
};

template <bool BF16>
__device__ __forceinline__ typename Elem<BF16>::T2 min2_nan(typename Elem<BF16>::T2 a,
                                                            typename Elem<BF16>::T2 b) {
  return __hmin2_nan(a, b);
}
template <bool BF16>
__device__ __forceinline__ typename Elem<BF16>::T2 max2_nan(typename Elem<BF16>::T2 a,
                                                            typename Elem<BF16>::T2 b) {
  return __hmax2_nan(a, b);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// fp32 x >= 0 -> dtype with directed rounding, back in fp32
template <bool BF16>
__device__ __forceinline__ float round_up(float x) {
  if constexpr (BF16) {
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float((u + 0xffffu) & 0xffff0000u);
  } else {
    return __half2float(__float2half_ru(x));
  }
}
template <bool BF16>
__device__ __forceinline__ float round_down(float x) {
  if constexpr (BF16) return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  else return __half2float(__float2half_rd(x));
}

// The step of a group with extremes lo, hi (both finite) and n = 2^bits - 1:
// (hi - lo) / n rounded up to dtype, so that n steps from lo reach hi; rounded
// down where lo + n*step would leave the dtype's range.  Halves keep hi - lo
// finite for any finite bf16.  Explicit roundings: the result is specified to
// the bit.  `down` says that it was rounded down.
template <bool BF16, int BITS>
__device__ __forceinline__ float group_step(float lo, float hi, bool& down) {
  constexpr float n = (float)((1 << BITS) - 1);
  const float want = __fmul_rn(__fsub_rn(0.5f * hi, 0.5f * lo), 2.0f / n);
  // the least fp32 that rounds to infinity: max + half a last place
  constexpr float kPast = BF16 ? 3.3961775292304601e38f : 65520.f;
  float s = round_up<BF16>(want);
  down = __fmaf_rn(n, s, lo) >= kPast;
  if (down) s = round_down<BF16>(want);
  return s < kTinyStep ? 0.f : s;
}

// Reciprocal of half a step (0 for a step of 0 or NaN: codes 0).
__device__ __forceinline__ float step_inverse(float step) {
  return step > 0.f ? __frcp_rn(0.5f * step) : 0.f;
}

// Codes of 8 finite values of a group, min(rint((x/2 - lo/2) * inv), n): one
// word at 4 bits, two at 8.  Adding 2^23 leaves the value, rounded to nearest
// even, in the low mantissa bits.  Only a step that was rounded down needs the
// minimum (CLAMP): any other is at least (hi - lo)/n less the 2^-22 of three fp32
// roundings, so that the product is at most n (1 + 2^-21) and rounds to n.
template <bool BF16, int BITS, bool CLAMP>
__device__ __forceinline__ uint2 encode8(const Vec8<BF16>& x, float lo, float inv) {
  constexpr float n = (float)((1 << BITS) - 1);
  const float lo2 = 0.5f * lo;
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // x/2 is exact, so the fused form rounds once as the difference does
    float2 f = ffma2(Elem<BF16>::unpack(x.v[i]), make_float2(0.5f, 0.5f), make_float2(-lo2, -lo2));
    f = fmul2(f, make_float2(inv, inv));
    if constexpr (CLAMP) f = make_float2(fminf(f.x, n), fminf(f.y, n));
    // not as a pair: the product and the sum would be fused, which rounds once
    c[2 * i] = __float_as_uint(__fadd_rn(f.x, 8388608.f));
    c[2 * i + 1] = __float_as_uint(__fadd_rn(f.y, 8388608.f));
  }
  uint2 w = make_uint2(0u, 0u);
  if constexpr (BITS == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = c[2 * i] + (c[2 * i + 1] << 4);  // a byte, rest unused
    w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  } else {
    w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    w.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  }
  return w;
}

// The values that 8 codes stand for: one fused multiply-add in fp32, rounded
// once to dtype.  A code becomes a float by placing its byte in 2^23 (int to
// float conversions run at a quarter of the rate).
template <bool BF16, int BITS>
__device__ __forceinline__ Vec8<BF16> decode8(uint2 w, float step, float lo) {
  Vec8<BF16> r;
  const uint32_t even = w.x & 0x0f0f0f0fu, odd = (w.x >> 4) & 0x0f0f0f0fu;  // 4 bits
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t c0, c1;
    if constexpr (BITS == 4) {
      c0 = __byte_perm(even, 0x4b000000u, 0x7550 + i);
      c1 = __byte_perm(odd, 0x4b000000u, 0x7550 + i);
    } else {
      const uint32_t x = i < 2 ? w.x : w.y;
      c0 = __byte_perm(x, 0x4b000000u, i & 1 ? 0x7552 : 0x7550);
      c1 = __byte_perm(x, 0x4b000000u, i & 1 ? 0x7553 : 0x7551);
    }
    r.v[i] = Elem<BF16>::pack(
        __fmaf_rn(__fadd_rn(__uint_as_float(c0), -8388608.f), step, lo),
        __fmaf_rn(__fadd_rn(__uint_as_float(c1), -8388608.f), step, lo));
  }
  return r;
}

// a (scale, min) pair of the cache's dtype in fp32
template <bool BF16>
__device__ __forceinline__ float2 param(uint32_t raw) {
  typename Elem<BF16>::T2 h;
  *reinterpret_cast<uint32_t*>(&h) = raw;
  return Elem<BF16>::unpack(h);
}

// A signed 8-bit scale for values of magnitude up to `top`: NaN when top is
// not finite; codes are 0 where it is below kTinyStep.
__device__ __forceinline__ float scale127(float top) {
  return finite(top) ? __fmul_rn(top, 1.0f / 127.0f) : __int_as_float(0x7fc00000);
}
__device__ __forceinline__ int code127(float v, float scale, float inv) {
  if (!(scale >= kTinyStep)) return 0;
  return __float2int_rn(fminf(fmaxf(__fmul_rn(v, inv), -127.f), 127.f));
}

}  // namespace kvq
}  // namespace b2a

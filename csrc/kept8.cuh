// The 8-bit kept-activation format and the row views its kernels read and write.
//
// A row of C values is cut into blocks of 32 consecutive channels (the last may be short).  A block is
// held as one scale byte b and 32 signed codes:
//
//   b = clamp(floor(log2(max |x|)) + 127, 7, 254),  step = 2^(b - 133),  code = clamp(rne(x / step), -127, 127)
//
// i.e. the OCP microscaling MXINT8 layout (shared power-of-two scale, 6 fraction bits) with the scale
// kept in the range where the step and every value code * step are normal fp32 / bf16 numbers.  Why a
// power of two: x / step and code * step are exact, so the codes do not depend on the order or the
// precision of the arithmetic, and a value (7 bits times a power of two) fits bf16's 8-bit significand
// without a second rounding: it can feed a bf16 tensor-core operand as it is.  The error is at most half a step
// (one step where an fp32 value above 127.5 steps is clamped); on normally distributed blocks it is 0.5-1 % of
// the block's RMS.  A block that holds an Inf or a NaN gets b = 255 and reads back as NaN: a
// non-finite activation shows in the gradients instead of being stored as a number.
//
// Storage: codes [rows, Cp] int8 with Cp = C rounded up to 32 (16-byte aligned rows), scales
// [rows, nbp] uint8 with nbp = Cp / 32 rounded up to 4; padding codes are 0, padding scale bytes 127.
#pragma once

#include "common.cuh"

namespace pan {

constexpr int kKeptBlock = 32;
constexpr uint32_t kKeptPadByte = 127;

// n / d for n < 2^31 by a multiply and a shift (Granlund and Montgomery, "Division by invariant
// integers using multiplication", 1994).
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

// Rows of a [rows, C] view whose leading dimensions are at most two strided levels:
// row r starts at p + (r / inner) * outer_stride + (r % inner) * inner_stride (elements).
struct RowView {
  const void* p;
  long long outer_stride, inner_stride;
  FastDiv inner;
};

template <typename T>
__device__ __forceinline__ const T* row_ptr(const RowView& v, uint32_t r) {
  const uint32_t o = v.inner.div(r);
  return reinterpret_cast<const T*>(v.p) + (long long)o * v.outer_stride +
         (long long)(r - o * v.inner.d) * v.inner_stride;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements as fp32: V = 8 by 16-byte accesses, V = 1 by one element.
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else if constexpr (sizeof(T) == 2) {
    load8(p, v);
  } else {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 2) {
    store8(p, v);
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// ---------------------------------------------------------------- codes
// Scale byte from the bits of max |x|.  NaN has the largest bits, then Inf: both give 255.
__device__ __forceinline__ uint32_t kept8_byte(uint32_t amax_bits) { return max(amax_bits >> 23, 7u); }
// 1 / step of a finite block (b = 255 gives some finite number; its codes are never read as values).
__device__ __forceinline__ float kept8_inv_step(uint32_t b) { return __uint_as_float((260u - b) << 23); }
__device__ __forceinline__ float kept8_step(uint32_t b) {
  return b == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float((b - 6u) << 23);
}

// Bits whose low byte is the code of x: adding 1.5 * 2^23 rounds x * inv (exact) to a whole number,
// half to even, and leaves it in two's complement in the low mantissa bits.  A NaN clamps to a number.
__device__ __forceinline__ uint32_t kept8_code(float x, float inv) {
  const float magic = 12582912.f;
  return __float_as_uint(fminf(fmaxf(fmaf(x, inv, magic), magic - 127.f), magic + 127.f));
}

// Largest |x| bits over the 32 / V lanes that hold one block (V = 8: four lanes, V = 1: the warp).
// Every lane of the warp takes part.
template <int V>
__device__ __forceinline__ uint32_t kept8_amax(const float (&v)[V]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  if constexpr (V == 1) {
    m = __reduce_max_sync(0xffffffffu, m);
  } else {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  }
  return m;
}

__device__ __forceinline__ uint32_t pack4_low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <int V>
__device__ __forceinline__ void kept8_store_codes(int8_t* p, const float (&v)[V], uint32_t b) {
  const float inv = kept8_inv_step(b);
  if constexpr (V == 1) {
    *p = (int8_t)(kept8_code(v[0], inv) & 0xffu);
  } else {
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = kept8_code(v[i], inv);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(pack4_low_bytes(c[0], c[1], c[2], c[3]), pack4_low_bytes(c[4], c[5], c[6], c[7]));
  }
}

// Eight codes times their step.
__device__ __forceinline__ void kept8_values(uint2 w, float step, float (&v)[8]) {
  // byte k as an unsigned offset code in the mantissa of 2^23: 2^23 + (code + 128), exactly
  const uint32_t u0 = w.x ^ 0x80808080u, u1 = w.y ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (__uint_as_float(__byte_perm(u0, 0x4b000000u, 0x7540 + i)) - 8388736.f) * step;
    v[4 + i] = (__uint_as_float(__byte_perm(u1, 0x4b000000u, 0x7540 + i)) - 8388736.f) * step;
  }
}

// V codes from `p` times the step of scale byte b.
template <int V>
__device__ __forceinline__ void kept8_load(const int8_t* p, uint32_t b, float (&v)[V]) {
  const float step = kept8_step(b);
  if constexpr (V == 1) v[0] = (float)*p * step;
  else kept8_values(*reinterpret_cast<const uint2*>(p), step, v);
}

// Scale byte of block `blk` of a row; the block's writer also fills the row's padding bytes.
__device__ __forceinline__ void kept8_store_byte(uint8_t* row_scales, int blk, int nb, int nbp, uint32_t b) {
  row_scales[blk] = (uint8_t)b;
  if (blk == nb - 1)
    for (int i = nb; i < nbp; ++i) row_scales[i] = (uint8_t)kKeptPadByte;
}

}  // namespace pan

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

// ---------------------------------------------------------------- packed fp32 pairs
// Two fp32 operations an instruction: these kernels are as often bound by instruction issue as by DRAM.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mov.b64 rc, {%6, %7};\n\tfma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// Eight consecutive elements as they lie in memory, and as fp32 pairs.
template <typename T>
struct Frag;
template <>
struct Frag<__nv_bfloat16> {
  uint4 raw;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  }
};
template <>
struct Frag<float> {
  float4 raw[2];
  __device__ __forceinline__ void load(const float* p) {
    raw[0] = reinterpret_cast<const float4*>(p)[0];
    raw[1] = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { raw[0] = raw[1] = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    v[0] = make_float2(raw[0].x, raw[0].y);
    v[1] = make_float2(raw[0].z, raw[0].w);
    v[2] = make_float2(raw[1].x, raw[1].y);
    v[3] = make_float2(raw[1].z, raw[1].w);
  }
};

__device__ __forceinline__ void store_pairs(__nv_bfloat16* p, const float2 (&v)[4]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y),
                                            pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
}
__device__ __forceinline__ void store_pairs(float* p, const float2 (&v)[4]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
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

__device__ __forceinline__ void kept8_store_code(int8_t* p, float v, uint32_t b) {
  *p = (int8_t)(kept8_code(v, kept8_inv_step(b)) & 0xffu);
}

// Eight codes as numbers.
__device__ __forceinline__ void kept8_numbers(uint2 w, float2 (&v)[4]) {
  // byte k as an unsigned offset code in the mantissa of 2^23: 2^23 + (code + 128), exactly
  const uint32_t u[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 m = make_float2(__uint_as_float(__byte_perm(u[i / 2], 0x4b000000u, 0x7540 + i % 2 * 2)),
                                 __uint_as_float(__byte_perm(u[i / 2], 0x4b000000u, 0x7541 + i % 2 * 2)));
    v[i] = add2(m, twice(-8388736.f));
  }
}
__device__ __forceinline__ float kept8_number(int8_t code) {
  return __uint_as_float(((uint8_t)code ^ 0x80u) | 0x4b000000u) - 8388736.f;
}
// ... times their step.
__device__ __forceinline__ void kept8_values(uint2 w, float step, float2 (&v)[4]) {
  kept8_numbers(w, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], twice(step));
}
__device__ __forceinline__ void kept8_values(uint2 w, float step, float (&v)[8]) {
  float2 p[4];
  kept8_values(w, step, p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = p[i].x, v[2 * i + 1] = p[i].y;
}

// Scale byte and codes of a fragment whose block is held by four neighbouring lanes; every lane of the
// warp takes part.
__device__ __forceinline__ void kept8_encode(const Frag<float>& f, uint32_t& b, uint2& codes) {
  const float v[8] = {f.raw[0].x, f.raw[0].y, f.raw[0].z, f.raw[0].w, f.raw[1].x, f.raw[1].y, f.raw[1].z, f.raw[1].w};
  b = kept8_byte(kept8_amax<8>(v));
  const float inv = kept8_inv_step(b);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = kept8_code(v[i], inv);
  codes = make_uint2(pack4_low_bytes(c[0], c[1], c[2], c[3]), pack4_low_bytes(c[4], c[5], c[6], c[7]));
}

// In bf16 pairs: |x| is clamped to 127 steps, and one fused multiply-add |x| / step + 128 rounds it half to
// even to a whole number whose low seven mantissa bits are the magnitude (128 .. 255 has a unit of 1 in
// bf16).  Four magnitudes a word then take their signs as bytes: -m = (0x80 - m) ^ 0x80 without borrows.
__device__ __forceinline__ void kept8_encode(const Frag<__nv_bfloat16>& f, uint32_t& b, uint2& codes) {
  const uint32_t w[4] = {f.raw.x, f.raw.y, f.raw.z, f.raw.w};
  uint32_t a[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = w[i] & 0x7fff7fffu;
  uint32_t m = __vmaxu2(__vmaxu2(a[0], a[1]), __vmaxu2(a[2], a[3]));
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
  b = max(max(m & 0xffffu, m >> 16) >> 7, 7u);
  const uint32_t lim = ((b << 7) | 0x7eu) * 0x10001u;  // 127 steps
  const uint32_t inv = ((260u - b) << 7) * 0x10001u;
  uint32_t z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b32 t;\n\tmin.bf16x2 t, %1, %2;\n\tfma.rn.bf16x2 %0, t, %3, %4;\n\t}"
        : "=r"(z[i]) : "r"(a[i]), "r"(lim), "r"(inv), "r"(0x43004300u));
  uint32_t c[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t mag = __byte_perm(z[2 * i], z[2 * i + 1], 0x6420);
    uint32_t neg;  // 0xff where the element's sign bit is set
    asm("prmt.b32 %0, %1, %2, 0xfdb9;" : "=r"(neg) : "r"(w[2 * i]), "r"(w[2 * i + 1]));
    c[i] = ((0x80808080u - (mag & neg)) ^ 0x80808080u) | (mag & ~neg);
  }
  codes = make_uint2(c[0], c[1]);
}

// Scale byte of block `blk` of a row; the block's writer also fills the row's padding bytes.
__device__ __forceinline__ void kept8_store_byte(uint8_t* row_scales, int blk, int nb, int nbp, uint32_t b) {
  row_scales[blk] = (uint8_t)b;
  if (blk == nb - 1)
    for (int i = nb; i < nbp; ++i) row_scales[i] = (uint8_t)kKeptPadByte;
}

}  // namespace pan

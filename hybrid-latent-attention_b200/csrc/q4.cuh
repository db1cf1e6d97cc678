// The 4-bit format shared by the latent cache (q4_history.cu, q4_rows.cu) and the weights (q4_linear.cu).
//
// A group of 32 consecutive columns of a row shares one e4m3 scale s; a value is (n - 8) * s * ts with the
// code n in 1..15 and one tensor scale ts.  (n - 8) * s has at most 3 + 4 significant bits, so it is exact
// in bf16 (8 bits): the kernels feed the tensor cores bf16 values without a rounding, and ts is applied to
// the fp32 accumulators.  Codes travel in 32-bit words of 8 columns, nibble i column 2i and nibble i + 4
// column 2i + 1: one shift and one and-or leave two neighbouring columns in the two halves of a register.
//
// A latent cache page is page / 16 tiles of 16 rows, 17 W bytes each (W = latent width, G = W / 32 groups):
//   K codes  [G][16 rows][16 B]    a row's group is one 16-byte chunk
//   V codes  [W / 8][16 rows][4 B] the rows of 8 columns side by side: V is contracted over rows
//   K scales [16 rows][G]   V scales [G][16 rows]
// Every byte belongs to one row, so rows are committed independently of one another.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace hla {

constexpr int kQ4Group = 32;  // columns that share a scale
constexpr uint32_t kQ4ScaleNaN = 0x7f;         // e4m3's NaN: the scale of a group that holds one
constexpr uint32_t kQ4Zeros = 0x88888888u;     // a word of codes 8

// A packed weight [N, K] is [N / 16][K / 128] tiles (zero padded) of 16 rows x 128 columns: codes
// [2][32 lanes][16 B], scales [32 lanes][2], lane 4 g + c and half h holding row 8 h + g, columns 32 c .. -
// the A fragment of mma.m16n8k16 read straight from global memory, one 16-byte load per half.
constexpr int kQ4WeightTile = 1088;

struct Q4Tile {  // byte offsets inside a 16-row tile of latent width W
  int W;
  __host__ __device__ explicit Q4Tile(int w) : W(w) {}
  __host__ __device__ int bytes() const { return 17 * W; }
  __host__ __device__ int k_codes(int group, int row) const { return group * 256 + row * 16; }
  __host__ __device__ int v_codes(int octet, int row) const { return 8 * W + octet * 64 + row * 4; }
  __host__ __device__ int k_scale(int row, int group) const { return 16 * W + row * (W / kQ4Group) + group; }
  __host__ __device__ int v_scale(int group, int row) const { return 16 * W + W / 2 + group * 16 + row; }
};

// (x & mask) | bits in one instruction (written in C it becomes two: both constants are immediates).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(bits));
  return d;
}
__device__ __forceinline__ uint32_t bf2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// The largest value, or NaN where one is NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two e4m3 bytes (low 16 bits of v) -> bf16x2 (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_bf2(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v), __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  return pack_bf16(f.x, f.y);
}

// A scale pair as the dequantiser wants it: s and -24 s.
struct Q4Scale {
  uint32_t s, c;
  __device__ __forceinline__ explicit Q4Scale(uint32_t s2) : s(s2), c(bf2_mul(s2, 0xc1c0c1c0u)) {}  // -24
};

// (n - 8) * s of nibbles i and i + 4 of a word: the nibbles moved to bits 3..6 of each half are the top
// mantissa bits of a bf16 in [16, 32), i.e. 16 + n, and (16 + n) s - 24 s = (n - 8) s, exact at every
// step (24 s has 6 significant bits).
template <int I>
__device__ __forceinline__ uint32_t q4_pair(uint32_t w, const Q4Scale& s) {
  const uint32_t sh = I == 0 ? w << 3 : w >> (4 * I - 3);
  return bf2_fma(and_or(sh, 0x00780078u, 0x41804180u), s.s, s.c);
}

// The same in fp16, which needs one shift and two multiplications by 16 for the four pairs of a word instead of
// four shifts: a nibble at bits 4..7 of a half under the exponent of 64 is 64 + n, and (64 + n) s - 72 s =
// (n - 8) s (72 s has 8 significant bits, 72 * 448 < 65504: exact).
struct Q4ScaleH {
  uint32_t s, c;
};
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t v) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(static_cast<uint16_t>(v)));
  return d;
}
__device__ __forceinline__ Q4ScaleH q4_scale_h(uint32_t s2) { return Q4ScaleH{s2, h2_mul(s2, 0xd480d480u)}; }  // -72
// Scales of two groups (bytes b0 | b1 << 8), each for both halves of a pair.
__device__ __forceinline__ void q4_scales_h(uint32_t bytes, Q4ScaleH& a, Q4ScaleH& b) {
  const Q4ScaleH p = q4_scale_h(e4m3x2_to_h2(bytes));
  a = Q4ScaleH{__byte_perm(p.s, 0, 0x1010), __byte_perm(p.c, 0, 0x1010)};
  b = Q4ScaleH{__byte_perm(p.s, 0, 0x3232), __byte_perm(p.c, 0, 0x3232)};
}
// The four pairs of a word: r[i] = columns 2i, 2i + 1 (or rows, where the halves of w come from two rows).
// `sixteen` is 16 in a value the compiler cannot see through: the two shifts to the left then run as
// multiplications beside the HFMA2s, while shifts, ANDs and byte permutes all share the other pipe (2 clocks an
// instruction each; 5 + 6 a word instead of 7 + 4).
__device__ __forceinline__ void q4_word_h(uint32_t w, const Q4ScaleH& s, uint32_t sixteen, uint32_t& r0, uint32_t& r1,
                                          uint32_t& r2, uint32_t& r3) {
  constexpr uint32_t kMask = 0x00f000f0u, kMagic = 0x54005400u;
  const uint32_t t = w >> 8;
  r0 = h2_fma(and_or(w * sixteen, kMask, kMagic), s.s, s.c);
  r1 = h2_fma(and_or(w, kMask, kMagic), s.s, s.c);
  r2 = h2_fma(and_or(t * sixteen, kMask, kMagic), s.s, s.c);
  r3 = h2_fma(and_or(t, kMask, kMagic), s.s, s.c);
}

// Scale byte of a group: e4m3(amax / (7 ts)), a true division so that ties fall as the format says.
__device__ __forceinline__ uint32_t q4_scale_byte(float amax, float ts) {
  return __nv_cvt_float_to_fp8(__fdiv_rn(amax, 7.f * ts), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float q4_scale_value(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}
// Codes of a group whose step is s * ts: 8 + x / step rounded to nearest, ties to even, clamped to 1..15 (by
// clamping x to 7 steps: |x| / step < 7.5 except where the scale saturated or was rounded in e4m3's subnormal range).
// An infinity takes the group's largest code; a step of 0 gives 8.  (Groups with a NaN take kQ4ScaleNaN and kQ4Zeros.)
// No division: z = x * inv + 1.5 * 2^23 + 8 has the rounded sum in its low bits.  inv = 1 / step is itself rounded, so
// where x / step is (almost) half way z may have gone the wrong way; the remainder x - q step tells: more than half a
// step, or half a step from an odd code, moves the code by one towards it.  (fmaf rounds the remainder once; it is exact
// where ts has up to 17 significant bits: 8 bits minus 3 x 4 x 17.)
struct Q4Coder {
  float step, inv, lim;
  uint32_t half;  // bits of step / 2
  __device__ __forceinline__ explicit Q4Coder(float step_) {
    step = step_;
    inv = step_ > 0.f ? __frcp_rn(step_) : 0.f;
    lim = 7.f * step_;
    half = step_ > 0.f ? __float_as_uint(0.5f * step_) : 0x7f800000u;
  }
  __device__ __forceinline__ uint32_t operator()(float x) const {
    constexpr float kMagic = 12582912.f + 8.f;
    x = fminf(fmaxf(x, -lim), lim);
    const uint32_t z = __float_as_uint(fmaf(x, inv, kMagic));
    const uint32_t r = __float_as_uint(fmaf(kMagic - __uint_as_float(z), step, x));
    const uint32_t towards = static_cast<uint32_t>(static_cast<int32_t>(r) >> 31) | 1u;
    return (z + ((r & 0x7fffffffu) + (z & 1u) > half ? towards : 0u)) & 15u;
  }
};
// The word of 8 columns' codes.
__device__ __forceinline__ uint32_t q4_word(const uint32_t (&n)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= (n[2 * i] << (4 * i)) | (n[2 * i + 1] << (16 + 4 * i));
  return w;
}
// Scale byte and codes of bf16 values for a power-of-two tensor scale (2^-117 .. 2^116: the smallest step, 2^-9 ts, is a
// normal number and 7 of the largest, 448 ts, are finite), without divisions and in 6 instructions a value instead of 16:
// * amax / 7 has at most 5 significant bits where it is half way between two e4m3 numbers, and is otherwise 2^-11 or
//   more away from that, relative; so amax * (1 / 7), right to 2^-23, is rounded to 16 bits and falls as the quotient.
// * a quotient of 8 by 4 significant bits that is not half way between two integers is at least 1/1000 away from that,
//   so x * inv rounds like it for an inv within 2^-20; half way a value below and one above 1 / step give the two
//   integers, of which the even one is (a + b + ((a + b) / 2) % 2) / 2, computed for two columns in a register.
// amax: the group's largest value, which says whether anything has to be clamped (see above).
__device__ __forceinline__ bool q4_pow2(float ts) {
  const uint32_t b = __float_as_uint(ts);
  return (b & 0x7fffffu) == 0 && b - (10u << 23) <= (233u << 23);
}
// Any other (normal) tensor scale: values and scale are multiplied by the power of two that puts the scale into [1, 4),
// which changes no code; steps, reciprocals and remainders then stay among fp32's normal numbers.
__device__ __forceinline__ float q4_norm(float ts) {
  const uint32_t e = __float_as_uint(ts) >> 23;
  return __uint_as_float((254u - (e < 253u ? e : 253u)) << 23);
}
__device__ __forceinline__ uint32_t q4_scale_byte_pow2(float amax, float ts) {
  const float seventh = __uint_as_float(__float_as_uint(1.f / 7.f) + (127u << 23) - __float_as_uint(ts));  // 1 / (7 ts)
  const float q = __uint_as_float((__float_as_uint(amax * seventh) + 0x80u) & 0xffffff00u);
  return __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float rcp_approx(float x) {  // to 1 ulp (0 is infinite)
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t q4_word_pow2(const float (&f)[8], float amax, float step) {
  constexpr float kMagic = 12582912.f + 8.f;
  // a step of 0 (every value below 2^-10 * 7 ts) leaves the codes at 8
  const uint32_t inv = __float_as_uint(rcp_approx(step));
  const float lo = step > 0.f ? __uint_as_float(inv - 2u) : 0.f, hi = step > 0.f ? __uint_as_float(inv + 2u) : 0.f;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = f[i];
  if (!(amax <= 7.4f * step)) {
    const float lim = 7.f * step;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -lim), lim);
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t s[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      s[k] = __float_as_uint(fmaf(x[2 * i + k], lo, kMagic)) + __float_as_uint(fmaf(x[2 * i + k], hi, kMagic));
    uint32_t t = __byte_perm(s[0], s[1], 0x5410);
    t += (t >> 1) & 0x00010001u;
    w |= (i == 0 ? t >> 1 : t << (4 * i - 1)) & (0x000f000fu << (4 * i));
  }
  return w;
}

}  // namespace hla

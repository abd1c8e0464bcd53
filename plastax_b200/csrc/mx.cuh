// Microscaled (MX) values: blocks of 32 that share a power-of-two scale byte
// (E8M0: 2^(byte - 127), 255 = not a number) with codes in e4m3, e5m2 (one
// byte each) or e2m1 (two to a byte, the even element in the low nibble).
//
// Encoding of a block x_0..x_31: the scale is the smallest power of two s >=
// 2^-127 with max|x_i| <= L * s (L the format's largest value, so nothing
// saturates and at most one bit of the range is unused), the code of x_i the
// nearest element to x_i / s, ties to even. The division is a product with
// 2^-e, exact down to where the code is 0 anyway. A block that holds an
// infinity or a NaN gets the scale 255 and reads NaN whole: a partial sum over
// it is then NaN too, as it would be in float32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "pxb_common.cuh"

namespace pxb {

constexpr int kMxBlock = 32;
constexpr int32_t kMxMaxBatch = 1 << 30;  // a row's padded samples stay within 32 bits

// A value's bits as another type of its size.
template <typename To, typename From>
__device__ __forceinline__ To same_bits(const From &v) {
  static_assert(sizeof(To) == sizeof(From), "sizes differ");
  To t;
  memcpy(&t, &v, sizeof(To));
  return t;
}

template <int FMT>
struct MxFormat;
template <>
struct MxFormat<PXB_MX_E4M3> {
  static constexpr int bits = 8, top_exp = 8;
  static constexpr uint32_t top_mant = 0x600000u;  // 448 = 1.75 * 2^8
};
template <>
struct MxFormat<PXB_MX_E5M2> {
  static constexpr int bits = 8, top_exp = 15;
  static constexpr uint32_t top_mant = 0x600000u;  // 57344 = 1.75 * 2^15
};
template <>
struct MxFormat<PXB_MX_E2M1> {
  static constexpr int bits = 4, top_exp = 2;
  static constexpr uint32_t top_mant = 0x400000u;  // 6 = 1.5 * 2^2
};

template <int FMT>
__host__ __device__ constexpr int mx_block_bytes() {
  return kMxBlock * MxFormat<FMT>::bits / 8;
}

__host__ __device__ inline int mx_bits(int fmt) { return fmt == PXB_MX_E2M1 ? 4 : 8; }
__host__ __device__ inline int64_t mx_blocks(int64_t n) { return (n + kMxBlock - 1) / kMxBlock; }

// The value of a scale byte.
__device__ __forceinline__ float mx_scale_value(uint32_t s) {
  // the exponent field; 0 (2^-127, a subnormal) and 255 (not a number) set the same mantissa bit
  return __uint_as_float((s << 23) | (((s + 1) & 0xfeu) == 0 ? 0x00400000u : 0u));
}

// The scale byte of a block whose largest magnitude has these bits.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int e = static_cast<int>(amax_bits >> 23) - MxFormat<FMT>::top_exp +
                ((amax_bits & 0x7fffffu) > MxFormat<FMT>::top_mant ? 1 : 0);
  return static_cast<uint32_t>(e < 0 ? 0 : e);
}

// 2^-e of a scale byte e + 127 (0 for the byte 255, whose codes are all 0).
__device__ __forceinline__ float mx_inverse_scale(uint32_t s) {
  return s == 255u ? 0.0f : __uint_as_float((254u - s) << 23);
}

// Eight consecutive values -> eight codes (8 bytes, or 4 for e2m1), given
// 2^-e. `keep`: a value that is not zero takes at least the smallest
// magnitude of its sign, so its sign survives.
template <int FMT>
__device__ __forceinline__ uint64_t mx_encode8(const float (&x)[8], uint32_t scale, bool keep) {
  if (scale == 255u) return 0;
  const float inv = mx_inverse_scale(scale);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(x[i], inv);
  // Each pair leaves the assembly as a whole register and the pairs are joined
  // here: packed inside it (mov.b32 {a, b}), two pairs of equal values that the
  // compiler had merged came out with an undefined upper half.
  uint32_t lo, hi = 0;
  if constexpr (FMT == PXB_MX_E2M1) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}"
          : "=r"(c[i]) : "f"(y[2 * i]), "f"(y[2 * i + 1]));
    lo = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    if (keep) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (x[i] != 0.0f && (lo & (0x7u << (4 * i))) == 0) lo |= 0x1u << (4 * i);
    }
  } else {
    uint16_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (FMT == PXB_MX_E4M3)
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(c[i]) : "f"(y[2 * i]), "f"(y[2 * i + 1]));
      else
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %2, %1;" : "=h"(c[i]) : "f"(y[2 * i]), "f"(y[2 * i + 1]));
    }
    lo = __byte_perm(c[0], c[1], 0x5410);
    hi = __byte_perm(c[2], c[3], 0x5410);
    if (keep) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (x[i] != 0.0f && (lo & (0x7fu << (8 * i))) == 0) lo |= 0x1u << (8 * i);
        if (x[i + 4] != 0.0f && (hi & (0x7fu << (8 * i))) == 0) hi |= 0x1u << (8 * i);
      }
    }
  }
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// Four bytes of codes (4 in 8 bits, 8 in e2m1) -> pairs of values before the
// scale. Every element is a half; the conversions are the hardware's. For words
// loaded whole (mx_decode2 takes parts of one).
template <int FMT>
__device__ __forceinline__ void mx_decode_word(uint32_t c, __half2 (&h)[32 / (2 * MxFormat<FMT>::bits)]) {
  uint32_t r[32 / (2 * MxFormat<FMT>::bits)];
  if constexpr (FMT == PXB_MX_E2M1)
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(c));
  else if constexpr (FMT == PXB_MX_E4M3)
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(r[0]), "=r"(r[1]) : "r"(c));
  else
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e5m2x2 %0, a;\n\t"
        "cvt.rn.f16x2.e5m2x2 %1, b;\n\t}" : "=r"(r[0]), "=r"(r[1]) : "r"(c));
#pragma unroll
  for (int i = 0; i < 32 / (2 * MxFormat<FMT>::bits); ++i) h[i] = same_bits<__half2>(r[i]);
}

// The two values of e2m1's byte, or of two bytes of the others, in c's low bits.
template <int FMT>
__device__ __forceinline__ float2 mx_decode2(uint32_t c) {
  __half2_raw h;
  if constexpr (FMT == PXB_MX_E2M1) h = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(c), __NV_E2M1);
  else h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c), FMT == PXB_MX_E4M3 ? __NV_E4M3 : __NV_E5M2);
  return __half22float2(static_cast<__half2>(h));
}

// Eight codes -> eight values before the scale.
template <int FMT>
__device__ __forceinline__ void mx_decode8(uint64_t codes, float (&v)[8]) {
  constexpr int kWords = FMT == PXB_MX_E2M1 ? 1 : 2, kPairs = 4 / kWords;
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    __half2 h[kPairs];
    mx_decode_word<FMT>(static_cast<uint32_t>(codes >> (32 * w)), h);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 d = __half22float2(h[i]);
      v[(w * kPairs + i) * 2] = d.x;
      v[(w * kPairs + i) * 2 + 1] = d.y;
    }
  }
}

// The eight codes of a lane's samples (an octet of a row: 8 bytes, or 4).
template <int FMT>
__device__ __forceinline__ uint64_t mx_load8(const uint8_t *__restrict__ codes, int64_t octet) {
  if constexpr (FMT == PXB_MX_E2M1) return __ldg(reinterpret_cast<const uint32_t *>(codes) + octet);
  else return __ldg(reinterpret_cast<const unsigned long long *>(codes) + octet);
}
template <int FMT>
__device__ __forceinline__ void mx_store8(uint8_t *__restrict__ codes, int64_t octet, uint64_t v) {
  if constexpr (FMT == PXB_MX_E2M1) reinterpret_cast<uint32_t *>(codes)[octet] = static_cast<uint32_t>(v);
  else reinterpret_cast<unsigned long long *>(codes)[octet] = v;
}

// The largest magnitude's bits of a lane's eight values, as an unsigned order
// in which infinities and NaN come last.
__device__ __forceinline__ uint32_t mx_amax8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

// A unit's activation. A ReLU keeps what is not a number (act_fn's comparison
// makes it 0): a poisoned block must not read as a silent unit.
__device__ __forceinline__ float mx_act(int kind, float x) {
  return kind == PXB_ACT_RELU ? (x <= 0.0f ? 0.0f : x) : act_fn(kind, x);
}

// Division by a launch constant: n / d for n < 2^32 as a multiply-high
// (round-up method; exact for every 32-bit n with a 33-bit magic number).
struct FastDiv {
  uint32_t d, mul, shift;
  explicit FastDiv(uint32_t div) : d(div), mul(0), shift(0) {
    while ((uint64_t(1) << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    const uint64_t t = __umulhi(n, mul);
    return static_cast<uint32_t>((t + n) >> shift);
  }
};

// CTAs for a kernel whose CTAs step through `items`, `per_cta` at a time: one
// full wave at most (a grid of 8 an SM where 6 fit would leave a second wave a
// third full).
template <auto KERNEL>
inline int mx_grid(int64_t items, int per_cta, int threads) {
  static const int resident = [threads] {
    int n = 0;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, 0) == cudaSuccess && n > 0 ? n : 1;
  }();
  return grid_for(items, per_cta, resident);
}

__host__ inline bool mx_format_ok(int fmt) { return fmt >= PXB_MX_E4M3 && fmt <= PXB_MX_E2M1; }

}  // namespace pxb

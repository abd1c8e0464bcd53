// Microscaled unit rows: quantisation, reading back, the forward apply that
// leaves a checkpoint, and the unit gradient that reads one.
//
// A row of B samples is ceil(B / 32) blocks (mx.cuh); the samples past B in
// the last block are code 0. All four are one pass over the rows: a lane owns
// an octet (eight consecutive samples of a unit), four lanes a block, so a
// block's largest magnitude takes two shuffles and its codes leave as one
// 8-byte (e2m1: 4-byte) store per lane.
#include "mx.cuh"

namespace pxb {

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

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}

// Eight consecutive values of a row, zero past `left`.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *__restrict__ p, int64_t step, int left, float (&v)[8]) {
  if (VEC && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4 *>(p);
      const T *h = reinterpret_cast<const T *>(&a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(h[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f32(p[i * step]) : 0.0f;
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *__restrict__ p, int left, const float (&v)[8]) {
  if (VEC && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 a;
      T *h = reinterpret_cast<T *>(&a);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(v[i]);
      *reinterpret_cast<uint4 *>(p) = a;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) p[i] = from_f32<T>(v[i]);
}

// A lane's octet into its block's codes and scale (every lane of the warp
// calls; the four lanes of a block are neighbours and agree on `on`).
template <int FMT>
__device__ __forceinline__ void encode_octet(const float (&v)[8], bool keep, bool on, int64_t octet, uint8_t *codes,
                                             uint8_t *scales) {
  uint32_t m = mx_amax8(v);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const uint32_t s = mx_scale_byte<FMT>(m);
  const uint64_t c = mx_encode8<FMT>(v, s, keep);
  if (on) {
    mx_store8<FMT>(codes, octet, c);
    if ((octet & 3) == 0) scales[octet >> 2] = static_cast<uint8_t>(s);
  }
}

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(256) mx_quantize_kernel(uint32_t blocks, FastDiv per_row, int32_t batch,
                                                          const T *__restrict__ x, int64_t su, int64_t sb, bool keep,
                                                          const int64_t *__restrict__ ids, int32_t num_units,
                                                          uint8_t *__restrict__ codes, uint8_t *__restrict__ scales) {
  const int64_t octets = static_cast<int64_t>(blocks) * 4;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t o0 = blockIdx.x * static_cast<int64_t>(blockDim.x) + (threadIdx.x & ~31); o0 < octets; o0 += stride) {
    int64_t o = o0 + (threadIdx.x & 31);
    bool on = o < octets;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (on) {
      const uint32_t blk = static_cast<uint32_t>(o >> 2), u = per_row.div(blk);
      const int32_t b = static_cast<int32_t>(blk - u * per_row.d) * kMxBlock + static_cast<int32_t>(o & 3) * 8;
      load8<T, VEC>(x + u * su + b * sb, sb, batch - b, v);
      if (ids != nullptr) {
        const int64_t row = ids[u];
        on = row >= 0 && row < num_units;
        o += (row - u) * (4 * static_cast<int64_t>(per_row.d));
      }
    }
    encode_octet<FMT>(v, keep, on, o, codes, scales);
  }
}

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(uint32_t blocks, FastDiv per_row, int32_t batch,
                                                            const uint8_t *__restrict__ codes,
                                                            const uint8_t *__restrict__ scales, T *__restrict__ out,
                                                            int64_t ld) {
  const int64_t octets = static_cast<int64_t>(blocks) * 4;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t o = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; o < octets; o += stride) {
    const uint32_t blk = static_cast<uint32_t>(o >> 2), u = per_row.div(blk);
    const int32_t b = static_cast<int32_t>(blk - u * per_row.d) * kMxBlock + static_cast<int32_t>(o & 3) * 8;
    const float s = mx_scale_value(scales[blk]);
    float v[8];
    mx_decode8<FMT>(mx_load8<FMT>(codes, o), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], s);
    store8<T, VEC>(out + u * ld + b, batch - b, v);
  }
}

// The forward's masked apply, in place, and the checkpoint of its result: the
// units at `target` take act(acc); an input keeps its value. Both leave their
// codes; no other row is read or written.
template <int FMT, bool VEC>
__global__ void __launch_bounds__(256) mx_unit_apply_kernel(uint32_t blocks, FastDiv per_row, int32_t batch,
                                                            int32_t act_kind, float *__restrict__ rows,
                                                            const int32_t *__restrict__ level, int32_t target,
                                                            const uint8_t *__restrict__ roles,
                                                            uint8_t *__restrict__ codes,
                                                            uint8_t *__restrict__ scales) {
  const int64_t octets = static_cast<int64_t>(blocks) * 4;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t o0 = blockIdx.x * static_cast<int64_t>(blockDim.x) + (threadIdx.x & ~31); o0 < octets; o0 += stride) {
    const int64_t o = o0 + (threadIdx.x & 31);
    bool on = o < octets;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (on) {
      const uint32_t blk = static_cast<uint32_t>(o >> 2), u = per_row.div(blk);
      on = level == nullptr || level[u] == target;
      if (on) {
        const int32_t b = static_cast<int32_t>(blk - u * per_row.d) * kMxBlock + static_cast<int32_t>(o & 3) * 8;
        float *p = rows + static_cast<int64_t>(u) * batch + b;
        load8<float, VEC>(p, 1, batch - b, v);
        const uint8_t role = roles != nullptr ? roles[u] : 0;
        if (role != 1) {
          const int kind = unit_act_kind(act_kind, role);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = i < batch - b ? act_fn(kind, v[i]) : 0.0f;
          store8<float, VEC>(p, batch - b, v);
        }
      }
    }
    encode_octet<FMT>(v, true, on, o, codes, scales);
  }
}

// out = (acc + seed) * act'(checkpointed activation).
template <int FMT, bool VEC>
__global__ void __launch_bounds__(256) mx_unit_grad_kernel(uint32_t blocks, FastDiv per_row, int32_t batch,
                                                           int32_t act_kind, const float *acc, const float *seed,
                                                           const uint8_t *__restrict__ codes,
                                                           const uint8_t *__restrict__ scales,
                                                           const int32_t *__restrict__ level, int32_t target,
                                                           const uint8_t *__restrict__ roles, float *out) {
  const int64_t octets = static_cast<int64_t>(blocks) * 4;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t o = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; o < octets; o += stride) {
    const uint32_t blk = static_cast<uint32_t>(o >> 2), u = per_row.div(blk);
    if (level != nullptr && level[u] != target) continue;
    const uint8_t role = roles != nullptr ? roles[u] : 0;
    if (role == 1) continue;
    const int32_t b = static_cast<int32_t>(blk - u * per_row.d) * kMxBlock + static_cast<int32_t>(o & 3) * 8;
    if (b >= batch) continue;
    const int kind = unit_act_kind(act_kind, role);
    const int64_t at = static_cast<int64_t>(u) * batch + b;
    float a[8], g[8];
    load8<float, VEC>(acc + at, 1, batch - b, g);
    if (seed != nullptr) {
      float sd[8];
      load8<float, VEC>(seed + at, 1, batch - b, sd);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = __fadd_rn(g[i], sd[i]);
    }
    mx_decode8<FMT>(mx_load8<FMT>(codes, o), a);
    const float s = mx_scale_value(scales[blk]);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = __fmul_rn(g[i], act_prime_from_act(kind, __fmul_rn(a[i], s)));
    store8<float, VEC>(out + at, batch - b, g);
  }
}

// Rows, blocks a row and the 32-bit block count every launch indexes by.
static int check_rows(const char *fn, int32_t num_units, int32_t batch, int fmt, int64_t *blocks) {
  PXB_REQUIRE(num_units >= 0 && batch >= 0, "%s: negative size", fn);
  PXB_REQUIRE(mx_format_ok(fmt), "%s: unknown format %d", fn, fmt);
  *blocks = static_cast<int64_t>(num_units) * mx_blocks(batch);
  PXB_REQUIRE(*blocks < (int64_t(1) << 32), "%s: %lld blocks of 32 samples are past 2^32", fn,
              static_cast<long long>(*blocks));
  return PXB_OK;
}

static bool aligned(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// One instance of the statements per format (F) / element type (T).
#define PXB_MX_FMT8(FMT, ...)                                                       \
  do {                                                                              \
    if ((FMT) == PXB_MX_E4M3) { constexpr int F = PXB_MX_E4M3; __VA_ARGS__; }        \
    else { constexpr int F = PXB_MX_E5M2; __VA_ARGS__; }                             \
  } while (0)
#define PXB_MX_FMT(FMT, ...)                                                        \
  do {                                                                              \
    if ((FMT) == PXB_MX_E2M1) { constexpr int F = PXB_MX_E2M1; __VA_ARGS__; }        \
    else PXB_MX_FMT8(FMT, __VA_ARGS__);                                              \
  } while (0)
#define PXB_MX_DTYPE(DT, ...)                                                       \
  do {                                                                              \
    if ((DT) == PXB_DT_F32) { using T = float; __VA_ARGS__; }                        \
    else if ((DT) == PXB_DT_BF16) { using T = __nv_bfloat16; __VA_ARGS__; }          \
    else { using T = __half; __VA_ARGS__; }                                          \
  } while (0)

}  // namespace pxb

using namespace pxb;

extern "C" int pxb_mx_quantize(int32_t num_rows, int32_t batch, const void *x, int32_t dtype, int64_t stride_row,
                               int64_t stride_sample, int32_t fmt, int32_t keep_nonzero, const int64_t *ids,
                               int32_t num_units, uint8_t *codes, uint8_t *scales, void *stream) {
  int64_t blocks = 0;
  if (int rc = check_rows("pxb_mx_quantize", num_units, batch, fmt, &blocks)) return rc;
  if (int rc = check_rows("pxb_mx_quantize", num_rows, batch, fmt, &blocks)) return rc;
  PXB_REQUIRE(ids != nullptr || num_rows <= num_units, "pxb_mx_quantize: %d rows do not fit in %d", num_rows,
              num_units);
  PXB_REQUIRE(dtype >= PXB_DT_F32 && dtype <= PXB_DT_F16, "pxb_mx_quantize: unknown type %d", dtype);
  if (blocks == 0) return PXB_OK;
  PXB_REQUIRE(x && codes && scales, "pxb_mx_quantize: a pointer is NULL");
  PXB_REQUIRE(aligned(codes, 16), "pxb_mx_quantize: codes must be 16-byte aligned");
  const int size = dtype == PXB_DT_F32 ? 4 : 2;
  const bool vec = stride_sample == 1 && aligned16(x) && (stride_row * size) % 16 == 0;
  const FastDiv per_row(static_cast<uint32_t>(mx_blocks(batch)));
  const int grid = grid_for(blocks * 4, 256, 16);
  cudaStream_t st = as_stream(stream);
  const uint32_t nb = static_cast<uint32_t>(blocks);
  PXB_MX_DTYPE(dtype, PXB_MX_FMT(fmt, {
    const T *xt = static_cast<const T *>(x);
    if (vec) mx_quantize_kernel<T, F, true><<<grid, 256, 0, st>>>(nb, per_row, batch, xt, stride_row, stride_sample, keep_nonzero != 0, ids, num_units, codes, scales);
    else mx_quantize_kernel<T, F, false><<<grid, 256, 0, st>>>(nb, per_row, batch, xt, stride_row, stride_sample, keep_nonzero != 0, ids, num_units, codes, scales);
  }));
  PXB_LAUNCHED("mx_quantize_kernel");
  return PXB_OK;
}

extern "C" int pxb_mx_dequantize(int32_t num_units, int32_t batch, const uint8_t *codes, const uint8_t *scales,
                                 int32_t fmt, void *out, int32_t dtype, int64_t ld, void *stream) {
  int64_t blocks = 0;
  if (int rc = check_rows("pxb_mx_dequantize", num_units, batch, fmt, &blocks)) return rc;
  PXB_REQUIRE(dtype >= PXB_DT_F32 && dtype <= PXB_DT_F16, "pxb_mx_dequantize: unknown type %d", dtype);
  PXB_REQUIRE(ld >= batch, "pxb_mx_dequantize: rows overlap");
  if (blocks == 0) return PXB_OK;
  PXB_REQUIRE(codes && scales && out, "pxb_mx_dequantize: a pointer is NULL");
  PXB_REQUIRE(aligned(codes, 16), "pxb_mx_dequantize: codes must be 16-byte aligned");
  const int size = dtype == PXB_DT_F32 ? 4 : 2;
  const bool vec = aligned16(out) && (ld * size) % 16 == 0;
  const FastDiv per_row(static_cast<uint32_t>(mx_blocks(batch)));
  const int grid = grid_for(blocks * 4, 256, 16);
  cudaStream_t st = as_stream(stream);
  const uint32_t nb = static_cast<uint32_t>(blocks);
  PXB_MX_DTYPE(dtype, PXB_MX_FMT(fmt, {
    T *ot = static_cast<T *>(out);
    if (vec) mx_dequantize_kernel<T, F, true><<<grid, 256, 0, st>>>(nb, per_row, batch, codes, scales, ot, ld);
    else mx_dequantize_kernel<T, F, false><<<grid, 256, 0, st>>>(nb, per_row, batch, codes, scales, ot, ld);
  }));
  PXB_LAUNCHED("mx_dequantize_kernel");
  return PXB_OK;
}

extern "C" int pxb_mx_unit_apply(int32_t num_units, int32_t batch, int32_t act_kind, float *rows,
                                 const int32_t *level, int32_t target_level, const uint8_t *roles, int32_t fmt,
                                 uint8_t *codes, uint8_t *scales, void *stream) {
  int64_t blocks = 0;
  if (int rc = check_rows("pxb_mx_unit_apply", num_units, batch, fmt, &blocks)) return rc;
  PXB_REQUIRE(fmt != PXB_MX_E2M1, "pxb_mx_unit_apply: a checkpoint has 8 bits (e4m3 or e5m2)");
  PXB_REQUIRE(act_code_ok(act_kind), "pxb_mx_unit_apply: unknown activation code %d", act_kind);
  if (blocks == 0) return PXB_OK;
  PXB_REQUIRE(rows && codes && scales, "pxb_mx_unit_apply: a pointer is NULL");
  PXB_REQUIRE(aligned(codes, 16), "pxb_mx_unit_apply: codes must be 16-byte aligned");
  const bool vec = aligned16(rows) && batch % 4 == 0;
  const FastDiv per_row(static_cast<uint32_t>(mx_blocks(batch)));
  const int grid = grid_for(blocks * 4, 256, 8);
  cudaStream_t st = as_stream(stream);
  const uint32_t nb = static_cast<uint32_t>(blocks);
  PXB_MX_FMT8(fmt, {
    if (vec) mx_unit_apply_kernel<F, true><<<grid, 256, 0, st>>>(nb, per_row, batch, act_kind, rows, level, target_level, roles, codes, scales);
    else mx_unit_apply_kernel<F, false><<<grid, 256, 0, st>>>(nb, per_row, batch, act_kind, rows, level, target_level, roles, codes, scales);
  });
  PXB_LAUNCHED("mx_unit_apply_kernel");
  return PXB_OK;
}

extern "C" int pxb_mx_unit_grad(int32_t num_units, int32_t batch, int32_t act_kind, const float *acc,
                                const float *seed, const uint8_t *codes, const uint8_t *scales, int32_t fmt,
                                const int32_t *level, int32_t target_level, const uint8_t *roles, float *out,
                                void *stream) {
  int64_t blocks = 0;
  if (int rc = check_rows("pxb_mx_unit_grad", num_units, batch, fmt, &blocks)) return rc;
  PXB_REQUIRE(fmt != PXB_MX_E2M1, "pxb_mx_unit_grad: a checkpoint has 8 bits (e4m3 or e5m2)");
  PXB_REQUIRE(act_code_ok(act_kind), "pxb_mx_unit_grad: unknown activation code %d", act_kind);
  if (blocks == 0) return PXB_OK;
  PXB_REQUIRE(acc && codes && scales && out, "pxb_mx_unit_grad: a pointer is NULL");
  PXB_REQUIRE(aligned(codes, 16), "pxb_mx_unit_grad: codes must be 16-byte aligned");
  const bool vec = aligned16(acc) && aligned16(out) && (seed == nullptr || aligned16(seed)) && batch % 4 == 0;
  const FastDiv per_row(static_cast<uint32_t>(mx_blocks(batch)));
  const int grid = grid_for(blocks * 4, 256, 16);
  cudaStream_t st = as_stream(stream);
  const uint32_t nb = static_cast<uint32_t>(blocks);
  PXB_MX_FMT8(fmt, {
    if (vec) mx_unit_grad_kernel<F, true><<<grid, 256, 0, st>>>(nb, per_row, batch, act_kind, acc, seed, codes, scales, level, target_level, roles, out);
    else mx_unit_grad_kernel<F, false><<<grid, 256, 0, st>>>(nb, per_row, batch, act_kind, acc, seed, codes, scales, level, target_level, roles, out);
  });
  PXB_LAUNCHED("mx_unit_grad_kernel");
  return PXB_OK;
}

// Microscaled unit rows: quantisation, reading back, the forward apply that
// leaves a checkpoint, and the unit gradient that reads one.
//
// A row of B samples is ceil(B / 32) blocks (mx.cuh); the samples past B in
// the last block are code 0. All four are one pass over the rows: a lane owns
// an octet (eight consecutive samples of a unit), four lanes a block, so a
// block's largest magnitude takes two shuffles and its codes leave as one
// 8-byte (e2m1: 4-byte) store per lane.
#include <initializer_list>

#include "mx.cuh"

namespace pxb {

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// How a warp's 32 octets (its tile) lie in the rows.
//
// ALIGNED: octets of all rows in a line; a lane moves its octet in 16-byte
// accesses (rows on 16-byte boundaries).
// RUN, RUN2, TILE: rows at any element. An octet a lane would be eight
// accesses 32 bytes apart, each touching every sector of the tile; instead the
// warp moves the tile in runs of addresses -- lane l the elements l, l + 32,
// ... -- and turns it into octets through its own kilobyte of shared memory.
// RUN: a tile is 256 samples of one row; RUN2: the same in pairs of 16-bit
// elements (rows on 4-byte boundaries); TILE: `width` blocks (1, 2 or 4) of 8 /
// width rows, for rows of 128 samples at most.
enum Layout { ALIGNED, RUN, RUN2, TILE };

struct Grid {
  int32_t rows, batch, nb, width;  // width: a tile's blocks a row (not ALIGNED)
  FastDiv per_row;                 // ALIGNED: blocks a row; else tiles a row
  uint32_t tiles;
};

struct Octet {
  uint32_t u;   // row
  int32_t b;    // first sample
  int64_t at;   // index among all octets
  bool on;      // within the rows
};

template <int LAYOUT>
__device__ __forceinline__ Octet octet_of(const Grid &g, uint32_t tile, int lane) {
  Octet o;
  if constexpr (LAYOUT != ALIGNED) {
    const uint32_t group = g.per_row.div(tile), seg = tile - group * g.per_row.d;
    const int blk = lane >> 2, shift = LAYOUT == TILE ? 31 - __clz(g.width) : 3;
    o.u = group * (8 >> shift) + (blk >> shift);
    const int32_t k = (seg << shift) + (blk & ((1 << shift) - 1));
    o.b = k * kMxBlock + (lane & 3) * 8;
    o.on = o.u < static_cast<uint32_t>(g.rows) && k < g.nb;
    o.at = (static_cast<int64_t>(o.u) * g.nb + k) * 4 + (lane & 3);
  } else {
    o.at = static_cast<int64_t>(tile) * 32 + lane;
    const uint32_t blk = static_cast<uint32_t>(o.at >> 2);
    o.u = g.per_row.div(blk);
    o.b = static_cast<int32_t>(blk - o.u * g.per_row.d) * kMxBlock + (lane & 3) * 8;
    o.on = o.at < static_cast<int64_t>(g.rows) * g.nb * 4;
  }
  return o;
}

// The move q of lane l in a tile: kEach neighbouring elements of row `u` from
// sample `b` on; none where u is outside the rows.
template <int LAYOUT>
struct Moves {
  static constexpr int kEach = LAYOUT == RUN2 ? 2 : 1, kMoves = 8 / kEach;
  uint32_t u0;
  int32_t b0;
  int shift;  // TILE: log2 of the tile's blocks a row
  __device__ __forceinline__ Moves(const Grid &g, uint32_t tile, int lane) {
    const uint32_t group = g.per_row.div(tile), seg = tile - group * g.per_row.d;
    shift = LAYOUT == TILE ? 31 - __clz(g.width) : 3;
    u0 = group * (8 >> shift);
    b0 = static_cast<int32_t>(seg) * 256 + lane * kEach;  // TILE has one tile a row
  }
  __device__ __forceinline__ uint32_t u(int q) const { return LAYOUT == TILE ? u0 + (q >> shift) : u0; }
  __device__ __forceinline__ int32_t b(int q) const {
    return LAYOUT == TILE ? b0 + (q & ((1 << shift) - 1)) * kMxBlock : b0 + q * 32 * kEach;
  }
};

template <typename T, int N>
struct Pack {
  T v[N];
};

// What a lane has read of its tile, before it is turned into its octet: the
// words as they came, so that nothing waits between the loads.
template <typename T, int LAYOUT>
struct Raw {
  T v[8];
};
template <typename T>
struct Raw<T, RUN2> {
  uint32_t v[4];
};
template <typename T>
struct Raw<T, ALIGNED> {
  uint4 v[sizeof(T) / 2];
  float tail[8];
};

// The lane's share of the tile from rows `su` elements apart; zero outside.
// `keep(u)`: whether row u is read.
template <typename T, int LAYOUT, typename Keep>
__device__ __forceinline__ void fetch(const Grid &g, uint32_t tile, const Octet &o, const T *x, int64_t su, Keep keep,
                                      Raw<T, LAYOUT> &r) {
  if constexpr (LAYOUT == ALIGNED) {
    const T *p = x + o.u * su + o.b;
    if (o.on && o.b + 8 <= g.batch) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.tail[i] = o.on && o.b + i < g.batch ? to_f32(p[i]) : 0.0f;
    }
  } else {
    const Moves<LAYOUT> m(g, tile, threadIdx.x & 31);
    if constexpr (LAYOUT == TILE) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint32_t u = m.u(q);
        const bool ok = u < static_cast<uint32_t>(g.rows) && m.b(q) < g.batch && keep(u);
        r.v[q] = ok ? x[u * su + m.b(q)] : T(0.0f);
      }
    } else {
      const int32_t end = m.u0 < static_cast<uint32_t>(g.rows) && keep(m.u0) ? g.batch : 0;
      const T *p = x + m.u0 * su + m.b0;
#pragma unroll
      for (int q = 0; q < Moves<LAYOUT>::kMoves; ++q) {
        if constexpr (LAYOUT == RUN) {
          r.v[q] = m.b(q) < end ? p[q * 32] : T(0.0f);
        } else {
          r.v[q] = m.b(q) < (end & ~1) ? *reinterpret_cast<const uint32_t *>(p + q * 64) : 0u;
        }
      }
      if (LAYOUT == RUN2 && (end & 1)) {  // the sample without a partner
#pragma unroll
        for (int q = 0; q < Moves<LAYOUT>::kMoves; ++q)
          if (m.b(q) == end - 1) r.v[q] = *reinterpret_cast<const uint16_t *>(p + q * 64);
      }
    }
  }
}

template <typename T, int LAYOUT>
__device__ __forceinline__ void settle(const Grid &g, const Octet &o, const Raw<T, LAYOUT> &r, float *buf,
                                       float (&v)[8]) {
  if constexpr (LAYOUT == ALIGNED) {
    if (o.on && o.b + 8 <= g.batch) {
#pragma unroll
      for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q) {
        const auto h = same_bits<Pack<T, 16 / sizeof(T)>>(r.v[q]);
#pragma unroll
        for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) v[q * (16 / sizeof(T)) + i] = to_f32(h.v[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r.tail[i];
    }
  } else {
    const int lane = threadIdx.x & 31;
    T *b = reinterpret_cast<T *>(buf);
    __syncwarp();
#pragma unroll
    for (int q = 0; q < Moves<LAYOUT>::kMoves; ++q) {
      if constexpr (LAYOUT == RUN2) reinterpret_cast<uint32_t *>(b)[q * 32 + lane] = r.v[q];
      else b[q * 32 + lane] = r.v[q];
    }
    __syncwarp();
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q) {
      const auto h = same_bits<Pack<T, 16 / sizeof(T)>>(reinterpret_cast<const uint4 *>(b)[lane * (sizeof(T) / 2) + q]);
#pragma unroll
      for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) v[q * (16 / sizeof(T)) + i] = to_f32(h.v[i]);
    }
  }
}

// The lane's octet out to rows `ld` elements apart. `keep(u)`: whether row u
// is written.
template <typename T, int LAYOUT, typename Keep>
__device__ __forceinline__ void put(const Grid &g, uint32_t tile, const Octet &o, T *out, int64_t ld, Keep keep,
                                    float *buf, const float (&v)[8]) {
  if constexpr (LAYOUT != ALIGNED) {
    const int lane = threadIdx.x & 31;
    T *b = reinterpret_cast<T *>(buf);
    __syncwarp();
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q) {
      Pack<T, 16 / sizeof(T)> h;
#pragma unroll
      for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) h.v[i] = from_f32<T>(v[q * (16 / sizeof(T)) + i]);
      reinterpret_cast<uint4 *>(b)[lane * (sizeof(T) / 2) + q] = same_bits<uint4>(h);
    }
    __syncwarp();
    const Moves<LAYOUT> m(g, tile, lane);
    if constexpr (LAYOUT == TILE) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint32_t u = m.u(q);
        if (u < static_cast<uint32_t>(g.rows) && m.b(q) < g.batch && keep(u)) out[u * ld + m.b(q)] = b[q * 32 + lane];
      }
    } else {
      const int32_t end = m.u0 < static_cast<uint32_t>(g.rows) && keep(m.u0) ? g.batch : 0;
      T *p = out + m.u0 * ld + m.b0;
#pragma unroll
      for (int q = 0; q < Moves<LAYOUT>::kMoves; ++q) {
        if constexpr (LAYOUT == RUN) {
          if (m.b(q) < end) p[q * 32] = b[q * 32 + lane];
        } else {
          const uint32_t two = reinterpret_cast<const uint32_t *>(b)[q * 32 + lane];
          if (m.b(q) < (end & ~1)) *reinterpret_cast<uint32_t *>(p + q * 64) = two;
          if ((end & 1) && m.b(q) == end - 1) p[q * 64] = same_bits<Pack<T, 2>>(two).v[0];
        }
      }
    }
  } else {
    const bool on = o.on && keep(o.u);
    T *p = out + o.u * ld + o.b;
    if constexpr (sizeof(T) == 4) {
      // two lanes swap halves of their octets, so that each store instruction writes whole sectors: the first the even
      // lanes' octets, the second the odd lanes'
      const int lane = threadIdx.x & 31;
      const bool odd = lane & 1, full = on && o.b + 8 <= g.batch;
      const unsigned fulls = __ballot_sync(0xffffffffu, full);
      float4 got;
      got.x = __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[4], 1);
      got.y = __shfl_xor_sync(0xffffffffu, odd ? v[1] : v[5], 1);
      got.z = __shfl_xor_sync(0xffffffffu, odd ? v[2] : v[6], 1);
      got.w = __shfl_xor_sync(0xffffffffu, odd ? v[3] : v[7], 1);
      if (fulls >> (lane & ~1) & 1) *reinterpret_cast<float4 *>(odd ? p - 4 : p) = odd ? got : make_float4(v[0], v[1], v[2], v[3]);
      if (fulls >> (lane | 1) & 1) *reinterpret_cast<float4 *>(odd ? p + 4 : p + 8) = odd ? make_float4(v[4], v[5], v[6], v[7]) : got;
      if (full) return;
    } else if (on && o.b + 8 <= g.batch) {
      Pack<T, 8> h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h.v[i] = from_f32<T>(v[i]);
      *reinterpret_cast<uint4 *>(p) = same_bits<uint4>(h);
      return;
    }
    if (on) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (o.b + i < g.batch) p[i] = from_f32<T>(v[i]);
    }
  }
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

constexpr int kThreads = 256, kWarps = kThreads / 32;
struct All {
  __device__ __forceinline__ bool operator()(uint32_t) const { return true; }
};

// Warps step through the tiles two at a time, so that two tiles' loads are in
// flight together.
#define PXB_MX_TILES(g)                                                                                 \
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;                                           \
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kWarps;                                      \
  for (uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * kWarps + warp; t0 < (g).tiles; t0 += 2 * step)

template <typename T, int FMT, int LAYOUT>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(Grid g, const T *__restrict__ x, int64_t su, bool keep,
                                                               const int64_t *__restrict__ ids,
                                                               int32_t num_units, uint8_t *__restrict__ codes,
                                                               uint8_t *__restrict__ scales) {
  __shared__ __align__(16) float tiles[LAYOUT != ALIGNED ? kWarps : 1][256];
  PXB_MX_TILES(g) {
    Octet o[2];
    Raw<T, LAYOUT> r[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint64_t t = t0 + k * step;
      o[k] = octet_of<LAYOUT>(g, static_cast<uint32_t>(t), lane);
      if (t >= g.tiles) o[k].on = false;
      else fetch<T, LAYOUT>(g, static_cast<uint32_t>(t), o[k], x, su, All(), r[k]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (t0 + k * step >= g.tiles) break;
      float v[8];
      settle<T, LAYOUT>(g, o[k], r[k], tiles[LAYOUT != ALIGNED ? warp : 0], v);
      int64_t at = o[k].at;
      bool on = o[k].on;
      if (ids != nullptr && on) {
        const int64_t row = ids[o[k].u];
        on = row >= 0 && row < num_units;
        at += (row - o[k].u) * (4 * static_cast<int64_t>(g.nb));
      }
      encode_octet<FMT>(v, keep, on, at, codes, scales);
    }
  }
}

// Samples at any stride. A lane takes a whole block of one unit, the lanes of
// a warp 32 neighbouring units: a sample-major batch (units adjacent) is then
// read in full lines, and the block's scale and codes need no other lane.
template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) mx_quantize_strided_kernel(int32_t rows, int32_t batch, int32_t nb,
                                                                       FastDiv groups, const T *__restrict__ x,
                                                                       int64_t su, int64_t sb, bool keep,
                                                                       const int64_t *__restrict__ ids,
                                                                       int32_t num_units, uint8_t *__restrict__ codes,
                                                                       uint8_t *__restrict__ scales) {
  const int lane = threadIdx.x & 31;
  const uint64_t total = static_cast<uint64_t>(groups.d) * nb, step = static_cast<uint64_t>(gridDim.x) * kWarps;
  for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < total; t += step) {
    const uint32_t k = groups.div(static_cast<uint32_t>(t));
    const int64_t u = static_cast<int64_t>(static_cast<uint32_t>(t) - k * groups.d) * 32 + lane;
    if (u >= rows) continue;
    const int32_t b = static_cast<int32_t>(k) * kMxBlock;
    const T *p = x + u * su + b * sb;
    float v[4][8];
    uint32_t m = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[q][i] = b + q * 8 + i < batch ? to_f32(p[(q * 8 + i) * sb]) : 0.0f;
      m = max(m, mx_amax8(v[q]));
    }
    const int64_t row = ids != nullptr ? ids[u] : u;
    if (row < 0 || row >= num_units) continue;
    const uint32_t s = mx_scale_byte<FMT>(m);
    const int64_t at = row * nb + k;
    uint64_t c[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) c[q] = mx_encode8<FMT>(v[q], s, keep);
    uint4 *out = reinterpret_cast<uint4 *>(codes + at * mx_block_bytes<FMT>());
    if constexpr (FMT == PXB_MX_E2M1) {
      out[0] = make_uint4(c[0], c[1], c[2], c[3]);
    } else {
      out[0] = make_uint4(c[0], c[0] >> 32, c[1], c[1] >> 32);
      out[1] = make_uint4(c[2], c[2] >> 32, c[3], c[3] >> 32);
    }
    scales[at] = static_cast<uint8_t>(s);
  }
}

template <typename T, int FMT, int LAYOUT>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(Grid g, const uint8_t *__restrict__ codes,
                                                                 const uint8_t *__restrict__ scales, T *out,
                                                                 int64_t ld) {
  __shared__ __align__(16) float tiles[LAYOUT != ALIGNED ? kWarps : 1][256];
  PXB_MX_TILES(g) {
    Octet o[2];
    uint64_t c[2] = {0, 0};
    uint32_t s[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint64_t t = t0 + k * step;
      o[k] = octet_of<LAYOUT>(g, static_cast<uint32_t>(t), lane);
      if (t >= g.tiles) o[k].on = false;
      if (o[k].on) {
        c[k] = mx_load8<FMT>(codes, o[k].at);
        s[k] = __ldg(scales + (o[k].at >> 2));
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (t0 + k * step >= g.tiles) break;
      float v[8];
      mx_decode8<FMT>(c[k], v);
      const float sc = mx_scale_value(s[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], sc);
      put<T, LAYOUT>(g, static_cast<uint32_t>(t0 + k * step), o[k], out, ld, All(),
                     tiles[LAYOUT != ALIGNED ? warp : 0], v);
    }
  }
}

// The units a masked pass works on, and whether it changes their rows.
struct Mask {
  const int32_t *__restrict__ level;
  int32_t target;
  const uint8_t *__restrict__ roles;
  __device__ __forceinline__ bool here(uint32_t u) const { return level == nullptr || __ldg(level + u) == target; }
  __device__ __forceinline__ uint8_t role(uint32_t u) const { return roles == nullptr ? 0 : __ldg(roles + u); }
};

// The forward's masked apply, in place, and the checkpoint of its result: the
// units at the mask's level take act(rows); an input keeps its row. Both leave
// their codes; no other row is read or written.
template <int FMT, int LAYOUT>
__global__ void __launch_bounds__(kThreads) mx_unit_apply_kernel(Grid g, int32_t act_kind, float *rows, Mask m,
                                                                 uint8_t *__restrict__ codes,
                                                                 uint8_t *__restrict__ scales) {
  __shared__ __align__(16) float tiles[LAYOUT != ALIGNED ? kWarps : 1][256];
  const auto here = [&](uint32_t u) { return m.here(u); };
  const auto moves = [&](uint32_t u) { return m.here(u) && m.role(u) != 1; };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float *buf = tiles[LAYOUT != ALIGNED ? warp : 0];
  for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kWarps + warp; t < g.tiles;
       t += static_cast<uint64_t>(gridDim.x) * kWarps) {
    Octet o = octet_of<LAYOUT>(g, static_cast<uint32_t>(t), lane);
    o.on = o.on && m.here(o.u);
    if (!__any_sync(0xffffffffu, o.on)) continue;
    Raw<float, LAYOUT> r;
    fetch<float, LAYOUT>(g, static_cast<uint32_t>(t), o, rows, g.batch, here, r);
    float v[8];
    settle<float, LAYOUT>(g, o, r, buf, v);
    if (o.on) {
      const uint8_t role = m.role(o.u);
      if (role != 1) {
        const int kind = unit_act_kind(act_kind, role);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = o.b + i < g.batch ? mx_act(kind, v[i]) : 0.0f;
      }
    }
    put<float, LAYOUT>(g, static_cast<uint32_t>(t), o, rows, g.batch, moves, buf, v);
    encode_octet<FMT>(v, true, o.on, o.at, codes, scales);
  }
}

// out = (acc + seed) * act'(checkpointed activation).
template <int FMT, int LAYOUT>
__global__ void __launch_bounds__(kThreads, 4) mx_unit_grad_kernel(Grid g, int32_t act_kind, const float *acc,
                                                                const float *seed, const uint8_t *__restrict__ codes,
                                                                const uint8_t *__restrict__ scales, Mask m,
                                                                float *out) {
  __shared__ __align__(16) float tiles[LAYOUT != ALIGNED ? kWarps : 1][256];
  const auto moves = [&](uint32_t u) { return m.here(u) && m.role(u) != 1; };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float *buf = tiles[LAYOUT != ALIGNED ? warp : 0];
  for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kWarps + warp; t < g.tiles;
       t += static_cast<uint64_t>(gridDim.x) * kWarps) {
    Octet o = octet_of<LAYOUT>(g, static_cast<uint32_t>(t), lane);
    const uint8_t role = o.on ? m.role(o.u) : 1;
    o.on = o.on && role != 1 && m.here(o.u);
    if (!__any_sync(0xffffffffu, o.on)) continue;
    Raw<float, LAYOUT> ra, rs;
    fetch<float, LAYOUT>(g, static_cast<uint32_t>(t), o, acc, g.batch, moves, ra);
    if (seed != nullptr) fetch<float, LAYOUT>(g, static_cast<uint32_t>(t), o, seed, g.batch, moves, rs);
    const uint64_t c = o.on ? mx_load8<FMT>(codes, o.at) : 0;
    const float sc = mx_scale_value(o.on ? __ldg(scales + (o.at >> 2)) : 0);
    float v[8], a[8];
    settle<float, LAYOUT>(g, o, ra, buf, v);
    if (seed != nullptr) {
      settle<float, LAYOUT>(g, o, rs, buf, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fadd_rn(v[i], a[i]);
    }
    const int kind = unit_act_kind(act_kind, role);
    mx_decode8<FMT>(c, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], act_prime_from_act(kind, __fmul_rn(a[i], sc)));
    put<float, LAYOUT>(g, static_cast<uint32_t>(t), o, out, g.batch, moves, buf, v);
  }
}

// Rows, blocks a row and the 32-bit block count every launch indexes by.
static int check_rows(const char *fn, int32_t num_units, int32_t batch, int fmt, int64_t *blocks) {
  PXB_REQUIRE(num_units >= 0 && batch >= 0 && batch <= kMxMaxBatch, "%s: bad size", fn);
  PXB_REQUIRE(mx_format_ok(fmt), "%s: unknown format %d", fn, fmt);
  *blocks = static_cast<int64_t>(num_units) * mx_blocks(batch);
  PXB_REQUIRE(*blocks < (int64_t(1) << 32), "%s: %lld blocks of 32 samples are past 2^32", fn,
              static_cast<long long>(*blocks));
  return PXB_OK;
}

// The layout for rows `ld` elements of `size` bytes apart from p (any of a
// pass's row buffers: the first that is off the boundary decides).
static int layout_of(int32_t batch, int size, std::initializer_list<const void *> ps, int64_t ld) {
  uintptr_t bits = static_cast<uintptr_t>(ld * size);
  for (const void *p : ps) bits |= reinterpret_cast<uintptr_t>(p);
  if ((bits & 15) == 0) return ALIGNED;
  if (batch <= 4 * kMxBlock) return TILE;
  return size == 2 && (bits & 3) == 0 ? RUN2 : RUN;
}

static Grid grid_of(int32_t rows, int32_t batch, int layout) {
  const int32_t nb = static_cast<int32_t>(mx_blocks(batch));
  if (layout == ALIGNED)
    return Grid{rows, batch, nb, 0, FastDiv(static_cast<uint32_t>(nb)),
                static_cast<uint32_t>((static_cast<int64_t>(rows) * nb + 7) / 8)};
  const int32_t width = layout != TILE ? 8 : nb <= 1 ? 1 : nb <= 2 ? 2 : 4, segs = (nb + width - 1) / width;
  const int64_t groups = (static_cast<int64_t>(rows) * width + 7) / 8;
  return Grid{rows, batch, nb, width, FastDiv(static_cast<uint32_t>(segs)), static_cast<uint32_t>(groups * segs)};
}

// One instance of the statements per format (F), element type (T), layout (L).
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
#define PXB_MX_ROWS(LAY, ...)                                                       \
  do {                                                                              \
    if ((LAY) == ALIGNED) { constexpr int L = ALIGNED; __VA_ARGS__; }                \
    else if ((LAY) == TILE) { constexpr int L = TILE; __VA_ARGS__; }                 \
    else { constexpr int L = RUN; __VA_ARGS__; }                                     \
  } while (0)
#define PXB_MX_ROWS2(LAY, ...)                                                      \
  do {                                                                              \
    if (sizeof(T) == 2 && (LAY) == RUN2) { constexpr int L = sizeof(T) == 2 ? RUN2 : RUN; __VA_ARGS__; } \
    else PXB_MX_ROWS(LAY, __VA_ARGS__);                                              \
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
  PXB_REQUIRE(aligned16(codes), "pxb_mx_quantize: codes must be 16-byte aligned");
  const int size = dtype == PXB_DT_F32 ? 4 : 2;
  cudaStream_t st = as_stream(stream);
  if (stride_sample != 1 && batch > 1) {
    const FastDiv groups(static_cast<uint32_t>((static_cast<int64_t>(num_rows) + 31) / 32));
    const int32_t nb = static_cast<int32_t>(mx_blocks(batch));
    PXB_MX_DTYPE(dtype, PXB_MX_FMT(fmt, {
      mx_quantize_strided_kernel<T, F><<<mx_grid<mx_quantize_strided_kernel<T, F>>(static_cast<int64_t>(groups.d) * nb, kWarps, kThreads), kThreads, 0, st>>>(num_rows, batch, nb, groups, static_cast<const T *>(x),
                                                                  stride_row, stride_sample, keep_nonzero != 0, ids, num_units, codes, scales);
    }));
    PXB_LAUNCHED("mx_quantize_strided_kernel");
    return PXB_OK;
  }
  const int layout = layout_of(batch, size, {x}, stride_row);
  const Grid g = grid_of(num_rows, batch, layout);
  PXB_MX_DTYPE(dtype, PXB_MX_FMT(fmt, PXB_MX_ROWS2(layout, {
    mx_quantize_kernel<T, F, L><<<mx_grid<mx_quantize_kernel<T, F, L>>(g.tiles, kWarps, kThreads), kThreads, 0, st>>>(g, static_cast<const T *>(x), stride_row, keep_nonzero != 0, ids, num_units, codes, scales);
  })));
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
  PXB_REQUIRE(aligned16(codes), "pxb_mx_dequantize: codes must be 16-byte aligned");
  const int size = dtype == PXB_DT_F32 ? 4 : 2;
  const int layout = layout_of(batch, size, {out}, ld);
  const Grid g = grid_of(num_units, batch, layout);
  cudaStream_t st = as_stream(stream);
  PXB_MX_DTYPE(dtype, PXB_MX_FMT(fmt, PXB_MX_ROWS2(layout, {
    mx_dequantize_kernel<T, F, L><<<mx_grid<mx_dequantize_kernel<T, F, L>>(g.tiles, kWarps, kThreads), kThreads, 0, st>>>(g, codes, scales, static_cast<T *>(out), ld);
  })));
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
  PXB_REQUIRE(aligned16(codes), "pxb_mx_unit_apply: codes must be 16-byte aligned");
  const int layout = layout_of(batch, 4, {rows}, batch);
  const Grid g = grid_of(num_units, batch, layout);
  cudaStream_t st = as_stream(stream);
  PXB_MX_FMT8(fmt, PXB_MX_ROWS(layout, {
    mx_unit_apply_kernel<F, L><<<mx_grid<mx_unit_apply_kernel<F, L>>(g.tiles, kWarps, kThreads), kThreads, 0, st>>>(g, act_kind, rows, Mask{level, target_level, roles}, codes, scales);
  }));
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
  PXB_REQUIRE(aligned16(codes), "pxb_mx_unit_grad: codes must be 16-byte aligned");
  const int layout = layout_of(batch, 4, {acc, seed, out}, batch);
  const Grid g = grid_of(num_units, batch, layout);
  cudaStream_t st = as_stream(stream);
  PXB_MX_FMT8(fmt, PXB_MX_ROWS(layout, {
    mx_unit_grad_kernel<F, L><<<mx_grid<mx_unit_grad_kernel<F, L>>(g.tiles, kWarps, kThreads), kThreads, 0, st>>>(g, act_kind, acc, seed, codes, scales, Mask{level, target_level, roles}, out);
  }));
  PXB_LAUNCHED("mx_unit_grad_kernel");
  return PXB_OK;
}

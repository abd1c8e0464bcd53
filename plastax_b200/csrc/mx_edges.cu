// Edge products over microscaled rows: the gradient of every connection from
// checkpointed activations, and the forward of a frozen arena.
#include <cooperative_groups.h>

#include "mx.cuh"
#include "optim.cuh"

namespace pxb {

// ---------------------------------------------------------------------------
// stat[s] = (sum_b g[to, b] * a[from, b]) / B
// ---------------------------------------------------------------------------
struct EdgeGrad {
  int64_t cap;
  const int32_t *__restrict__ from, *__restrict__ to;
  const uint8_t *__restrict__ dead;
  const float *__restrict__ g;
  const uint8_t *__restrict__ codes, *__restrict__ scales;
  int32_t batch, nb;
  uint32_t n;
  float *dw, *weight;
  OptParams op;
  float *m, *v, *t;
};

// A slot as it was read (three loads in flight together), and whether it
// takes a gradient.
struct Slot {
  int32_t f, t;
  uint8_t dead;
  __device__ __forceinline__ bool live(uint32_t n) const {
    return !dead && static_cast<uint32_t>(f) < n && static_cast<uint32_t>(t) < n;
  }
};

__device__ __forceinline__ Slot load_slot(const EdgeGrad &k, int64_t s) {
  Slot r{0, 0, 1};
  if (s < k.cap) r = Slot{__ldg(k.from + s), __ldg(k.to + s), __ldg(k.dead + s)};
  return r;
}

// Offsets into the gradient rows and the codes: 32 bits where the rows end
// below 4 GiB (one add a load, from a uniform base), else 64.
template <bool WIDE>
struct Offset {
  using type = uint32_t;
};
template <>
struct Offset<true> {
  using type = uint64_t;
};

// Four gradients from byte offset `at`, whose first sample is b: 0 past the
// batch (FULL: the whole slice lies below it).
template <bool VEC, bool FULL, typename O>
__device__ __forceinline__ float4 load_grad(const float *__restrict__ g, O at, int32_t batch, int32_t b) {
  const float *p = reinterpret_cast<const float *>(reinterpret_cast<const char *>(g) + at);
  if (VEC && FULL) return __ldg(reinterpret_cast<const float4 *>(p));
  if (!VEC && FULL) return make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (VEC) {
    if (b < batch) v = __ldg(reinterpret_cast<const float4 *>(p));
    return v;
  }
  if (b < batch) v.x = __ldg(p);
  if (b + 1 < batch) v.y = __ldg(p + 1);
  if (b + 2 < batch) v.z = __ldg(p + 2);
  if (b + 3 < batch) v.w = __ldg(p + 3);
  return v;
}

// A lane's four activations of a slice of source row f, as two pairs.
template <int FMT, typename O>
__device__ __forceinline__ void load_acts(const EdgeGrad &k, int32_t f, int32_t slice, int sub, float2 (&a)[2]) {
  const O blk = static_cast<O>(f) * static_cast<O>(k.nb) + static_cast<O>(slice);
  const uint32_t c = __ldg(reinterpret_cast<const uint32_t *>(k.codes + blk * 32) + sub);
  const float sc = mx_scale_value(__ldg(k.scales + blk));
  __half2 h[2];
  mx_decode_word<FMT>(c, h);
  const float2 lo = __half22float2(h[0]), hi = __half22float2(h[1]);
  a[0] = make_float2(__fmul_rn(lo.x, sc), __fmul_rn(lo.y, sc));
  a[1] = make_float2(__fmul_rn(hi.x, sc), __fmul_rn(hi.y, sc));
}

__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d) : "l"(same_bits<unsigned long long>(a)), "l"(same_bits<unsigned long long>(b)),
        "l"(same_bits<unsigned long long>(c)));
  return same_bits<float2>(d);
}

// Sums over the lanes OFF, OFF / 2, ... LANES apart: half of the N values left go
// to the other side each time, until one is left; a lane ends with the values
// from `base` on.
template <int OFF, int LANES, int N, int A>
__device__ __forceinline__ void fold_lanes(float (&f)[A], int lane, int &base) {
  if constexpr (OFF >= LANES && OFF > 0) {
    if constexpr (N > 1) {
      const bool upper = (lane & OFF) != 0;
#pragma unroll
      for (int q = 0; q < N / 2; ++q) {
        const float send = upper ? f[q] : f[q + N / 2], keep = upper ? f[q + N / 2] : f[q];
        f[q] = keep + __shfl_xor_sync(0xffffffffu, send, OFF);
      }
      base += upper ? N / 2 : 0;
      fold_lanes<OFF / 2, LANES, N / 2>(f, lane, base);
    } else {
      f[0] += __shfl_xor_sync(0xffffffffu, f[0], OFF);
      fold_lanes<OFF / 2, LANES, 1>(f, lane, base);
    }
  }
}

// One slice of slot_sums: the group's eight slots' products into p. UNIFORM:
// their source is `f` for the whole group.
template <int FMT, bool VEC, bool FULL, bool UNIFORM, int DEPTH, typename O>
__device__ __forceinline__ void slice_sums(const EdgeGrad &k, int32_t f, O row, int32_t slice, float2 (&p)[8]) {
  const int sub = threadIdx.x & 7;
  const int32_t b = slice * kMxBlock + sub * 4;
  float2 a[2];
  int32_t cur = UNIFORM ? f : __shfl_sync(0xffffffffu, f, 0, 8);
  load_acts<FMT, O>(k, cur, slice, sub, a);
#pragma unroll
  for (int j0 = 0; j0 < 8; j0 += DEPTH) {
    float4 gv[DEPTH];
#pragma unroll
    for (int j = 0; j < DEPTH; ++j)
      gv[j] = load_grad<VEC, FULL, O>(k.g, __shfl_sync(0xffffffffu, row, j0 + j, 8) + static_cast<O>(b) * 4, k.batch, b);
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
      if (!UNIFORM) {
        const int32_t fj = __shfl_sync(0xffffffffu, f, j0 + j, 8);
        if (fj != cur) {
          cur = fj;
          load_acts<FMT, O>(k, fj, slice, sub, a);
        }
      }
      p[j0 + j] = ffma2(make_float2(gv[j].x, gv[j].y), a[0], p[j0 + j]);
      p[j0 + j] = ffma2(make_float2(gv[j].z, gv[j].w), a[1], p[j0 + j]);
    }
  }
}

// sum_b g[to, b] * a[from, b] over the slices first, first + step, ... of the
// warp's 32 slots; lane l returns slot l's. Eight lanes share a slot, four
// samples each, so one load instruction covers a 32-sample slice of four
// slots. A lane keeps the partial sums of its group's eight slots over every
// slice; halving them across the group's lanes at the end (4 + 2 + 1
// exchanges) leaves each lane its own slot's sum. The arena is source-major but
// for regrown slots: where each group's slots share a source, its codes are
// read and widened once a slice, else once a run.
template <int FMT, bool VEC, bool WIDE, int DEPTH>
__device__ __forceinline__ float slot_sums(const EdgeGrad &k, const Slot &slot, int first, int step) {
  using O = typename Offset<WIDE>::type;
  const bool mine = slot.live(k.n);
  const unsigned live = __ballot_sync(0xffffffffu, mine);
  if (live == 0) return 0.0f;
  const int lane = threadIdx.x & 31;
  // a slot without a gradient stands at its group's first source and at row 0: its sum is not read
  const int lead = __ffs(live >> (lane & 24) & 0xffu) - 1;
  const int32_t first_f = __shfl_sync(0xffffffffu, mine ? slot.f : 0, lead < 0 ? 0 : lead, 8);
  const int32_t f = mine ? slot.f : first_f;
  const bool uniform = __all_sync(0xffffffffu, f == first_f);
  const O row = static_cast<O>(mine ? slot.t : 0) * static_cast<O>(k.batch) * 4;
  float2 p[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) p[j] = make_float2(0.0f, 0.0f);
  for (int32_t slice = first; slice < k.nb; slice += step) {
    const bool full = (slice + 1) * kMxBlock <= k.batch;
    if (full && uniform) slice_sums<FMT, VEC, true, true, DEPTH, O>(k, f, row, slice, p);
    else if (full) slice_sums<FMT, VEC, true, false, DEPTH, O>(k, f, row, slice, p);
    else slice_sums<FMT, VEC, false, false, DEPTH, O>(k, f, row, slice, p);
  }
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = p[j].x + p[j].y;
  int which = 0;
  fold_lanes<4, 1, 8>(q, lane, which);
  return q[0];
}

__device__ __forceinline__ void finish_slot(const EdgeGrad &k, int64_t s, bool live, float sum) {
  const float stat = __fdiv_rn(sum, static_cast<float>(k.batch));
  if (k.dw != nullptr) {
    k.dw[s] = live ? stat : 0.0f;
  } else if (live) {
    float w = k.weight[s];
    opt_step(k.op, stat, w, k.m, k.v, k.t, s);
    k.weight[s] = w;
  }
}

// Every warp takes 32 slots at a time over the whole batch. What costs is the
// gradient rows, 128 bytes a slot and slice, and a shuffle of their offset for
// each load: over 2^22 slots of 65,536 units (128 samples, 119 us) the loads'
// data pipe is 66 % busy, L1 71 %, L2 47 %, and warps wait for loads (7 of 12
// cycles between issues) with 46 % of them resident: latency and that pipe, no
// rate of a memory. MIN_BLOCKS: a warp reads one slice of its rows after
// another, so what the rows' reuse in L1 depends on is the units, not the
// batch. 2^19 slots with three and with four blocks an SM: 1,000 units and 128
// samples 20.4 and 21.7 us, 2,794 and 256 36.0 and 37.7, 16,384 and 256 36.3 and
// 35.7, 65,536 and 256 40.8 and 39.8 (8,192 units: alike).
template <int FMT, bool VEC, bool WIDE, int MIN_BLOCKS>
__global__ void __launch_bounds__(256, MIN_BLOCKS) mx_edge_grad_kernel(EdgeGrad k) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t s = blockIdx.x * int64_t(256) + threadIdx.x; s - (threadIdx.x & 31) < k.cap; s += stride) {
    const Slot slot = load_slot(k, s);
    const float sum = slot_sums<FMT, VEC, WIDE, 8>(k, slot, 0, 1);
    if (s < k.cap) finish_slot(k, s, slot.live(k.n), sum);
  }
}

// Few slots and a long batch: the CTAs of a cluster share 256 slots, CTA r
// taking the slices r, r + ranks, ...; the partial sums join through the
// cluster's shared memory in rank order.
template <int FMT, bool VEC, bool WIDE>
__global__ void __launch_bounds__(256) mx_edge_grad_split_kernel(EdgeGrad k) {
  namespace cg = cooperative_groups;
  __shared__ float part[256];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int64_t base = blockIdx.x / ranks * int64_t(256);
  const Slot slot = load_slot(k, base + threadIdx.x);
  part[threadIdx.x] = slot_sums<FMT, VEC, WIDE, 8>(k, slot, rank, ranks);
  cluster.sync();
  const int at = static_cast<int>(threadIdx.x), share = 256 / ranks;
  if (at / share == rank && base + at < k.cap) {
    float sum = 0.0f;
    for (int r = 0; r < ranks; ++r) sum += cluster.map_shared_rank(part, r)[at];
    finish_slot(k, base + at, slot.live(k.n), sum);
  }
  cluster.sync();  // the peers have read this CTA's sums
}

// --- small nets, many edges ---------------------------------------------------
// Where the slots are a good part of all pairs of units, every pair's sum is a
// matrix product, D[t, f] = sum_b g[t, b] * a[f, b], and the slots pick theirs
// from it. With 256 samples, us so and slot by slot: 400 x 300 units and 2^20
// slots 14 and 74, 1000 x 1000 and 2^19 27 and 37 (43 partly regrown). An 8-bit
// activation is a bfloat16 exactly (four significant bits, a power of two), and
// a float32 gradient is the sum of three bfloat16 (8 + 8 + 8 bits), both down to
// 2^-133, so three tensor-core products, added in float32, hold what the float32
// products do but for parts below that. Only the 64 x 64 tiles that some slot
// touches are computed; the product lies in the caller's scratch, n^2 floats,
// in L2. Latency bounds the middle kernel (18 us of the 27 under the profiler):
// two barriers a 32-sample slice around one buffer, and every source tile
// splits the gradient rows into their parts again (1.5 instructions a cycle,
// 25 % of the warps, first stall shared memory, tensor pipes 30 % busy); the
// launches around it cost as much again.
constexpr int kPairTile = 64, kPairUnits = 4096, kPairSlots = 49152;

__host__ __device__ inline int pair_tiles(uint32_t n) { return static_cast<int>((n + kPairTile - 1) / kPairTile); }

// One bit a tile that some slot touches, by source tile, then target tile. A CTA
// takes slots in a row (they share few sources) and gathers its bits in shared
// memory, so few words reach L2 from it.
__global__ void __launch_bounds__(512) mx_pair_mark_kernel(EdgeGrad k, uint32_t *__restrict__ marks) {
  __shared__ uint32_t bits[kPairUnits / kPairTile * (kPairUnits / kPairTile) / 32];
  const int tiles = pair_tiles(k.n), words = (tiles * tiles + 31) / 32;
  for (int i = threadIdx.x; i < words; i += 512) bits[i] = 0;
  __syncthreads();
  const int64_t each = ((k.cap + gridDim.x - 1) / gridDim.x + 31) & ~int64_t(31);
  const int64_t first = blockIdx.x * each, last = min(k.cap, first + each);
  for (int64_t s = first + threadIdx.x; s < last; s += 512) {
    const Slot slot = load_slot(k, s);
    if (!slot.live(k.n)) continue;
    const int at = slot.f / kPairTile * tiles + slot.t / kPairTile;
    if ((bits[at >> 5] >> (at & 31) & 1) == 0) atomicOr(&bits[at >> 5], 1u << (at & 31));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < words; i += 512)
    if (bits[i] != 0) atomicOr(marks + i, bits[i]);
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void *row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(row))) : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return same_bits<uint32_t>(__floats2bfloat162_rn(lo, hi));
}

__device__ __forceinline__ __nv_bfloat162 cut_bf16(float x, float y) {
  return __halves2bfloat162(__float2bfloat16_rz(x), __float2bfloat16_rz(y));
}

// Two gradients as their three bfloat16 parts. The first two are rounded toward
// zero: 8 + 8 + 8 bits hold a float32 all the same, and the largest float32
// values, which would round up to infinity, stay finite. One that is not finite
// stands in the first part alone.
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&p)[3]) {
  const __nv_bfloat162 h = cut_bf16(x, y);
  const float2 hf = __bfloat1622float2(h);
  float rx = __fsub_rn(x, hf.x), ry = __fsub_rn(y, hf.y);
  if (!isfinite(hf.x)) rx = 0.0f;
  if (!isfinite(hf.y)) ry = 0.0f;
  const __nv_bfloat162 m = cut_bf16(rx, ry);
  const float2 mf = __bfloat1622float2(m);
  p[0] = same_bits<uint32_t>(h);
  p[1] = same_bits<uint32_t>(m);
  p[2] = pack_bf16(__fsub_rn(rx, mf.x), __fsub_rn(ry, mf.y));
}

// A CTA of eight warps a tile; a warp 16 x 32 of it. 32 samples (a block) at a
// time: the gradients' parts and the activations go to shared memory in
// bfloat16 while the next block's words are on their way to registers. Rows of
// 40 elements keep ldmatrix's eight rows on banks of their own.
template <int FMT, bool VEC>
__global__ void __launch_bounds__(256) mx_pair_product_kernel(EdgeGrad k, const uint32_t *__restrict__ marks,
                                                              float *__restrict__ pairs) {
  constexpr int kPitch = 40;
  __shared__ __align__(16) uint16_t gs[3][kPairTile][kPitch], as[kPairTile][kPitch];
  const int tiles = pair_tiles(k.n);
  const int mark = blockIdx.x * tiles + blockIdx.y;
  if (marks != nullptr && (marks[mark >> 5] >> (mark & 31) & 1) == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t t0 = blockIdx.y * kPairTile, f0 = blockIdx.x * kPairTile;
  const int wm = (warp >> 1) * 16, wn = (warp & 1) * 32;
  // this thread's words of a block: two quads of gradients, rows tid / 8 + 32 i; eight codes, a quarter of a row
  const int gq = tid & 7, gr = tid >> 3, ar = tid >> 2, aq = tid & 3;
  const bool a_in = f0 + ar < k.n;
  float4 g[2];
  uint2 c;
  uint32_t sc;
  const auto fetch = [&](int32_t slice) {
    const int32_t b = slice * kMxBlock + gq * 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t row = t0 + gr + 32 * i;
      g[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < k.n) g[i] = load_grad<VEC, false, uint64_t>(k.g, (static_cast<uint64_t>(row) * k.batch + b) * 4, k.batch, b);
    }
    c = make_uint2(0, 0);
    sc = 0;
    if (a_in) {
      const int64_t blk = static_cast<int64_t>(f0 + ar) * k.nb + slice;
      c = __ldg(reinterpret_cast<const uint2 *>(k.codes) + blk * 4 + aq);
      sc = __ldg(k.scales + blk);
    }
  };
  float d[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.0f;
  fetch(0);
  for (int32_t slice = 0; slice < k.nb; ++slice) {
    __syncthreads();  // the last block has been read
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t lo[3], hi[3];
      split_bf16(g[i].x, g[i].y, lo);
      split_bf16(g[i].z, g[i].w, hi);
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<uint2 *>(&gs[p][gr + 32 * i][gq * 4]) = make_uint2(lo[p], hi[p]);
    }
    {
      const float s = mx_scale_value(sc);
      const uint32_t w[2] = {c.x, c.y};
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        __half2 h[2];
        mx_decode_word<FMT>(w[i], h);
        const float2 x = __half22float2(h[0]), y = __half22float2(h[1]);
        o[2 * i] = pack_bf16(__fmul_rn(x.x, s), __fmul_rn(x.y, s));
        o[2 * i + 1] = pack_bf16(__fmul_rn(y.x, s), __fmul_rn(y.y, s));
      }
      *reinterpret_cast<uint4 *>(&as[ar][aq * 8]) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (slice + 1 < k.nb) fetch(slice + 1);
    __syncthreads();
    // a block's sum by itself, then added with rounding: the tensor cores cut what lies below their largest addend's
    // last bit, and over a whole batch in one accumulator that was 9 times a float32 sum's error (256 samples)
    float e[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j][0] = e[j][1] = e[j][2] = e[j][3] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < kMxBlock; kk += 16) {
      // B fragments of the warp's 32 columns: two loads of 16 columns x 16 samples
      uint32_t b[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        ldmatrix_x4(b[j], &as[wn + j * 16 + (lane & 7) + ((lane >> 4) << 3)][kk + ((lane >> 3) & 1) * 8]);
#pragma unroll
      for (int p = 2; p >= 0; --p) {  // the smallest parts first
        uint32_t a[4];
        ldmatrix_x4(a, &gs[p][wm + (lane & 15)][kk + (lane >> 4) * 8]);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_bf16(e[j], a, b[j >> 1][(j & 1) * 2], b[j >> 1][(j & 1) * 2 + 1]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int z = 0; z < 4; ++z) d[j][z] += e[j][z];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t t = t0 + wm + (lane >> 2) + 8 * h, f = f0 + wn + j * 8 + (lane & 3) * 2;
      if (t >= k.n) continue;
      float *o = pairs + static_cast<int64_t>(t) * k.n + f;
      if (f < k.n) o[0] = d[j][2 * h];
      if (f + 1 < k.n) o[1] = d[j][2 * h + 1];
    }
}

__global__ void __launch_bounds__(256) mx_pair_pick_kernel(EdgeGrad k, const float *__restrict__ pairs) {
  for (int64_t s = blockIdx.x * int64_t(256) + threadIdx.x; s < k.cap; s += static_cast<int64_t>(gridDim.x) * 256) {
    const Slot slot = load_slot(k, s);
    const bool live = slot.live(k.n);
    finish_slot(k, s, live, live ? __ldg(pairs + static_cast<int64_t>(slot.t) * k.n + slot.f) : 0.0f);
  }
}

// ---------------------------------------------------------------------------
// out[units[i], :] = act(sum_e w[e] * x[src[e], :])
// ---------------------------------------------------------------------------
struct Conns {
  int32_t num_dst, fmt;
  int64_t num_edges, num_blocks;
  const int32_t *__restrict__ units;
  const int64_t *__restrict__ offsets;
  const int32_t *__restrict__ src;
  const float *__restrict__ weight;
  const int64_t *__restrict__ block_offsets;
  const uint8_t *__restrict__ codes;
  const uint8_t *__restrict__ scales;
};

// The weight of in-edge `edge`: element `at` (under 32) of block `blk`.
__device__ __forceinline__ float conn_weight(const Conns &c, int64_t edge, int64_t blk, int at) {
  if (c.fmt == PXB_MX_F32) return __ldg(c.weight + edge);
  if (blk >= c.num_blocks) return 0.0f;
  const float s = mx_scale_value(__ldg(c.scales + blk));
  float v;
  if (c.fmt == PXB_MX_E2M1) {
    v = mx_decode2<PXB_MX_E2M1>((__ldg(c.codes + blk * 16 + (at >> 1)) >> (4 * (at & 1))) & 0xfu).x;
  } else {
    const uint32_t code = __ldg(c.codes + blk * 32 + at);
    v = c.fmt == PXB_MX_E4M3 ? mx_decode2<PXB_MX_E4M3>(code).x : mx_decode2<PXB_MX_E5M2>(code).x;
  }
  return __fmul_rn(v, s);
}

// A lane's octet of results: float32, or its block's codes (every lane of the
// warp calls; the four lanes of a block are neighbours).
template <int OF>
__device__ __forceinline__ void store_codes(const float (&v)[8], bool on, int64_t octet, uint8_t *codes,
                                            uint8_t *scales) {
  uint32_t m = mx_amax8(v);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const uint32_t s = mx_scale_byte<OF>(m);
  const uint64_t c = mx_encode8<OF>(v, s, false);
  if (on) {
    mx_store8<OF>(codes, octet, c);
    if ((octet & 3) == 0) scales[octet >> 2] = static_cast<uint8_t>(s);
  }
}

struct Out {
  int32_t fmt;
  uint32_t rows;
  float *x;
  uint8_t *codes, *scales;
  bool vec;  // float32 rows on 16-byte boundaries
};

struct Rows {
  const float *__restrict__ x;
  const uint8_t *__restrict__ codes;
  const uint8_t *__restrict__ scales;
  int32_t batch, nb;
  uint32_t rows;
};

// A launch's items: (destination, chunk of the batch), `wpd` warps of a CTA to
// an item, 8 / wpd items a tile, a tile a cluster (of one CTA or more).
struct Items {
  uint32_t total, tiles;
  FastDiv chunks;
  int wpd;
};

struct Item {
  int64_t e0, blk0;
  int32_t blocks, tail;  // of 32 edges, the last with `tail`
  int32_t chunk;
};

__device__ __forceinline__ Item load_item(const Conns &c, const Items &n, uint32_t item) {
  const uint32_t i = n.chunks.div(item);
  Item t;
  t.chunk = static_cast<int32_t>(item - i * n.chunks.d);
  t.e0 = max(int64_t(0), __ldg(c.offsets + i));
  t.blk0 = c.fmt == PXB_MX_F32 ? 0 : max(int64_t(0), __ldg(c.block_offsets + i));
  const int64_t edges = max(int64_t(0), min(c.num_edges, __ldg(c.offsets + i + 1)) - t.e0);
  t.blocks = static_cast<int32_t>(min((edges + 31) >> 5, int64_t(0x7fffffff)));
  t.tail = static_cast<int32_t>(edges - (static_cast<int64_t>(t.blocks) - 1) * 32);
  return t;
}

// Lane's edge of block k: its source (-1 for none) and weight.
__device__ __forceinline__ void load_edge(const Conns &c, const Item &it, int32_t k, int lane, uint32_t rows, int32_t &s,
                                          float &w) {
  s = -1;
  w = 0.0f;
  if (k < it.blocks - 1 || (k == it.blocks - 1 && lane < it.tail)) {
    const int64_t e = it.e0 + static_cast<int64_t>(k) * 32 + lane;
    const int32_t v = __ldg(c.src + e);
    const float x = conn_weight(c, e, it.blk0 + k, lane);
    if (static_cast<uint32_t>(v) < rows) s = v, w = x;
  }
}

// One octet of an item's sums -> activation -> float32 or codes (every lane of
// the warp calls; the four lanes of a block are neighbours).
template <int CHUNK, typename Sum>
__device__ __forceinline__ void finish_octet(const Conns &c, const Rows &r, int act_kind, const Out &out, const Items &n,
                                             uint32_t item, int o, bool live, Sum sum) {
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int32_t u = -1, b = 0;
  if (live) {
    const uint32_t i = n.chunks.div(item);
    u = __ldg(c.units + i);
    b = static_cast<int32_t>(item - i * n.chunks.d) * CHUNK + o;
    sum(v);
#pragma unroll
    for (int z = 0; z < 8; ++z) v[z] = b + z < r.batch ? mx_act(act_kind, v[z]) : 0.0f;
  }
  const bool on = live && b < r.nb * kMxBlock && static_cast<uint32_t>(u) < out.rows;
  if (out.fmt == PXB_MX_F32) {
    float *dst = out.x + static_cast<int64_t>(u) * r.batch + b;
    if (on && out.vec && b + 8 <= r.batch) {
      reinterpret_cast<float4 *>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4 *>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if (on) {
#pragma unroll
      for (int z = 0; z < 8; ++z)
        if (b + z < r.batch) dst[z] = v[z];
    }
  } else {
    const int64_t at = static_cast<int64_t>(u) * r.nb * 4 + (b >> 3);
    if (out.fmt == PXB_MX_E4M3) store_codes<PXB_MX_E4M3>(v, on, at, out.codes, out.scales);
    else if (out.fmt == PXB_MX_E5M2) store_codes<PXB_MX_E5M2>(v, on, at, out.codes, out.scales);
    else store_codes<PXB_MX_E2M1>(v, on, at, out.codes, out.scales);
  }
}

// The sums of a tile's items lie in shared memory, one set a warp (`stride`
// floats apart, CHUNK samples each). An item of one warp is finished by it;
// else the CTA's first threads, of the cluster's first CTA, join an item's sets
// in order and finish it.
template <int CHUNK>
__device__ __forceinline__ void finish_items(const Conns &c, const Rows &r, int act_kind, const Out &out, const Items &n,
                                             uint32_t tile, int ranks, float *part, int stride) {
  constexpr int kOctets = (CHUNK < kMxBlock ? kMxBlock : CHUNK) / 8;  // an item's octets: whole blocks
  namespace cg = cooperative_groups;
  const auto add = [](float(&v)[8], const float *q, int o) {
#pragma unroll
    for (int z = 0; z < 8; ++z)
      if (CHUNK % 8 == 0 ? o < CHUNK : o + z < CHUNK) v[z] += q[o + z];
  };
  if (n.wpd == 1 && ranks == 1) {
    __syncwarp();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t item = tile * 8 + warp;
#pragma unroll
    for (int t = 0; t < (kOctets + 31) / 32 * 32; t += 32) {
      const int o = (t + lane) * 8;
      finish_octet<CHUNK>(c, r, act_kind, out, n, item, o, item < n.total && t + lane < kOctets,
                               [&](float(&v)[8]) { add(v, part + warp * stride, o); });
    }
    __syncwarp();
    return;
  }
  const cg::cluster_group cluster = cg::this_cluster();
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  if (ranks == 1 || cluster.block_rank() == 0) {
    const int per_cta = 8 / n.wpd;
    // every warp steps through whole rounds, so that a block's four lanes meet in the shuffles
    for (int t = threadIdx.x; t < ((per_cta * kOctets + 31) & ~31); t += 256) {
      const int j = t / kOctets, o = (t - j * kOctets) * 8;
      const uint32_t item = tile * per_cta + j;
      finish_octet<CHUNK>(c, r, act_kind, out, n, item, o, j < per_cta && item < n.total, [&](float(&v)[8]) {
        for (int k = 0; k < ranks; ++k) {
          const float *q = ranks > 1 ? cluster.map_shared_rank(part, k) : part;
          for (int m = 0; m < n.wpd; ++m) add(v, q + (j * n.wpd + m) * stride, o);
        }
      });
    }
  }
  if (ranks > 1) cluster.sync();
  else __syncthreads();
}

// 16 bytes of a source row (a piece: a block of 32 samples in e2m1, 16 samples
// in 8 bits, 4 in float32) and the factor of its values.
template <int XF>
struct Piece {
  static constexpr int kSamples = XF == PXB_MX_F32 ? 4 : XF == PXB_MX_E2M1 ? 32 : 16;
  static constexpr int kMaxLanes = XF == PXB_MX_F32 ? 32 : 256 / kSamples;  // lanes a row takes at most
  uint4 v;
  float w;
};

// A piece of the row at byte offset `row` for an edge of weight w. `valid`:
// the edge has a source; where not, `row` is 0, whose values the factor 0 (for
// e2m1, whose codes are all finite) or zeros in their place leave out.
template <int XF, bool VEC, typename O>
__device__ __forceinline__ Piece<XF> load_piece(const Rows &r, O row, float w, bool valid, int32_t piece) {
  Piece<XF> p;
  if constexpr (XF == PXB_MX_F32) {
    p.v = make_uint4(0, 0, 0, 0);
    p.w = valid ? w : 0.0f;
    if (!valid) return p;
    const float *x = reinterpret_cast<const float *>(reinterpret_cast<const char *>(r.x) + row) + piece * 4;
    if (VEC) {
      p.v = __ldg(reinterpret_cast<const uint4 *>(x));
    } else {
      const uint32_t *u = reinterpret_cast<const uint32_t *>(x);
      const int32_t left = r.batch - piece * 4;
      p.v.x = __ldg(u);
      if (left > 1) p.v.y = __ldg(u + 1);
      if (left > 2) p.v.z = __ldg(u + 2);
      if (left > 3) p.v.w = __ldg(u + 3);
    }
  } else {
    constexpr int kShift = XF == PXB_MX_E2M1 ? 4 : 5;  // a block's bytes of codes
    p.v = __ldg(reinterpret_cast<const uint4 *>(r.codes + row) + piece);
    const uint32_t s = __ldg(r.scales + (row >> kShift) + (piece >> (kShift - 4)));
    // as mx_scale_value, but for 255: infinite, so that the sums are not finite and sum_scaled takes the item
    const float f = __fmul_rn(w, __uint_as_float(max(s << 23, 0x00400000u)));
    p.w = valid ? f : 0.0f;
    if (XF != PXB_MX_E2M1 && !valid) p.v = make_uint4(0, 0, 0, 0);
  }
  return p;
}

// acc += w * values, two at a time.
template <int XF>
__device__ __forceinline__ void add_piece(const Piece<XF> &p, float2 (&acc)[Piece<XF>::kSamples / 2]) {
  const uint32_t v[4] = {p.v.x, p.v.y, p.v.z, p.v.w};
  const float2 w = make_float2(p.w, p.w);
  if constexpr (XF == PXB_MX_F32) {
    acc[0] = ffma2(w, make_float2(__uint_as_float(v[0]), __uint_as_float(v[1])), acc[0]);
    acc[1] = ffma2(w, make_float2(__uint_as_float(v[2]), __uint_as_float(v[3])), acc[1]);
  } else {
    constexpr int kPairs = 32 / (2 * MxFormat<XF>::bits);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h[kPairs];
      mx_decode_word<XF>(v[i], h);
#pragma unroll
      for (int q = 0; q < kPairs; ++q) acc[i * kPairs + q] = ffma2(w, __half22float2(h[q]), acc[i * kPairs + q]);
    }
  }
}

// An item's sums again, each value with its scale before the weight, as a
// float32 row would hold it: for where weight times scale left float32's range
// though products with the block's small values do not (or a block is not a
// number). add_piece then had an infinite factor, which leaves every sum of its
// piece infinite or not a number, so one look at one sum an item finds it.
// (The order does not matter otherwise: a power of two, and one rounding.)
template <int XF, int LANES, typename O>
__device__ __forceinline__ void sum_scaled(const Conns &c, const Rows &r, const Item &it, int32_t first, int32_t step,
                                           int32_t piece, O row_bytes, float2 (&acc)[Piece<XF>::kSamples / 2]) {
  constexpr int kShift = XF == PXB_MX_E2M1 ? 4 : 5, kPairs = 32 / (2 * MxFormat<XF>::bits), kGroups = 32 / LANES;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int q = 0; q < Piece<XF>::kSamples / 2; ++q) acc[q] = make_float2(0.0f, 0.0f);
#pragma unroll 1
  for (int32_t k = first; k < it.blocks; k += step) {
    int32_t src;
    float weight;
    load_edge(c, it, k, lane, r.rows, src, weight);
#pragma unroll 1
    for (int j = 0; j < 32; j += kGroups) {
      const int32_t f = __shfl_sync(0xffffffffu, src, j + lane / LANES);
      const float w = __shfl_sync(0xffffffffu, weight, j + lane / LANES);
      if (f < 0) continue;
      const O row = static_cast<O>(f) * row_bytes;
      const uint4 codes = __ldg(reinterpret_cast<const uint4 *>(r.codes + row) + piece);
      const float s = mx_scale_value(__ldg(r.scales + (row >> kShift) + (piece >> (kShift - 4))));
      const uint32_t v[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __half2 h[kPairs];
        mx_decode_word<XF>(v[i], h);
#pragma unroll
        for (int q = 0; q < kPairs; ++q) {
          const float2 x = __half22float2(h[q]);
          acc[i * kPairs + q] = ffma2(make_float2(w, w), make_float2(__fmul_rn(x.x, s), __fmul_rn(x.y, s)),
                                      acc[i * kPairs + q]);
        }
      }
    }
  }
}

// A warp takes a block of 32 edges of an item: lane j holds edge j's row and
// weight, and fetches the next block's while this one's rows come. A row is
// LANES pieces, so 32 / LANES edges are read side by side, each load
// instruction full, two in flight a lane. MX rows: the loop waits for loads and
// issues about three instructions a pair of samples (two conversions and a
// paired FMA, on two pipes), so warps count for more than loads a warp: 64
// registers, 32 warps an SM (32,768 x 96 in-edges, 100 samples of e2m1, 89 us:
// 2.7 instructions a cycle, ALU pipe 48 %, L2 22 %). Float32 rows: two loads in
// flight a lane are the bound (256 samples, 343 us: 9.4 TB/s of rows, L2 40 %,
// 14 cycles of waiting for loads between issues; a 1000 x 1000 pair, 19 us).
template <int XF, int LANES, bool VEC, bool WIDE>
__global__ void __launch_bounds__(256, 4) mx_product_kernel(Conns c, Rows r, int act_kind, Out out, Items n) {
  using O = typename Offset<WIDE>::type;
  constexpr int A = Piece<XF>::kSamples, kGroups = 32 / LANES, kChunk = LANES * A, kDepth = LANES < 2 ? 1 : 2;
  __shared__ __align__(16) float part[8][kChunk];
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LANES, grp = lane / LANES;
  const int team = warp / n.wpd, member = warp % n.wpd, per_cta = 8 / n.wpd;
  const int32_t pieces = XF == PXB_MX_F32 ? (r.batch + 3) / 4 : r.nb * (kMxBlock / A);
  const O row_bytes = XF == PXB_MX_F32 ? static_cast<O>(r.batch) * 4 : static_cast<O>(pieces) * 16;
  const int32_t step = n.wpd * ranks;
  for (uint32_t tile = blockIdx.x / ranks; tile < n.tiles; tile += gridDim.x / ranks) {
    const uint32_t item = tile * per_cta + team;
    float2 acc[A / 2];
#pragma unroll
    for (int q = 0; q < A / 2; ++q) acc[q] = make_float2(0.0f, 0.0f);
    if (item < n.total) {
      const Item it = load_item(c, n, item);
      const int32_t piece = min(it.chunk * LANES + sub, pieces - 1);  // past the row: the last again, its sums unread
      int32_t k = member + rank * n.wpd;
      if constexpr (LANES == 1) {  // four blocks at once: a lane's edge has one piece
#pragma unroll 1
        for (; k < it.blocks; k += 4 * step) {
          int32_t s[4];
          float w[4];
          Piece<XF> p[4];
#pragma unroll
          for (int d = 0; d < 4; ++d) load_edge(c, it, k + d * step, lane, r.rows, s[d], w[d]);
#pragma unroll
          for (int d = 0; d < 4; ++d)
            p[d] = load_piece<XF, VEC, O>(r, s[d] < 0 ? O(0) : static_cast<O>(s[d]) * row_bytes, w[d], s[d] >= 0, piece);
#pragma unroll
          for (int d = 0; d < 4; ++d) add_piece<XF>(p[d], acc);
        }
      }
      int32_t next;
      float next_w;
      load_edge(c, it, k, lane, r.rows, next, next_w);
#pragma unroll 1
      for (; k < it.blocks; k += step) {
        const O row = next < 0 ? O(0) : static_cast<O>(next) * row_bytes;
        const unsigned valid = __ballot_sync(0xffffffffu, next >= 0);
        const float w = next_w;
        load_edge(c, it, k + step, lane, r.rows, next, next_w);
        const int cnt = k == it.blocks - 1 ? it.tail : 32;
#pragma unroll 1
        for (int j = 0; j < cnt; j += kGroups * kDepth) {
          Piece<XF> p[kDepth];
#pragma unroll
          for (int d = 0; d < kDepth; ++d) {
            const int at = j + d * kGroups + grp;
            p[d] = load_piece<XF, VEC, O>(r, __shfl_sync(0xffffffffu, row, at), __shfl_sync(0xffffffffu, w, at),
                                          (valid >> at) & 1, piece);
          }
#pragma unroll
          for (int d = 0; d < kDepth; ++d) add_piece<XF>(p[d], acc);
        }
      }
      if constexpr (XF != PXB_MX_F32) {
        if (__any_sync(0xffffffffu, !(fabsf(acc[0].x) < INFINITY)))
          sum_scaled<XF, LANES, O>(c, r, it, member + rank * n.wpd, step, piece, row_bytes, acc);
      }
    }
    // the edges read side by side join
    float f[A];
#pragma unroll
    for (int q = 0; q < A / 2; ++q) f[2 * q] = acc[q].x, f[2 * q + 1] = acc[q].y;
    int base = sub * A;
    fold_lanes<16, LANES, A>(f, lane, base);
    constexpr int kHeld = A > kGroups ? A / kGroups : 1;
#pragma unroll
    for (int q = 0; q < kHeld; ++q) part[warp][base + q] = f[q];
    finish_items<kChunk>(c, r, act_kind, out, n, tile, ranks, &part[0][0], kChunk);
  }
}

// Up to 16 samples (4 * Q) of float32 rows and many short destinations: eight
// lanes a destination, four consecutive edges of a weight block each (their
// codes are one load, their scale one), so a warp works on four destinations
// and the set-up and the ending of each cost a quarter of a warp's. 32,768
// destinations of 64 in-edges: one sample 10 us against 27 with a warp each,
// eight samples 18 against 38, 16 samples 34 against 42 (rows that need single
// loads: 13 samples 52 against 44, so past eight samples only whole vectors).
template <int Q, bool VEC>
__global__ void __launch_bounds__(256) mx_product_short_kernel(Conns c, Rows r, int act_kind, Out out) {
  constexpr int N = 4 * Q;
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const int64_t teams = static_cast<int64_t>(gridDim.x) * 32;
  // whole warps step together (the shuffles below take every lane)
  for (int64_t i0 = (blockIdx.x * int64_t(256) + threadIdx.x) / 32 * 4; i0 < c.num_dst; i0 += teams) {
    const int64_t i = i0 + (lane >> 3);
    float f[N];
#pragma unroll
    for (int b = 0; b < N; ++b) f[b] = 0.0f;
    if (i < c.num_dst) {
      const int64_t e0 = max(int64_t(0), __ldg(c.offsets + i)), e1 = min(c.num_edges, __ldg(c.offsets + i + 1));
      int64_t blk = c.fmt == PXB_MX_F32 ? 0 : max(int64_t(0), __ldg(c.block_offsets + i));
      for (int64_t e = e0 + sub * 4; e < e1; e += 32, ++blk) {
        const int cnt = static_cast<int>(min(int64_t(4), e1 - e));
        int32_t s[4];
        float w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] = q < cnt ? __ldg(c.src + e + q) : -1;
        if (c.fmt == PXB_MX_F32) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q < cnt) w[q] = __ldg(c.weight + e + q);
        } else if (blk < c.num_blocks) {
          const float scale = mx_scale_value(__ldg(c.scales + blk));
          float2 lo, hi;
          if (c.fmt == PXB_MX_E2M1) {
            const uint32_t code = __ldg(reinterpret_cast<const uint16_t *>(c.codes + blk * 16) + sub);
            lo = mx_decode2<PXB_MX_E2M1>(code & 0xffu), hi = mx_decode2<PXB_MX_E2M1>(code >> 8);
          } else {
            const uint32_t code = __ldg(reinterpret_cast<const uint32_t *>(c.codes + blk * 32) + sub);
            if (c.fmt == PXB_MX_E4M3) lo = mx_decode2<PXB_MX_E4M3>(code & 0xffffu), hi = mx_decode2<PXB_MX_E4M3>(code >> 16);
            else lo = mx_decode2<PXB_MX_E5M2>(code & 0xffffu), hi = mx_decode2<PXB_MX_E5M2>(code >> 16);
          }
          w[0] = __fmul_rn(lo.x, scale), w[1] = __fmul_rn(lo.y, scale);
          w[2] = __fmul_rn(hi.x, scale), w[3] = __fmul_rn(hi.y, scale);
        }
        constexpr int kAtOnce = Q == 4 ? 2 : 4;  // edges whose rows are in flight together
#pragma unroll
        for (int q0 = 0; q0 < 4; q0 += kAtOnce) {
          float x[kAtOnce][N];
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q) {
            const bool on = static_cast<uint32_t>(s[q0 + q]) < r.rows;
            const float *p = r.x + static_cast<int64_t>(on ? s[q0 + q] : 0) * r.batch;
            if (!on) w[q0 + q] = 0.0f;
            if constexpr (VEC) {
#pragma unroll
              for (int z = 0; z < Q; ++z) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (on && z * 4 < r.batch) v = __ldg(reinterpret_cast<const float4 *>(p) + z);
                x[q][4 * z] = v.x, x[q][4 * z + 1] = v.y, x[q][4 * z + 2] = v.z, x[q][4 * z + 3] = v.w;
              }
            } else {
#pragma unroll
              for (int b = 0; b < N; ++b) x[q][b] = on && b < r.batch ? __ldg(p + b) : 0.0f;
            }
          }
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
            for (int b = 0; b < N; ++b) f[b] = fmaf(w[q0 + q], x[q][b], f[b]);
        }
      }
    }
    const int32_t u = i < c.num_dst ? __ldg(c.units + i) : -1;
    const bool on = static_cast<uint32_t>(u) < out.rows;
    if (out.fmt == PXB_MX_F32) {
      int base = 0;
      fold_lanes<4, 1, N>(f, lane, base);
#pragma unroll
      for (int z = 0; z < (N > 8 ? N / 8 : 1); ++z)
        if (on && base + z < r.batch) out.x[static_cast<int64_t>(u) * r.batch + base + z] = mx_act(act_kind, f[z]);
      continue;
    }
#pragma unroll
    for (int off = 4; off > 0; off >>= 1)  // in fold_lanes' order: the same sums
#pragma unroll
      for (int b = 0; b < N; ++b) f[b] += __shfl_xor_sync(0xffffffffu, f[b], off);
    if (!on || sub >= 4) continue;  // a lane an octet of the block
    uint32_t m = 0;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < N; ++b) {
      const float y = b < r.batch ? mx_act(act_kind, f[b]) : 0.0f;
      m = max(m, __float_as_uint(y) & 0x7fffffffu);
      if (sub == b / 8) v[b % 8] = y;
    }
    const int64_t at = static_cast<int64_t>(u) * 4 + sub;
    uint32_t sb;
    if (out.fmt == PXB_MX_E2M1) {
      sb = mx_scale_byte<PXB_MX_E2M1>(m);
      mx_store8<PXB_MX_E2M1>(out.codes, at, mx_encode8<PXB_MX_E2M1>(v, sb, false));
    } else if (out.fmt == PXB_MX_E4M3) {
      sb = mx_scale_byte<PXB_MX_E4M3>(m);
      mx_store8<PXB_MX_E4M3>(out.codes, at, mx_encode8<PXB_MX_E4M3>(v, sb, false));
    } else {
      sb = mx_scale_byte<PXB_MX_E5M2>(m);
      mx_store8<PXB_MX_E5M2>(out.codes, at, mx_encode8<PXB_MX_E5M2>(v, sb, false));
    }
    if (sub == 0) out.scales[u] = static_cast<uint8_t>(sb);
  }
}

// How many warps share a destination (`wpd`, up to a CTA's eight) and, past
// that, CTAs: until every SM has 32 warps' worth or a warp has one block of 32
// edges left. By the mean in-degree: where the items fill the SMs, a destination
// far above it is one warp's (or eight lanes') work from end to end. 32,768
// destinations of 64 in-edges, one of them with 0 / 4,096 / 65,536 more: one
// float32 sample 12 / 54 / 690 us, 64 samples of e2m1 49 / 156 / 1,980 us.
static void split_items(int64_t items, int64_t mean, int *wpd, int *ranks) {
  const int64_t warps = static_cast<int64_t>(sm_count()) * 32;
  *wpd = *ranks = 1;
  while (*wpd < 8 && items * *wpd < warps && mean > 32 * *wpd) *wpd *= 2;
  if (*wpd == 8)
    while (*ranks < 8 && items * 8 * *ranks < warps && mean > 32 * 8 * *ranks) *ranks *= 2;
}

template <auto KERNEL>
static int launch_items(const Conns &c, const Rows &r, int act, const Out &out, int32_t chunks, cudaStream_t st) {
  const int64_t items = static_cast<int64_t>(c.num_dst) * chunks;
  PXB_REQUIRE(items < (int64_t(1) << 32) - 8, "pxb_mx_product: %lld destinations and chunks are past 2^32",
              static_cast<long long>(items));
  int wpd, ranks;
  split_items(items, c.num_edges / c.num_dst, &wpd, &ranks);
  const int64_t tiles = (items * wpd + 7) / 8;
  const Items n{static_cast<uint32_t>(items), static_cast<uint32_t>(tiles), FastDiv(static_cast<uint32_t>(chunks)), wpd};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(mx_grid<KERNEL>(tiles, 1, 256) * ranks));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  PXB_CUDA(cudaLaunchKernelEx(&cfg, KERNEL, c, r, act, out, n));
  return PXB_OK;
}

template <int XF, int LANES>
static int launch_product(const Conns &c, const Rows &r, int act, const Out &out, bool vec, cudaStream_t st) {
  if constexpr (XF == PXB_MX_F32 && (LANES == 1 || LANES == 2 || LANES == 4)) {
    // four short destinations a warp, as soon as that fills the SMs half
    if ((LANES < 4 || vec) && r.batch <= 4 * LANES && c.num_dst >= sm_count() * 64 && c.num_edges / c.num_dst <= 512) {
#define PXB_SHORT(V)                                                                                               \
  mx_product_short_kernel<LANES, V>                                                                                \
      <<<mx_grid<mx_product_short_kernel<LANES, V>>(c.num_dst, 32, 256), 256, 0, st>>>(c, r, act, out)
      if (vec) PXB_SHORT(true);
      else if constexpr (LANES < 4) PXB_SHORT(false);
#undef PXB_SHORT
      PXB_LAUNCHED("mx_product_short_kernel");
      return PXB_OK;
    }
  }
  const int32_t pieces = XF == PXB_MX_F32 ? (r.batch + 3) / 4 : r.nb * (kMxBlock / Piece<XF>::kSamples);
  if constexpr (LANES < Piece<XF>::kMaxLanes) {
    if (pieces > LANES) return launch_product<XF, LANES * 2>(c, r, act, out, vec, st);
  }
  const int32_t chunks = (pieces + LANES - 1) / LANES;
  const int64_t row_bytes = XF == PXB_MX_F32 ? int64_t(r.batch) * 4 : int64_t(pieces) * 16;
  const bool wide = r.rows * row_bytes >= (int64_t(1) << 32);
  if constexpr (XF == PXB_MX_F32) {
    if (!vec)
      return wide ? launch_items<mx_product_kernel<XF, LANES, false, true>>(c, r, act, out, chunks, st)
                  : launch_items<mx_product_kernel<XF, LANES, false, false>>(c, r, act, out, chunks, st);
  }
  return wide ? launch_items<mx_product_kernel<XF, LANES, true, true>>(c, r, act, out, chunks, st)
              : launch_items<mx_product_kernel<XF, LANES, true, false>>(c, r, act, out, chunks, st);
}

// Scratch of the pair product (0 where slot by slot is as good): the pairs'
// sums, then a bit a tile. At a twelfth of all pairs of units the two are alike
// (300,000 slots of 2,000 units: 25 us each). The pairs are those of all the
// net's units, not of the levels that a bucket joins, so a deeper net's bucket
// stays slot by slot although its own level pair is as full (2^19 slots of 1000
// x 1000 units: 27 us in a net of 2,000 units, 37 in one of 2,794); and
// enough work to pay for four launches. A tile is one CTA over the whole batch,
// so a small net's long batch is few CTAs' work however many slots it has, and
// the slots have to be worth that: 64 units, 4,096 samples, slot by slot and so:
// 32,768 slots 63 and 82 us, 65,536 slots 112 and 83 (16, 128 and 300 units and
// 1,024 to 16,384 samples: the same border).
static size_t pair_scratch(int64_t cap, int32_t batch, int64_t n) {
  if (n > kPairUnits || cap * 12 < n * n || cap * batch < (int64_t(1) << 26) || cap < kPairSlots) return 0;
  const int64_t tiles = pair_tiles(static_cast<uint32_t>(n));
  return static_cast<size_t>(n * n * 4 + (tiles * tiles + 31) / 32 * 4);
}

template <int FMT, bool VEC>
static int launch_pairs(const EdgeGrad &k, void *scratch, cudaStream_t st) {
  float *pairs = static_cast<float *>(scratch);
  uint32_t *marks = reinterpret_cast<uint32_t *>(pairs + static_cast<int64_t>(k.n) * k.n);
  const int tiles = pair_tiles(k.n);
  if (tiles * tiles <= sm_count()) {
    marks = nullptr;  // a tile an SM at most: all of them
  } else {
    PXB_CUDA(cudaMemsetAsync(marks, 0, (static_cast<size_t>(tiles) * tiles + 31) / 32 * 4, st));
    mx_pair_mark_kernel<<<grid_for(k.cap, 512, 2), 512, 0, st>>>(k, marks);
    PXB_LAUNCHED("mx_pair_mark_kernel");
  }
  mx_pair_product_kernel<FMT, VEC><<<dim3(tiles, tiles), 256, 0, st>>>(k, marks, pairs);
  PXB_LAUNCHED("mx_pair_product_kernel");
  mx_pair_pick_kernel<<<grid_for(k.cap, 256, 8), 256, 0, st>>>(k, pairs);
  PXB_LAUNCHED("mx_pair_pick_kernel");
  return PXB_OK;
}

template <int FMT, bool VEC, bool WIDE>
static int launch_edge_grad(const EdgeGrad &k, cudaStream_t st) {
  const int64_t blocks = (k.cap + 255) / 256;
  int ranks = 1;
  while (ranks < 8 && ranks * 2 <= k.nb && blocks * ranks <= sm_count()) ranks *= 2;
  if (ranks > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks * ranks));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ranks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    PXB_CUDA(cudaLaunchKernelEx(&cfg, mx_edge_grad_split_kernel<FMT, VEC, WIDE>, k));
    return PXB_OK;
  }
  const int grid = grid_for((k.cap + 31) / 32, 8, 8);
  if (k.n <= 4096) mx_edge_grad_kernel<FMT, VEC, WIDE, 3><<<grid, 256, 0, st>>>(k);
  else mx_edge_grad_kernel<FMT, VEC, WIDE, 4><<<grid, 256, 0, st>>>(k);
  PXB_LAUNCHED("mx_edge_grad_kernel");
  return PXB_OK;
}

}  // namespace pxb

using namespace pxb;

extern "C" int pxb_mx_edge_grad(int64_t cap, const int32_t *from_id, const int32_t *to_id, const uint8_t *dead,
                                const float *g, const uint8_t *codes, const uint8_t *scales, int32_t fmt,
                                int32_t batch, int32_t num_units, float *dw, float *weight, const pxb_optimizer *opt,
                                float *opt_m, float *opt_v, float *opt_t, void *scratch, size_t scratch_bytes,
                                void *stream) {
  PXB_REQUIRE(cap >= 0 && batch >= 1 && batch <= kMxMaxBatch && num_units >= 0, "pxb_mx_edge_grad: bad sizes");
  PXB_REQUIRE(fmt == PXB_MX_E4M3 || fmt == PXB_MX_E5M2, "pxb_mx_edge_grad: a checkpoint has 8 bits (e4m3 or e5m2)");
  if (cap == 0) return PXB_OK;
  PXB_REQUIRE((opt == nullptr) == (dw != nullptr), "pxb_mx_edge_grad: give dw or an optimizer, not both or neither");
  PXB_REQUIRE(from_id && to_id && dead, "pxb_mx_edge_grad: a pointer is NULL");
  PXB_REQUIRE(num_units == 0 || (g && codes && scales), "pxb_mx_edge_grad: a pointer is NULL");
  PXB_REQUIRE(aligned16(codes), "pxb_mx_edge_grad: codes must be 16-byte aligned");
  OptParams op{};
  if (opt != nullptr) {
    PXB_REQUIRE(opt->kind >= PXB_OPT_SGD && opt->kind <= PXB_OPT_RMSPROP, "pxb_mx_edge_grad: bad optimizer");
    PXB_REQUIRE(weight, "pxb_mx_edge_grad: weight is NULL");
    PXB_REQUIRE(opt->kind == PXB_OPT_SGD || opt_v, "pxb_mx_edge_grad: optimizer state column is NULL");
    PXB_REQUIRE(opt->kind != PXB_OPT_ADAM || (opt_m && opt_t), "pxb_mx_edge_grad: adam needs opt/m and opt/t");
    op = OptParams{opt->kind, opt->lr, opt->b1, opt->b2, opt->eps, opt->weight_decay, nullptr};
  }
  const bool vec = aligned16(g) && batch % 4 == 0;
  const EdgeGrad k{cap, from_id, to_id, dead, g, codes, scales, batch,
                   static_cast<int32_t>(mx_blocks(batch)), static_cast<uint32_t>(num_units), dw, weight, op, opt_m,
                   opt_v, opt_t};
  cudaStream_t st = as_stream(stream);
  // 32-bit offsets hold the gradients' bytes and the codes' (32 a unit at least: more than the gradients' at few samples)
  const int64_t row_bytes = batch > mx_blocks(batch) * 8 ? int64_t(batch) * 4 : mx_blocks(batch) * 32;
  const bool wide = !vec || num_units * row_bytes >= (int64_t(1) << 32);
  if (scratch != nullptr) {
    const size_t need = pair_scratch(cap, batch, num_units);
    if (scratch_bytes < need) {
      set_error("pxb_mx_edge_grad: scratch of %zu bytes, %zu needed", scratch_bytes, need);
      return PXB_ESCRATCH;
    }
    PXB_REQUIRE(aligned16(scratch), "pxb_mx_edge_grad: scratch must be 16-byte aligned");
    if (need > 0) {
      if (fmt == PXB_MX_E4M3) return vec ? launch_pairs<PXB_MX_E4M3, true>(k, scratch, st) : launch_pairs<PXB_MX_E4M3, false>(k, scratch, st);
      return vec ? launch_pairs<PXB_MX_E5M2, true>(k, scratch, st) : launch_pairs<PXB_MX_E5M2, false>(k, scratch, st);
    }
  }
#define PXB_EG(F) \
  return !vec ? launch_edge_grad<F, false, true>(k, st) \
              : wide ? launch_edge_grad<F, true, true>(k, st) : launch_edge_grad<F, true, false>(k, st)
  if (fmt == PXB_MX_E4M3) PXB_EG(PXB_MX_E4M3);
  PXB_EG(PXB_MX_E5M2);
#undef PXB_EG
}

extern "C" int pxb_mx_edge_grad_scratch_bytes(int64_t cap, int32_t batch, int32_t num_units, size_t *bytes) {
  PXB_REQUIRE(bytes != nullptr, "pxb_mx_edge_grad_scratch_bytes: bytes is NULL");
  PXB_REQUIRE(cap >= 0 && batch >= 1 && num_units >= 0, "pxb_mx_edge_grad_scratch_bytes: bad sizes");
  *bytes = num_units == 0 ? 0 : pair_scratch(cap, batch, num_units);
  return PXB_OK;
}

extern "C" int pxb_mx_product(const pxb_mx_conns *conns, int32_t num_src, int32_t batch, const float *x,
                              const uint8_t *x_codes, const uint8_t *x_scales, int32_t x_fmt, int32_t act_kind,
                              int32_t num_out, float *out, uint8_t *out_codes, uint8_t *out_scales, int32_t out_fmt,
                              void *stream) {
  PXB_REQUIRE(conns != nullptr, "pxb_mx_product: conns is NULL");
  PXB_REQUIRE(num_src >= 0 && num_out >= 0 && batch >= 0 && conns->num_dst >= 0 && conns->num_edges >= 0 &&
                  conns->num_blocks >= 0 && batch <= kMxMaxBatch, "pxb_mx_product: bad sizes");
  PXB_REQUIRE(x_fmt >= PXB_MX_E4M3 && x_fmt <= PXB_MX_F32 && out_fmt >= PXB_MX_E4M3 && out_fmt <= PXB_MX_F32 &&
                  conns->fmt >= PXB_MX_E4M3 && conns->fmt <= PXB_MX_F32, "pxb_mx_product: unknown format");
  PXB_REQUIRE(act_kind >= PXB_ACT_IDENTITY && act_kind <= PXB_ACT_SIGMOID,
              "pxb_mx_product: unknown activation code %d", act_kind);
  if (conns->num_dst == 0 || batch == 0) return PXB_OK;
  PXB_REQUIRE(conns->units && conns->offsets, "pxb_mx_product: a pointer is NULL");
  PXB_REQUIRE(conns->fmt == PXB_MX_F32 || conns->block_offsets, "pxb_mx_product: block_offsets is NULL");
  if (conns->num_edges > 0) {
    PXB_REQUIRE(conns->src, "pxb_mx_product: a pointer is NULL");
    PXB_REQUIRE(conns->fmt == PXB_MX_F32 ? conns->weight != nullptr
                                         : conns->num_blocks == 0 || (conns->codes && conns->scales),
                "pxb_mx_product: the weights' pointers are NULL");
    PXB_REQUIRE(num_src == 0 || (x_fmt == PXB_MX_F32 ? x != nullptr : x_codes && x_scales),
                "pxb_mx_product: x is NULL");
  }
  PXB_REQUIRE(out_fmt == PXB_MX_F32 ? out != nullptr : out_codes && out_scales, "pxb_mx_product: out is NULL");
  PXB_REQUIRE(aligned16(x_codes) && aligned16(out_codes) && aligned16(conns->codes),
              "pxb_mx_product: codes must be 16-byte aligned");
  const Conns c{conns->num_dst, conns->fmt, num_src > 0 ? conns->num_edges : 0, conns->num_blocks, conns->units, conns->offsets, conns->src,
                conns->weight, conns->block_offsets, conns->codes, conns->scales};
  const int32_t nb = static_cast<int32_t>(mx_blocks(batch));
  cudaStream_t st = as_stream(stream);
  const bool whole = batch % 4 == 0;
  const Out o{out_fmt, static_cast<uint32_t>(num_out), out, out_codes, out_scales, whole && aligned16(out)};
  const Rows r{x, x_codes, x_scales, batch, nb, static_cast<uint32_t>(num_src)};
  if (x_fmt == PXB_MX_F32) return launch_product<PXB_MX_F32, 1>(c, r, act_kind, o, whole && aligned16(x), st);
  if (x_fmt == PXB_MX_E4M3) return launch_product<PXB_MX_E4M3, 2>(c, r, act_kind, o, true, st);
  if (x_fmt == PXB_MX_E5M2) return launch_product<PXB_MX_E5M2, 2>(c, r, act_kind, o, true, st);
  return launch_product<PXB_MX_E2M1, 1>(c, r, act_kind, o, true, st);
}

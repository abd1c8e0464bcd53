// Edge products over microscaled rows: the gradient of every connection from
// checkpointed activations, and the forward of a frozen arena.
#include "mx.cuh"
#include "optim.cuh"

namespace pxb {

// ---------------------------------------------------------------------------
// stat[s] = (sum_b g[to, b] * a[from, b]) / B
// ---------------------------------------------------------------------------
// A warp owns 32 slots; eight lanes share a slot, four samples each, so one
// load instruction covers a 32-sample slice of four slots. A lane keeps the
// partial sums of its group's eight slots over every slice; halving them
// across the group's lanes at the end (4 + 2 + 1 exchanges) leaves lane l
// with slot l's sum.
template <int FMT, bool VEC>
__global__ void __launch_bounds__(256) mx_edge_grad_kernel(
    int64_t cap, const int32_t *__restrict__ from, const int32_t *__restrict__ to, const uint8_t *__restrict__ dead,
    const float *__restrict__ g, const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int32_t batch,
    uint32_t n, float *__restrict__ dw, float *__restrict__ weight, OptParams op, float *m_col, float *v_col,
    float *t_col) {
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const int32_t nb = (batch + kMxBlock - 1) / kMxBlock;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  for (int64_t base = ((blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5) * 32; base < cap;
       base += warps * 32) {
    const int64_t s = base + lane;
    int32_t f = -1, t = -1;
    if (s < cap && !dead[s]) {
      f = from[s];
      t = to[s];
      if (static_cast<uint32_t>(f) >= n || static_cast<uint32_t>(t) >= n) f = t = -1;
    }
    float p[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (__any_sync(0xffffffffu, t >= 0)) {
      for (int32_t k = 0; k < nb; ++k) {
        const int32_t b = k * kMxBlock + sub * 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int32_t fj = __shfl_sync(0xffffffffu, f, j, 8), tj = __shfl_sync(0xffffffffu, t, j, 8);
          if (tj < 0) continue;
          const float *gr = g + static_cast<int64_t>(tj) * batch + b;
          float4 gv = make_float4(0.f, 0.f, 0.f, 0.f);
          if (VEC) {
            if (b < batch) gv = __ldg(reinterpret_cast<const float4 *>(gr));
          } else {
            if (b < batch) gv.x = __ldg(gr);
            if (b + 1 < batch) gv.y = __ldg(gr + 1);
            if (b + 2 < batch) gv.z = __ldg(gr + 2);
            if (b + 3 < batch) gv.w = __ldg(gr + 3);
          }
          const int64_t blk = static_cast<int64_t>(fj) * nb + k;
          const uint32_t c = __ldg(reinterpret_cast<const uint32_t *>(codes) + blk * 8 + sub);
          const float2 lo = mx_decode2<FMT>(c & 0xffffu), hi = mx_decode2<FMT>(c >> 16);
          const float dot = gv.x * lo.x + gv.y * lo.y + gv.z * hi.x + gv.w * hi.y;
          p[j] = fmaf(dot, mx_scale_value(__ldg(scales + blk)), p[j]);
        }
      }
#pragma unroll
      for (int half = 4; half > 0; half >>= 1) {
        const bool upper = (lane & half) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const float send = upper ? p[i] : p[i + half], keep = upper ? p[i + half] : p[i];
          p[i] = keep + __shfl_xor_sync(0xffffffffu, send, half);
        }
      }
    }
    if (s < cap) {
      const float stat = __fdiv_rn(p[0], static_cast<float>(batch));
      if (dw != nullptr) {
        dw[s] = t >= 0 ? stat : 0.0f;
      } else if (t >= 0) {
        float w = weight[s];
        opt_step(op, stat, w, m_col, v_col, t_col, s);
        weight[s] = w;
      }
    }
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
};

template <int XF>
struct Rows {
  const float *__restrict__ x;
  const uint8_t *__restrict__ codes;
  const uint8_t *__restrict__ scales;
  int32_t batch, nb;
};

// A warp owns one destination and a chunk of 256 samples. A lane holds eight
// consecutive samples; where a row has fewer than 32 octets, 32 / LANES edges
// run side by side and their sums join at the end by shuffles.
template <int XF, int LANES, bool VEC>
__global__ void __launch_bounds__(256) mx_product_kernel(Conns c, uint32_t num_src, Rows<XF> r, int act_kind, Out out,
                                                         int32_t chunks) {
  constexpr int kGroups = 32 / LANES;
  const int lane = threadIdx.x & 31, sub = lane % LANES, grp = lane / LANES;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  const int64_t total = static_cast<int64_t>(c.num_dst) * chunks;
  for (int64_t item = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5; item < total;
       item += warps) {
    const int32_t i = static_cast<int32_t>(item / chunks);
    const int32_t b = static_cast<int32_t>(item - static_cast<int64_t>(i) * chunks) * 256 + sub * 8;
    const int64_t e0 = max(int64_t(0), c.offsets[i]), e1 = min(c.num_edges, c.offsets[i + 1]);
    const int64_t blk0 = c.fmt == PXB_MX_F32 ? 0 : max(int64_t(0), c.block_offsets[i]);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t e = e0; e < e1; e += 32) {
      int32_t s = -1;
      float w = 0.0f;
      if (e + lane < e1) {
        s = __ldg(c.src + e + lane);
        if (static_cast<uint32_t>(s) >= num_src) s = -1;
        w = conn_weight(c, e + lane, blk0 + ((e - e0) >> 5), lane);
      }
      const int cnt = static_cast<int>(min(int64_t(32), e1 - e));
      for (int j = 0; j < cnt; j += kGroups) {
        const int32_t sj = __shfl_sync(0xffffffffu, s, j + grp);
        const float wj = __shfl_sync(0xffffffffu, w, j + grp);
        if (sj < 0 || b >= r.batch) continue;
        float v[8];
        if constexpr (XF == PXB_MX_F32) {
          const float *xr = r.x + static_cast<int64_t>(sj) * r.batch + b;
          if (VEC && b + 8 <= r.batch) {
            const float4 lo = __ldg(reinterpret_cast<const float4 *>(xr));
            const float4 hi = __ldg(reinterpret_cast<const float4 *>(xr) + 1);
            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = b + q < r.batch ? __ldg(xr + q) : 0.0f;
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[q] = fmaf(wj, v[q], acc[q]);
        } else {
          const int64_t row = static_cast<int64_t>(sj) * r.nb;
          mx_decode8<XF>(mx_load8<XF>(r.codes, row * 4 + (b >> 3)), v);
          const float ws = __fmul_rn(wj, mx_scale_value(__ldg(r.scales + row + (b >> 5))));
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[q] = fmaf(ws, v[q], acc[q]);
        }
      }
    }
#pragma unroll
    for (int off = LANES; off < 32; off <<= 1)
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += __shfl_xor_sync(0xffffffffu, acc[q], off);
    const int32_t u = c.units[i];
    const bool on = grp == 0 && b < r.nb * kMxBlock && static_cast<uint32_t>(u) < out.rows;
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = b + q < r.batch ? act_fn(act_kind, acc[q]) : 0.0f;
    if (out.fmt == PXB_MX_F32) {
      float *o = out.x + static_cast<int64_t>(u) * r.batch + b;
      if (on && VEC && b + 8 <= r.batch) {
        reinterpret_cast<float4 *>(o)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        reinterpret_cast<float4 *>(o)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      } else if (on) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (b + q < r.batch) o[q] = acc[q];
      }
    } else {
      const int64_t o = static_cast<int64_t>(u) * r.nb * 4 + (b >> 3);
      if (out.fmt == PXB_MX_E4M3) store_codes<PXB_MX_E4M3>(acc, on, o, out.codes, out.scales);
      else if (out.fmt == PXB_MX_E5M2) store_codes<PXB_MX_E5M2>(acc, on, o, out.codes, out.scales);
      else store_codes<PXB_MX_E2M1>(acc, on, o, out.codes, out.scales);
    }
  }
}

template <int XF>
static int launch_product(const Conns &c, int32_t num_src, const Rows<XF> &r, int act, const Out &out, bool vec,
                          cudaStream_t st) {
  const int32_t octets = r.nb * 4, chunks = (octets + 31) / 32;
  const int grid = grid_for(static_cast<int64_t>(c.num_dst) * chunks, 8, 8);
#define PXB_MXP(L)                                                                                         \
  do {                                                                                                     \
    if (vec) mx_product_kernel<XF, L, true><<<grid, 256, 0, st>>>(c, num_src, r, act, out, chunks);         \
    else mx_product_kernel<XF, L, false><<<grid, 256, 0, st>>>(c, num_src, r, act, out, chunks);            \
  } while (0)
  if (octets <= 4) PXB_MXP(4);
  else if (octets <= 8) PXB_MXP(8);
  else if (octets <= 16) PXB_MXP(16);
  else PXB_MXP(32);
#undef PXB_MXP
  PXB_LAUNCHED("mx_product_kernel");
  return PXB_OK;
}

}  // namespace pxb

using namespace pxb;

extern "C" int pxb_mx_edge_grad(int64_t cap, const int32_t *from_id, const int32_t *to_id, const uint8_t *dead,
                                const float *g, const uint8_t *codes, const uint8_t *scales, int32_t fmt,
                                int32_t batch, int32_t num_units, float *dw, float *weight, const pxb_optimizer *opt,
                                float *opt_m, float *opt_v, float *opt_t, void *stream) {
  PXB_REQUIRE(cap >= 0 && batch >= 1 && num_units >= 0, "pxb_mx_edge_grad: bad sizes");
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
  const int grid = grid_for((cap + 31) / 32, 8, 8);
  cudaStream_t st = as_stream(stream);
  const bool vec = aligned16(g) && batch % 4 == 0;
  const uint32_t n = static_cast<uint32_t>(num_units);
#define PXB_EG(F, V)                                                                                               \
  mx_edge_grad_kernel<F, V><<<grid, 256, 0, st>>>(cap, from_id, to_id, dead, g, codes, scales, batch, n, dw, weight, \
                                                  op, opt_m, opt_v, opt_t)
  if (fmt == PXB_MX_E4M3) {
    if (vec) PXB_EG(PXB_MX_E4M3, true);
    else PXB_EG(PXB_MX_E4M3, false);
  } else {
    if (vec) PXB_EG(PXB_MX_E5M2, true);
    else PXB_EG(PXB_MX_E5M2, false);
  }
#undef PXB_EG
  PXB_LAUNCHED("mx_edge_grad_kernel");
  return PXB_OK;
}

extern "C" int pxb_mx_product(const pxb_mx_conns *conns, int32_t num_src, int32_t batch, const float *x,
                              const uint8_t *x_codes, const uint8_t *x_scales, int32_t x_fmt, int32_t act_kind,
                              int32_t num_out, float *out, uint8_t *out_codes, uint8_t *out_scales, int32_t out_fmt,
                              void *stream) {
  PXB_REQUIRE(conns != nullptr, "pxb_mx_product: conns is NULL");
  PXB_REQUIRE(num_src >= 0 && num_out >= 0 && batch >= 0 && conns->num_dst >= 0 && conns->num_edges >= 0 &&
                  conns->num_blocks >= 0, "pxb_mx_product: bad sizes");
  PXB_REQUIRE(x_fmt >= PXB_MX_E4M3 && x_fmt <= PXB_MX_F32 && out_fmt >= PXB_MX_E4M3 && out_fmt <= PXB_MX_F32 &&
                  conns->fmt >= PXB_MX_E4M3 && conns->fmt <= PXB_MX_F32, "pxb_mx_product: unknown format");
  PXB_REQUIRE(act_kind >= PXB_ACT_IDENTITY && act_kind <= PXB_ACT_SIGMOID,
              "pxb_mx_product: unknown activation code %d", act_kind);
  if (conns->num_dst == 0 || batch == 0) return PXB_OK;
  PXB_REQUIRE(conns->units && conns->offsets, "pxb_mx_product: a pointer is NULL");
  if (conns->num_edges > 0) {
    PXB_REQUIRE(conns->src, "pxb_mx_product: a pointer is NULL");
    PXB_REQUIRE(conns->fmt == PXB_MX_F32 ? conns->weight != nullptr
                                         : conns->block_offsets && (conns->num_blocks == 0 || (conns->codes && conns->scales)),
                "pxb_mx_product: the weights' pointers are NULL");
    PXB_REQUIRE(num_src == 0 || (x_fmt == PXB_MX_F32 ? x != nullptr : x_codes && x_scales),
                "pxb_mx_product: x is NULL");
  }
  PXB_REQUIRE(out_fmt == PXB_MX_F32 ? out != nullptr : out_codes && out_scales, "pxb_mx_product: out is NULL");
  PXB_REQUIRE(aligned16(x_codes) && aligned16(out_codes), "pxb_mx_product: codes must be 16-byte aligned");
  const Conns c{conns->num_dst, conns->fmt, conns->num_edges, conns->num_blocks, conns->units, conns->offsets, conns->src,
                conns->weight, conns->block_offsets, conns->codes, conns->scales};
  const int32_t nb = static_cast<int32_t>(mx_blocks(batch));
  const bool vec = batch % 4 == 0 && aligned16(x) && aligned16(out);
  cudaStream_t st = as_stream(stream);
  const Out o{out_fmt, static_cast<uint32_t>(num_out), out, out_codes, out_scales};
#define PXB_MXD(XF) \
  launch_product<XF>(c, num_src, Rows<XF>{x, x_codes, x_scales, batch, nb}, act_kind, o, vec, st)
  if (x_fmt == PXB_MX_F32) return PXB_MXD(PXB_MX_F32);
  if (x_fmt == PXB_MX_E4M3) return PXB_MXD(PXB_MX_E4M3);
  if (x_fmt == PXB_MX_E5M2) return PXB_MXD(PXB_MX_E5M2);
  return PXB_MXD(PXB_MX_E2M1);
#undef PXB_MXD
}

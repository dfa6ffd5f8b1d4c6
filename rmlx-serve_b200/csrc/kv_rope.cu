// Append with the position rotation applied on the way: what a transformer
// layer does between its projections and its attention, in one launch.  The
// query rows of T tokens are rotated into a buffer, the key rows are rotated
// into the pool's slots, the value rows are copied into them; a quantised
// pool quantises the f32 rotated row directly.
//
// With R = rotary_dim, a_i = position[axis(i)] * inv_freq[i] for i < R / 2
// and (x1, x2) the i-th pair of a row (elements i and i + R/2, or 2i and
// 2i + 1 when interleaved):
//   y1 = x1 cos a_i - x2 sin a_i,   y2 = x2 cos a_i + x1 sin a_i;
// elements from R on pass through unchanged.
//
// The angle of a far position does not fit f32 (at 100,000 radians its ulp
// is 2^-7), so the product and the reduction to one turn are done in f64
// (about 2^-52 relative: 1e-6 rad at position 2^31) and only the remainder,
// below half a turn, is rounded to f32 for sincospif.  A token's R / 2 pairs
// are computed once per CTA into shared memory and serve all of its query
// and key heads.
//
// Bytes per token: (q_heads + 2 heads) rows in, the same out; a few flops per
// byte, so HBM bounds the long calls and the launch the short ones.
#include <algorithm>

#include "quant.cuh"

namespace rmlx {

struct RopeArgs {
  const uint8_t *q, *k, *v;
  uint8_t* qo;
  int64_t qts, qhs, ots, ohs, ts, hs;  // byte strides: q, q_out, k and v (token, head)
  const int32_t *slots, *pos, *axis;
  const float* inv;
  int64_t pos_stride;
  int half, naxes;     // rotary_dim / 2
  int hq, T, layer;
  int cpr, upr;        // 8-element chunks and work units (chunk pairs) of a row
  int tokens_per_cta;
};

// cos and sin of pair i of token t.
__device__ __forceinline__ float2 rope_angle(const RopeArgs& a, int t, int i, int32_t* err) {
  int ax = 0;
  if (a.axis) {
    ax = __ldg(a.axis + i);
    if (ax < 0 || ax >= a.naxes) {
      atomicOr(err, DEV_ERR_AXIS);
      ax = 0;
    }
  }
  const double p = (double)__ldg(a.pos + ax * a.pos_stride + t);
  double turns = p * (double)__ldg(a.inv + i) * 0.15915494309189533577;  // 1 / (2 pi)
  turns -= rint(turns);
  float2 cs;
  sincospif((float)(2.0 * turns), &cs.y, &cs.x);
  return cs;
}

// Slot of token t, -1 when the token is skipped or its slot lies outside the pool (flagged).
__device__ __forceinline__ int32_t rope_slot(const PoolGeo& g, const RopeArgs& a, int t, int32_t* err) {
  int32_t s = __ldg(a.slots + t);
  if (s >= (int64_t)g.nblocks * g.bs) {
    atomicOr(err, DEV_ERR_SLOT);
    s = -1;
  }
  return s;
}

// One 8-element chunk as it lies in memory.
template <int DT>
struct Raw8 {
  static constexpr int BYTES = 8 * Elem<DT>::size, N = BYTES / 16;
  uint4 w[N];
  __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = ld_stream_coherent(p + 16 * i);  // q_out may be q
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
#pragma unroll
    for (int i = 0; i < N; ++i) st_stream(p + 16 * i, w[i]);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (DT == RMLX_F32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[4 * i] = __uint_as_float(w[i].x), f[4 * i + 1] = __uint_as_float(w[i].y);
        f[4 * i + 2] = __uint_as_float(w[i].z), f[4 * i + 3] = __uint_as_float(w[i].w);
      }
    } else {
      const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == RMLX_BF16) {
          f[2 * i] = __uint_as_float(u[i] << 16);
          f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
          f[2 * i] = x.x;
          f[2 * i + 1] = x.y;
        }
      }
    }
  }
};

// Rotates the 8 pairs held as chunks a and b; i0 is the first pair's index.
template <bool IL>
__device__ __forceinline__ void rotate8(float (&a)[8], float (&b)[8], const float2* cs) {
  if (IL) {  // pairs of adjacent elements: four in each chunk
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 r = cs[i], s = cs[4 + i];
      const float a1 = a[2 * i], a2 = a[2 * i + 1], b1 = b[2 * i], b2 = b[2 * i + 1];
      a[2 * i] = a1 * r.x - a2 * r.y;
      a[2 * i + 1] = a2 * r.x + a1 * r.y;
      b[2 * i] = b1 * s.x - b2 * s.y;
      b[2 * i + 1] = b2 * s.x + b1 * s.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 r = cs[i];
      const float x1 = a[i], x2 = b[i];
      a[i] = x1 * r.x - x2 * r.y;
      b[i] = x2 * r.x + x1 * r.y;
    }
  }
}

// A CTA takes tokens_per_cta tokens (blockIdx.x) and a share of their work
// units (blockIdx.y).  A unit is two 8-element chunks of one row: the two
// halves' chunks that hold the same pairs (or two adjacent chunks), so one
// thread reads and writes both sides of its pairs and q_out may be q itself.
// BITS != 0: the K and V rows go through the group quantiser instead, one
// lane per 8 elements (a lane of the second half re-reads its partner chunk,
// which its neighbour has brought into L1).
template <int DT, bool IL, int BITS, bool MF32>
__global__ void __launch_bounds__(256) append_rope_kernel(PoolGeo g, RopeArgs a, int tpg, int32_t* err) {
  using E = Elem<DT>;
  constexpr int CB = 8 * E::size;  // bytes of a chunk
  extern __shared__ float2 cs[];   // [token][pair]
  pdl_wait();
  pdl_release();
  const int t0 = blockIdx.x * a.tokens_per_cta;
  const int nt = min(a.tokens_per_cta, a.T - t0);
  for (int x = threadIdx.x; x < nt * a.half; x += blockDim.x) {
    const int j = x / a.half;
    cs[x] = rope_angle(a, t0 + j, x - j * a.half, err);
  }
  __syncthreads();
  const int hc = a.half / 8;  // chunks of half of the rotary part
  const int rows = a.hq + (BITS ? 0 : 2 * g.heads);
  const int step = gridDim.y * blockDim.x;
  for (int x = blockIdx.y * blockDim.x + threadIdx.x; x < nt * rows * a.upr; x += step) {
    const int r = x / a.upr, u = x - r * a.upr;
    const int j = r / rows, h = r - j * rows;
    const int t = t0 + j;
    const uint8_t* src;
    uint8_t* dst;
    bool rot = u < hc;
    if (h < a.hq) {
      src = a.q + t * a.qts + h * a.qhs;
      dst = a.qo + t * a.ots + h * a.ohs;
    } else {
      const int hk = h - a.hq, kv = hk >= g.heads, hh = kv ? hk - g.heads : hk;
      const int32_t s = rope_slot(g, a, t, err);
      if (s < 0) continue;
      const int blk = s / g.bs, off = s - blk * g.bs;
      src = (kv ? a.v : a.k) + t * a.ts + hh * a.hs;
      dst = g.base + g.tile_off(blk, a.layer, kv, hh) + (int64_t)off * g.row_bytes;
      if (kv) rot = false;
    }
    // a unit of the rotary part holds chunks u and u + hc (halves), any other 2u and 2u + 1
    const bool split = !IL && u < hc;
    const int c0 = split ? u : 2 * u;
    const int c1 = split ? u + hc : c0 + 1;
    Raw8<DT> ra, rb;
    ra.load(src + c0 * CB);
    if (c1 < a.cpr) rb.load(src + c1 * CB);
    if (rot) {
      float fa[8], fb[8];
      ra.get(fa);
      rb.get(fb);
      rotate8<IL>(fa, fb, cs + j * a.half + 8 * u);
      E::store8(dst + c0 * CB, fa);
      E::store8(dst + c1 * CB, fb);
    } else {
      ra.store(dst + c0 * CB);
      if (c1 < a.cpr) rb.store(dst + c1 * CB);
    }
  }
  if constexpr (BITS != 0) {
    const int units = nt * 2 * g.heads * a.cpr;
    for (int x0 = blockIdx.y * blockDim.x; x0 < units; x0 += step) {
      const int x = x0 + threadIdx.x;
      const int r = x / a.cpr, c = x - r * a.cpr;
      const int j = r / (2 * g.heads), hk = r - j * 2 * g.heads;
      const int kv = hk >= g.heads, h = kv ? hk - g.heads : hk;
      const int t = t0 + j;
      const int32_t s = x < units ? rope_slot(g, a, t, err) : -1;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (s >= 0) {
        const uint8_t* src = (kv ? a.v : a.k) + t * a.ts + h * a.hs;
        E::load8(src + c * CB, f);
        if (!kv && c < 2 * hc) {
          const float2* w = cs + j * a.half;
          if (IL) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 y = w[4 * c + i];
              const float x1 = f[2 * i], x2 = f[2 * i + 1];
              f[2 * i] = x1 * y.x - x2 * y.y;
              f[2 * i + 1] = x2 * y.x + x1 * y.y;
            }
          } else {
            const bool lo = c < hc;
            const int p = lo ? c : c - hc;
            float b[8];
            E::load8(src + (lo ? c + hc : p) * CB, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 y = w[8 * p + i];
              f[i] = lo ? f[i] * y.x - b[i] * y.y : f[i] * y.x + b[i] * y.y;
            }
          }
        }
      }
      quantise8<BITS ? BITS : 8, MF32>(g, f, s >= 0, s, a.layer, kv, h, c, tpg);
    }
  }
}

}  // namespace rmlx

using namespace rmlx;

namespace {

using RopeFn = void (*)(PoolGeo, RopeArgs, int, int32_t*);
template <int DT, bool IL>
RopeFn pick_rope(int bits, bool mf32) {
  if (bits == 0) return append_rope_kernel<DT, IL, 0, false>;
  if (bits == 8) return mf32 ? append_rope_kernel<DT, IL, 8, true> : append_rope_kernel<DT, IL, 8, false>;
  return mf32 ? append_rope_kernel<DT, IL, 4, true> : append_rope_kernel<DT, IL, 4, false>;
}
template <bool IL>
RopeFn pick_rope(const rmlx_pool_config& c) {
  const bool mf32 = c.meta_dtype == RMLX_F32;
  return c.dtype == RMLX_F32   ? pick_rope<RMLX_F32, IL>(c.quant_bits, mf32)
         : c.dtype == RMLX_F16 ? pick_rope<RMLX_F16, IL>(c.quant_bits, mf32)
                               : pick_rope<RMLX_BF16, IL>(c.quant_bits, mf32);
}

}  // namespace

extern "C" rmlx_status rmlx_kv_append_rope(rmlx_kv_pool* p, int32_t layer, const rmlx_rope* rope,
                                           const int32_t* positions, int64_t position_axis_stride, const void* q,
                                           int32_t q_heads, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                                           int64_t q_out_token_stride, int64_t q_out_head_stride, const void* k,
                                           const void* v, int64_t token_stride, int64_t head_stride,
                                           const int32_t* slot_mapping, int32_t num_tokens, void* stream) {
  if (!p || !rope) return fail(RMLX_E_BAD_ARG, "NULL pool or rope");
  const rmlx_pool_config& c = p->cfg;
  if (layer < 0 || layer >= c.num_layers) return fail(RMLX_E_RANGE, "layer %d outside the pool's %d layers", layer, c.num_layers);
  if (c.head_dim % 8) return fail(RMLX_E_BAD_ARG, "append with rotation needs a head_dim that is a multiple of 8");
  if (rope->rotary_dim <= 0 || rope->rotary_dim % 16 || rope->rotary_dim > c.head_dim || rope->rotary_dim > 1024)
    return fail(RMLX_E_BAD_ARG, "rotary_dim must be a multiple of 16 in [16, min(head_dim, 1024)], got %d", rope->rotary_dim);
  if (rope->num_axes < 1) return fail(RMLX_E_BAD_ARG, "num_axes must be at least 1");
  if (!rope->inv_freq) return fail(RMLX_E_BAD_ARG, "NULL inv_freq");
  if (q_heads < 0 || q_heads > 65536) return fail(RMLX_E_BAD_ARG, "q_heads outside [0, 65536]");
  if (num_tokens < 0) return fail(RMLX_E_BAD_ARG, "num_tokens < 0");
  if (num_tokens == 0) return RMLX_OK;
  if (!positions || !k || !v || !slot_mapping) return fail(RMLX_E_BAD_ARG, "NULL positions, k, v or slot_mapping");
  if (q_heads && (!q || !q_out)) return fail(RMLX_E_BAD_ARG, "NULL q or q_out with q_heads = %d", q_heads);
  const int es = c.dtype == RMLX_F32 ? 4 : 2;
  RopeArgs a;
  a.q = (const uint8_t*)q, a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.qo = (uint8_t*)q_out;
  a.qts = q_token_stride * es, a.qhs = q_head_stride * es, a.ots = q_out_token_stride * es;
  a.ohs = q_out_head_stride * es, a.ts = token_stride * es, a.hs = head_stride * es;
  if (!aligned16(k) || !aligned16(v) || (a.ts % 16) || (a.hs % 16))
    return fail(RMLX_E_BAD_ARG, "k/v pointers and strides must be 16-byte aligned");
  if (q_heads && (!aligned16(q) || !aligned16(q_out) || (a.qts % 16) || (a.qhs % 16) || (a.ots % 16) || (a.ohs % 16)))
    return fail(RMLX_E_BAD_ARG, "q/q_out pointers and strides must be 16-byte aligned");
  if (q_heads && q == q_out && ((num_tokens > 1 && a.qts != a.ots) || (q_heads > 1 && a.qhs != a.ohs)))
    return fail(RMLX_E_BAD_ARG, "q_out is q with other strides");
  a.slots = slot_mapping, a.pos = positions, a.axis = rope->pair_axis, a.inv = rope->inv_freq;
  a.pos_stride = position_axis_stride;
  a.half = rope->rotary_dim / 2, a.naxes = rope->num_axes;
  a.hq = q_heads, a.T = num_tokens, a.layer = layer;
  a.cpr = c.head_dim / 8, a.upr = (a.cpr + 1) / 2;
  // Four tokens a CTA in long calls; one, with its rows dealt to several
  // CTAs, while that leaves SMs without work.
  const int64_t units = (int64_t)(q_heads + 2 * c.num_kv_heads) * a.upr;
  if (units * 4 > INT32_MAX) return fail(RMLX_E_BAD_ARG, "too many heads in one append");
  a.tokens_per_cta = num_tokens >= 8 * p->num_sms ? 4 : 1;
  const int gx = (num_tokens + a.tokens_per_cta - 1) / a.tokens_per_cta;
  const int64_t want = (2 * (int64_t)p->num_sms + gx - 1) / gx;
  const int gy = (int)std::max<int64_t>(1, std::min<int64_t>(want, (units + 255) / 256));
  DeviceGuard dg(p->device);
  RopeFn fn = rope->interleaved ? pick_rope<true>(c) : pick_rope<false>(c);
  cudaError_t e = launch_pdl(fn, dim3((unsigned)gx, (unsigned)gy), dim3(256),
                             (size_t)a.tokens_per_cta * a.half * sizeof(float2), (cudaStream_t)stream, p->geo(), a,
                             c.quant_bits ? c.group_size / 8 : 1, p->err);
  if (e != cudaSuccess) return cuda_check(e, "append with rotation launch");
  return cuda_check(cudaGetLastError(), "append with rotation launch");
}

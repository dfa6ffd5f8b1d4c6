// Element conversions and the group quantiser of one lane's 8 elements,
// shared by the quantise-on-append kernels (kv_pool.cu, kv_rope.cu).
#pragma once
#include "kv_pool_internal.cuh"

namespace rmlx {

template <int DT>  // rmlx_dtype
struct Elem;
template <>
struct Elem<RMLX_F32> {
  static constexpr int size = 4;
  // 8 consecutive elements -> f32
  __device__ __forceinline__ static void load8(const uint8_t* p, float* f) {
    uint4 a = ld_stream(p), b = ld_stream(p + 16);
    f[0] = __uint_as_float(a.x), f[1] = __uint_as_float(a.y), f[2] = __uint_as_float(a.z), f[3] = __uint_as_float(a.w);
    f[4] = __uint_as_float(b.x), f[5] = __uint_as_float(b.y), f[6] = __uint_as_float(b.z), f[7] = __uint_as_float(b.w);
  }
  __device__ __forceinline__ static void store8(uint8_t* p, const float* f) {
    st_stream(p, make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])));
    st_stream(p + 16,
              make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])));
  }
};
template <>
struct Elem<RMLX_F16> {
  static constexpr int size = 2;
  __device__ __forceinline__ static void load8(const uint8_t* p, float* f) {
    uint4 a = ld_stream(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
      float2 x = __half22float2(h);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ __forceinline__ static void store8(uint8_t* p, const float* f) {
    st_stream(p, make_uint4(pack(f[0], f[1]), pack(f[2], f[3]), pack(f[4], f[5]), pack(f[6], f[7])));
  }
};
template <>
struct Elem<RMLX_BF16> {
  static constexpr int size = 2;
  __device__ __forceinline__ static void load8(const uint8_t* p, float* f) {
    uint4 a = ld_stream(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ __forceinline__ static void store8(uint8_t* p, const float* f) {
    st_stream(p, make_uint4(pack(f[0], f[1]), pack(f[2], f[3]), pack(f[4], f[5]), pack(f[6], f[7])));
  }
};

// Rust `x.round().clamp(0.0, qmax) as u8`: half-away rounding, clamp that
// passes NaN through, saturating cast with NaN -> 0.
__device__ __forceinline__ uint32_t quant_code(float v, float mn, float scale, float qmax) {
  float x = roundf(__fdiv_rn(__fsub_rn(v, mn), scale));
  if (x < 0.0f) x = 0.0f;
  if (x > qmax) x = qmax;
  return (x == x) ? (uint32_t)x : 0u;
}

// The codes of 8 elements: quant_code's, mostly without its division.  With x
// = (v - mn) / scale <= 256 and inv = 1 / scale rounded, d * inv is within x
// 2^-24 <= 2^-16 of x, and so is the rounded quotient that quant_code rounds.
// Where d * inv lies more than 2^-13 from every tie, all three round to the
// same code; elements nearer to one (1 in 4096), NaN, and scales whose
// reciprocal loses digits take quant_code itself.
__device__ __forceinline__ void quantise_codes(const float (&f)[8], float mn, float scale, float qmax, uint32_t (&code)[8]) {
  const float inv = scale > 1e-30f && scale < 1e30f ? __frcp_rn(scale) : __uint_as_float(0x7fffffffu);
  bool sure = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = __fsub_rn(f[e], mn);
    const float t = __fmaf_rn(d, inv, 12582912.0f);  // 1.5 * 2^23: the nearest integer in the low bits
    const float off = __fmaf_rn(d, inv, 12582912.0f - t);
    sure = sure && fabsf(off) <= 0.5f - 1.0f / 8192.0f;
    code[e] = __float_as_uint(t) & 0xffu;
  }
  if (!sure) {
#pragma unroll
    for (int e = 0; e < 8; ++e) code[e] = quant_code(f[e], mn, scale, qmax);
  }
}

// Quantises this lane's 8 elements f (chunk c of the row of KV head h) and
// stores codes and, once per group, (scale, zero) in pool slot s of `layer`.
// A group is tpg adjacent lanes, reduced with xor shuffles: every lane of
// the warp calls this, the ones without a row with valid = false.
template <int BITS, bool META_F32>
__device__ __forceinline__ void quantise8(const PoolGeo& g, const float (&f)[8], bool valid, int32_t s, int layer,
                                          int kv, int h, int c, int tpg) {
  const float qmax = (float)((1u << BITS) - 1);
  float mx = -INFINITY, mn = INFINITY;
#pragma unroll
  for (int e = 0; e < 8; ++e) mx = fmaxf(mx, f[e]);
#pragma unroll
  for (int e = 0; e < 8; ++e) mn = fminf(mn, f[e]);
  for (int o = 1; o < tpg; o <<= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  if (!valid) return;
  const float range = __fsub_rn(mx, mn);
  const float scale = (range == 0.0f) ? 1.0f : __fdiv_rn(range, qmax);
  const int blk = s / g.bs, off = s - blk * g.bs;
  uint8_t* tile = g.base + g.tile_off(blk, layer, kv, h);
  uint8_t* code_row = tile + (int64_t)off * g.row_bytes;
  uint32_t code[8];
  quantise_codes(f, mn, scale, qmax, code);
  if (BITS == 8) {
    *reinterpret_cast<uint2*>(code_row + c * 8) =
        make_uint2(code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24);
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= code[e] << (4 * e);
    *reinterpret_cast<uint32_t*>(code_row + c * 4) = w;
  }
  if ((c & (tpg - 1)) == 0) {
    const int q = c / tpg;
    uint8_t* meta_row = tile + (int64_t)g.bs * g.row_bytes + (int64_t)off * g.meta_row_bytes;
    if (META_F32) {
      reinterpret_cast<float*>(meta_row)[2 * q] = scale;
      reinterpret_cast<float*>(meta_row)[2 * q + 1] = mn;
    } else {
      reinterpret_cast<__half2*>(meta_row)[q] = __halves2half2(__float2half_rn(scale), __float2half_rn(mn));
    }
  }
}

}  // namespace rmlx

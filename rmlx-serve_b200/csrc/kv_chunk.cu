// Attention of a chunk of new tokens per sequence over the paged pool
// (prefill, chunked prefill, verification of drafted tokens): the consumer
// of the K/V tiles for more than one query token per sequence.
//
// Sequence s holds seq_lens[s] rows, the last q_lens[s] of them the chunk's
// own.  Chunk token i stands at position p = seq_lens[s] - q_lens[s] + i and
// sees keys j <= p (and j > p - window when a window is set); for query head
// h * G + g, with KV head h:
//   out = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m).
// A token that sees no key gives zeros.
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <numeric>
#include <type_traits>

#include "dequant.cuh"
#include "kv_pool_internal.cuh"
#include "tcgen05.cuh"

namespace rmlx {

struct ChunkArgs {
  const uint8_t* q;
  uint8_t* out;
  const int32_t *bt, *q_lens, *seq_lens;
  int64_t qts, qhs;  // byte strides of q: token, head
  int layer, G, bt_stride, nseq, nq, window;
  int max_len;  // rows that a row of the block tables can hold
  int gs_log2, bits, mf32;
  int bs_log2;  // of the block size, -1 when it is no power of two
  float scale_log2;
  uint64_t wait_ns;  // limit of a wait
};

// ---------------------------------------------------------------------------
// The plan.  A tile is up to 256 query rows of one sequence and KV head: the
// G query heads of 256 / G consecutive chunk tokens, so that every K/V row
// loaded serves all of them.  An item is (tile, KV head) with the 128-key
// tiles that its mask leaves; its cost is that number plus CH_OVERHEAD.  The
// launch's items are laid end to end and cut into equal shares, one per CTA,
// so a share may begin and end inside an item: such portions write partial
// results that a second kernel joins.  Every CTA works out its own share from
// q_lens and seq_lens, with no counter shared between CTAs or launches.
// ---------------------------------------------------------------------------
constexpr int CH_ROWS = 256;    // query rows of a tile: two M = 128 accumulators
constexpr int CH_KEYS = 128;    // keys of a key tile
constexpr int CH_HALF = 64;     // keys whose weights are made together
// Two softmax warpgroups, the MMA warp, and load warps: three with TMA, seven
// where they read and dequantise rows themselves.
constexpr int ch_threads(bool tma) { return tma ? 384 : 512; }
constexpr int CH_MAX_WARPS = 16;
constexpr int CH_RAW = 4;       // most tiles of codes in flight
constexpr int CH_OVERHEAD = 3;  // cost of an item besides its key tiles, in key tiles
constexpr int CH_MIN_COST = 4;  // smallest share
// Weights are made as 2^(score - running maximum + bias).  A lagging maximum lets
// them grow to 2^(8 + bias), which f16 holds up to a bias of 7; below 2^-14 f16
// loses digits and below 2^-25 everything, so that without the bias the tail behind
// one key of nearly all the weight came out short (16 nats behind it 6 %, 17.5
// nats all).  bf16 has f32's range.
template <int CT>
constexpr float CH_BIAS = CT == RMLX_F16 ? 7.0f : 0.0f;

// Chunk token range, key tiles and masks of tile mt of a sequence.
struct TileGeo {
  int t0, rows, pos0, k_lo, nk, lo, hi;  // first token, rows, its position, first key tile, key tiles, keys [lo, hi)
};
__device__ __forceinline__ TileGeo tile_geo(int qlen, int len, int mt, int tpt, int G, int window) {
  TileGeo t;
  t.t0 = mt * tpt;
  const int n = min(tpt, qlen - t.t0);
  t.rows = n * G;
  t.pos0 = len - qlen + t.t0;
  t.hi = t.pos0 + n;
  t.lo = window && t.pos0 >= window ? t.pos0 - window + 1 : 0;
  t.k_lo = t.lo / CH_KEYS;
  t.nk = t.hi > 0 ? (t.hi - 1) / CH_KEYS + 1 - t.k_lo : 0;
  return t;
}

// A CTA's place in the plan, walked item by item by every warp.
struct ItemIter {
  int s, mt, head, qoff, qlen, len;
  int64_t off, left;  // position inside the item's cost, cost left in the share
  // the current portion
  TileGeo t;
  int k0, k1;   // its key tiles, relative to t.k_lo
  bool starts;  // it holds the item's beginning
};
__device__ __forceinline__ bool next_portion(ItemIter& it, const ChunkArgs& a, int heads, int tpt, bool first) {
  if (!first) {
    it.off = 0;
    if (++it.head == heads) {
      it.head = 0;
      if ((++it.mt) * tpt >= it.qlen) it.mt = 0, it.qoff += it.qlen, it.qlen = 0;
    }
  }
  if (it.left <= 0) return false;
  while (it.qlen <= 0) {  // the next sequence with chunk tokens
    if (++it.s >= a.nseq) return false;
    it.qlen = max(__ldg(a.q_lens + it.s), 0);
    it.len = min(max(__ldg(a.seq_lens + it.s), 0), a.max_len);
  }
  it.t = tile_geo(it.qlen, it.len, it.mt, tpt, a.G, a.window);
  const int64_t end = min(it.off + it.left, (int64_t)it.t.nk + CH_OVERHEAD);
  it.left -= end - it.off;
  it.starts = it.off == 0;
  it.k0 = (int)max(it.off - CH_OVERHEAD, (int64_t)0);
  it.k1 = (int)max(end - CH_OVERHEAD, (int64_t)0);
  return true;
}

// Sums of x[i] over the CTA's earlier threads into x[i], over all into total[i].
// words: N CH_MAX_WARPS 64-bit words of shared memory, read by nobody else before the next barrier.
template <int N>
__device__ __forceinline__ void block_prefix(int64_t (&x)[N], int64_t (&total)[N], int64_t* words) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    y[i] = x[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t z = __shfl_up_sync(0xffffffffu, y[i], o);
      if (lane >= o) y[i] += z;
    }
    if (lane == 31) words[i * CH_MAX_WARPS + warp] = y[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // every warp scans the warps' sums, one a lane
    int64_t w = lane < warps ? words[i * CH_MAX_WARPS + lane] : 0;
    const int64_t own = __shfl_sync(0xffffffffu, w, warp);
#pragma unroll
    for (int o = 1; o < CH_MAX_WARPS; o <<= 1) {
      const int64_t z = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += z;
    }
    total[i] = __shfl_sync(0xffffffffu, w, CH_MAX_WARPS - 1);
    x[i] = y[i] - x[i] + __shfl_sync(0xffffffffu, w, warp) - own;
  }
}

// n / d with 32 bits where they do (a 64-bit division takes some hundred clocks).
__device__ __forceinline__ int64_t div_small(int64_t n, int64_t d) {
  if (((n | d) >> 32) == 0) return (uint32_t)n / (uint32_t)d;
  return n / d;
}

// Cuts the work and leaves this CTA's share in *out (left = 0: none).
// scratch: 3 CH_MAX_WARPS 64-bit words, 2 (nseq + 1) words.  False when q_lens sum past
// a.nq.  Each thread walks a run of sequences, then a run of tiles.
__device__ __forceinline__ bool make_plan(const ChunkArgs& a, int heads, int tpt, uint8_t* scratch, ItemIter* out,
                                          int32_t* err) {
  int64_t* words = reinterpret_cast<int64_t*>(scratch);
  int32_t* cub = reinterpret_cast<int32_t*>(words + 3 * CH_MAX_WARPS);  // tiles before a sequence
  int32_t* cut = cub + a.nseq + 1;                                      // chunk tokens before it
  const int tid = threadIdx.x;
  if (tid == 0) out->left = 0;
  const int nt = blockDim.x, per_s = a.nseq <= nt ? 1 : (a.nseq + nt - 1) / nt;
  const int s0 = min(a.nseq, tid * per_s), s1 = min(a.nseq, s0 + per_s);
  int64_t before[2] = {0, 0}, all[2];  // tokens, tiles
  for (int s = s0; s < s1; ++s) {
    const int q = max(__ldg(a.q_lens + s), 0), len = __ldg(a.seq_lens + s);
    before[0] += q;
    before[1] += q ? (q - 1) / tpt + 1 : 0;
    if (q > 0 && len > a.max_len && blockIdx.x == 0) atomicOr(err, DEV_ERR_BLOCK);
  }
  block_prefix(before, all, words);
  if (all[0] > a.nq) return false;
  int token = (int)before[0], tile = (int)before[1];
  for (int s = s0; s < s1; ++s) {
    cub[s] = tile, cut[s] = token;
    const int q = max(__ldg(a.q_lens + s), 0);
    token += q;
    tile += q ? (q - 1) / tpt + 1 : 0;
  }
  if (tid == 0) cub[a.nseq] = (int)all[1], cut[a.nseq] = (int)all[0];
  __syncthreads();
  const int T = (int)all[1], per = T <= nt ? 1 : (T + nt - 1) / nt;
  const int beg = (int)min((int64_t)T, (int64_t)tid * per), end = min(T, beg + per);
  auto walk = [&](auto&& f) {  // f(sequence, its chunk length, its rows, tile, an item's cost)
    if (beg >= end) return;
    int s = find_seq(cub, a.nseq, beg);
    for (int i = beg; i < end; ++s) {
      const int qlen = cut[s + 1] - cut[s], len = min(max(__ldg(a.seq_lens + s), 0), a.max_len);
      for (const int stop = min(end, cub[s + 1]); i < stop; ++i) {
        const int mt = i - cub[s];
        f(s, qlen, len, mt, tile_geo(qlen, len, mt, tpt, a.G, a.window).nk + CH_OVERHEAD);
      }
    }
  };
  int64_t cost[1] = {0}, total[1];
  walk([&](int, int, int, int, int one) { cost[0] += (int64_t)heads * one; });
  const int64_t mine = cost[0];
  block_prefix(cost, total, words + 2 * CH_MAX_WARPS);
  const int64_t n = total[0] >= (int64_t)gridDim.x * CH_MIN_COST ? gridDim.x : max((int)total[0] / CH_MIN_COST, 1);
  if (blockIdx.x >= n) return true;
  const int64_t b0 = div_small(total[0] * blockIdx.x, n), b1 = div_small(total[0] * (blockIdx.x + 1), n);
  if (b0 < b1 && cost[0] <= b0 && b0 < cost[0] + mine) {
    int64_t c0 = cost[0];
    walk([&](int s, int qlen, int len, int mt, int one) {
      if (c0 <= b0 && b0 < c0 + (int64_t)heads * one) {
        const int head = (int)div_small(b0 - c0, one);
        out->s = s, out->mt = mt, out->qoff = cut[s], out->qlen = qlen, out->len = len;
        out->head = head, out->off = b0 - c0 - (int64_t)head * one;
        out->left = b1 - b0;
      }
      c0 += (int64_t)heads * one;
    });
  }
  return true;
}

// One partial result in the workspace: CH_ROWS unnormalised output rows, column
// by column, then a (max, sum) pair per row; what it is a part of in a descriptor.  Slot 0 of
// a CTA continues an item that an earlier CTA began, slot 1 begins one that a
// later CTA goes on with.
struct PartDesc {
  int32_t valid, last, token0, head, rows, pad[3];
};
__host__ __device__ constexpr size_t part_floats(int hd) { return (size_t)CH_ROWS * (hd + 2); }

// ---------------------------------------------------------------------------
// The kernel.  S = Q K^T and O += P V on the tcgen05 tensor cores, S, P and O
// in TMEM, K and V in a ring of shared-memory stages.  Warps 0-3 and 4-7 are
// two softmax warpgroups (A and B), one thread a row; warp 8 issues the MMAs;
// warp 9 loads K and V tiles by TMA and warps 10-11 the queries (pools that
// TMA cannot read: warps 9-15 load all).
//   more than 128 rows: A and B hold rows 0-127 and 128-255 and every key tile
//     is used twice;
//   up to 128 rows: A and B hold the same rows and take the even and the odd
//     key tiles, joined at the end.
// While one warpgroup does its softmax the tensor cores work for the other.  A
// warpgroup takes its 128 scores in halves: the first half's product runs while
// the second half's weights are computed.  P overwrites the first half of its
// scores.  O is rescaled only when a row's maximum has grown by more than 2^8
// since the last time (weights stay below 2^8, times the bias of f16; the final
// division undoes both).
// Measured for an 8192-token prompt (8 x 128, G = 4, bf16): 559 us, 984 TFLOP/s
// of the causal work, in bursts of 20 calls; 616 us at the power limit.  A key tile
// takes a warpgroup about 2460 clocks of softmax and 1750 of waiting for the two
// products, the tensor cores 2060.  Slower were: two threads a row (654 us), an
// MMA warp for each warpgroup (726), weights through shared memory so that the
// score buffer is free sooner (715), score buffers of 64 keys (N = 64 costs the
// tensor cores 56 clocks an MMA for half of what N = 128 does in 64).
//
// A V row that the mask hides is weighed with 0, which leaves NaN where it
// holds infinities or NaN.  Rows behind the last visible key are zeroed in
// shared memory; should a row's output come out NaN all the same, its warp
// computes that row again from the pool, reading visible rows only.
//
// Quantised pools: codes are dequantised to f16 in shared memory (K of f16 pools in
// two parts, CH_SPLIT) and the products run in f16 (11 bits; bf16's 8 would add
// more error than the codes), a query row scaled by a power of two to f16's upper
// end.  Groups whose values leave f16's range become NaN, and their rows take that
// path too, as do rows that groups of tiny values matter to.
// Where a box of codes and of (scale, zero) rows is whole 16-byte pieces, one
// warp fetches them by bulk copies (1-16 tokens over 4-bit pools of 1024-8192
// rows 184 us; with copies by the converting warps 10 us more).
// ---------------------------------------------------------------------------
struct ChunkParams {
  PoolGeo g;
  ChunkArgs a;
  int tpt;                 // chunk tokens of a tile
  int box;                 // rows of a TMA box, or of a bulk copy of codes: a power of two
  int raw_depth;           // tiles of codes in flight by bulk copies, 0: codes are copied by the load warps
  float* parts;
  PartDesc* desc;
};

// f16 pools over codes: K in two f16 parts, a stage each.  Their outputs have three
// bits more than bf16 ones, and K in one part cost most of them (rows with
// outliers: error 2.2 to 4 times that of the output's own rounding, with two parts
// 1.3 to 1.5); bf16 outputs show none of it (1.02 to 1.1).  The second part costs
// a half of the time again: 8-bit chunks 357 us instead of 230.
template <int DT, int BITS>
constexpr bool CH_SPLIT = BITS && DT == RMLX_F16;

template <int HD, int BITS, bool SPLIT>
struct ChunkSmem {
  static constexpr int QTILE = 128 * HD * 2;
  static constexpr int STAGE = CH_KEYS * HD * 2;
  // Quantised pools give two stages up for codes in flight (RAW): 3 tiles of
  // 8-bit codes with f16 scales, or 4 of 4-bit codes.  A fourth stage beside 3 tiles
  // of 4-bit codes serves K in two parts (1-16 tokens over 4-bit rows 12 % shorter).
  static constexpr bool FOURTH = SPLIT && BITS == 4 && HD == 128;
  static constexpr int STAGES = BITS ? (HD == 128 ? 3 + FOURTH : 6) : HD == 128 ? 5 : 8;
  static constexpr int UNITS = BITS ? CH_KEYS * HD * BITS / 128 : 0;  // of a tile
  static constexpr int RAW_BYTES = BITS == 8 ? UNITS * 60 : FOURTH ? UNITS * 56 : UNITS * 96;
  static constexpr int Q = 0, KV = 2 * QTILE, RAW = KV + STAGES * STAGE, CTRL = RAW + RAW_BYTES;
  // control block: barriers, then the plan, (max, sum) of warpgroup B, query scales, items with tiny groups
  static constexpr int BARS = CTRL, PLAN = CTRL + 352, ML = PLAN + 128, QSCALE = ML + 1024, TINY = QSCALE + 512;
  static constexpr int BYTES = TINY + 64;
};
// barrier numbers
constexpr int BAR_FULL = 0, BAR_EMPTY = 8, BAR_QFULL = 16, BAR_QEMPTY = 17, BAR_OFREE = 18, BAR_ML = 19, BAR_O = 20,
              BAR_S = 22, BAR_V = 24, BAR_P = 26, BAR_DRAIN = 30, BAR_RAWF = 31,
              BAR_RAWE = 35;  // P: warpgroup * 2 + half; RAW: up to CH_RAW slots

template <int DT>
__device__ __forceinline__ float unpack_lo(uint32_t w) {
  return DT == RMLX_BF16 ? __uint_as_float(w << 16) : __half2float(__ushort_as_half((uint16_t)w));
}
template <int DT>
__device__ __forceinline__ float unpack_hi(uint32_t w) {
  return DT == RMLX_BF16 ? __uint_as_float(w & 0xffff0000u) : __half2float(__ushort_as_half((uint16_t)(w >> 16)));
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (DT == RMLX_BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Weights of a row's 64 scores: 2^(c s + nb), stored to TMEM in the products'
// type (an MMA's operands have one 16-bit type; half a step of it costs about what
// the output's own rounding does: error 1.2 to 1.4 times that of f32 weights), and
// their f32 sum, of the unrounded ones.  All go to the special-function unit (4 a clock and
// SM quarter): with 1/8 to 1/2 of them as polynomials on the FMA pipe the
// softmax was shorter and the whole kernel slower (8192-token prompt 586 us,
// with a quarter 624 us).
template <int CT>
__device__ __forceinline__ float weights(const uint32_t (&v)[CH_HALF], float c, float nb, uint32_t tm_p) {
  const uint64_t c2 = f32x2(c, c), n2 = f32x2(nb, nb);
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int h = 0; h < CH_HALF / 32; ++h) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = 32 * h + 2 * i;
      float e0, e1;
      f32x2_split(fma_f32x2((uint64_t)v[k + 1] << 32 | v[k], c2, n2), e0, e1);
      e0 = ex2(e0);
      e1 = ex2(e1);
      sum[i & 1] = add_f32x2(sum[i & 1], f32x2(e0, e1));
      w[i] = pack2<CT>(e0, e1);
    }
    tmem_st16(tm_p + 16 * h, w);
  }
  float a, b;
  f32x2_split(add_f32x2(sum[0], sum[1]), a, b);
  return a + b;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Byte offset of 16-byte column c of row r in an operand tile: 128-byte
// swizzled atoms of 8 rows x 64 elements.  Query tiles keep a half's 128 rows
// together; K/V stages keep the halves of each 8 rows together, as a TMA box
// of a block's rows leaves them.
template <int HD>
__device__ __forceinline__ uint32_t q_off(int r, int c) {
  return (c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}
template <int HD>
__device__ __forceinline__ uint32_t kv_off(int r, int c) {
  return (r >> 3) * (HD * 16) + (c >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// (scale, zero) pair q of a stored row, as it lies in memory (f16: in one word).
__device__ __forceinline__ uint2 load_meta(const uint8_t* meta, int q, bool mf32) {
  if (mf32) return __ldg(reinterpret_cast<const uint2*>(meta) + q);
  return make_uint2(__ldg(reinterpret_cast<const uint32_t*>(meta) + q), 0u);
}
// A group's scale and zero as the conversion takes them.  Its values lie
// between zr and zr + qmax sc: where they leave f16's range the scale becomes NaN,
// and the rows that see the group take the exact path.  True when the group is
// tiny: its largest value is below 2^-13, where f16's smallest step (a rounding of
// 2^-25) costs more than 2^-12 of it.  With f16 scales and zeros none is: all
// values are multiples of 2^-24, and those below 2^-13 are f16 numbers.
template <int BITS>
struct Group {
  float sc, zr;
  __half2 sc2, zr2;
  __device__ __forceinline__ bool set(uint2 meta, bool mf32) {
    float s = mf32 ? __uint_as_float(meta.x) : unpack_lo<RMLX_F16>(meta.x);
    const float z = mf32 ? __uint_as_float(meta.y) : unpack_hi<RMLX_F16>(meta.x);
    const float top = fmaxf(fabsf(z), fabsf(fmaf((float)((1 << BITS) - 1), s, z)));
    const float least = s == 1.0f ? fabsf(z) : top;  // a flat group has scale 1 and no code but 0
    if (!(top <= 65504.0f)) s = __uint_as_float(0x7fffffffu);
    sc = s, zr = z;
    sc2 = __float2half2_rn(s), zr2 = __float2half2_rn(z);
    return mf32 && least > 0.0f && least < 1.220703125e-4f;
  }
};
// Eight elements as f16 pairs from their codes, a byte each.  A code becomes
// the f16 1024 + code by a byte permute, then code exactly; f16 scale and
// zero give code * scale + zero with one rounding, f32 ones with one of f32 more.
template <int BITS, bool MF32>
__device__ __forceinline__ uint4 dequant8(uint2 w, const Group<BITS>& g) {
  uint4 r;
  uint32_t* o = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = __byte_perm(i < 2 ? w.x : w.y, 0x64646464u, (i & 1) ? 0x4342 : 0x4140);
    const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&m), __floats2half2_rn(1024.0f, 1024.0f));
    __half2 v;
    if (MF32) {
      const float2 f = __half22float2(c);
      v = __floats2half2_rn(fmaf(f.x, g.sc, g.zr), fmaf(f.y, g.sc, g.zr));
    } else {
      v = __hfma2(c, g.sc2, g.zr2);
    }
    o[i] = *reinterpret_cast<uint32_t*>(&v);
  }
  return r;
}
// a b + c of f16 factors in f32, with one rounding.
__device__ __forceinline__ float fma_f32_f16(__half a, __half b, float c) {
  float d;
  asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(d) : "h"(__half_as_ushort(a)), "h"(__half_as_ushort(b)), "f"(c));
  return d;
}
// What dequant8's f16 elements leave of the values, in f16: both together hold 22
// bits of them, or 2^-25.  Mixed-precision multiply-adds take the f16 factors as
// they are (with conversions of codes and elements to f32 8-bit chunks took 386 us).
template <int BITS, bool MF32>
__device__ __forceinline__ uint4 dequant8_rest(uint2 w, const Group<BITS>& g, uint4 hi) {
  uint4 r;
  const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w};
  uint32_t* o = reinterpret_cast<uint32_t*>(&r);
  const __half minus = __ushort_as_half(0xbc00);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = __byte_perm(i < 2 ? w.x : w.y, 0x64646464u, (i & 1) ? 0x4342 : 0x4140);
    const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&m), __floats2half2_rn(1024.0f, 1024.0f));
    const __half2 x = *reinterpret_cast<const __half2*>(&h[i]);
    float v0, v1;
    if (MF32) {
      const float2 f = __half22float2(c);
      v0 = fmaf(f.x, g.sc, g.zr), v1 = fmaf(f.y, g.sc, g.zr);
    } else {
      v0 = fma_f32_f16(__low2half(c), __low2half(g.sc2), g.zr), v1 = fma_f32_f16(__high2half(c), __low2half(g.sc2), g.zr);
    }
    o[i] = pack2<RMLX_F16>(fma_f32_f16(__low2half(x), minus, v0), fma_f32_f16(__high2half(x), minus, v1));
  }
  return r;
}
// Eight 4-bit codes, low nibble first, as bytes.
__device__ __forceinline__ uint2 nibbles(uint32_t w) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
  return make_uint2(__byte_perm(lo, hi, 0x5140), __byte_perm(lo, hi, 0x7362));
}

// Every lane has 64 bytes of a row of its own, going to dst (if valid).  Lanes
// of a group of four trade 16-byte pieces so that a store instruction writes
// whole 64-byte runs: a lane a row would write 16 bytes of 32 lines at once.
__device__ __forceinline__ void store_rows64(uint32_t (&w)[16], uint8_t* dst, bool valid, int lane) {
  const unsigned long long at = valid ? reinterpret_cast<unsigned long long>(dst) : 0;
  // transpose the 4 x 4 pieces: exchange blocks of 2, then single ones
#pragma unroll
  for (int s = 2; s; s >>= 1) {
    const bool up = lane & s;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (a & s) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t keep = up ? w[4 * (a | s) + e] : w[4 * a + e], give = up ? w[4 * a + e] : w[4 * (a | s) + e];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, s);
        w[4 * a + e] = up ? got : keep;
        w[4 * (a | s) + e] = up ? keep : got;
      }
    }
  }
  // lane 4 g + c now holds piece c of the rows of lanes 4 g .. 4 g + 3
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const unsigned long long row = __shfl_sync(0xffffffffu, at, (lane & 28) | r);
    if (row)
      reinterpret_cast<uint4*>(row)[lane & 3] = make_uint4(w[4 * r], w[4 * r + 1], w[4 * r + 2], w[4 * r + 3]);
  }
}

// This lane's head_dim / 32 elements of U stored rows (K or V) as they lie in
// memory: plain rows', or codes with the (scale, zero) of their group.
template <int HD, int BITS, int U>
struct LaneRows {
  static constexpr int EPL = HD / 32, BYTES = EPL * (BITS ? BITS : 16) / 8;
  uint32_t w[U][BYTES == 8 ? 2 : 1];
  uint2 meta[U];
  // tile[u]: the tile of row u (slot row[u] of its block)
  __device__ __forceinline__ void load(const PoolGeo& g, const ChunkArgs& a, const uint8_t* const (&tile)[U],
                                       const int (&row)[U], int lane) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint8_t* p = tile[u] + (int64_t)row[u] * g.row_bytes + lane * BYTES;
      if constexpr (BYTES == 8) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
        w[u][0] = x.x, w[u][1] = x.y;
      } else if constexpr (BYTES == 4) {
        w[u][0] = __ldg(reinterpret_cast<const uint32_t*>(p));
      } else if constexpr (BYTES == 2) {
        w[u][0] = __ldg(reinterpret_cast<const uint16_t*>(p));
      } else {
        w[u][0] = __ldg(p);
      }
    }
    if constexpr (BITS != 0) {
      const int q = (lane * EPL) >> a.gs_log2;
      auto at = [&](int u) { return tile[u] + (int64_t)g.bs * g.row_bytes + (int64_t)row[u] * g.meta_row_bytes; };
      if (a.mf32) {
#pragma unroll
        for (int u = 0; u < U; ++u) meta[u] = __ldg(reinterpret_cast<const uint2*>(at(u)) + q);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t m = __ldg(reinterpret_cast<const uint32_t*>(at(u)) + q);
          meta[u] = make_uint2(__float_as_uint(unpack_lo<RMLX_F16>(m)), __float_as_uint(unpack_hi<RMLX_F16>(m)));
        }
      }
    }
  }
  // Row u in f32; codes are not rounded to the pool's type (8 bits of a bf16 value would cost more than the codes' own).
  template <int DT>
  __device__ __forceinline__ void get(int u, float (&f)[EPL]) const {
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      if constexpr (BITS == 0)
        f[e] = (e & 1) ? unpack_hi<DT>(w[u][e >> 1]) : unpack_lo<DT>(w[u][e >> 1]);
      else
        f[e] = __fadd_rn(__fmul_rn((float)((w[u][0] >> (BITS * e)) & ((1u << BITS) - 1)), __uint_as_float(meta[u].x)),
                         __uint_as_float(meta[u].y));
    }
  }
};

// What a warp's lanes know of an item's portion whose rows are computed again.
struct AgainRows {
  const int32_t* btrow;
  float* part;            // where a portion's partial rows go, nullptr when the rows are whole
  int64_t token0, orow;   // first chunk token of the tile in q; this lane's row in out
  int head, k_first, k_end;
  int row, lim, low;      // this lane's row of the tile: it sees keys low <= key < lim
};

// The exact path: the rows of the lanes in `bad` again in f32, four rows and four
// keys at a time by the whole warp, with the running maximum and sum of a softmax
// in the log2 domain.  A row that none of the four sees is never read, and one that
// a row's mask hides has no part in that row.  Lane 4 r + u ends up with the score
// of row r and key u (15 shuffles for 16 sums over the lanes, and one that joins the
// warp's halves) and keeps its row's maximum and its own share of the sum.  Bound
// by instruction issue: about 100 ns a row and key in each of eight warps (82 of a
// plain pool); a row and a key at a time took 950.  Out of line, and four keys
// instead of eight, so that its registers are not the main loop's.
template <int DT, int HD, int BITS>
__device__ __noinline__ void attend_rows_again(const ChunkParams& p, const AgainRows& it, unsigned bad, int32_t* err) {
  constexpr int EPL = HD / 32, R = 4, U = 4;
  constexpr unsigned FULL = 0xffffffffu;
  const PoolGeo& g = p.g;
  const ChunkArgs& a = p.a;
  const int lane = threadIdx.x & 31, u_own = lane % U, r_own = lane / U % R;
  const int64_t vdelta = (int64_t)g.heads * g.tile_bytes;
  auto block_of = [&](int j) { return a.bs_log2 >= 0 ? j >> a.bs_log2 : j / g.bs; };
  bool out_of_pool = false;
#pragma unroll 1
  while (bad) {
    int from[R], n = 0;  // the lanes whose rows are taken; a last row stands in for missing ones
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (bad) {
        from[r] = __ffs(bad) - 1, bad &= bad - 1, ++n;
      } else {
        from[r] = from[r ? r - 1 : 0];
      }
    }
    float q[R][EPL], acc[R][EPL];
    int k0 = INT32_MAX, k1 = 0, own0 = 0, own1 = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = __shfl_sync(FULL, it.row, from[r]);
      const int r0 = max(__shfl_sync(FULL, it.low, from[r]), it.k_first), r1 = min(__shfl_sync(FULL, it.lim, from[r]), it.k_end);
      k0 = min(k0, r0), k1 = max(k1, r1);
      if (r == r_own) own0 = r0, own1 = r1;
      const int tok = row / a.G;
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q + (it.token0 + tok) * a.qts +
                                                             (it.head * a.G + row - tok * a.G) * a.qhs) + lane * EPL;
#pragma unroll
      for (int e = 0; e < EPL; ++e) q[r][e] = unpack_lo<DT>(__ldg(qp + e)), acc[r][e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
#pragma unroll 1
    for (int j0 = k0; j0 < k1; j0 += U) {
      const uint8_t* tile[U];
      int slot[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = min(j0 + u, k1 - 1), b = block_of(j);
        const int32_t blk = __ldg(it.btrow + b);
        const bool good = blk >= 0 && blk < g.nblocks;
        out_of_pool |= !good;
        tile[u] = g.base + g.tile_off(good ? blk : 0, a.layer, 0, it.head);
        slot[u] = j - b * g.bs;
      }
      LaneRows<HD, BITS, U> kr, vr;
      kr.load(g, a, tile, slot, lane);
      float s[R * U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[EPL];
        kr.template get<DT>(u, f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          s[r * U + u] = 0.0f;
#pragma unroll
          for (int e = 0; e < EPL; ++e) s[r * U + u] = fmaf(q[r][e], f[e], s[r * U + u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) tile[u] += vdelta;
      vr.load(g, a, tile, slot, lane);
#pragma unroll
      for (int o = R * U / 2; o; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
          const float keep = up ? s[i + o] : s[i], give = up ? s[i] : s[i + o];
          s[i] = keep + __shfl_xor_sync(FULL, give, o);
        }
      }
#pragma unroll
      for (int o = R * U; o < 32; o <<= 1) s[0] += __shfl_xor_sync(FULL, s[0], o);
      const bool sees = j0 + u_own >= own0 && j0 + u_own < own1;
      const float x = sees ? s[0] * a.scale_log2 : -INFINITY;
      float top = x;
#pragma unroll
      for (int o = U / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
      top = fmaxf(top, m);
      const float base = top == -INFINITY ? 0.0f : top;  // scores of -inf before any other: exp2(-inf - 0) = 0
      const float f = exp2f(m - base), w = exp2f(x - base);
      m = top;
      l = fmaf(l, f, w);
      const float mine = sees ? w : -1.0f;  // below 0: hidden, whatever the row holds
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float fr = __shfl_sync(FULL, f, r * U);
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[r][e] *= fr;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[EPL];
        vr.template get<DT>(u, v);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float pr = __shfl_sync(FULL, mine, r * U + u);
          const bool use = !(pr < 0.0f);  // NaN counts
#pragma unroll
          for (int e = 0; e < EPL; ++e) acc[r][e] = use ? fmaf(pr, v[e], acc[r][e]) : acc[r][e];
        }
      }
    }
#pragma unroll
    for (int o = U / 2; o; o >>= 1) l += __shfl_xor_sync(FULL, l, o);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float rl = __shfl_sync(FULL, l, r * U), rm = __shfl_sync(FULL, m, r * U);
      const int row = __shfl_sync(FULL, it.row, from[r]);
      const int64_t orow = __shfl_sync(FULL, it.orow, from[r]);
      if (r >= n) continue;
      if (it.part) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) it.part[(size_t)(lane * EPL + e) * CH_ROWS + row] = acc[r][e];
        if (lane == 0) reinterpret_cast<float2*>(it.part + (size_t)CH_ROWS * HD)[row] = make_float2(rm, rl);
      } else {
        const float il = rl == 0.0f ? 0.0f : 1.0f / rl;
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          reinterpret_cast<uint16_t*>(a.out)[orow * HD + lane * EPL + e] = (uint16_t)pack2<DT>(acc[r][e] * il, 0.0f);
      }
    }
  }
  if (out_of_pool && lane == 0) atomicOr(err, DEV_ERR_BLOCK);
}

template <int DT, int HD, int BITS, bool TMA>
__global__ void __launch_bounds__(ch_threads(TMA), 1)
    chunk_attn_kernel(const __grid_constant__ ChunkParams p, const __grid_constant__ CUtensorMap map, int32_t* err) {
  constexpr bool SPLIT = CH_SPLIT<DT, BITS>;
  using S = ChunkSmem<HD, BITS, SPLIT>;
  constexpr int CT = BITS ? RMLX_F16 : DT;  // type of the products' operands
  constexpr int ST = S::STAGES;
  constexpr uint32_t IDESC_S = mma_idesc(CT == RMLX_BF16, 128, CH_KEYS, false);
  constexpr uint32_t IDESC_O = mma_idesc(CT == RMLX_BF16, 128, HD, true);
  constexpr uint32_t TM_S = 0, TM_O = 256;  // TMEM columns: S/P of A and B, then O of A and B
  // Load warps beside the one that issues TMA or bulk copies (none does where
  // rows are copied by the load warps themselves): they load queries, and rows
  // or codes.
  const bool raw = BITS && p.raw_depth;
  const int qwarps = TMA ? 2 : raw ? 6 : 7;
  extern __shared__ __align__(1024) uint8_t smem[];  // swizzle atoms are 1024 bytes
  const uint32_t sb = smem_u32(smem);
  const PoolGeo& g = p.g;
  const ChunkArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto bar = [&](int i) { return sb + S::BARS + 8 * i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::BARS + 336);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::BARS + 340);
  ItemIter* plan = reinterpret_cast<ItemIter*>(smem + S::PLAN);
  float2* ml_b = reinterpret_cast<float2*>(smem + S::ML);
  uint8_t* qscale = smem + S::QSCALE;  // [2][CH_ROWS] f32 exponents, by item parity
  // [K, V][item % 8]: number, from 1, of an item with a tiny group there (loads run at most four items ahead of an epilogue)
  volatile uint32_t* tiny = reinterpret_cast<volatile uint32_t*>(smem + S::TINY);

  if (threadIdx.x < 16) tiny[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < ST; ++i) {
      mbar_init(bar(BAR_FULL + i), TMA ? 1 : qwarps);
      mbar_init(bar(BAR_EMPTY + i), 1);
    }
    mbar_init(bar(BAR_QFULL), qwarps);
    mbar_init(bar(BAR_QEMPTY), 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(bar(BAR_S + x), 1);
      mbar_init(bar(BAR_V + x), 1);
      mbar_init(bar(BAR_O + x), 1);
      mbar_init(bar(BAR_P + 2 * x), 4);
      mbar_init(bar(BAR_P + 2 * x + 1), 4);
    }
    mbar_init(bar(BAR_DRAIN), 1);
    for (int i = 0; i < CH_RAW; ++i) mbar_init(bar(BAR_RAWF + i), 1), mbar_init(bar(BAR_RAWE + i), 6);
    mbar_init(bar(BAR_OFREE), 8);
    mbar_init(bar(BAR_ML), 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) tmem_alloc(sb + S::BARS + 340, 512);
  pdl_wait();
  pdl_release();
  PartDesc* desc = p.desc + 2 * blockIdx.x;
  if (threadIdx.x < 2) desc[threadIdx.x].valid = desc[threadIdx.x].last = 0;
  if (!make_plan(a, g.heads, p.tpt, smem + S::KV, plan, err) && threadIdx.x == 0) atomicOr(err, DEV_ERR_Q_ROWS);
  fence_async_smem();  // the plan's scratch becomes the K/V ring
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  ItemIter it = *plan;
  const int qheads = g.heads * a.G;
  uint32_t copies = 0;  // TMA or bulk loads that this warp has issued

  if (warp < 8) {
    // ---- softmax warpgroups -----------------------------------------------
    const int x = warp >> 2, wq = warp & 3;
    const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
    const uint32_t tm_s = tmem + lane_off + TM_S + 128 * x, tm_o = tmem + lane_off + TM_O + HD * x;
    uint32_t ns = 0, nitem = 0, nml = 0, no[2] = {0, 0};  // phases: S tiles, items, (max, sum) handed over, O of A and B
    for (bool more = next_portion(it, a, g.heads, p.tpt, true); more;
         more = next_portion(it, a, g.heads, p.tpt, false)) {
      const int nk = it.k1 - it.k0;
      const bool two = it.t.rows > 128;
      const int row = (two ? 128 * x : 0) + wq * 32 + lane;
      const int tok = row / a.G, gq = row - tok * a.G;
      const bool valid = row < it.t.rows;
      const int64_t orow = (int64_t)(it.qoff + it.t.t0 + tok) * qheads + it.head * a.G + gq;
      if (nk == 0) {
        // an item with no visible key at all: zeros
        if (it.starts && it.t.nk == 0 && valid && (two || x == 0)) {
          uint4* o = reinterpret_cast<uint4*>(p.a.out + orow * HD * 2);
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) o[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        continue;
      }
      // half tiles: two a tile, one of the last tile where no key of its second half is visible
      const bool odd = it.t.hi - (it.t.k_lo + it.k1 - 1) * CH_KEYS <= CH_HALF;
      const int mine = two ? 2 * nk - odd : 2 * (x == 0 ? (nk + 1) / 2 : nk / 2) - (odd && x == ((nk - 1) & 1));
      const bool active = (two ? 128 * x : 0) + wq * 32 < it.t.rows;
      const int pos = it.t.pos0 + tok;
      const int lim = valid ? max(pos + 1, 0) : INT32_MAX;  // visible keys: low <= key < lim
      const int low = valid && a.window && pos >= a.window ? pos - a.window + 1 : 0;
      // A lane without a row scores whatever lies in shared memory: with a maximum
      // that nothing exceeds it has no say in when the warp moves its rows' maxima,
      // and the rows' bits do not depend on what ran before.
      float m = valid ? -INFINITY : INFINITY, l = 0.0f, c = a.scale_log2;
      bool ok = true;
      for (int j = 0; j < mine; ++j) {
        const int b = j & 1;
        if (b == 0 && !(ok = mbar_wait(bar(BAR_S + x), ns++ & 1, abort_flag, a.wait_ns, err))) break;
        if (active) {
          tc_fence_after();
          if (BITS && j == 0) c = a.scale_log2 * __uint_as_float((uint32_t)qscale[(nitem & 1) * CH_ROWS + row] << 23);
          uint32_t v[CH_HALF];
          tmem_ld32(tm_s + CH_HALF * b, v);
          tmem_ld32(tm_s + CH_HALF * b + 32, v + 32);
          const int kb = (it.t.k_lo + it.k0 + (two ? j >> 1 : (j & ~1) + x)) * CH_KEYS + CH_HALF * b;
          const bool masked = __any_sync(0xffffffffu, kb + CH_HALF > lim || kb < low);
          tmem_ld_wait32(v);
          tmem_ld_wait32(v + 32);
          if (masked) {
            const int r1 = lim - kb, r0 = low - kb;
#pragma unroll
            for (int i = 0; i < CH_HALF; ++i)
              if (i >= r1 || i < r0) v[i] = 0xff800000u;  // -inf
          }
          float mx4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mx4[i] = fmaxf(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
#pragma unroll
          for (int i = 8; i < CH_HALF; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mx4[k] = fmaxf(mx4[k], fmaxf(__uint_as_float(v[i + 2 * k]), __uint_as_float(v[i + 2 * k + 1])));
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          if (__any_sync(0xffffffffu, (mx - m) * c > 8.0f)) {
            const float n = fmaxf(m, mx);
            const float f = n == m ? 1.0f : ex2((m - n) * c);
            m = n;
            l *= f;
            if (j > 0) {
              // products into O have to be done: those of earlier tiles are (these scores were issued
              // behind them), the tile's first half signals its own
              if (b && !(ok = mbar_wait(bar(BAR_V + x), (ns - 1) & 1, abort_flag, a.wait_ns, err))) break;
              tc_fence_after();
#pragma unroll 1
              for (int i = 0; i < HD; i += 16) {
                uint32_t o[16];
                tmem_ld16(tm_o + i, o);
                tmem_ld_wait16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st16(tm_o + i, o);
              }
              tc_wait_st();
            }
          }
          const float nb = m == -INFINITY ? 0.0f : CH_BIAS<CT> - m * c;
          l += weights<CT>(v, c, nb, tm_s + CH_HALF * b);
          tc_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(BAR_P + 2 * x + b));
      }
      if (!ok) break;
      // ---- epilogue ---------------------------------------------------------
      float ml = m == -INFINITY ? -INFINITY : m * c - CH_BIAS<CT>;  // in the log2 domain: O and l are in units of 2^ml
      const bool whole = it.k0 == 0 && it.k1 == it.t.nk;
      const int slot = it.k0 == 0 ? 1 : 0;
      float* part = p.parts + (size_t)(2 * blockIdx.x + slot) * part_floats(HD);
      if (!whole && threadIdx.x == 0) {
        desc[slot].last = it.k1 == it.t.nk, desc[slot].token0 = it.qoff + it.t.t0;
        desc[slot].head = it.head, desc[slot].rows = it.t.rows, desc[slot].valid = 1;
      }
      bool writes = active;
      float fa = 1.0f, fb = 0.0f;
      const bool has[2] = {true, two || nk > 1};  // A and B have tiles
      if (!two) {
        if (x == 1) {
          if (nitem > 0 && !(ok = mbar_wait(bar(BAR_OFREE), (nitem - 1) & 1, abort_flag, a.wait_ns, err))) break;
          ml_b[wq * 32 + lane] = make_float2(ml, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(BAR_ML));
          writes = false;
        } else {
          if (!(ok = mbar_wait(bar(BAR_ML), nml & 1, abort_flag, a.wait_ns, err))) break;
          const float2 b = ml_b[wq * 32 + lane];
          const float n = fmaxf(ml, b.x);
          const float base = n == -INFINITY ? 0.0f : n;
          fa = ex2(ml - base);
          fb = ex2(b.x - base);  // 0 without tiles
          l = l * fa + b.y * fb;
          ml = n;
        }
        ++nml;
      }
#pragma unroll
      for (int y = 0; y < 2 && ok; ++y) {
        // a warpgroup reads its own O, and A reads B's too when they share rows
        if (has[y] && (y == x || (!two && x == 0))) ok = mbar_wait(bar(BAR_O + y), no[y] & 1, abort_flag, a.wait_ns, err);
        no[y] += has[y];
      }
      if (!ok) break;
      ++nitem;
      if (writes) {
        tc_fence_after();
        const float il = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
        float nan = l;  // becomes NaN with any NaN among the outputs
        // Tiny groups lie in f16 with an error of up to 2^-25.  In V that is more than
        // 2^-12 of a group's largest output where this is below 2^-13: such a row is
        // computed again (f16 outputs are rounded by 2^-25 themselves).  In K it moves a
        // score by 2^-25 scale sum |q|, at most 2^-12 unless head_dim times the row's
        // largest element (below 2^15 in units of c) is above 2^13 / scale.
        const bool tiny_v = BITS && DT == RMLX_BF16 && tiny[8 + ((nitem - 1) & 7)] == nitem;
        const float faint = (whole ? 1.0f : l) * 1.220703125e-4f;
        bool again = BITS && tiny[(nitem - 1) & 7] == nitem && c * HD > 0.25f * 1.4426950408889634f;
#pragma unroll 1
        for (int i = 0; i < HD; i += 32) {
          uint32_t o[32];
          tmem_ld32(tm_o + i, o);
          tmem_ld_wait32(o);
          float f[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(o[e]);
          if (!two) {
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] *= fa;
            if (has[1]) {
              tmem_ld32(tm_o + HD + i, o);
              tmem_ld_wait32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) f[e] = fmaf(__uint_as_float(o[e]), fb, f[e]);
            }
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            f[e] = l == 0.0f ? 0.0f : f[e] * il;
            nan = fmaf(f[e], 0.0f, nan);
          }
          if (tiny_v) {  // the largest of each group's columns, or of these 32
            float top[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              top[k] = fabsf(f[8 * k]);
#pragma unroll
              for (int e = 1; e < 8; ++e) top[k] = fmaxf(top[k], fabsf(f[8 * k + e]));
            }
            if (a.gs_log2 > 3) top[0] = top[1] = fmaxf(top[0], top[1]), top[2] = top[3] = fmaxf(top[2], top[3]);
            if (a.gs_log2 > 4) top[0] = top[1] = top[2] = top[3] = fmaxf(top[0], top[2]);
            again |= fminf(fminf(top[0], top[1]), fminf(top[2], top[3])) < faint;
          }
          if (whole) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = pack2<DT>(f[2 * e], f[2 * e + 1]);
            store_rows64(w, p.a.out + (orow * HD + i) * 2, valid, lane);
          } else if (valid) {
#pragma unroll
            for (int e = 0; e < 32; ++e) part[(size_t)(i + e) * CH_ROWS + row] = f[e];  // a warp's lanes side by side
          }
        }
        if (valid && !whole) reinterpret_cast<float2*>(part + (size_t)CH_ROWS * HD)[row] = make_float2(ml, l);
        // rows whose output holds NaN, or too few digits: again, from visible rows only
        const unsigned bad = __ballot_sync(0xffffffffu, valid && (nan != nan || again));
        if (bad) {
          __syncwarp();  // other lanes store these rows again: behind what this lane has stored of them
          AgainRows rows;
          rows.btrow = a.bt + (int64_t)it.s * a.bt_stride;
          rows.part = whole ? nullptr : part;
          rows.token0 = it.qoff + it.t.t0, rows.orow = orow, rows.head = it.head;
          rows.k_first = (it.t.k_lo + it.k0) * CH_KEYS, rows.k_end = (it.t.k_lo + it.k1) * CH_KEYS;
          rows.row = row, rows.lim = lim, rows.low = low;
          attend_rows_again<DT, HD, BITS>(p, rows, bad, err);
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(BAR_OFREE));
    }
  } else if (warp == 8) {
    // ---- MMA issue ----------------------------------------------------------
    uint32_t nitem = 0, pp = 0;  // items; a phase bit for each P buffer
    uint32_t st = 0, ph = 0;     // the ring's next stage and its phase
    bool ok = true;
    auto wait = [&](int b, uint32_t parity) { return ok = ok && mbar_wait(bar(b), parity & 1, abort_flag, a.wait_ns, err); };
    auto advance = [&] {
      if (++st == ST) st = 0, ph ^= 1;
    };
    // operand descriptors of the first stage; a stage, or 64 rows, adds its bytes / 16
    constexpr uint32_t HALF = CH_HALF * HD * 2 / 16;
    const uint64_t qd = smem_desc(sb + S::Q, 16, 1024), kd = smem_desc(sb + S::KV, 16, HD * 16),
                   vd = smem_desc(sb + S::KV, 1024, HD * 16);
    struct KeyStages {
      uint32_t hi, lo;
    };
    auto scores = [&](int x, int qt, KeyStages k) {  // S[x] = Q[qt] K^T
      const uint64_t q = qd + (uint32_t)(qt * (S::QTILE / 16));
      mma_ss_rows<HD>(tmem + TM_S + 128 * x, q, kd + k.hi * (S::STAGE / 16), IDESC_S, 0);
      if (SPLIT) mma_ss_rows<HD>(tmem + TM_S + 128 * x, q, kd + k.lo * (S::STAGE / 16), IDESC_S, 1);
      tc_commit(bar(BAR_S + x));
    };
    auto next_stage = [&] {  // once it is full; the ring's next one after it
      const uint32_t s = st;
      wait(BAR_FULL + s, ph);
      advance();
      return s;
    };
    auto next_keys = [&] {
      KeyStages k;
      k.hi = next_stage();
      k.lo = SPLIT ? next_stage() : k.hi;
      return k;
    };
    auto free_keys = [&](KeyStages k) {
      tc_commit(bar(BAR_EMPTY + k.hi));
      if (SPLIT) tc_commit(bar(BAR_EMPTY + k.lo));
    };
    auto values = [&](int x, uint32_t stage, int h, int keys, bool first) {  // O[x] (+)= P[x][h] V
      const uint64_t v0 = vd + (stage * (S::STAGE / 16) + h * HALF);
      const uint32_t o = tmem + TM_O + HD * x, s = tmem + TM_S + 128 * x + CH_HALF * h;
      if (keys >= CH_HALF - 15) {
        mma_ts_64<HD>(o, s, v0, IDESC_O, !first);
      } else {
        for (int kk = 0; 16 * kk < keys; ++kk) mma_ts_16(o, s + 8 * kk, v0 + kk * (HD * 2), IDESC_O, kk > 0 || !first);
      }
    };
    auto weights_ready = [&](int x, int h) {
      if (!wait(BAR_P + 2 * x + h, pp >> (2 * x + h))) return false;
      pp ^= 1u << (2 * x + h);
      tc_fence_after();
      return true;
    };
    for (bool more = next_portion(it, a, g.heads, p.tpt, true); more;
         more = next_portion(it, a, g.heads, p.tpt, false)) {
      const int nk = it.k1 - it.k0;
      if (nk == 0) continue;
      const bool two = it.t.rows > 128;
      auto keys_of = [&](int j) { return min(CH_KEYS, it.t.hi - (it.t.k_lo + it.k0 + j) * CH_KEYS); };
      auto fill = [&](uint32_t stage, int keys) {
        // V rows behind the last visible key that share its MMA step: zeros
        if (TMA && (keys & 15)) {
          for (int i = lane; i < (16 - (keys & 15)) * (HD / 8); i += 32)
            sts128(sb + S::KV + stage * S::STAGE + kv_off<HD>(keys + i / (HD / 8), i % (HD / 8)), make_uint4(0u, 0u, 0u, 0u));
          fence_async_smem();
          __syncwarp();
        }
      };
      const int lead = two ? 1 : min(2, nk);
      if (!wait(BAR_QFULL, nitem)) break;
      for (int i = 0; i < lead; ++i) {
        const KeyStages k = next_keys();
        if (!ok) break;
        tc_fence_after();
        scores(two ? 0 : i, 0, k);
        if (two) scores(1, 1, k);
        free_keys(k);
      }
      if (!ok) break;
      if (lead == nk) tc_commit(bar(BAR_QEMPTY));
      if (nitem > 0 && !wait(BAR_OFREE, nitem - 1)) break;
      for (int j = 0; j < nk; ++j) {
        const uint32_t sv = next_stage();
        if (!ok) break;
        const int keys = keys_of(j), jn = j + lead;
        fill(sv, keys);
        KeyStages sk = {0, 0};
        if (jn < nk) {
          sk = next_keys();
          if (!ok) break;
        }
        for (int y = 0; y < (two ? 2 : 1); ++y) {
          const int x = two ? y : j & 1;
          const bool first = j < lead;
          if (!weights_ready(x, 0)) break;
          values(x, sv, 0, keys, first);
          tc_commit(bar(BAR_V + x));
          if (keys > CH_HALF) {
            if (!weights_ready(x, 1)) break;
            values(x, sv, 1, keys - CH_HALF, false);
          }
          if (jn < nk) {
            scores(x, two ? y : 0, sk);
          } else {
            tc_commit(bar(BAR_O + x));
          }
        }
        if (!ok) break;
        tc_commit(bar(BAR_EMPTY + sv));
        if (jn < nk) {
          free_keys(sk);
          if (jn == nk - 1) tc_commit(bar(BAR_QEMPTY));
        }
      }
      if (!ok) break;
      ++nitem;
    }
  } else {
    // ---- loads ----------------------------------------------------------------
    uint32_t n = 0, nitem = 0;   // loads, items
    uint32_t ns = 0;             // stages filled (elsewhere than in SPLIT kernels a load is a stage)
    bool ok = true;
    const bool issues = (TMA || raw) && warp == 9, loads_q = !issues;
    const bool loads_kv = issues || !TMA;
    const int qw = TMA || raw ? warp - 10 : warp - 9;
    for (bool more = next_portion(it, a, g.heads, p.tpt, true); more;
         more = next_portion(it, a, g.heads, p.tpt, false)) {
      const int nk = it.k1 - it.k0;
      if (nk == 0) continue;
      const bool two = it.t.rows > 128;
      const int32_t* btrow = a.bt + (int64_t)it.s * a.bt_stride;
      if (loads_q) {
        if (nitem > 0 && !(ok = mbar_wait(bar(BAR_QEMPTY), (nitem - 1) & 1, abort_flag, a.wait_ns, err))) break;
        constexpr int CPR = HD / 8, RPW = 32 / CPR;  // 16-byte chunks of a row, rows of a warp's pass
        const uint8_t* qbase = a.q + (int64_t)(it.qoff + it.t.t0) * a.qts + (int64_t)it.head * a.G * a.qhs;
        const int ch = lane % CPR;
        const int step = qwarps * RPW;
        if (!BITS) {
          // every row's copy in flight at once
          for (int r = qw * RPW + lane / CPR; r < it.t.rows; r += step) {
            const int tok = r / a.G;
            cp_async16(sb + S::Q + (r >> 7) * S::QTILE + q_off<HD>(r & 127, ch),
                       qbase + tok * a.qts + (r - tok * a.G) * a.qhs + ch * 16);
          }
          cp_async_wait_all();
        } else {
          constexpr int U = 8;
          for (int r0 = (qw * RPW) + lane / CPR; r0 < it.t.rows + (int)(lane / CPR); r0 += U * step) {
            uint4 w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int r = r0 + u * step;
              w[u] = make_uint4(0u, 0u, 0u, 0u);
              if (r < it.t.rows) {
                const int tok = r / a.G;
                w[u] = ld_stream(qbase + tok * a.qts + (r - tok * a.G) * a.qhs + ch * 16);
              }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int r = r0 + u * step;
              // the row in f16, its largest element scaled by a power of two to 2^14 .. 2^15
              // (the others keep their bits down to 2^-28 of it)
              uint32_t* q4 = reinterpret_cast<uint32_t*>(&w[u]);
              float mx = 0.0f;
#pragma unroll
              for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(fabsf(unpack_lo<DT>(q4[i])), fabsf(unpack_hi<DT>(q4[i]))));
#pragma unroll
              for (int o = 1; o < CPR; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
              int e = (int)(__float_as_uint(mx) >> 23);  // 2^(e - 127) <= max
              e = e == 255 ? 127 : max(e - 14, 1);       // infinities: as they are
              const float inv = 1.0f / __uint_as_float((uint32_t)e << 23);
#pragma unroll
              for (int i = 0; i < 4; ++i) q4[i] = pack2<RMLX_F16>(unpack_lo<DT>(q4[i]) * inv, unpack_hi<DT>(q4[i]) * inv);
              if (ch == 0 && r < CH_ROWS) qscale[(nitem & 1) * CH_ROWS + r] = (uint8_t)e;
              if (r < it.t.rows) sts128(sb + S::Q + (r >> 7) * S::QTILE + q_off<HD>(r & 127, ch), w[u]);
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(BAR_QFULL));
      }
      ++nitem;
      if (!loads_kv) continue;
      const int lead = two ? 1 : min(2, nk);
      // loads in the order of their use: K 0 .. lead - 1, then V j and K j + lead
      const int loads = 2 * nk;
      auto which = [&](int i, int& j, int& kv) {
        if (i < lead) j = i, kv = 0;
        else if (i - lead >= 2 * (nk - lead)) j = i - nk, kv = 1;  // the last ones are all V
        else j = (i - lead) >> 1, kv = ((i - lead) & 1) ^ 1, j += kv ? 0 : lead;
      };
      if constexpr (TMA) {
        for (int i = 0; i < loads; ++i) {
          int j, kv;
          which(i, j, kv);
          const uint32_t stage = n % ST, dst = sb + S::KV + stage * S::STAGE;
          if (!(ok = mbar_wait(bar(BAR_EMPTY + stage), ((n / ST) & 1) ^ 1, abort_flag, a.wait_ns, err))) break;
          ++n;
          // one box of p.box rows a lane
          const int kb = (it.t.k_lo + it.k0 + j) * CH_KEYS, at = kb + lane * p.box;
          const bool want = lane * p.box < CH_KEYS && at < it.t.hi;
          // boxes below the window hold the first visible one in their place: their blocks may be gone
          const int t = max(at, it.t.lo & -p.box);
          int blk = 0, b = 0;
          if (want) {
            b = t / g.bs;
            blk = __ldg(btrow + b);
            if (blk < 0 || blk >= g.nblocks) {
              atomicOr(err, DEV_ERR_BLOCK);
              blk = 0;
            }
          }
          const int boxes = __popc(__ballot_sync(0xffffffffu, want));
          if (lane == 0) mbar_arrive_expect_tx(bar(BAR_FULL + stage), boxes * p.box * HD * 2);
          __syncwarp();
          if (want)
            tma_load_4d(dst + lane * p.box * (HD * 2), &map, 0, 0, 0,
                        (int)((((int64_t)blk * g.layers + a.layer) * 2 + kv) * g.heads + it.head) * (g.bs / 8) +
                            (t - b * g.bs) / 8,
                        bar(BAR_FULL + stage));
        }
      } else if (raw) {
        // Codes of a tile, then its (scale, zero) rows, as they lie in the blocks:
        // warp 9 copies both a block's run at a time, the others convert them.
        constexpr int EPU = BITS ? 128 / (BITS ? BITS : 1) : 8, UPR = HD / EPU, UNITS = CH_KEYS * UPR, W = 6;
        constexpr int N = (UNITS + 32 * W - 1) / (32 * W);
        constexpr int RB = HD * BITS / 8;
        const int mb = g.meta_row_bytes, depth = p.raw_depth;
        const uint32_t raw_tile = CH_KEYS * (RB + mb);
        const int64_t block_bytes = (int64_t)g.layers * 2 * g.heads * g.tile_bytes;
        const uint8_t* head_base = g.base + g.tile_off(0, a.layer, 0, it.head);
        for (int i = 0; i < loads; ++i) {
          int j, kv;
          which(i, j, kv);
          const uint32_t slot = n % depth, phase = (n / depth) & 1, dst = sb + S::RAW + slot * raw_tile;
          const int kb = (it.t.k_lo + it.k0 + j) * CH_KEYS;
          if (warp == 9) {
            if (!(ok = mbar_wait(bar(BAR_RAWE + slot), phase ^ 1, abort_flag, a.wait_ns, err))) break;
            const int at = kb + lane * p.box;
            const bool want = lane * p.box < CH_KEYS && at < it.t.hi;
            const int t = max(at, it.t.lo & -p.box);  // as in the TMA loads
            int blk = 0, r = 0;
            if (want) {
              const int b = t / g.bs;
              r = t - b * g.bs;
              blk = __ldg(btrow + b);
              if (blk < 0 || blk >= g.nblocks) {
                atomicOr(err, DEV_ERR_BLOCK);
                blk = 0;
              }
            }
            const int boxes = __popc(__ballot_sync(0xffffffffu, want));
            if (lane == 0) mbar_arrive_expect_tx(bar(BAR_RAWF + slot), boxes * p.box * (RB + mb));
            __syncwarp();
            if (want) {
              const uint8_t* tile = head_base + blk * block_bytes + (kv ? (int64_t)g.heads * g.tile_bytes : 0);
              bulk_load(dst + lane * p.box * RB, tile + r * RB, p.box * RB, bar(BAR_RAWF + slot));
              bulk_load(dst + CH_KEYS * RB + lane * p.box * mb, tile + g.bs * RB + r * mb, p.box * mb, bar(BAR_RAWF + slot));
            }
          } else {
            if (!(ok = mbar_wait(bar(BAR_RAWF + slot), phase, abort_flag, a.wait_ns, err))) break;
            const bool both = SPLIT && kv == 0;
            if (!SPLIT) ns = n;
            const uint32_t stage = ns % ST, rest = (ns + 1) % ST;
            const uint32_t out = sb + S::KV + stage * S::STAGE, out2 = sb + S::KV + rest * S::STAGE;
            if (!(ok = mbar_wait(bar(BAR_EMPTY + stage), ((ns / ST) & 1) ^ 1, abort_flag, a.wait_ns, err))) break;
            if (both && !(ok = mbar_wait(bar(BAR_EMPTY + rest), (((ns + 1) / ST) & 1) ^ 1, abort_flag, a.wait_ns, err))) break;
            ns += both ? 2 : 1;
            const int ch = lane % UPR;
            auto convert = [&](auto mf32, auto one) {  // f32 scales and zeros; a unit's elements are all of one group
              constexpr bool MF32 = decltype(mf32)::value;
              // every unit's loads first, so that the conversions overlap
              auto unit = [&](int y) { return (y * W + qw) * 32 + lane; };
              auto there = [&](int y) { return (y + 1) * W * 32 <= UNITS || unit(y) < UNITS; };
              auto pair = [&](int y, int e) {
                const uint32_t meta = dst + CH_KEYS * RB + unit(y) / UPR * mb;
                const int q = (ch * EPU + e) >> a.gs_log2;
                return MF32 ? lds64(meta + q * 8) : make_uint2(lds32(meta + q * 4), 0u);
              };
              uint4 ws[N];
              uint2 sz[N];
              bool small = false;
#pragma unroll
              for (int y = 0; y < N; ++y)
                if (there(y)) ws[y] = lds128(dst + unit(y) * 16), sz[y] = pair(y, 0);
#pragma unroll
              for (int y = 0; y < N; ++y) {
                if (!there(y)) continue;
                const int row = unit(y) / UPR;
                const bool live = kb + row < it.t.hi;  // else zeros: behind the last visible row
                const uint32_t cw[4] = {ws[y].x, ws[y].y, ws[y].z, ws[y].w};
                Group<BITS ? BITS : 8> grp;
                small |= grp.set(live ? sz[y] : make_uint2(0u, 0u), MF32);
                uint4 o[EPU / 8];
#pragma unroll
                for (int e = 0; e < EPU / 8; ++e) {
                  if (!decltype(one)::value && e > 0) small |= grp.set(live ? pair(y, 8 * e) : make_uint2(0u, 0u), MF32);
                  const uint2 codes = BITS == 4 ? nibbles(cw[e & 3]) : make_uint2(cw[2 * (e & 1)], cw[2 * (e & 1) + 1]);
                  o[e] = dequant8<BITS ? BITS : 8, MF32>(codes, grp);
                  if (both) sts128(out2 + kv_off<HD>(row, ch * (EPU / 8) + e), dequant8_rest<BITS ? BITS : 8, MF32>(codes, grp, o[e]));
                }
#pragma unroll
                for (int e = 0; e < EPU / 8; ++e) sts128(out + kv_off<HD>(row, ch * (EPU / 8) + e), o[e]);
              }
              if (MF32 && small) tiny[8 * kv + ((nitem - 1) & 7)] = nitem;
            };
            const bool one = (1 << a.gs_log2) >= EPU;
            if (!a.mf32 && one) convert(std::false_type(), std::true_type());
            else if (!a.mf32) convert(std::false_type(), std::false_type());
            else if (one) convert(std::true_type(), std::true_type());
            else convert(std::true_type(), std::false_type());
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(bar(BAR_FULL + stage));
              if (both) mbar_arrive(bar(BAR_FULL + rest));
              mbar_arrive(bar(BAR_RAWE + slot));
            }
          }
          ++n;
        }
      } else {
        // A unit is 16 bytes of a stored row: 8 elements, or 16 or 32 codes.  Rows
        // go straight into their stage; codes, with the scale and zero of a unit's
        // first group, into a ring of their own, from which the thread that
        // copied them converts them `depth` - 1 loads later (with registers
        // instead of the ring one tile was in flight: 4-bit chunks 290 us).
        constexpr int EPU = BITS ? 128 / (BITS ? BITS : 1) : 8, UPR = HD / EPU, UNITS = CH_KEYS * UPR;
        constexpr int N = (UNITS + 32 * 7 - 1) / (32 * 7);
        const int depth = BITS == 0 ? 3 : S::FOURTH ? 2 : BITS == 4 ? 4 : a.mf32 ? 2 : 3;
        const int ch = lane % UPR;  // the same for all of a lane's units
        const int64_t block_bytes = (int64_t)g.layers * 2 * g.heads * g.tile_bytes;
        const uint8_t* head_base = g.base + g.tile_off(0, a.layer, 0, it.head);
        const int u0 = qw * 32 + lane;
        const uint32_t raw_meta = sb + S::RAW + depth * UNITS * 16;
        auto key_of = [&](int j, int y) { return (it.t.k_lo + it.k0 + j) * CH_KEYS + (u0 + y * 7 * 32) / UPR; };
        auto seen = [&](int key) { return key >= it.t.lo && key < it.t.hi; };  // the others are zeros
        // block ids (-1: no row) and rows in them of a load's units, a load ahead of the units themselves
        auto fetch_ids = [&](int i, int32_t (&blk)[N], int32_t (&row)[N]) {
          int j, kv;
          which(i, j, kv);
          int b[N];
          if (a.bs_log2 >= 0) {
#pragma unroll
            for (int y = 0; y < N; ++y) b[y] = key_of(j, y) >> a.bs_log2, row[y] = key_of(j, y) & (g.bs - 1);
          } else {
#pragma unroll
            for (int y = 0; y < N; ++y) b[y] = key_of(j, y) / g.bs, row[y] = key_of(j, y) - b[y] * g.bs;
          }
#pragma unroll
          for (int y = 0; y < N; ++y) {
            blk[y] = -1;
            if (u0 + y * 7 * 32 < UNITS && seen(key_of(j, y))) blk[y] = __ldg(btrow + b[y]);
          }
        };
        // straight-line, so that the units' address arithmetic overlaps
        bool bad = false;
        auto copy = [&](int i, const int32_t (&blk)[N], const int32_t (&row)[N], uint32_t stage, int slot) {
          int j, kv;
          which(i, j, kv);
          const uint8_t* base = head_base + (kv ? (int64_t)g.heads * g.tile_bytes : 0);
#pragma unroll
          for (int y = 0; y < N; ++y) {
            const int u = u0 + y * 7 * 32;
            const bool unit = u < UNITS, want = unit && seen(key_of(j, y));
            const bool good = want && (uint32_t)blk[y] < (uint32_t)g.nblocks;  // else zeros
            bad |= want && !good;
            const uint8_t* tile = base + (good ? blk[y] : 0) * block_bytes;
            if (BITS == 0) {
              cp_async16_zfill(sb + S::KV + stage * S::STAGE + kv_off<HD>(u / UPR, ch), tile + row[y] * g.row_bytes + ch * 16, unit, good);
            } else {
              cp_async16_zfill(sb + S::RAW + (slot * UNITS + u) * 16, tile + row[y] * g.row_bytes + ch * 16, unit, good);
              const uint8_t* meta = tile + g.bs * g.row_bytes + row[y] * g.meta_row_bytes;
              const int q = (ch * EPU) >> a.gs_log2;
              if (a.mf32) cp_async_zfill<8>(raw_meta + (slot * UNITS + u) * 8, meta + q * 8, unit, good);
              else cp_async_zfill<4>(raw_meta + (slot * UNITS + u) * 4, meta + q * 4, unit, good);
            }
          }
        };
        // mf32: f32 scales and zeros; one: a unit's elements are all of one group
        auto convert_as = [&](int i, uint32_t stage, uint32_t rest, int slot, auto mf32, auto one) {
          constexpr bool MF32 = decltype(mf32)::value;
          int j, kv;
          which(i, j, kv);
          bool small = false;
#pragma unroll
          for (int y = 0; y < N; ++y) {
            const int u = u0 + y * 7 * 32;
            if (u >= UNITS) continue;
            const uint4 w = lds128(sb + S::RAW + (slot * UNITS + u) * 16);
            const uint32_t cw[4] = {w.x, w.y, w.z, w.w};
            Group<BITS ? BITS : 8> grp;
            small |= grp.set(MF32 ? lds64(raw_meta + (slot * UNITS + u) * 8) : make_uint2(lds32(raw_meta + (slot * UNITS + u) * 4), 0u),
                             MF32);
            const uint8_t* meta = nullptr;
            if (!decltype(one)::value) {
              const int t = key_of(j, y);
              const int b = a.bs_log2 >= 0 ? t >> a.bs_log2 : t / g.bs;
              const int32_t blk = seen(t) ? __ldg(btrow + b) : -1;
              if (blk >= 0 && blk < g.nblocks)
                meta = head_base + (kv ? (int64_t)g.heads * g.tile_bytes : 0) + blk * block_bytes + g.bs * g.row_bytes +
                       (t - b * g.bs) * g.meta_row_bytes;
            }
            uint4 o[EPU / 8];
#pragma unroll
            for (int e = 0; e < EPU / 8; ++e) {
              if (!decltype(one)::value && e > 0 && meta)
                small |= grp.set(load_meta(meta, (ch * EPU + 8 * e) >> a.gs_log2, MF32), MF32);
              const uint2 codes = BITS == 4 ? nibbles(cw[e & 3]) : make_uint2(cw[2 * (e & 1)], cw[2 * (e & 1) + 1]);
              o[e] = dequant8<BITS ? BITS : 8, MF32>(codes, grp);
              if (SPLIT && kv == 0)
                sts128(sb + S::KV + rest * S::STAGE + kv_off<HD>(u / UPR, ch * (EPU / 8) + e), dequant8_rest<BITS ? BITS : 8, MF32>(codes, grp, o[e]));
            }
#pragma unroll
            for (int e = 0; e < EPU / 8; ++e)
              sts128(sb + S::KV + stage * S::STAGE + kv_off<HD>(u / UPR, ch * (EPU / 8) + e), o[e]);
          }
          if (MF32 && small) tiny[8 * kv + ((nitem - 1) & 7)] = nitem;
        };
        auto convert = [&](int i, uint32_t stage, uint32_t rest, int slot) {
          const bool one = (1 << a.gs_log2) >= EPU;
          if (!a.mf32 && one) convert_as(i, stage, rest, slot, std::false_type(), std::true_type());
          else if (!a.mf32) convert_as(i, stage, rest, slot, std::false_type(), std::false_type());
          else if (one) convert_as(i, stage, rest, slot, std::true_type(), std::true_type());
          else convert_as(i, stage, rest, slot, std::true_type(), std::false_type());
        };
        auto empty = [&](uint32_t i) { return ok = mbar_wait(bar(BAR_EMPTY + i % ST), ((i / ST) & 1) ^ 1, abort_flag, a.wait_ns, err); };
        int32_t ids[N], rows[N];
        fetch_ids(0, ids, rows);
        int in = 0, out = 0;  // ring slots of the next copy and the next conversion
        for (int i = 0; i < loads + depth - 1; ++i) {
          if (i < loads) {
            if (BITS == 0 && !empty(n + i)) break;
            copy(i, ids, rows, (n + i) % ST, in);
            if (++in == depth) in = 0;
            if (i + 1 < loads) fetch_ids(i + 1, ids, rows);
          }
          cp_async_commit();
          const int d = i - (depth - 1);
          if (d < 0) continue;
          if (depth == 2) cp_async_wait<1>();
          else if (depth == 3) cp_async_wait<2>();
          else cp_async_wait<3>();
          if constexpr (BITS != 0) {
            int j, kv;
            which(d, j, kv);
            const bool both = SPLIT && kv == 0;
            if (!SPLIT) ns = n + d;
            if (!empty(ns) || (both && !empty(ns + 1))) break;
            convert(d, ns % ST, (ns + 1) % ST, out);
            if (++out == depth) out = 0;
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(bar(BAR_FULL + ns % ST));
              if (both) mbar_arrive(bar(BAR_FULL + (ns + 1) % ST));
            }
            ns += both ? 2 : 1;
          } else {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(BAR_FULL + (n + d) % ST));
          }
        }
        n += loads;
        if (bad) atomicOr(err, DEV_ERR_BLOCK);
      }
      if (!ok) break;
    }
    if (issues) copies = n;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // A wait ran out, in whichever role: the others' MMAs and copies may still be in
    // flight, and nothing may be when the CTA ends.
    if (warp == 8) {
      tc_commit(bar(BAR_DRAIN));
      for (int i = 0; i < 2000 && !mbar_try(bar(BAR_DRAIN), 0); ++i) {
      }
    } else if (warp == 9) {
      const uint32_t slots = raw ? p.raw_depth : ST;
      for (uint32_t i = copies > slots ? copies - slots : 0; i < copies; ++i)
        for (int k = 0; k < 2000 && !mbar_try(bar((raw ? BAR_RAWF : BAR_FULL) + i % slots), (i / slots) & 1); ++k) {
        }
    }
    cp_async_wait_all();
    if (threadIdx.x < 2) desc[threadIdx.x].valid = desc[threadIdx.x].last = 0;  // no part to join
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 8) tmem_free(tmem, 512);
}

// Joins the portions of the items that more than one CTA worked on.  Block
// (c, y): rows 32 y .. of the item that CTA c began and others went on with, a
// lane a row, a warp 1 / 8 of the columns.  Part by part, each waiting for the
// last, an item of 30 parts took 87 us.
template <int DT, int HD>
__global__ void __launch_bounds__(256) chunk_combine_kernel(ChunkParams p, int nparts) {
  constexpr int COLS = HD / 8;
  pdl_release();
  pdl_wait();
  const PartDesc d = p.desc[2 * blockIdx.x + 1];
  const int lane = threadIdx.x & 31, col = (threadIdx.x >> 5) * COLS, row = blockIdx.y * 32 + lane;
  if (!d.valid || (int)blockIdx.y * 32 >= d.rows) return;
  int n = 0;  // parts: this CTA's, and those of the next CTAs up to the item's last
  for (int c0 = blockIdx.x + 1; c0 < nparts && !n; c0 += 32) {
    const unsigned last = __ballot_sync(0xffffffffu, c0 + lane < nparts && p.desc[2 * (c0 + lane)].last);
    if (last) n = c0 - blockIdx.x + __ffs(last);
  }
  if (n == 0) return;  // its last part's CTA gave up
  const float* first = p.parts + (size_t)(2 * blockIdx.x + 1) * part_floats(HD);  // a CTA's slot 1; the others' slot 0
  auto part = [&](int i) { return i == 0 ? first : first + (size_t)(2 * i - 1) * part_floats(HD); };
  auto max_sum = [&](int i) {
    return i < n ? __ldcg(reinterpret_cast<const float2*>(part(i) + (size_t)CH_ROWS * HD) + row) : make_float2(-INFINITY, 0.0f);
  };
  // every pass has the loads of several parts in flight: an item may have as many parts as there are SMs
  float m = -INFINITY, l = 0.0f, acc[COLS];
  for (int i = 0; i < n; i += 8) {
    float2 x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = max_sum(i + k);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, x[k].x);
  }
  const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int e = 0; e < COLS; ++e) acc[e] = 0.0f;
  for (int i = 0; i < n; i += 4) {
    float o[4][COLS];
    float2 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = max_sum(i + k);
#pragma unroll
      for (int e = 0; e < COLS; ++e) o[k][e] = i + k < n ? __ldcg(part(i + k) + (size_t)(col + e) * CH_ROWS + row) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = ex2(x[k].x - base);
      l = fmaf(x[k].y, f, l);
#pragma unroll
      for (int e = 0; e < COLS; ++e) acc[e] = fmaf(o[k][e], f, acc[e]);
    }
  }
  if (row >= d.rows) return;
  const float il = l == 0.0f ? 0.0f : 1.0f / l;
  const int tok = row / p.a.G, gq = row - tok * p.a.G;
  uint4* o = reinterpret_cast<uint4*>(
      p.a.out + ((((int64_t)(d.token0 + tok) * p.g.heads + d.head) * p.a.G + gq) * HD + col) * 2);
#pragma unroll
  for (int e = 0; e < COLS / 8; ++e)
    o[e] = make_uint4(pack2<DT>(acc[8 * e] * il, acc[8 * e + 1] * il), pack2<DT>(acc[8 * e + 2] * il, acc[8 * e + 3] * il),
                      pack2<DT>(acc[8 * e + 4] * il, acc[8 * e + 5] * il), pack2<DT>(acc[8 * e + 6] * il, acc[8 * e + 7] * il));
}

}  // namespace rmlx

using namespace rmlx;

namespace {

using ChunkFn = void (*)(ChunkParams, CUtensorMap, int32_t*);
using ChunkCombineFn = void (*)(ChunkParams, int);
template <int DT, int HD>
ChunkFn pick_chunk(int bits, bool tma) {
  if (bits == 8) return chunk_attn_kernel<DT, HD, 8, false>;
  if (bits == 4) return chunk_attn_kernel<DT, HD, 4, false>;
  return tma ? chunk_attn_kernel<DT, HD, 0, true> : chunk_attn_kernel<DT, HD, 0, false>;
}

// Shared memory of a launch, and what of it holds codes in flight.
struct ChunkBytes {
  size_t smem;
  int raw;
};
template <int HD, bool F16>
ChunkBytes chunk_bytes(int bits) {
  using S8 = ChunkSmem<HD, 8, F16>;
  using S4 = ChunkSmem<HD, 4, F16>;
  if (bits == 8) return {S8::BYTES, S8::RAW_BYTES};
  if (bits == 4) return {S4::BYTES, S4::RAW_BYTES};
  return {ChunkSmem<HD, 0, false>::BYTES, 0};
}

size_t chunk_workspace(const rmlx_kv_pool* p) {
  return (size_t)p->num_sms * 2 * (part_floats(p->cfg.head_dim) * sizeof(float) + sizeof(PartDesc));
}

// The pool as TMA sees it: [group of 8 rows][64-column half][row][64 elements],
// loaded a box of `box` rows at a time into 128-byte-swizzled shared memory.
// Every coordinate but the group's is 0, so a box starts on a 16-byte boundary.
rmlx_status chunk_map(rmlx_kv_pool* p, int box, CUtensorMap* map) {
  using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  if (!encode) return fail(RMLX_E_CUDA, "the driver has no cuTensorMapEncodeTiled");
  // a driver call needs the device's context bound to this thread, which may have made no CUDA call before
  const rmlx_status s = cuda_check(cudaSetDevice(p->device), "cudaSetDevice");
  if (s != RMLX_OK) return s;
  const rmlx_pool_config& c = p->cfg;
  const cuuint64_t hd = c.head_dim;
  const cuuint64_t dims[4] = {64, 8, hd / 64, (cuuint64_t)c.num_blocks * c.num_layers * 2 * c.num_kv_heads * (c.block_size / 8)};
  const cuuint64_t strides[3] = {hd * 2, 128, hd * 16};
  const cuuint32_t boxes[4] = {64, 8, (cuuint32_t)hd / 64, (cuuint32_t)box / 8}, ones[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, c.dtype == RMLX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            4, p->base, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(RMLX_E_CUDA, "cuTensorMapEncodeTiled: error %d", (int)r);
  return RMLX_OK;
}

}  // namespace

extern "C" {

rmlx_status rmlx_kv_chunk_attention_workspace_size(const rmlx_kv_pool* p, int32_t q_heads_per_kv, size_t* bytes) {
  if (!p || !bytes) return fail(RMLX_E_BAD_ARG, "NULL pool or bytes");
  if (q_heads_per_kv < 1 || q_heads_per_kv > 16) return fail(RMLX_E_BAD_ARG, "q_heads_per_kv must be in [1, 16]");
  const int hd = p->cfg.head_dim;
  *bytes = hd == 64 || hd == 128 ? chunk_workspace(p) : 0;
  return RMLX_OK;
}

rmlx_status rmlx_kv_chunk_attention(rmlx_kv_pool* p, int32_t layer, const void* q, int64_t q_token_stride,
                                    int64_t q_head_stride, int32_t q_heads_per_kv, const int32_t* block_tables,
                                    int32_t block_table_stride, const int32_t* q_lens, const int32_t* seq_lens,
                                    int32_t num_seqs, int32_t num_q_tokens, float softmax_scale, int32_t window,
                                    void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (!p) return fail(RMLX_E_BAD_ARG, "NULL pool");
  const rmlx_pool_config& c = p->cfg;
  if (c.dtype != RMLX_F16 && c.dtype != RMLX_BF16) return fail(RMLX_E_BAD_ARG, "chunk attention needs an F16 or BF16 pool");
  if (c.head_dim != 64 && c.head_dim != 128) return fail(RMLX_E_BAD_ARG, "chunk attention supports head_dim 64 or 128");
  if (q_heads_per_kv < 1 || q_heads_per_kv > 16) return fail(RMLX_E_BAD_ARG, "q_heads_per_kv must be in [1, 16]");
  if (layer < 0 || layer >= c.num_layers) return fail(RMLX_E_RANGE, "layer %d out of range", layer);
  if (num_seqs < 0 || num_seqs > RMLX_MAX_SEQS_PER_LAUNCH) return fail(RMLX_E_BAD_ARG, "num_seqs out of range");
  if (num_q_tokens < 0) return fail(RMLX_E_BAD_ARG, "num_q_tokens < 0");
  if (window < 0) return fail(RMLX_E_BAD_ARG, "window < 0");
  if (num_seqs == 0 || num_q_tokens == 0) return RMLX_OK;
  if (!q || !out || !block_tables || !q_lens || !seq_lens || !workspace) return fail(RMLX_E_BAD_ARG, "NULL argument");
  const int64_t qts = q_token_stride * 2, qhs = q_head_stride * 2;
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || (qts % 16) || (qhs % 16))
    return fail(RMLX_E_BAD_ARG, "q, out, workspace and the strides of q must be 16-byte aligned");
  if (block_table_stride < 1) return fail(RMLX_E_BAD_ARG, "block_table_stride must be at least 1");
  if (!(softmax_scale > 0.0f) || softmax_scale > 1e30f) return fail(RMLX_E_BAD_ARG, "softmax_scale must be positive");
  size_t need = 0;
  rmlx_status s = rmlx_kv_chunk_attention_workspace_size(p, q_heads_per_kv, &need);
  if (s != RMLX_OK) return s;
  if (workspace_bytes < need) return fail(RMLX_E_BAD_ARG, "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  ChunkArgs a;
  a.q = (const uint8_t*)q, a.out = (uint8_t*)out;
  a.bt = block_tables, a.q_lens = q_lens, a.seq_lens = seq_lens;
  a.qts = qts, a.qhs = qhs;
  a.layer = layer, a.G = q_heads_per_kv, a.bt_stride = block_table_stride, a.nseq = num_seqs, a.nq = num_q_tokens;
  a.window = window;
  a.bs_log2 = is_pow2(c.block_size) ? log2i(c.block_size) : -1;
  a.max_len = (int)std::min<int64_t>((int64_t)block_table_stride * c.block_size, 1 << 30);
  a.gs_log2 = c.quant_bits ? log2i(c.group_size) : 0, a.bits = c.quant_bits, a.mf32 = c.meta_dtype == RMLX_F32;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;  // log2(e)
  a.wait_ns = p->wait_ns;
  DeviceGuard dg(p->device);
  const bool bf = c.dtype == RMLX_BF16;
  ChunkParams prm;
  prm.g = p->geo();
  prm.a = a;
  prm.tpt = CH_ROWS / q_heads_per_kv;
  // TMA reads whole groups of 8 stored rows; a box is the most rows that both a block and a key tile hold a whole number of
  prm.box = std::gcd(c.block_size, CH_KEYS);
  const bool tma = !c.quant_bits && c.block_size % 8 == 0;
  const ChunkBytes bytes = c.head_dim == 128 ? (bf ? chunk_bytes<128, false>(c.quant_bits) : chunk_bytes<128, true>(c.quant_bits))
                                             : (bf ? chunk_bytes<64, false>(c.quant_bits) : chunk_bytes<64, true>(c.quant_bits));
  // codes and their (scale, zero) rows by bulk copies where a box of either is whole 16-byte pieces (and 32 lanes issue a tile's)
  prm.raw_depth = 0;
  if (c.quant_bits && prm.box >= 4 && prm.box * p->meta_row_bytes % 16 == 0) {
    const int depth = std::min<int>(CH_RAW, bytes.raw / (CH_KEYS * (int)(p->row_bytes + p->meta_row_bytes)));
    if (depth >= 2) prm.raw_depth = depth;
  }
  prm.parts = static_cast<float*>(workspace);
  prm.desc = reinterpret_cast<PartDesc*>(prm.parts + (size_t)p->num_sms * 2 * part_floats(c.head_dim));
  static_assert(sizeof(CUtensorMap) == sizeof(p->chunk_map), "tensor map");
  if (!__atomic_load_n(&p->chunk_fn, __ATOMIC_ACQUIRE)) {  // the first calls of a pool, from one thread or several
    static std::mutex first;
    std::lock_guard<std::mutex> lock(first);
    if (!p->chunk_fn) {
      if (tma && (s = chunk_map(p, prm.box, reinterpret_cast<CUtensorMap*>(p->chunk_map))) != RMLX_OK) return s;
      ChunkFn fn = c.head_dim == 128 ? (bf ? pick_chunk<RMLX_BF16, 128>(c.quant_bits, tma) : pick_chunk<RMLX_F16, 128>(c.quant_bits, tma))
                                     : (bf ? pick_chunk<RMLX_BF16, 64>(c.quant_bits, tma) : pick_chunk<RMLX_F16, 64>(c.quant_bits, tma));
      if ((s = prepare_smem(fn, bytes.smem)) != RMLX_OK) return s;
      p->chunk_combine_fn = reinterpret_cast<void*>(
          c.head_dim == 128 ? (bf ? chunk_combine_kernel<RMLX_BF16, 128> : chunk_combine_kernel<RMLX_F16, 128>)
                            : (bf ? chunk_combine_kernel<RMLX_BF16, 64> : chunk_combine_kernel<RMLX_F16, 64>));
      __atomic_store_n(&p->chunk_fn, reinterpret_cast<void*>(fn), __ATOMIC_RELEASE);  // last: what it stands for is ready
    }
  }
  ChunkFn fn = reinterpret_cast<ChunkFn>(p->chunk_fn);
  ChunkCombineFn fc = reinterpret_cast<ChunkCombineFn>(p->chunk_combine_fn);
  cudaError_t e = launch_pdl(fn, dim3(p->num_sms), dim3(ch_threads(tma)), bytes.smem, (cudaStream_t)stream, prm,
                             *reinterpret_cast<const CUtensorMap*>(p->chunk_map), p->err);
  if (e != cudaSuccess) return cuda_check(e, "chunk attention launch");
  e = launch_pdl(fc, dim3(p->num_sms, CH_ROWS / 32), dim3(256), 0, (cudaStream_t)stream, prm, (int)p->num_sms);
  if (e != cudaSuccess) return cuda_check(e, "chunk attention combine launch");
  return cuda_check(cudaGetLastError(), "chunk attention launch");
}

}  // extern "C"

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
#include <algorithm>

#include "dequant.cuh"
#include "kv_pool_internal.cuh"

namespace rmlx {

struct ChunkArgs {
  const uint8_t* q;
  uint8_t* out;
  const int32_t *bt, *q_lens, *seq_lens;
  int64_t qts, qhs;  // byte strides of q: token, head
  int layer, G, bt_stride, nseq, nq, window;
  int gs_log2, bits, mf32;
  float scale_log2;
};

// This lane's head_dim / 32 elements of stored row `row` (K or V) of a tile,
// dequantised in f32 when the pool holds codes (not rounded to the pool's
// type: 8 bits of a bf16 value would cost more than the codes' own).
template <int DT, int HD>
__device__ __forceinline__ void load_row(const PoolGeo& g, const ChunkArgs& a, const uint8_t* tile, int row, int lane,
                                         float (&f)[HD / 32]) {
  constexpr int EPL = HD / 32;
  const int e0 = lane * EPL;
  if (a.bits == 0) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(tile + (int64_t)row * g.row_bytes) + e0;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      if (DT == RMLX_BF16) f[e] = __uint_as_float((uint32_t)__ldg(p + e) << 16);
      else f[e] = __half2float(__ushort_as_half(__ldg(p + e)));
    }
    return;
  }
  const uint8_t* codes = tile + (int64_t)row * g.row_bytes;
  const uint8_t* meta = tile + (int64_t)g.bs * g.row_bytes + (int64_t)row * g.meta_row_bytes;
  const int q = e0 >> a.gs_log2;
  float sc, zr;
  if (a.mf32) {
    sc = __ldg(reinterpret_cast<const float*>(meta) + 2 * q);
    zr = __ldg(reinterpret_cast<const float*>(meta) + 2 * q + 1);
  } else {
    sc = __half2float(__ushort_as_half(__ldg(reinterpret_cast<const uint16_t*>(meta) + 2 * q)));
    zr = __half2float(__ushort_as_half(__ldg(reinterpret_cast<const uint16_t*>(meta) + 2 * q + 1)));
  }
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    const int i = e0 + e;
    const int c = a.bits == 8 ? __ldg(codes + i) : (__ldg(codes + (i >> 1)) >> (4 * (i & 1))) & 15;
    f[e] = __fadd_rn(__fmul_rn((float)c, sc), zr);
  }
}

// One query row against keys [k0, k1) by one warp, a key at a time, with the
// running maximum m and sum l of a softmax in the log2 domain; acc is this
// lane's head_dim / 32 elements of the unnormalised output.  Rows that the
// mask hides are never read.
template <int DT, int HD>
__device__ __forceinline__ void attend_row(const PoolGeo& g, const ChunkArgs& a, const int32_t* btrow, int h, int k0,
                                           int k1, const float (&qf)[HD / 32], int lane, int32_t* err, float& m,
                                           float& l, float (&acc)[HD / 32]) {
  constexpr int EPL = HD / 32;
  constexpr unsigned FULL = 0xffffffffu;
  const int64_t vdelta = (int64_t)g.heads * g.tile_bytes;
  for (int j = k0; j < k1; ++j) {
    const int b = j / g.bs;
    const int32_t blk = b < a.bt_stride ? __ldg(btrow + b) : -1;
    if (blk < 0 || blk >= g.nblocks) {
      if (lane == 0) atomicOr(err, DEV_ERR_BLOCK);
      continue;
    }
    const uint8_t* tile = g.base + g.tile_off(blk, a.layer, 0, h);
    float kf[EPL], vf[EPL];
    load_row<DT, HD>(g, a, tile, j - b * g.bs, lane, kf);
    load_row<DT, HD>(g, a, tile + vdelta, j - b * g.bs, lane, vf);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) s = fmaf(qf[e], kf[e], s);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
    s *= a.scale_log2;
    const float n = fmaxf(m, s);
    const float base = n == -INFINITY ? 0.0f : n;  // a score of -inf before any other: exp2(-inf - 0) = 0
    const float f = exp2f(m - base), p = exp2f(s - base);
    m = n;
    l = fmaf(l, f, p);
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = fmaf(acc[e], f, p * vf[e]);
  }
}

// One warp per (token, query head).
template <int DT, int HD>
__global__ void __launch_bounds__(256) chunk_attn_rows_kernel(PoolGeo g, ChunkArgs a, int32_t* err) {
  constexpr int EPL = HD / 32;
  extern __shared__ int32_t smem[];
  int32_t* cub = smem;
  int32_t* cut = smem + a.nseq + 1;
  pdl_wait();
  pdl_release();
  scan_seq_lens(a.q_lens, a.nseq, 1, cub, cut);
  if (cut[a.nseq] > a.nq) {
    if (threadIdx.x == 0) atomicOr(err, DEV_ERR_Q_ROWS);
    return;
  }
  const int lane = threadIdx.x & 31, qheads = g.heads * a.G;
  const int64_t total = (int64_t)cut[a.nseq] * qheads;
  const int64_t nwarps = ((int64_t)gridDim.x * blockDim.x) >> 5;
  for (int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; w < total; w += nwarps) {
    const int t = (int)(w / qheads), hq = (int)(w - (int64_t)t * qheads);
    const int s = find_seq(cut, a.nseq, t);
    const int n = cut[s + 1] - cut[s], len = max(__ldg(a.seq_lens + s), 0);
    const int pos = len - n + (t - cut[s]);
    float qf[EPL], acc[EPL], m = -INFINITY, l = 0.0f;
    const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q + t * a.qts + hq * a.qhs) + lane * EPL;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      qf[e] = DT == RMLX_BF16 ? __uint_as_float((uint32_t)__ldg(qp + e) << 16) : __half2float(__ushort_as_half(__ldg(qp + e)));
      acc[e] = 0.0f;
    }
    const int k0 = a.window && pos >= a.window ? pos - a.window + 1 : 0;
    attend_row<DT, HD>(g, a, a.bt + (int64_t)s * a.bt_stride, hq / a.G, k0, pos + 1, qf, lane, err, m, l, acc);
    const float il = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* o = reinterpret_cast<uint16_t*>(a.out) + ((int64_t)t * qheads + hq) * HD + lane * EPL;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const float x = acc[e] * il;
      o[e] = DT == RMLX_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
    }
  }
}

}  // namespace rmlx

using namespace rmlx;

extern "C" {

rmlx_status rmlx_kv_chunk_attention_workspace_size(const rmlx_kv_pool* p, int32_t q_heads_per_kv, size_t* bytes) {
  if (!p || !bytes) return fail(RMLX_E_BAD_ARG, "NULL pool or bytes");
  if (q_heads_per_kv < 1 || q_heads_per_kv > 16) return fail(RMLX_E_BAD_ARG, "q_heads_per_kv must be in [1, 16]");
  *bytes = 16;
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
  a.gs_log2 = c.quant_bits ? log2i(c.group_size) : 0, a.bits = c.quant_bits, a.mf32 = c.meta_dtype == RMLX_F32;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;  // log2(e)
  DeviceGuard dg(p->device);
  const bool bf = c.dtype == RMLX_BF16;
  auto fn = c.head_dim == 128 ? (bf ? chunk_attn_rows_kernel<RMLX_BF16, 128> : chunk_attn_rows_kernel<RMLX_F16, 128>)
                              : (bf ? chunk_attn_rows_kernel<RMLX_BF16, 64> : chunk_attn_rows_kernel<RMLX_F16, 64>);
  const size_t smem = (size_t)(num_seqs + 1) * 2 * sizeof(int32_t);
  if ((s = prepare_smem(fn, smem)) != RMLX_OK) return s;
  const int64_t rows = (int64_t)num_q_tokens * c.num_kv_heads * q_heads_per_kv;
  const int grid = (int)std::min<int64_t>((rows + 7) / 8, persistent_grid(fn, 256, smem, p->num_sms));
  cudaError_t e = launch_pdl(fn, dim3(grid), dim3(256), smem, (cudaStream_t)stream, p->geo(), a, p->err);
  if (e != cudaSuccess) return cuda_check(e, "chunk attention launch");
  return cuda_check(cudaGetLastError(), "chunk attention launch");
}

}  // extern "C"

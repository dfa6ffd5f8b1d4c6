"""Attention of a chunk of new tokens over the paged pool (rmlx_kv_chunk_attention).

The reference is softmax(scale q K^T) V in float64 over the pool's rows.  Error of an element, with A = sum_j p_j |v_j| (p the softmax):
  * each weight is rounded to the pool's type before P V: half a step, eps / 2;
  * the output is rounded to the pool's type: eps / 2 of |out| <= A;
  * scores are f32 sums of exact products of 16-bit values: below
    D 2^-24 sum |q_d k_d| scale, 7e-5 for these inputs; the exponential and the
    sum of weights add a few 2^-22: together below 2e-4 of A
so |error| <= (eps + 2e-4) A, plus half a step among the subnormals of f16.

A quantised pool's rows are code * scale + zero in float64 from the pool's
bytes.  Its products may run in f16 whatever the pool's type: weights, V and K
each rounded by half a step of f16 (2^-11), a rounded K moving a score by at
most delta = 2^-11 scale sum |q_d k_d| and so a weight, and the sum of weights,
by a factor of exp(delta) each: |error| <= (eps / 2 + 2 * 2^-11 + 2 delta + 2e-4) A.
"""
import numpy as np
import pytest
import torch

import rmlx_kv
import oracle as orc
from test_gpu_append_rope import TORCH, pool_bytes, pool_rows

pytestmark = pytest.mark.gpu


def reference(k, v, q, n, window, scale):
    """k, v [H, L, D] and q [n, H, G, D] in float64 -> out and A, both [n, H, G, D]."""
    L = k.shape[1]
    pos = torch.arange(L - n, L, device=q.device)[:, None]
    key = torch.arange(L, device=q.device)[None]
    seen = key <= pos
    if window:
        seen &= key > pos - window
    s = torch.einsum("nhgd,hld->hgnl", q, k) * scale
    s = s.masked_fill(~seen, -np.inf)
    p = torch.softmax(s, -1)
    p = torch.where(seen.any(-1)[:, None], p, torch.zeros_like(p))  # a token with no key
    p = torch.where(seen, p, torch.zeros_like(p))
    v = torch.where((pos.max() >= key[0])[:, None], v, torch.zeros_like(v))
    reach = torch.einsum("nhgd,hld->hgnl", q.abs(), k.abs()).amax(-1).permute(2, 0, 1)[..., None] * scale
    return torch.einsum("hgnl,hld->nhgd", p, v), torch.einsum("hgnl,hld->nhgd", p, v.abs()), reach


def stored_rows(pool, layer, dt):
    """The layer's rows in float64, [block][K, V][head][slot][dim], codes dequantised without rounding."""
    c = pool.cfg
    b = pool_bytes(pool).view(c.num_blocks, c.num_layers, 2, c.num_kv_heads, -1)[:, layer]
    bs, D, bits = c.block_size, c.head_dim, c.quant_bits
    if not bits:
        return b.contiguous().view(TORCH[dt]).unflatten(-1, (bs, D)).double()
    row, ng = D * bits // 8, D // c.group_size
    codes = b[..., :bs * row].unflatten(-1, (bs, row))
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    kind = torch.float32 if c.meta_dtype == orc.F32 else torch.float16
    meta = b[..., bs * row:bs * row + bs * pool.layout.meta_row_bytes].contiguous().view(kind).double()
    meta = meta.unflatten(-1, (bs, ng, 2))
    return (codes.double().unflatten(-1, (ng, -1)) * meta[..., :1] + meta[..., 1:]).flatten(-2)


def fill(pool, dt, bits, g):
    """N(0, 1) rows in every slot of every layer, through the append (which quantises)."""
    c = pool.cfg
    T = c.num_blocks * c.block_size
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    for layer in range(c.num_layers):
        k, v = (torch.randn(T, c.num_kv_heads, c.head_dim, generator=g, device="cuda").to(TORCH[dt]) for _ in range(2))
        pool.append(k, v, slots, T, layer_begin=layer, num_layers=1)


def tables(lens, bs, N, g, spare=0):
    need = [-(-max(int(n), 0) // bs) for n in lens]
    perm = torch.randperm(N, generator=g, device="cuda").to(torch.int32)
    bt = torch.zeros(len(lens), max(max(need), 1) + spare, dtype=torch.int32, device="cuda")
    o = 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[o:o + n]
        o += n
    assert o <= N
    return bt


def dev(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(pool, layer, q, G, bt, q_lens, lens, window, out, dt):
    """Every sequence's out rows against the reference over the stored rows."""
    c = pool.cfg
    H, D = c.num_kv_heads, c.head_dim
    rows = stored_rows(pool, layer, dt)
    eps = torch.finfo(TORCH[dt]).eps
    at = 0
    for s, (n, L) in enumerate(zip(q_lens, lens)):
        L = max(L, 0)
        got = out[at:at + n].double().view(n, H, G, D)
        if n and L == 0:
            assert (got == 0).all()
        elif n:
            kv = rows[bt[s, :-(-L // c.block_size)].long()]  # [block][K, V][head][slot][dim]
            k, v = (kv[:, i].transpose(0, 1).reshape(H, -1, D)[:, :L] for i in (0, 1))
            skip = max(n - L, 0)  # tokens before the sequence's first row see nothing
            assert (got[:skip] == 0).all()
            want, A, reach = reference(k, v, q[at + skip:at + n].double().view(n - skip, H, G, D), n - skip, window, D ** -0.5)
            err = (got[skip:] - want).abs()
            assert torch.isfinite(got).all()
            rel = eps / 2 + 2.0 ** -10 + 2.0 ** -10 * reach + 2e-4 if c.quant_bits else eps + 2e-4
            tol = rel * A + (2.0 ** -24 if dt == orc.F16 else 1e-38)
            assert (err <= tol).all(), (n, L, float((err / tol).max()))
        at += n


def run(H, G, D, bs, dt, q_lens, ctx, window=0, bits=0, gs=64, meta=orc.F16, layers=2, layer=1, seed=0, spare=1):
    g = torch.Generator("cuda").manual_seed(seed + 1000 * D + G)
    lens = [n + c for n, c in zip(q_lens, ctx)]
    N = sum(-(-max(n, 0) // bs) for n in lens) + 2
    pool = rmlx_kv.KVPool(layers, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=gs, meta_dtype=meta)
    fill(pool, dt, bits, g)
    bt = tables(lens, bs, N, g, spare)
    T = sum(q_lens)
    qkv = torch.randn(T + 3, H * G + 2 * H, D, generator=g, device="cuda").to(TORCH[dt])
    out = torch.full((T + 3, H * G, D), 9.0, dtype=TORCH[dt], device="cuda")
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
    pool.chunk_attention(layer, qkv, G, bt, bt.shape[1], dev(q_lens), dev(lens), len(lens), T + 3, D ** -0.5, out, ws,
                         window=window, q_token_stride=qkv.shape[1] * D)
    assert pool.check() == 0
    assert (out[T:] == 9.0).all()  # rows behind the last chunk
    check(pool, layer, qkv[:, :H * G], G, bt, q_lens, lens, window, out, dt)
    pool.close()


@pytest.mark.parametrize("dt", [orc.BF16, orc.F16])
@pytest.mark.parametrize("D", [64, 128])
def test_ragged_batch(cuda, dt, D):
    """Lengths of zero and one, tile edges, a sequence with nothing but its chunk, one with no row at all."""
    run(2, 4, D, 16, dt, [1, 5, 0, 16, 33, 128, 129, 200, 7, 3], [0, 300, 40, 0, 95, 0, 511, 57, 1000, -3])


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 11, 16])
def test_group_sizes(cuda, G):
    run(2, G, 128, 16, orc.BF16, [1, 40, 150], [77, 128, 3], seed=G)


@pytest.mark.parametrize("bs", [1, 2, 8, 20, 24, 32, 48, 64, 128, 256])
def test_block_sizes(cuda, bs):
    """Blocks that hold less than a tile, more than one, and end inside one."""
    run(2, 4, 64, bs, orc.F16, [3, 70, 1, 140], [0, 200, 129, 380], seed=bs)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("D", [64, 128])
def test_windows(cuda, window, D):
    run(1, 4, D, 16, orc.BF16, [1, 60, 300, 9], [500, 200, 0, 1100], window=window, seed=window % 97)


@pytest.mark.parametrize("bits,gs,meta,D,bs,dt", [
    (8, 64, orc.F16, 128, 16, orc.BF16), (4, 64, orc.F16, 128, 16, orc.BF16), (8, 64, orc.F32, 64, 16, orc.F16),
    (4, 32, orc.F32, 64, 16, orc.F16), (8, 8, orc.F16, 128, 16, orc.F16), (4, 8, orc.F32, 128, 16, orc.BF16),
    (8, 128, orc.F32, 128, 8, orc.BF16), (4, 128, orc.F16, 128, 48, orc.F16), (8, 16, orc.F16, 64, 5, orc.BF16),
    (4, 64, orc.F32, 64, 1, orc.BF16), (8, 32, orc.F32, 128, 20, orc.F16), (4, 16, orc.F16, 64, 256, orc.F16)])
def test_quantised_pools(cuda, bits, gs, meta, D, bs, dt):
    run(2, 4, D, bs, dt, [1, 40, 130, 0, 66], [130, 300, 20, 9, 0], bits=bits, gs=gs, meta=meta, seed=bits + gs)
    run(1, 5, D, bs, dt, [70], [333], window=90, bits=bits, gs=gs, meta=meta, seed=bits + gs + 1)


def test_long_context_few_rows(cuda):
    run(1, 8, 128, 16, orc.BF16, [5, 1], [20000, 9001], layers=1, layer=0)
    run(2, 4, 64, 16, orc.F16, [3], [30001], layers=1, layer=0)


def test_long_prompt(cuda):
    run(2, 4, 128, 16, orc.BF16, [2500], [0], layers=1, layer=0)
    run(1, 1, 64, 16, orc.F16, [3001], [700], layers=1, layer=0)


def test_many_sequences(cuda):
    rng = np.random.default_rng(3)
    n = rng.integers(0, 6, 700).tolist()
    c = rng.integers(0, 90, 700).tolist()
    run(1, 4, 64, 16, orc.BF16, n, c, layers=1, layer=0)


def test_eight_thousand_sequences(cuda):
    run(1, 2, 64, 8, orc.F16, [1, 0, 2] * 2730, [3, 2, 0] * 2730, layers=1, layer=0)


def test_offsets_past_32_bits(cuda):
    """Blocks whose bytes lie beyond 4 GiB into the pool."""
    H, D, bs, dt, L = 8, 128, 16, orc.BF16, 8
    pool = rmlx_kv.KVPool(L, H, D, bs, 9000, dtype=dt)
    assert pool.layout.bytes > 2 ** 32
    rows = pool_rows(pool, dt)
    g = torch.Generator("cuda").manual_seed(5)
    first = 8960
    rows[first:] = torch.randn(rows[first:].shape, generator=g, device="cuda").to(TORCH[dt])
    q_lens, lens = [9, 20], [300, 111]
    bt = tables(lens, bs, 40, g) + first
    q = torch.randn(29, H * 2, D, generator=g, device="cuda").to(TORCH[dt])
    out = torch.empty_like(q)
    ws = torch.empty(pool.chunk_attention_workspace_size(2), dtype=torch.uint8, device="cuda")
    pool.chunk_attention(L - 1, q, 2, bt, bt.shape[1], dev(q_lens), dev(lens), 2, 29, D ** -0.5, out, ws)
    assert pool.check() == 0
    check(pool, L - 1, q, 2, bt, q_lens, lens, 0, out, dt)


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("bs,D", [(16, 128), (5, 64)])
def test_masked_rows_have_no_influence(cuda, junk, bs, D):
    """Junk in slots behind a sequence's end, in rows below the window and in K and V of later tokens."""
    H, G, dt = 2, 4, orc.BF16
    g = torch.Generator("cuda").manual_seed(8)
    q_lens, lens = [6, 40, 1], [133, 40, 90]
    N = sum(-(-n // bs) for n in lens)
    results = []
    bt = tables(lens, bs, N, g)
    kv = torch.randn(N, 1, 2, H, bs, D, generator=g, device="cuda").to(TORCH[dt])
    q = torch.randn(47, H * G, D, generator=g, device="cuda").to(TORCH[dt])
    seen_below = {0: 130, 1: 20, 2: 90}  # sequence -> junk starts at this row (tokens before it must not care)
    window = 50
    for dirty in (False, True):
        pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt)
        rows = pool_rows(pool, dt)
        rows.copy_(kv)
        if dirty:
            for s, start in seen_below.items():
                for r in range(start, bt.shape[1] * bs):
                    if r < -(-lens[s] // bs) * bs:
                        rows[int(bt[s, r // bs]), :, :, :, r % bs] = junk
            for r in range(0, 90 - window):  # the last sequence's rows below its one token's window
                rows[int(bt[2, r // bs]), :, :, :, r % bs] = junk
        out = torch.empty_like(q)
        ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
        pool.chunk_attention(0, q, G, bt, bt.shape[1], dev(q_lens), dev(lens), 3, 47, D ** -0.5, out, ws, window=window)
        assert pool.check() == 0
        results.append(out)
    clean, dirty = (r.float() for r in results)
    eps = torch.finfo(TORCH[dt]).eps
    for a, b in ((0, 3), (6, 26), (46, 47)):  # tokens that see no junk: positions 127..129, 0..19 and 89
        assert torch.isfinite(dirty[a:b]).all()
        # both are within eps |v|max of the same exact value; weights are the same up to the order of sums
        assert (dirty[a:b] - clean[a:b]).abs().max() <= 2 * (eps + 2e-4) * kv.float().abs().max()
    if junk != junk:
        assert torch.isnan(dirty[3:6]).all() and torch.isnan(dirty[26:46]).all()  # rows that do see it


def test_every_row_through_the_exact_path(cuda):
    """V holds an infinity that all tokens but the first few see: NaN or infinity there, the others exact."""
    H, G, D, bs, dt = 1, 4, 64, 16, orc.BF16
    g = torch.Generator("cuda").manual_seed(16)
    pool = rmlx_kv.KVPool(1, H, D, bs, 320, dtype=dt)
    fill(pool, dt, 0, g)
    rows = pool_rows(pool, dt)
    bt = torch.arange(320, dtype=torch.int32, device="cuda")[None]
    at = 4930
    q = torch.randn(200, G, D, generator=g, device="cuda").to(TORCH[dt])
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
    clean, out = torch.empty_like(q), torch.empty_like(q)
    pool.chunk_attention(0, q, G, bt, 320, dev([200]), dev([5120]), 1, 200, D ** -0.5, clean, ws)
    rows[at // bs, 0, 1, 0, at % bs] = float("inf")
    pool.chunk_attention(0, q, G, bt, 320, dev([200]), dev([5120]), 1, 200, D ** -0.5, out, ws)
    assert pool.check() == 0
    first = at - 4920  # tokens before the infinity
    assert torch.isfinite(out[:first]).all()
    assert (out[:first].float() - clean[:first].float()).abs().max() <= 2 * (2.0 ** -7 + 2e-4) * 5.5
    assert (out[first:] == float("inf")).all()


def test_masked_rows_quantised(cuda):
    """Junk scales and zeros behind the end of a sequence and in later tokens of a quantised pool."""
    H, G, D, bs, dt = 1, 4, 128, 16, orc.BF16
    g = torch.Generator("cuda").manual_seed(9)
    lens = [70]
    outs = []
    q = torch.randn(10, G, D, generator=g, device="cuda").to(TORCH[dt])
    k, v = (torch.randn(80, H, D, generator=g, device="cuda").to(TORCH[dt]) for _ in range(2))
    for dirty in (False, True):
        pool = rmlx_kv.KVPool(1, H, D, bs, 5, dtype=dt, quant_bits=8, group_size=64, meta_dtype=orc.F16)
        kk, vv = k.clone(), v.clone()
        if dirty:
            kk[65:], vv[65:] = float("inf"), float("nan")
        pool.append(kk, vv, torch.arange(80, dtype=torch.int32, device="cuda"), 80)
        out = torch.empty_like(q)
        ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
        bt = torch.arange(5, dtype=torch.int32, device="cuda")
        pool.chunk_attention(0, q, G, bt, 5, dev([10]), dev(lens), 1, 10, D ** -0.5, out, ws)
        assert pool.check() == 0
        outs.append(out.float())
    assert torch.isfinite(outs[1][:5]).all()
    assert (outs[0][:5] - outs[1][:5]).abs().max() <= 2 * (2.0 ** -7 + 2e-4) * v.float().abs().max()
    assert torch.isnan(outs[1][5:]).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kscale,vscale,qscale", [(1.0, 1e6, 1.0), (1e6, 1.0, 1e-6), (1e-6, 1e-7, 1e6), (30.0, 40.0, 1e-2), (1e-3, 1e-3, 1e20)])
def test_value_ranges_of_quantised_pools(cuda, bits, kscale, vscale, qscale):
    """bf16 rows far outside f16's range, and near its smallest values; the exact path takes the rows that see them."""
    H, G, D, bs, dt = 2, 4, 128, 16, orc.BF16
    g = torch.Generator("cuda").manual_seed(14)
    pool = rmlx_kv.KVPool(1, H, D, bs, 20, dtype=dt, quant_bits=bits, group_size=32, meta_dtype=orc.F32)
    if qscale > 1e10:  # scores of order 1 from keys of 1e-20
        kscale = 1e-20
    k, v = ((torch.randn(320, H, D, generator=g, device="cuda") * s).to(TORCH[dt]) for s in (kscale, vscale))
    v[:200, :, :32] = 3e-6 * vscale  # groups of one value
    v[200:, :, 64:96] = 0
    pool.append(k, v, torch.arange(320, dtype=torch.int32, device="cuda"), 320)
    q = (torch.randn(45, H * G, D, generator=g, device="cuda") * qscale).to(TORCH[dt])
    out = torch.empty_like(q)
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
    bt = torch.arange(20, dtype=torch.int32, device="cuda")[None]
    pool.chunk_attention(0, q, G, bt, 20, dev([45]), dev([310]), 1, 45, D ** -0.5, out, ws)
    assert pool.check() == 0
    check(pool, 0, q, G, bt, [45], [310], 0, out, dt)


def test_large_scores(cuda):
    """Scores of thousands: one key takes all the weight, and -inf scores beside it."""
    H, G, D, bs, dt = 1, 1, 64, 16, orc.F16
    g = torch.Generator("cuda").manual_seed(10)
    pool = rmlx_kv.KVPool(1, H, D, bs, 40, dtype=dt)
    rows = pool_rows(pool, dt)
    rows.copy_(torch.randn(rows.shape, generator=g, device="cuda"))
    rows[:, :, 0] *= 60
    bt = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    q = (40 * torch.randn(200, 1, D, generator=g, device="cuda")).to(TORCH[dt])
    out = torch.empty_like(q)
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
    pool.chunk_attention(0, q, G, bt, 40, dev([200]), dev([640]), 1, 200, D ** -0.5, out, ws)
    assert pool.check() == 0
    k, v = (rows[:, 0, i, 0].reshape(640, D).double() for i in (0, 1))
    s = (q[:, 0].double() @ k.t()) * D ** -0.5
    s = s.masked_fill(torch.arange(640, device="cuda")[None] > torch.arange(440, 640, device="cuda")[:, None], -np.inf)
    # an f32 score of size S is off by up to D 2^-24 sum |q k| scale; weights by that factor
    bound = (D * 2.0 ** -24) * (q[:, 0].double().abs() @ k.abs().t()).amax(-1) * D ** -0.5
    p = torch.softmax(s, -1)
    err = (out[:, 0].double() - p @ v).abs()
    A = p @ v.abs()
    assert (err <= (2.0 ** -10 + 2e-4) * A + (2 * bound)[:, None] * v.abs().max() + 2.0 ** -24).all()


def test_one_token_equals_decode_attention(cuda):
    """The same arguments through rmlx_kv_decode_attention: both within their bound of the same value."""
    H, G, D, bs, dt = 4, 4, 128, 16, orc.F16
    g = torch.Generator("cuda").manual_seed(4)
    lens = [1, 50, 700, 1300]
    N = sum(-(-n // bs) for n in lens)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt)
    fill(pool, dt, 0, g)
    bt = tables(lens, bs, N, g)
    q = torch.randn(4, H * G, D, generator=g, device="cuda").to(TORCH[dt])
    a, b = torch.empty_like(q), torch.empty_like(q)
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
    wd = torch.empty(pool.attention_workspace_size(G, 4, sum(lens)), dtype=torch.uint8, device="cuda")
    pool.chunk_attention(0, q, G, bt, bt.shape[1], dev([1] * 4), dev(lens), 4, 4, D ** -0.5, a, ws)
    pool.decode_attention(0, q, G, bt, bt.shape[1], dev(lens), 4, D ** -0.5, b, wd)
    assert pool.check() == 0
    assert (a.float() - b.float()).abs().max() <= 2 * (2.0 ** -10 + 2e-4) * 5.5  # |v| < 5.5


def test_prefill_in_chunks_with_prefix_reuse(cuda):
    """The batch planner admits prompts (the second reuses the first's blocks), each prompt is rotated, appended and
    attended in chunks; the result is that of the whole prompt at once, and decode goes on from it."""
    H, G, D, bs, dt = 2, 4, 128, 16, orc.BF16
    g = torch.Generator("cuda").manual_seed(6)
    mgr = rmlx_kv.PagedCacheManager(bs, 64)
    from rmlx_kv.batch import KVBatch
    prefix = rmlx_kv.PrefixCacheManager(64)
    batch = KVBatch(mgr, prefix, 4)
    pool = rmlx_kv.KVPool(1, H, D, bs, 64, dtype=dt)
    inv = (10000.0 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))).float()
    rope = rmlx_kv.Rope(inv, D)
    rng = np.random.default_rng(1)
    shared = rng.integers(0, 1000, 96).tolist()
    prompts = {1: shared + rng.integers(0, 1000, 60).tolist(), 2: shared + rng.integers(0, 1000, 41).tolist()}
    table = torch.randn(1000, (G + 2) * H, D, generator=g, device="cuda").to(TORCH[dt])  # a "projection" per token id
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
    whole = {}
    for uid, prompt in prompts.items():
        row, cached, slots = batch.add(uid, prompt)
        if uid == 2:
            assert cached == 96
        bt = dev(batch.tables()[0].tolist())[row:row + 1].contiguous()
        outs, done = [], cached
        slots = dev(slots.tolist())
        for step in (17, 1, len(prompt)):
            n = min(step, len(prompt) - done)
            x = table[torch.tensor(prompt[done:done + n], device="cuda")]
            q, k, v = x.split([H * G, H, H], 1)
            pos = torch.arange(done, done + n, dtype=torch.int32, device="cuda")
            qr = torch.empty(n, H * G, D, dtype=TORCH[dt], device="cuda")
            out = torch.empty_like(qr)
            w = x.shape[1] * D
            pool.append_rope(0, k, v, slots[done - cached:], n, pos, rope, q=q, q_out=qr, q_heads=H * G,
                             token_stride=w, q_token_stride=w)
            pool.chunk_attention(0, qr, G, bt, bt.shape[1], dev([n]), dev([done + n]), 1, n, D ** -0.5, out, ws)
            check(pool, 0, qr, G, bt, [n], [done + n], 0, out, dt)
            outs.append((qr, out))
            done += n
        assert done == len(prompt)
        whole[uid] = torch.cat([o[0] for o in outs]), torch.cat([o[1] for o in outs])
        n = len(prompt) - cached
        out = torch.empty_like(whole[uid][1])
        pool.chunk_attention(0, whole[uid][0], G, bt, bt.shape[1], dev([n]), dev([len(prompt)]), 1, n, D ** -0.5, out, ws)
        check(pool, 0, whole[uid][0], G, bt, [n], [len(prompt)], 0, out, dt)
        if uid == 1:
            batch.remove(1, cache_prefix=True)
    assert pool.check() == 0


def test_a_graph_follows_its_lengths(cuda):
    """A captured call replayed after its lengths, tables and queries changed on the device; then with no chunk at all."""
    H, G, D, bs, dt = 2, 4, 128, 16, orc.BF16
    g = torch.Generator("cuda").manual_seed(17)
    pool = rmlx_kv.KVPool(1, H, D, bs, 400, dtype=dt)
    fill(pool, dt, 0, g)
    width, T = 150, 400
    bt = torch.zeros(3, width, dtype=torch.int32, device="cuda")
    q_lens, lens = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(T, H * G, D, dtype=TORCH[dt], device="cuda")
    out = torch.zeros_like(q)
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.chunk_attention(0, q, G, bt, width, q_lens, lens, 3, T, D ** -0.5, out, ws)
    for n, L in (([1, 1, 1], [5, 900, 2300]), ([300, 0, 90], [310, 70, 2000]), ([7, 200, 64], [2400, 200, 64]), ([0, 0, 0], [9, 9, 9])):
        new = tables(L, bs, 400, g)
        bt.zero_()
        bt[:, :new.shape[1]] = new
        q_lens.copy_(dev(n))
        lens.copy_(dev(L))
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        out.fill_(4.0)
        graph.replay()
        torch.cuda.synchronize()
        assert pool.check() == 0
        assert (out[sum(n):] == 4.0).all()
        check(pool, 0, q, G, bt, n, L, 0, out, dt)


def test_graphs_streams_and_bad_arguments(cuda):
    H, G, D, bs, dt = 2, 4, 64, 16, orc.BF16
    g = torch.Generator("cuda").manual_seed(12)
    pool = rmlx_kv.KVPool(1, H, D, bs, 80, dtype=dt)
    fill(pool, dt, 0, g)
    size = pool.chunk_attention_workspace_size(G)
    sets = []
    for q_lens, lens in (([30, 5], [400, 300]), ([3, 60], [500, 60])):
        bt = tables(lens, bs, 80, g)
        q = torch.randn(sum(q_lens), H * G, D, generator=g, device="cuda").to(TORCH[dt])
        sets.append([q_lens, lens, bt, q, torch.empty_like(q), torch.empty(size, dtype=torch.uint8, device="cuda"),
                     dev(q_lens), dev(lens)])

    def call(s, stream=None):
        pool.chunk_attention(0, s[3], G, s[2], s[2].shape[1], s[6], s[7], 2, s[3].shape[0], D ** -0.5, s[4], s[5], stream=stream)

    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(s)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, graph, st in zip(sets, graphs, streams):
            s[4].zero_()
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for s in sets:
            check(pool, 0, s[3], G, s[2], s[0], s[1], 0, s[4], dt)
    for s, st in zip(sets, streams):  # the two at once on two streams, each with its workspace
        s[4].zero_()
    torch.cuda.synchronize()
    for s, st in zip(sets, streams):
        call(s, st)
    torch.cuda.synchronize()
    for s in sets:
        check(pool, 0, s[3], G, s[2], s[0], s[1], 0, s[4], dt)
    assert pool.check() == 0

    q_lens, lens, bt, q, out, ws, dq, dl = sets[0]
    # more rows in q_lens than the launch has: flagged, nothing written
    out.fill_(3.0)
    pool.chunk_attention(0, q, G, bt, bt.shape[1], dq, dl, 2, q.shape[0] - 1, D ** -0.5, out, ws)
    assert pool.check() == 16 and (out == 3.0).all()
    pool.chunk_attention(0, q, G, bt, bt.shape[1], dev([2 ** 30] * 2), dl, 2, q.shape[0], D ** -0.5, out, ws)
    assert pool.check() == 16 and (out == 3.0).all()
    four = bt[[0, 1, 0, 1]].contiguous()  # lengths whose 32-bit sum is 0
    pool.chunk_attention(0, q, G, four, bt.shape[1], dev([2 ** 30] * 4), dev([9] * 4), 4, q.shape[0], D ** -0.5, out, ws)
    assert pool.check() == 16 and (out == 3.0).all()
    # a bad block of one sequence, a table that is too short for the other: flagged; a third is right
    bad = torch.cat([bt, bt[:1]])[:, :bt.shape[1]].contiguous()
    bad[0, 3] = 80
    bad[1, 0] = -1
    q3 = torch.cat([q, q[:30]])
    out3 = torch.empty_like(q3)
    pool.chunk_attention(0, q3, G, bad, bad.shape[1], dev(q_lens + [30]), dev(lens + [400]), 3, q3.shape[0], D ** -0.5, out3, ws)
    assert pool.check() == 2
    check(pool, 0, q3[35:], G, bad[2:].contiguous(), [30], [400], 0, out3[35:], dt)
    for long in (10 ** 6, 2 ** 31 - 1):
        pool.chunk_attention(0, q, G, bt, bt.shape[1], dq, dev([400, long]), 2, q.shape[0], D ** -0.5, out, ws)
        assert pool.check() == 2
        check(pool, 0, q[:30], G, bt[:1].contiguous(), [30], [400], 0, out[:30], dt)

    def refused(status=5, **kw):
        args = dict(layer=0, q=q, q_heads_per_kv=G, block_tables=bt, block_table_stride=bt.shape[1], q_lens=dq, seq_lens=dl,
                    num_seqs=2, num_q_tokens=q.shape[0], softmax_scale=0.1, out=out, workspace=ws)
        args.update(kw)
        with pytest.raises(rmlx_kv.RmlxError) as e:
            pool.chunk_attention(**args)
        assert e.value.status == status

    refused(1, layer=1)
    refused(q_heads_per_kv=0)
    refused(q_heads_per_kv=17)
    refused(num_seqs=-1)
    refused(num_seqs=8193)
    refused(num_q_tokens=-1)
    refused(window=-1)
    refused(softmax_scale=0.0)
    refused(softmax_scale=float("nan"))
    refused(block_table_stride=0)
    refused(q=None)
    refused(q=q.data_ptr() + 2)
    refused(q_token_stride=12)
    refused(q_lens=None)
    refused(workspace_bytes=size - 1)
    with pytest.raises(rmlx_kv.RmlxError):
        pool.chunk_attention_workspace_size(17)
    for kw in (dict(dtype=orc.F32), dict(head_dim=96)):
        args = dict(num_layers=1, num_kv_heads=1, head_dim=64, block_size=16, num_blocks=2, dtype=dt)
        args.update(kw)
        other = rmlx_kv.KVPool(**args)
        with pytest.raises(rmlx_kv.RmlxError):
            other.chunk_attention(0, q, G, bt, bt.shape[1], dq, dl, 2, q.shape[0], 0.1, out, ws)
    assert pool.check() == 0

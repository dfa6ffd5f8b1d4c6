"""Chunk attention (rmlx_kv_chunk_attention) where a value's range, not its formula, makes it hard.

Bound of an element, with A = sum_j p_j |v_j| (p the softmax) and S = sum_j |v_j| over the row's visible keys:
  * f16 products (f16 pools and all quantised ones): a weight is held relative to a running maximum m that is at most
    the row's maximum and is scaled by 2^7, so it is rounded by half a step of f16, 2^-11 of it, or, below f16's
    normal numbers, by at most 2^-25 2^-7 of the largest weight, which the sum of weights is never below:
    |error| <= 2^-11 A + 2^-32 S.  bf16 products have f32's range: 2^-8 A (half a step of bf16 is 2^-9).
  * the output's rounding: eps / 2 of |out| <= A, and half a step among the subnormals of f16 (2^-25);
  * f32 scores, exponentials and sums: 2e-4 of A (as derived in test_gpu_chunk_attention.py), for scores of at most
    64: a larger score s adds its own rounding, 2^-23 s, to each weight;
  * quantised pools: a stored value code * scale + zero is rounded to f16 (2^-11 of it): 2^-11 A for V, and a score
    off by delta <= 2^-11 scale sum |q_d k_d| for K, which moves weights and their sum by exp(2 delta) together.
    Below f16's normal numbers the rounding is 2^-25: in f16 pools that is half a step of the output's own; in bf16
    ones it stands only where the largest output of the element's group is 2^-13 or more, so 2^-12 of that largest.
"""
import numpy as np
import pytest
import torch

import oracle as orc
import rmlx_kv
from test_gpu_append_rope import TORCH, pool_rows
from test_gpu_chunk_attention import dev, stored_rows, tables

pytestmark = pytest.mark.gpu


def attend(pool, q, G, bt, q_lens, lens, out=None, ws=None, window=0, scale=None):
    """One call over contiguous q rows; the result."""
    out = torch.empty_like(q) if out is None else out
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda") if ws is None else ws
    pool.chunk_attention(0, q, G, bt, bt.shape[1], dev(q_lens), dev(lens), len(lens), q.shape[0],
                         pool.cfg.head_dim ** -0.5 if scale is None else scale, out, ws, window=window)
    return out


def check_rows(pool, q, G, bt, q_lens, lens, out, dt, window=0):
    """Every out row against float64 over the stored rows, within the bound above."""
    c = pool.cfg
    H, D, bs = c.num_kv_heads, c.head_dim, c.block_size
    rows = stored_rows(pool, 0, dt)
    eps = torch.finfo(TORCH[dt]).eps
    f16 = bool(c.quant_bits) or dt == orc.F16
    at = 0
    for s, (n, L) in enumerate(zip(q_lens, lens)):
        blocks = bt[s, :-(-L // bs)].long().clamp(0, c.num_blocks - 1)  # a table may name no block below the window
        kv = rows[blocks]
        k, v = (kv[:, i].transpose(0, 1).reshape(H, -1, D)[:, :L] for i in (0, 1))
        pos = torch.arange(L - n, L, device="cuda")[:, None]
        key = torch.arange(L, device="cuda")[None]
        seen = (key <= pos) & ((key > pos - window) if window else True)
        used = seen.any(0)
        k, v = (torch.where(used[None, :, None], x, torch.zeros_like(x)) for x in (k, v))
        x = q[at:at + n].double().view(n, H, G, D)
        sc = torch.einsum("nhgd,hld->hgnl", x, k) * D ** -0.5
        reach = torch.einsum("nhgd,hld->hgnl", x.abs(), k.abs()).masked_fill(~seen, 0).amax(-1).permute(2, 0, 1)[..., None] * D ** -0.5
        p = torch.softmax(sc.masked_fill(~seen, -np.inf), -1)
        want = torch.einsum("hgnl,hld->nhgd", p, v)
        A = torch.einsum("hgnl,hld->nhgd", p, v.abs())
        S = torch.einsum("nl,hld->nhd", seen.double(), v.abs())[:, :, None]
        rel = (2.0 ** -11 if f16 else 2.0 ** -8) + eps / 2 + 2e-4 + 2.0 ** -23 * reach
        if c.quant_bits:
            rel = rel + 2.0 ** -11 + 2 * 2.0 ** -11 * reach
        tol = rel * A + (2.0 ** -32 * S if f16 else 0) + (2.0 ** -25 if dt == orc.F16 else 1e-38)
        if c.quant_bits and dt == orc.F16:
            tol = tol + 2.0 ** -25
        elif c.quant_bits and c.meta_dtype == orc.F32:
            top = want.abs().unflatten(-1, (-1, min(c.group_size, 32))).amax(-1, keepdim=True)
            tol = tol + (2.0 ** -25 * (top >= 2.0 ** -13)).expand(*top.shape[:-1], min(c.group_size, 32)).flatten(-2)
        got = out[at:at + n].double().view(n, H, G, D)
        assert torch.isfinite(got).all()
        err = (got - want).abs()
        assert (err <= tol).all(), (n, L, float((err / tol).max()))
        at += n


@pytest.mark.parametrize("dt,bits,meta", [(orc.F16, 0, orc.F16), (orc.BF16, 0, orc.F16), (orc.BF16, 8, orc.F16), (orc.BF16, 4, orc.F32)])
@pytest.mark.parametrize("gap", [10.0, 14.0, 16.0, 17.5, 20.0])
@pytest.mark.parametrize("D,q_lens,ctx", [(128, [3, 70], [5000, 900]), (64, [2], [40000])])
def test_tail_behind_one_key(cuda, dt, bits, meta, gap, D, q_lens, ctx):
    """The first key holds nearly all the weight and its value is 0: the output is the tail's alone, `gap` nats below.
    The second shape splits one item over many parts, with the first key in one of them."""
    H, G, bs = 2, 4, 16
    lens = [n + c for n, c in zip(q_lens, ctx)]
    g = torch.Generator("cuda").manual_seed(int(gap * 10) + D)
    N = sum(-(-n // bs) for n in lens)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=32, meta_dtype=meta)
    sign = torch.where(torch.rand(D, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    q = (sign + 0.02 * torch.randn(sum(q_lens), H * G, D, generator=g, device="cuda")).to(TORCH[dt])
    bt = tables(lens, bs, N, g)
    slots = torch.arange(N * bs, device="cuda", dtype=torch.int32)
    k = 0.05 * torch.randn(N * bs, H, D, generator=g, device="cuda")
    v = 1 + 0.5 * torch.randn(N * bs, H, D, generator=g, device="cuda")
    for s in range(len(lens)):
        k[int(bt[s, 0]) * bs] = sign * gap * D ** -0.5
        v[int(bt[s, 0]) * bs] = 0
    pool.append(k.to(TORCH[dt]), v.to(TORCH[dt]), slots, N * bs)
    out = attend(pool, q, G, bt, q_lens, lens)
    assert pool.check() == 0
    check_rows(pool, q, G, bt, q_lens, lens, out, dt)


@pytest.mark.parametrize("dt,bits", [(orc.BF16, 0), (orc.F16, 0), (orc.BF16, 8), (orc.BF16, 4)])
def test_same_bits_whatever_ran_before(cuda, dt, bits):
    """The same call after calls that leave other queries in shared memory gives the same bits: 5 tokens of 4 heads
    fill 20 lanes of a warp's 32, and the others must have no say."""
    H, G, D, bs = 8, 4, 128, 16
    g = torch.Generator("cuda").manual_seed(31)
    q_lens, lens = [5] * 40 + [33], [900 + 37 * i for i in range(41)]
    N = sum(-(-n // bs) for n in lens)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=64, meta_dtype=orc.F16)
    slots = torch.arange(N * bs, device="cuda", dtype=torch.int32)
    k, v = (torch.randn(N * bs, H, D, generator=g, device="cuda").to(TORCH[dt]) for _ in range(2))
    pool.append(k, v, slots, N * bs)
    bt = tables(lens, bs, N, g)
    q = (1.5 * torch.randn(sum(q_lens), H * G, D, generator=g, device="cuda")).to(TORCH[dt])
    results = []
    for size in (0.0, 0.5, 4.0, 30.0):
        before = (size * torch.randn(64 * 41, H * G, D, generator=g, device="cuda")).to(TORCH[dt])
        attend(pool, before, G, bt, [64] * 41, lens)
        results.append(attend(pool, q, G, bt, q_lens, lens))
    assert pool.check() == 0
    for r in results[1:]:
        assert torch.equal(results[0].view(torch.int16), r.view(torch.int16))


@pytest.mark.parametrize("bits,meta", [(8, orc.F32), (4, orc.F16)])
def test_query_rows_of_many_sizes(cuda, bits, meta):
    """One element of a bf16 query row is 2^23 times the others, and its keys are as much smaller: the small elements
    decide the scores and keep their eight bits."""
    H, G, D, bs, dt = 1, 4, 128, 16, orc.BF16
    g = torch.Generator("cuda").manual_seed(32)
    L, n = 320, 45
    pool = rmlx_kv.KVPool(1, H, D, bs, L // bs, dtype=dt, quant_bits=bits, group_size=32, meta_dtype=meta)
    k, v = (torch.randn(L, H, D, generator=g, device="cuda") for _ in range(2))
    k[:, :, :32] *= 1e-3
    k[:, :, 32:] *= 3000
    pool.append(k.to(TORCH[dt]), v.to(TORCH[dt]), torch.arange(L, device="cuda", dtype=torch.int32), L)
    q = torch.randn(n, H * G, D, generator=g, device="cuda")
    q[..., 32:] *= 2.0 ** -9
    q[..., 5] = 2.0 ** 14
    q = q.to(TORCH[dt])
    bt = torch.arange(L // bs, dtype=torch.int32, device="cuda")[None]
    out = attend(pool, q, G, bt, [n], [310])
    assert pool.check() == 0
    check_rows(pool, q, G, bt, [n], [310], out, dt)


def event_ms(f, n=3):
    f()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    for _ in range(n):
        f()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / n


@pytest.mark.parametrize("dt,bits,meta", [(orc.BF16, 8, orc.F32), (orc.BF16, 4, orc.F16), (orc.F16, 8, orc.F32)])
@pytest.mark.parametrize("what", ["v", "k"])
def test_one_tiny_group_costs_little(cuda, dt, bits, meta, what):
    """One group of values below f16's normal numbers, in one row that every token sees: right, and at the speed of
    a call without it (a tenth of it at least; every row taking the exact path is some hundred times slower)."""
    H, G, D, bs = 4, 4, 128, 16
    g = torch.Generator("cuda").manual_seed(33)
    q_lens, lens = [300, 40], [4000, 2000]
    N = sum(-(-n // bs) for n in lens)
    bt = tables(lens, bs, N, g)
    k, v = (torch.randn(N * bs, H, D, generator=g, device="cuda") for _ in range(2))
    q = torch.randn(sum(q_lens), H * G, D, generator=g, device="cuda").to(TORCH[dt])
    ms = []
    for tiny in (False, True):
        pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=32, meta_dtype=meta)
        kk, vv = k.clone(), v.clone()
        if tiny:
            for s in range(2):
                (vv if what == "v" else kk)[int(bt[s, 3]) * bs + 5, :, 32:64] *= 2e-5
        pool.append(kk.to(TORCH[dt]), vv.to(TORCH[dt]), torch.arange(N * bs, device="cuda", dtype=torch.int32), N * bs)
        ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        ms.append(event_ms(lambda: attend(pool, q, G, bt, q_lens, lens, out, ws)))
        assert pool.check() == 0
        check_rows(pool, q, G, bt, q_lens, lens, out, dt)
    assert ms[1] <= 10 * ms[0] + 0.2, ms


@pytest.mark.parametrize("dt,bits,meta,gs", [(orc.BF16, 8, orc.F32, 8), (orc.BF16, 4, orc.F32, 16), (orc.BF16, 8, orc.F32, 64),
                                             (orc.F16, 4, orc.F32, 32), (orc.BF16, 8, orc.F16, 32)])
@pytest.mark.parametrize("size", [1e-4, 3e-6, 1e-9])
@pytest.mark.parametrize("D,q_lens,lens", [(128, [40, 3], [310, 90]), (64, [2], [9000])])
def test_tiny_columns(cuda, dt, bits, meta, gs, size, D, q_lens, lens):
    """V columns of one group hold tiny values in every key, next to ordinary ones: each output keeps its own digits."""
    if meta == orc.F16 or dt == orc.F16:
        size = max(size, 3e-6)  # 1e-9 is 0 in f16
    H, G, bs = 2, 4, 16
    g = torch.Generator("cuda").manual_seed(34)
    N = sum(-(-n // bs) for n in lens)
    bt = tables(lens, bs, N, g)
    k, v = (torch.randn(N * bs, H, D, generator=g, device="cuda") for _ in range(2))
    v[:, :, gs * 1 % D:gs * 1 % D + gs] *= size
    if gs < D:
        v[:, 1, :gs] = 0  # all zero: no digits to keep
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=gs, meta_dtype=meta)
    pool.append(k.to(TORCH[dt]), v.to(TORCH[dt]), torch.arange(N * bs, device="cuda", dtype=torch.int32), N * bs)
    q = torch.randn(sum(q_lens), H * G, D, generator=g, device="cuda").to(TORCH[dt])
    out = attend(pool, q, G, bt, q_lens, lens)
    assert pool.check() == 0
    check_rows(pool, q, G, bt, q_lens, lens, out, dt)


@pytest.mark.parametrize("dt,kscale,qscale", [(orc.BF16, 1e-5, 1e5), (orc.BF16, 1e-8, 1e8), (orc.F16, 2e-5, 3e4), (orc.BF16, 1e-5, 1e3)])
def test_tiny_keys_under_large_queries(cuda, dt, kscale, qscale):
    """Scores of order 1 (and of 0.01) from keys that f16 holds badly or not at all."""
    H, G, D, bs = 2, 4, 128, 16
    g = torch.Generator("cuda").manual_seed(35)
    L, n = 320, 45
    pool = rmlx_kv.KVPool(1, H, D, bs, L // bs, dtype=dt, quant_bits=8, group_size=32, meta_dtype=orc.F32)
    k, v = (torch.randn(L, H, D, generator=g, device="cuda") for _ in range(2))
    pool.append((k * kscale).to(TORCH[dt]), v.to(TORCH[dt]), torch.arange(L, device="cuda", dtype=torch.int32), L)
    q = (torch.randn(n, H * G, D, generator=g, device="cuda").clamp(-2, 2) * qscale).to(TORCH[dt])
    bt = torch.arange(L // bs, dtype=torch.int32, device="cuda")[None]
    out = attend(pool, q, G, bt, [n], [310])
    assert pool.check() == 0
    check_rows(pool, q, G, bt, [n], [310], out, dt)


@pytest.mark.parametrize("dt,bits,meta,bs,D", [(orc.BF16, 0, orc.F16, 16, 128), (orc.F16, 0, orc.F16, 64, 64), (orc.BF16, 0, orc.F16, 5, 64),
                                               (orc.BF16, 8, orc.F16, 16, 128), (orc.BF16, 4, orc.F32, 32, 64), (orc.F16, 8, orc.F32, 5, 128),
                                               (orc.BF16, 4, orc.F16, 1, 128)])
def test_freed_blocks_below_the_window(cuda, dt, bits, meta, bs, D):
    """Table entries of blocks that lie wholly below every token's window may be anything: they are not read."""
    H, G, window = 2, 4, 100
    g = torch.Generator("cuda").manual_seed(36)
    q_lens, lens = [1, 9, 150], [1000, 333, 701]
    N = sum(-(-n // bs) for n in lens)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=32, meta_dtype=meta)
    k, v = (torch.randn(N * bs, H, D, generator=g, device="cuda").to(TORCH[dt]) for _ in range(2))
    pool.append(k, v, torch.arange(N * bs, device="cuda", dtype=torch.int32), N * bs)
    bt = tables(lens, bs, N, g)
    q = torch.randn(sum(q_lens), H * G, D, generator=g, device="cuda").to(TORCH[dt])
    whole = attend(pool, q, G, bt, q_lens, lens, window=window)
    assert pool.check() == 0
    check_rows(pool, q, G, bt, q_lens, lens, whole, dt, window=window)
    for s, (n, L) in enumerate(zip(q_lens, lens)):
        bt[s, :max(L - n - window + 1, 0) // bs] = [-1, N, 2 ** 31 - 1][s]
    out = attend(pool, q, G, bt, q_lens, lens, window=window)
    assert pool.check() == 0
    check_rows(pool, q, G, bt, q_lens, lens, out, dt, window=window)


@pytest.mark.parametrize("dt,bits", [(orc.BF16, 0), (orc.F16, 0), (orc.BF16, 8)])
@pytest.mark.parametrize("D,n,L", [(128, 60, 100), (128, 60, 2000), (64, 3, 20000)])
def test_rows_computed_again_repeat(cuda, dt, bits, D, n, L):
    """NaN in the last row, which the mask hides from all tokens but the last: their rows are computed again, in whole
    items (100 rows) and in parts, and come back finite, right and the same every time."""
    H, G, bs = 2, 4, 16
    g = torch.Generator("cuda").manual_seed(37)
    N = -(-L // bs)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=32, meta_dtype=orc.F32)
    k, v = (torch.randn(N * bs, H, D, generator=g, device="cuda") for _ in range(2))
    v[L - 1] = float("nan")
    pool.append(k.to(TORCH[dt]), v.to(TORCH[dt]), torch.arange(N * bs, device="cuda", dtype=torch.int32), N * bs)
    bt = torch.arange(N, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(n, H * G, D, generator=g, device="cuda").to(TORCH[dt])
    first = attend(pool, q, G, bt, [n], [L])
    for _ in range(10):
        assert torch.equal(attend(pool, q, G, bt, [n], [L]).view(torch.int16), first.view(torch.int16))
    assert pool.check() == 0
    assert torch.isnan(first[-1]).all()
    check_rows(pool, q[:-1], G, bt, [n - 1], [L - 1], first[:-1], dt)


def test_no_first_store_outlives_the_second(cuda):
    """Every row of many whole items is stored twice, first as NaN by one lane and then by others: no NaN is left."""
    H, G, D, bs, dt, S = 8, 16, 128, 16, orc.BF16, 64
    g = torch.Generator("cuda").manual_seed(39)
    pool = rmlx_kv.KVPool(1, H, D, bs, S * 2, dtype=dt)
    k, v = (torch.randn(S * 32, H, D, generator=g, device="cuda") for _ in range(2))
    v[31::32] = float("nan")
    pool.append(k.to(TORCH[dt]), v.to(TORCH[dt]), torch.arange(S * 32, device="cuda", dtype=torch.int32), S * 32)
    bt = torch.arange(S * 2, dtype=torch.int32, device="cuda").view(S, 2)
    q = torch.randn(S * 16, H * G, D, generator=g, device="cuda").to(TORCH[dt])
    for _ in range(5):
        out = attend(pool, q, G, bt, [16] * S, [32] * S).view(S, 16, H * G, D)
        assert torch.isfinite(out[:, :15]).all() and torch.isnan(out[:, 15]).all()
    assert pool.check() == 0


@pytest.mark.parametrize("bits", [0, 8])
def test_rows_computed_again_in_time(cuda, bits):
    """Every row of the last tile over 8192 keys through the exact path: some 75 to 100 times as long as a call
    without (a row and a key at a time took 700 times as long, and a million keys ran into the waits' limit)."""
    H, G, D, bs, dt, n, L = 8, 4, 128, 16, orc.BF16, 512, 8192
    g = torch.Generator("cuda").manual_seed(38)
    k, v = (torch.randn(L, H, D, generator=g, device="cuda") for _ in range(2))
    q = torch.randn(n, H * G, D, generator=g, device="cuda").to(TORCH[dt])
    bt = torch.arange(L // bs, dtype=torch.int32, device="cuda")[None]
    ms = []
    for junk in (False, True):
        if junk:
            v[L - 1] = float("nan")
        pool = rmlx_kv.KVPool(1, H, D, bs, L // bs, dtype=dt, quant_bits=bits, group_size=64, meta_dtype=orc.F32)
        pool.append(k.to(TORCH[dt]), v.to(TORCH[dt]), torch.arange(L, device="cuda", dtype=torch.int32), L)
        ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        ms.append(event_ms(lambda: attend(pool, q, G, bt, [n], [L], out, ws)))
        assert pool.check() == 0
    assert torch.isfinite(out[:-1]).all() and torch.isnan(out[-1]).all()
    assert ms[1] <= 250 * ms[0], ms


@pytest.mark.parametrize("bits,meta,gs,D,bs", [(8, orc.F16, 64, 128, 16), (4, orc.F16, 64, 128, 16), (8, orc.F32, 32, 64, 16),
                                               (4, orc.F32, 64, 64, 5), (8, orc.F16, 8, 128, 1)])
@pytest.mark.parametrize("n,L", [(70, 1500), (3, 9000)])
def test_f16_pools_over_codes_lose_little(cuda, bits, meta, gs, D, bs, n, L):
    """Rows with outliers in an f16 pool over codes: the error's norm against that of rounding the exact output to f16.
    Weights, V and the output are rounded by half a step of f16 each, which in values of random sign are independent
    shares of one size: sqrt(3) in all.  (With K in one f16 part its roundings alone came to 3.)"""
    H, G, dt = 2, 4, orc.F16
    g = torch.Generator("cuda").manual_seed(40 + D)
    N = -(-L // bs)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=gs, meta_dtype=meta)
    k, v = (torch.randn(N * bs, H, D, generator=g, device="cuda") for _ in range(2))
    k, v = (torch.where(torch.rand(x.shape, generator=g, device="cuda") < 0.01, 8 * x, x).to(TORCH[dt]) for x in (k, v))
    pool.append(k, v, torch.arange(N * bs, device="cuda", dtype=torch.int32), N * bs)
    bt = torch.randperm(N, generator=g, device="cuda").to(torch.int32)[None]
    q = torch.randn(n, H * G, D, generator=g, device="cuda").to(TORCH[dt])
    out = attend(pool, q, G, bt, [n], [L])
    assert pool.check() == 0
    check_rows(pool, q, G, bt, [n], [L], out, dt)
    kv = stored_rows(pool, 0, dt)[bt[0].long()]
    kk, vv = (kv[:, i].transpose(0, 1).reshape(H, -1, D)[:, :L] for i in (0, 1))
    s = torch.einsum("nhgd,hld->hgnl", q.double().view(n, H, G, D), kk) * D ** -0.5
    hidden = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
    want = torch.einsum("hgnl,hld->nhgd", torch.softmax(s.masked_fill(hidden, -np.inf), -1), vv).reshape(n, H * G, D)
    assert (out.double() - want).norm() <= 2 * (want.half().double() - want).norm()


@pytest.mark.parametrize("dt,bits,bs", [(orc.BF16, 0, 16), (orc.F16, 0, 5), (orc.BF16, 8, 16), (orc.F16, 4, 16)])
def test_query_strides(cuda, dt, bits, bs):
    """Queries laid out [head][token][dim], and one row for all tokens (stride 0): the bits of contiguous copies."""
    H, G, D, n, L = 2, 4, 128, 150, 400
    g = torch.Generator("cuda").manual_seed(41)
    N = -(-L // bs)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=64, meta_dtype=orc.F16)
    k, v = (torch.randn(N * bs, H, D, generator=g, device="cuda").to(TORCH[dt]) for _ in range(2))
    pool.append(k, v, torch.arange(N * bs, device="cuda", dtype=torch.int32), N * bs)
    bt = torch.arange(N, dtype=torch.int32, device="cuda")[None]
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")
    by_head = torch.randn(H * G, n, D, generator=g, device="cuda").to(TORCH[dt])
    for q, strides in ((by_head.transpose(0, 1), dict(q_token_stride=D, q_head_stride=n * D)),
                       (by_head[:, :1].transpose(0, 1).expand(n, -1, -1), dict(q_token_stride=0, q_head_stride=n * D))):
        out = torch.empty(n, H * G, D, dtype=TORCH[dt], device="cuda")
        pool.chunk_attention(0, by_head, G, bt, N, dev([n]), dev([L]), 1, n, D ** -0.5, out, ws, **strides)
        want = attend(pool, q.contiguous(), G, bt, [n], [L])
        assert pool.check() == 0
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))

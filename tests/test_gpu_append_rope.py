"""The append with position rotation (rmlx_kv_append_rope) on the GPU.

The expected rows are rotated in float64.  Error of a computed row before it
is rounded to the pool's type, with x1, x2 the pair: the reduced angle is
rounded to f32 (at most half a turn of pi: pi 2^-25 = 9.4e-8 rad; the f64
product adds 1e-6 * 2^-31 per position), sincospif is good to an ulp (1.2e-7),
the two products and their sum round by 2^-24 each: in all below
4e-7 (|x1| + |x2|).  The store then rounds by half a step, eps / 2 of the
value.  A quantised pool with f32 scale and zero is off by half a code step
more.
"""
import numpy as np
import pytest
import torch

import oracle as orc
import rmlx_kv

pytestmark = pytest.mark.gpu
TORCH = {orc.F32: torch.float32, orc.F16: torch.float16, orc.BF16: torch.bfloat16}


class PoolBytes:
    def __init__(self, pool):
        self.pool = pool
        self.__cuda_array_interface__ = {"shape": (pool.layout.bytes,), "typestr": "|u1",
                                         "data": (pool.layout.base, False), "version": 3}


def pool_bytes(pool):
    return torch.as_tensor(PoolBytes(pool), device="cuda")


def pool_rows(pool, dt):
    """[block][layer][K, V][head][slot][dim] of a plain pool, a view."""
    c = pool.cfg
    return pool_bytes(pool).view(TORCH[dt]).view(c.num_blocks, c.num_layers, 2, c.num_kv_heads, c.block_size, c.head_dim)


def rotate64(x, pos, inv_freq, R, interleaved, axis):
    """Rows [T, heads, D] rotated in float64, and |x1| + |x2| of each rotated element."""
    x = x.double()
    ang = torch.stack([pos[int(a)].double() * inv_freq[i].double() for i, a in enumerate(axis)], 1)[:, None]
    i = torch.arange(R // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., a] = x[..., a] * ang.cos() - x[..., b] * ang.sin()
    y[..., b] = x[..., b] * ang.cos() + x[..., a] * ang.sin()
    mag[..., a] = mag[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, mag


def within(got, want, mag, dt):
    half = torch.finfo(TORCH[dt]).eps / 2
    tiny = torch.finfo(TORCH[dt]).tiny * 2 * half  # half a step among the subnormals
    err = (got.double() - want).abs()
    tol = half * want.abs() + 4e-7 * (1 + half) * mag + tiny
    assert (err <= tol).all(), float((err - tol).max())


def inputs(T, H, Hq, D, dt, seed, axes=1, far=2000):
    g = torch.Generator("cuda").manual_seed(seed)
    qkv = torch.randn(T, Hq + 2 * H, D, generator=g, device="cuda").to(TORCH[dt])
    pos = torch.randint(0, far, (axes, T), generator=g, device="cuda", dtype=torch.int32)
    return g, qkv, pos


def freqs(R, base=10000.0):
    return (base ** (-torch.arange(R // 2, device="cuda", dtype=torch.float64) / (R // 2))).float()


CASES = [
    # T, H, G, D, R, block, dtype, interleaved, axes
    (1, 8, 4, 128, 128, 16, orc.BF16, False, 1),
    (64, 8, 4, 128, 128, 16, orc.F16, False, 1),
    (37, 2, 3, 64, 32, 8, orc.BF16, True, 1),
    (300, 1, 8, 128, 64, 1, orc.F16, False, 3),
    (1500, 3, 5, 96, 48, 48, orc.BF16, True, 3),     # four tokens a CTA, odd head counts
    (1203, 2, 2, 72, 16, 20, orc.F16, False, 1),     # an odd number of chunks: the last unit holds one
    (33, 2, 2, 80, 80, 16, orc.F32, False, 2),
    (1300, 2, 1, 256, 256, 16, orc.F32, True, 1),
    (5, 4, 0, 128, 128, 16, orc.BF16, False, 1),     # keys only
]


@pytest.mark.parametrize("T,H,G,D,R,bs,dt,il,axes", CASES)
def test_rows(cuda, T, H, G, D, R, bs, dt, il, axes):
    g, qkv, pos = inputs(T, H, H * G, D, dt, 7 * T + D, axes)
    N = -(-T // bs) + 3
    pool = rmlx_kv.KVPool(2, H, D, bs, N, dtype=dt)
    rows = pool_rows(pool, dt)
    rows.fill_(7.0)
    slots = torch.randperm(N * bs, generator=g, device="cuda")[:T].to(torch.int32)
    if T > 4:
        slots[T // 2] = -1
    axis = torch.randint(0, axes, (R // 2,), generator=g, device="cuda", dtype=torch.int32)
    inv = freqs(R)
    rope = rmlx_kv.Rope(inv, R, interleaved=il, pair_axis=axis if axes > 1 else None, num_axes=axes)
    q, k, v = qkv.split([H * G, H, H], 1)
    width = qkv.shape[1] * D
    q_out = torch.full((T + 2, max(H * G, 1), D), 5.0, dtype=TORCH[dt], device="cuda")
    pool.append_rope(1, k, v, slots, T, pos, rope, q=q if G else None, q_out=q_out if G else None, q_heads=H * G,
                     token_stride=width, q_token_stride=width)
    assert pool.check() == 0
    ax = axis.tolist() if axes > 1 else [0] * (R // 2)
    if G:
        want, mag = rotate64(q, pos, inv, R, il, ax)
        within(q_out[:T], want, mag, dt)
        assert (q_out[:T, :, R:] == q[..., R:]).all()
        assert (q_out[T:] == 5.0).all()
    want, mag = rotate64(k, pos, inv, R, il, ax)
    live = slots >= 0
    at = slots[live].long()
    got = rows[at // bs, 1, :, :, at % bs]  # [t, 2, H, D]
    within(got[:, 0], want[live], mag[live], dt)
    assert torch.equal(got[:, 1], v[live])
    rows[at // bs, 1, :, :, at % bs] = 7.0
    assert (rows == 7.0).all()  # nothing else was written


@pytest.mark.parametrize("dt,bits,meta,gs,D", [(orc.BF16, 8, orc.F16, 64, 128), (orc.F16, 4, orc.F32, 32, 64),
                                               (orc.F32, 8, orc.F32, 128, 128), (orc.BF16, 4, orc.F16, 8, 96),
                                               (orc.BF16, 0, orc.F32, 64, 128), (orc.F32, 0, orc.F32, 64, 64)])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("T", [3, 1300])
def test_position_zero_is_the_append(cuda, dt, bits, meta, gs, D, il, T):
    """At position 0 every pair turns by nothing: the same bytes as rmlx_kv_append, quantised pools included."""
    H, bs = 2, 16
    N = -(-T // bs)
    g, qkv, pos = inputs(T, H, H, D, dt, 11, 1)
    pos.zero_()
    pools = [rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=gs, meta_dtype=meta) for _ in range(2)]
    slots = torch.randperm(N * bs, generator=g, device="cuda")[:T].to(torch.int32)
    q, k, v = (x.contiguous() for x in qkv.split([H, H, H], 1))
    pools[0].append(k, v, slots, T)
    q_out = torch.empty_like(q)
    R = 32
    pools[1].append_rope(0, k, v, slots, T, pos, rmlx_kv.Rope(freqs(R), R, interleaved=il), q=q, q_out=q_out, q_heads=H)
    torch.cuda.synchronize()
    assert torch.equal(*[pool_bytes(p) for p in pools])
    assert torch.equal(q_out, q)


@pytest.mark.parametrize("bits,gs,D,R,il", [(8, 64, 128, 128, False), (8, 128, 128, 64, False), (4, 32, 128, 128, True),
                                            (4, 64, 64, 32, False), (8, 8, 64, 16, True), (8, 32, 96, 96, False)])
@pytest.mark.parametrize("T", [40, 1300])
def test_quantised_rows(cuda, bits, gs, D, R, il, T):
    H, bs, dt = 3, 16, orc.F32
    N = -(-T // bs)
    g, qkv, pos = inputs(T, H, 0, D, dt, 13 + T, 1, far=100000)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=gs, meta_dtype=orc.F32)
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    inv = freqs(R)
    k, v = (x.contiguous() for x in qkv.split([H, H], 1))
    pool.append_rope(0, k, v, slots, T, pos, rmlx_kv.Rope(inv, R, interleaved=il))
    out = [torch.empty(H, T, D, device="cuda") for _ in range(2)]
    bt = torch.arange(N, device="cuda", dtype=torch.int32)
    pool.gather(0, bt, N, torch.tensor([T], dtype=torch.int32, device="cuda"), 1, *out)
    assert pool.check() == 0
    for got, rows, rot in ((out[0], k, True), (out[1], v, False)):
        want, mag = rotate64(rows, pos, inv, R if rot else 0, il, [0] * (R // 2 if rot else 0)) if rot else (
            rows.double(), torch.zeros_like(rows, dtype=torch.float64))
        grp = want.unflatten(-1, (-1, gs))
        step = (grp.amax(-1, keepdim=True) - grp.amin(-1, keepdim=True)) / (2 ** bits - 1)
        step = step.expand_as(grp).flatten(-2)
        # half a code step, the rows' own error (it moves the ends of the group too), and a few f32 roundings
        tol = 0.5 * step + 3 * 4e-7 * mag.amax(-1, keepdim=True) + 8 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True)
        err = (got.transpose(0, 1).double() - want).abs()
        assert (err <= tol).all(), float((err - tol).max())


def test_far_positions(cuda):
    """Angles near 2^31 radians, and negative ones, keep their fraction of a turn (2^31 * 2^-52 = 5e-7 rad more error)."""
    T, H, D, R = 64, 1, 64, 64
    g, qkv, _ = inputs(T, H, H, D, orc.F32, 3)
    pos = torch.randint(2 ** 30, 2 ** 31 - 1, (1, T), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    pos[0, ::2] *= -1
    pool = rmlx_kv.KVPool(1, H, D, 16, 4, dtype=orc.F32)
    inv = freqs(R)
    q = qkv[:, :1].contiguous()
    q_out = torch.empty_like(q)
    pool.append_rope(0, qkv[:, 1], qkv[:, 2], torch.arange(T, device="cuda", dtype=torch.int32), T, pos,
                     rmlx_kv.Rope(inv, R), q=q, q_out=q_out, q_heads=1, token_stride=3 * D)
    want, mag = rotate64(q, pos, inv, R, False, [0] * (R // 2))
    err = (q_out.double() - want).abs()
    assert (err <= 2.0 ** -24 * want.abs() + (4e-7 + 2e-6) * mag).all()


def test_in_place_other_stream_and_graph(cuda):
    T, H, G, D, dt = 50, 2, 4, 128, orc.BF16
    g, qkv, pos = inputs(T, H, H * G, D, dt, 21)
    pool = rmlx_kv.KVPool(1, H, D, 16, 8, dtype=dt)
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    inv = freqs(D)
    rope = rmlx_kv.Rope(inv, D)
    width = qkv.shape[1] * D
    want, mag = rotate64(qkv[:, :H * G], pos, inv, D, False, [0] * (D // 2))
    work = qkv.clone()
    q, k, v = work.split([H * G, H, H], 1)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    call = dict(q=q, q_out=q, q_heads=H * G, token_stride=width, q_token_stride=width, q_out_token_stride=width)
    pool.append_rope(0, k, v, slots, T, pos, rope, stream=stream, **call)
    stream.synchronize()
    within(q, want, mag, dt)
    assert torch.equal(work[:, H * G:], qkv[:, H * G:])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.append_rope(0, k, v, slots, T, pos, rope, **call)
    for _ in range(2):
        work.copy_(qkv)
        pool_rows(pool, dt).zero_()
        graph.replay()
        torch.cuda.synchronize()
        within(q, want, mag, dt)
        assert (pool_rows(pool, dt)[:, 0, 0].abs().sum() > 0)
    assert pool.check() == 0


def test_flagged_on_the_device(cuda):
    """Slots past the pool and axes out of range are flagged; nothing is written for such a slot."""
    H, D = 1, 64
    g, qkv, pos = inputs(4, H, 0, D, orc.F16, 5, 2)
    pool = rmlx_kv.KVPool(1, H, D, 16, 2, dtype=orc.F16)
    k, v = (x.contiguous() for x in qkv.split([H, H], 1))
    slots = torch.tensor([0, 32, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    pool.append_rope(0, k, v, slots, 4, pos, rmlx_kv.Rope(freqs(16), 16))
    assert pool.check() == 1
    rows = pool_rows(pool, orc.F16)
    assert torch.equal(rows[0, 0, 1, 0, 0], v[0, 0])
    rows[0, 0, :, 0, 0] = 0
    assert (rows == 0).all()
    axis = torch.tensor([0, 1, 2, -1, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
    pool.append_rope(0, k, v, slots[:1], 1, pos, rmlx_kv.Rope(freqs(16), 16, pair_axis=axis, num_axes=2))
    assert pool.check() == 8


def test_refusals(cuda):
    H, D = 1, 64
    pool = rmlx_kv.KVPool(1, H, D, 16, 2, dtype=orc.F16)
    x = torch.zeros(8, 4, D, dtype=torch.float16, device="cuda")
    i = torch.zeros(8, dtype=torch.int32, device="cuda")
    rope = rmlx_kv.Rope(freqs(32), 32)

    def refused(status, layer=0, rope=rope, k=x, T=8, pos=i, **kw):
        with pytest.raises(rmlx_kv.RmlxError) as e:
            pool.append_rope(layer, k, x, i, T, pos, rope, **kw)
        assert e.value.status == status

    bad, rng = 5, 1
    refused(rng, layer=1)
    refused(rng, layer=-1)
    refused(bad, T=-1)
    refused(bad, rope=rmlx_kv.Rope(freqs(24), 24))
    refused(bad, rope=rmlx_kv.Rope(freqs(80), 80))
    refused(bad, rope=rmlx_kv.Rope(freqs(32), 32, num_axes=0))
    refused(bad, k=None)
    refused(bad, pos=None)
    refused(bad, q_heads=1)
    refused(bad, q_heads=-1, q=x, q_out=x)
    refused(bad, token_stride=68)
    refused(bad, q=x, q_out=x, q_heads=1, q_token_stride=68)
    refused(bad, k=x.data_ptr() + 2)
    refused(bad, q=x.data_ptr() + 2, q_out=x, q_heads=1)
    pool.append_rope(0, None, None, None, 0, None, rope)  # no tokens: nothing to do
    odd = rmlx_kv.KVPool(1, 1, 12, 16, 2, dtype=orc.F32)
    with pytest.raises(rmlx_kv.RmlxError):
        odd.append_rope(0, x, x, i, 1, i, rmlx_kv.Rope(freqs(16), 16))
    assert pool.check() == 0

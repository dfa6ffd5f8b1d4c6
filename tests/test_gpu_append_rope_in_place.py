"""The append with rotation where q_out is q: the same bits as into another buffer."""
import pytest
import torch

import oracle as orc
import rmlx_kv
from test_gpu_append_rope import TORCH, freqs, inputs, pool_bytes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,D,R,il,bits", [
    (orc.BF16, 128, 128, False, 0), (orc.F16, 128, 64, True, 0), (orc.BF16, 72, 48, False, 0), (orc.F32, 64, 32, True, 0),
    (orc.BF16, 128, 128, False, 8), (orc.F16, 128, 64, True, 4), (orc.F32, 64, 32, True, 8), (orc.F16, 96, 96, True, 8)])
@pytest.mark.parametrize("T", [1, 50, 1301, 5000])  # one token a CTA, and four from 8 tokens an SM on
def test_same_bits_in_place(cuda, dt, D, R, il, bits, T):
    H, G, bs = 2, 4, 16
    g, qkv, pos = inputs(T, H, H * G, D, dt, 51)
    slots = torch.randperm(-(-T // bs) * bs, generator=g, device="cuda")[:T].to(torch.int32)
    rope = rmlx_kv.Rope(freqs(R), R, interleaved=il)
    width = qkv.shape[1] * D
    pools, rows = [], []
    for in_place in (False, True):
        pool = rmlx_kv.KVPool(1, H, D, bs, -(-T // bs), dtype=dt, quant_bits=bits, group_size=32, meta_dtype=orc.F32)
        work = qkv.clone()
        q, k, v = work.split([H * G, H, H], 1)
        out = q if in_place else torch.empty(T, H * G, D, dtype=TORCH[dt], device="cuda")
        pool.append_rope(0, k, v, slots, T, pos, rope, q=q, q_out=out, q_heads=H * G, token_stride=width,
                         q_token_stride=width)
        assert pool.check() == 0
        assert torch.equal(work[:, H * G:], qkv[:, H * G:])
        pools.append(pool_bytes(pool).clone())
        rows.append(out.contiguous().view(torch.uint8))
    assert torch.equal(*rows) and torch.equal(*pools)


def test_in_place_strides(cuda):
    """q_out = q takes q's strides; other ones, which would write a row over one that is still to be read, are refused."""
    T, H, G, D, dt = 30, 1, 4, 64, orc.F16
    g, qkv, pos = inputs(T, H, H * G, D, dt, 52)
    pool = rmlx_kv.KVPool(1, H, D, 16, 2, dtype=dt)
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    rope = rmlx_kv.Rope(freqs(D), D)
    q, k, v = qkv.split([H * G, H, H], 1)
    width = qkv.shape[1] * D
    call = dict(q=q, q_out=q, q_heads=H * G, token_stride=width, q_token_stride=width)
    before = qkv.clone()
    for kw in (dict(q_out_token_stride=H * G * D), dict(q_out_head_stride=2 * D), dict(q_out_token_stride=0)):
        with pytest.raises(rmlx_kv.RmlxError) as e:
            pool.append_rope(0, k, v, slots, T, pos, rope, **call, **kw)
        assert e.value.status == 5
    assert torch.equal(qkv, before)
    want = torch.empty(T, H * G, D, dtype=TORCH[dt], device="cuda")
    pool.append_rope(0, k, v, slots, T, pos, rope, **{**call, "q_out": want})
    pool.append_rope(0, k, v, slots, T, pos, rope, **call)
    assert pool.check() == 0
    assert torch.equal(q, want) and torch.equal(qkv[:, H * G:], before[:, H * G:])
    # one token: strides between tokens mean nothing
    pool.append_rope(0, k, v, slots, 1, pos, rope, **{**call, "q_out_token_stride": 8})
    assert pool.check() == 0

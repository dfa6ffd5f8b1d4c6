"""Bounded waits of the chunk attention: one that runs out ends the launch with bit 32 and leaves the GPU as it was.

Rows that are computed again keep a CTA's other warps waiting while they take their time (here some tens of
milliseconds: about 100 ns a row and key, 32 rows a warp, up to 28,000 keys), and all of it ends by itself.
"""
import pytest
import torch

import oracle as orc
import rmlx_kv
from test_gpu_append_rope import TORCH
from test_gpu_chunk_attention import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs,bits", [(16, 0), (5, 0), (16, 8)])  # TMA, rows loaded one by one, bulk copies
def test_a_wait_that_runs_out(cuda, bs, bits):
    H, G, D, dt, n, L = 8, 4, 128, orc.BF16, 512, 65536
    g = torch.Generator("cuda").manual_seed(41)
    N = -(-L // bs)
    pool = rmlx_kv.KVPool(1, H, D, bs, N, dtype=dt, quant_bits=bits, group_size=64, meta_dtype=orc.F16)
    k, v = (torch.randn(L, H, D, generator=g, device="cuda").to(TORCH[dt]) for _ in range(2))
    slots = torch.arange(L, device="cuda", dtype=torch.int32)
    pool.append(k, v, slots, L)
    bt = torch.arange(N, dtype=torch.int32, device="cuda")
    q = torch.randn(n, H * G, D, generator=g, device="cuda").to(TORCH[dt])
    ws = torch.empty(pool.chunk_attention_workspace_size(G), dtype=torch.uint8, device="cuda")

    def call():
        out = torch.full_like(q, 3.0)
        pool.chunk_attention(0, q, G, bt, N, dev([n]), dev([L]), 1, n, D ** -0.5, out, ws)
        return out, pool.check()

    clean, status = call()
    assert status == 0 and torch.isfinite(clean).all()
    at = slots[L - n:L - n + 1]  # a row that every token sees: all are NaN, and are computed again
    nan = torch.full_like(v[:1], float("nan"))
    pool.append(k[L - n:L - n + 1].contiguous(), nan, at, 1)
    pool.set_wait_limit(0.001)
    for _ in range(2):
        assert call()[1] == 32
    pool.set_wait_limit(30)
    out, status = call()
    assert status == 0 and torch.isnan(out).all()
    pool.append(k[L - n:L - n + 1].contiguous(), v[L - n:L - n + 1].contiguous(), at, 1)
    out, status = call()
    assert status == 0 and torch.equal(out.view(torch.int16), clean.view(torch.int16))


def test_refused_limits(cuda):
    pool = rmlx_kv.KVPool(1, 1, 64, 16, 2, dtype=orc.F16)
    for seconds in (0.0, -1.0, float("nan"), 1e7):
        with pytest.raises(rmlx_kv.RmlxError) as e:
            pool.set_wait_limit(seconds)
        assert e.value.status == 5
    pool.set_wait_limit(1e6)

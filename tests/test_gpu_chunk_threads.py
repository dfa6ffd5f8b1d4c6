"""First calls of the chunk attention on a new pool from several threads at once, each with its stream and workspace."""
import threading

import pytest
import torch

import oracle as orc
import rmlx_kv
from test_gpu_append_rope import TORCH
from test_gpu_chunk_attention import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [0, 8])
def test_first_calls_at_once(cuda, bits):
    H, G, D, bs, dt, n, L, threads = 2, 4, 64, 16, orc.F16, 9, 80, 8
    g = torch.Generator("cuda").manual_seed(61)
    k, v = (torch.randn(L, H, D, generator=g, device="cuda").to(TORCH[dt]) for _ in range(2))
    q = torch.randn(n, H * G, D, generator=g, device="cuda").to(TORCH[dt])
    bt = torch.arange(L // bs, dtype=torch.int32, device="cuda")
    slots = torch.arange(L, device="cuda", dtype=torch.int32)
    q_lens, lens = dev([n]), dev([L])
    streams = [torch.cuda.Stream() for _ in range(threads)]
    outs = [torch.empty_like(q) for _ in range(threads)]
    first = None
    for _ in range(25):
        pool = rmlx_kv.KVPool(1, H, D, bs, L // bs, dtype=dt, quant_bits=bits, group_size=32, meta_dtype=orc.F16)
        pool.append(k, v, slots, L)
        size = pool.chunk_attention_workspace_size(G)
        spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(threads)]
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        gate, errors = threading.Barrier(threads), []

        def call(i):
            gate.wait()
            try:
                pool.chunk_attention(0, q, G, bt, L // bs, q_lens, lens, 1, n, D ** -0.5, outs[i], spaces[i], stream=streams[i])
            except Exception as e:  # noqa: BLE001 - reported below
                errors.append(e)

        ts = [threading.Thread(target=call, args=(i,)) for i in range(threads)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
        torch.cuda.synchronize()
        assert not errors and pool.check() == 0
        first = outs[0].clone() if first is None else first
        assert torch.isfinite(first).all()
        for o in outs:
            assert torch.equal(o.view(torch.int16), first.view(torch.int16))

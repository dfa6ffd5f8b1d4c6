"""Workloads of the paged pool's prompt-side operators: the append with position rotation
(KVPool.append_rope) and the attention of a chunk of new tokens over the paged cache
(KVPool.chunk_attention), alone and as a serving step runs them together.

`run` computes a case with elementary torch operations in f32 (angles in f64), or, with `own` set,
with the package's entry points.  The pool's bytes are laid out as include/rmlx_kv.h states:
[block][layer][K, V][head][tile], a tile being block_size rows (plain) or block_size code rows
followed by block_size rows of (scale, zero) pairs (quantised), padded to 16 bytes.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LAYERS, LAYER = 2, 1  # the pool's layers, and the one that a pass works on
GROUP = 64            # quantisation group, with f16 scale and zero
DEVICE = "cuda"


def _case(name, op, **kw):
    base = dict(dtype="bf16", heads=8, group=4, dim=128, block=16, bits=0, seqs=1, q_lo=1, q_hi=1, ctx_lo=0, ctx_hi=0,
                rotary=128, interleaved=False, axes=1, window=0)
    return {"name": name, "op": op, **base, **kw}


def listed():
    return [
        # one decode step's tokens of a batch of 64: the append at its smallest, launch latency counts
        _case("append decode", "append", seqs=64, ctx_lo=512, ctx_hi=4096),
        # the prompts of a whole prefill batch at once, ragged lengths: a bandwidth-bound append
        _case("append prompts", "append", seqs=16, q_lo=1024, q_hi=4096),
        # a few images' and texts' tokens with (time, height, width) positions, seven queries per key head
        _case("append axes f16", "append", dtype="f16", heads=4, group=7, seqs=3, q_lo=700, q_hi=1500, ctx_hi=100000, axes=3),
        # prompts into an 8-bit pool, read back dequantised as the gather path's next step reads them
        _case("append quant8", "append", bits=8, seqs=8, q_lo=512, q_hi=2048),
        # five drafted tokens per sequence verified over cached contexts: every cached byte is read once
        _case("attend verify", "attend", seqs=64, q_lo=5, q_hi=5, ctx_lo=512, ctx_hi=4096),
        # one long prompt with nothing cached: a compute-bound triangle
        _case("attend prompt", "attend", seqs=1, q_lo=8192, q_hi=8192),
        # prefill chunks of ragged sizes over cached prefixes
        _case("attend chunks", "attend", seqs=16, q_lo=100, q_hi=512, ctx_lo=512, ctx_hi=4096),
        # one key head's shard of a larger model over long contexts
        _case("attend shard f16", "attend", dtype="f16", heads=1, group=8, seqs=4, q_lo=64, q_hi=128, ctx_lo=2048, ctx_hi=32768),
        # chunks over 8-bit pools
        _case("attend quant8", "attend", bits=8, seqs=8, q_lo=129, q_hi=384, ctx_lo=1024, ctx_hi=8192),
        # a few tokens per sequence over 4-bit pools
        _case("attend quant4", "attend", bits=4, seqs=32, q_lo=1, q_hi=16, ctx_lo=1024, ctx_hi=8192),
        # the smallest step: a few short turns of a small model, append and attention together
        _case("step turns f16", "step", dtype="f16", heads=4, group=2, dim=64, rotary=32, interleaved=True, seqs=4, q_lo=1, q_hi=37, ctx_hi=100),
        # a sliding-window model's chunks, append and attention together
        _case("step window", "step", seqs=2, q_lo=1024, q_hi=2048, ctx_lo=2048, ctx_hi=6000, window=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["append", "append", "attend", "attend", "step"])
        dim = rng.choice([64, 128, 128])
        c = _case("", op, dtype=rng.choice(["bf16", "bf16", "f16"]), heads=rng.choice([1, 2, 4, 8]), group=rng.choice([1, 2, 4, 4, 5, 8]),
                  dim=dim, block=rng.choice([8, 16, 16, 16, 32, 64]), seqs=_log(rng, 1, 64),
                  rotary=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3)
        del c["name"]
        q = _log(rng, 1, 8192)
        c["q_lo"], c["q_hi"] = max(1, int(q * rng.uniform(0.3, 1.0))), q
        if op == "append":
            c["bits"] = rng.choice([0, 0, 8])
            c["axes"] = rng.choice([1, 1, 3])
            c["ctx_hi"] = 0 if c["bits"] else _log(rng, 1, 100000)
        else:
            ctx = _log(rng, 1, 32768)
            c["ctx_lo"], c["ctx_hi"] = int(ctx * rng.uniform(0.1, 1.0)), ctx
            c["bits"] = rng.choice([0, 0, 8, 4]) if op == "attend" else 0
            c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        q_lens, ctx = _lens(c)
        padded = c["seqs"] * c["heads"] * c["group"] * max(q_lens) * max(a + b for a, b in zip(q_lens, ctx))
        w = work(c)
        if w["bytes"] <= 8e8 and w["flops"] <= 5e11 and (op == "append" or padded <= 1.5e9):
            return c


def _lens(c):
    """The case's chunk lengths and the lengths of what each sequence had before."""
    rng = random.Random("%(seqs)d %(q_lo)d %(q_hi)d %(ctx_lo)d %(ctx_hi)d" % c)
    return [rng.randint(c["q_lo"], c["q_hi"]) for _ in range(c["seqs"])], [rng.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["seqs"])]


def _row_bytes(c):
    """Bytes of a stored row and of its (scale, zero) pairs."""
    if not c["bits"]:
        return c["dim"] * torch.finfo(DTYPES[c["dtype"]]).bits // 8, 0
    return c["dim"] * c["bits"] // 8, c["dim"] // GROUP * 4


def _visible(c):
    """(query, key) pairs that the masks leave, and the cached rows that some query sees."""
    pairs = rows = 0
    for n, before in zip(*_lens(c)):
        if c["window"]:
            seen = [min(before + i + 1, c["window"]) for i in range(n)]
            pairs += sum(seen)
            rows += min(before + n, c["window"] + n - 1)
        else:
            pairs += n * before + n * (n + 1) // 2
            rows += before + n
    return pairs, rows


def work(case):
    c = case
    es = torch.finfo(DTYPES[c["dtype"]]).bits // 8
    row, meta = _row_bytes(c)
    tokens, qh = sum(_lens(c)[0]), c["heads"] * c["group"]
    total = flops = 0
    if c["op"] in ("append", "step"):
        total += tokens * (2 * qh + 2 * c["heads"]) * c["dim"] * es + tokens * 2 * c["heads"] * (row + meta) + tokens * 4 * (1 + c["axes"])
        flops += tokens * (qh + c["heads"]) * c["rotary"] * 3
        if c["bits"]:
            total += tokens * 2 * c["heads"] * (row + meta + c["dim"] * es)  # the gather of the dequantised rows
    if c["op"] in ("attend", "step"):
        pairs, rows = _visible(c)
        total += 2 * tokens * qh * c["dim"] * es + 2 * rows * c["heads"] * (row + meta)
        flops += 4 * c["dim"] * qh * pairs
    return {"bytes": total, "flops": flops}


class _PoolBytes:
    """A KVPool's device memory for torch; keeps the pool alive as long as a tensor looks at it."""

    def __init__(self, pool):
        self.pool = pool
        self.__cuda_array_interface__ = {"shape": (pool.layout.bytes,), "typestr": "|u1", "data": (pool.layout.base, False), "version": 3}


def _quantise(x, bits):
    """Rows [..., dim] in f32 as codes and the (scale, zero) of each group."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = torch.where(hi == lo, torch.ones_like(lo), (hi - lo) / (2 ** bits - 1))
    u = (g - lo) / scale
    codes = (u.floor() + (u - u.floor() >= 0.5)).clamp(0, 2 ** bits - 1).to(torch.uint8).flatten(-2)
    if bits == 4:
        codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return codes, torch.cat([scale, lo], -1).to(torch.float16).flatten(-2)


def _inputs(case, seed):
    """Everything but the pool's handle: the same for a plain pass and for the package's."""
    c = case
    gen = torch.Generator(DEVICE).manual_seed(int(seed) * 7919 + 17)
    dt, es = DTYPES[c["dtype"]], torch.finfo(DTYPES[c["dtype"]]).bits // 8
    q_lens, before = _lens(c)
    if c["op"] == "append":  # the pool holds the blocks that the new rows go to
        base = [b // c["block"] * c["block"] for b in before]
    else:
        base = [0] * len(before)
    ends = [b - z + n for b, z, n in zip(before, base, q_lens)]
    need = [-(-e // c["block"]) for e in ends]
    blocks = sum(need)
    ids = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
    s = {"case": c, "tokens": sum(q_lens), "need": need}
    dev = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=DEVICE)  # noqa: E731
    s["q_lens"], s["seq_lens"] = dev(q_lens), dev(ends)
    first = dev([sum(need[:i]) for i in range(len(need))], torch.int64)
    width = max(need)
    col = torch.arange(width, device=DEVICE)
    s["tables"] = torch.where(col[None] < dev(need)[:, None], ids[(first[:, None] + col).clamp(max=blocks - 1)], torch.zeros_like(ids[:1])).contiguous()
    # each new token's sequence, its place among the chunk's tokens and in the sequence, and its slot
    s["seq_of"] = torch.repeat_interleave(torch.arange(len(q_lens), device=DEVICE), dev(q_lens, torch.int64), output_size=s["tokens"])
    start = dev([sum(q_lens[:i]) for i in range(len(q_lens))], torch.int64)
    s["nth"] = torch.arange(s["tokens"], device=DEVICE) - start[s["seq_of"]]
    place = s["nth"] + (dev(before) - dev(base))[s["seq_of"]]
    s["slots"] = (s["tables"][s["seq_of"], place // c["block"]] * c["block"] + place % c["block"]).to(torch.int32)
    pos = (s["nth"] + dev(before, torch.int64)[s["seq_of"]]).to(torch.int32)
    if c["axes"] > 1:  # images' rows and columns beside the time axis
        side = torch.randint(0, 64, (c["axes"] - 1, s["tokens"]), generator=gen, device=DEVICE, dtype=torch.int32)
        pos = torch.cat([pos[None], pos[None] + side])
    s["positions"] = pos.reshape(c["axes"], -1).contiguous()
    half = c["rotary"] // 2
    s["inv_freq"] = (500000.0 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)).float()
    s["pair_axis"] = (torch.arange(half, device=DEVICE) * c["axes"] // half).to(torch.int32)
    # new rows as one projection writes them: [token][query heads, key heads, value heads][dim]
    qh = c["heads"] * c["group"]
    s["qkv"] = torch.randn(s["tokens"], qh + 2 * c["heads"], c["dim"], generator=gen, device=DEVICE, dtype=torch.float32).to(dt)
    row, meta = _row_bytes(c)
    tile = -(-c["block"] * (row + meta) // 16) * 16
    shape = (blocks, LAYERS, 2, c["heads"])
    if c["op"] == "append":
        s["bytes"] = torch.zeros(*shape, tile, dtype=torch.uint8, device=DEVICE)
    elif not c["bits"]:
        s["bytes"] = torch.randn(*shape, c["block"] * c["dim"], generator=gen, device=DEVICE, dtype=torch.float32).to(dt).view(torch.uint8)
    else:
        x = torch.randn(*shape, c["block"], c["dim"], generator=gen, device=DEVICE)
        x = torch.where(torch.rand(x.shape, generator=gen, device=DEVICE) < 0.01, 8 * x, x)
        codes, sz = _quantise(x, c["bits"])
        s["bytes"] = torch.cat([codes.flatten(-2), sz.flatten(-2).view(torch.uint8)], -1).contiguous()
    if c["op"] == "append" and c["bits"]:
        # rows of a gather of whole sequences, [sequence][head][token]: which token, which head
        key = (s["seq_of"][:, None] * c["heads"] + torch.arange(c["heads"], device=DEVICE)[None]).t().reshape(-1)
        order = torch.argsort(key, stable=True)
        s["rows"] = (order % s["tokens"], order // s["tokens"])
        s["gathered"] = [torch.zeros(s["tokens"] * c["heads"], c["dim"], dtype=dt, device=DEVICE) for _ in range(2)]
    s["scale"] = c["dim"] ** -0.5
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    c = case
    if own:
        at = os.path.join(os.getcwd(), "rmlx-serve_b200")
        if at not in sys.path:
            sys.path.insert(1, at)
        import rmlx_kv
        kind = {"bf16": rmlx_kv.BF16, "f16": rmlx_kv.F16, "f32": rmlx_kv.F32}[c["dtype"]]
        pool = rmlx_kv.KVPool(LAYERS, c["heads"], c["dim"], c["block"], sum(s["need"]), dtype=kind, quant_bits=c["bits"], group_size=GROUP, meta_dtype=rmlx_kv.F16)
        mine = torch.as_tensor(_PoolBytes(pool), device=DEVICE).view(s["bytes"].shape)
        mine.copy_(s["bytes"])
        s["bytes"], s["pool"] = mine, pool
        s["rope"] = rmlx_kv.Rope(s["inv_freq"], c["rotary"], interleaved=c["interleaved"], pair_axis=s["pair_axis"] if c["axes"] > 1 else None, num_axes=c["axes"])
        qh = c["heads"] * c["group"]
        s["q_out"] = torch.empty(s["tokens"], qh, c["dim"], dtype=DTYPES[c["dtype"]], device=DEVICE)
        s["out"] = torch.empty_like(s["q_out"])
        if c["op"] != "append":
            s["workspace"] = torch.empty(pool.chunk_attention_workspace_size(c["group"]), dtype=torch.uint8, device=DEVICE)
    return s


def _own_append(s):
    c = s["case"]
    qh, width = c["heads"] * c["group"], s["qkv"].shape[1] * c["dim"]
    q, k, v = s["qkv"].split([qh, c["heads"], c["heads"]], 1)
    s["pool"].append_rope(LAYER, k, v, s["slots"], s["tokens"], s["positions"], s["rope"], q=q, q_out=s["q_out"], q_heads=qh,
                          token_stride=width, head_stride=c["dim"], q_token_stride=width, q_head_stride=c["dim"])


def _own_attend(s, q, token_stride):
    c = s["case"]
    s["pool"].chunk_attention(LAYER, q, c["group"], s["tables"], s["tables"].shape[1], s["q_lens"], s["seq_lens"], c["seqs"], s["tokens"], s["scale"],
                              s["out"], s["workspace"], window=c["window"], q_token_stride=token_stride)


def _run_own(s):
    c = s["case"]
    if c["op"] == "attend":
        _own_attend(s, s["qkv"], s["qkv"].shape[1] * c["dim"])
        return s["out"]
    _own_append(s)
    if c["op"] == "step":
        _own_attend(s, s["q_out"], s["q_out"].shape[1] * c["dim"])
        return {"q": s["q_out"], "out": s["out"], "pool": s["bytes"].view(DTYPES[c["dtype"]])}
    if c["bits"]:
        s["pool"].gather(LAYER, s["tables"], s["tables"].shape[1], s["seq_lens"], c["seqs"], *s["gathered"])
        return {"q": s["q_out"], "k": s["gathered"][0], "v": s["gathered"][1]}
    return {"q": s["q_out"], "pool": s["bytes"].view(DTYPES[c["dtype"]])}


def _rotate(x, s):
    """Rows [tokens, heads, dim] in f32 with their first `rotary` dims rotated."""
    c = s["case"]
    r = c["rotary"]
    angle = s["positions"][s["pair_axis"].long()].t().double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if c["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., r:]], -1)
    a, b = x[..., : r // 2], x[..., r // 2 : r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)


def _plain_append(s):
    c = s["case"]
    dt, qh = DTYPES[c["dtype"]], c["heads"] * c["group"]
    x = s["qkv"].float()
    q, k, v = _rotate(x[:, :qh], s), _rotate(x[:, qh : qh + c["heads"]], s), x[:, qh + c["heads"] :]
    blk, off = s["slots"].long() // c["block"], s["slots"].long() % c["block"]
    kv = torch.stack([k, v], 1)  # [token][K, V][head][dim]
    if not c["bits"]:
        rows = s["bytes"].view(dt).unflatten(-1, (c["block"], c["dim"]))
        rows[blk, LAYER, :, :, off] = kv.to(dt)
        return q.to(dt)
    row, meta = _row_bytes(c)
    codes, sz = _quantise(kv, c["bits"])
    n = c["block"] * row
    s["bytes"][..., :n].unflatten(-1, (c["block"], row))[blk, LAYER, :, :, off] = codes
    s["bytes"][..., n : n + c["block"] * meta].unflatten(-1, (c["block"], meta))[blk, LAYER, :, :, off] = sz.view(torch.uint8)
    return q.to(dt)


def _tile_rows(s):
    """The layer's stored rows, [block][K, V][head][slot][dim], in f32: of a quantised pool, code * scale + zero."""
    c = s["case"]
    b = s["bytes"][:, LAYER]
    if not c["bits"]:
        return b.view(DTYPES[c["dtype"]]).unflatten(-1, (c["block"], c["dim"])).float()
    row, meta = _row_bytes(c)
    codes = b[..., : c["block"] * row].unflatten(-1, (c["block"], row))
    if c["bits"] == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    at = c["block"] * row
    sz = b[..., at : at + c["block"] * meta].contiguous().view(torch.float16).float().unflatten(-1, (c["block"], c["dim"] // GROUP, 2))
    return (codes.float().unflatten(-1, (-1, GROUP)) * sz[..., :1] + sz[..., 1:]).flatten(-2)


def _plain_attend(s, q):
    """Every sequence padded to the longest, [sequence][head][query in the group, token][key]."""
    c = s["case"]
    rows = _tile_rows(s)
    n, longest = max(_lens(c)[0]), s["tables"].shape[1] * c["block"]
    kv = rows[s["tables"].long()]  # [seq][table column][K, V][head][slot][dim]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, c["seqs"], c["heads"], longest, c["dim"])
    pad = torch.zeros(c["seqs"], n, c["heads"], c["group"], c["dim"], device=q.device)
    pad[s["seq_of"], s["nth"]] = q.float().unflatten(1, (c["heads"], c["group"]))
    x = pad.permute(0, 2, 3, 1, 4).reshape(c["seqs"], c["heads"], c["group"] * n, c["dim"])
    scores = (x @ kv[0].transpose(-1, -2)).mul_(s["scale"]).unflatten(2, (c["group"], n))
    at = (s["seq_lens"] - s["q_lens"])[:, None] + torch.arange(n, device=q.device)  # a token's place in its sequence
    key = torch.arange(longest, device=q.device)
    hidden = key > at[..., None]
    if c["window"]:
        hidden = hidden | (key <= at[..., None] - c["window"])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    # rows behind a sequence's end are not part of it: whatever lies there is weighed with nothing
    v = kv[1].masked_fill((key >= s["seq_lens"][:, None])[:, None, :, None], 0.0)
    o = (p.flatten(2, 3) @ v).unflatten(2, (c["group"], n)) / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4)[s["seq_of"], s["nth"]].flatten(1, 2).to(DTYPES[c["dtype"]])


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s)
    if c["op"] == "attend":
        return _plain_attend(s, s["qkv"][:, : c["heads"] * c["group"]])
    q = _plain_append(s)
    if c["op"] == "step":
        return {"q": q, "out": _plain_attend(s, q), "pool": s["bytes"].view(DTYPES[c["dtype"]])}
    if c["bits"]:
        rows = _tile_rows(s)
        blk, off = s["slots"].long() // c["block"], s["slots"].long() % c["block"]
        token, head = s["rows"]
        got = rows[blk[token], :, head, off[token]].to(DTYPES[c["dtype"]])
        return {"q": q, "k": got[:, 0], "v": got[:, 1]}
    return {"q": q, "pool": s["bytes"].view(DTYPES[c["dtype"]])}


def exact(case, seed):
    s, c = _inputs(case, seed), case
    qh, H, D, bs = c["heads"] * c["group"], c["heads"], c["dim"], c["block"]
    q_lens, lens = s["q_lens"].tolist(), s["seq_lens"].tolist()
    result = {}
    x = s["qkv"].double()
    q = x[:, :qh]
    row, meta = _row_bytes(c)
    stored = s["bytes"].view(DTYPES[c["dtype"]]).double().view(-1, LAYERS, 2, H, bs, D) if not c["bits"] else None
    if c["op"] != "attend":
        # each pair as a complex number, turned by its angle
        half = c["rotary"] // 2
        turn = torch.stack([s["positions"][int(a)].double() * f for a, f in zip(s["pair_axis"].tolist(), s["inv_freq"].double())], 1)
        turn = torch.polar(torch.ones_like(turn), turn)[:, None]
        first = torch.arange(half, device=x.device) * (2 if c["interleaved"] else 1)
        second = first + (1 if c["interleaved"] else half)
        k = x[:, qh : qh + H].clone()
        q = q.clone()
        for y in (q, k):
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
        result["q"] = q
        v = x[:, qh + H :]
        slots = s["slots"].tolist()
        if c["bits"]:
            out = []
            for rows in (k, v):
                g = rows.reshape(s["tokens"], H, D // GROUP, GROUP)
                lo = g.min(-1).values
                step = (g.max(-1).values - lo) / (2 ** c["bits"] - 1)
                step[step == 0] = 1.0
                code = torch.clamp(torch.floor((g - lo[..., None]) / step[..., None] + 0.5), 0, 2 ** c["bits"] - 1)
                value = (code * step.half().double()[..., None] + lo.half().double()[..., None]).reshape(s["tokens"], H, D)
                at, parts = 0, []
                for n in q_lens:
                    parts.append(value[at : at + n].transpose(0, 1).reshape(n * H, D))
                    at += n
                out.append(torch.cat(parts))
            result["k"], result["v"] = out
            return result
        where = torch.tensor(slots, device=x.device)
        for which, rows in ((0, k), (1, v)):
            flat = stored[:, LAYER, which].permute(0, 2, 1, 3).reshape(-1, H, D)
            flat[where] = rows
            stored[:, LAYER, which] = flat.view(-1, bs, H, D).permute(0, 2, 1, 3)
        result["pool"] = stored.view(*s["bytes"].shape[:-1], -1)
        if c["op"] == "append":
            return result
        # the attention's exact value is that of the rows before their rounding
    out = torch.zeros(s["tokens"], qh, D, dtype=torch.float64, device=x.device)
    at = 0
    for i, (n, total) in enumerate(zip(q_lens, lens)):
        ids = s["tables"][i, : -(-total // bs)].long()
        for h in range(H):
            if c["bits"]:
                pair = []
                for which in (0, 1):
                    raw = s["bytes"][ids, LAYER, which, h]
                    codes = raw[:, : bs * row].reshape(-1, row)
                    if c["bits"] == 4:
                        codes = torch.stack((codes % 16, codes // 16), 2).reshape(-1, D)
                    sz = raw[:, bs * row : bs * (row + meta)].contiguous().view(torch.float16).double().view(-1, D // GROUP, 2)
                    pair.append((codes.double().view(-1, D // GROUP, GROUP) * sz[..., 0:1] + sz[..., 1:2]).view(-1, D)[:total])
            else:
                pair = [stored[ids, LAYER, which, h].reshape(-1, D)[:total] for which in (0, 1)]
            place = torch.arange(total - n, total, device=x.device)[:, None]
            key = torch.arange(total, device=x.device)[None]
            seen = (key <= place) & ((key > place - c["window"]) if c["window"] else True)
            for j in range(h * c["group"], (h + 1) * c["group"]):
                w = torch.softmax(torch.where(seen, q[at : at + n, j] @ pair[0].t() * D ** -0.5, -math.inf), -1)
                out[at : at + n, j] = w @ pair[1]
        at += n
    if c["op"] == "attend":
        return out
    result["out"] = out
    return result

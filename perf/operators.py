"""Measured cases of the bounded-cache operators: attention over a sliding window
with sink tokens (single tokens and prompt chunks), rotary embedding with the
K/V append, and block copies of the paged cache.

``run`` computes a case either in plain torch operations or, with ``own`` set,
through this package's entry points; ``exact`` computes it in 64 bits from the
definition, one sequence at a time.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}


def listed():
    """The cases: each operator from its smallest calls to its largest."""
    return [
        # One short conversation: every block visible, the call is its latency.
        dict(name="decode_1_short", op="decode", dtype="bf16", batch=1, heads=14, kv_heads=2,
             head_dim=64, block=16, window=256, sinks=4, min_len=77, max_len=77, shape_seed=1),
        # A served batch of conversations of 1 to 16384 tokens, four sink tokens.
        dict(name="decode_64_d64", op="decode", dtype="bf16", batch=64, heads=14, kv_heads=2,
             head_dim=64, block=16, window=1024, sinks=4, min_len=1, max_len=16384, shape_seed=2),
        # A full batch with a wide window on the wider heads: the most cache read.
        dict(name="decode_256_d128", op="decode", dtype="bf16", batch=256, heads=28, kv_heads=4,
             head_dim=128, block=16, window=4096, sinks=16, min_len=512, max_len=32768,
             shape_seed=3),
        # A 32-bit cache (parity runs), an odd window and no sinks, larger blocks.
        dict(name="decode_24_f32", op="decode", dtype="f32", batch=24, heads=8, kv_heads=2,
             head_dim=64, block=32, window=777, sinks=0, min_len=1, max_len=4096, shape_seed=4),
        # A short question appended to a long conversation.
        dict(name="chunk_1x33", op="chunk", dtype="bf16", chunks=1, min_chunk=33, max_chunk=33,
             max_prior=6000, heads=14, kv_heads=2, head_dim=64, block=16, window=1024, sinks=4,
             shape_seed=5),
        # The mixed step's prompt chunks: 8 x 512 tokens behind cached prefixes.
        dict(name="chunk_8x512_d64", op="chunk", dtype="bf16", chunks=8, min_chunk=512,
             max_chunk=512, max_prior=4096, heads=14, kv_heads=2, head_dim=64, block=16,
             window=1024, sinks=4, shape_seed=6),
        # Ragged long prompts on the wider heads, a window that spans several chunks.
        dict(name="chunk_6_ragged_d128", op="chunk", dtype="bf16", chunks=6, min_chunk=100,
             max_chunk=2048, max_prior=16384, heads=28, kv_heads=4, head_dim=128, block=16,
             window=4096, sinks=16, shape_seed=7),
        # One decoded token, half layout over the whole head.
        dict(name="rotary_1", op="rotary", dtype="bf16", tokens=1, heads=14, kv_heads=2,
             head_dim=64, rotary_dim=64, block=16, interleaved=False, scaling="none",
             max_position=32768),
        # A prompt step of 4096 tokens, interleaved pairs over half of the head, positions
        # up to a million with scaled frequencies.
        dict(name="rotary_4096_partial", op="rotary", dtype="bf16", tokens=4096, heads=28,
             kv_heads=4, head_dim=128, rotary_dim=64, block=16, interleaved=True, scaling="yarn",
             max_position=1000000),
        # A 32-bit step of odd size.
        dict(name="rotary_333_f32", op="rotary", dtype="f32", tokens=333, heads=8, kv_heads=2,
             head_dim=64, rotary_dim=64, block=16, interleaved=False, scaling="linear",
             max_position=131072),
        # Forking: three children copy the last block of one conversation, all layers.
        dict(name="pages_fork_3", op="pages", dtype="bf16", layers=24, kv_heads=2, head_dim=64,
             block=16, blocks=512, pairs=3, fork=True),
        # Compacting a fragmented pool: 1024 blocks move, all layers.
        dict(name="pages_compact_1024", op="pages", dtype="bf16", layers=24, kv_heads=2,
             head_dim=64, block=16, blocks=2560, pairs=1024, fork=False),
    ]


# The most work a drawn case of each operator may have: its largest listed case's.
_LARGEST = {"decode": "decode_256_d128", "chunk": "chunk_6_ragged_d128",
            "rotary": "rotary_4096_partial", "pages": "pages_compact_1024"}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges, without a name."""
    limits = {c["name"]: work(c) for c in listed()}
    while True:
        case = _draw(rng)
        cost, most = work(case), limits[_LARGEST[case["op"]]]
        if cost["bytes"] <= most["bytes"] and cost["flops"] <= most["flops"]:
            return case


def _draw(rng):
    op = rng.choice(["decode", "decode", "chunk", "chunk", "rotary", "pages"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 16])
    head_dim = rng.choice([64, 128])
    block = rng.choice([16, 16, 16, 32])
    if op == "decode":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        max_len = _log_int(rng, 16, 32768)
        return dict(op=op, dtype=dtype, batch=_log_int(rng, 1, 256), heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim, block=block,
                    window=_log_int(rng, 16, 8192), sinks=rng.choice([0, 1, 4, 16, 40]),
                    min_len=rng.randint(1, max_len), max_len=max_len,
                    shape_seed=rng.randint(0, 1 << 30))
    if op == "chunk":
        max_chunk = _log_int(rng, 1, 2048)
        return dict(op=op, dtype="bf16", chunks=rng.randint(1, 12), min_chunk=rng.randint(1, max_chunk),
                    max_chunk=max_chunk, max_prior=_log_int(rng, 1, 16384), heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim, block=block,
                    window=_log_int(rng, 16, 8192), sinks=rng.choice([0, 1, 4, 16, 40]),
                    shape_seed=rng.randint(0, 1 << 30))
    if op == "rotary":
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), tokens=_log_int(rng, 1, 4096),
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4]),
                    block=block, interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "yarn"]),
                    max_position=_log_int(rng, 4096, 1000000))
    blocks = _log_int(rng, 64, 4096)
    return dict(op=op, dtype=rng.choice(["bf16", "f32"]), layers=rng.randint(1, 32),
                kv_heads=rng.choice([1, 2, 4, 8]), head_dim=head_dim, block=block, blocks=blocks,
                pairs=_log_int(rng, 1, blocks // 2), fork=rng.random() < 0.5)


# ------------------------------------------------------------------ shapes of a case


def _lengths(case):
    """Decode: the context length of each sequence, log-uniform."""
    r = np.random.RandomState(case["shape_seed"])
    lo, hi = math.log(case["min_len"]), math.log(case["max_len"])
    lens = np.exp(r.uniform(lo, hi, case["batch"])).round().astype(int)
    return np.clip(lens, case["min_len"], case["max_len"]).tolist()


def _chunks(case):
    """Chunk: (new tokens, cached tokens before them) of each chunk."""
    r = np.random.RandomState(case["shape_seed"])
    n = r.randint(case["min_chunk"], case["max_chunk"] + 1, case["chunks"])
    prior = r.randint(0, case["max_prior"] + 1, case["chunks"])
    return [(int(a), int(b)) for a, b in zip(n, prior)]


def _visible(length, window, sinks):
    """Keys that the token at position length - 1 sees."""
    low = max(0, length - window)
    return length - low + min(sinks, low)


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "decode":
        H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
        lens = _lengths(case)
        seen = sum(_visible(n, case["window"], case["sinks"]) for n in lens)
        blocks = sum(-(-_visible(n, case["window"], case["sinks"]) // case["block"]) for n in lens)
        return {"bytes": 2 * seen * Hkv * D * e + 2 * len(lens) * H * D * e + 4 * blocks
                + 4 * len(lens),
                "flops": 4 * H * D * seen}
    if case["op"] == "chunk":
        H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
        keys = products = tokens = 0
        for n, prior in _chunks(case):
            low = max(0, prior + 1 - case["window"])
            keys += prior + n - low + min(case["sinks"], low)
            products += sum(_visible(prior + i + 1, case["window"], case["sinks"])
                            for i in range(n))
            tokens += n
        return {"bytes": 2 * keys * Hkv * D * e + 2 * tokens * H * D * e + 4 * keys // case["block"],
                "flops": 4 * H * D * products}
    if case["op"] == "rotary":
        T, H, Hkv, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        return {"bytes": 2 * T * (H + 2 * Hkv) * D * e + 8 * T + 4 * case["rotary_dim"],
                "flops": 3 * T * (H + Hkv) * case["rotary_dim"]}
    page = case["layers"] * case["kv_heads"] * case["block"] * case["head_dim"] * e
    return {"bytes": 4 * case["pairs"] * page + 8 * case["pairs"], "flops": 0}


# ------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _paged(case, totals, lows, seed):
    """K and V pools, and block tables in which the blocks that no later token sees
    (behind the sinks, before ``lows``) have been freed (-1).  The keys of the sink
    tokens lie along the queries' mean, as sink tokens' do."""
    g = _generator(seed)
    Hkv, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    dtype = _DTYPES[case["dtype"]]
    sink_blocks = -(-case["sinks"] // bs)
    held = []
    for total, low in zip(totals, lows):
        n = -(-total // bs)
        held.append([b for b in range(n) if b < sink_blocks or b >= low // bs])
    used = sum(len(h) for h in held)
    nb = used + 3
    order = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).tolist()
    table = np.full((len(totals), max(-(-t // bs) for t in totals)), -1, dtype=np.int32)
    at, sink_slots = 0, []
    for r, h in enumerate(held):
        table[r, h] = order[at: at + len(h)]
        at += len(h)
        sink_slots += [int(table[r, p // bs]) * bs + p % bs
                       for p in range(min(case["sinks"], totals[r]))]
    shape = (Hkv, nb, bs, D)
    k = torch.randn(shape, generator=g, device="cuda")
    mean = torch.randn((Hkv, 1, D), generator=g, device="cuda")
    if sink_slots:
        idx = torch.tensor(sink_slots, device="cuda")
        flat = k.view(Hkv, nb * bs, D)
        flat[:, idx] += mean
    v = torch.randn(shape, generator=g, device="cuda")
    T = len(totals) if case["op"] == "decode" else sum(n for n, _ in _chunks(case))
    groups = case["heads"] // Hkv
    q = torch.randn((T, Hkv, groups, D), generator=g, device="cuda") + 0.3 * mean.view(1, Hkv, 1, D)
    return dict(case=case, q=q.reshape(T, case["heads"], D).to(dtype), k=k.to(dtype), v=v.to(dtype),
                table=torch.from_numpy(table).cuda(), scale=D ** -0.5,
                lens=torch.tensor(totals, dtype=torch.int32, device="cuda"))


def _inverse_frequencies(case):
    """Rotary frequencies in 64 bits: plain, positions divided by 4, or YaRN's blend
    of the two (a ramp over the pairs that turn 1 to 32 times in 32768 positions)."""
    half = case["rotary_dim"] // 2
    freq = 1e6 ** (-np.arange(half, dtype=np.float64) / half)
    if case["scaling"] == "none":
        return freq, 1.0
    if case["scaling"] == "linear":
        return freq / 4.0, 1.0
    turns = 32768 * freq / (2 * math.pi)
    keep = np.clip((np.log(turns)) / math.log(32.0), 0.0, 1.0)
    return freq * keep + freq / 32.0 * (1.0 - keep), 0.1 * math.log(32.0) + 1.0


def prepare(case, seed):
    if case["op"] == "decode":
        lens = _lengths(case)
        return _paged(case, lens, [max(0, n - case["window"]) for n in lens], seed)
    if case["op"] == "chunk":
        chunks = _chunks(case)
        totals = [n + p for n, p in chunks]
        state = _paged(case, totals, [max(0, p + 1 - case["window"]) for _, p in chunks], seed)
        offsets = np.concatenate([[0], np.cumsum([n for n, _ in chunks])]).astype(np.int32)
        state["cu_q"] = torch.from_numpy(offsets).cuda()
        return state
    g = _generator(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        T, H, Hkv, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        nb = -(-T // case["block"]) + 2
        freq, amplitude = _inverse_frequencies(case)
        return dict(
            case=case, amplitude=amplitude, freq=torch.from_numpy(freq).cuda(),
            qkv=torch.randn((T, (H + 2 * Hkv) * D), generator=g, device="cuda").to(dtype),
            pos=torch.randint(0, case["max_position"], (T,), generator=g, device="cuda",
                              dtype=torch.int32),
            slots=torch.randperm(nb * case["block"], generator=g, device="cuda")[:T].int(),
            k=torch.randn((Hkv, nb, case["block"], D), generator=g, device="cuda").to(dtype),
            v=torch.randn((Hkv, nb, case["block"], D), generator=g, device="cuda").to(dtype))
    shape = (case["layers"], case["kv_heads"], case["blocks"], case["block"], case["head_dim"])
    order = torch.randperm(case["blocks"], generator=g, device="cuda").int()
    n = case["pairs"]
    src = order[:n].clone()
    if case["fork"]:
        src = src[torch.arange(n, device="cuda") // 3]  # three children of each parent
    return dict(case=case, src=src, dst=order[n: 2 * n].clone(),
                k=torch.randn(shape, generator=g, device="cuda").to(dtype),
                v=torch.randn(shape, generator=g, device="cuda").to(dtype))


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return _RUN_OWN[op](state)
    return _RUN_PLAIN[op](state)


def _own_decode(s):
    from batchstream_inference_engine_b200 import ops

    return ops.window_attention_batched(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"],
                                        window=s["case"]["window"], sinks=s["case"]["sinks"])


def _own_chunk(s):
    from batchstream_inference_engine_b200 import ops

    return ops.window_prefill_attention(s["q"], s["k"], s["v"], s["table"], s["cu_q"], s["lens"],
                                        s["scale"], max_query_len=s["case"]["max_chunk"],
                                        window=s["case"]["window"], sinks=s["case"]["sinks"])


def _own_rotary(s):
    from batchstream_inference_engine_b200 import ops

    q = ops.rotary_append(s["qkv"], s["freq"], s["pos"], s["slots"], s["k"], s["v"],
                          s["case"]["heads"], interleaved=s["case"]["interleaved"],
                          amplitude=s["amplitude"])
    return [q, s["k"], s["v"]]


def _own_pages(s):
    from batchstream_inference_engine_b200 import ops

    ops.copy_blocks(s["k"], s["v"], s["src"], s["dst"])
    return [s["k"], s["v"]]


def _softmax(scores, mask):
    """Softmax over the last axis of the entries that ``mask`` keeps."""
    scores = scores.masked_fill(~mask, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_decode(s):
    case = s["case"]
    Hkv, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    B, groups = s["q"].shape[0], case["heads"] // case["kv_heads"]
    lens = s["lens"].long()[:, None]
    low = (lens - case["window"]).clamp(min=0)
    span = min(case["window"], case["max_len"])
    sink = torch.arange(case["sinks"], device="cuda")[None].expand(B, -1)
    recent = low + torch.arange(span, device="cuda")[None]
    pos = torch.cat([sink, recent], 1)
    mask = torch.cat([sink < low, recent < lens], 1)
    safe = torch.where(mask, pos, torch.zeros_like(pos))
    block = torch.gather(s["table"].long(), 1, safe // bs).clamp(min=0)
    slot = block * bs + safe % bs
    q = s["q"].float().view(B, Hkv, groups, D)
    out = torch.empty((B, Hkv, groups, D), device="cuda")
    for h in range(Hkv):
        keys = s["k"][h].reshape(-1, D)[slot].float()
        values = s["v"][h].reshape(-1, D)[slot].float()
        p = _softmax(torch.matmul(q[:, h], keys.transpose(1, 2)) * s["scale"], mask[:, None])
        out[:, h] = torch.matmul(p, values)
    return out.view(B, case["heads"], D).to(s["q"].dtype)


def _plain_chunk(s):
    case = s["case"]
    Hkv, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    groups = case["heads"] // Hkv
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    at = 0
    for r, (n, prior) in enumerate(_chunks(case)):
        low = max(0, prior + 1 - case["window"])
        pos = torch.cat([torch.arange(min(case["sinks"], low), device="cuda"),
                         torch.arange(low, prior + n, device="cuda")])
        mine = prior + torch.arange(n, device="cuda")[:, None]
        mask = (pos <= mine) & ((pos < case["sinks"]) | (pos > mine - case["window"]))
        slot = s["table"][r].long()[pos // bs] * bs + pos % bs
        q = s["q"][at: at + n].float().view(n, Hkv, groups, D)
        for h in range(Hkv):
            keys = s["k"][h].reshape(-1, D)[slot].float()
            values = s["v"][h].reshape(-1, D)[slot].float()
            p = _softmax(torch.matmul(q[:, h].transpose(0, 1), keys.t()) * s["scale"], mask)
            mixed = torch.matmul(p, values).transpose(0, 1)
            out[at: at + n, h * groups: (h + 1) * groups] = mixed.to(out.dtype)
        at += n
    return out


def _plain_rotary(s):
    case = s["case"]
    T, H, Hkv, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    rd = case["rotary_dim"]
    angle = s["pos"].double()[:, None] * s["freq"]
    cos = (angle.cos() * s["amplitude"]).float()[:, None]
    sin = (angle.sin() * s["amplitude"]).float()[:, None]
    x = s["qkv"].view(T, H + 2 * Hkv, D).float()
    head, rest = x[:, : H + Hkv, :rd], x[:, : H + Hkv, rd:]
    if case["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., : rd // 2], head[..., rd // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    turned = torch.cat([turned, rest], -1).to(s["qkv"].dtype)
    slots = s["slots"].long()
    s["k"].view(Hkv, -1, D)[:, slots] = turned[:, H:].transpose(0, 1)
    s["v"].view(Hkv, -1, D)[:, slots] = x[:, H + Hkv:].to(s["v"].dtype).transpose(0, 1)
    return [turned[:, :H].contiguous(), s["k"], s["v"]]


def _plain_pages(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, :, dst] = s["k"][:, :, src]
    s["v"][:, :, dst] = s["v"][:, :, src]
    return [s["k"], s["v"]]


_RUN_OWN = {"decode": _own_decode, "chunk": _own_chunk, "rotary": _own_rotary, "pages": _own_pages}
_RUN_PLAIN = {"decode": _plain_decode, "chunk": _plain_chunk, "rotary": _plain_rotary,
              "pages": _plain_pages}


# ------------------------------------------------------------------ 64 bits


def _attend64(q, keys, values, seen, scale):
    """q [n, H, D] over keys and values [Hkv, L, D], seen [n, L]: 64-bit attention."""
    n, H, D = q.shape
    groups = H // keys.shape[0]
    scores = torch.einsum("nkgd,kld->kgnl", q.double().reshape(n, -1, groups, D), keys) * scale
    scores = torch.where(seen, scores, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
    log_sum = torch.logsumexp(scores, -1, keepdim=True)
    return torch.einsum("kgnl,kld->nkgd", torch.exp(scores - log_sum), values).reshape(n, H, D)


def exact(case, seed):
    """What ``run`` returns, in 64 bits; None for copies, which compute nothing."""
    if case["op"] == "pages":
        return None
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    if case["op"] == "decode":
        spans = [(i, 1, n - 1) for i, n in enumerate(_lengths(case))]
    else:
        spans, at = [], 0
        for n, prior in _chunks(case):
            spans.append((at, n, prior))
            at += n
    bs, W, S = case["block"], case["window"], case["sinks"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, (at, n, prior) in enumerate(spans):
        table = s["table"][r].tolist()
        where = [(p, table[p // bs] * bs + p % bs) for p in range(prior + n)
                 if p < S or p > prior - W]
        position = torch.tensor([p for p, _ in where], device="cuda")
        slot = torch.tensor([x for _, x in where], device="cuda")
        keys = s["k"].flatten(1, 2)[:, slot].double()
        values = s["v"].flatten(1, 2)[:, slot].double()
        for i in range(0, n, 256):  # rows of the chunk, 256 at a time
            m = min(256, n - i)
            token = torch.arange(prior + i, prior + i + m, device="cuda")[:, None]
            distance = token - position
            seen = (distance >= 0) & ((distance < W) | (position < S))
            out[at + i: at + i + m] = _attend64(s["q"][at + i: at + i + m], keys, values, seen,
                                                s["scale"])
    return out


def _exact_rotary(case, s):
    T, H, Hkv, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    rd = case["rotary_dim"]
    x = s["qkv"].double().reshape(T, H + 2 * Hkv, D)
    first = torch.arange(rd // 2, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else rd // 2)
    turn = torch.polar(torch.full((T, 1, rd // 2), s["amplitude"], dtype=torch.float64,
                                  device="cuda"),
                       (s["pos"].double()[:, None] * s["freq"]).reshape(T, 1, rd // 2))
    z = torch.complex(x[:, : H + Hkv, first], x[:, : H + Hkv, second]) * turn
    y = x.clone()
    y[:, : H + Hkv, first] = z.real
    y[:, : H + Hkv, second] = z.imag
    k, v = s["k"].double(), s["v"].double()
    k.flatten(1, 2)[:, s["slots"].long()] = y[:, H: H + Hkv].transpose(0, 1)
    v.flatten(1, 2)[:, s["slots"].long()] = y[:, H + Hkv:].transpose(0, 1)
    return [y[:, :H], k, v]

"""Measured cases of the 4-bit cache and of draft verification: rotary embedding with
the quantising K/V append, attention over the 4-bit cache (single tokens and prompt
chunks), and the verification of drafted tokens against the target's probabilities.

``run`` computes a case either in plain torch operations or, with ``own`` set,
through this package's entry points; ``exact`` computes it in 64 bits from the
definition.

The 4-bit cache: a group is 32 consecutive dims of one token and kv head.  With m the
largest magnitude of a group over 8, rounded up to 4 significant bits, its scale is s = m,
or -m when the largest magnitude is positive; its codes are n = rint(x / s) + 8 in 0 .. 15,
its values s (n - 8).  A block of bs tokens holds bs * D / 2 bytes of codes, then
bs * D / 32 bf16 scales; of 8 dims in 4 bytes, dim 2i is nibble i and dim 2i + 1 nibble
i + 4.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}
_GROUP = 32
_TINY = 2.0 ** -100  # groups whose largest magnitude is below are zeros


def listed():
    """The cases: each operator from its smallest calls to its largest."""
    return [
        # One decoded token: the call is its latency.
        dict(name="append_1", op="append", dtype="bf16", tokens=1, heads=14, kv_heads=2,
             head_dim=64, rotary_dim=64, block=16, interleaved=False, max_position=32768),
        # A prompt step of 4096 tokens on the wider heads.
        dict(name="append_4096_d128", op="append", dtype="bf16", tokens=4096, heads=28, kv_heads=4,
             head_dim=128, rotary_dim=128, block=16, interleaved=False, max_position=1000000),
        # One short conversation.
        dict(name="decode_1_short", op="decode", dtype="bf16", batch=1, heads=14, kv_heads=2,
             head_dim=64, block=16, min_len=77, max_len=77, shape_seed=1),
        # A served batch of conversations of 1 to 16384 tokens.
        dict(name="decode_64_d64", op="decode", dtype="bf16", batch=64, heads=14, kv_heads=2,
             head_dim=64, block=16, min_len=1, max_len=16384, shape_seed=2),
        # A full batch of long conversations on the wider heads: the most cache read.
        dict(name="decode_256_d128", op="decode", dtype="bf16", batch=256, heads=28, kv_heads=4,
             head_dim=128, block=16, min_len=512, max_len=32768, shape_seed=3),
        # 32-bit queries (parity runs), larger blocks.
        dict(name="decode_24_f32", op="decode", dtype="f32", batch=24, heads=8, kv_heads=2,
             head_dim=64, block=32, min_len=1, max_len=4096, shape_seed=4),
        # A drafted step: 64 conversations with a token and four drafts each.
        dict(name="chunk_64x5", op="chunk", dtype="bf16", chunks=64, min_chunk=5, max_chunk=5,
             max_prior=8192, heads=14, kv_heads=2, head_dim=64, block=16, shape_seed=5),
        # The mixed step's prompt chunks: 8 x 512 tokens behind cached prefixes.
        dict(name="chunk_8x512_d64", op="chunk", dtype="bf16", chunks=8, min_chunk=512,
             max_chunk=512, max_prior=4096, heads=14, kv_heads=2, head_dim=64, block=16,
             shape_seed=6),
        # Ragged long prompts on the wider heads.
        dict(name="chunk_6_ragged_d128", op="chunk", dtype="bf16", chunks=6, min_chunk=100,
             max_chunk=2048, max_prior=16384, heads=28, kv_heads=4, head_dim=128, block=16,
             shape_seed=7),
        # One conversation whose four drafts were looked up in its prompt (no probabilities).
        dict(name="verify_1x4", op="verify", dtype="bf16", batch=1, min_drafts=4, max_drafts=4,
             vocab=151936, draft_probs=False, greedy=0.0, shape_seed=8),
        # A served batch with four drafts each from a small model, sampled.
        dict(name="verify_64x4_probs", op="verify", dtype="bf16", batch=64, min_drafts=4,
             max_drafts=4, vocab=151936, draft_probs=True, greedy=0.0, shape_seed=9),
        # A ragged batch, some of it greedy, 32-bit logits of an odd vocabulary.
        dict(name="verify_200_ragged_f32", op="verify", dtype="f32", batch=200, min_drafts=0,
             max_drafts=7, vocab=32003, draft_probs=True, greedy=0.3, shape_seed=10),
    ]


# The most work a drawn case of each operator may have: its largest listed case's.
_LARGEST = {"append": "append_4096_d128", "decode": "decode_256_d128",
            "chunk": "chunk_6_ragged_d128", "verify": "verify_64x4_probs"}


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
    op = rng.choice(["append", "decode", "decode", "chunk", "chunk", "verify"])
    if op == "verify":
        most = rng.randint(0, 8)
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), batch=_log_int(rng, 1, 256),
                    min_drafts=rng.randint(0, most), max_drafts=most,
                    vocab=_log_int(rng, 500, 151936), draft_probs=rng.random() < 0.5,
                    greedy=rng.choice([0.0, 0.0, 0.5, 1.0]), shape_seed=rng.randint(0, 1 << 30))
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 16])
    head_dim = rng.choice([64, 128])
    block = rng.choice([16, 16, 16, 32])
    if op == "append":
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), tokens=_log_int(rng, 1, 4096),
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4]),
                    block=block, interleaved=rng.random() < 0.5,
                    max_position=_log_int(rng, 4096, 1000000))
    if op == "decode":
        max_len = _log_int(rng, 16, 32768)
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]),
                    batch=_log_int(rng, 1, 256), heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, block=block, min_len=rng.randint(1, max_len),
                    max_len=max_len, shape_seed=rng.randint(0, 1 << 30))
    max_chunk = _log_int(rng, 1, 2048)
    return dict(op=op, dtype="bf16", chunks=_log_int(rng, 1, 64), min_chunk=rng.randint(1, max_chunk),
                max_chunk=max_chunk, max_prior=_log_int(rng, 1, 16384), heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, block=block,
                shape_seed=rng.randint(0, 1 << 30))


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


def _drafts(case):
    """Verify: drafts of each sequence."""
    r = np.random.RandomState(case["shape_seed"])
    return r.randint(case["min_drafts"], case["max_drafts"] + 1, case["batch"]).tolist()


def _row_bytes(head_dim):
    return head_dim // 2 + head_dim // 16


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "verify":
        rows = sum(n + 1 for n in _drafts(case))
        return {"bytes": rows * case["vocab"] * e + 16 * rows, "flops": 3 * rows * case["vocab"]}
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        # The rows come in, the rotated queries and the packed rows go out; the pool that
        # is read back as values is as large as the rows.
        T = case["tokens"]
        return {"bytes": T * (2 * H + 2 * Hkv) * D * e + 2 * T * Hkv * (2 * _row_bytes(D) + 2 * D)
                + 8 * T + 4 * case["rotary_dim"],
                "flops": 3 * T * (H + Hkv) * case["rotary_dim"] + 6 * T * Hkv * D}
    if case["op"] == "decode":
        lens = _lengths(case)
        seen, tokens, keys = sum(lens), len(lens), sum(lens)
    else:
        seen = tokens = keys = 0
        for n, prior in _chunks(case):
            seen += n * prior + n * (n + 1) // 2
            keys += prior + n
            tokens += n
    return {"bytes": 2 * keys * Hkv * _row_bytes(D) + 2 * tokens * H * D * e
            + 4 * keys // case["block"] + 4 * tokens,
            "flops": 4 * H * D * seen}


# ------------------------------------------------------------------ the 4-bit format


def _quantise(x):
    """(codes, scales) of [..., D] values in 64 bits."""
    g = x.unflatten(-1, (-1, _GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(torch.maximum(-lo, hi) / 8.0)
    size = torch.ldexp(torch.ceil(mantissa * 16.0) / 16.0, exponent)
    size = torch.where(torch.maximum(-lo, hi) < _TINY, torch.zeros_like(size), size)
    scale = torch.where(-lo >= hi, size, -size)
    ratio = torch.where(scale == 0.0, torch.zeros_like(g), g / torch.where(
        scale == 0.0, torch.ones_like(scale), scale))
    codes = (torch.round(ratio) + 8.0).clamp(0.0, 15.0)
    return codes.flatten(-2).to(torch.uint8), scale.squeeze(-1).to(torch.bfloat16)


def _pack_codes(codes):
    """[..., D] codes -> [..., D / 2] bytes."""
    nibbles = codes.unflatten(-1, (-1, 4, 2)).transpose(-1, -2).flatten(-3).unflatten(-1, (-1, 2))
    return nibbles[..., 0] | (nibbles[..., 1] << 4)


def _unpack_codes(data):
    """[..., D / 2] bytes -> [..., D] codes."""
    nibbles = torch.stack([data & 15, data >> 4], -1).flatten(-2)
    return nibbles.unflatten(-1, (-1, 2, 4)).transpose(-1, -2).flatten(-3)


def _write_rows(pool, head, slots, codes, scales):
    """Packed rows of one kv head into pool [Hkv, NB, bs, row bytes] at `slots`."""
    _, nb, bs, row = pool.shape
    D = codes.shape[-1]
    blocks = pool[head].view(nb, bs * row)
    data = blocks[:, : bs * D // 2].unflatten(1, (bs, D // 2))
    data[slots // bs, slots % bs] = _pack_codes(codes)
    size = blocks[:, bs * D // 2:].unflatten(1, (bs, D // 16))
    size[slots // bs, slots % bs] = scales.contiguous().view(torch.uint8)


def _read_head(pool, head):
    """All rows of one kv head as fp32 values [NB * bs, D]."""
    _, nb, bs, row = pool.shape
    D = row * 16 // 9
    blocks = pool[head].reshape(nb, bs * row)
    codes = _unpack_codes(blocks[:, : bs * D // 2].reshape(nb * bs, D // 2))
    scales = blocks[:, bs * D // 2:].contiguous().view(torch.bfloat16).reshape(nb * bs, D // _GROUP)
    centred = codes.float().sub_(8.0).view(nb * bs, D // _GROUP, _GROUP)
    return centred.mul_(scales.float()[..., None]).view(nb * bs, D)


# ------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _random_pool(g, kv_heads, nb, bs, D, outliers):
    """A pool of packed random rows; `outliers`: a few dims are larger than the rest, as in
    keys."""
    pool = torch.empty((kv_heads, nb, bs, _row_bytes(D)), dtype=torch.uint8, device="cuda")
    size = torch.ones(D, device="cuda")
    if outliers:
        size[torch.randperm(D, generator=g, device="cuda")[: D // 32]] = 4.0
    step = max(1, (1 << 25) // (bs * D))  # blocks packed at a time
    for h in range(kv_heads):
        for b in range(0, nb, step):
            n = min(step, nb - b)
            x = torch.randn((n * bs, D), generator=g, device="cuda") * size
            codes, scales = _quantise(x)
            _write_rows(pool[h: h + 1, b: b + n], 0, torch.arange(n * bs, device="cuda"), codes,
                        scales)
    return pool


def _paged(case, totals, seed):
    g = _generator(seed)
    Hkv, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    need = [-(-t // bs) for t in totals]
    nb = sum(need) + 3
    order = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).tolist()
    table = np.full((len(totals), max(need)), -1, dtype=np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at: at + n]
        at += n
    T = len(totals) if case["op"] == "decode" else sum(n for n, _ in _chunks(case))
    return dict(case=case, table=torch.from_numpy(table).cuda(), scale=D ** -0.5,
                k=_random_pool(g, Hkv, nb, bs, D, True), v=_random_pool(g, Hkv, nb, bs, D, False),
                q=torch.randn((T, case["heads"], D), generator=g,
                              device="cuda").to(_DTYPES[case["dtype"]]),
                lens=torch.tensor(totals, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    if case["op"] == "decode":
        return _paged(case, _lengths(case), seed)
    if case["op"] == "chunk":
        chunks = _chunks(case)
        state = _paged(case, [n + p for n, p in chunks], seed)
        offsets = np.concatenate([[0], np.cumsum([n for n, _ in chunks])]).astype(np.int32)
        state["cu_q"] = torch.from_numpy(offsets).cuda()
        return state
    g = _generator(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "append":
        T, H, Hkv, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        bs, half = case["block"], case["rotary_dim"] // 2
        nb = -(-T // bs) + 1
        freq = 1e6 ** (-np.arange(half, dtype=np.float64) / half)
        return dict(
            case=case, freq=torch.from_numpy(freq).cuda(),
            qkv=torch.randn((T, (H + 2 * Hkv) * D), generator=g, device="cuda").to(dtype),
            pos=torch.randint(0, case["max_position"], (T,), generator=g, device="cuda",
                              dtype=torch.int32),
            slots=torch.randperm(nb * bs, generator=g, device="cuda")[:T].int(),
            every=torch.arange(nb * bs, device="cuda", dtype=torch.int32),
            k=_random_pool(g, Hkv, nb, bs, D, True), v=_random_pool(g, Hkv, nb, bs, D, False))
    drafts = _drafts(case)
    rows, V = sum(n + 1 for n in drafts), case["vocab"]
    # The target's logits: a spread of scores, a few favoured tokens a row.
    logits = torch.randn((rows, V), generator=g, device="cuda").mul_(2.0)
    favoured = torch.randint(0, V, (rows, 4), generator=g, device="cuda")
    logits.scatter_(1, favoured, 12.0 + 2.0 * torch.randn((rows, 4), generator=g, device="cuda"))
    # The draft model sees about the same.
    near = logits + 0.4 * torch.randn((rows, V), generator=g, device="cuda")
    probs = torch.softmax(near, -1)
    if case["draft_probs"]:
        tokens = torch.multinomial(probs, 1, generator=g)[:, 0]
    else:
        tokens = near.argmax(-1)
    warm = torch.rand((case["batch"],), generator=g, device="cuda") >= case["greedy"]
    temperature = 0.6 + 0.6 * torch.rand((case["batch"],), generator=g, device="cuda")
    offsets = np.concatenate([[0], np.cumsum([n + 1 for n in drafts])]).astype(np.int32)
    return dict(case=case, logits=logits.to(dtype), tokens=tokens.int(),
                probs=probs if case["draft_probs"] else None,
                temperature=torch.where(warm, temperature, torch.zeros_like(temperature)),
                cu=torch.from_numpy(offsets).cuda(),
                uniforms=torch.rand((rows,), generator=g, device="cuda"))


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return _RUN_OWN[op](state)
    return _RUN_PLAIN[op](state)


def _own_append(s):
    from batchstream_inference_engine_b200 import ops

    q = ops.rotary_append_int4(s["qkv"], s["freq"], s["pos"], s["slots"], s["k"], s["v"],
                               s["case"]["heads"], interleaved=s["case"]["interleaved"])
    k, v = ops.read_int4(s["k"], s["v"], s["every"])
    return [q, k, v]


def _own_decode(s):
    from batchstream_inference_engine_b200 import ops

    return ops.int4_attention_batched(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"])


def _own_chunk(s):
    from batchstream_inference_engine_b200 import ops

    return ops.int4_prefill_attention(s["q"], s["k"], s["v"], s["table"], s["cu_q"], s["lens"],
                                      s["scale"], max_query_len=s["case"]["max_chunk"])


def _own_verify(s):
    from batchstream_inference_engine_b200 import ops

    tokens, accepted = ops.verify_drafts(s["logits"], s["tokens"], s["cu"], s["uniforms"],
                                         temperature=s["temperature"], draft_probs=s["probs"])
    return [tokens, accepted]


def _plain_append(s):
    case = s["case"]
    T, H, Hkv, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    rd = case["rotary_dim"]
    # 64 bits: angles of far positions, and keys next to the border of two codes.
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    x = s["qkv"].view(T, H + 2 * Hkv, D).double()
    head, rest = x[:, : H + Hkv, :rd], x[:, : H + Hkv, rd:]
    if case["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., : rd // 2], head[..., rd // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    turned = torch.cat([turned, rest], -1)
    slots = s["slots"].long()
    out = [turned[:, :H].to(s["qkv"].dtype)]
    for pool, rows in ((s["k"], turned[:, H:]), (s["v"], x[:, H + Hkv:])):
        codes, scales = _quantise(rows)
        for h in range(Hkv):
            _write_rows(pool, h, slots, codes[:, h], scales[:, h])
        out.append(torch.stack([_read_head(pool, h) for h in range(Hkv)], 1).to(torch.bfloat16))
    return out


def _softmax(scores, mask):
    """Softmax over the last axis of the entries that ``mask`` keeps."""
    scores = scores.masked_fill(~mask, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_decode(s):
    case = s["case"]
    Hkv, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    B, groups = s["q"].shape[0], case["heads"] // case["kv_heads"]
    pos = torch.arange(int(s["table"].shape[1]) * bs, device="cuda")[None]
    q = s["q"].float().view(B, Hkv, groups, D)
    out = torch.empty((B, Hkv, groups, D), device="cuda")
    some = max(1, (1 << 28) // (pos.shape[1] * D))  # sequences at a time
    for h in range(Hkv):
        keys, values = _read_head(s["k"], h), _read_head(s["v"], h)
        for b in range(0, B, some):
            rows = slice(b, b + some)
            mask = pos < s["lens"][rows].long()[:, None]
            block = s["table"][rows].long().clamp(min=0).repeat_interleave(bs, 1)
            slot = block * bs + pos % bs
            p = _softmax(torch.matmul(q[rows, h], keys[slot].transpose(1, 2)) * s["scale"],
                         mask[:, None])
            out[rows, h] = torch.matmul(p, values[slot])
    return out.view(B, case["heads"], D).to(s["q"].dtype)


def _plain_chunk(s):
    case = s["case"]
    Hkv, D, bs = case["kv_heads"], case["head_dim"], case["block"]
    groups = case["heads"] // Hkv
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    for h in range(Hkv):
        all_keys, all_values = _read_head(s["k"], h), _read_head(s["v"], h)
        at = 0
        for r, (n, prior) in enumerate(_chunks(case)):
            pos = torch.arange(prior + n, device="cuda")
            mask = pos <= prior + torch.arange(n, device="cuda")[:, None]
            slot = s["table"][r].long()[pos // bs] * bs + pos % bs
            q = s["q"][at: at + n, h * groups: (h + 1) * groups].float()
            p = _softmax(torch.matmul(q.transpose(0, 1), all_keys[slot].t()) * s["scale"], mask)
            mixed = torch.matmul(p, all_values[slot]).transpose(0, 1)
            out[at: at + n, h * groups: (h + 1) * groups] = mixed.to(out.dtype)
            at += n
    return out


def _plain_verify(s):
    case = s["case"]
    cu = s["cu"].long()
    B, N, V = case["batch"], s["logits"].shape[0], case["vocab"]
    rows = torch.arange(N, device="cuda")
    seq = torch.searchsorted(cu[1:], rows, right=True)
    step = rows - cu[seq]
    last = rows == cu[seq + 1] - 1
    temperature = s["temperature"].double()[seq]
    greedy = temperature == 0.0
    drafts = s["tokens"].long()
    z = s["logits"].double()
    top = z.amax(-1, keepdim=True)
    best = torch.where(z == top, torch.arange(V, device="cuda"), V).amin(-1)
    # 64 bits: long sums, and draws next to the border of two tokens.
    p = torch.exp((z - top) / torch.where(greedy, 1.0, temperature)[:, None])
    p = p / p.sum(-1, keepdim=True)
    p_draft = p.gather(1, drafts[:, None])[:, 0]
    if s["probs"] is not None:
        q_draft = s["probs"].gather(1, drafts[:, None])[:, 0].double()
    else:
        q_draft = torch.ones_like(p_draft)
    take = torch.where(greedy, best == drafts, s["uniforms"].double() * q_draft < p_draft) & ~last
    # Accepted: the drafts ahead of a sequence's first row that is not taken.
    first = torch.full((B,), N, device="cuda").scatter_reduce(
        0, seq, torch.where(take, N, step), "amin")
    end = cu[:-1] + first  # the row that the step's last token is drawn from
    weights = p[end]
    rejected = ~last[end]
    if s["probs"] is not None:
        left = (weights - s["probs"][end].double()).clamp(min=0.0)
    else:
        left = weights.scatter(1, drafts[end][:, None], 0.0)
    use = rejected & (left.sum(-1) > 0.0)
    weights = torch.where(use[:, None], left, weights)
    below = weights.cumsum(-1)
    target = s["uniforms"].double()[cu[1:] - 1] * below[:, -1]
    drawn = (below <= target[:, None]).sum(-1)
    final = torch.where(greedy[end], best[end], drawn)
    tokens = torch.where(step < first[seq], drafts, torch.full_like(drafts, -1))
    tokens[end] = final
    return [tokens.int(), first.int()]


_RUN_OWN = {"append": _own_append, "decode": _own_decode, "chunk": _own_chunk,
            "verify": _own_verify}
_RUN_PLAIN = {"append": _plain_append, "decode": _plain_decode, "chunk": _plain_chunk,
              "verify": _plain_verify}


# ------------------------------------------------------------------ 64 bits


def _values64(pool, slots):
    """Rows of a pool at `slots`, every kv head: [Hkv, n, D] in 64 bits, byte by byte."""
    Hkv, nb, bs, row = pool.shape
    D = row * 16 // 9
    flat = pool.reshape(Hkv, nb * bs * row)
    start = (slots // bs) * (bs * row)
    at = start + (slots % bs) * (D // 2)
    d = torch.arange(D, device="cuda")
    nibble = (d % 8) // 2 + 4 * (d % 2)
    byte = flat[:, at[:, None] + (d // 8) * 4 + nibble // 2].int()
    code = (byte >> (4 * (nibble % 2)).int()) & 15
    where = start + bs * D // 2 + (slots % bs) * (D // 16)
    group = where[:, None] + 2 * torch.arange(D // 32, device="cuda")
    bits = flat[:, group].int() | (flat[:, group + 1].int() << 8)
    scale = (bits << 16).view(torch.float32).double()
    return (code.double() - 8.0) * scale.repeat_interleave(32, -1)


def _attend64(q, keys, values, seen, scale):
    """q [n, H, D] over keys and values [Hkv, L, D], seen [n, L]: 64-bit attention."""
    n, H, D = q.shape
    groups = H // keys.shape[0]
    scores = torch.einsum("nkgd,kld->kgnl", q.double().reshape(n, -1, groups, D), keys) * scale
    scores = torch.where(seen, scores, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
    log_sum = torch.logsumexp(scores, -1, keepdim=True)
    return torch.einsum("kgnl,kld->nkgd", torch.exp(scores - log_sum), values).reshape(n, H, D)


def exact(case, seed):
    """What ``run`` returns, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "verify":
        return _exact_verify(case, s)
    if case["op"] == "decode":
        spans = [(i, 1, n - 1) for i, n in enumerate(_lengths(case))]
    else:
        spans, at = [], 0
        for n, prior in _chunks(case):
            spans.append((at, n, prior))
            at += n
    bs = case["block"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, (at, n, prior) in enumerate(spans):
        position = torch.arange(prior + n, device="cuda")
        slot = s["table"][r].long().repeat_interleave(bs)[: prior + n] * bs + position % bs
        keys, values = _values64(s["k"], slot), _values64(s["v"], slot)
        for i in range(0, n, 256):  # rows of the chunk, 256 at a time
            m = min(256, n - i)
            token = torch.arange(prior + i, prior + i + m, device="cuda")[:, None]
            out[at + i: at + i + m] = _attend64(s["q"][at + i: at + i + m], keys, values,
                                                token >= position, s["scale"])
    return out


def _exact_append(case, s):
    T, H, Hkv, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    rd = case["rotary_dim"]
    x = s["qkv"].double().reshape(T, H + 2 * Hkv, D)
    first = torch.arange(rd // 2, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else rd // 2)
    angle = (s["pos"].double()[:, None] * s["freq"]).reshape(T, 1, rd // 2)
    z = torch.complex(x[:, : H + Hkv, first], x[:, : H + Hkv, second]) * torch.polar(
        torch.ones_like(angle), angle)
    y = x.clone()
    y[:, : H + Hkv, first] = z.real
    y[:, : H + Hkv, second] = z.imag
    out = [y[:, :H]]
    every = s["every"].long()
    for pool, rows in ((s["k"], y[:, H: H + Hkv]), (s["v"], y[:, H + Hkv:])):
        # The step is the least m * 2^e >= largest / 8 with 8 <= m < 16.
        g = rows.reshape(T, Hkv, D // 32, 32)
        largest = g.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(largest.clamp(min=_TINY) / 8.0)) - 3.0
        e = torch.where(torch.exp2(e + 4.0) <= largest / 8.0, e + 1.0, e)
        e = torch.where(torch.exp2(e + 3.0) > largest / 8.0, e - 1.0, e)
        step = torch.ceil(largest / 8.0 / torch.exp2(e)) * torch.exp2(e)
        step = torch.where(largest < _TINY, 0.0, step)
        negative = (g == -largest).any(-1, keepdim=True)
        step = torch.where(negative, step, -step)
        ratio = torch.where(step == 0.0, 0.0, g / step)
        down = torch.floor(ratio)
        part = ratio - down
        up = (part > 0.5) | ((part == 0.5) & (torch.remainder(down, 2.0) == 1.0))
        near = torch.where(up, down + 1.0, down)
        held = torch.where(near > 7.0, 7.0, torch.where(near < -8.0, -8.0, near)) * step
        values = _values64(pool, every)
        values[:, s["slots"].long()] = held.reshape(T, Hkv, D).transpose(0, 1)
        out.append(values.transpose(0, 1))
    return out


def _exact_verify(case, s):
    """One sequence after the other, from the definition."""
    cu, V = s["cu"].tolist(), case["vocab"]
    uniforms, temperature = s["uniforms"].tolist(), s["temperature"].tolist()
    drafts = s["tokens"].tolist()
    tokens, accepted = [], []
    for b in range(case["batch"]):
        n = 0
        while True:
            r = cu[b] + n
            row = s["logits"][r].double()
            final = r == cu[b + 1] - 1
            if temperature[b] == 0.0:
                best = int((row == row.max()).nonzero()[0])
                if not final and best == drafts[r]:
                    n += 1
                    continue
                tokens += drafts[cu[b]: r] + [best]
                break
            p = torch.softmax(row / temperature[b], -1)
            q = None if s["probs"] is None else s["probs"][r].double()
            x = drafts[r]
            if not final and uniforms[r] * (1.0 if q is None else float(q[x])) < float(p[x]):
                n += 1
                continue
            w = p
            if not final:
                if q is None:
                    left = p.clone()
                    left[x] = 0.0
                else:
                    left = torch.relu(p - q)
                w = left if float(left.sum()) > 0.0 else p
            sums = torch.cumsum(w, 0)
            limit = uniforms[cu[b + 1] - 1] * float(sums[-1])
            tokens += drafts[cu[b]: r] + [int((sums > limit).nonzero()[0])]
            break
        tokens += [-1] * (cu[b + 1] - len(tokens))
        accepted.append(n)
    return [torch.tensor(tokens, dtype=torch.int32, device="cuda"),
            torch.tensor(accepted, dtype=torch.int32, device="cuda")]

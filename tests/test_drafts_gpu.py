"""Verification of drafted tokens on the GPU, against the definition in 64 bits.

Tokens and counts are whole numbers and compared as such.  The kernel accepts by a fp32 sum
of exponentials (off by 2^-20 of it at most, and less by far), so cases are made in which no
acceptance is nearer to its border than that; draws are in fp64, and none is nearer to the
border of two tokens than 2^-40 of the weights' sum.  The reference checks both.
"""

import math

import pytest
import torch

from batchstream_inference_engine_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(drafts, vocab, dtype=torch.float32, seed=0, probs=True, spread=2.0, near=0.5,
         temperature=1.0):
    """A batch with drafts[b] drafts in sequence b, drawn from a model near the target's."""
    g = torch.Generator().manual_seed(seed)
    N = sum(n + 1 for n in drafts)
    logits = (torch.randn(N, vocab, generator=g) * spread).to(dtype)
    other = logits.float() + near * torch.randn(N, vocab, generator=g)
    q = torch.softmax(other, -1)
    tokens = torch.multinomial(q, 1, generator=g)[:, 0].int() if probs else other.argmax(-1).int()
    cu = torch.tensor([0] + [n + 1 for n in drafts]).cumsum(0).int()
    return dict(logits=logits, draft_tokens=tokens, cu_rows=cu,
                uniforms=torch.rand(N, generator=g), temperature=temperature,
                draft_probs=q if probs else None)


def reference(c):
    cu, u = c["cu_rows"].tolist(), c["uniforms"].double()
    B, N = len(cu) - 1, c["logits"].shape[0]
    temps = c["temperature"]
    temps = temps.tolist() if torch.is_tensor(temps) else [temps] * B
    tokens, accepted = torch.full((N,), -1, dtype=torch.int32), []
    for b in range(B):
        taken = 0
        for r in range(cu[b], cu[b + 1]):
            row, x, last = c["logits"][r].double(), int(c["draft_tokens"][r]), r == cu[b + 1] - 1
            if temps[b] == 0.0:
                best = int((row == row.max()).nonzero()[0])
                tokens[r] = best
                if not last and x == best:
                    taken += 1
                    continue
                break
            p = torch.softmax(row / torch.tensor(temps[b], dtype=torch.float32).double(), -1)
            q = c["draft_probs"][r].double() if c["draft_probs"] is not None else None
            if not last:
                have, need = float(p[x]), float(u[r]) * (1.0 if q is None else float(q[x]))
                assert abs(have - need) > 2.0 ** -20 * have, "a case on the border"
                if need < have:
                    tokens[r] = x
                    taken += 1
                    continue
            w = p.clone()
            if not last:
                left = (p - q).clamp(min=0) if q is not None else p.clone()
                if q is None:
                    left[x] = 0.0
                w = left if float(left.sum()) > 0 else p
            run = w.cumsum(0)
            at = float(u[cu[b + 1] - 1]) * float(run[-1])
            assert float((run - at).abs().min()) > 2.0 ** -40 * float(run[-1]), "a draw on the border"
            tokens[r] = int((run > at).nonzero()[0])
            break
        accepted.append(taken)
    return tokens, torch.tensor(accepted, dtype=torch.int32)


def call(c):
    return ops.verify_drafts(**{k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()})


def check(c):
    tokens, accepted = call(c)
    assert ops.take_status() == 0
    want_tokens, want_accepted = reference(c)
    assert torch.equal(accepted.cpu(), want_accepted)
    assert torch.equal(tokens.cpu(), want_tokens)
    return want_accepted


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 7, 500, 8192, 8193, 32003, 151936])
def test_vocabularies(dtype, probs, vocab):
    c = make([4, 0, 2, 7, 1, 3], vocab, dtype, seed=vocab, probs=probs)
    c["uniforms"] *= 0.999  # (a vocabulary of one leaves no room above)
    check(c)


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("batch", [1, 2, 40, 148, 300, 700])
def test_batches(batch, probs):
    # Clusters of every size, and more sequences than a pass of the row search.
    c = make([i % 6 for i in range(batch)], 1237, seed=batch, probs=probs,
             temperature=torch.tensor([(0.0, 0.7, 1.0, 1.6)[i % 4] for i in range(batch)]))
    taken = check(c)
    if batch >= 40:  # every outcome is there
        drafts = torch.tensor([i % 6 for i in range(batch)])
        assert bool((taken == 0).any()) and bool((taken == drafts).any())
        assert bool(((taken > 0) & (taken < drafts)).any())


@pytest.mark.parametrize("temperature", [0.0, 1e-30, 1e-3, 0.3, 5.0, 1e30])
def test_temperatures(temperature):
    c = make([3] * 20, 997, seed=3, probs=temperature >= 0.3, temperature=temperature, near=0.2)
    if 0.0 < temperature < 0.1:  # all the weight at the largest logit: no ties
        c["logits"][:, 500] = 20.0
        c["draft_tokens"][::2] = 500
    check(c)


def test_draft_probs_in_bf16_and_strided_rows():
    c = make([4] * 9, 777, torch.bfloat16, seed=5)
    c["draft_probs"] = c["draft_probs"].bfloat16()
    check(c)
    want = call(c)
    wide = {}
    for name in ("logits", "draft_probs"):
        t = torch.full((45, 800), math.nan, dtype=torch.bfloat16, device=DEV)
        t[:, 5: 782] = c[name].to(DEV)
        wide[name] = t[:, 5: 782]
    got = call({**c, **wide})
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    spread = torch.zeros(45, 1554, dtype=torch.bfloat16, device=DEV)
    spread[:, ::2] = c["logits"].to(DEV)
    got = call({**c, "logits": spread[:, ::2]})
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert ops.take_status() == 0


def test_equal_models_accept_everything():
    c = make([5] * 30, 2000, seed=6, near=0.0)
    c["draft_probs"] = c["draft_probs"] * 0.999  # above p nowhere, so u q < p
    taken = check(c)
    assert taken.tolist() == [5] * 30


def test_greedy_ties_go_to_the_first_and_nan_counts_as_the_largest():
    logits = torch.zeros(4, 20000)
    logits[0, [77, 9000, 19999]] = 3.0
    logits[1, 15000] = math.nan
    logits[1, 3] = math.inf
    logits[2] = -math.inf
    logits[3, 8191], logits[3, 8192] = 1.0, 1.0
    c = dict(logits=logits, draft_tokens=torch.tensor([77, 15000, 0, 5], dtype=torch.int32),
             cu_rows=torch.tensor([0, 4], dtype=torch.int32), uniforms=torch.zeros(4),
             temperature=0.0, draft_probs=None)
    tokens, accepted = call(c)
    assert tokens.tolist() == [77, 15000, 0, 8191] and accepted.tolist() == [3]
    assert tokens.tolist() == ops.argmax_rows(logits.to(DEV)).tolist()
    assert ops.take_status() == 0


def test_masked_tokens_are_never_drawn():
    for probs in (True, False):
        c = make([2] * 50, 3000, seed=8, probs=probs)
        allowed = torch.randperm(3000, generator=torch.Generator().manual_seed(1))[:7]
        mask = torch.ones(3000, dtype=torch.bool)
        mask[allowed] = False
        c["logits"][:, mask] = -math.inf
        check(c)
        tokens, _ = call(c)
        assert set(tokens.unique().tolist()) <= set(allowed.tolist()) | {-1}


def test_nothing_left_falls_back():
    # A certain draft with all the weight, and draft probabilities above p everywhere.
    c = make([1, 1], 300, seed=9, probs=False)
    c["logits"][0] = -math.inf
    c["logits"][0, 7] = 1.0
    c["draft_tokens"][0] = 7
    c["uniforms"][0] = 1.0  # not below 1: rejected all the same
    tokens, accepted = call(c)
    assert tokens[:2].tolist() == [7, -1] and int(accepted[0]) == 0
    c = make([1] * 40, 300, seed=10)
    c["draft_probs"] = torch.ones_like(c["draft_probs"])
    c["uniforms"][::2] = 0.99
    check(c)
    assert ops.take_status() == 0


@pytest.mark.parametrize("u", [-0.5, 0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, math.nan])
def test_uniforms_at_and_past_the_ends(u):
    # The first token of any weight, and the last.
    c = make([0] * 6, 5000, seed=11, probs=False)
    c["logits"][:, :100] = -math.inf
    c["logits"][:, 4900:] = -math.inf
    c["uniforms"][:] = u
    tokens, accepted = call(c)
    assert ops.take_status() == 0 and accepted.tolist() == [0] * 6
    if u <= 0.0:
        assert tokens.tolist() == [100] * 6
    elif u >= 1.0 or math.isnan(u):
        assert tokens.tolist() == [4899] * 6
    else:
        assert torch.equal(tokens.cpu(), reference(c)[0])


def test_draws_follow_the_target():
    # 40000 drafted tokens against a target of 16 tokens: each first token's frequency within 5
    # standard deviations of its probability, whatever the draft model.
    n, vocab = 20000, 16
    g = torch.Generator().manual_seed(12)
    target = torch.randn(vocab, generator=g)
    p = torch.softmax(target, -1)
    for probs in (True, False):
        q = torch.softmax(torch.randn(vocab, generator=g), -1)
        draft = torch.multinomial(q, n, replacement=True, generator=g).int()
        if not probs:
            draft[:] = int(q.argmax())
        rows = torch.stack([draft, torch.zeros(n, dtype=torch.int32)], 1).flatten()
        tokens, _ = call(dict(
            logits=target.expand(2 * n, vocab).contiguous(), draft_tokens=rows,
            cu_rows=torch.arange(0, 2 * n + 1, 2).int(), uniforms=torch.rand(2 * n, generator=g),
            temperature=1.0, draft_probs=q.expand(2 * n, vocab).contiguous() if probs else None))
        count = torch.bincount(tokens.view(n, 2)[:, 0].cpu().long(), minlength=vocab).double()
        assert bool(((count / n - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all())
    assert ops.take_status() == 0


def test_padding_sequences_and_rows_of_none():
    c = make([2, 1, 3], 600, seed=13)
    want = call(c)
    pad = dict(c)
    pad["cu_rows"] = torch.tensor([0, 0, 3, 3, 5, 9, 9], dtype=torch.int32)
    for name in ("logits", "draft_probs"):
        pad[name] = torch.cat([c[name], torch.full((4, 600), math.nan)])
    pad["draft_tokens"] = torch.cat([c["draft_tokens"], torch.full((4,), 1 << 30, dtype=torch.int32)])
    pad["uniforms"] = torch.cat([c["uniforms"], torch.full((4,), math.nan)])
    tokens, accepted = call(pad)
    assert ops.take_status() == 0
    assert torch.equal(tokens[:9], want[0]) and tokens[9:].tolist() == [-1] * 4
    a = want[1].tolist()
    assert accepted.tolist() == [0, a[0], 0, a[1], a[2], 0]
    empty = call(dict(c, logits=c["logits"][:0], draft_tokens=c["draft_tokens"][:0],
                      uniforms=c["uniforms"][:0], draft_probs=None,
                      cu_rows=torch.zeros(3, dtype=torch.int32)))
    assert empty[0].numel() == 0 and empty[1].tolist() == [0, 0]
    none = call(dict(c, cu_rows=torch.zeros(1, dtype=torch.int32)))
    assert none[0].tolist() == [-1] * 9 and none[1].numel() == 0


@pytest.mark.parametrize("change,message", [
    ("offsets", "context length"), ("past", "context length"), ("draft", "index"),
    ("nan", "not finite"), ("empty", "not finite"), ("inf", "not finite"),
    ("temperature", "not finite"),
])
def test_bad_input_is_reported_and_spares_the_others(change, message):
    c = make([2, 2, 2], 900, seed=14, probs=False, temperature=torch.tensor([1.0, 1.0, 1.0]))
    want = call(c)
    c = {k: v.clone() if torch.is_tensor(v) else v for k, v in c.items()}
    best = c["logits"][3].argmax()
    spared = [0, 2]
    if change == "offsets":
        c["cu_rows"][2] = 1  # the last sequence's rows then lie over the first's
        spared = []
    elif change == "past":
        c["cu_rows"][3] = 10
        spared = [0, 1]
    elif change == "draft":
        c["draft_tokens"][3] = 900
    elif change == "nan":
        c["logits"][3, 5] = math.nan
    elif change == "empty":
        c["logits"][3] = -math.inf
    elif change == "inf":
        c["logits"][3, 8] = math.inf
    else:
        c["temperature"][1] = -1.0
    tokens, accepted = call(c)
    with pytest.raises(RuntimeError, match=message):
        ops.take_status()
    for b in spared:
        assert torch.equal(tokens[3 * b: 3 * b + 3], want[0][3 * b: 3 * b + 3])
        assert accepted[b] == want[1][b]
    if change == "offsets":
        assert int(accepted[1]) == 0 and accepted[0] == want[1][0]
    if change in ("nan", "empty", "inf"):
        assert int(accepted[1]) == 0
        assert tokens[3:6].tolist() == [{"nan": 5, "empty": 0, "inf": 8}[change], -1, -1]
    if change == "draft":
        assert int(accepted[1]) == 0 and 0 <= int(tokens[3]) < 900
    if change == "temperature" and int(accepted[1]) == 0:
        assert int(tokens[3]) == int(best)


def test_streams_and_captured_calls():
    cases = [make([4] * 11, 30000, torch.bfloat16, seed=s) for s in (20, 21)]
    want = [call(c) for c in cases]
    runs = []
    for c in cases:
        dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.verify_drafts(**dev)
        runs.append((graph, dev, out, torch.cuda.Stream()))
    for _ in range(10):
        for graph, _, _, s in runs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, out, _), w in zip(runs, want):
            assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
            out[0].zero_(), out[1].zero_()
        torch.cuda.synchronize()
    # The same graph with the other batch's inputs.
    for name, t in runs[0][1].items():
        if torch.is_tensor(t):
            t.copy_(cases[1][name])
    runs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(runs[0][2][0], want[1][0]) and torch.equal(runs[0][2][1], want[1][1])
    assert ops.take_status() == 0


def test_wrappers_refuse():
    c = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in make([2, 1], 50).items()}
    ops.verify_drafts(**c)
    for kw in (dict(logits=c["logits"].half()), dict(logits=c["logits"][0]),
               dict(draft_tokens=c["draft_tokens"].long()), dict(draft_tokens=c["draft_tokens"][:4]),
               dict(cu_rows=c["cu_rows"].long()), dict(cu_rows=c["cu_rows"][:0]),
               dict(uniforms=c["uniforms"].double()), dict(uniforms=c["uniforms"][:4]),
               dict(temperature=-0.1), dict(temperature=math.inf), dict(temperature=math.nan),
               dict(temperature=torch.ones(1, device=DEV)), dict(temperature=torch.ones(2)),
               dict(draft_probs=c["draft_probs"][:, :49]), dict(draft_probs=c["draft_probs"].half()),
               dict(logits=c["logits"].cpu())):
        with pytest.raises(RuntimeError):
            ops.verify_drafts(**{**c, **kw})
    assert ops.take_status() == 0

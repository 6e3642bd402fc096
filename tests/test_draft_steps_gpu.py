"""Steps with drafted tokens on the engine: what they leave behind for the steps and forks that
follow.  fp32 pools hold what plain steps would have written (tokens are compared); of 4-bit
ones the 64-bit reference of test_int4_engine_gpu checks text, keys and values."""

import pytest
import torch

from batchstream_inference_engine_b200 import ops
from batchstream_inference_engine_b200.backend import PagedBackend

from .test_bounded_engine_gpu import VOCAB
from .test_int4_engine_gpu import (CONFIG, DEV, WINDOWED, backend_of, check_generated, generate,
                                  prompts)

pytestmark = pytest.mark.gpu


def ending_backend(model, pool, end, blocks=64):
    class Ends:
        def is_end_of_generation(self, token):
            return token == end

    return PagedBackend(model, blocks, 16, 48, vocab=Ends(), max_seqs=8, pool_dtype=pool)


@pytest.mark.parametrize("pool", [torch.float32, torch.uint8])
@pytest.mark.parametrize("behind", [0, 1, 4])
def test_forks_of_sequences_that_a_drafted_step_ended(pool, behind):
    # The ending token is the last draft, in the middle, and (no such draft) the token behind.
    text = prompts((20,))[0]
    plain = backend_of(pool=pool)
    (i,), want = generate(plain, [text], 40)
    want = want[i]
    at = next(k for k in range(3, 40) if want[k] not in want[:k])
    for follow in (want[1: at + 1 + behind], want[1:at]):
        model = plain._model
        runs = []
        for drafted in (False, True):
            backend = ending_backend(model, pool, want[at])
            drafts = list(follow)
            (s,), out = generate(backend, [text], 1)
            tokens = out[s][:1]
            while not backend._sequences[s].finished:
                if drafted:
                    got = backend.draft_step({s: drafts})[s]
                    assert pool == torch.uint8 or len(got) == at  # all hold, in one step
                    tokens += [o.token for o in got]
                    drafts = []
                else:
                    tokens.append(backend.step()[s].token)
            assert pool == torch.uint8 or tokens == want[: at + 1]
            child = backend.fork_sequence(s, [9, 8, 7])
            more = []
            while len(more) < 12 and not (more and backend._sequences[child].finished):
                more += [o.token for o in backend.step().values()]
            runs.append((tokens, more))
            check = text + tokens + [9, 8, 7]
            cache = backend._sequences[child].cache
            assert cache.length == len(check) + len(more) - 1
            if pool == torch.uint8:
                check_generated(backend, child, check, more, torch.float32)
        assert pool == torch.uint8 or runs[0] == runs[1]
    assert ops.take_status() == 0


def held_after(length, window, sinks, size=16):
    """Blocks that a sequence of so many cached tokens holds after plain steps."""
    gone = max(0, length - window + 1) // size - -(-sinks // size) if window else 0
    return -(-length // size) - max(0, gone)


@pytest.mark.parametrize("config", [CONFIG, WINDOWED])
@pytest.mark.parametrize("pool", [torch.float32, torch.uint8])
def test_rejected_drafts_leave_what_plain_steps_leave(config, pool):
    # Chunks whose rejected end reaches into a new block, past the border where the window
    # gives one up.
    texts = prompts((130, 20))
    _, want = generate(backend_of(config, pool=pool), texts, 80)
    backend = backend_of(config, pool=pool)
    ids, out = generate(backend, texts, 1)
    turn = rejected = 0
    while min(len(v) for v in out.values()) < 60:
        drafts = {}
        for i in ids:
            drafts[i] = want[i][len(out[i]): len(out[i]) + turn % 4]
            drafts[i] += [(t + 1) % VOCAB for t in want[i][len(out[i]) + len(drafts[i]):][:20 - turn % 7]]
        for i, steps in backend.draft_step(drafts).items():
            tokens = [o.token for o in steps]
            assert tokens[:-1] == drafts[i][: len(tokens) - 1]
            rejected += len(drafts[i]) + 1 - len(tokens)
            out[i] += tokens
        lengths = [backend._sequences[i].cache.length for i in ids]
        assert lengths == [len(t) + len(out[i]) - 1 for t, i in zip(texts, ids)]
        assert backend.blocks_in_use == sum(
            held_after(n, config.attention_window, config.attention_sinks) for n in lengths)
        turn += 1
    assert rejected > 100
    if pool == torch.float32:
        for i in ids:
            assert out[i][:80] == want[i][: len(out[i])]
    assert ops.take_status() == 0


@pytest.mark.parametrize("pool", [torch.float32, torch.uint8])
def test_drafts_in_a_pool_that_the_outputs_fill(pool):
    # As many blocks as 40 tokens each need: with 30 drafts each, every step runs.
    texts = prompts()
    blocks = sum(-(-(len(t) + 40) // 16) for t in texts)
    _, want = generate(backend_of(pool=pool), texts, 80)
    backend = backend_of(pool=pool, blocks=blocks)
    ids, out = generate(backend, texts, 1)
    while any(len(v) < 40 for v in out.values()):
        # (A request generates 40 tokens, so its drafts are no more than are left.)
        drafts = {i: want[i][len(out[i]):][: min(30, 39 - len(out[i]))] for i in ids}
        drafts[ids[0]] = [(t + 1) % VOCAB for t in drafts[ids[0]]]  # none of them holds
        for i, steps in backend.draft_step(drafts).items():
            out[i] += [o.token for o in steps]
            if len(out[i]) >= 40:
                backend.release_sequence(i)
                ids = [j for j in ids if j != i]
    assert backend.blocks_in_use == 0 and not ids
    if pool == torch.float32:
        assert all(out[i] == want[i][:40] for i in out)
    assert ops.take_status() == 0


@torch.inference_mode()
def step_logits(model, groups):
    """The logits of every token of a step, which counts none of them as cached."""
    hidden = model._hidden(groups, list(range(sum(len(tokens) for tokens, _ in groups))))
    return torch.nn.functional.linear(hidden, model.embed)


@pytest.mark.parametrize("pool", [torch.float32, torch.uint8])
def test_verify_tokens_with_draft_probabilities(pool):
    # The model's step with probabilities gives what verify_drafts gives of the same step's
    # logits; temperatures by sequence, greedy among them.
    texts = prompts((50, 7, 33))
    backend = backend_of(pool=pool)
    model = backend._model
    ids, out = generate(backend, texts, 1)
    g = torch.Generator().manual_seed(11)
    accepted = rejected = 0
    for turn in range(8):
        caches = [backend._sequences[i].cache for i in ids]
        lengths = [c.length for c in caches]
        n = [int(torch.randint(0, 5, (1,), generator=g)) for _ in ids]
        T = sum(n) + len(ids)
        groups, at = [], [0]
        for i, k, cache in zip(ids, n, caches):
            groups.append([out[i][-1], *torch.randint(0, VOCAB, (k,), generator=g).tolist()])
            at.append(at[-1] + k + 1)
        # Every other turn's first drafts come from a sharper target: most of them hold.
        probs = torch.softmax(step_logits(model, list(zip(groups, caches))).float() * 3, -1)
        for b, tokens in enumerate(groups):
            for k in range(len(tokens) - 1):
                if turn % 2 == 0 and k == 0:
                    tokens[1] = int(torch.multinomial(probs[at[b]].cpu(), 1, generator=g))
        groups = list(zip(groups, caches))
        logits = step_logits(model, groups)
        uniforms = torch.rand(T, generator=g).to(DEV)
        temperature = torch.tensor([0.9, 0.0, 1.4], device=DEV)
        drafts = [t for tokens, _ in groups for t in (*tokens[1:], 0)]
        want, taken = ops.verify_drafts(
            logits, torch.tensor(drafts, dtype=torch.int32, device=DEV),
            torch.tensor(at, dtype=torch.int32, device=DEV), uniforms, temperature, probs)
        got = model.verify_tokens(groups, temperature, uniforms, probs)
        for b, tokens in enumerate(got):
            k = int(taken[b])
            assert tokens == want[at[b]: at[b] + k + 1].tolist()
            assert caches[b].length == lengths[b] + k + 1
            out[ids[b]] += tokens
            accepted += k
            rejected += n[b] - k
    assert accepted > 3 and rejected > 3 and ops.take_status() == 0
    with pytest.raises(RuntimeError, match="draft_probs"):
        model.verify_tokens(groups, temperature, uniforms, probs[:, :-1])
    assert [c.length for c in caches] == [len(t) + len(out[i]) - 1 for t, i in zip(texts, ids)]

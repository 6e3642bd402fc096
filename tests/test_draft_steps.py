"""Steps with drafted tokens on the host (no GPU): what a sequence holds after one, by a
stand-in for the model that keeps the text in the cache's slots."""

import pytest
import torch

from batchstream_inference_engine_b200 import torch_model
from batchstream_inference_engine_b200.backend import PagedBackend
from batchstream_inference_engine_b200.block_allocator import OutOfBlocks
from batchstream_inference_engine_b200.torch_model import (ModelConfig, PagedKVPool, TorchModel,
                                                          random_weights)

from .test_bounded_cache import TINY, mirrored

END = 49
PROMPT = [1, 2, 3, 4]


class Vocab:
    def is_end_of_generation(self, token):
        return token == END


class Backend(PagedBackend):
    """A backend whose model goes on with the tokens of `follow`, by position."""

    def __init__(self, follow, monkeypatch, num_blocks=40, block_size=1, max_position=64, **config):
        config = ModelConfig(**TINY, **config)
        model = TorchModel(config, random_weights(config, vocab_size=50, intermediate_size=16),
                           device="cpu", dtype=torch.float32, max_position=max_position)
        super().__init__(model, num_blocks, block_size, 100, vocab=Vocab(), max_seqs=8)
        self.follow, self.slots = follow, {}
        monkeypatch.setattr(model, "next_tokens", None)
        monkeypatch.setattr(model, "launch_tokens", self._launch_tokens)
        monkeypatch.setattr(model, "verify_tokens", self._verify_tokens)

    def _write(self, tokens, cache):
        cache.reserve(len(tokens))
        for i, token in enumerate(tokens):
            self.slots[self.pool.allocator.locate(cache.seq_id, cache.length + i)] = token

    def _launch_tokens(self, groups):
        ids = []
        for tokens, cache in groups:
            self._write(tokens, cache)
            ids.append(self.follow[cache.length + len(tokens)])
        self._model._advance(self.pool, groups)

        class Ids:
            ref = staticmethod(lambda i: -1 - i)
            result = staticmethod(lambda: ids)

        return Ids

    def _verify_tokens(self, groups, temperature=0.0, uniforms=None, draft_probs=None):
        out = []
        for tokens, cache in groups:
            self._write(tokens, cache)
            n = 0
            while n + 1 < len(tokens) and tokens[1 + n] == self.follow[cache.length + 1 + n]:
                n += 1
            out.append(self.follow[cache.length + 1: cache.length + 2 + n])
            self._model._advance(self.pool, [(tokens[: 1 + n], cache)])
        return out

    def text(self, seq_id):
        """The tokens that a sequence has cached, and those it still has to feed."""
        s = self._sequences[seq_id]
        cached = [self.slots[self.pool.allocator.locate(seq_id, p)] for p in range(s.cache.length)]
        return cached + list(s.pending) + ([] if s.next_token is None else [s.next_token])


@pytest.mark.parametrize("drafts,end", [
    ([5, 6, END, 8, 9], 2),  # in the middle of the drafts that hold
    ([5, 6, END], 2),        # the last of them
    ([5, 6], 2),             # the token after them
    ([5, 7], 2),             # after the ones that hold, a draft that does not
    ([END, 8], 0),
])
def test_a_sequence_that_a_drafted_step_ended_is_forked_as_after_plain_steps(monkeypatch, drafts,
                                                                             end):
    text = PROMPT + [30] + ([5, 6] if end else []) + [END]
    follow = text + [8, 9, 10, 11, 12]
    backend = Backend(follow, monkeypatch)
    s = backend.start_sequence(PROMPT)
    assert backend.step()[s].token == 30
    out = []
    while not out or not out[-1].finished:
        out += backend.draft_step({s: drafts if not out else []})[s]
    assert [o.token for o in out] == text[len(PROMPT) + 1:]
    assert [o.finished for o in out] == [False] * end + [True]
    # As after plain steps: everything up to the ending token, and nothing behind it.
    assert backend.text(s) == text
    assert backend._sequences[s].cache.length in (len(text) - 1, len(text))
    child = backend.fork_sequence(s, [20, 21])
    assert backend.text(child) == text + [20, 21]
    assert backend._sequences[child].next_token is None
    assert backend.draft_step({}) == {} and backend.text(s) == text
    with pytest.raises(RuntimeError, match="finished"):
        backend.fork_sequence(s, [])


def host_model(monkeypatch, accept, **config):
    """A model whose step runs on the host, without its layers: sequences accept as many
    drafts as `accept` says, one entry a group."""
    config = ModelConfig(**TINY, **config)
    model = TorchModel(config, random_weights(config, vocab_size=50, intermediate_size=16),
                       device="cpu", dtype=torch.float32, max_position=64)
    monkeypatch.setattr(model, "_stage", lambda values: torch.tensor(values, dtype=torch.int32))
    monkeypatch.setattr(model, "_raise_status", lambda: None)
    monkeypatch.setattr(model, "_layers", lambda pool, tokens, positions, slots, last, attend:
                        torch.zeros(last.numel(), config.hidden_size))
    monkeypatch.setattr(torch_model.ops, "step_metadata", lambda *a, **kw: (torch.zeros(9),) * 4)

    def verify_drafts(logits, tokens, cu, uniforms, temperature, probs):
        out = torch.full((tokens.numel(),), -1, dtype=torch.int32)
        for b, n in enumerate(accept):
            out[cu[b]: cu[b] + n] = tokens[cu[b]: cu[b] + n]
            out[cu[b] + n] = 7
        return out, torch.tensor(accept, dtype=torch.int32)

    monkeypatch.setattr(torch_model.ops, "verify_drafts", verify_drafts)
    return model


def test_blocks_of_rejected_drafts_are_given_back(monkeypatch):
    model = host_model(monkeypatch, [1, 0, 5])
    pool = PagedKVPool(model.config, 40, 2, device="cpu", dtype=torch.float32, max_seqs=4)
    caches = [pool.new_cache(i) for i in range(3)]
    for cache, n in zip(caches, (3, 4, 1)):
        cache.reserve(n)
        cache.advance(n)
    caches[2].reserve(11)  # what a caller holds ahead of its tokens stays
    pool.allocator.sync_device()
    free, held = pool.free_blocks, [list(pool.block_table(i)) for i in range(3)]
    got = model.verify_tokens([([1, 2, 3, 4, 5], caches[0]), ([1, 2, 3, 4], caches[1]),
                               ([1, 2, 3, 4, 5, 6], caches[2])])
    assert got == [[2, 7], [7], [2, 3, 4, 5, 6, 7]]
    assert [c.length for c in caches] == [5, 5, 7]
    tables = [pool.block_table(i) for i in range(3)]
    assert [len(t) for t in tables] == [3, 3, 6] and tables[2] == held[2]
    assert pool.free_blocks == free - 2  # as plain steps of 2, 1 and 6 tokens would leave
    assert tables[0][:2] == held[0] and tables[1][:2] == held[1]
    assert sorted(pool.allocator._free + sum(tables, [])) == list(range(40))
    # The device mirror learns of the blocks that come in their place.
    for cache in caches[:2]:
        cache.reserve(6)
    pool.allocator.sync_device()
    for i in range(2):
        table = pool.block_table(i)
        row = pool.allocator.device_tables[pool.allocator.row(i)]
        assert row[: len(table)].tolist() == table


def test_a_drafted_step_that_cannot_run_gives_back_what_it_took(monkeypatch):
    model = host_model(monkeypatch, [0, 0])
    pool = PagedKVPool(model.config, 8, 2, device="cpu", dtype=torch.float32, max_seqs=4)
    caches = [pool.new_cache(i) for i in range(2)]
    for cache in caches:
        cache.reserve(2)
        cache.advance(2)
    free = list(pool.allocator._free)
    with pytest.raises(OutOfBlocks):
        model.verify_tokens([([1, 2, 3, 4, 5], caches[0]), ([1] * 9, caches[1])])
    assert [c.length for c in caches] == [2, 2] and pool.allocator._free == free
    pool = PagedKVPool(model.config, 40, 2, device="cpu", dtype=torch.float32, max_seqs=4)
    cache = pool.new_cache(0)
    cache.reserve(62)
    cache.advance(62)
    free = list(pool.allocator._free)
    with pytest.raises(RuntimeError, match="rotary table"):
        model.verify_tokens([([1, 2, 3], cache)])
    assert cache.length == 62 and pool.allocator._free == free


def test_shrink_gives_up_the_last_blocks():
    a = mirrored(num_blocks=8)
    a.allocate(0, 20)
    a.fork(0, 1, 8)
    a.sync_device()
    table = list(a.block_table(0))
    assert a.shrink(0, 20) == 0 and a.shrink(0, 17) == 0 and a.shrink(0, 16) == 1
    assert a.block_table(0) == table[:4] and a._free[-1] == table[4]
    assert a.shrink(0, 1) == 2  # the shared one of the three stays in use
    assert a.block_table(0) == table[:1] and a.block_table(1) == table[:2]
    a.allocate(0, 20)
    a.sync_device()
    assert a.device_tables[a.row(0), :5].tolist() == a.block_table(0)
    assert a.shrink(7, 0) == 0  # (unknown: nothing to give up)
    a.trim(0, 13)
    assert a.block_table(0)[:3] == [-1] * 3
    assert a.shrink(0, 8) == 2 and a.block_table(0) == [-1] * 2
    a.allocate(0, 16)
    assert a.trim(0, 16) == 2 and a.block_table(0) == [-1] * 4


def started(backend, *lengths):
    """Sequences that have generated a token behind prompts of so many tokens."""
    ids = [backend.start_sequence(backend.follow[:n]) for n in lengths]
    assert set(backend.step()) == set(ids)
    return ids


def test_drafts_stop_at_the_last_position(monkeypatch):
    backend = Backend([t % 40 for t in range(80)], monkeypatch, num_blocks=80)
    near, far = started(backend, 60, 5)
    seen = []
    verify = backend._model.verify_tokens

    def verify_tokens(groups, *args):
        seen.append([len(tokens) for tokens, _ in groups])
        backend._model._check_positions([c.length for _, c in groups], seen[-1])
        return verify(groups, *args)

    monkeypatch.setattr(backend._model, "verify_tokens", verify_tokens)
    follow = backend.follow
    got = backend.draft_step({near: follow[61:70], far: follow[6:15]})
    # 60 tokens are cached: the step holds four more, and the other sequence all of its.
    assert seen == [[4, 10]]
    assert [len(got[near]), len(got[far])] == [4, 10]
    assert [o.token for o in got[far]] == follow[6:16]


@pytest.mark.parametrize("free", [0, 1, 2, 3, 5, 50])
def test_drafts_take_the_blocks_that_the_steps_tokens_leave(monkeypatch, free):
    # Blocks of two tokens: the first sequence needs one for its own next token, the second
    # has room for one draft, the third needs one too.
    backend = Backend([t % 40 for t in range(80)], monkeypatch, block_size=2)
    a, b, c = started(backend, 8, 7, 6)
    taken = backend.pool.new_cache(99)
    taken.reserve(2 * max(0, backend.pool.free_blocks - 2 - free))
    drafts = {a: [1] * 5, b: [1] * 5, c: [1] * 5}
    seen = []
    verify = backend._model.verify_tokens

    def verify_tokens(groups, *args):
        seen.append([len(tokens) - 1 for tokens, _ in groups])
        for tokens, cache in groups:
            cache.reserve(len(tokens))
        return verify(groups, *args)

    monkeypatch.setattr(backend._model, "verify_tokens", verify_tokens)
    got = backend.draft_step(drafts)
    assert all(len(got[i]) >= 1 for i in (a, b, c))
    # Each is given what is left in turn: one draft in its own block, two a block from there on
    # (b's own block is the one its next token begins).
    want = {0: [1, 0, 1], 1: [3, 0, 1], 2: [5, 0, 1], 3: [5, 2, 1], 5: [5, 5, 1], 50: [5, 5, 5]}
    assert seen == [want[free]]


def test_a_step_without_room_for_its_own_tokens_is_refused_as_a_plain_one(monkeypatch):
    backend = Backend([t % 40 for t in range(80)], monkeypatch, num_blocks=20, block_size=2)
    a, = started(backend, 8)
    taken = backend.pool.new_cache(99)
    taken.reserve(2 * backend.pool.free_blocks)
    for step in (backend.step, lambda: backend.draft_step({a: [1, 2]})):
        with pytest.raises(OutOfBlocks):
            step()

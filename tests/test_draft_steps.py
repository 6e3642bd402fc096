"""Steps with drafted tokens on the host (no GPU): what a sequence holds after one, by a
stand-in for the model that keeps the text in the cache's slots."""

import pytest
import torch

from batchstream_inference_engine_b200.backend import PagedBackend
from batchstream_inference_engine_b200.torch_model import ModelConfig, TorchModel, random_weights

from .test_bounded_cache import TINY

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
        super().__init__(model, num_blocks, block_size, 64, vocab=Vocab(), max_seqs=8)
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

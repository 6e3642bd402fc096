"""Steps with drafted tokens on the engine: what they leave behind for the steps and forks that
follow.  fp32 pools hold what plain steps would have written (tokens are compared); of 4-bit
ones the 64-bit reference of test_int4_engine_gpu checks text, keys and values."""

import pytest
import torch

from batchstream_inference_engine_b200 import ops
from batchstream_inference_engine_b200.backend import PagedBackend

from .test_int4_engine_gpu import backend_of, check_generated, generate, prompts

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

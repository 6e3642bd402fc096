"""One model on pool after pool, each gone before the next is made."""

import pytest
import torch

from batchstream_inference_engine_b200 import ops
from batchstream_inference_engine_b200.backend import PagedBackend

from .test_int4_engine_gpu import backend_of, generate, prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.uint8])
def test_one_model_on_pool_after_pool(dtype):
    model = backend_of(pool=dtype)._model
    texts = prompts()
    want = None
    for blocks in (64, 40, 64, 90, 33, 64, 40, 120, 64, 50):
        backend = PagedBackend(model, blocks, 16, 48, max_seqs=8, pool_dtype=dtype)
        guard = torch.full((1 << 16,), 7, dtype=torch.uint8, device=model.device)
        out = list(generate(backend, texts, 12)[1].values())
        assert want is None or out == want
        want = out
        assert bool((guard == 7).all()) and len(model._graphs) == 1
        del backend
    assert len(model._graphs) == 0 and ops.take_status() == 0

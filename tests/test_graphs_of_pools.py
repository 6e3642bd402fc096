"""A model's captured steps name the memory of the pool they were captured for: they live as
long as it does, and no other pool gets them (no GPU)."""

import gc

import torch

from batchstream_inference_engine_b200.torch_model import PagedKVPool

from .test_step_graphs import TINY, tiny_model


def test_a_pool_in_the_place_of_another_gets_graphs_of_its_own(monkeypatch):
    model = tiny_model()
    captured = []
    monkeypatch.setattr(model, "_capture", lambda pool, key: (len(captured), captured.append(key)))
    for turn in range(20):
        pool = PagedKVPool(TINY, 4, 4, device="cpu", dtype=torch.float32, max_seqs=2)
        for _ in range(2):
            assert model._graph(pool, (1, 0, 0))[0] == 2 * turn
            assert model._graph(pool, (2, 0, 0))[0] == 2 * turn + 1
        assert len(model._graphs) == 1
        del pool
        gc.collect()
        assert len(model._graphs) == 0
    assert len(captured) == 40


def test_graphs_of_two_pools(monkeypatch):
    model = tiny_model()
    monkeypatch.setattr(model, "_capture", lambda pool, key: (id(pool), key))
    pools = [PagedKVPool(TINY, 4, 4, device="cpu", dtype=torch.float32) for _ in range(2)]
    for pool in pools * 2:
        assert model._graph(pool, (4, 0, 0)) == (id(pool), (4, 0, 0))
    assert len(model._graphs) == 2

"""Block copies of the paged cache on the GPU (exact), and the pool operations that
use them: forks, trimming and compaction."""

import pytest
import torch

from batchstream_inference_engine_b200 import ops
from batchstream_inference_engine_b200.torch_model import ModelConfig, PagedKVPool

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def pools(shape, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2)]


def want(pool, pairs):
    out = pool.clone()
    axis = pool.dim() - 3
    for s, d in pairs:
        out.select(axis, d).copy_(pool.select(axis, s))
    return out


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [
    (3, 2, 20, 16, 64), (2, 20, 16, 128), (1, 1, 20, 1, 1), (2, 3, 20, 5, 7), (24, 2, 20, 16, 64),
    (1, 8, 20, 32, 256), (2, 1, 20, 4, 2),
])
@pytest.mark.parametrize("pairs", [
    [(3, 7)], [(0, 19), (0, 1), (0, 2), (5, 4)], [(i, i + 10) for i in range(10)], []])
def test_copies(dtype, shape, pairs):
    k, v = pools(shape, dtype)
    want_k, want_v = want(k, pairs), want(v, pairs)
    ops.copy_blocks(k, v, ints([s for s, _ in pairs]), ints([d for _, d in pairs]))
    assert ops.take_status() == 0
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_many_pairs():
    k, v = pools((4, 2, 5000, 4, 8), torch.bfloat16)
    order = torch.randperm(5000, generator=torch.Generator().manual_seed(1)).tolist()
    pairs = list(zip(order[:2500], order[2500:]))
    want_k, want_v = want(k, pairs), want(v, pairs)
    ops.copy_blocks(k, v, ints(order[:2500]), ints(order[2500:]))
    assert ops.take_status() == 0
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_pool_past_four_gigabytes():
    # 6.4 GB each: byte offsets past 2^32, element offsets past 2^31.
    shape = (2, 4, 25000, 16, 1024)
    k = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    k[-1, -1, -1] = 3.0
    v[0, 2, -1] = 4.0
    ops.copy_blocks(k, v, ints([24999]), ints([24000]))
    assert ops.take_status() == 0
    assert bool((k[-1, -1, 24000] == 3.0).all()) and bool((v[0, 2, 24000] == 4.0).all())
    assert float(k[:, :, 24000].float().sum()) == 3.0 * 16 * 1024
    assert float(v[:, :, 24000].float().sum()) == 4.0 * 16 * 1024


def test_padding_and_pairs_onto_themselves_do_nothing():
    k, v = pools((2, 2, 12, 16, 64), torch.bfloat16)
    want_k, want_v = want(k, [(1, 2)]), want(v, [(1, 2)])
    # -1 anywhere is padding, also beside a real pair's blocks; 5 -> 5 is idle, and a
    # block copied from may have several readers.
    ops.copy_blocks(k, v, ints([-1, 1, 2, 5, -1]), ints([3, 2, -1, 5, -1]))
    assert ops.take_status() == 0
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


@pytest.mark.parametrize("src,dst,done", [
    ([1, 2, 6], [4, 4, 7], [(6, 7)]),        # a destination named twice
    ([1, 2, 6], [2, 9, 7], [(2, 9), (6, 7)]),  # 1 -> 2 would race with 2 -> 9
    ([3, 5, 6], [5, 5, 7], [(6, 7)]),        # one of the two is 5 -> 5
])
def test_pairs_that_clash_are_reported_and_skipped(src, dst, done):
    k, v = pools((2, 2, 12, 16, 64), torch.bfloat16)
    want_k, want_v = want(k, done), want(v, done)
    ops.copy_blocks(k, v, ints(src), ints(dst))
    with pytest.raises(RuntimeError, match="another pair"):
        ops.take_status()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_blocks_outside_the_pool_are_reported_and_skipped():
    for src, dst in (([12, 1], [3, 2]), ([3, 1], [12, 2]), ([1 << 30, 1], [3, 2])):
        k, v = pools((2, 2, 12, 16, 64), torch.bfloat16)
        want_k, want_v = want(k, [(1, 2)]), want(v, [(1, 2)])
        ops.copy_blocks(k, v, ints(src), ints(dst))
        with pytest.raises(RuntimeError, match="block table entry"):
            ops.take_status()
        assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_unaligned_pools_and_strided_lists():
    shape = (2, 2, 12, 16, 64)
    k0, v0 = pools(shape, torch.bfloat16)
    n = k0.numel()
    bufs = [torch.empty(n + 1, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    k, v = (b[1:].view(shape) for b in bufs)
    k.copy_(k0)
    v.copy_(v0)
    both = ints([[1, 2], [5, 9], [1, 3]])
    ops.copy_blocks(k, v, both[:, 0], both[:, 1])
    assert ops.take_status() == 0
    pairs = [(1, 2), (5, 9), (1, 3)]
    assert torch.equal(k, want(k0, pairs)) and torch.equal(v, want(v0, pairs))


def test_captured_copy_follows_its_pairs():
    k, v = pools((2, 2, 12, 16, 64), torch.bfloat16)
    src, dst = ints([1, -1]), ints([2, -1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_blocks(k, v, src, dst)
    for pairs in ([(1, 2)], [(3, 4), (2, 5)], []):
        padded = pairs + [(-1, -1)] * (2 - len(pairs))
        src.copy_(ints([s for s, _ in padded]))
        dst.copy_(ints([d for _, d in padded]))
        want_k, want_v = want(k, pairs), want(v, pairs)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_refusals():
    k, v = pools((2, 2, 12, 16, 64), torch.bfloat16)
    a, b = ints([1]), ints([2])
    for args in ((k, v[:1], a, b), (k, v.float(), a, b), (k.transpose(1, 2), v, a, b),
                 (k, v, a.long(), b), (k, v, ints([1, 2]), b), (k, v, a, b.cpu()),
                 (k[0, 0], v[0, 0], a, b), (k.half(), v.half(), a, b)):
        with pytest.raises(RuntimeError):
            ops.copy_blocks(*args)
    assert ops.take_status() == 0


# ------------------------------------------------------------------ pool


CONFIG = ModelConfig(num_layers=3, hidden_size=64, num_heads=4, num_kv_heads=2, rope_theta=1e4,
                     rms_norm_eps=1e-6)


def tokens_of(pool, cache):
    """K of every cached token [L, Hkv, n, D] read through the block table."""
    table = torch.tensor(pool.block_table(cache.seq_id), device=DEV)
    p = torch.arange(cache.length, device=DEV)
    return pool.keys.flatten(2, 3)[:, :, table[p // pool.block_size] * pool.block_size
                                   + p % pool.block_size]


def test_pool_fork_and_compact_keep_every_sequence():
    pool = PagedKVPool(CONFIG, 40, 16, device=DEV, max_seqs=8)
    pool.keys.normal_()
    pool.values.normal_()
    caches = []
    for s, n in enumerate((50, 33, 100)):
        cache = pool.new_cache(s)
        cache.reserve(n)
        cache.advance(n)
        caches.append(cache)
    pool.release(caches.pop(1))
    before = [tokens_of(pool, c) for c in caches]
    child = pool.fork(caches[1], 7)
    assert child.length == 100 and torch.equal(tokens_of(pool, child), before[1])
    free = pool.free_blocks
    moved = pool.compact()
    assert moved > 0 and pool.free_blocks == free
    used = {b for c in (*caches, child) for b in pool.block_table(c.seq_id)}
    assert max(used) == len(used) - 1
    for c, b in zip((*caches, child), (*before, before[1])):
        assert torch.equal(tokens_of(pool, c), b)
    assert pool.compact() == 0
    assert ops.take_status() == 0

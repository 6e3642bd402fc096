"""Host side of the bounded cache (no GPU): forks, trimming and compaction in the
allocator, rotary frequencies, the model's windows, and what the operators refuse."""

import ctypes
import json
import math
import random

import pytest
import torch

from batchstream_inference_engine_b200 import _lib, ops
from batchstream_inference_engine_b200.backend import PagedBackend
from batchstream_inference_engine_b200.block_allocator import (EMPTY_BLOCK, BlockAllocator,
                                                               OutOfBlocks)
from batchstream_inference_engine_b200.torch_model import ModelConfig, TorchModel, random_weights


def mirrored(num_blocks=32, block_size=4, max_seqs=6):
    return BlockAllocator(num_blocks, block_size, max_seqs=max_seqs,
                          max_blocks_per_seq=num_blocks, device="cpu")


# ------------------------------------------------------------------ allocator


def test_fork_shares_whole_blocks_and_copies_the_partial_one():
    a = mirrored()
    a.allocate(0, 10)
    before = a.free_blocks
    pairs = a.fork(0, 1, 10)
    parent, child = a.block_table(0), a.block_table(1)
    assert child[:2] == parent[:2] and child[2] not in parent
    assert pairs == [(parent[2], child[2])] and a.free_blocks == before - 1
    assert a.row(1) != a.row(0)


def test_fork_at_a_block_boundary_copies_nothing():
    a = mirrored()
    a.allocate(0, 12)
    assert a.fork(0, 1, 8) == [] and a.block_table(1) == a.block_table(0)[:2]
    assert a.fork(0, 2, 0) == [] and a.block_table(2) == []


def test_shared_blocks_return_to_the_free_list_with_their_last_holder():
    a = mirrored(num_blocks=8)
    a.allocate(0, 8)
    a.fork(0, 1, 8)
    a.fork(1, 2, 8)
    table = list(a.block_table(0))
    a.free(0)
    a.free(2)
    assert a.free_blocks == 6
    a.free(1)
    assert a.free_blocks == 8 and a._free[-2:] == table  # in table order, as ever


def test_fork_refusals_take_nothing():
    a = mirrored(num_blocks=3, max_seqs=2)
    a.allocate(0, 10)
    with pytest.raises(ValueError):
        a.fork(0, 0, 4)
    with pytest.raises(ValueError):
        a.fork(0, 1, 13)
    with pytest.raises(ValueError):
        a.fork(0, 1, -1)
    with pytest.raises(KeyError):
        a.fork(9, 1, 4)
    with pytest.raises(OutOfBlocks):
        a.fork(0, 1, 10)  # the partial block needs one more
    assert a.free_blocks == 0 and a._free_rows == [1] and not a._refs
    a.fork(0, 1, 8)
    with pytest.raises(OutOfBlocks):
        a.fork(0, 2, 8)  # no table row left
    assert all(n == 2 for n in a._refs.values())


def test_trim_gives_up_the_blocks_between_sinks_and_window():
    a = mirrored()
    a.allocate(0, 40)  # 10 blocks
    table = list(a.block_table(0))
    assert a.trim(0, 3) == 0 and a.block_table(0) == table
    assert a.trim(0, 21, keep_first=5) == 3  # blocks 2, 3, 4
    assert a.block_table(0) == table[:2] + [EMPTY_BLOCK] * 3 + table[5:]
    assert a.trim(0, 21, keep_first=5) == 0
    assert a.trim(0, 1000, keep_first=5) == 5  # everything past the sinks
    assert a.trim(0, -5, keep_first=5) == 0
    a.allocate(0, 44)  # grows behind the trimmed entries
    assert len(a.block_table(0)) == 11 and a.block_table(0)[10] != EMPTY_BLOCK
    a.free(0)
    assert sorted(a._free) == list(range(32))


def test_trim_with_fewer_sinks_than_before():
    a = mirrored()
    a.allocate(0, 40)
    table = list(a.block_table(0))
    assert a.trim(0, 21, keep_first=9) == 2  # blocks 3 and 4
    assert a.trim(0, 7, keep_first=4) == 0  # block 0 stays, block 1 holds token 7
    assert a.trim(0, 8, keep_first=4) == 1
    assert a.trim(0, 33, keep_first=0) == 5  # blocks 0, 2, 5, 6, 7
    assert a.block_table(0) == [EMPTY_BLOCK] * 8 + table[8:]
    a.free(0)
    assert sorted(a._free) == list(range(32)) and not a._trimmed and not a._kept


def test_trims_in_any_order_give_up_what_each_asks_for():
    rng = random.Random(1)
    for _ in range(300):
        a = mirrored(num_blocks=16, block_size=3)
        a.allocate(0, 48)
        gone = set()
        for _ in range(6):
            first, keep = rng.randint(-3, 60), rng.randint(0, 30)
            want = {i for i in range(16) if 3 * i + 3 <= first and 3 * i >= keep} - gone
            assert a.trim(0, first, keep_first=keep) == len(want)
            gone |= want
            assert {i for i, b in enumerate(a.block_table(0)) if b == EMPTY_BLOCK} == gone


def test_trimming_a_shared_block_keeps_it_for_the_other_sequence():
    a = mirrored()
    a.allocate(0, 16)
    a.fork(0, 1, 16)
    table = list(a.block_table(1))
    free = a.free_blocks
    assert a.trim(0, 9) == 0 and a.free_blocks == free
    assert a.block_table(1) == table and a.block_table(0)[:2] == [EMPTY_BLOCK] * 2
    assert a.trim(1, 9) == 2
    a.fork(1, 2, 16)
    assert a.block_table(2) == a.block_table(1)
    for s in (0, 1, 2):
        a.free(s)
    assert sorted(a._free) == list(range(32)) and not a._refs and not a._trimmed


def test_fork_refuses_tokens_whose_blocks_are_gone():
    a = mirrored()
    a.allocate(0, 30)
    a.trim(0, 17, keep_first=4)  # blocks 1 to 3; block 4 holds token 17
    for tokens in (5, 8, 13, 15):
        with pytest.raises(ValueError):
            a.fork(0, 1, tokens)
    assert 1 not in a._tables and len(a._free_rows) == 5 and not a._refs
    assert a.fork(0, 3, 4) == [] and a.block_table(3) == a.block_table(0)[:1]  # the sinks alone
    assert a.fork(0, 1, 30) == [(a.block_table(0)[7], a.block_table(1)[7])]
    assert a.block_table(1)[:7] == a.block_table(0)[:7]
    a.trim(0, 1000)  # the partial last block too
    with pytest.raises(ValueError):
        a.fork(0, 2, 30)


def test_compact_moves_the_highest_blocks_into_the_lowest_holes():
    a = mirrored(num_blocks=12)
    for s in range(3):
        a.allocate(s, 12)  # blocks 11..9, 8..6, 5..3
    a.free(1)
    a.fork(0, 3, 12)
    a.sync_device()
    pairs = a.compact()
    assert pairs == [(9, 0), (10, 1), (11, 2)]  # 3, 4, 5 stay
    assert a.block_table(0) == [2, 1, 0] and a.block_table(3) == [2, 1, 0]
    assert a.block_table(2) == [5, 4, 3]
    assert sorted(a._free) == list(range(6, 12))
    a.sync_device()
    assert a.device_tables[a.row(0), :3].tolist() == [2, 1, 0]
    assert a.device_tables[a.row(3), :3].tolist() == [2, 1, 0]
    assert a.compact() == []
    a.free(0)
    a.free(3)
    a.free(2)
    assert sorted(a._free) == list(range(12))


def test_compact_of_an_empty_pool_and_of_a_full_one():
    a = mirrored(num_blocks=4)
    assert a.compact() == [] and a.free_blocks == 4
    a.allocate(0, 16)
    assert a.compact() == []


def test_random_forks_trims_and_compactions_account_for_every_block():
    rng = random.Random(0)
    a = mirrored(num_blocks=64, max_seqs=12)
    content = {}  # block -> the tokens it holds, as a pool would
    tokens = {}  # sequence -> its tokens
    next_id = 0
    for _ in range(3000):
        op = rng.random()
        live = list(tokens)
        try:
            if op < 0.25:
                n = rng.randint(0, 30)
                a.allocate(next_id, n)
                tokens[next_id] = []
                next_id += 1
            elif op < 0.5 and live:
                s = rng.choice(live)
                n = rng.randint(1, 9)
                a.allocate(s, len(tokens[s]) + n)
                for _ in range(n):
                    p = len(tokens[s])
                    block, offset = a.locate(s, p)
                    content.setdefault(block, {})[offset] = (s, p)
                    tokens[s].append((s, p))
            elif op < 0.65 and live:
                s = rng.choice(live)
                for src, dst in a.fork(s, next_id, len(tokens[s])):
                    content[dst] = dict(content.get(src, {}))
                tokens[next_id] = list(tokens[s])
                next_id += 1
            elif op < 0.8 and live:
                s = rng.choice(live)
                a.trim(s, len(tokens[s]) - 7, keep_first=rng.choice([0, 3, 5]))
            elif op < 0.85:
                moves = a.compact()
                assert not {s for s, _ in moves} & {d for _, d in moves}
                old = dict(content)
                for src, dst in moves:
                    content[dst] = dict(old.get(src, {}))
            elif live:
                s = rng.choice(live)
                a.free(s)
                del tokens[s]
        except OutOfBlocks:
            pass
        a.sync_device()
        held = [b for s in tokens for b in set(a.block_table(s)) - {EMPTY_BLOCK}]
        for b in set(held):
            assert a._refs.get(b, 1) == held.count(b)
        assert sorted(set(held) | set(a._free)) == list(range(64))
        assert not set(held) & set(a._free) and len(set(a._free)) == len(a._free)
        for s in tokens:
            table = a.block_table(s)
            for p, token in enumerate(tokens[s]):
                if table[p // 4] != EMPTY_BLOCK:
                    assert content[table[p // 4]][p % 4] == token
            # The device row holds every entry that a kernel may read.
            row = a.device_tables[a.row(s), : len(table)].tolist()
            assert all(x == y for x, y in zip(row, table) if y != EMPTY_BLOCK)


# ------------------------------------------------------------------ frequencies


def test_plain_and_linear_frequencies():
    f, amp = ops.rope_frequencies(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and amp == 1.0
    # exp(x log theta) against powers: a few fp64 roundings.
    want = torch.tensor([10000.0 ** (-2 * i / 8) for i in range(4)], dtype=torch.float64)
    assert torch.allclose(f, want, rtol=1e-14, atol=0)
    g, _ = ops.rope_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.equal(g, f / 4.0)


def test_ntk_keeps_the_fastest_pair_and_slows_the_slowest_by_the_factor():
    f, _ = ops.rope_frequencies(64, 1e6, device="cpu")
    g, amp = ops.rope_frequencies(64, 1e6, {"type": "ntk", "factor": 8.0}, device="cpu")
    assert amp == 1.0 and g[0] == f[0]
    assert math.isclose(f[-1] / g[-1], 8.0, rel_tol=1e-12)
    one, _ = ops.rope_frequencies(2, 1e6, {"type": "ntk", "factor": 8.0}, device="cpu")
    assert one.tolist() == [1.0]


def test_yarn_ramps_from_the_plain_frequencies_to_the_interpolated_ones():
    scaling = {"type": "yarn", "factor": 16.0, "original_max_position": 4096}
    f, _ = ops.rope_frequencies(128, 10000.0, device="cpu")
    g, amp = ops.rope_frequencies(128, 10000.0, scaling, device="cpu")
    assert math.isclose(amp, 0.1 * math.log(16.0) + 1.0)
    ratio = f / g
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns > 40], f[turns > 40])
    assert torch.allclose(ratio[turns < 0.9], torch.full((), 16.0, dtype=torch.float64))
    assert bool((ratio[1:] >= ratio[:-1]).all()) and 1.0 < ratio[30] < 16.0
    _, amp = ops.rope_frequencies(128, 1e4, dict(scaling, attention_factor=1.0), device="cpu")
    assert amp == 1.0


def test_banded_frequencies_by_wavelength():
    scaling = {"type": "banded", "factor": 8.0, "original_max_position": 8192,
               "low_freq_factor": 1.0, "high_freq_factor": 4.0}
    f, _ = ops.rope_frequencies(128, 500000.0, device="cpu")
    g, amp = ops.rope_frequencies(128, 500000.0, scaling, device="cpu")
    wavelength = 2 * math.pi / f
    assert amp == 1.0
    for x, y, w in zip(f.tolist(), g.tolist(), wavelength.tolist()):
        if w < 8192 / 4:
            assert y == x
        elif w > 8192:
            assert math.isclose(y, x / 8, rel_tol=1e-14)
        else:
            smooth = (8192 / w - 1.0) / 3.0
            assert math.isclose(y, (1 - smooth) * x / 8 + smooth * x, rel_tol=1e-12)


@pytest.mark.parametrize("dim,theta,scaling", [
    (7, 1e4, None), (0, 1e4, None), (8, 0.0, None), (8, 1e4, {"type": "odd", "factor": 2.0}),
    (8, 1e4, {"type": "linear", "factor": 0.5}), (8, 1e4, {"type": "linear", "factor": math.inf}),
    (8, 1e4, {"type": "banded", "factor": 2.0, "original_max_position": 64,
              "low_freq_factor": 4.0, "high_freq_factor": 4.0}),
])
def test_bad_frequency_requests_are_refused(dim, theta, scaling):
    with pytest.raises(RuntimeError):
        ops.rope_frequencies(dim, theta, scaling, device="cpu")


# ------------------------------------------------------------------ model and backend


TINY = dict(num_layers=1, hidden_size=32, num_heads=4, num_kv_heads=2, rope_theta=1e4,
            rms_norm_eps=1e-6)


def test_config_defaults_are_the_reference_model():
    c = ModelConfig(**TINY)
    assert c.attention_window == 0 and c.rotary_from_tables
    assert ModelConfig(**TINY, rotary_dim=8).rotary_from_tables
    assert not ModelConfig(**TINY, rotary_dim=4).rotary_from_tables
    assert not ModelConfig(**TINY, rope_interleaved=True).rotary_from_tables
    scaled = ModelConfig(**TINY, rope_scaling={"type": "linear", "factor": 2.0})
    assert not scaled.rotary_from_tables and isinstance(hash(scaled), int)


CHECKPOINT = {"num_hidden_layers": 4, "hidden_size": 64, "num_attention_heads": 4,
              "num_key_value_heads": 2, "rope_theta": 1e6, "rms_norm_eps": 1e-6,
              "max_position_embeddings": 4096}
YARN = {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024}


@pytest.mark.parametrize("keys,fields", [
    ({}, {}),
    ({"sliding_window": 2048, "use_sliding_window": False, "max_window_layers": 2}, {}),
    ({"sliding_window": None, "layer_types": ["full_attention"] * 4, "rope_scaling": None}, {}),
    ({"sliding_window": 2048, "use_sliding_window": True, "max_window_layers": 4}, {}),
    ({"sliding_window": 2048, "use_sliding_window": True, "max_window_layers": 0},
     {"attention_window": 2048}),
    ({"sliding_window": 2048}, {"attention_window": 2048}),
    ({"sliding_window": 2048, "use_sliding_window": True, "max_window_layers": None},
     {"attention_window": 2048}),
    ({"sliding_window": 99, "layer_types": ["sliding_attention"] * 4}, {"attention_window": 99}),
    ({"partial_rotary_factor": 0.5}, {"rotary_dim": 8}),
    ({"rope_parameters": {"rope_type": "default", "rope_theta": 1e6,
                          "partial_rotary_factor": 0.25}}, {"rotary_dim": 4}),
    ({"rope_scaling": {"type": "linear", "factor": 2.0}},
     {"rope_scaling": {"type": "linear", "factor": 2.0}}),
    ({"rope_scaling": YARN},
     {"rope_scaling": {"type": "yarn", "factor": 4.0, "original_max_position": 1024}}),
    ({"rope_scaling": {"rope_type": "yarn", "factor": 4.0, "attention_factor": 1.0,
                       "beta_fast": 16}},
     {"rope_scaling": {"type": "yarn", "factor": 4.0, "attention_factor": 1.0, "beta_fast": 16,
                       "original_max_position": 4096}}),
    ({"rope_scaling": {"rope_type": "banded", "factor": 8.0, "low_freq_factor": 1.0,
                       "high_freq_factor": 4.0, "original_max_position_embeddings": 512}},
     {"rope_scaling": {"type": "banded", "factor": 8.0, "low_freq_factor": 1.0,
                       "high_freq_factor": 4.0, "original_max_position": 512}}),
])
def test_checkpoints_reach_the_bounded_forms(tmp_path, keys, fields):
    path = tmp_path / "config.json"
    path.write_text(json.dumps(CHECKPOINT | keys))
    config = ModelConfig.from_file(path)
    plain = dict(num_layers=4, hidden_size=64, num_heads=4, num_kv_heads=2, rope_theta=1e6,
                 rms_norm_eps=1e-6)
    assert config == ModelConfig(**plain, **fields)
    if config.rope_scaling:
        ops.rope_frequencies(16, 1e6, config.rope_scaling, device="cpu")


@pytest.mark.parametrize("keys", [
    {"sliding_window": 2048, "use_sliding_window": True, "max_window_layers": 3},
    {"sliding_window": 2048, "layer_types": ["sliding_attention", "full_attention"] * 2},
    {"sliding_window": 2048, "layer_types": ["chunked_attention"] * 4},
    {"layer_types": ["sliding_attention"] * 4}, {"partial_rotary_factor": 0.3},
    {"partial_rotary_factor": 2.0}, {"rope_scaling": {"type": "dynamic", "factor": 2.0}},
    {"rope_scaling": {"type": "default", "sections": [1, 2]}},
    {"rope_scaling": dict(YARN, mscale=0.7)}, {"rope_scaling": dict(YARN, truncate=False)},
    {"rope_scaling": YARN, "rope_parameters": {"rope_type": "default"}},
    {"rope_parameters": {"rope_type": "default", "rope_theta": 5e5}},
])
def test_checkpoint_forms_without_a_kernel_are_refused(tmp_path, keys):
    path = tmp_path / "config.json"
    path.write_text(json.dumps(CHECKPOINT | keys))
    with pytest.raises(ValueError):
        ModelConfig.from_file(path)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (5, 2), (9, 30), (100, 3)])
def test_attention_flops_count_the_visible_keys(window, sinks):
    config = ModelConfig(**TINY, attention_window=window, attention_sinks=sinks)
    weights = random_weights(config, vocab_size=50, intermediate_size=16)
    model = TorchModel(config, weights, device="cpu", dtype=torch.float32, max_position=64)
    starts, lengths = [0, 3, 17, 40], [6, 1, 12, 1]
    seen = sum(1 for s, n in zip(starts, lengths) for p in range(s, s + n)
               for j in range(p + 1) if not window or j < sinks or j > p - window)
    assert model._attention_flops(starts, lengths) == 4 * 4 * 8 * seen




def test_fork_sequence_composes_the_child_prompt():
    config = ModelConfig(**TINY)
    model = TorchModel(config, random_weights(config, vocab_size=50, intermediate_size=16),
                       device="cpu", dtype=torch.float32, max_position=64)
    backend = PagedBackend(model, num_blocks=16, block_size=4, prefill_chunk=8, max_seqs=8)
    a = backend.start_sequence([1, 2, 3, 4, 5])
    seq = backend._sequences[a]
    # Four prompt tokens cached (one whole block), one still to come.
    seq.cache.reserve(4)
    seq.cache.advance(4)
    for _ in range(4):
        seq.pending.popleft()
    b = backend.fork_sequence(a, [7, 8])
    child = backend._sequences[b]
    assert list(child.pending) == [5, 7, 8] and child.cache.length == 4
    assert backend.pool.block_table(b) == backend.pool.block_table(a)
    # The parent generates: its last token comes first in the child's prompt.
    seq.pending.clear()
    seq.next_token = 11
    c = backend.fork_sequence(a, [9])
    assert list(backend._sequences[c].pending) == [11, 9]
    assert backend._sequences[c].next_token is None
    d = backend.fork_sequence(a, [])
    assert not backend._sequences[d].pending and backend._sequences[d].next_token == 11
    seq.finished = True
    with pytest.raises(RuntimeError, match="finished"):
        backend.fork_sequence(a, [])
    seq.feeds = object()
    with pytest.raises(RuntimeError, match="unfinished"):
        backend.fork_sequence(a, [1])
    for s in (a, b, c, d):
        backend.release_sequence(s)
    assert backend.blocks_in_use == 0


@pytest.mark.parametrize("window,sinks,block,chunk", [
    (1, 0, 1, 1), (70, 5, 16, 32), (64, 16, 16, 16), (5, 33, 4, 9), (100, 0, 7, 1), (3, 2, 16, 40)])
def test_sequence_blocks_bound_what_a_windowed_sequence_holds(window, sinks, block, chunk):
    config = ModelConfig(**TINY, attention_window=window, attention_sinks=sinks)
    model = TorchModel(config, random_weights(config, vocab_size=50, intermediate_size=16),
                       device="cpu", dtype=torch.float32, max_position=4096)
    backend = PagedBackend(model, num_blocks=400, block_size=block, prefill_chunk=chunk,
                           max_seqs=64)
    rng = random.Random(window)
    most = 0
    for seq in range(30):
        cache = backend.pool.new_cache(seq)
        cache.reserve(0)
        while cache.length < 700:
            n = rng.choice([1, rng.randint(1, chunk), chunk])
            cache.reserve(n)
            most = max(most, sum(b != EMPTY_BLOCK for b in backend.pool.block_table(seq)))
            cache.advance(n)
            backend.pool.trim(cache, window, sinks)
        backend.pool.release(cache)
    assert 0.9 * backend.sequence_blocks - 1 <= most <= backend.sequence_blocks
    budget = backend.block_budget()
    assert budget.fits_ever(4096 // block * block) and not budget.fits_ever(4096 + block)
    budget.try_reserve(4000)
    assert 400 - budget.available == min(-(-4000 // block), backend.sequence_blocks)
    budget.try_reserve(1)
    budget.release(4000)
    assert budget.available == 399


def test_without_a_window_the_budget_is_the_plain_one():
    model = TorchModel(ModelConfig(**TINY), random_weights(ModelConfig(**TINY), vocab_size=50,
                                                           intermediate_size=16),
                       device="cpu", dtype=torch.float32, max_position=64)
    backend = PagedBackend(model, num_blocks=10, block_size=4, prefill_chunk=8, max_seqs=8)
    assert backend.sequence_blocks is None
    budget = backend.block_budget()
    assert budget.fits_ever(40) and not budget.fits_ever(41)
    assert budget.try_reserve(37) and budget.available == 0


def test_only_rotary_tables_limit_positions():
    for kw, limited in (({}, True), ({"rope_scaling": {"type": "linear", "factor": 2.0}}, False)):
        config = ModelConfig(**TINY, **kw)
        model = TorchModel(config, random_weights(config, vocab_size=50, intermediate_size=16),
                           device="cpu", dtype=torch.float32, max_position=64)
        model._check_positions([60, 0], [4, 64])
        if limited:
            with pytest.raises(RuntimeError, match="rotary table"):
                model._check_positions([0, 64], [1, 1])
        else:
            model._check_positions([0, 64], [1, 1])


class Ids:
    """A launched step whose ids are known."""

    def __init__(self, ids):
        self._ids = ids

    def ref(self, i):
        return -1 - i

    def result(self):
        return self._ids


def test_fork_of_a_sequence_that_ended_with_a_step_in_flight(monkeypatch):
    # The pipelined loop launches one step past an end-of-generation token.
    config = ModelConfig(**TINY)
    model = TorchModel(config, random_weights(config, vocab_size=50, intermediate_size=16),
                       device="cpu", dtype=torch.float32, max_position=64)
    end = 49
    answers = iter([[5], [end], [7]])

    def launch_tokens(groups):
        for tokens, cache in groups:
            cache.reserve(len(tokens))
            cache.advance(len(tokens))
        return Ids(next(answers))

    monkeypatch.setattr(model, "launch_tokens", launch_tokens)

    class Vocab:
        def is_end_of_generation(self, token):
            return token == end

    backend = PagedBackend(model, num_blocks=16, block_size=4, prefill_chunk=8, vocab=Vocab(),
                           max_seqs=8)
    s = backend.start_sequence([1, 2])
    first = backend.launch()
    second = backend.launch()
    backend.finish(first)
    third = backend.launch()  # the host does not know yet that `end` was generated
    assert backend.finish(second)[s].finished
    with pytest.raises(RuntimeError, match="unfinished"):
        backend.fork_sequence(s, [8, 9])
    assert backend.finish(third) == {}
    child = backend._sequences[backend.fork_sequence(s, [8, 9])]
    # 1 2, 5 and the ending token are cached: a whole block, so that nothing is copied.
    assert child.cache.length == 4 and list(child.pending) == [8, 9]
    assert child.next_token is None
    with pytest.raises(RuntimeError, match="finished"):
        backend.fork_sequence(s, [])


def test_forks_and_compactions_that_cannot_copy_change_nothing():
    # A pool without a GPU has no kernel for its copies.
    config = ModelConfig(**TINY)
    model = TorchModel(config, random_weights(config, vocab_size=50, intermediate_size=16),
                       device="cpu", dtype=torch.float32, max_position=64)
    backend = PagedBackend(model, num_blocks=16, block_size=4, prefill_chunk=8, max_seqs=4)
    pool = backend.pool
    cache = pool.new_cache(100)
    cache.reserve(6)
    cache.advance(6)
    alloc = pool.allocator
    before = (dict(alloc._tables), sorted(alloc._free), list(alloc._free_rows), dict(alloc._refs))
    with pytest.raises(RuntimeError):
        pool.fork(cache, 101)
    table = list(pool.block_table(100))
    assert alloc.moves() and min(table) > 2
    with pytest.raises(RuntimeError):
        pool.compact()
    after = (dict(alloc._tables), sorted(alloc._free), list(alloc._free_rows), dict(alloc._refs))
    assert after == before and pool.block_table(100) == table


# ------------------------------------------------------------------ refusals of the C ABI


def window_args(**change):
    """A valid bs_window_attention_batched call (no pointer is read before the
    checks are done; zero sequences, so nothing is launched)."""
    args = dict(query=1, q_stride=64 * 4, key_pool=1, value_pool=1, tables=1, table_stride=8,
                table_rows=2, seq_rows=None, lens=1, num_seqs=0, heads=4, kv_heads=2, head_dim=64,
                block_size=16, num_blocks=8, max_blocks=8, dtype=0, scaling=0.125, window=32,
                sinks=4, out=1, o_stride=64 * 4, ws=None, ws_bytes=0, status=None, stream=None)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=7), "dtype"), (dict(num_seqs=-1), "count"), (dict(heads=5), "groups"),
    (dict(kv_heads=0), "groups"), (dict(head_dim=0), "positive"), (dict(block_size=0), "positive"),
    (dict(num_blocks=0), "positive"), (dict(max_blocks=9), "max_blocks"),
    (dict(max_blocks=0), "positive"), (dict(table_rows=0), "table_rows"),
    (dict(window=0), "window"), (dict(window=-3), "window"), (dict(sinks=-1), "sinks"),
    (dict(q_stride=100), "strides"), (dict(o_stride=100), "strides"),
    (dict(head_dim=264, q_stride=4096, o_stride=4096), "head_dim"),
    (dict(heads=34, q_stride=4096, o_stride=4096), "groups"),
    (dict(max_blocks=1 << 27, table_stride=1 << 27), "2\\^30"),
    (dict(num_blocks=1 << 28), "2\\^31"),
])
def test_window_attention_refuses(change, message):
    assert _lib.lib().bs_window_attention_batched(*window_args()) == 0
    with pytest.raises(RuntimeError, match=message):
        _lib.check(_lib.lib().bs_window_attention_batched(*window_args(**change)))


def test_window_prefill_refuses_bad_sizes():
    lib = _lib.lib()

    def call(**change):
        args = dict(query=1, q_stride=256, cu_q=1, num_rows=0, num_tokens=0, max_query_len=5,
                    lens=1, seq_rows=None, key_pool=1, value_pool=1, tables=1, table_stride=8,
                    table_rows=2, max_blocks=8, heads=4, kv_heads=2, head_dim=64, block_size=16,
                    num_blocks=8, dtype=0, scaling=0.125, window=32, sinks=4, out=1, o_stride=256,
                    ws=None, ws_bytes=0, status=None, stream=None)
        args.update(change)
        return lib.bs_window_prefill_attention(*args.values())

    assert call() == 0
    for change in (dict(window=0), dict(sinks=-1), dict(max_query_len=-1), dict(num_tokens=-2),
                   dict(num_rows=2, num_tokens=4, max_query_len=0),
                   dict(num_rows=2, num_tokens=4, cu_q=None)):
        assert call(**change) != 0, change


def rotary_call(**change):
    args = dict(qkv=1, stride=512, dtype=0, freq=1, rotary_dim=64, inter=0, amp=1.0, pos=1, slots=1,
                tokens=0, heads=4, kv_heads=2, head_dim=64, q=1, k=1, v=1, pool_dtype=0,
                num_blocks=8, block_size=16, status=None, stream=None)
    args.update(change)
    return _lib.lib().bs_rotary_append(*args.values())


@pytest.mark.parametrize("change", [
    dict(dtype=3), dict(pool_dtype=-1), dict(tokens=-1), dict(heads=0), dict(kv_heads=0),
    dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=66), dict(amp=math.nan),
    dict(amp=math.inf), dict(stride=511), dict(num_blocks=0), dict(block_size=0),
    dict(num_blocks=1 << 30), dict(tokens=1, freq=None), dict(tokens=1, slots=None),
])
def test_rotary_append_refuses(change):
    assert rotary_call() == 0
    assert rotary_call(**change) != 0


@pytest.mark.parametrize("change", [
    dict(dtype=5), dict(layers=0), dict(kv_heads=0), dict(num_blocks=0), dict(block_size=-1),
    dict(head_dim=0), dict(pairs=-1), dict(num_blocks=1 << 31), dict(layers=1 << 60),
    dict(pairs=2, src=None), dict(pairs=2, k=None),
])
def test_copy_blocks_refuses(change):
    base = dict(k=1, v=1, dtype=0, layers=2, kv_heads=2, num_blocks=8, block_size=16, head_dim=64,
                src=1, dst=1, pairs=0, status=None, stream=None)
    lib = _lib.lib()
    assert lib.bs_copy_blocks(*base.values()) == 0
    assert lib.bs_copy_blocks(*dict(base, **change).values()) != 0


def test_workspace_queries_refuse_a_null_result():
    lib = _lib.lib()
    null = ctypes.POINTER(ctypes.c_uint64)()
    assert lib.bs_window_attention_batched_workspace_bytes(1, 4, 2, 64, 16, 8, 0, 32, 4, null) != 0
    assert lib.bs_window_prefill_attention_workspace_bytes(8, 1, 8, 4, 2, 64, 16, 8, 0, 32, 4,
                                                           null) != 0


@pytest.mark.parametrize("name", ["window_attention_batched", "window_prefill_attention",
                                  "rotary_append", "copy_blocks"])
def test_operators_refuse_host_tensors(name):
    z = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    calls = {
        "window_attention_batched": lambda: ops.window_attention_batched(
            z, pool, pool, i[None], i, 1.0, 4),
        "window_prefill_attention": lambda: ops.window_prefill_attention(
            z, pool, pool, i[None], i, i, 1.0, 1, 4),
        "rotary_append": lambda: ops.rotary_append(z.view(1, -1), i.double(), i, i, pool, pool, 0),
        "copy_blocks": lambda: ops.copy_blocks(pool, pool, i, i),
    }
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        calls[name]()


@pytest.mark.parametrize("theta, scaling", [
    (1e4, {"type": "linear"}),
    (1e4, {"type": "yarn", "factor": 4.0}),
    (1e4, {"type": "yarn", "factor": 4.0, "original_max_position": -1}),
    (1e4, {"type": "yarn", "factor": 4.0, "original_max_position": 4096, "beta_fast": 0.0}),
    (1.0, {"type": "yarn", "factor": 4.0, "original_max_position": 4096}),
    (1e4, {"type": "banded", "factor": 4.0, "original_max_position": 4096,
           "low_freq_factor": 1.0}),
    (1e4, {"type": "ntk", "factor": float("inf")}),
    (1e4, {}),
])
def test_incomplete_scaling_is_refused(theta, scaling):
    with pytest.raises(RuntimeError):
        ops.rope_frequencies(64, theta, scaling, device="cpu")

"""The engine on a model with a sliding window, sink tokens and a scaled, partial,
interleaved rotary embedding: every operator of the bounded cache together, with
forks, trimming and compaction while sequences run.

The reference is the model's formula over a whole token sequence at once, in 64
bits, on the weights the engine holds.  A generated token must be a near-maximum of
the reference's logits at its position, given the tokens before it: within twice the
engine's logit error.  That error is held to 1e-3 of the largest logit in fp32 (as
the full-attention engine's); in bf16 each of the roughly 13 roundings of a layer
and of the head may move the hidden state by 2^-8 of itself: 2 layers, 27 roundings,
0.11 of the largest logit if they all pushed one way.
"""

import dataclasses

import numpy as np
import pytest
import torch

from batchstream_inference_engine_b200 import ops
from batchstream_inference_engine_b200.backend import PagedBackend
from batchstream_inference_engine_b200.serve import BlockBudget, serve
from batchstream_inference_engine_b200.torch_model import (ModelConfig, PagedKVPool, TorchModel,
                                                          random_weights)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VOCAB = 640
CONFIG = ModelConfig(num_layers=2, hidden_size=256, num_heads=4, num_kv_heads=2, rope_theta=1e4,
                     rms_norm_eps=1e-6, attention_window=70, attention_sinks=5, rotary_dim=32,
                     rope_interleaved=True,
                     rope_scaling={"type": "yarn", "factor": 8.0, "original_max_position": 512})
REL = {torch.float32: 1e-3, torch.bfloat16: 27 * 2.0 ** -8}


def weights_of(config=CONFIG):
    return random_weights(config, vocab_size=VOCAB, intermediate_size=384, seed=3, std=0.08)


def reference_logits(config, weights, tokens, dtype):
    """Logits [n, vocab] of every position in 64 bits."""
    w = {k: v.to(dtype).double().to(DEV) for k, v in weights.items()}
    n, H, Hkv, D = len(tokens), config.num_heads, config.num_kv_heads, config.head_dim
    x = w["model.embed_tokens.weight"][torch.tensor(tokens, device=DEV)]

    def norm(x, weight):
        return weight * x * torch.rsqrt((x * x).mean(-1, keepdim=True) + config.rms_norm_eps)

    rd = config.rotary_dim or D
    freq, amp = ops.rope_frequencies(rd, config.rope_theta, config.rope_scaling, device=DEV)
    turn = torch.polar(torch.full((n, rd // 2), amp, dtype=torch.float64, device=DEV),
                       torch.arange(n, device=DEV)[:, None] * freq)[:, None]

    def rotate(x):
        z = torch.view_as_complex(x[..., :rd].reshape(*x.shape[:-1], rd // 2, 2)) * turn
        return torch.cat([torch.view_as_real(z).flatten(-2), x[..., rd:]], -1)

    p = torch.arange(n, device=DEV)
    see = (p[None] <= p[:, None]) & ((p[None] < config.attention_sinks)
                                     | (p[None] > p[:, None] - config.attention_window))
    for layer in range(config.num_layers):
        pre = f"model.layers.{layer}."
        lin = lambda name, x: x @ w[pre + name + ".weight"].t() + w.get(pre + name + ".bias", 0)  # noqa: E731,B023
        y = norm(x, w[pre + "input_layernorm.weight"])
        q = rotate(lin("self_attn.q_proj", y).view(n, H, D)).view(n, Hkv, H // Hkv, D)
        k = rotate(lin("self_attn.k_proj", y).view(n, Hkv, D))
        v = lin("self_attn.v_proj", y).view(n, Hkv, D)
        s = torch.einsum("thgd,jhd->hgtj", q, k) * D ** -0.5
        a = torch.softmax(s.masked_fill(~see, float("-inf")), -1)
        x = x + lin("self_attn.o_proj", torch.einsum("hgtj,jhd->thgd", a, v).reshape(n, H * D))
        y = norm(x, w[pre + "post_attention_layernorm.weight"])
        gate = torch.nn.functional.silu(lin("mlp.gate_proj", y))
        x = x + lin("mlp.down_proj", gate * lin("mlp.up_proj", y))
    return norm(x, w["model.norm.weight"]) @ w["model.embed_tokens.weight"].t()


def check_generated(weights, prompt, generated, dtype):
    logits = reference_logits(CONFIG, weights, prompt + generated, dtype)
    rows = logits[len(prompt) - 1: len(prompt) - 1 + len(generated)]
    picked = rows[torch.arange(len(generated)), torch.tensor(generated, device=DEV)]
    slack = 2 * REL[dtype] * rows.abs().amax(-1)
    assert bool((picked >= rows.amax(-1) - slack).all())


class NoEnd:
    """Ids only; no token ends generation."""

    def is_end_of_generation(self, token):
        return False


@pytest.fixture
def exact_gemm():
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = prev


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pipelined,graphs", [(False, False), (False, True), (True, True)])
def test_served_tokens(exact_gemm, dtype, pipelined, graphs):
    weights = weights_of()
    model = TorchModel(CONFIG, weights, device=DEV, dtype=dtype, max_position=1024,
                       step_graphs=graphs, max_graph_batch=16, max_graph_prefill=128)
    backend = PagedBackend(model, num_blocks=96, block_size=16, prefill_chunk=96, vocab=NoEnd(),
                           max_seqs=16)
    rng = np.random.default_rng(1)
    specs = [(rng.integers(0, VOCAB, int(n)).tolist(), int(m))
             for n, m in zip((3, 200, 70, 71, 30, 410, 1, 64), (150, 20, 40, 8, 60, 12, 100, 30))]
    requests = serve(backend, specs, 5, BlockBudget(96, 16), pipelined=pipelined)
    assert not any(r.failed for r in requests) and backend.blocks_in_use == 0
    for (prompt, n), request in zip(specs, requests):
        assert len(request.tokens) == n
        check_generated(weights, prompt, request.tokens, dtype)


def test_logits_along_a_long_sequence(exact_gemm):
    # fp32 logits, one chunk and then single tokens, 400 tokens through a window of 70.
    weights = weights_of()
    model = TorchModel(CONFIG, weights, device=DEV, dtype=torch.float32, max_position=1024)
    pool = PagedKVPool(CONFIG, 40, 16, device=DEV, dtype=torch.float32)
    pool.keys.fill_(float("nan"))
    pool.values.fill_(float("nan"))
    cache = pool.new_cache(0)
    tokens = np.random.default_rng(2).integers(0, VOCAB, 400).tolist()
    ref = reference_logits(CONFIG, weights, tokens, torch.float32)
    at = 0
    for n in (150, 90, 1, 1, 1, 17, 1, 64, 1, 1):
        got = model.forward_batch([(tokens[at: at + n], cache)])[0].double()
        at += n
        want = ref[at - 1]
        assert float((got - want).abs().max()) <= 1e-3 * float(want.abs().max()), at
        # One sink block, and at most ceil(70 / 16) + 1 blocks of the window.
        assert 40 - pool.free_blocks <= 1 + 6
    ops.take_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("graphs", [False, True])
def test_forks_and_compaction_between_steps(exact_gemm, dtype, graphs):
    weights = weights_of()
    model = TorchModel(CONFIG, weights, device=DEV, dtype=dtype, max_position=1024,
                       step_graphs=graphs, max_graph_batch=16, max_graph_prefill=128)
    backend = PagedBackend(model, num_blocks=64, block_size=16, prefill_chunk=96, vocab=NoEnd(),
                           max_seqs=16)
    rng = np.random.default_rng(4)
    prompts = {backend.start_sequence(p): p
               for p in (rng.integers(0, VOCAB, 130).tolist(), rng.integers(0, VOCAB, 20).tolist())}
    tokens = {s: [] for s in prompts}

    def steps(n):
        for _ in range(n):
            for s, out in backend.step().items():
                tokens[s].append(out.token)

    steps(9)
    a, b = list(prompts)
    # Two children of a with other suffixes, one that goes on as a does, and one of b.
    suffixes = [rng.integers(0, VOCAB, 5).tolist(), rng.integers(0, VOCAB, 100).tolist(), []]
    for suffix in suffixes:
        child = backend.fork_sequence(a, suffix)
        prompts[child] = prompts[a] + tokens[a] + suffix
        tokens[child] = []
    twin = child
    child = backend.fork_sequence(b, [7])
    prompts[child] = prompts[b] + tokens[b] + [7]
    tokens[child] = []
    done = len(tokens[a])
    steps(6)
    backend.release_sequence(b)
    assert backend.compact() > 0
    used = 64 - backend.pool.free_blocks
    assert all(x < used for s in tokens if s != b for x in backend.pool.block_table(s))
    finished = tokens.pop(b)
    steps(40)
    check_generated(weights, prompts[b], finished, dtype)
    for s, generated in tokens.items():
        assert generated
        check_generated(weights, prompts[s], generated, dtype)
    assert len(tokens[twin]) == len(tokens[a]) - done
    if dtype == torch.float32:  # the same inputs along the same path, up to near-ties
        check_generated(weights, prompts[twin], tokens[a][done:], dtype)
    for s in tokens:
        backend.release_sequence(s)
    assert backend.blocks_in_use == 0
    assert ops.take_status() == 0


def test_fork_refuses_while_a_step_is_in_flight(exact_gemm):
    model = TorchModel(CONFIG, weights_of(), device=DEV, dtype=torch.bfloat16, max_position=256)
    backend = PagedBackend(model, num_blocks=32, block_size=16, prefill_chunk=64, vocab=NoEnd())
    s = backend.start_sequence([1, 2, 3])
    launched = backend.launch()
    with pytest.raises(RuntimeError, match="unfinished"):
        backend.fork_sequence(s, [4])
    backend.finish(launched)
    backend.fork_sequence(s, [4])


@pytest.mark.parametrize("graphs", [False, True])
def test_scaled_rotary_before_full_attention(exact_gemm, graphs, monkeypatch):
    # Without a window the full decode follows the rotary append directly and starts
    # ahead of its end: the same tokens as without that overlap.
    config = dataclasses.replace(CONFIG, attention_window=0, attention_sinks=0)
    weights = weights_of()
    rng = np.random.default_rng(8)
    specs = [(rng.integers(0, VOCAB, int(n)).tolist(), 24) for n in (300, 5, 90, 1, 200, 33, 64, 17)]
    served = []
    for overlap in (True, False):
        if not overlap:
            plain = ops.paged_attention_batched
            monkeypatch.setattr(ops, "paged_attention_batched",
                                lambda *a, **kw: plain(*a, **{**kw, "after_append": False}))
        model = TorchModel(config, weights, device=DEV, dtype=torch.bfloat16, max_position=1024,
                           step_graphs=graphs, max_graph_batch=16, max_graph_prefill=128)
        backend = PagedBackend(model, num_blocks=128, block_size=16, prefill_chunk=96,
                               vocab=NoEnd(), max_seqs=16)
        requests = serve(backend, specs, 8, BlockBudget(128, 16))
        assert not any(r.failed for r in requests)
        served.append([r.tokens for r in requests])
    assert served[0] == served[1]


def test_default_rotary_over_frequencies_and_a_full_window(exact_gemm):
    # A window that covers the sequence and the plain frequencies in half layout:
    # linear scaling by 1 takes the new operators through the reference's model.
    config = dataclasses.replace(CONFIG, attention_window=1 << 20, attention_sinks=0, rotary_dim=0,
                                 rope_interleaved=False,
                                 rope_scaling={"type": "linear", "factor": 1.0})
    plain = dataclasses.replace(config, attention_window=0, rope_scaling=None)
    weights = weights_of()
    tokens = np.random.default_rng(5).integers(0, VOCAB, 90).tolist()
    logits = []
    for c in (config, plain):
        model = TorchModel(c, weights, device=DEV, dtype=torch.float32, max_position=256)
        pool = PagedKVPool(c, 16, 16, device=DEV, dtype=torch.float32)
        logits.append(model.forward_batch([(tokens, pool.new_cache(0))])[0])
    # The table-driven embedding rounds cos and sin to bf16 (2^-9 of 1 each), so q and k
    # are off by up to 2^-8 of themselves; through 2 layers of scores and values.
    assert float((logits[0] - logits[1]).abs().max()) <= 0.05 * float(logits[1].abs().max())


@pytest.mark.parametrize("graphs", [False, True])
def test_a_skipped_block_copy_fails_the_next_step_of_any_model(exact_gemm, graphs):
    # Block copies report in the second status word, which a model without a window or
    # another rotary form does not write otherwise.
    config = ModelConfig(num_layers=2, hidden_size=256, num_heads=4, num_kv_heads=2,
                         rope_theta=1e4, rms_norm_eps=1e-6)
    model = TorchModel(config, weights_of(config), device=DEV, dtype=torch.bfloat16,
                       max_position=256, step_graphs=graphs, max_graph_batch=4)
    backend = PagedBackend(model, num_blocks=32, block_size=16, prefill_chunk=64, vocab=NoEnd(),
                           max_seqs=4)
    a = backend.start_sequence(list(range(1, 20)))
    backend.step()
    child = backend.fork_sequence(a, [5])
    backend.step()
    backend.step()
    backend.pool._copy([(3, 4), (5, 4)])  # clashing pairs, as a broken allocator would give
    with pytest.raises(RuntimeError, match="named by another pair"):
        backend.step()
    backend.step()
    for s in (a, child):
        backend.release_sequence(s)


@pytest.mark.parametrize("pipelined,graphs", [(False, False), (True, True)])
def test_conversations_longer_than_the_pool(exact_gemm, pipelined, graphs):
    # 20 blocks hold 320 tokens; each request runs to between 330 and 700.
    weights = weights_of()
    model = TorchModel(CONFIG, weights, device=DEV, dtype=torch.float32, max_position=1024,
                       step_graphs=graphs, max_graph_batch=8, max_graph_prefill=64)
    backend = PagedBackend(model, num_blocks=20, block_size=16, prefill_chunk=32, vocab=NoEnd(),
                           max_seqs=4)
    assert backend.sequence_blocks == 9  # one of the sinks, eight of 69 + 32 tokens
    rng = np.random.default_rng(9)
    specs = [(rng.integers(0, VOCAB, n).tolist(), m) for n, m in ((500, 200), (10, 400), (330, 3))]
    requests = serve(backend, specs, 4, backend.block_budget(), pipelined=pipelined)
    assert not any(r.failed for r in requests) and backend.blocks_in_use == 0
    for (prompt, n), request in zip(specs, requests):
        assert len(request.tokens) == n
        check_generated(weights, prompt, request.tokens, torch.float32)

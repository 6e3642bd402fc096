"""The engine on a 4-bit cache, and its steps with drafted tokens.

The reference is the model's formula over a whole token sequence at once, in 64 bits, on the
weights the engine holds and on the keys and values that its cache holds (read back, so that
an element which the engine's rounding moved across the border of two codes is the same on
both sides); the tolerances are those of test_bounded_engine_gpu.  What the cache holds must be
within its step, |s|, of the formula's own keys and values.
"""

import dataclasses

import pytest
import torch

from batchstream_inference_engine_b200 import ops
from batchstream_inference_engine_b200.backend import PagedBackend
from batchstream_inference_engine_b200.torch_model import (ModelConfig, PagedKVPool, TorchModel,
                                                          random_weights)

from . import int4_format as fmt
from .test_bounded_engine_gpu import REL, VOCAB

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CONFIG = ModelConfig(num_layers=2, hidden_size=256, num_heads=4, num_kv_heads=2, rope_theta=1e4,
                     rms_norm_eps=1e-6)
WINDOWED = dataclasses.replace(CONFIG, attention_window=70, attention_sinks=5, rotary_dim=32,
                               rope_interleaved=True)


def weights_of(config=CONFIG):
    return random_weights(config, vocab_size=VOCAB, intermediate_size=384, seed=3, std=0.08)


def backend_of(config=CONFIG, dtype=torch.float32, pool=torch.uint8, graphs=True, blocks=64,
               chunk=48):
    model = TorchModel(config, weights_of(config), device=DEV, dtype=dtype, max_position=4096,
                       step_graphs=graphs)
    return PagedBackend(model, blocks, 16, chunk, max_seqs=8, pool_dtype=pool)


def held_rows(pool, cache):
    """What the pool holds for a sequence: per layer (keys, values) [n, Hkv, D]."""
    table = pool.allocator.block_table(cache.seq_id)
    slots = torch.tensor([table[p // 16] * 16 + p % 16 for p in range(cache.length)],
                         dtype=torch.int32, device=DEV)
    return [ops.read_int4(k, v, slots) for k, v in zip(pool.keys, pool.values)]


def reference_logits(weights, tokens, dtype, held):
    """Logits [n, vocab] of every position in 64 bits, over the cached keys and values."""
    c = CONFIG
    w = {k: v.to(dtype).double().to(DEV) for k, v in weights.items()}
    n, H, Hkv, D = len(tokens), c.num_heads, c.num_kv_heads, c.head_dim
    x = w["model.embed_tokens.weight"][torch.tensor(tokens, device=DEV)]

    def norm(x, weight):
        return weight * x * torch.rsqrt((x * x).mean(-1, keepdim=True) + c.rms_norm_eps)

    freq, _ = ops.rope_frequencies(D, c.rope_theta, device=DEV)
    angle = (torch.arange(n, device=DEV)[:, None] * freq)[:, None]

    def rotate(x):
        a, b = x[..., : D // 2], x[..., D // 2:]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    p = torch.arange(n, device=DEV)
    see = p[None] <= p[:, None]
    for layer in range(c.num_layers):
        pre = f"model.layers.{layer}."
        lin = lambda name, x: x @ w[pre + name + ".weight"].t() + w.get(pre + name + ".bias", 0)  # noqa: E731,B023
        y = norm(x, w[pre + "input_layernorm.weight"])
        q = rotate(lin("self_attn.q_proj", y).view(n, H, D)).view(n, Hkv, H // Hkv, D)
        own = (rotate(lin("self_attn.k_proj", y).view(n, Hkv, D)), lin("self_attn.v_proj", y).view(n, Hkv, D))
        k, v = (t.double() for t in held[layer])
        for got, want in zip((k, v), own):
            # Off by |s| at most, and by the engine's own error of the row.
            scale = fmt.quantise(want)[1].abs().repeat_interleave(32, -1)
            slack = REL[dtype] * want.abs().amax()
            assert bool(((got - want).abs() <= 1.2 * scale + 2 * slack).all())
        s = torch.einsum("thgd,jhd->hgtj", q, k) * D ** -0.5
        a = torch.softmax(s.masked_fill(~see, float("-inf")), -1)
        x = x + lin("self_attn.o_proj", torch.einsum("hgtj,jhd->thgd", a, v).reshape(n, H * D))
        y = norm(x, w[pre + "post_attention_layernorm.weight"])
        gate = torch.nn.functional.silu(lin("mlp.gate_proj", y))
        x = x + lin("mlp.down_proj", gate * lin("mlp.up_proj", y))
    return norm(x, w["model.norm.weight"]) @ w["model.embed_tokens.weight"].t()


def check_generated(backend, seq_id, prompt, generated, dtype):
    """Each generated token is a near-maximum of the reference's logits."""
    cache = backend._sequences[seq_id].cache
    text = (prompt + generated)[: cache.length]
    logits = reference_logits(weights_of(), text, dtype, held_rows(backend.pool, cache))
    rows = logits[len(prompt) - 1:]
    picked = torch.tensor((prompt + generated)[len(prompt): len(prompt) + rows.shape[0]], device=DEV)
    rows = rows[: picked.numel()]
    short = rows.amax(-1) - rows.gather(1, picked[:, None])[:, 0]
    assert bool((short <= 2 * REL[dtype] * rows.abs().amax()).all())


def prompts(lengths=(50, 7, 33), seed=4):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in lengths]


def generate(backend, texts, steps):
    ids = [backend.start_sequence(t) for t in texts]
    out = {i: [] for i in ids}
    while min(len(v) for v in out.values()) < steps:
        for i, o in backend.step().items():
            out[i].append(o.token)
    return ids, out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("graphs", [False, True])
def test_engine_on_a_4_bit_cache(dtype, graphs):
    backend = backend_of(dtype=dtype, graphs=graphs)
    texts = prompts()
    ids, out = generate(backend, texts, 20)
    for i, text in zip(ids, texts):
        check_generated(backend, i, text, out[i], dtype)
    assert ops.take_status() == 0


def test_forks_and_compaction_of_a_4_bit_cache():
    backend = backend_of(dtype=torch.bfloat16)
    text = prompts((37,))[0]
    (parent,), out = generate(backend, [text], 5)
    child = backend.fork_sequence(parent, [])
    other = backend.fork_sequence(parent, [9, 8, 7])
    more = {parent: [], child: [], other: []}
    for _ in range(6):
        for i, o in backend.step().items():
            more[i].append(o.token)
    assert more[parent] == more[child]
    backend.release_sequence(parent)
    assert backend.compact() > 0
    for _ in range(4):
        for i, o in backend.step().items():
            more[i].append(o.token)
    check_generated(backend, child, text, out[parent] + more[child], torch.bfloat16)
    check_generated(backend, other, text + out[parent] + [9, 8, 7], more[other], torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_windowed_engine_on_a_4_bit_cache(dtype):
    # Far past the window, with trimmed blocks: graphs and eager steps agree.
    texts = prompts((130, 20))
    runs = []
    for graphs in (False, True):
        backend = backend_of(WINDOWED, dtype=dtype, graphs=graphs, blocks=24)
        _, out = generate(backend, texts, 60)
        assert backend.blocks_in_use <= 2 * backend.sequence_blocks
        runs.append([v[:60] for v in out.values()])
    same = [[a == b for a, b in zip(x, y)] for x, y in zip(*runs)]
    # (Another GEMM in the padded step may turn a near-tie: the first tokens are the same.)
    assert all(all(s[:8]) for s in same)
    assert ops.take_status() == 0


@pytest.mark.parametrize("pool", [torch.float32, torch.uint8])
def test_draft_steps_give_the_tokens_of_plain_steps(pool):
    texts = prompts()
    ids, want = generate(backend_of(pool=pool), texts, 80)
    backend = backend_of(pool=pool)
    ids, out = generate(backend, texts, 1)
    g = torch.Generator().manual_seed(5)
    accepted = 0
    for turn in range(12):
        drafts = {}
        for i in ids:
            n = int(torch.randint(0, 5, (1,), generator=g))
            follow = want[i][len(out[i]): len(out[i]) + n]
            if follow and turn % 3 == 2:  # the last draft is wrong
                follow[-1] = (follow[-1] + 1) % VOCAB
            drafts[i] = follow
        steps = backend.draft_step(drafts)
        for i in ids:
            tokens = [o.token for o in steps[i]]
            assert 1 <= len(tokens) <= len(drafts[i]) + 1
            assert tokens[:-1] == drafts[i][: len(tokens) - 1]
            if pool == torch.float32 and turn % 3 != 2:
                assert len(tokens) == len(drafts[i]) + 1  # all right, all accepted
            accepted += len(tokens) - 1
            out[i] += tokens
            cache = backend._sequences[i].cache
            assert cache.length == len(texts[ids.index(i)]) + len(out[i]) - 1
        if min(len(v) for v in out.values()) >= 20:
            break
    assert accepted > 10
    for i, text in zip(ids, texts):
        if pool == torch.uint8:
            check_generated(backend, i, text, out[i], torch.float32)
        else:
            assert out[i] == want[i][: len(out[i])]
    # Plain steps go on from there.
    before = {i: list(v) for i, v in out.items()}
    for i, o in backend.step().items():
        assert pool == torch.uint8 or o.token == want[i][len(before[i])]
    assert ops.take_status() == 0


def test_draft_steps_at_a_temperature():
    texts = prompts()
    runs = []
    for _ in range(2):
        backend = backend_of()
        ids, out = generate(backend, texts, 1)
        g = torch.Generator(device=DEV).manual_seed(6)
        for turn in range(6):
            drafts = {i: [out[i][-1], (7 * turn) % VOCAB] for i in ids[:2]}
            for i, steps in backend.draft_step(drafts, temperature=0.8, generator=g).items():
                tokens = [o.token for o in steps]
                assert tokens[:-1] == drafts.get(i, [])[: len(tokens) - 1]
                assert all(0 <= t < VOCAB for t in tokens)
                out[i] += tokens
        runs.append(out)
    assert runs[0] == runs[1]


def test_drafts_past_the_end_of_generation_are_dropped():
    texts = prompts((20,))
    (i,), want = generate(backend_of(), texts, 8)

    class Ends:
        def is_end_of_generation(self, token):
            return token == want[i][4]

    model = backend_of()._model
    backend = PagedBackend(model, 64, 16, 48, vocab=Ends(), max_seqs=8, pool_dtype=torch.uint8)
    (j,), out = generate(backend, texts, 1)
    end = want[i].index(want[i][4])
    if end == 0:
        pytest.skip("the first token ends it")
    steps = backend.draft_step({j: want[i][1:8]})[j]
    tokens = [o.token for o in steps]
    assert tokens == want[i][1: 1 + len(tokens)]
    if len(tokens) >= end:
        assert [o.finished for o in steps] == [False] * (end - 1) + [True]
        assert backend.draft_step({}) == {}


def test_model_refuses():
    model = TorchModel(CONFIG, weights_of(), device=DEV)
    pool = PagedKVPool(CONFIG, 8, 16, device=DEV, dtype=torch.uint8)
    cache = pool.new_cache(0)
    with pytest.raises(RuntimeError, match="uniforms"):
        model.verify_tokens([([1, 2], cache)], temperature=0.5)
    with pytest.raises(RuntimeError, match="references"):
        model.verify_tokens([([-1, 2], cache)])
    with pytest.raises(RuntimeError, match="input token"):
        model.verify_tokens([([1], pool.new_cache(1)), ([], cache)])
    with pytest.raises(RuntimeError, match="one group"):
        model.verify_tokens([([1, 2], cache), ([3], cache)])
    with pytest.raises(RuntimeError, match="index"):
        model.verify_tokens([([1, VOCAB], cache)])
    assert model.verify_tokens([]) == []
    assert cache.length == 0 and ops.take_status() == 0
    odd = dataclasses.replace(CONFIG, hidden_size=160, num_heads=4, num_kv_heads=2)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        PagedKVPool(odd, 8, 16, device=DEV, dtype=torch.uint8)

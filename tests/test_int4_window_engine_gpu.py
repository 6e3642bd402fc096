"""The engine on a 4-bit cache with a sliding window, sinks and a partial interleaved rotary
embedding, against the model's formula in 64 bits over what its cache holds (as in
test_int4_engine_gpu, whose tolerances these are): plain and drafted steps far past the window.
The checked backend gives no block up, so that every key it attends can be read back; one that
does gives the same tokens."""

import pytest
import torch

from batchstream_inference_engine_b200 import ops

from . import int4_format as fmt
from .test_bounded_engine_gpu import REL, VOCAB
from .test_int4_engine_gpu import (DEV, WINDOWED, backend_of, generate, held_rows, prompts,
                                   weights_of)

pytestmark = pytest.mark.gpu


def reference_logits(tokens, dtype, held, c=WINDOWED):
    """Logits [n, vocab] of every position in 64 bits, over the cached keys and values."""
    w = {k: v.to(dtype).double().to(DEV) for k, v in weights_of(c).items()}
    n, H, Hkv, D, rd = len(tokens), c.num_heads, c.num_kv_heads, c.head_dim, c.rotary_dim
    x = w["model.embed_tokens.weight"][torch.tensor(tokens, device=DEV)]
    p = torch.arange(n, device=DEV)
    # By the definition, not by the framework's frequencies.
    freq = c.rope_theta ** (-torch.arange(0, rd, 2, dtype=torch.float64, device=DEV) / rd)
    angle = (p[:, None] * freq)[:, None]
    ahead = p[:, None] - p[None]
    see = (ahead >= 0) & ((ahead < c.attention_window) | (p[None] < c.attention_sinks))

    def norm(x, weight):
        return weight * x * torch.rsqrt((x * x).mean(-1, keepdim=True) + c.rms_norm_eps)

    def rotate(x):
        x = x.clone()
        a, b = x[..., 0:rd:2].clone(), x[..., 1:rd:2].clone()
        x[..., 0:rd:2] = a * angle.cos() - b * angle.sin()
        x[..., 1:rd:2] = b * angle.cos() + a * angle.sin()
        return x

    for layer in range(c.num_layers):
        pre = f"model.layers.{layer}."

        def lin(name, x):
            return x @ w[pre + name + ".weight"].t() + w.get(pre + name + ".bias", 0)  # noqa: B023

        y = norm(x, w[pre + "input_layernorm.weight"])
        q = rotate(lin("self_attn.q_proj", y).view(n, H, D)).view(n, Hkv, H // Hkv, D)
        own = (rotate(lin("self_attn.k_proj", y).view(n, Hkv, D)),
               lin("self_attn.v_proj", y).view(n, Hkv, D))
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
    rows = reference_logits(text, dtype, held_rows(backend.pool, cache))[len(prompt) - 1:]
    picked = torch.tensor(generated[: rows.shape[0]], device=DEV)
    rows = rows[: picked.numel()]
    short = rows.amax(-1) - rows.gather(1, picked[:, None])[:, 0]
    assert bool((short <= 2 * REL[dtype] * rows.abs().amax()).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("graphs", [False, True])
def test_plain_steps(dtype, graphs, monkeypatch):
    texts = prompts((130, 20, 75))
    trimmed = backend_of(WINDOWED, dtype=dtype, graphs=graphs, blocks=40)
    ids, want = generate(trimmed, texts, 100)
    assert trimmed.blocks_in_use <= 3 * trimmed.sequence_blocks
    whole = backend_of(WINDOWED, dtype=dtype, graphs=graphs)
    monkeypatch.setattr(whole.pool, "trim", lambda *a: 0)
    ids, out = generate(whole, texts, 100)
    assert out == want  # what the window does not see does not count
    for i, text in zip(ids, texts):
        check_generated(whole, i, text, out[i], dtype)
    assert ops.take_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_drafted_steps(dtype, monkeypatch):
    texts = prompts((130, 20, 60))
    _, want = generate(backend_of(WINDOWED, dtype=dtype, blocks=40), texts, 90)
    runs = []
    for whole in (False, True):
        backend = backend_of(WINDOWED, dtype=dtype, blocks=64 if whole else 40)
        if whole:
            monkeypatch.setattr(backend.pool, "trim", lambda *a: 0)
        ids, out = generate(backend, texts, 1)
        turn = 0
        while turn < 40 or min(len(v) for v in out.values()) <= 60:  # past the window
            drafts = {}
            for i in ids:  # some right, then wrong ones
                drafts[i] = want[i][len(out[i]): len(out[i]) + (turn + i) % 6]
                drafts[i] += [(len(drafts[i]) + 3 * turn) % VOCAB] * (turn % 4)
            for i, steps in backend.draft_step(drafts).items():
                tokens = [o.token for o in steps]
                assert tokens[:-1] == drafts[i][: len(tokens) - 1]
                out[i] += tokens
            turn += 1
        runs.append({i: list(v) for i, v in out.items()})
    assert runs[0] == runs[1]
    for i, text in zip(ids, texts):
        check_generated(backend, i, text, out[i], dtype)
    assert ops.take_status() == 0

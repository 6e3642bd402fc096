"""The 4-bit cache and draft verification without a GPU: shapes, refusals of the C ABI and
of the wrappers."""

import ctypes
import math

import pytest
import torch

from batchstream_inference_engine_b200 import _lib, ops

from . import int4_format as fmt


def test_pool_shapes():
    assert ops.int4_pool_shape(4, 100, 16, 128) == (4, 100, 16, 72)
    assert ops.int4_pool_shape(2, 7, 5, 64) == (2, 7, 5, 36)
    for head_dim, block in ((48, 16), (0, 16), (32, 5), (96, 1)):
        with pytest.raises(RuntimeError):
            ops.int4_pool_shape(2, 7, block, head_dim)


def test_the_format_holds_bf16_numbers_within_its_bound():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 64, generator=g, dtype=torch.float64) * torch.exp(
        4 * torch.randn(500, 1, generator=g, dtype=torch.float64))
    codes, scales = fmt.quantise(x)
    held = fmt.values(codes, scales)
    assert torch.equal(held, held.bfloat16().double())  # exactly
    s = scales.abs().repeat_interleave(32, -1)
    assert bool(((held - x).abs() <= torch.where(x.abs() > 7.5 * s, s, s / 2)).all())
    pool = fmt.pack(codes.view(5, 10, 10, 64), scales.view(5, 10, 10, 2))
    assert pool.shape == ops.int4_pool_shape(5, 10, 10, 64)
    assert torch.equal(fmt.unpack(pool).view(500, 64), held)


def attention_args(**change):
    """A valid bs_int4_attention_batched call (zero sequences, so nothing is launched)."""
    args = dict(query=1, q_stride=64 * 4, key_pool=1, value_pool=1, tables=1, table_stride=8,
                table_rows=2, seq_rows=None, lens=1, num_seqs=0, heads=4, kv_heads=2, head_dim=64,
                block_size=16, num_blocks=8, max_blocks=8, dtype=0, scaling=0.125, window=0,
                sinks=4, out=1, o_stride=64 * 4, ws=None, ws_bytes=0, status=None, stream=None)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=7), "dtype"), (dict(num_seqs=-1), "count"), (dict(heads=5), "groups"),
    (dict(head_dim=0), "positive"), (dict(head_dim=48), "multiple of 32"),
    (dict(head_dim=32, block_size=5), "even"), (dict(block_size=0), "positive"),
    (dict(num_blocks=0), "positive"), (dict(max_blocks=9), "max_blocks"),
    (dict(table_rows=0), "table_rows"), (dict(window=-3), "window"), (dict(sinks=-1), "sinks"),
    (dict(q_stride=100), "strides"), (dict(o_stride=100), "strides"),
    (dict(head_dim=288, q_stride=4096, o_stride=4096), "head_dim"),
    (dict(heads=34, q_stride=4096, o_stride=4096), "groups"),
    (dict(max_blocks=1 << 27, table_stride=1 << 27), "2\\^30"),
    (dict(num_blocks=1 << 28), "2\\^31"),
])
def test_attention_refuses(change, message):
    assert _lib.lib().bs_int4_attention_batched(*attention_args()) == 0
    with pytest.raises(RuntimeError, match=message):
        _lib.check(_lib.lib().bs_int4_attention_batched(*attention_args(**change)))


def test_prefill_refuses_bad_sizes():
    lib = _lib.lib()

    def call(**change):
        args = dict(query=1, q_stride=256, cu_q=1, num_rows=0, num_tokens=0, max_query_len=5,
                    lens=1, seq_rows=None, key_pool=1, value_pool=1, tables=1, table_stride=8,
                    table_rows=2, max_blocks=8, heads=4, kv_heads=2, head_dim=64, block_size=16,
                    num_blocks=8, dtype=0, scaling=0.125, window=0, sinks=0, out=1, o_stride=256,
                    ws=None, ws_bytes=0, status=None, stream=None)
        args.update(change)
        return lib.bs_int4_prefill_attention(*args.values())

    assert call() == 0
    for change in (dict(window=-1), dict(sinks=-1), dict(max_query_len=-1), dict(num_tokens=-2),
                   dict(head_dim=40), dict(head_dim=32, block_size=3),
                   dict(num_rows=2, num_tokens=4, max_query_len=0),
                   dict(num_rows=2, num_tokens=4, cu_q=None)):
        assert call(**change) != 0, change


def append_call(**change):
    args = dict(qkv=16, stride=512, dtype=0, freq=16, rotary_dim=64, inter=0, amp=1.0, pos=16,
                slots=16, tokens=0, heads=4, kv_heads=2, head_dim=64, q=16, k=16, v=16,
                num_blocks=8, block_size=16, status=None, stream=None)
    args.update(change)
    return _lib.lib().bs_rotary_append_int4(*args.values())


@pytest.mark.parametrize("change", [
    dict(dtype=3), dict(tokens=-1), dict(heads=-1), dict(kv_heads=0), dict(rotary_dim=-2),
    dict(rotary_dim=63), dict(rotary_dim=66), dict(amp=math.nan), dict(amp=math.inf),
    dict(stride=511), dict(num_blocks=0), dict(block_size=0), dict(num_blocks=1 << 30),
    dict(head_dim=48, rotary_dim=48), dict(head_dim=32, rotary_dim=32, block_size=3),
    dict(tokens=1, freq=None), dict(tokens=1, pos=None), dict(tokens=1, slots=None),
    dict(tokens=1, k=None), dict(tokens=1, q=None), dict(tokens=1, k=18),
])
def test_append_refuses(change):
    assert append_call() == 0
    assert append_call(heads=0, q=None, rotary_dim=0, freq=None, pos=None) == 0
    assert append_call(**change) != 0


@pytest.mark.parametrize("change", [
    dict(tokens=-1), dict(kv_heads=0), dict(num_blocks=0), dict(block_size=0), dict(head_dim=0),
    dict(head_dim=100), dict(head_dim=1056), dict(num_blocks=1 << 30), dict(tokens=2, slots=None),
    dict(tokens=2, k=None), dict(tokens=2, v=17), dict(tokens=2, k_out=24),
])
def test_read_refuses(change):
    base = dict(k=16, v=16, slots=16, tokens=0, kv_heads=2, num_blocks=8, block_size=16,
                head_dim=64, k_out=16, v_out=16, status=None, stream=None)
    lib = _lib.lib()
    assert lib.bs_read_int4(*base.values()) == 0
    assert lib.bs_read_int4(*dict(base, **change).values()) != 0


@pytest.mark.parametrize("change", [
    dict(dtype=5), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31), dict(seqs=-1),
    dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
    dict(temperature=1e300), dict(rows=4, stride=49), dict(rows=4, probs=16, probs_stride=49),
    dict(rows=4, probs=16, probs_dtype=3), dict(rows=4, ws=None), dict(rows=4, ws_bytes=63),
    dict(rows=4, ws=8), dict(rows=4, logits=None), dict(rows=4, tokens=None),
    dict(rows=4, seqs=1, accepted=None), dict(seqs=1, cu=None), dict(rows=1 << 31),
])
def test_verify_drafts_refuses(change):
    base = dict(logits=16, stride=50, dtype=0, rows=0, vocab=50, drafts=16, cu=16, seqs=0,
                uniforms=16, temperatures=None, temperature=1.0, probs=None, probs_stride=50,
                probs_dtype=1, tokens=16, accepted=16, ws=16, ws_bytes=64, status=None, stream=None)
    lib = _lib.lib()
    assert lib.bs_verify_drafts(*base.values()) == 0
    assert lib.bs_verify_drafts(*dict(base, **change).values()) != 0


def test_workspace_queries():
    lib, got = _lib.lib(), ctypes.c_uint64(0)
    null = ctypes.POINTER(ctypes.c_uint64)()
    assert lib.bs_int4_attention_batched_workspace_bytes(1, 4, 2, 64, 16, 8, 0, 0, 0, null) != 0
    assert lib.bs_int4_prefill_attention_workspace_bytes(8, 1, 8, 4, 2, 64, 16, 8, 0, 0, 0,
                                                         null) != 0
    assert lib.bs_verify_drafts_workspace_bytes(4, 50, 0, null) != 0
    assert lib.bs_verify_drafts_workspace_bytes(5, 8192, 1, ctypes.byref(got)) == 0
    assert got.value == 5 * 3 * 16  # a row may begin inside a 16-byte unit


def test_operators_refuse_host_tensors():
    z = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 2, 16, 36, dtype=torch.uint8)
    i = torch.zeros(1, dtype=torch.int32)
    f = torch.zeros(1)
    for call in (lambda: ops.int4_attention_batched(z, pool, pool, i[None], i, 1.0),
                 lambda: ops.int4_prefill_attention(z, pool, pool, i[None], i, i, 1.0, 1),
                 lambda: ops.rotary_append_int4(z.view(1, -1), i.double(), i, i, pool, pool, 0),
                 lambda: ops.read_int4(pool, pool, i),
                 lambda: ops.verify_drafts(z[0], i, i, f)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()

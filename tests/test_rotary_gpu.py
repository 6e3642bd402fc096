"""Rotary embedding with the K/V append from frequencies, on the GPU, against the
formula in 64 bits.

Tolerance, with u = 2^-24: cos and sin come from fp64 angles and are rounded to fp32
after the amplitude (u each, plus the fp64 angle's own error, below 2^-20 at
positions up to 2^31: 2^-53 of a few times 2^31 radians), the product and the sum
round once each: 4 u (|x| + |y|) amp + 2^-20 (|x| + |y|) amp at the farthest
positions, and the output rounds by half a step (bf16 2^-8, fp32 2^-24) of its value.
Copied dims are exact.
"""

import math

import pytest
import torch

from batchstream_inference_engine_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Case:
    def __init__(self, T, H, Hkv, D, rotary_dim, interleaved, dtype, pool_dtype, scaling=None,
                 far=2000, block=16, seed=0, theta=1e6):
        g = torch.Generator().manual_seed(seed)
        self.T, self.H, self.Hkv, self.D, self.rd = T, H, Hkv, D, rotary_dim
        self.inter, self.dtype, self.pool_dtype = interleaved, dtype, pool_dtype
        self.freq, self.amp = ops.rope_frequencies(rotary_dim, theta, scaling, device=DEV)
        self.qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=g).to(dtype).to(DEV)
        self.pos = torch.randint(0, far, (T,), generator=g).int().to(DEV)
        nb = -(-T // block) + 3
        self.slots = torch.randperm(nb * block, generator=g)[:T].int().to(DEV)
        self.k = torch.randn(Hkv, nb, block, D, generator=g).to(pool_dtype).to(DEV)
        self.v = torch.randn(Hkv, nb, block, D, generator=g).to(pool_dtype).to(DEV)

    def run(self, **kw):
        k, v = self.k.clone(), self.v.clone()
        args = dict(interleaved=self.inter, amplitude=self.amp)
        args.update(kw)
        q = ops.rotary_append(self.qkv, self.freq, self.pos, self.slots, k, v, self.H, **args)
        return q, k, v

    def reference(self):
        """Rotated rows [T, H + 2 Hkv, D] in 64 bits and their tolerances before
        the output's rounding."""
        x = self.qkv.double().view(self.T, -1, self.D)
        y, tol = x.clone(), torch.zeros_like(x)
        rot = slice(0, self.H + self.Hkv)
        i = torch.arange(self.rd // 2, device=DEV)
        a, b = (2 * i, 2 * i + 1) if self.inter else (i, i + self.rd // 2)
        angle = (self.pos.double()[:, None] * self.freq)[:, None]
        cos, sin = self.amp * angle.cos(), self.amp * angle.sin()
        xa, xb = x[:, rot][..., a], x[:, rot][..., b]
        y[:, rot, a] = xa * cos - xb * sin  # noqa: E203
        y[:, rot, b] = xb * cos + xa * sin
        reach = (self.pos.double() + 1)[:, None, None] * 2.0 ** -50  # the angle's own rounding
        t = (4 * 2.0 ** -24 + reach) * (xa.abs() + xb.abs()) * abs(self.amp)
        tol[:, rot, a] = t
        tol[:, rot, b] = t
        return y, tol

    def check(self, q, k, v, live=None):
        y, tol = self.reference()
        live = torch.ones(self.T, dtype=torch.bool, device=DEV) if live is None else live

        def close(got, want, slack, dtype):
            bound = slack + half_step(dtype) * (want.abs() + slack)
            err = (got.double() - want).abs()
            assert bool((err <= bound).all()), float((err / bound.clamp_min(1e-300)).max())

        close(q, y[:, : self.H], tol[:, : self.H], self.dtype)
        keep_k, keep_v = self.k.clone(), self.v.clone()
        s = self.slots[live].long()
        for pool, keep, part, off in ((k, keep_k, "k", self.H), (v, keep_v, "v", self.H + self.Hkv)):
            flat, old = pool.view(self.Hkv, -1, self.D), keep.view(self.Hkv, -1, self.D)
            want = y[live][:, off: off + self.Hkv].transpose(0, 1)
            slack = tol[live][:, off: off + self.Hkv].transpose(0, 1)
            close(flat[:, s], want, slack, self.pool_dtype)
            old[:, s] = flat[:, s]
            assert torch.equal(pool, keep), part  # no other slot changed


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,Hkv,D,rotary_dim", [
    (14, 2, 64, 64), (28, 4, 128, 64), (4, 4, 80, 32), (3, 1, 8, 8), (5, 1, 7, 2), (2, 2, 256, 256),
    (6, 2, 96, 24), (1, 1, 2, 2), (8, 2, 64, 10), (2, 1, 576, 64),
])
@pytest.mark.parametrize("dtype,pool_dtype", [
    (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
    (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_shapes(interleaved, H, Hkv, D, rotary_dim, dtype, pool_dtype):
    c = Case(37, H, Hkv, D, rotary_dim, interleaved, dtype, pool_dtype, seed=D)
    c.check(*c.run())
    assert ops.take_status() == 0


@pytest.mark.parametrize("scaling", [
    None, {"type": "linear", "factor": 8.0}, {"type": "ntk", "factor": 4.0},
    {"type": "yarn", "factor": 32.0, "original_max_position": 4096},
    {"type": "banded", "factor": 8.0, "original_max_position": 8192, "low_freq_factor": 1.0,
     "high_freq_factor": 4.0}])
@pytest.mark.parametrize("far", [4096, 1 << 20, (1 << 31) - 1])
def test_scaled_frequencies_at_far_positions(scaling, far):
    for dtype in (torch.float32, torch.bfloat16):
        c = Case(50, 4, 2, 64, 64, False, dtype, dtype, scaling=scaling, far=far, seed=7)
        c.pos[0], c.pos[1] = far, 0
        c.check(*c.run())
    assert ops.take_status() == 0


@pytest.mark.parametrize("T", [1, 2, 7, 129, 1000, 5000])
@pytest.mark.parametrize("interleaved", [False, True])
def test_token_counts(T, interleaved):
    c = Case(T, 14, 2, 64, 64, interleaved, torch.bfloat16, torch.bfloat16, seed=T)
    c.check(*c.run())
    assert ops.take_status() == 0


def test_no_tokens():
    c = Case(1, 14, 2, 64, 64, False, torch.bfloat16, torch.bfloat16)
    q = ops.rotary_append(c.qkv[:0], c.freq, c.pos[:0], c.slots[:0], c.k, c.v, 14)
    assert q.shape == (0, 14, 64)


@pytest.mark.parametrize("D,rotary_dim", [(64, 64), (64, 32), (8, 6)])
def test_padding_bad_slots_and_bad_positions(D, rotary_dim):
    c = Case(9, 4, 2, D, rotary_dim, False, torch.bfloat16, torch.bfloat16, seed=2)
    live = torch.ones(9, dtype=torch.bool, device=DEV)
    c.slots[3] = -1
    live[3] = False
    c.check(*c.run(), live=live)
    assert ops.take_status() == 0
    c.slots[5] = c.k.size(1) * 16
    live[5] = False
    c.check(*c.run(), live=live)
    with pytest.raises(RuntimeError, match="slot"):
        ops.take_status()
    # A bad position leaves the row's q and k unwritten; v is still appended.
    d = Case(4, 4, 2, D, rotary_dim, False, torch.bfloat16, torch.bfloat16, seed=3)
    q0, k0, v0 = d.run()
    d.pos[2] = -1
    out = torch.full((4, 4, D), 55.0, dtype=torch.bfloat16, device=DEV)
    q, k, v = d.run(query_out=out)
    with pytest.raises(RuntimeError, match="position"):
        ops.take_status()
    assert bool((q[2] == 55.0).all()) and torch.equal(q[[0, 1, 3]], q0[[0, 1, 3]])
    s = int(d.slots[2])
    assert torch.equal(k.view(2, -1, D)[:, s], d.k.view(2, -1, D)[:, s])
    assert torch.equal(v, v0)


def test_strided_rows_lists_and_unaligned_buffers():
    c = Case(20, 14, 2, 64, 64, False, torch.bfloat16, torch.bfloat16, seed=5)
    q0, k0, v0 = c.run()
    wide = torch.zeros(20, 18 * 64 + 24, dtype=torch.bfloat16, device=DEV)
    for shift in (8, 3):  # 16-byte rows, then rows that are not
        wide[:, shift: shift + 18 * 64] = c.qkv
        k, v = c.k.clone(), c.v.clone()
        pos2 = torch.stack([c.pos, c.pos + 1], 1)[:, 0]
        slots2 = torch.stack([c.slots, c.slots], 1)[:, 0]
        out = torch.empty(20 * 14 * 64 + shift, dtype=torch.bfloat16, device=DEV)
        q = ops.rotary_append(wide[:, shift: shift + 18 * 64], c.freq, pos2, slots2, k, v, 14,
                              query_out=out[shift:].view(20, 14, 64))
        assert torch.equal(q, q0) and torch.equal(k, k0) and torch.equal(v, v0)
    assert ops.take_status() == 0


def test_interleaved_of_permuted_dims_is_the_half_layout():
    c = Case(33, 4, 2, 64, 64, False, torch.float32, torch.float32, seed=6)
    q0, _, _ = c.run()
    perm = torch.stack([torch.arange(32), torch.arange(32) + 32], 1).flatten().to(DEV)
    rows = c.qkv.view(33, 8, 64)[..., perm].reshape(33, -1).contiguous()
    q = ops.rotary_append(rows, c.freq, c.pos, c.slots, c.k.clone(), c.v.clone(), 4,
                          interleaved=True)
    assert torch.equal(q, q0[..., perm])


def test_matches_the_table_driven_op_up_to_its_roundings():
    # rope_append rounds cos and sin, both products and the sum to bf16: at most
    # 2^-8 (|x| + |y|) for each of the tables and the products, 2^-8 of the result.
    c = Case(64, 14, 2, 64, 64, False, torch.bfloat16, torch.bfloat16, seed=8, far=500)
    q, k, v = c.run()
    angle = torch.arange(500).double()[:, None] * c.freq.cpu()
    angle = torch.cat([angle, angle], -1)
    cos, sin = angle.cos().bfloat16().to(DEV), angle.sin().bfloat16().to(DEV)
    k2, v2 = c.k.clone(), c.v.clone()
    q2 = ops.rope_append(c.qkv, cos, sin, c.pos, c.slots, k2, v2, 14)
    x = c.qkv.float().view(64, -1, 64)[:, :14]
    reach = x.abs() + torch.cat([x[..., 32:], x[..., :32]], -1).abs()
    assert bool(((q.float() - q2.float()).abs() <= 5 * 2.0 ** -8 * reach).all())
    assert torch.equal(v, v2)


def test_captured_replays_follow_positions_and_slots():
    c = Case(12, 14, 2, 64, 64, True, torch.bfloat16, torch.bfloat16, seed=9)
    k, v = c.k.clone(), c.v.clone()
    out = torch.empty(12, 14, 64, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary_append(c.qkv, c.freq, c.pos, c.slots, k, v, 14, interleaved=True, query_out=out)
    for shift in (0, 5, 100):
        c.pos.add_(shift)
        c.slots.copy_(c.slots.flip(0))
        k.copy_(c.k)
        v.copy_(c.v)
        graph.replay()
        c.check(out, k, v)


def test_wrapper_refuses():
    c = Case(5, 14, 2, 64, 64, False, torch.bfloat16, torch.bfloat16)

    def call(**kw):
        args = dict(qkv=c.qkv, frequencies=c.freq, positions=c.pos, slot_mapping=c.slots,
                    key_pool=c.k, value_pool=c.v, num_heads=14)
        args.update(kw)
        return ops.rotary_append(**args)

    call()
    for kw in (dict(frequencies=c.freq.float()), dict(frequencies=torch.cat([c.freq, c.freq])),
               dict(frequencies=c.freq[:0]), dict(positions=c.pos.long()),
               dict(slot_mapping=c.slots[:4]), dict(slot_mapping=c.slots.long()),
               dict(qkv=c.qkv[:4]), dict(qkv=c.qkv[:, 1:]), dict(num_heads=13),
               dict(key_pool=c.k[:1]), dict(value_pool=c.v.float()), dict(amplitude=math.nan),
               dict(query_out=torch.empty(5, 14, 64, device=DEV)),
               dict(query_out=torch.empty(5, 64, 14, dtype=torch.bfloat16, device=DEV).transpose(1, 2)),
               dict(positions=c.pos.cpu()), dict(qkv=c.qkv.half())):
        with pytest.raises(RuntimeError):
            call(**kw)
    assert ops.take_status() == 0


def test_query_out_must_not_overlap_qkv():
    # q in place would be read by other threads after it was written.
    c = Case(5, 14, 2, 64, 64, False, torch.bfloat16, torch.bfloat16)
    rows = c.qkv.contiguous()
    inside = rows.view(-1)[: 5 * 14 * 64].view(5, 14, 64)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.rotary_append(rows, c.freq, c.pos, c.slots, c.k, c.v, 14, query_out=inside)


@pytest.mark.parametrize("pool_dtype,head_dim", [(torch.bfloat16, 64), (torch.float32, 72)])
def test_slots_past_32_bit_offsets(pool_dtype, head_dim):
    # More than 2^31 elements a pool, the slots at its end; the same rows as in a small pool.
    blocks = 1_100_000
    c = Case(5, 14, 2, head_dim, head_dim, False, torch.bfloat16, pool_dtype)
    assert 2 * blocks * 16 * head_dim > 2 ** 31
    k = torch.zeros(2, blocks, 16, head_dim, dtype=pool_dtype, device=DEV)
    v = torch.zeros_like(k)
    small_k = torch.zeros(2, 8, 16, head_dim, dtype=pool_dtype, device=DEV)
    small_v = torch.zeros_like(small_k)
    slots = torch.tensor([0, 127, 5, 64, 126], dtype=torch.int32, device=DEV)
    want = ops.rotary_append(c.qkv, c.freq, c.pos, slots, small_k, small_v, 14)
    got = ops.rotary_append(c.qkv, c.freq, c.pos, slots + (blocks - 8) * 16, k, v, 14)
    assert ops.take_status() == 0
    assert torch.equal(got, want)
    assert torch.equal(k[:, blocks - 8:], small_k) and torch.equal(v[:, blocks - 8:], small_v)

"""The 4-bit cache on the GPU: the append's bytes against the format in 64 bits, reading
rows back, and attention over it, single tokens and prompt chunks, against the formula.

Attention's tolerances are those of test_window_gpu (its ``Paged.reference``): the numbers
that codes stand for are exact, so nothing is added for them but this: an element of the
cache may be exactly 0, and where the keys that weigh have 0 the relative terms are no larger
than the output of the keys that do not.  Weights below 2^-126 of the row's largest are 0 in
fp32 (their products with V below that too, and bf16 rounds there to multiples of 2^-133), so
n visible keys of at most max |v| each add 2^-125 n max |v|.  What the append stores is
compared bit for bit: the rotated key's fp64 error (2^-50 of it) moves an element across
the border of two codes once in some 10^13.
"""

import math

import pytest
import torch

from batchstream_inference_engine_b200 import ops

from . import int4_format as fmt
from .test_window_gpu import BORDERS, SENTINEL, Paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Packed(Paged):
    """``Paged`` over 4-bit pools.  Slots that no query token sees hold codes of 15 and NaN
    scales."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.keys = [fmt.held(k).float() for k in self.keys]
        self.values = [fmt.held(v).float() for v in self.values]
        self.k, self.v = self._packed(self.k), self._packed(self.v)

    def _packed(self, pool):
        x = pool.cpu().float()
        seen = x.isfinite().all(-1, keepdim=True)
        codes, scales = fmt.quantise(torch.where(seen, x, torch.zeros_like(x)))
        codes = torch.where(seen, codes, torch.full_like(codes, 15))
        scales = torch.where(seen, scales, torch.full_like(scales, math.nan))
        return fmt.pack(codes, scales).to(DEV)

    def reference(self):
        ref, tol = super().reference()
        most = [0.0 if n == 0 else n * float(v.abs().max()) for n, v in zip(self.lens, self.values)]
        return ref, tol + 2.0 ** -125 * max(most, default=0.0)

    def decode(self, **kw):
        out = torch.full((self.T, self.H, self.D), SENTINEL, dtype=self.dtype, device=DEV)
        kw.setdefault("query", self.q.to(DEV))
        got = ops.int4_attention_batched(key_pool=self.k, value_pool=self.v,
                                         block_tables=self.table, context_lens=self.len_d,
                                         scaling=self.scale, window=self.args[0],
                                         sinks=self.args[1], out=out, **kw)
        assert got is out
        return out

    def chunks(self, **kw):
        out = torch.full((self.T, self.H, self.D), SENTINEL, dtype=self.dtype, device=DEV)
        kw.setdefault("max_query_len", max(self.news))
        got = ops.int4_prefill_attention(self.q.to(DEV), self.k, self.v, self.table, self.cu,
                                         self.len_d, self.scale, window=self.args[0],
                                         sinks=self.args[1], out=out, **kw)
        assert got is out
        return out


# ------------------------------------------------------------------ append and read


def rotated(qkv, freq, pos, heads, rd, interleaved, amplitude):
    """Rotated q and k heads in 64 bits, [T, heads, D]."""
    x = qkv.double()[:, :heads].clone()
    if rd:
        angle = pos.double()[:, None, None] * freq
        c, s = angle.cos() * amplitude, angle.sin() * amplitude
        first = (slice(0, rd, 2) if interleaved else slice(0, rd // 2))
        second = (slice(1, rd, 2) if interleaved else slice(rd // 2, rd))
        a, b = x[..., first].clone(), x[..., second].clone()
        x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    return x


def append_case(dtype, T, H, Hkv, D, bs, rd, seed=0, high=100000):
    g = torch.Generator().manual_seed(seed)
    nb = -(-T // bs) + 2
    qkv = torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype)
    pos = torch.randint(0, high, (T,), generator=g, dtype=torch.int32)
    slots = torch.randperm(nb * bs, generator=g)[:T].int()
    freq = 1e4 ** (-torch.arange(rd // 2, dtype=torch.float64) * 2 / max(rd, 1))
    pool = torch.randint(0, 256, ops.int4_pool_shape(Hkv, nb, bs, D), generator=g,
                         dtype=torch.uint8)
    return qkv, pos, slots, freq, pool


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,Hkv,D,bs,rd,interleaved,amplitude", [
    (1, 14, 2, 64, 16, 64, False, 1.0), (37, 28, 4, 128, 16, 128, False, 1.0),
    (37, 8, 2, 128, 16, 64, True, 1.25), (300, 4, 4, 64, 5, 32, True, 1.0),
    (9, 3, 1, 32, 4, 32, False, 1.0), (9, 3, 1, 96, 6, 20, False, 0.5), (5, 2, 1, 256, 32, 6, True, 1.0),
    (33, 0, 2, 64, 16, 0, False, 1.0), (33, 4, 2, 160, 16, 0, False, 1.0),
])
def test_append_stores_the_format(dtype, T, H, Hkv, D, bs, rd, interleaved, amplitude):
    qkv, pos, slots, freq, before = append_case(dtype, T, H, Hkv, D, bs, rd, seed=T + D)
    slots[T // 2] = -1 if T > 2 else slots[T // 2]
    k, v = before.to(DEV), before.to(DEV)
    q = ops.rotary_append_int4(qkv.to(DEV), freq.to(DEV), pos.to(DEV), slots.to(DEV), k, v, H,
                               interleaved=interleaved, amplitude=amplitude)
    assert ops.take_status() == 0
    x = rotated(qkv, freq, pos, H + Hkv, rd, interleaved, amplitude)
    # fp32 products of rounded cos and sin, then one rounding to the dtype.
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    size = qkv.double()[:, :H].abs().amax(-1, keepdim=True) if H else torch.zeros(T, 0, 1)
    tol = half * x[:, :H].abs() + 4 * 2.0 ** -24 * 2 * size * max(amplitude, 1.0)
    assert bool(((q.cpu().double() - x[:, :H]).abs() <= tol).all())
    for pool, rows in ((k, x[:, H:]), (v, qkv.double()[:, H + Hkv:])):
        nb = before.shape[1]
        codes, scales = fmt.quantise(rows)
        want = before.clone().view(Hkv, nb, -1)
        new = fmt.pack(*(torch.zeros(Hkv, nb * bs, n, dtype=t.dtype).index_copy(
            1, slots.clamp(min=0).long()[slots >= 0], t.transpose(0, 1)[:, slots >= 0])
            .view(Hkv, nb, bs, n) for t, n in ((codes, D), (scales, D // 32))))
        new = new.view(Hkv, nb, -1)
        mask = torch.zeros(nb * bs, dtype=torch.bool)
        mask[slots[slots >= 0].long()] = True
        mask = mask.view(nb, bs, 1)
        bytes_of = torch.cat([mask.expand(-1, -1, D // 2).flatten(1),
                              mask.expand(-1, -1, D // 16).flatten(1)], 1)
        want = torch.where(bytes_of, new, want)
        assert torch.equal(pool.cpu().view(Hkv, nb, -1), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_of_ties_and_extremes(dtype):
    # Position 0, so that keys are stored as they come: values half way between codes, both
    # extremes equal, one sided groups, zeros, subnormals, huge values.
    D = 64
    rows = torch.zeros(12, D)
    rows[0] = torch.arange(-32, 32) / 4.0
    rows[1, :32] = torch.arange(32) * 0.25
    rows[2] = torch.cat([torch.tensor([4.0, -4.0]), torch.arange(62) * 0.125 - 3.5])
    rows[3] = torch.cat([torch.tensor([-8.0]), torch.arange(63) * 0.25 - 7.5])
    rows[4, 0], rows[4, 33] = 2.0 ** -99, -2.0 ** -101
    rows[5, 0], rows[5, 33] = 2.0 ** 119, -2.0 ** 119 * 1.75
    rows[6] = 2.0 ** -126
    rows[7] = 1.0
    rows[8] = -1.0
    rows[9] = torch.randn(D, generator=torch.Generator().manual_seed(1)).bfloat16().float()
    rows[10] = torch.linspace(-1.9, 1.9, D).bfloat16().float() * 1.125
    rows[11] = torch.arange(64).float().sub(40).mul(0.1875)
    T = rows.shape[0]
    qkv = torch.cat([rows, rows.flip(0)], 1).to(dtype)  # one k head, one v head
    pools = [torch.zeros(ops.int4_pool_shape(1, 1, 16, D), dtype=torch.uint8, device=DEV)
             for _ in range(2)]
    index = torch.arange(T, dtype=torch.int32, device=DEV)
    freq = torch.ones(D // 2, dtype=torch.float64, device=DEV)
    ops.rotary_append_int4(qkv.to(DEV), freq, torch.zeros_like(index), index, *pools, 0)
    assert ops.take_status() == 0
    back = ops.read_int4(*pools, index)
    for pool, got, x in zip(pools, back, (rows, rows.flip(0))):
        want = fmt.held(x.to(dtype))
        assert torch.equal(got[:, 0].cpu().double(), want)
        assert torch.equal(fmt.unpack(pool.cpu())[0, 0, :T], want)
        # The bound that the documentation gives.
        s = fmt.quantise(x.to(dtype))[1].abs().repeat_interleave(32, -1)
        x = x.to(dtype).double()
        top = x.unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, -1)
        assert bool(((want - x).abs() <= torch.where(x.abs() > 7.5 * s, s, s / 2)
                     + 2.0 ** -100).all()) and bool((want.abs() <= 8 * s).all())
        assert bool((8 * s <= top * 1.125).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 2.0 ** 120])
def test_append_reports_values_it_cannot_hold(bad):
    D, T = 128, 3
    qkv = torch.randn(T, 3 * D, generator=torch.Generator().manual_seed(2))
    pools = [torch.full(ops.int4_pool_shape(1, 1, 16, D), 7, dtype=torch.uint8, device=DEV)
             for _ in range(2)]
    index = torch.arange(T, dtype=torch.int32, device=DEV)
    none = torch.zeros(0, dtype=torch.float64, device=DEV)
    broken = qkv.clone()
    broken[1, D + 40] = bad       # k, second group
    broken[2, 2 * D + 127] = -bad  # v, last group
    ops.rotary_append_int4(broken.to(DEV), none, index, index, *pools, 1)
    with pytest.raises(RuntimeError, match="not finite or too large"):
        ops.take_status()
    k, v = (t[:, 0].cpu().double() for t in ops.read_int4(*pools, index))
    want_k, want_v = fmt.held(qkv[:, D: 2 * D]), fmt.held(qkv[:, 2 * D:])
    want_k[1, 32:64] = 0.0
    want_v[2, 96:] = 0.0
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert ops.take_status() == 0


def test_append_reports_positions_and_slots():
    qkv, pos, slots, freq, before = append_case(torch.bfloat16, 4, 2, 1, 64, 16, 64)
    pos[1] = -1
    slots[2] = before.shape[1] * 16
    k, v = before.to(DEV), before.to(DEV)
    out = torch.full((4, 2, 64), SENTINEL, dtype=torch.bfloat16, device=DEV)
    ops.rotary_append_int4(qkv.to(DEV), freq.to(DEV), pos.to(DEV), slots.to(DEV), k, v, 2,
                           query_out=out)
    with pytest.raises(RuntimeError, match="slot outside the pool.*position|position"):
        ops.take_status()
    assert bool((out[1] == SENTINEL).all()) and not bool((out[2] == SENTINEL).any())
    kept = ops.read_int4(k, v, slots[1:2].to(DEV))
    old = ops.read_int4(before.to(DEV), before.to(DEV), slots[1:2].to(DEV))
    assert torch.equal(kept[0].view(torch.int16), old[0].view(torch.int16))  # no key without a position
    assert torch.equal(kept[1][0, 0].cpu().double(), fmt.held(qkv[1, 3]))


def test_append_unaligned_and_strided_rows():
    for dtype in (torch.bfloat16, torch.float32):
        qkv, pos, slots, freq, before = append_case(dtype, 21, 4, 2, 64, 16, 64, seed=5)
        want = [before.to(DEV), before.to(DEV)]
        q = ops.rotary_append_int4(qkv.to(DEV), freq.to(DEV), pos.to(DEV), slots.to(DEV), *want, 4)
        wide = torch.zeros(21, 8 * 64 + 3, dtype=dtype, device=DEV)
        wide[:, 1: 1 + 8 * 64] = qkv.view(21, -1).to(DEV)
        got = [before.to(DEV), before.to(DEV)]
        q2 = ops.rotary_append_int4(wide[:, 1: 1 + 8 * 64], freq.to(DEV), pos.to(DEV),
                                    slots.to(DEV), *got, 4)
        assert torch.equal(q, q2)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert ops.take_status() == 0


def test_read_rows():
    g = torch.Generator().manual_seed(3)
    for D, bs in ((64, 16), (128, 32), (32, 6), (96, 10), (256, 4)):
        x = torch.randn(3, 5, bs, D, generator=g)
        k, v = fmt.pack(*fmt.quantise(x)), fmt.pack(*fmt.quantise(2 * x))
        slots = torch.randint(0, 5 * bs, (77,), generator=g, dtype=torch.int32)
        slots[5] = -3
        got = ops.read_int4(k.to(DEV), v.to(DEV), slots.to(DEV))
        for t, pool in zip(got, (k, v)):
            want = fmt.unpack(pool).view(3, -1, D)[:, slots.clamp(min=0).long()].transpose(0, 1)
            want[5] = 0.0
            assert torch.equal(t.cpu().double(), want)
    assert ops.take_status() == 0
    slots[9] = 5 * bs
    got = ops.read_int4(k.to(DEV), v.to(DEV), slots.to(DEV))
    with pytest.raises(RuntimeError, match="slot outside the pool"):
        ops.take_status()
    assert not bool(got[0][9].any())
    assert ops.read_int4(k.to(DEV), v.to(DEV), slots[:0].to(DEV))[0].shape == (0, 3, 256)


def test_blocks_of_4_bit_pools_are_copied():
    g = torch.Generator().manual_seed(4)
    pools = [torch.randint(0, 256, (3, *ops.int4_pool_shape(2, 9, 16, d)), generator=g,
                           dtype=torch.uint8) for d in (64, 64, 96)]
    k, v = pools[0].to(DEV), pools[1].to(DEV)
    src = torch.tensor([1, 7, -1, 4], dtype=torch.int32, device=DEV)
    dst = torch.tensor([0, 8, 2, 3], dtype=torch.int32, device=DEV)
    ops.copy_blocks(k, v, src, dst)
    ops.copy_blocks(pools[2].to(DEV)[0], pools[2].to(DEV)[1], src, dst)
    for got, want in ((k, pools[0]), (v, pools[1])):
        want[:, :, [0, 8, 3]] = want[:, :, [1, 7, 4]]
        assert torch.equal(got.cpu(), want)
    assert ops.take_status() == 0


# ------------------------------------------------------------------ single tokens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5), (1, 0), (1, 1), (16, 16), (200, 33),
                                          (5, 2000), (300, 1 << 40)])
def test_decode_at_every_border(dtype, head_dim, window, sinks):
    c = Packed(BORDERS, [1] * len(BORDERS), 14, 2, head_dim, 16, dtype, window or 1 << 40, sinks,
               seed=window)
    if not window:
        c.args = (0, 0)
        out = c.decode()
        c.args = (1 << 40, 0)
    else:
        out = c.decode()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,head_dim,block", [
    (8, 8, 64, 16), (16, 1, 64, 16), (28, 4, 128, 16), (32, 2, 128, 32), (5, 1, 96, 16),
    (6, 2, 256, 16), (4, 2, 32, 4), (9, 3, 160, 48), (24, 2, 64, 64), (18, 2, 128, 48),
    (2, 1, 64, 5), (8, 1, 224, 6), (1, 1, 128, 16),
])
def test_decode_shapes(dtype, heads, kv_heads, head_dim, block):
    lens = [1, 0, 7, 33, 130, 131, 300, 65]
    c = Packed(lens, [1] * len(lens), heads, kv_heads, head_dim, block, dtype, 90, 6, seed=heads)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("lens", [[9000], [5000, 1], [1], [4099] * 3, [64], [65], [2000] * 9])
def test_decode_long_rows_are_split_and_joined(dtype, head_dim, lens):
    c = Packed(lens, [1] * len(lens), 14, 2, head_dim, 16, dtype, 1 << 40, 0, seed=3)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)
    for _ in range(3):
        assert torch.equal(c.decode(), out)


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(14, 2, 64), (28, 4, 128), (16, 1, 64)])
@pytest.mark.parametrize("lens,new", [([30000], 1), ([25000, 3, 700], 1), ([30000, 40], 2),
                                      ([300 + 9 * i for i in range(250)], 2)])
def test_rows_cut_across_spans_of_the_batch(heads, kv_heads, head_dim, lens, new):
    if new * heads // kv_heads > 16:
        new = 1
    c = Packed(lens, [new] * len(lens), heads, kv_heads, head_dim, 16, torch.bfloat16, 1 << 40, 0,
               seed=13)
    run = c.decode if new == 1 else c.chunks
    out = run()
    assert ops.take_status() == 0
    c.check(out)
    assert torch.equal(run(), out)


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(14, 2, 64), (28, 4, 128), (16, 1, 128)])
@pytest.mark.parametrize("window", [1 << 40, 256])
def test_decode_large_batch_many_lengths(heads, kv_heads, head_dim, window):
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 900, (300,), generator=g).tolist()
    c = Packed(lens, [1] * 300, heads, kv_heads, head_dim, 16, torch.bfloat16, window, 4, seed=6)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)
    assert torch.equal(c.decode(), out)


def test_decode_more_sequences_than_the_span_scan_stages():
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(0, 60, (7000,), generator=g).tolist()
    c = Packed(lens, [1] * 7000, 2, 1, 64, 16, torch.bfloat16, 1 << 40, 0, seed=7)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("dtype,heads,kv_heads,head_dim", [
    (torch.float32, 14, 2, 64), (torch.bfloat16, 16, 2, 96), (torch.bfloat16, 14, 2, 64),
    (torch.bfloat16, 28, 4, 128)])
@pytest.mark.parametrize("rows,window", [(3, 100), (8, 1 << 40), (24, 777), (64, 1 << 40)])
def test_decode_by_clusters_and_by_records(dtype, heads, kv_heads, head_dim, rows, window):
    lens = [(0, 1, 17, 64, 120, 128, 130, 145, 300, 900)[i % 10] + i // 10 for i in range(rows)]
    c = Packed(lens, [1] * rows, heads, kv_heads, head_dim, 16, dtype, window, 4, seed=40)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)
    assert torch.equal(out, c.decode())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 20.0])
def test_decode_scales(dtype, scale):
    c = Packed([70, 300, 1100], [1] * 3, 14, 2, 64, 16, dtype, 400, 5, seed=14)
    c.scale = scale
    c.check(c.decode())


def test_decode_output_may_be_the_query():
    for dtype in (torch.bfloat16, torch.float32):
        c = Packed([5000, 70, 3], [1] * 3, 14, 2, 64, 16, dtype, 4000, 4, seed=13)
        want = c.decode()
        q = c.q.to(DEV)
        ops.int4_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, 4000, 4, out=q)
        assert torch.equal(q, want)


def test_decode_of_an_all_padding_batch_and_of_none():
    c = Packed([0, 0, 0], [1, 1, 1], 14, 2, 64, 16, torch.bfloat16, 40, 4)
    assert bool((c.decode() == SENTINEL).all())
    empty = torch.empty(0, 14, 64, dtype=torch.bfloat16, device=DEV)
    assert ops.int4_attention_batched(empty, c.k, c.v, c.table, c.len_d, 0.1).shape == (0, 14, 64)
    assert ops.take_status() == 0


def test_decode_strided_query_and_output_rows_and_lists():
    lens = [70, 3, 200, 41, 0, 90]
    c = Packed(lens, [1] * 6, 14, 2, 64, 16, torch.bfloat16, 1 << 40, 0, seed=8)
    plain = c.decode()
    fused = torch.randn(6, 18 * 64, device=DEV).bfloat16()
    fused[:, : 14 * 64] = c.q.to(DEV).view(6, -1)
    wide = torch.full((6, 20, 64), SENTINEL, dtype=torch.bfloat16, device=DEV)
    order = [4, 2, 0, 5, 1, 3]
    table = torch.full((6, c.table.size(1) + 5), -7, dtype=torch.int32, device=DEV)
    table[order, : c.table.size(1)] = c.table
    lens2 = torch.zeros(12, dtype=torch.int32, device=DEV)
    lens2[::2] = c.len_d
    rows2 = torch.full((12,), 99, dtype=torch.int32, device=DEV)
    rows2[::2] = torch.tensor(order, dtype=torch.int32, device=DEV)
    ops.int4_attention_batched(fused.view(6, 18, 64)[:, :14], c.k, c.v, table, lens2[::2], c.scale,
                               seq_rows=rows2[::2], out=wide[:, 3:17])
    assert ops.take_status() == 0
    assert torch.equal(wide[:, 3:17], plain)
    assert bool((wide[:, :3] == SENTINEL).all()) and bool((wide[:, 17:] == SENTINEL).all())


def test_decode_unaligned_pool_and_query():
    # Pools 4 bytes and a query 2 bytes into their storage: no tensor-core loads, same sums.
    c = Packed([70, 3, 200], [1] * 3, 14, 2, 64, 16, torch.bfloat16, 40, 5, seed=9)

    def shifted(t, by):
        buf = torch.empty(t.numel() + by, dtype=t.dtype, device=DEV)
        buf[by:] = t.reshape(-1)
        return buf[by:].view(t.shape)

    q = shifted(c.q.to(DEV), 1)
    out = shifted(torch.zeros(3, 14, 64, dtype=torch.bfloat16, device=DEV), 1)
    ops.int4_attention_batched(q, shifted(c.k, 4), shifted(c.v, 4), c.table, c.len_d, c.scale, 40,
                               5, out=out)
    assert ops.take_status() == 0
    c.check(out)
    c.check(ops.int4_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, 40, 5))
    with pytest.raises(RuntimeError, match="4-byte aligned"):
        ops.int4_attention_batched(q, shifted(c.k, 1), c.v, c.table, c.len_d, c.scale, 40, 5)


@pytest.mark.parametrize("change,message", [
    ("block", "block table"), ("length", "context length"), ("negative", "context length"),
    ("row", "sequence row"),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [40, 1 << 40])
def test_decode_reports_bad_input_and_spares_the_other_rows(dtype, change, message, window):
    c = Packed([70, 50, 200], [1] * 3, 14, 2, 64, 16, dtype, window, 5, seed=10)
    good = c.decode()
    rows = torch.arange(3, dtype=torch.int32, device=DEV)
    if change == "block":
        c.table[1, 2] = c.k.size(1)
    elif change == "length":
        c.len_d[1] = c.table.size(1) * 16 + 1
    elif change == "negative":
        c.len_d[1] = -5
    else:
        rows[1] = 3
    out = c.decode(seq_rows=rows)
    with pytest.raises(RuntimeError, match=message):
        ops.take_status()
    assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    if change != "block":
        assert bool((out[1] == SENTINEL).all())


@pytest.mark.parametrize("far", [-1e30, 1e30, -1e8, 2e35])
@pytest.mark.parametrize("new,head_dim", [(1, 64), (1, 128), (100, 64), (100, 128)])
def test_scores_far_from_zero(new, head_dim, far):
    # One dim of every key makes all scores of a row the same huge number (the query's
    # other dims are 0): the output is the mean of the visible values.
    c = Packed([300], [new], 14, 2, head_dim, 16, torch.bfloat16, 120, 0, seed=8)
    c.q[..., 0] = 1.0
    c.q[..., 1:] = 0.0
    x = fmt.unpack(c.k.cpu()).nan_to_num(0.0)
    x[..., 0] = far
    c.k = fmt.pack(*fmt.quantise(x)).to(DEV)
    out = (c.decode if new == 1 else c.chunks)().double().cpu()
    assert ops.take_status() == 0
    for t, p in enumerate(range(300 - new, 300)):
        v = c.values[0][:, max(0, p - 119): p + 1].double()
        want = v.mean(1).repeat_interleave(7, 0)
        size = v.abs().mean(1).repeat_interleave(7, 0)
        # Weights of exactly 1: the sums' roundings (n + 64 of them) and the output's.
        tol = 2 * 200 * 2.0 ** -24 * size + 2.0 ** -8 * (want.abs() + 2.0 ** -8 * size)
        assert bool(((out[t] - want).abs() <= tol).all()), t


# ------------------------------------------------------------------ chunks


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,head_dim,block", [
    (14, 2, 64, 16), (28, 4, 128, 16), (8, 8, 64, 16), (16, 1, 64, 32), (3, 1, 96, 16),
    (4, 2, 32, 4), (6, 2, 256, 16), (15, 3, 128, 64),
])
@pytest.mark.parametrize("window,sinks", [(60, 6), (1 << 40, 0)])
def test_chunk_shapes(dtype, heads, kv_heads, head_dim, block, window, sinks):
    news = [1, 5, 16, 17, 40, 130, 3]
    priors = [0, 3, 16, 31, 0, 200, 77]
    c = Packed([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, block, dtype,
               window, sinks, seed=heads)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (64, 0), (64, 64), (100, 130), (37, 1),
                                          (1000, 7), (0, 0), (20, 1 << 40)])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(14, 2, 64), (8, 2, 128)])
def test_chunk_windows(window, sinks, heads, kv_heads, head_dim):
    news = [300, 9, 64, 1, 128]
    priors = [500, 1000, 0, 129, 190]
    c = Packed([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, 16,
               torch.bfloat16, window or 1 << 40, sinks, seed=sinks % 1000)
    if not window:
        c.args = (0, 0)
    out = c.chunks()
    c.args = (window or 1 << 40, sinks)
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("news,priors", [
    ([512] * 8, [3485, 2609, 2094, 1105, 1261, 167, 308, 67]), ([2000], [3000]), ([33], [6000]),
    ([1], [0]), ([5] * 40, [90 + 31 * i for i in range(40)]), ([9, 1, 200], [4000, 15, 0]),
])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(14, 2, 64), (28, 4, 128)])
def test_chunk_batches(news, priors, heads, kv_heads, head_dim):
    c = Packed([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, 16,
               torch.bfloat16, 1 << 40, 0, seed=21)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)
    for _ in range(3):
        assert torch.equal(c.chunks(), out)


def test_chunk_padding_rows_and_rows_past_the_last_chunk():
    news, priors = [20, 0, 35], [50, 10, 0]
    c = Packed([p + n for p, n in zip(priors, news)], news, 14, 2, 64, 16, torch.bfloat16, 1 << 40,
               0, seed=31)
    plain = c.chunks()
    c.check(plain)
    T = c.T + 15
    q = torch.randn(T, 14, 64, device=DEV).bfloat16()
    q[: c.T] = c.q.to(DEV)
    cu = torch.cat([c.cu, c.cu[-1:], c.cu[-1:] + 9])
    ctx = torch.cat([c.len_d, torch.zeros(2, dtype=torch.int32, device=DEV)])
    rows = torch.tensor([0, 1, 2, 0, 77], dtype=torch.int32, device=DEV)
    out = torch.full((T, 14, 64), SENTINEL, dtype=torch.bfloat16, device=DEV)
    ops.int4_prefill_attention(q, c.k, c.v, c.table, cu, ctx, c.scale, 64, seq_rows=rows, out=out)
    assert ops.take_status() == 0
    assert torch.equal(out[: c.T], plain) and bool((out[c.T:] == SENTINEL).all())


@pytest.mark.parametrize("scale", [0.0, -0.3, 20.0])
@pytest.mark.parametrize("dtype,head_dim", [(torch.bfloat16, 64), (torch.bfloat16, 128),
                                            (torch.float32, 64)])
def test_chunk_scales(scale, dtype, head_dim):
    news, priors = [150, 30], [300, 90]
    c = Packed([p + n for p, n in zip(priors, news)], news, 8, 2, head_dim, 16, dtype, 200, 4,
               seed=34)
    c.scale = scale
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("rows", [256, 257, 700])
def test_chunk_many_sequences(rows):
    news = [1 + (7 * i) % 5 for i in range(rows)]
    priors = [(37 * i) % 90 for i in range(rows)]
    c = Packed([p + n for p, n in zip(priors, news)], news, 4, 2, 64, 16, torch.bfloat16, 1 << 40, 0,
               seed=36)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("change,message", [
    ("block", "block table"), ("context", "context length"), ("table", "context length"),
    ("row", "sequence row"), ("long", "context length"), ("outside", "context length"),
    ("backwards", "context length"),
])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_chunk_reports_bad_input_and_spares_the_others(change, message, head_dim):
    news, priors = [40, 30, 50], [60, 70, 10]
    c = Packed([p + n for p, n in zip(priors, news)], news, 14, 2, head_dim, 16, torch.bfloat16, 40,
               5, seed=33)
    good = c.chunks()
    rows = torch.arange(3, dtype=torch.int32, device=DEV)
    kw, skipped = {}, slice(40, 70)
    if change == "block":
        c.table[1, 5] = -1
    elif change == "context":
        c.len_d[1] = 29
    elif change == "table":
        c.len_d[1] = c.table.size(1) * 16 + 1
    elif change == "row":
        rows[1] = -1
    else:
        skipped = slice(70, 120)
        if change == "long":
            kw["max_query_len"] = 40  # the last chunk holds 50
        elif change == "outside":
            c.cu[3] = 121  # one token past the query's rows
            c.len_d[2] += 1
            kw["max_query_len"] = 64
        else:
            c.cu[3] = 60  # ends before it begins
    out = c.chunks(seq_rows=rows, **kw)
    with pytest.raises(RuntimeError, match=message):
        ops.take_status()
    if change != "block":
        assert bool((out[skipped] == SENTINEL).all())
    keep = torch.ones(120, dtype=torch.bool)
    keep[skipped] = False
    assert torch.equal(out[keep.to(DEV)], good[keep.to(DEV)])


# Chunks of a few tokens (the decode kernel's form of several tokens a row).


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (6, 2), (5, 1), (7, 1), (16, 2), (11, 1),
                                            (16, 1)])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("longest", [2, 3, 5, 8, 13])
def test_short_chunks(heads, kv_heads, head_dim, longest):
    # Ends before, at and behind the borders of 16 and 32 keys, chunks longer than what is behind
    # them, and a long sequence that several warps and CTAs share.
    priors = [0, 1, 10, 14, 15, 16, 30, 31, 33, 61, 128, 5000, 700]
    news = [1 + (3 * i + longest - 1) % longest for i in range(len(priors))]
    c = Packed([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, 16,
               torch.bfloat16, 1 << 40, 0, seed=heads + longest)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 17), (15, 0), (16, 16), (17, 33),
                                          (64, 3), (200, 1 << 40), (200, 5), (4000, 1)])
@pytest.mark.parametrize("heads,kv_heads,head_dim,block", [(14, 2, 64, 16), (8, 2, 128, 32)])
def test_short_chunk_windows(window, sinks, heads, kv_heads, head_dim, block):
    news = [5, 3, 1, 5, 4, 5, 2]
    priors = [500, 0, 13, 194, 3000, 40, 5000]
    c = Packed([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, block,
               torch.bfloat16, window, sinks, seed=sinks % 1000)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("rows,longest,window", [(1, 4, 100), (1, 5, 1 << 40), (6, 5, 777),
                                                 (40, 7, 1 << 40), (300, 2, 64)])
def test_short_chunks_by_clusters_and_by_records(heads, kv_heads, head_dim, rows, longest, window):
    news = [1 + (5 * i + longest - 1) % longest for i in range(rows)]
    priors = [(997 * i + 2000) % 3000 for i in range(rows)]
    c = Packed([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, 16,
               torch.bfloat16, window, 3, seed=rows)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)
    for _ in range(3):
        assert torch.equal(c.chunks(), out)


def test_short_chunks_of_more_sequences_than_the_span_scan_stages():
    rows = 9000
    news = [1 + (7 * i) % 3 for i in range(rows)]
    priors = [(37 * i) % 40 for i in range(rows)]
    c = Packed([p + n for p, n in zip(priors, news)], news, 2, 1, 64, 16, torch.bfloat16, 1 << 40, 0,
               seed=37)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


def test_short_chunk_padding_and_strides():
    news, priors = [2, 0, 5, 1], [50, 10, 300, 0]
    c = Packed([p + n for p, n in zip(priors, news)], news, 14, 2, 64, 16, torch.bfloat16, 1 << 40,
               0, seed=31)
    plain = c.chunks()
    c.check(plain)
    T = c.T + 9
    wide = torch.randn(T, 14 * 64 + 24, device=DEV).bfloat16()
    q = wide[:, 8:-16].unflatten(1, (14, 64))
    q[: c.T] = c.q.to(DEV)
    cu = torch.cat([c.cu, c.cu[-1:], c.cu[-1:] + 4])
    ctx = torch.cat([c.len_d, torch.zeros(2, dtype=torch.int32, device=DEV)])
    rows = torch.tensor([0, 1, 2, 3, 0, 77], dtype=torch.int32, device=DEV)
    room = torch.full((T, 16 * 64), SENTINEL, dtype=torch.bfloat16, device=DEV)
    out = room[:, : 14 * 64].unflatten(1, (14, 64))
    ops.int4_prefill_attention(q, c.k, c.v, c.table, cu, ctx, c.scale, 8, seq_rows=rows, out=out)
    assert ops.take_status() == 0
    assert torch.equal(out[: c.T], plain) and bool((out[c.T:] == SENTINEL).all())
    assert bool((room[:, 14 * 64:] == SENTINEL).all())


@pytest.mark.parametrize("far", [-1e30, 1e30, 2e35])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_short_chunk_scores_far_from_zero(head_dim, far):
    test_scores_far_from_zero(2, head_dim, far)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("head_dim,priors", [(64, [300, 20]), (128, [300, 20]), (64, [5000, 9])])
def test_short_chunk_rows_of_non_finite_queries_stay_alone(head_dim, priors, bad):
    c = Packed([p + 2 for p in priors], [2] * 2, 14, 2, head_dim, 16, torch.bfloat16, 1 << 40, 0,
               seed=35)
    want = c.chunks()
    c.check(want)
    c.q[1, 3, 5] = bad
    out = c.chunks()
    assert ops.take_status() == 0
    assert not bool(out[1, 3].isfinite().all())
    keep = torch.ones(4, 14, dtype=torch.bool)
    keep[1, 3] = False
    assert torch.equal(out[keep.to(DEV)], want[keep.to(DEV)])


@pytest.mark.parametrize("scale", [0.0, -0.3, 20.0])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_short_chunk_scales(scale, head_dim):
    news, priors = [5, 3], [300, 90]
    c = Packed([p + n for p, n in zip(priors, news)], news, 8, 2, head_dim, 16, torch.bfloat16, 200,
               4, seed=34)
    c.scale = scale
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("change,message", [
    ("block", "block table"), ("context", "context length"), ("table", "context length"),
    ("row", "sequence row"), ("long", "context length"), ("outside", "context length"),
    ("backwards", "context length"),
])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_short_chunk_reports_bad_input_and_spares_the_others(change, message, head_dim):
    news, priors = [4, 3, 5], [60, 70, 10]
    c = Packed([p + n for p, n in zip(priors, news)], news, 14, 2, head_dim, 16, torch.bfloat16, 40,
               5, seed=33)
    ref, tol = c.reference()
    good = c.chunks()
    rows = torch.arange(3, dtype=torch.int32, device=DEV)
    kw, skipped = {}, slice(4, 7)
    if change == "block":
        c.table[1, 4] = -1
    elif change == "context":
        c.len_d[1] = 2
    elif change == "table":
        c.len_d[1] = c.table.size(1) * 16 + 1
    elif change == "row":
        rows[1] = -1
    else:
        skipped = slice(7, 12)
        if change == "long":
            kw["max_query_len"] = 4  # the last chunk holds 5
        elif change == "outside":
            c.cu[3] = 13  # one token past the query's rows
            c.len_d[2] += 1
            kw["max_query_len"] = 6
        else:
            c.cu[3] = 6  # ends before it begins
    out = c.chunks(seq_rows=rows, **kw)
    with pytest.raises(RuntimeError, match=message):
        ops.take_status()
    if change != "block":
        assert bool((out[skipped] == SENTINEL).all())
    spared = [t for t in range(12) if not skipped.start <= t < skipped.stop]
    # (Another max_query_len may cut a chunk and share its keys out differently: the same sums in
    # another order, each within the tolerance of the reference.)
    if "max_query_len" not in kw:
        assert torch.equal(out[spared], good[spared])
    assert bool(((out.double().cpu() - ref).abs() <= tol)[spared].all())


@pytest.mark.parametrize("dtype,head_dim,blocks", [
    (torch.bfloat16, 128, 1_000_000), (torch.bfloat16, 64, 2_000_000), (torch.float32, 96, 1_300_000)])
def test_pool_past_32_bit_offsets(dtype, head_dim, blocks):
    # More than 2^31 bytes a pool, the sequences in the last blocks of the last head.
    news, priors = [20, 150], [700, 0]
    c = Packed([p + n for p, n in zip(priors, news)], news, 14, 2, head_dim, 16, dtype, 400, 4,
               seed=38)
    few, row = c.k.shape[1], c.k.shape[3]
    assert 2 * blocks * 16 * row > 2 ** 31
    for name in ("k", "v"):
        big = torch.zeros(2, blocks, 16, row, dtype=torch.uint8, device=DEV)
        big[:, blocks - few:] = getattr(c, name)
        setattr(c, name, big)
    c.table[c.table < few] += blocks - few
    c.check(c.chunks())
    one = Packed([720, 150], [1, 1], 14, 2, head_dim, 16, dtype, 400, 4, seed=39)
    few = one.k.shape[1]
    for name in ("k", "v"):
        getattr(c, name)[:, blocks - few:] = getattr(one, name)
        setattr(one, name, getattr(c, name))
    one.table[one.table < few] += blocks - few
    one.check(one.decode())
    # Append to, and read, the last slots.
    x = torch.randn(3, 4 * head_dim, generator=torch.Generator().manual_seed(9))
    slots = torch.arange(blocks * 16 - 3, blocks * 16, dtype=torch.int32, device=DEV)
    none = torch.zeros(0, dtype=torch.float64, device=DEV)
    ops.rotary_append_int4(x.to(DEV), none, slots, slots, c.k, c.v, 0)
    k, v = ops.read_int4(c.k, c.v, slots)
    assert torch.equal(k.cpu().double(), fmt.held(x[:, : 2 * head_dim]).view(3, 2, -1))
    assert torch.equal(v.cpu().double(), fmt.held(x[:, 2 * head_dim:]).view(3, 2, -1))
    assert ops.take_status() == 0


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 14, 2), (128, 8, 2)])
def test_prompt_then_tokens_then_drafts(head_dim, heads, kv_heads):
    # A conversation as it is served: a prompt in two chunks, single tokens, then a chunk of
    # drafts, each appended and attended over; checked against attention over what the cache
    # holds of the same keys and values.
    g = torch.Generator().manual_seed(11)
    steps = [70, 45, 1, 1, 1, 5]
    total = sum(steps)
    nb = -(-total // 16) + 2
    table = torch.randperm(nb, generator=g)[: -(-total // 16)].int().to(DEV)[None]
    pools = [torch.full(ops.int4_pool_shape(kv_heads, nb, 16, head_dim), 255, dtype=torch.uint8,
                        device=DEV) for _ in range(2)]
    freq, amplitude = ops.rope_frequencies(head_dim, 1e4, device=DEV)
    qkv = torch.randn(total, heads + 2 * kv_heads, head_dim, generator=g).bfloat16()
    x = rotated(qkv, freq.cpu(), torch.arange(total), heads + kv_heads, head_dim, False, amplitude)
    keys, vals = fmt.held(x[:, heads:]), fmt.held(qkv[:, heads + kv_heads:])
    at = 0
    for n in steps:
        pos = torch.arange(at, at + n, dtype=torch.int32, device=DEV)
        slots = table[0, (pos // 16).long()] * 16 + pos % 16
        q = ops.rotary_append_int4(qkv[at: at + n].to(DEV), freq, pos, slots, *pools, heads)
        lens = torch.tensor([at + n], dtype=torch.int32, device=DEV)
        if n == 1:
            out = ops.int4_attention_batched(q, *pools, table, lens, head_dim ** -0.5)
        else:
            cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
            out = ops.int4_prefill_attention(q, *pools, table, cu, lens, head_dim ** -0.5, n)
        c = Packed([at + n], [n], heads, kv_heads, head_dim, 16, torch.bfloat16, 1 << 40, 0)
        c.q = q.cpu()
        c.keys = [keys[: at + n].transpose(0, 1).float()]
        c.values = [vals[: at + n].transpose(0, 1).float()]
        c.check(out)
        at += n
    assert ops.take_status() == 0


def test_other_streams_and_two_calls_at_once():
    a = Packed([900, 30, 4000], [1] * 3, 14, 2, 64, 16, torch.bfloat16, 1 << 40, 0, seed=41)
    b = Packed([700] * 5, [60] * 5, 14, 2, 64, 16, torch.bfloat16, 1 << 40, 0, seed=42)
    want_a, want_b = a.decode(), b.chunks()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            out_a = a.decode()
            twice = a.decode()
        with torch.cuda.stream(s2):
            out_b = b.chunks()
        torch.cuda.synchronize()
        assert torch.equal(out_a, want_a) and torch.equal(twice, want_a)
        assert torch.equal(out_b, want_b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_calls_share_no_scratch(dtype):
    cases = [Packed([6000] * 2, [1] * 2, 14, 2, 64, 16, dtype, 1 << 40, 0, seed=s) for s in (51, 52)]
    chunks = [Packed([6000], [40], 14, 2, 64, 16, dtype, 1 << 40, 0, seed=s) for s in (53, 54)]
    runs = []
    for c, chunk in [(c, False) for c in cases] + [(c, True) for c in chunks]:
        want = c.chunks() if chunk else c.decode()
        q, out = c.q.to(DEV), torch.zeros_like(want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            if chunk:
                ops.int4_prefill_attention(q, c.k, c.v, c.table, c.cu, c.len_d, c.scale, 40, out=out)
            else:
                ops.int4_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, out=out)
        runs.append((graph, q, out, want, torch.cuda.Stream()))
    for _ in range(10):
        for graph, _, _, _, s in runs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out, want, _ in runs:
            assert torch.equal(out, want)
            out.zero_()
        torch.cuda.synchronize()
    assert ops.take_status() == 0


def test_captured_short_chunks_share_no_scratch_and_follow_their_inputs():
    # Few and many chunks (clusters, spans), replayed on two streams at once; then the first chunk
    # of each becomes padding, which leaves its rows as they were and moves nothing else.
    cases = [Packed([p + 2 for p in priors], [2] * len(priors), 14, 2, 64, 16, torch.bfloat16,
                    1 << 40, 0, seed=s)
             for s, priors in ((57, [100, 40, 9]), (58, [1000 + 7 * i for i in range(90)]),
                               (59, [3000 + 11 * i for i in range(70)]))]
    runs = []
    for c in cases:
        want = c.chunks()
        c.check(want)
        q, out = c.q.to(DEV), torch.zeros_like(want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.int4_prefill_attention(q, c.k, c.v, c.table, c.cu, c.len_d, c.scale, 2, out=out)
        runs.append((graph, q, out, want, torch.cuda.Stream()))
    for turn in range(6):
        for c, (graph, _, out, _, s) in zip(cases, runs):
            if turn == 3:
                c.len_d[0] = 0
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                out.fill_(SENTINEL)
        for graph, _, _, _, s in runs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for c, (_, q, out, want, _) in zip(cases, runs):
            if turn < 3:
                assert torch.equal(out, want)
                continue
            # (The spans are others now: the same sums in another order.)
            assert bool((out[:2] == SENTINEL).all())
            ref, tol = c.reference()
            assert bool(((out.double().cpu() - ref).abs() <= tol)[2:].all())
    assert ops.take_status() == 0


def test_a_captured_step_follows_its_inputs():
    # Append and attention in one graph, replayed for the next tokens of three sequences (one
    # of them padding at first).
    H, Hkv, D = 14, 2, 64
    g = torch.Generator().manual_seed(12)
    c = Packed([40, 90, 15], [1] * 3, H, Hkv, D, 16, torch.bfloat16, 1 << 40, 0, seed=61)
    table = torch.full((3, 8), 1 << 30, dtype=torch.int32, device=DEV)
    nb = 24
    table[:] = torch.randperm(nb, generator=g)[:24].view(3, 8).int()
    pools = [torch.full(ops.int4_pool_shape(Hkv, nb, 16, D), 255, dtype=torch.uint8, device=DEV)
             for _ in range(2)]
    freq = torch.zeros(0, dtype=torch.float64, device=DEV)
    qkv = torch.zeros(3, (H + 2 * Hkv) * D, dtype=torch.bfloat16, device=DEV)
    pos, slots, lens = (torch.zeros(3, dtype=torch.int32, device=DEV) for _ in range(3))
    out = torch.full((3, H, D), SENTINEL, dtype=torch.bfloat16, device=DEV)
    slots.fill_(-1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = ops.rotary_append_int4(qkv, freq, pos, slots, *pools, H)
        ops.int4_attention_batched(q, *pools, table, lens, c.scale, out=out)
    rows = [[], [], []]
    for step in range(40):
        new = torch.randn(3, H + 2 * Hkv, D, generator=g).bfloat16()
        live = [step < 30, True, step >= 5]
        p = [len(r) for r in rows]
        qkv.copy_(new.view(3, -1))
        slots.copy_(torch.tensor([int(table[r, p[r] // 16]) * 16 + p[r] % 16 if live[r] else -1
                                  for r in range(3)], dtype=torch.int32))
        lens.copy_(torch.tensor([p[r] + 1 if live[r] else 0 for r in range(3)], dtype=torch.int32))
        for r in range(3):
            if live[r]:
                rows[r].append(new[r])
        out.fill_(SENTINEL)
        graph.replay()
        if step % 13 == 0 or step == 39:
            ref = Packed([len(r) if live[i] else 0 for i, r in enumerate(rows)], [1] * 3, H, Hkv, D,
                         16, torch.bfloat16, 1 << 40, 0)
            ref.q = new[:, :H]
            for r in range(3):
                if live[r]:
                    x = torch.stack(rows[r]).double()
                    ref.keys[r] = fmt.held(x[:, H: H + Hkv]).transpose(0, 1).float()
                    ref.values[r] = fmt.held(x[:, H + Hkv:]).transpose(0, 1).float()
            ref.check(out)
    assert ops.take_status() == 0


# ------------------------------------------------------------------ refusals


def test_wrappers_refuse():
    c = Packed([70, 3], [1, 1], 14, 2, 64, 16, torch.bfloat16, 40, 5)
    q = c.q.to(DEV)

    def call(**kw):
        args = dict(query=q, key_pool=c.k, value_pool=c.v, block_tables=c.table,
                    context_lens=c.len_d, scaling=0.125, window=40, sinks=5)
        args.update(kw)
        return ops.int4_attention_batched(**args)

    call()
    for kw in (dict(query=q[0]), dict(query=q.half()), dict(query=q[..., :32]),
               dict(value_pool=c.v[:, :2]), dict(key_pool=c.k.transpose(1, 2)),
               dict(key_pool=c.k.view(torch.int8)), dict(key_pool=c.k[..., :35], value_pool=c.v[..., :35]),
               dict(block_tables=c.table.long()), dict(block_tables=c.table[0]),
               dict(context_lens=c.len_d.long()), dict(context_lens=c.len_d[:1]),
               dict(seq_rows=c.len_d[:1]), dict(window=-1), dict(sinks=-1),
               dict(out=torch.empty(2, 14, 64, device=DEV)),
               dict(max_blocks_per_seq=c.table.size(1) + 1), dict(context_lens=c.len_d.cpu()),
               dict(query=q[:, :13])):
        with pytest.raises(RuntimeError):
            call(**kw)
    with pytest.raises(RuntimeError):
        ops.int4_prefill_attention(q, c.k, c.v, c.table, c.cu[:2], c.len_d, 0.125, 1)
    with pytest.raises(RuntimeError):
        ops.int4_prefill_attention(q, c.k, c.v, c.table, c.cu, c.len_d, 0.125, 0)
    qkv = torch.zeros(2, 18 * 64, dtype=torch.bfloat16, device=DEV)
    index = torch.zeros(2, dtype=torch.int32, device=DEV)
    freq = torch.zeros(32, dtype=torch.float64, device=DEV)

    def append(**kw):
        args = dict(qkv=qkv, frequencies=freq, positions=index, slot_mapping=index - 1, key_pool=c.k,
                    value_pool=c.v, num_heads=14)
        args.update(kw)
        return ops.rotary_append_int4(**args)

    append()
    for kw in (dict(qkv=qkv.half()), dict(qkv=qkv[:, :-1]), dict(frequencies=freq.float()),
               dict(frequencies=freq.repeat(2)), dict(positions=index.long()),
               dict(slot_mapping=index[:1]), dict(num_heads=-1), dict(amplitude=math.inf),
               dict(key_pool=c.k.view(torch.int8)), dict(query_out=qkv[:, : 14 * 64]),
               dict(qkv=qkv[:1])):
        with pytest.raises(RuntimeError):
            append(**kw)
    with pytest.raises(RuntimeError):
        ops.read_int4(c.k, c.v, index.long())
    with pytest.raises(RuntimeError):
        ops.read_int4(c.k[0], c.v[0], index)
    with pytest.raises(RuntimeError):
        ops.copy_blocks(c.k[..., :35].contiguous(), c.v[..., :35].contiguous(), index, index)
    assert ops.take_status() == 0

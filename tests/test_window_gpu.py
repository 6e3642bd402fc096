"""Sliding-window attention with sink tokens on the GPU against the formula in 64
bits, for single tokens and prompt chunks.

Tolerance, element by element, with A = sum_j softmax_j |v_j| (the output if no
terms cancelled), n visible keys and u = 2^-24:

  * scores: a fp32 dot product of D terms, scaled, is off by at most
    (D + 8) u sum_d |q_d k_d| |scale|; delta is that at its largest, plus 2^-20 for
    the hardware exponential (2 ulp) and its argument's rounding; weights and
    their sum then move the output by at most 2 delta A;
  * sums: at most (n + 64) u A for each of the numerator and the denominator
    (any order of n + 64 additions, joins of partial results included);
  * bf16 only: the tensor-core kernels round each weight to bf16 before it
    multiplies V (half a step, 2^-8, of each term: 2^-8 A), and the output is
    rounded (2^-8 of its value);
  * fp32: the division and the output's rounding, 2 u of the value.
"""

import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from batchstream_inference_engine_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SENTINEL = 768.0


def visible(length, window, sinks):
    """Positions that the token at length - 1 sees."""
    return [j for j in range(length) if j < sinks or j > length - 1 - window]


class Paged:
    """Sequences of random K/V paged over a shuffled pool.  Every slot that no
    query token sees holds NaN (K) and infinity (V), and the table entries of
    blocks without a visible token are out of range."""

    def __init__(self, lens, news, heads, kv_heads, head_dim, block, dtype, window, sinks, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.args = (window, sinks)
        self.lens, self.news = lens, news
        self.H, self.Hkv, self.D, self.bs, self.dtype = heads, kv_heads, head_dim, block, dtype
        need = [-(-n // block) for n in lens]
        nb = sum(need) + 3
        order = torch.randperm(nb, generator=g).tolist()
        k = torch.full((kv_heads, nb * block, head_dim), math.nan)
        v = torch.full((kv_heads, nb * block, head_dim), math.inf)
        width = max(max(need), 1) + 1
        table = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
        self.keys, self.values = [], []
        at = 0
        for r, (n, new) in enumerate(zip(lens, news)):
            kk = torch.randn(kv_heads, n, head_dim, generator=g).to(dtype).float()
            vv = torch.randn(kv_heads, n, head_dim, generator=g).to(dtype).float()
            kk[:, : min(sinks, n)] *= 1.5  # sink tokens draw more weight
            kk = kk.to(dtype).float()
            self.keys.append(kk)
            self.values.append(vv)
            blocks = order[at: at + need[r]]
            at += need[r]
            first = max(0, n - new - window + 1)  # the first new token's window
            seen = [p for p in range(n) if p < sinks or p >= first] if new else []
            for p in seen:
                slot = blocks[p // block] * block + p % block
                k[:, slot], v[:, slot] = kk[:, p], vv[:, p]
                table[r, p // block] = blocks[p // block]
        self.k = k.view(kv_heads, nb, block, head_dim).to(dtype).to(DEV)
        self.v = v.view(kv_heads, nb, block, head_dim).to(dtype).to(DEV)
        self.table = table.to(DEV)
        self.T = sum(news)
        self.q = torch.randn(self.T, heads, head_dim, generator=g).to(dtype)
        self.scale = head_dim ** -0.5
        self.len_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
        offsets = [0]
        for new in news:
            offsets.append(offsets[-1] + new)
        self.cu = torch.tensor(offsets, dtype=torch.int32, device=DEV)

    def decode(self, **kw):
        out = torch.full((self.T, self.H, self.D), SENTINEL, dtype=self.dtype, device=DEV)
        got = ops.window_attention_batched(self.q.to(DEV), self.k, self.v, self.table, self.len_d,
                                           self.scale, *self.args, out=out, **kw)
        assert got is out
        return out

    def chunks(self, **kw):
        out = torch.full((self.T, self.H, self.D), SENTINEL, dtype=self.dtype, device=DEV)
        kw.setdefault("max_query_len", max(self.news))
        got = ops.window_prefill_attention(self.q.to(DEV), self.k, self.v, self.table, self.cu,
                                           self.len_d, self.scale, window=self.args[0],
                                           sinks=self.args[1], out=out, **kw)
        assert got is out
        return out

    def reference(self):
        """(outputs, tolerances) [T, H, D] in 64 bits; rows of empty sequences keep
        the sentinel."""
        window, sinks = self.args
        G = self.H // self.Hkv
        ref = torch.full((self.T, self.H, self.D), SENTINEL, dtype=torch.float64)
        tol = torch.zeros_like(ref)
        u = 2.0 ** -24
        at = 0
        for kk, vv, n, new in zip(self.keys, self.values, self.lens, self.news):
            if n == 0 or new == 0:
                at += new
                continue
            kk, vv = kk.double().to(DEV), vv.double().to(DEV)
            q = self.q[at: at + new].double().to(DEV).view(new, self.Hkv, G, self.D)
            pos = torch.arange(n - new, n, device=DEV)[:, None]
            j = torch.arange(n, device=DEV)[None]
            see = (j <= pos) & ((j < sinks) | (j > pos - window))
            s = torch.einsum("thgd,hkd->hgtk", q, kk) * self.scale
            p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            o = torch.einsum("hgtk,hkd->thgd", p, vv)
            big = torch.einsum("hgtk,hkd->thgd", p, vv.abs())
            size = torch.einsum("thgd,hkd->hgtk", q.abs(), kk.abs()) * abs(self.scale)
            size = size.masked_fill(~see, 0.0).amax(-1)  # [Hkv, G, new]
            delta = ((self.D + 8) * u * size + 2.0 ** -20).permute(2, 0, 1)[..., None]
            count = see.sum(-1).double()[:, None, None, None]
            t = 2 * delta * big + 2 * (count + 64) * u * big
            if self.dtype == torch.bfloat16:
                t = t + 2.0 ** -8 * big + 2.0 ** -8 * (o.abs() + t + 2.0 ** -8 * big)
            else:
                t = t + 2 * u * (o.abs() + t)
            ref[at: at + new] = o.reshape(new, self.H, self.D).cpu()
            tol[at: at + new] = t.reshape(new, self.H, self.D).cpu()
            at += new
        return ref, tol

    def check(self, out):
        ref, tol = self.reference()
        err = (out.double().cpu() - ref).abs()
        assert not out.isnan().any()
        bad = (err > tol).flatten(1).any(1).nonzero().flatten().tolist()
        assert not bad, (bad[:10], float((err / tol.clamp_min(1e-30)).max()))


# Lengths around every border of a window of 40 with 5 sinks in blocks of 16, an
# empty (padding) row, one token, and lengths far past the window.
BORDERS = [0, 1, 2, 15, 16, 17, 39, 40, 41, 44, 45, 46, 47, 48, 55, 56, 57, 64, 100, 0, 777, 1500]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,sinks", [(40, 5), (1, 0), (1, 1), (16, 16), (40, 0), (200, 33),
                                          (5, 2000), (1 << 40, 0), (300, 1 << 40)])
def test_decode_at_every_border(dtype, window, sinks):
    c = Paged(BORDERS, [1] * len(BORDERS), 14, 2, 64, 16, dtype, window, sinks, seed=window)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,head_dim,block", [
    (8, 8, 64, 16), (16, 1, 64, 16), (28, 4, 128, 16), (32, 2, 128, 32), (5, 1, 80, 16),
    (6, 2, 256, 16), (4, 2, 8, 4), (3, 1, 7, 5), (9, 3, 96, 48), (1, 1, 1, 1), (24, 2, 64, 64),
    (2, 1, 33, 16), (8, 1, 256, 3),
])
def test_decode_shapes(dtype, heads, kv_heads, head_dim, block):
    lens = [1, 0, 7, 33, 130, 131, 300, 65]
    c = Paged(lens, [1] * len(lens), heads, kv_heads, head_dim, block, dtype, 90, 6, seed=heads)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,window", [([9000], 1 << 30), ([5000, 1], 4096), ([1], 64),
                                         ([4099] * 3, 4000)])
def test_decode_long_rows_are_split_and_joined(dtype, lens, window):
    c = Paged(lens, [1] * len(lens), 14, 2, 64, 16, dtype, window, 4, seed=3)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)
    for _ in range(3):
        assert torch.equal(c.decode(), out)


def test_decode_large_batch_many_lengths():
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 900, (300,), generator=g).tolist()
    c = Paged(lens, [1] * 300, 14, 2, 64, 16, torch.bfloat16, 256, 4, seed=6)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)


def test_decode_more_sequences_than_the_span_scan_stages():
    # 5500 sequences: their lengths do not fit the stage memory, and there are more
    # segments than resident CTAs.
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(0, 60, (5500,), generator=g).tolist()
    c = Paged(lens, [1] * 5500, 2, 1, 64, 16, torch.bfloat16, 20, 3, seed=7)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("dtype,heads,kv_heads,head_dim", [
    (torch.float32, 14, 2, 64), (torch.float32, 8, 2, 256), (torch.bfloat16, 16, 2, 80),
    (torch.bfloat16, 14, 2, 64), (torch.bfloat16, 28, 4, 128)])
@pytest.mark.parametrize("rows,window", [(3, 100), (8, 777), (24, 777), (64, 777), (64, 200)])
def test_decode_by_clusters_and_by_records(dtype, heads, kv_heads, head_dim, rows, window):
    # Batches on both sides of the rules that let a sequence's CTAs join in a cluster,
    # of sequences on both sides of the sizes that one CTA takes alone, and empty ones.
    lens = [(0, 1, 17, 64, 120, 128, 130, 145, 300, 900)[i % 10] + i // 10 for i in range(rows)]
    c = Paged(lens, [1] * rows, heads, kv_heads, head_dim, 16, dtype, window, 4, seed=40)
    out = c.decode()
    assert ops.take_status() == 0
    c.check(out)
    assert torch.equal(out, c.decode())


def test_decode_output_may_be_the_query():
    for dtype in (torch.bfloat16, torch.float32):
        c = Paged([5000, 70, 3], [1] * 3, 14, 2, 64, 16, dtype, 4000, 4, seed=13)
        want = c.decode()
        q = c.q.to(DEV)
        ops.window_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, 4000, 4, out=q)
        assert torch.equal(q, want)


def test_decode_negative_and_zero_scale():
    # softmax of zeros weights every visible key alike; a negative scale turns the
    # order around.
    for dtype in (torch.bfloat16, torch.float32):
        for scale in (0.0, -0.3):
            c = Paged([70, 300], [1, 1], 14, 2, 64, 16, dtype, 40, 5, seed=14)
            c.scale = scale
            c.check(c.decode())


def test_decode_of_an_all_padding_batch_and_of_none():
    c = Paged([0, 0, 0], [1, 1, 1], 14, 2, 64, 16, torch.bfloat16, 40, 4)
    assert bool((c.decode() == SENTINEL).all())
    empty = torch.empty(0, 14, 64, dtype=torch.bfloat16, device=DEV)
    assert ops.window_attention_batched(empty, c.k, c.v, c.table, c.len_d, 0.1, 4).shape == (0, 14, 64)
    assert ops.take_status() == 0


def test_decode_strided_query_and_output_rows_and_lists():
    lens = [70, 3, 200, 41, 0, 90]
    c = Paged(lens, [1] * 6, 14, 2, 64, 16, torch.bfloat16, 40, 5, seed=8)
    plain = c.decode()
    # Query as the q part of fused rows, output as a slice of wider rows, every
    # other entry of longer lists, rows picked from a shuffled wider table.
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
    ops.window_attention_batched(fused.view(6, 18, 64)[:, :14], c.k, c.v, table, lens2[::2],
                                 c.scale, 40, 5, seq_rows=rows2[::2], out=wide[:, 3:17])
    assert ops.take_status() == 0
    assert torch.equal(wide[:, 3:17], plain)
    assert bool((wide[:, :3] == SENTINEL).all()) and bool((wide[:, 17:] == SENTINEL).all())
    # Heads that are not next to each other are copied first; a transposed table too.
    spread = torch.zeros(6, 14, 128, dtype=torch.bfloat16, device=DEV)
    spread[..., ::2] = c.q.to(DEV)
    out = torch.full_like(plain, SENTINEL)
    ops.window_attention_batched(spread[..., ::2], c.k, c.v, c.table.t().contiguous().t(), c.len_d,
                                 c.scale, 40, 5, out=out)
    assert torch.equal(out, plain)


def test_decode_unaligned_pool_and_query():
    # Views that start 2 bytes into their storage: every kernel choice must cope.
    lens = [70, 3, 200]
    c = Paged(lens, [1] * 3, 14, 2, 64, 16, torch.bfloat16, 40, 5, seed=9)

    def shifted(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    q = shifted(c.q.to(DEV))
    out = shifted(torch.zeros(3, 14, 64, dtype=torch.bfloat16, device=DEV))
    ops.window_attention_batched(q, shifted(c.k), shifted(c.v), c.table, c.len_d, c.scale, 40, 5,
                                 out=out)
    assert ops.take_status() == 0
    c.check(out)
    out2 = ops.window_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, 40, 5)
    c.check(out2)


@pytest.mark.parametrize("change,message", [
    ("block", "block table"), ("length", "context length"), ("negative", "context length"),
    ("row", "sequence row"),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_reports_bad_input_and_spares_the_other_rows(dtype, change, message):
    lens = [70, 50, 200]
    c = Paged(lens, [1] * 3, 14, 2, 64, 16, dtype, 40, 5, seed=10)
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


def test_decode_equals_full_attention_inside_the_window():
    # A window that covers every token: the framework's own full attention up to
    # its two roundings of the scores to bf16 (2^-8 of |s| each, which move a
    # weight by as much, hence the output by 2 * 2 * 2^-8 max |s| A) plus both
    # sides' own roundings.
    lens = [70, 33, 200]
    c = Paged(lens, [1] * 3, 14, 2, 64, 16, torch.bfloat16, 1 << 20, 0, seed=11)
    full = ops.paged_attention_batched(c.q.to(DEV), c.k, c.v, c.table, c.len_d, c.scale)
    ours = c.decode()
    ref, tol = c.reference()
    top = max(float((c.q[r].double().view(2, 7, 64) @ c.keys[r].double().transpose(1, 2)).abs().max())
              for r in range(3)) * c.scale
    bound = 2 * tol + 4 * 2.0 ** -8 * top * (tol / 2.0 ** -8)
    assert bool(((full.double() - ours.double()).abs().cpu() <= bound).all())


# ------------------------------------------------------------------ chunks


CHUNK_LAYOUTS = [
    # heads, kv heads, head_dim, block size
    (14, 2, 64, 16), (28, 4, 128, 16), (8, 8, 64, 16), (16, 1, 64, 32), (3, 1, 80, 16),
    (4, 2, 8, 4), (6, 2, 256, 16), (15, 3, 128, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,head_dim,block", CHUNK_LAYOUTS)
def test_chunk_shapes(dtype, heads, kv_heads, head_dim, block):
    news = [1, 5, 16, 17, 40, 130, 3]
    priors = [0, 3, 16, 31, 0, 200, 77]
    c = Paged([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, block, dtype,
              60, 6, seed=heads)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (64, 0), (64, 64), (100, 130), (37, 1),
                                          (1000, 7), (1 << 40, 0), (20, 1 << 40)])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(14, 2, 64), (8, 2, 128)])
def test_chunk_windows(dtype, window, sinks, heads, kv_heads, head_dim):
    news = [300, 9, 64, 1, 128]
    priors = [500, 1000, 0, 129, 190]
    c = Paged([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, 16, dtype,
              window, sinks, seed=sinks % 1000)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("news,priors,window", [
    ([512] * 8, [3485, 2609, 2094, 1105, 1261, 167, 308, 67], 1024),
    ([2000], [3000], 700), ([33], [6000], 4096), ([1], [0], 8), ([7] * 40, [90] * 40, 64),
])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(14, 2, 64), (28, 4, 128)])
def test_chunk_batches(news, priors, window, heads, kv_heads, head_dim):
    c = Paged([p + n for p, n in zip(priors, news)], news, heads, kv_heads, head_dim, 16,
              torch.bfloat16, window, 4, seed=21)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)
    for _ in range(3):
        assert torch.equal(c.chunks(), out)


@pytest.mark.parametrize("dtype,heads,kv_heads,head_dim", [
    (torch.bfloat16, 14, 2, 64), (torch.bfloat16, 8, 2, 128), (torch.float32, 8, 2, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_chunk_rows_are_not_touched_by_values_they_do_not_see(dtype, heads, kv_heads, head_dim, bad):
    # K and V of the token at position 250 (new token 50 of 150) and of the sink at
    # position 2 hold NaN or infinities.  Rows that do not see a bad key equal the
    # clean run's; rows that do are not finite.
    new, prior, window, sinks = 150, 200, 30, 0
    c = Paged([prior + new], [new], heads, kv_heads, head_dim, 16, dtype, window, sinks, seed=4)
    clean = c.chunks()
    at = 250
    slot = int(c.table[0, at // 16]) * 16 + at % 16
    c.v.view(kv_heads, -1, head_dim)[:, slot] = bad
    out = c.chunks()
    assert ops.take_status() == 0
    sees = [(at <= p < at + window) for p in range(prior, prior + new)]
    for t, seen in enumerate(sees):
        if seen:
            assert not out[t].isfinite().any(), t
        else:
            assert torch.equal(out[t], clean[t]), t
    # One dim only: the other dims of the rows that see it keep their values.
    c.v.view(kv_heads, -1, head_dim)[:, slot] = 0.25
    c.k.view(kv_heads, -1, head_dim)[:, slot] = 0.0
    base = c.chunks()
    c.v.view(kv_heads, -1, head_dim)[:, slot, 5] = bad
    out = c.chunks()
    keep = [d for d in range(head_dim) if d != 5]
    close = (out[..., keep].float() - base[..., keep].float()).abs() <= \
        2.0 ** -7 * base[..., keep].float().abs() + 2.0 ** -7
    assert bool(close.all())
    for t, seen in enumerate(sees):
        assert bool(out[t, :, 5].isfinite().all()) != seen
    c.k.view(kv_heads, -1, head_dim)[:, slot] = bad
    out = c.chunks()
    for t, seen in enumerate(sees):
        if not seen:
            assert torch.equal(out[t], clean[t]), t


def test_chunk_padding_rows_and_rows_past_the_last_chunk():
    news, priors = [20, 0, 35], [50, 10, 0]
    c = Paged([p + n for p, n in zip(priors, news)], news, 14, 2, 64, 16, torch.bfloat16, 40, 4,
              seed=31)
    plain = c.chunks()
    c.check(plain)
    # Two padding chunks (length 0: one empty, one of 9 tokens) and 6 rows behind.
    T = c.T + 15
    q = torch.randn(T, 14, 64, device=DEV).bfloat16()
    q[: c.T] = c.q.to(DEV)
    cu = torch.cat([c.cu, c.cu[-1:], c.cu[-1:] + 9])
    ctx = torch.cat([c.len_d, torch.zeros(2, dtype=torch.int32, device=DEV)])
    rows = torch.tensor([0, 1, 2, 0, 77], dtype=torch.int32, device=DEV)
    out = torch.full((T, 14, 64), SENTINEL, dtype=torch.bfloat16, device=DEV)
    ops.window_prefill_attention(q, c.k, c.v, c.table, cu, ctx, c.scale, 64, 40, 4, seq_rows=rows,
                                 out=out)
    assert ops.take_status() == 0
    assert torch.equal(out[: c.T], plain) and bool((out[c.T:] == SENTINEL).all())


@pytest.mark.parametrize("scale", [0.0, -0.3, 20.0])
@pytest.mark.parametrize("dtype,head_dim", [(torch.bfloat16, 64), (torch.bfloat16, 128),
                                            (torch.float32, 64)])
def test_chunk_scales(scale, dtype, head_dim):
    # 20 makes near one-hot rows whose maximum moves by far more than the rescaling
    # slack from step to step.
    news, priors = [150, 30], [300, 90]
    c = Paged([p + n for p, n in zip(priors, news)], news, 8, 2, head_dim, 16, dtype, 200, 4,
              seed=34)
    c.scale = scale
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


def test_chunk_bound_far_above_the_tokens():
    news, priors = [20, 150], [50, 0]
    for dtype in (torch.bfloat16, torch.float32):
        c = Paged([p + n for p, n in zip(priors, news)], news, 14, 2, 64, 16, dtype, 40, 4, seed=35)
        assert torch.equal(c.chunks(max_query_len=1 << 30), c.chunks(max_query_len=170))


@pytest.mark.parametrize("rows", [256, 257, 384, 385, 700])
def test_chunk_many_sequences(rows):
    # Up to 256 sequences are ranked inside every CTA, more run in order.
    news = [1 + (7 * i) % 5 for i in range(rows)]
    priors = [(37 * i) % 90 for i in range(rows)]
    c = Paged([p + n for p, n in zip(priors, news)], news, 4, 2, 64, 16, torch.bfloat16, 40, 4,
              seed=36)
    out = c.chunks()
    assert ops.take_status() == 0
    c.check(out)


@pytest.mark.parametrize("dtype,head_dim,blocks", [
    (torch.bfloat16, 128, 600_000), (torch.bfloat16, 64, 1_200_000), (torch.float32, 80, 850_000)])
def test_pool_past_32_bit_offsets(dtype, head_dim, blocks):
    # More than 2^31 elements a pool, the sequences in the last blocks of the last head.
    news, priors = [20, 150], [700, 0]
    c = Paged([p + n for p, n in zip(priors, news)], news, 14, 2, head_dim, 16, dtype, 400, 4,
              seed=38)
    few = c.k.shape[1]
    assert 2 * blocks * 16 * head_dim > 2 ** 31
    for name in ("k", "v"):
        small = getattr(c, name)
        big = torch.zeros(2, blocks, 16, head_dim, dtype=dtype, device=DEV)
        big[:, blocks - few:] = small
        setattr(c, name, big)
    c.table[c.table < few] += blocks - few
    c.check(c.chunks())
    one = Paged([720, 150], [1, 1], 14, 2, head_dim, 16, dtype, 400, 4, seed=39)
    few = one.k.shape[1]
    for name in ("k", "v"):
        getattr(c, name)[:, blocks - few:] = getattr(one, name)
        setattr(one, name, getattr(c, name))
    one.table[one.table < few] += blocks - few
    one.check(one.decode())
    assert ops.take_status() == 0


def test_chunk_strided_query_and_output():
    news, priors = [20, 150], [50, 0]
    c = Paged([p + n for p, n in zip(priors, news)], news, 14, 2, 64, 16, torch.bfloat16, 40, 4,
              seed=32)
    plain = c.chunks()
    fused = torch.randn(c.T, 18, 64, device=DEV).bfloat16()
    fused[:, :14] = c.q.to(DEV)
    wide = torch.full((c.T, 20, 64), SENTINEL, dtype=torch.bfloat16, device=DEV)
    ops.window_prefill_attention(fused[:, :14], c.k, c.v, c.table, c.cu, c.len_d, c.scale, 150, 40,
                                 4, out=wide[:, 3:17])
    assert ops.take_status() == 0
    assert torch.equal(wide[:, 3:17], plain)
    assert bool((wide[:, :3] == SENTINEL).all()) and bool((wide[:, 17:] == SENTINEL).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("change,message", [
    ("block", "block table"), ("context", "context length"), ("table", "context length"),
    ("row", "sequence row"), ("long", "context length"), ("outside", "context length"),
    ("backwards", "context length"),
])
def test_chunk_reports_bad_input_and_spares_the_others(dtype, change, message):
    news, priors = [40, 30, 50], [60, 70, 10]
    c = Paged([p + n for p, n in zip(priors, news)], news, 14, 2, 64, 16, dtype, 40, 5, seed=33)
    good = c.chunks()
    rows = torch.arange(3, dtype=torch.int32, device=DEV)
    kw = {}
    skipped = slice(40, 70)
    if change == "block":
        c.table[1, 5] = -1
    elif change == "context":
        c.len_d[1] = 29
    elif change == "table":
        c.len_d[1] = c.table.size(1) * 16 + 1
    elif change == "row":
        rows[1] = -1
    elif change == "long":
        kw["max_query_len"] = 40  # the last chunk holds 50
        skipped = slice(70, 120)
    elif change == "outside":
        c.cu[3] = 121  # one token past the query's rows
        c.len_d[2] += 1
        kw["max_query_len"] = 64
        skipped = slice(70, 120)
    else:
        c.cu[3] = 60  # ends before it begins
        skipped = slice(70, 120)
    out = c.chunks(seq_rows=rows, **kw)
    with pytest.raises(RuntimeError, match=message):
        ops.take_status()
    if change != "block":
        assert bool((out[skipped] == SENTINEL).all())
    keep = torch.ones(120, dtype=torch.bool)
    keep[skipped] = False
    assert torch.equal(out[keep.to(DEV)], good[keep.to(DEV)])


# ------------------------------------------------------------------ streams and graphs


def test_other_streams_and_two_calls_at_once():
    a = Paged([900, 30, 400], [1] * 3, 14, 2, 64, 16, torch.bfloat16, 300, 4, seed=41)
    b = Paged([700] * 5, [60] * 5, 14, 2, 64, 16, torch.bfloat16, 300, 4, seed=42)
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


def test_a_captured_call_reports_after_the_workspace_has_grown():
    c = Paged([70, 50], [1, 1], 14, 2, 64, 16, torch.bfloat16, 40, 5, seed=15)
    q, out = c.q.to(DEV), torch.zeros(2, 14, 64, dtype=torch.bfloat16, device=DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ops.window_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, 40, 5, out=out)
        assert ops.take_status() == 0
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.window_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, 40, 5, out=out)
        ops.workspace_for(torch.device("cuda", 0), 64 << 20)
        c.len_d[1] = -1
        graph.replay()
        with pytest.raises(RuntimeError, match="context length"):
            ops.take_status()
        c.len_d[1] = 50
        graph.replay()
        assert ops.take_status() == 0
        c.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_calls_share_no_scratch(dtype):
    # Two graphs whose calls need scratch, replayed at the same time on two streams.
    cases = [Paged([6000], [1], 14, 2, 64, 16, dtype, 5000, 4, seed=s) for s in (51, 52)]
    want = [c.decode() for c in cases]
    graphs, outs = [], []
    for c in cases:
        q = c.q.to(DEV)
        out = torch.zeros(1, 14, 64, dtype=dtype, device=DEV)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.window_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, 5000, 4, out=out)
        graphs.append((graph, q))
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
            out.zero_()
        torch.cuda.synchronize()
    assert ops.take_status() == 0


def test_a_captured_call_follows_its_inputs():
    c = Paged([600, 70, 300, 0], [1] * 4, 14, 2, 64, 16, torch.bfloat16, 128, 4, seed=61)
    q, out = c.q.to(DEV), torch.full((4, 14, 64), SENTINEL, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.window_attention_batched(q, c.k, c.v, c.table, c.len_d, c.scale, 128, 4, out=out)
    graph.replay()
    c.check(out)
    # Another batch of shorter rows in the same buffers; row 0 becomes padding.
    d = Paged([0, 50, 299, 1], [1] * 4, 14, 2, 64, 16, torch.bfloat16, 128, 4, seed=62)
    out.fill_(SENTINEL)
    q.copy_(d.q)
    c.k[:, : d.k.size(1)] = d.k
    c.v[:, : d.v.size(1)] = d.v
    c.table.fill_(1 << 30)
    c.table[:, : d.table.size(1)] = d.table
    c.len_d.copy_(d.len_d)
    graph.replay()
    d.check(out)
    assert ops.take_status() == 0


# ------------------------------------------------------------------ refusals


def test_wrappers_refuse():
    c = Paged([70, 3], [1, 1], 14, 2, 64, 16, torch.bfloat16, 40, 5)
    q = c.q.to(DEV)

    def call(**kw):
        args = dict(query=q, key_pool=c.k, value_pool=c.v, block_tables=c.table,
                    context_lens=c.len_d, scaling=0.125, window=40, sinks=5)
        args.update(kw)
        return ops.window_attention_batched(**args)

    call()
    for kw in (dict(query=q[0]), dict(query=q.float()), dict(query=q[..., :32]),
               dict(value_pool=c.v[:, :2]), dict(key_pool=c.k.transpose(1, 2)),
               dict(block_tables=c.table.long()), dict(block_tables=c.table[0]),
               dict(context_lens=c.len_d.long()), dict(context_lens=c.len_d[:1]),
               dict(seq_rows=c.len_d[:1]), dict(window=0), dict(sinks=-1),
               dict(out=torch.empty(2, 14, 64, device=DEV)),
               dict(out=torch.empty(2, 14, 32, dtype=torch.bfloat16, device=DEV)),
               dict(max_blocks_per_seq=c.table.size(1) + 1), dict(context_lens=c.len_d.cpu()),
               dict(query=q[:, :13])):
        with pytest.raises(RuntimeError):
            call(**kw)
    with pytest.raises(RuntimeError):
        ops.window_prefill_attention(q, c.k, c.v, c.table, c.cu[:2], c.len_d, 0.125, 1, 40)
    with pytest.raises(RuntimeError):
        ops.window_prefill_attention(q, c.k, c.v, c.table, c.cu, c.len_d, 0.125, 0, 40)
    assert ops.take_status() == 0


MERGES = """
import torch
from batchstream_inference_engine_b200 import ops
g = torch.Generator(device="cuda").manual_seed(0)
pool = lambda nb: torch.randn((2, nb, 16, 64), generator=g, device="cuda").bfloat16()
def call(rows, tokens, window, **kw):
    k, v = pool(rows * tokens // 16), pool(rows * tokens // 16)
    q = torch.randn((rows, 32, 64), generator=g, device="cuda").bfloat16()
    bt = torch.arange(k.size(1), dtype=torch.int32, device="cuda").view(rows, -1)
    lens = torch.full((rows,), tokens, dtype=torch.int32, device="cuda")
    if window:
        return lambda: ops.window_attention_batched(q, k, v, bt, lens, 0.125, window)
    return lambda: ops.paged_attention_batched(q, k, v, bt, lens, 0.125, **kw)
ORDERS = {
    # The merge pass takes 56 KB of shared memory behind the large calls, 33 KB or less
    # behind the small ones.
    "full first": (call(40, 4096, 0), call(1, 16384, 8192)),
    "window first": (call(40, 16384, 8192), call(1, 4096, 0, units_hint=512)),
}
large, small = ORDERS["%s"]
first = large()
small()
again = large()
assert torch.equal(first, again) and bool(first.isfinite().all())
assert ops.take_status() == 0
"""


@pytest.mark.parametrize("order", ["full first", "window first"])
def test_merge_passes_of_both_forms_in_one_process(order):
    # A process of its own: what the first large call sets up must outlast a small call
    # of the other form.
    root = Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", MERGES % order], cwd=root, capture_output=True,
                          text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("length,new,heads,kv_heads,window,dtype", [
    (300, 100, 14, 2, 120, torch.bfloat16), (478, 128, 2, 2, 351, torch.bfloat16),
    (300, 1, 14, 2, 120, torch.bfloat16), (300, 20, 14, 2, 120, torch.float32)])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("far", [-1e30, 1e30, -1e8, 3e37])
def test_scores_far_from_zero(length, new, heads, kv_heads, window, dtype, head_dim, far):
    # One dim of every key makes all scores of a row the same huge number (the query's
    # other dims are 0): the output is the mean of the visible values.
    c = Paged([length], [new], heads, kv_heads, head_dim, 16, dtype, window, 0, seed=8)
    c.q[..., 0] = 1.0
    c.q[..., 1:] = 0.0
    keys = c.k.view(kv_heads, -1, head_dim)
    keys[..., 0] = far
    out = (c.decode if new == 1 else c.chunks)().double().cpu()
    assert ops.take_status() == 0
    G = heads // kv_heads
    for t, p in enumerate(range(length - new, length)):
        v = c.values[0][:, max(0, p - window + 1): p + 1].double()
        mean, big = v.mean(1), v.abs().mean(1)
        # The weights are alike, but not 1: the maximum they are taken from is a rounded
        # product, up to 2^-24 of it off.  In bf16 each rounds by up to 2^-8 of itself.
        tol = 2 * (v.size(1) + 64) * 2.0 ** -24 * big
        if dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * big
        tol = tol + torch.finfo(dtype).eps / 2 * (mean.abs() + tol)
        err = (out[t] - mean.repeat_interleave(G, 0)).abs()
        assert bool((err <= tol.repeat_interleave(G, 0)).all()), (t, float(err.max()))


# (context, new tokens, heads, kv heads, window, sequences, keys of a part): the joins of
# four warps in one CTA, of 8 CTAs in a cluster, of spans over the batch, of the step
# ranges of a chunk (256 keys each), and of the CUDA-core kernel's ranges.
JOINS = [(49, 1, 14, 2, 64, 1, 1, torch.bfloat16), (1000, 1, 14, 2, 1024, 1, 120, torch.bfloat16),
         (16000, 1, 14, 2, 16000, 1, 200, torch.bfloat16),
         (900, 1, 14, 2, 1024, 200, 300, torch.bfloat16),
         (478, 128, 2, 2, 351, 1, 256, torch.bfloat16), (700, 30, 14, 2, 600, 1, 256, torch.bfloat16),
         (1000, 1, 14, 2, 1024, 1, 120, torch.float32), (700, 2, 14, 2, 600, 1, 256, torch.float32)]


@pytest.mark.parametrize("length,new,heads,kv_heads,window,seqs,part,dtype", JOINS)
@pytest.mark.parametrize("newest", [True, False])
def test_parts_without_a_finite_score_are_joined(length, new, heads, kv_heads, window, seqs, part,
                                                 dtype, newest):
    # The newest (or the oldest visible) keys, whole parts of a join, score NaN or -inf.
    c = Paged([length] * seqs, [new] * seqs, heads, kv_heads, 64, 16, dtype, window, 0, seed=7)
    run = c.decode if new == 1 else c.chunks
    c.q[..., 0] = c.q[..., 0].abs() + 0.5
    first = max(0, length - new - window + 1)
    at = range(length - part, length) if newest else range(first, first + part)
    table = c.table.cpu()
    slots = [int(table[r, p // 16]) * 16 + p % 16 for r in range(seqs) for p in at]
    keys = c.k.view(kv_heads, -1, 64)
    kept = keys[:, slots].clone()
    got = {}
    for value in (-math.inf, -1e30, math.nan):
        keys[:, slots] = kept
        keys[:, slots, 0] = value
        got[value] = run()
    assert ops.take_status() == 0
    pos = [p for p in range(length - new, length)] * seqs
    for t, p in enumerate(pos):
        sees = [j for j in at if p - window < j <= p]
        if sees:
            assert got[math.nan][t].isnan().all(), t
        if len(sees) < min(p + 1, window):  # another key is left
            # Weights of 0 either way.
            assert got[-1e30][t].isfinite().all() and torch.equal(got[-math.inf][t], got[-1e30][t]), t


@pytest.mark.parametrize("dtype,heads,head_dim,block,window,clustered,records", [
    # 444 CTAs run at once, or 48 clusters of 8, or 103 of 4.
    (torch.bfloat16, 16, 64, 8, 1000, (48, 60), (52,)),
    (torch.float32, 7, 48, 16, 1000, (48, 60), (52,)),
    (torch.float32, 7, 48, 16, 500, (96, 115), (108,))])
def test_clusters_while_they_take_no_more_waves(dtype, heads, head_dim, block, window, clustered,
                                                records):
    # Records need scratch, clusters do not.
    def scratch(rows):
        got = ctypes.c_uint64(0)
        _lib.check(_lib.lib().bs_window_attention_batched_workspace_bytes(
            rows, heads, 1, head_dim, block, 4096 // block, ops.dtype_code(dtype), window, 0,
            ctypes.byref(got)))
        return got.value

    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert [scratch(n) for n in clustered] == [0] * len(clustered)
        assert all(scratch(n) > 0 for n in records)
    for rows in (*clustered, *records):
        c = Paged([2 * window] * rows, [1] * rows, heads, 1, head_dim, block, dtype, window, 0,
                  seed=rows)
        out = c.decode()
        assert ops.take_status() == 0
        c.check(out)

"""Groups of rotated keys that only more than fp32 tells apart: extremes of either sign that
round up to one fp32 number, and largest elements just below a limit.  At position 0 a key is
its element times the amplitude, in fp64; the bytes are compared with the format's in 64 bits."""

import pytest
import torch

from batchstream_inference_engine_b200 import ops

from . import int4_format as fmt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def append(rows, amplitude, interleaved=False):
    """What the pool holds of fp32 keys [T, D] at position 0, fp64, and the keys in 64 bits."""
    T, D = rows.shape
    qkv = torch.cat([rows, torch.zeros_like(rows)], 1).to(DEV)
    pools = [torch.zeros(ops.int4_pool_shape(1, -(-T // 16), 16, D), dtype=torch.uint8, device=DEV)
             for _ in range(2)]
    index = torch.arange(T, dtype=torch.int32, device=DEV)
    freq = torch.ones(D // 2, dtype=torch.float64, device=DEV)
    ops.rotary_append_int4(qkv, freq, torch.zeros_like(index), index, *pools, 0,
                           interleaved=interleaved, amplitude=amplitude)
    return fmt.unpack(pools[0].cpu())[0].reshape(-1, D)[:T], rows.double() * amplitude


def round_up(x):
    """fp64 numbers rounded up to fp32."""
    f = x.float()
    return torch.where(f.double() < x, torch.nextafter(f, torch.full_like(f, torch.inf)), f)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_extremes_that_round_to_one_fp32_number(dim, interleaved):
    # Neighbouring fp32 numbers just below 2 times an amplitude near 0.56: steps of 0.56 fp32
    # steps of the products, so near half of the pairs round up to the same number.  (8 |s| is
    # 1.125, so that the sign decides what the largest element is held as.)
    amplitude, T = 0.5607, 64
    g = torch.Generator().manual_seed(dim)
    rows = torch.rand(T, dim, generator=g) - 0.5
    small = (2.0 - torch.arange(1, T + 1) * 2.0 ** -20).float()
    large = torch.nextafter(small, torch.full_like(small, 4.0))
    sign = torch.where(torch.arange(T) % 4 < 2, 1.0, -1.0)
    for group in range(dim // 32):
        first, second = 32 * group + 3, 32 * group + 17 + group
        rows[:, first], rows[:, second] = -sign * small, sign * large
    x = rows.double() * amplitude
    one = round_up(x[:, 3].abs()) == round_up(x[:, 17].abs())
    assert bool((x[:, 17].abs() > x[:, 3].abs()).all()) and 10 < int(one.sum()) < T
    got, x = append(rows, amplitude, interleaved)
    assert torch.equal(got, fmt.held(x))
    # The largest element is off by half a step, whichever its sign.
    s = fmt.quantise(x)[1][:, 0].abs()
    assert bool(((got - x)[:, 17].abs() <= s / 2).all())
    assert ops.take_status() == 0


def test_equal_extremes_keep_the_negative_one():
    rows = torch.rand(16, 64, generator=torch.Generator().manual_seed(1)) - 0.5
    rows[:, 5], rows[:, 11], rows[:, 40], rows[:, 50] = 1.75, -1.75, -1.5, 1.5
    got, x = append(rows, 0.3)
    assert torch.equal(got, fmt.held(x))
    assert bool((fmt.quantise(x)[1] > 0).all()) and ops.take_status() == 0


@pytest.mark.parametrize("below", [False, True])
def test_largest_elements_at_the_limits(below):
    # 2^120 and 2^-100, or 2^-40 of them less: as fp32 the same numbers.
    amplitude = 1.0 - 2.0 ** -40 if below else 1.0
    rows = torch.zeros(4, 64)
    rows[0, 3], rows[0, 40] = 2.0 ** -100, -2.0 ** -100
    rows[1, 3], rows[1, 4], rows[1, 40] = -2.0 ** -100, 2.0 ** -101, 2.0 ** -99
    rows[2, 3], rows[2, 40] = 1.0, -2.0
    got, x = append(rows, amplitude)
    assert torch.equal(got, fmt.held(x)) and ops.take_status() == 0
    assert bool((got[:2, :32] == 0).all()) == below
    rows[3, 3], rows[3, 40] = 2.0 ** 120, -3.0
    got, x = append(rows, amplitude)
    assert torch.equal(got, fmt.held(x))
    if below:
        assert ops.take_status() == 0 and float(got[3, 3]) == 2.0 ** 120
    else:
        with pytest.raises(RuntimeError, match="not finite or too large"):
            ops.take_status()
        assert bool((got[3, :32] == 0).all())

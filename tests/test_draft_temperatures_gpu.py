"""Draft verification at the smallest temperatures, bf16 logits among them: against the
definition in 64 bits, on the terms of test_drafts_gpu."""

import pytest
import torch

from batchstream_inference_engine_b200 import ops

from .test_drafts_gpu import call, check, make

pytestmark = pytest.mark.gpu

SMALLEST_NORMAL = 2.0 ** -126


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [1e-42, 1e-38, 1.2e-38, 1e-30, 1e-20, 1e-3])
def test_one_largest_logit_takes_all_the_weight(temperature, dtype):
    c = make([3] * 20, 997, dtype, seed=3, probs=False, temperature=temperature, near=0.2)
    c["logits"][:, 500] = 20.0
    c["draft_tokens"][::2] = 500
    tokens, accepted = call(c)
    assert ops.take_status() == 0
    for b in range(20):
        drafts = c["draft_tokens"][4 * b: 4 * b + 3].tolist()
        n = next((k for k, t in enumerate(drafts) if t != 500), 3)
        assert int(accepted[b]) == n
        assert tokens[4 * b: 4 * b + 4].tolist() == [500] * (n + 1) + [-1] * (3 - n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("unit", [2.0 ** -126, 2.0 ** -125, 2.0 ** -100, 2.0 ** -61, 2.0 ** -60, 1.0])
def test_logits_as_small_as_the_temperature(unit, probs, dtype):
    # Logits and temperature in units of a small number: the same distribution for all units.
    # (bf16 holds 8 bits: multiples of 1 / 8 below 16; 2^-129, the least step, is one.)
    g = torch.Generator().manual_seed(4)
    c = make([2] * 60, 50, seed=4, probs=probs, near=0.3)
    c["logits"] = (torch.randint(-64, 64, (180, 50), generator=g) / 8 * unit).to(dtype)
    if probs:
        c["draft_probs"] = torch.softmax(c["logits"].double() / unit / 1.1, -1).float()
        c["draft_tokens"] = torch.multinomial(c["draft_probs"], 1, generator=g)[:, 0].int()
    else:
        c["draft_tokens"] = c["logits"].argmax(-1).int()
    c["temperature"] = 1.5 * unit
    assert torch.equal(c["logits"].double() / unit * 8, (c["logits"].double() / unit * 8).round())
    taken = check(c)
    assert 0 < int(taken.sum()) < 120


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_temperatures_below_the_normal_numbers_take_the_largest_logit(dtype):
    # Ties too: the first of them, whatever the random numbers.
    c = make([2] * 9, 300, dtype, seed=5, probs=False)
    c["logits"][:, [7, 130, 299]] = 30.0
    c["draft_tokens"][:] = 7
    c["draft_tokens"][3::9] = 130
    c["uniforms"][:] = 0.9
    want = call({**c, "temperature": 0.0})
    assert set(want[1].tolist()) == {0, 2}
    for temperature in (1e-45, 1e-42, 1e-39, SMALLEST_NORMAL * (1 - 2.0 ** -23)):
        got = call({**c, "temperature": temperature})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        per = torch.full((9,), temperature)
        got = call({**c, "temperature": per})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = call({**c, "temperature": SMALLEST_NORMAL})  # drawn among the three
    assert got[0][got[0] >= 0].unique().tolist() != [7]
    assert ops.take_status() == 0

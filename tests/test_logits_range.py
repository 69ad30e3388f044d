"""The logit operators over the whole range of their arguments: temperatures
down to the smallest float beside biases and penalties, and logits up to the
largest float.  Oracles are the definitions in 64 bits."""

import math

import numpy as np
import pytest
import torch
from test_logits import DTYPES, U, check_pick, make, to_gpu


def stale():
    """Leaves numbers that no call gives in the memory that the next small outputs take."""
    junk = [torch.full((n,), 7_777_777, dtype=torch.int32, device="cuda") for n in (1, 16, 128) for _ in range(8)]
    torch.cuda.synchronize()
    del junk


# ---------------------------------------------------------------- pick

TEMPERATURES = [1e-45, 1e-30, 1e-12, 1e-10, 5e-10, 1e-9, 1e-8, 1e-6, 1e-3, 0.02, 1.0, 1e3, math.inf]


@pytest.mark.gpu
@pytest.mark.parametrize("rule", ["bias", "shared bias", "penalties", "both"])
@pytest.mark.parametrize("vocabulary", [300, 1025, 9000, 40_001])
def test_pick_at_any_temperature_under_rules(native_lib, vocabulary, rule):
    """Adjusted logits that are no floats: what is near the largest is settled in 64 bits."""
    rows = len(TEMPERATURES)
    for seed in range(4):
        s = make(seed + vocabulary, rows, vocabulary, torch.float32, 0 if "bias" in rule else 600, 0,
                 {"bias": "rows", "shared bias": "shared", "penalties": None, "both": "rows"}[rule])
        s["logits"][:, :256] -= 40.0  # the largest lies behind the first 256 symbols
        logits, rules = to_gpu(s)
        g = torch.Generator().manual_seed(seed)
        uniforms = torch.rand(rows, generator=g, dtype=torch.float64)
        if seed > 1:
            uniforms.fill_(1e-300 if seed == 2 else 0.999999)
        stale()
        check_pick(s, logits, rules, torch.tensor(TEMPERATURES).cuda(), uniforms.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_bias_that_forces_a_symbol(native_lib, dtype):
    """A bias beside which the logit it is added to is less than a float's step."""
    for vocabulary in (1024, 1025, 9000):
        s = make(vocabulary, 6, vocabulary, DTYPES[dtype], bias="rows")
        for i, force in enumerate((1e2, 1e5, 1e9, 1e20, 1e37, 3e38)):
            s["rules"]["bias"][i, 700:1020:40] = force
        logits, rules = to_gpu(s)
        uniforms = torch.full((6,), 0.5, dtype=torch.float64, device="cuda")
        for t in (0.0, 1e-9, 0.02, 1.0, 50.0):
            stale()
            check_pick(s, logits, rules, t, uniforms)


@pytest.mark.gpu
def test_a_weight_at_the_cut_off_is_written(native_lib):
    """A sum of logit and bias on the other side of e^-708 than its float: either answer, but an answer."""
    from leo_b200.logits import pick_symbols

    vocabulary, best, found = 9000, 1000, 0  # a block's part of the row, not a step's
    for k in range(64):
        heat = float(np.float32(1.0 + k / 64))
        edge = -65372.0 / (64 / math.log(2) / heat)
        e = float(np.float32(edge))
        b = float(np.float32(edge - e - 1e-7))  # the exact sum lies beyond the edge, its float before it
        if e <= edge or e + b >= edge or float(np.float32(e + b)) != e:
            continue
        found += 1
        logits = torch.full((1, vocabulary), -1e6)
        logits[0, 3], logits[0, best] = e, 0.0
        bias = torch.zeros(vocabulary)
        bias[3] = b
        stale()
        symbols, chance = pick_symbols(logits.cuda(), temperature=heat, bias=bias.cuda(),
                                       uniforms=torch.zeros(1, dtype=torch.float64, device="cuda"))
        symbol, chance = int(symbols[0]), float(chance[0])
        assert symbol in (3, best), symbol
        assert abs(chance - (0.0 if symbol == best else (e + b) / heat)) <= 1e-4
    assert found >= 8


# ---------------------------------------------------------------- loss

TOPS = [2.0**24, 2.0**27, 1e9, 2.0**30, 2.0**30 + 128, 1.5e9, 3e9, 5e9, 1e10, 1e20, 1e30, 9e36, 1e37, 1e38, 3e38]


def large_rows(vocabulary, dtype):
    """Rows whose largest logit has any magnitude: equal ones, one among small ones, neighbours."""
    rows = []
    for top in TOPS + [-t for t in TOPS]:
        value = torch.tensor(top, dtype=torch.float32).to(dtype)
        step = abs(float(value)) * torch.finfo(dtype).eps
        equal = torch.full((vocabulary,), float(value), dtype=torch.float64)
        rows.append(equal)
        near = equal - step * (torch.arange(vocabulary) % 5)
        rows.append(near)
        if top > 0:
            alone = torch.randn(vocabulary, generator=torch.Generator().manual_seed(1)).double()
            alone[vocabulary // 2] = float(value)
            rows.append(alone)
    return torch.stack(rows).clamp(-3.3e38, 3.3e38).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocabulary", [3, 257, 300, 1024, 5000, 70_001])
def test_loss_of_large_logits(native_lib, vocabulary, dtype):
    """Roundings: as at any size (test_logits), and a weight's exponent is rounded beside the
    rounding of top * log2(e), which is at most the distance of two floats there and so at most
    |z - top|, so 2 u |z - top| more; a weight below 2^-62 of the largest may be 0."""
    from leo_b200.logits import masked_cross_entropy

    x = large_rows(vocabulary, DTYPES[dtype])
    rows = x.shape[0]
    targets = torch.full((rows,), vocabulary // 2, dtype=torch.int32)
    losses, gradient = masked_cross_entropy(x.cuda(), targets.cuda())
    z = x.double()
    top = z.amax(1)
    far = (z - top[:, None]).abs()
    w = torch.exp(-far)
    total = w.sum(1)
    p = w / total[:, None]
    at = far[torch.arange(rows), targets.long()]
    want = torch.log(total) + at
    relative = (vocabulary / 32 + 28) * U + 3 * U * (far * w).sum(1) / total + vocabulary * 2.0**-62
    error = relative + 2 * U * (torch.log(total) + at)
    huge = want > 3.4e38  # the difference itself is no float any more
    assert bool(((losses.cpu().double() - want).abs() <= error + 2.0**-24 * want)[~huge].all())
    assert bool((losses.cpu()[huge] > 3.4e38).all())
    onehot = torch.nn.functional.one_hot(targets.long(), vocabulary).double()
    want = p - onehot
    error = p * (3 * far * U + 10 * U + relative[:, None]) + 2 * U * want.abs() + 2.0**-62
    eps = torch.finfo(gradient.dtype).eps
    off = (gradient.cpu().double() - want).abs() - error - eps / 2 * (want.abs() + error) * (1 + 2.0**-20)
    assert bool((off <= 0).all()), (float(off.max()), int(off.argmax()) // vocabulary)


@pytest.mark.gpu
def test_loss_of_a_row_of_a_mask_value(native_lib):
    """Finite values as masks are written: the symbols that have them are as likely as one another."""
    from leo_b200.logits import masked_cross_entropy

    for vocabulary in (257, 5000):
        for value in (-1e4, -1e9, -1e10, -1e30, float(torch.finfo(torch.bfloat16).min)):
            for dtype in (torch.float32, torch.bfloat16):
                x = torch.full((2, vocabulary), value, dtype=dtype, device="cuda")
                losses, gradient = masked_cross_entropy(x, torch.tensor([0, 7], dtype=torch.int32, device="cuda"))
                off = (losses.cpu().double() - math.log(vocabulary)).abs()
                assert bool((off <= (vocabulary / 32 + 40) * U).all()), (value, losses)
                # of a sum's and two more roundings, then the type's
                one = (gradient[0, 3:].cpu().double() * vocabulary - 1).abs().max()
                assert float(one) <= (vocabulary / 32 + 32) * U + torch.finfo(dtype).eps / 2 * 1.01, (value, one)

"""Penalties, biases and masks on logits, the pick of a symbol, and the masked
cross entropy, against their definitions in 64 bits.

Tolerances count roundings, u = 2^-24 being half a step of float32:
an adjusted logit passes at most five float32 roundings of values that its
parts bound; a softmax weight exp(z - top) is off by the rounding of z - top
(u |z - top|) and by four steps of an exponential, a sum of n of them by n / 32
additions in a row and a tree of 16; the last rounding to the output's type
adds finfo.eps / 2.  Symbols have to be equal.
"""

import ctypes as C
import math

import numpy as np
import pytest
import torch

U = 2.0**-24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(seed, rows, vocabulary, dtype, history=0, states=0, bias=None, pad=0):
    """Rules and logits on the CPU; rows `pad` elements apart."""
    g = torch.Generator().manual_seed(seed)
    wide = (4 * torch.randn(rows, vocabulary + pad, generator=g)).to(dtype)
    s = {"logits": wide[:, pad // 2:pad // 2 + vocabulary], "rules": {}}
    r = s["rules"]
    if history:
        r["history"] = torch.randint(-2, vocabulary + 3, (rows, history), generator=g, dtype=torch.int32)
        r["history"][:, ::2] = torch.randint(0, min(vocabulary, 9), r["history"][:, ::2].shape, generator=g)
        r["lengths"] = torch.randint(-1, history + 2, (rows,), generator=g, dtype=torch.int32)
        r["repetition"] = 0.8 + torch.rand(rows, generator=g)
        r["presence"] = torch.randn(rows, generator=g)
        r["frequency"] = torch.randn(rows, generator=g) / 4
    if bias:
        r["bias"] = torch.randn((vocabulary,) if bias == "shared" else (rows, vocabulary), generator=g)
        r["bias"][..., vocabulary // 2] = -math.inf
    if states:
        table = torch.rand(states, vocabulary, generator=g) < 0.5
        table[0] = False  # a state that allows nothing
        r["allowed"] = table
        r["state"] = torch.randint(-2, states + 1, (rows,), generator=g, dtype=torch.int32)
    return s


def mask_of(s):
    """[rows, vocabulary] booleans of what is allowed."""
    rows, vocabulary = s["logits"].shape
    table, state = s["rules"].get("allowed"), s["rules"].get("state")
    if table is None:
        return torch.ones(rows, vocabulary, dtype=torch.bool)
    if state is None:
        return table.expand(rows, vocabulary)
    ok = torch.zeros(rows, vocabulary, dtype=torch.bool)
    for i, k in enumerate(state.tolist()):
        if k == -1:
            ok[i] = True
        elif 0 <= k < len(table):
            ok[i] = table[k]
    return ok


def adjusted(s):
    """(adjusted logits, bound of the float32 error) in 64 bits, a symbol of the history at a time."""
    z = s["logits"].double().numpy().copy()
    rows, vocabulary = z.shape
    r = s["rules"]
    size = np.abs(z)
    if "history" in r:
        for i in range(rows):
            n = r["history"].shape[1]
            if "lengths" in r:
                n = max(0, min(n, int(r["lengths"][i])))
            spoken = [v for v in r["history"][i, :n].tolist() if 0 <= v < vocabulary]
            for v in set(spoken):
                c = spoken.count(v)
                rho, presence, frequency = (float(r[k][i]) if isinstance(r[k], torch.Tensor) else float(r[k])
                                            for k in ("repetition", "presence", "frequency"))
                z[i, v] = z[i, v] / rho if z[i, v] > 0 else z[i, v] * rho
                size[i, v] = abs(z[i, v]) + abs(presence) + c * abs(frequency)
                z[i, v] -= presence + frequency * c
    if "bias" in r:
        b = r["bias"].double().numpy()
        z = z + b
        size = size + np.abs(b)
    z, size = torch.from_numpy(z), torch.from_numpy(size)
    ok = mask_of(s)
    return torch.where(ok, z, -math.inf), torch.where(ok, 5 * U * size, 0.0)


def to_gpu(s, pad=0):
    """The rules as the calls take them."""
    from leo_b200.logits import pack_allowed

    r = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s["rules"].items()}
    if "allowed" in r:
        r["allowed"] = pack_allowed(r["allowed"])
    x = s["logits"]
    if pad:
        wide = torch.full((x.shape[0], x.shape[1] + pad), 77.0, dtype=x.dtype, device="cuda")
        wide[:, pad // 2:pad // 2 + x.shape[1]] = x.cuda()
        return wide[:, pad // 2:pad // 2 + x.shape[1]], r
    return x.cuda().contiguous(), r


def close(got, want, error, what):
    eps = torch.finfo(got.dtype).eps
    got = got.detach().cpu().double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    rest = ~finite & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest]), what
    tiny = 2.0**-24 if eps == 2.0**-10 else 2.0**-126
    off = ((got - want).abs() - error - eps / 2 * (want.abs() + error) * (1 + 2.0**-20) - tiny)[finite]
    assert bool((off <= 0).all()), (what, float(off.max()))


# ---------------------------------------------------------------- CPU


def test_pack_allowed():
    from leo_b200.logits import pack_allowed

    g = torch.Generator().manual_seed(0)
    for vocabulary in (1, 31, 32, 33, 257):
        table = torch.rand(5, vocabulary, generator=g) < 0.5
        words = pack_allowed(table)
        assert words.dtype == torch.int32 and words.shape == (5, (vocabulary + 31) // 32)
        for s in range(5):
            for v in range(vocabulary):
                assert bool((int(words[s, v // 32]) >> (v % 32)) & 1) == bool(table[s, v])
        assert all(int(w) & 0xFFFFFFFF < 1 << (vocabulary % 32 or 32) for w in words[:, -1])
    with pytest.raises(ValueError):
        pack_allowed(torch.zeros(3, 4))


def test_cpu_tensors_are_refused(native_lib):
    from leo_b200.logits import adjust_logits, masked_cross_entropy, pick_symbols

    x = torch.zeros(3, 5)
    for call in (lambda: adjust_logits(x), lambda: pick_symbols(x),
                 lambda: masked_cross_entropy(x, torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


BAD = {
    "vocabulary": dict(vocabulary=0),
    "dtype": dict(dtype=9),
    "null": dict(logits=None),
    "repetition": dict(repetition_value=0.0),
    "repetition nan": dict(repetition_value=math.nan),
    "presence": dict(presence_value=math.inf),
    "frequency": dict(frequency_value=math.nan),
    "states": dict(allowed=256, states=0),
    "rows of states": dict(allowed=256, states=2, allowed_stride=9),
    "mask stride": dict(allowed=256, states=3, allowed_stride=8),
    "negative stride": dict(stride=-1),
}


@pytest.mark.parametrize("bad", sorted(BAD))
def test_entry_points_refuse_before_device_work(native_lib, bad):
    from leo_b200.ctypes_types import LeoB200LogitRules

    b = dict(dtype=0, logits=256, stride=257, vocabulary=257, repetition_value=1.0, presence_value=0.0,
             frequency_value=0.0, allowed=None, states=0, allowed_stride=0)
    b.update(BAD[bad])
    rules = LeoB200LogitRules()
    for k in ("repetition_value", "presence_value", "frequency_value", "allowed", "states", "allowed_stride"):
        setattr(rules, k, b[k])
    head = (0, b["dtype"], b["logits"], b["stride"], 3, b["vocabulary"])
    calls = [native_lib.leo_b200_adjust_logits(*head, C.byref(rules), 256, 257, None),
             native_lib.leo_b200_pick_symbols(*head, C.byref(rules), None, 0.0, None, 256, 256, None)]
    if "_value" not in str(BAD[bad]):
        calls.append(native_lib.leo_b200_masked_cross_entropy(*head, 256, b["allowed"], b["allowed_stride"],
                                                              b["states"], None, None, 256, 256, 257, None))
    assert calls == [-1] * len(calls)
    assert native_lib.leo_b200_last_error()


def test_outputs_that_overlap_or_lack_are_refused(native_lib):
    from leo_b200.ctypes_types import LeoB200LogitRules

    rules = LeoB200LogitRules()
    rules.repetition_value = 1.0
    head = (0, 0, 256, 257, 3, 257)
    assert native_lib.leo_b200_adjust_logits(*head, C.byref(rules), 256, 256, None) == -1
    assert native_lib.leo_b200_adjust_logits(*head, C.byref(rules), None, 257, None) == -1
    assert native_lib.leo_b200_adjust_logits(*head, None, 256, 257, None) == -1
    assert native_lib.leo_b200_pick_symbols(*head, C.byref(rules), None, 0.0, None, None, None, None) == -1
    assert native_lib.leo_b200_pick_symbols(*head, C.byref(rules), None, -1.0, 256, 256, None, None) == -1
    assert native_lib.leo_b200_pick_symbols(*head, C.byref(rules), None, math.nan, 256, 256, None, None) == -1
    assert native_lib.leo_b200_pick_symbols(*head, C.byref(rules), None, 1.0, None, 256, None, None) == -1
    assert native_lib.leo_b200_pick_symbols(*head, C.byref(rules), 256, 0.0, None, 256, None, None) == -1
    assert native_lib.leo_b200_masked_cross_entropy(*head, None, None, 0, 0, None, None, 256, 256, 257, None) == -1
    assert native_lib.leo_b200_masked_cross_entropy(*head, 256, None, 0, 0, None, None, 256, 256, 256, None) == -1


# ---------------------------------------------------------------- GPU: adjust

CASES = [
    # rows, vocabulary, history, states, bias, pad
    (1, 1, 3, 0, None, 0),
    (3, 31, 0, 2, None, 0),
    (4, 257, 600, 5, "shared", 0),
    (5, 257, 40, 0, "rows", 3),
    (64, 260, 7, 3, "shared", 4),
    (2, 4096, 100, 3, None, 0),
    (3, 4097, 5000, 2, "rows", 1),
    (2, 40_001, 300, 3, "shared", 8),
    (1, 131_072, 64, 2, "rows", 0),
]
IDS = [f"{c[0]}x{c[1]}" for c in CASES]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_adjust(native_lib, case, dtype):
    from leo_b200.logits import adjust_logits

    rows, vocabulary, history, states, bias, pad = case
    s = make(rows + vocabulary, rows, vocabulary, DTYPES[dtype], history, states, bias)
    logits, rules = to_gpu(s, pad)
    before = logits.clone()
    want, error = adjusted(s)
    got = adjust_logits(logits, **rules)
    close(got, want, error, "adjusted")
    assert torch.equal(logits, before)
    wide = torch.full((rows, vocabulary + 5), 5.0, dtype=DTYPES[dtype], device="cuda")
    again = adjust_logits(logits, out=wide[:, 2:vocabulary + 2], **rules)
    assert torch.equal(again, got) and bool((wide[:, :2] == 5).all()) and bool((wide[:, vocabulary + 2:] == 5).all())
    inside = adjust_logits(logits, out=logits, **rules)  # in place
    assert inside is logits and torch.equal(logits, got)
    if pad:
        edge = logits.as_strided((rows, 1), (logits.stride(0), 1), logits.storage_offset() + vocabulary)
        if pad > 1:
            assert bool((edge == 77).all())


@pytest.mark.gpu
def test_numbers_and_plain_copies(native_lib):
    """Rules as numbers, and none at all."""
    from leo_b200.logits import adjust_logits

    s = make(3, 7, 300, torch.float32, history=50)
    s["rules"].update(repetition=1.3, presence=0.25, frequency=-0.5)
    del s["rules"]["lengths"]
    logits, rules = to_gpu(s)
    want, error = adjusted(s)
    close(adjust_logits(logits, **rules), want, error, "numbers")
    assert torch.equal(adjust_logits(logits), logits)
    empty = adjust_logits(logits[:0])
    assert empty.shape == (0, 300)


@pytest.mark.gpu
def test_masked_places_never_matter(native_lib):
    from leo_b200.logits import adjust_logits, masked_cross_entropy, pick_symbols

    s = make(5, 6, 700, torch.float32, states=4)
    s["rules"]["state"] = torch.tensor([1, 2, 3, 1, 2, 3], dtype=torch.int32)
    ok = mask_of(s).cuda()
    clean, rules = to_gpu(s)
    targets = ok.int().argmax(1).to(torch.int32)
    want = (adjust_logits(clean, **rules), *pick_symbols(clean, **rules),
            *masked_cross_entropy(clean, targets, **rules))
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).max, torch.finfo(torch.float32).min):
        x = torch.where(ok, clean, bad)
        got = (adjust_logits(x, **rules), *pick_symbols(x, **rules), *masked_cross_entropy(x, targets, **rules))
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- GPU: pick


def picked(s, temperature, uniforms):
    z, _ = adjusted(s)
    symbols, chances = [], []
    for i in range(z.shape[0]):
        row, t = z[i], float(temperature[i])
        if bool(torch.isnan(row).any()) or not t >= 0:
            symbols.append(-1)
            chances.append(math.nan)
            continue
        top = float(row.max())
        if top == -math.inf:
            symbols.append(-1)
            chances.append(-math.inf)
            continue
        heat = t if t else 1.0
        w = torch.where(row == top, 1.0, torch.exp((row - top) / heat))
        w = torch.where(row == -math.inf, 0.0, w)
        sums = torch.cumsum(w, 0)
        if t:
            over = torch.nonzero(sums > float(uniforms[i]) * float(sums[-1]))
            v = int(over[0, 0]) if len(over) else int(torch.nonzero(w > 0)[-1, 0])
        else:
            v = int(torch.nonzero(row == top)[0, 0])
        symbols.append(v)
        chances.append(math.log(float(w[v])) - math.log(float(sums[-1])))
    return torch.tensor(symbols, dtype=torch.int32), torch.tensor(chances, dtype=torch.float64)


def check_pick(s, logits, rules, temperature, uniforms):
    from leo_b200.logits import pick_symbols

    symbols, chance = pick_symbols(logits, temperature=temperature, uniforms=uniforms, **rules)
    t = temperature.cpu() if isinstance(temperature, torch.Tensor) else torch.full((logits.shape[0],), temperature)
    want, want_chance = picked(s, t, uniforms.cpu() if uniforms is not None else None)
    assert symbols.dtype == torch.int32 and symbols.cpu().tolist() == want.tolist()
    close(chance, want_chance, 1e-10, "log probability")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_pick(native_lib, case, dtype):
    rows, vocabulary, history, states, bias, pad = case
    s = make(7 * rows + vocabulary, rows, vocabulary, DTYPES[dtype], history, states, bias)
    logits, rules = to_gpu(s, pad)
    g = torch.Generator().manual_seed(rows)
    uniforms = torch.rand(rows, generator=g, dtype=torch.float64).cuda()
    check_pick(s, logits, rules, 0.0, None)
    check_pick(s, logits, rules, 1.7, uniforms)
    temperature = torch.rand(rows, generator=g)
    temperature[::3] = 0.0
    check_pick(s, logits, rules, temperature.cuda(), uniforms)


@pytest.mark.gpu
@pytest.mark.parametrize("vocabulary", [2, 257, 9000])
def test_pick_at_the_edges(native_lib, vocabulary):
    """Equal logits, uniforms at both ends, infinities, NaN, rows without anything."""
    from leo_b200.logits import pick_symbols

    rows = 12
    x = torch.zeros(rows, vocabulary)
    x[1:, 0] = -math.inf
    x[2] = -math.inf  # nothing
    x[3, 1] = math.nan
    x[4, 1] = math.inf  # one certain symbol
    x[5] = math.inf  # all of them
    x[6] = -3e38
    x[7, 1] = 3e38
    x[8] = -math.inf
    x[8, vocabulary - 1] = -80.0
    temperature = torch.tensor([0, 0, 0, 0, 0, 1, 1, 1, 1, -1, math.nan, math.inf])
    s = {"logits": x, "rules": {}}
    for u in (0.0, 0.5, 1.0 - 2.0**-53):
        uniforms = torch.full((rows,), u, dtype=torch.float64, device="cuda")
        for t in (temperature, torch.where(temperature == 0, 0.7, temperature)):
            check_pick(s, x.cuda(), {}, t.cuda(), uniforms)
    assert pick_symbols(x.cuda()[:0])[0].shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("vocabulary", [70, 900, 9000])
def test_pick_at_any_temperature(native_lib, vocabulary):
    """From the smallest float to infinity, where every symbol that is left is as likely."""
    g = torch.Generator().manual_seed(vocabulary)
    temperature = torch.tensor([1e-45, 1e-30, 1e-3, 1e3, 1e30, 3e38, math.inf, math.inf])
    x = torch.randn(8, vocabulary, generator=g)
    x[:, ::3] = -math.inf
    x[7] = -math.inf
    x[7, 5::7] = torch.randn(x[7, 5::7].shape, generator=g)
    uniforms = torch.rand(8, generator=g, dtype=torch.float64)
    check_pick({"logits": x, "rules": {}}, x.cuda(), {}, temperature.cuda(), uniforms.cuda())


@pytest.mark.gpu
def test_draws_follow_the_distribution(native_lib):
    """Evenly spread uniforms hit every symbol as often as its probability says, to one draw."""
    from leo_b200.logits import pick_symbols

    n, vocabulary = 4000, 37
    g = torch.Generator().manual_seed(4)
    row = torch.randn(1, vocabulary, generator=g)
    uniforms = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    symbols, _ = pick_symbols(row.expand(n, vocabulary).cuda(), temperature=0.8, uniforms=uniforms.cuda())
    count = torch.bincount(symbols.cpu().long(), minlength=vocabulary)
    p = torch.softmax(row[0].double() / float(np.float32(0.8)), 0)
    assert float((count - n * p).abs().max()) <= 1.0
    assert bool((symbols.diff() >= 0).all())


# ---------------------------------------------------------------- GPU: loss


def check_loss(s, logits, rules, targets, weights):
    from leo_b200.logits import masked_cross_entropy

    losses, gradient = masked_cross_entropy(logits, targets.cuda(), weights=None if weights is None else weights.cuda(),
                                            allowed=rules.get("allowed"), state=rules.get("state"))
    rows, vocabulary = s["logits"].shape
    z = torch.where(mask_of(s), s["logits"].double(), -math.inf)
    at = targets.long().clamp(0, vocabulary - 1)
    top = z.amax(1)
    z_at = z[torch.arange(rows), at]
    w = torch.exp(z - top[:, None])
    total = w.sum(1)
    want = torch.log(total) + (top - z_at)  # the difference first: log(total) would vanish beside a huge top
    empty = top == -math.inf
    want = torch.where((z_at == -math.inf) | empty, math.inf, want)
    p = w / total[:, None]
    onehot = torch.zeros_like(p)
    onehot[torch.arange(rows), at] = (z_at > -math.inf).double()
    scale = torch.ones(rows) if weights is None else weights
    grad = scale.double()[:, None] * (p - onehot)
    outside = targets >= vocabulary
    quiet = (targets < 0) | empty | outside
    grad = torch.where(quiet[:, None] | ~mask_of(s), 0.0, grad)
    want = torch.where(targets < 0, 0.0, torch.where(outside, math.nan, want))
    sums = (vocabulary / 32 + 16 + 8) * U
    far = torch.where(z == -math.inf, 0.0, z - top[:, None]).abs()
    relative = sums + ((far * w).nan_to_num().sum(1) / total).nan_to_num() * U + 4 * U
    loss_error = relative + 2 * U * (torch.log(total).abs() + (top - z_at).abs()).nan_to_num(0, 0, 0)
    close(losses, want, torch.where(torch.isfinite(want), loss_error, 0.0), "losses")
    grad_error = scale.double().abs()[:, None] * (p * (far * U + 10 * U + relative[:, None]) + 2 * U * (p - onehot).abs())
    close(gradient, grad, grad_error.nan_to_num(0.0), "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocabulary,states,pad", [
    (1, 1, 0, 0), (5, 2, 3, 0), (33, 31, 2, 1), (64, 257, 6, 0), (70, 257, 0, 3), (1000, 257, 4, 0), (9, 512, 3, 0),
    (9, 513, 0, 0), (7, 1023, 3, 1), (6, 1025, 2, 0), (5, 4100, 3, 0), (3, 33_001, 0, 8), (2, 131_072, 3, 0)])
def test_loss(native_lib, rows, vocabulary, states, pad, dtype):
    s = make(rows * vocabulary, rows, vocabulary, DTYPES[dtype], states=states)
    logits, rules = to_gpu(s, pad)
    g = torch.Generator().manual_seed(vocabulary)
    targets = torch.randint(-1, vocabulary + 1, (rows,), generator=g, dtype=torch.int32)
    weights = 2 * torch.randn(rows, generator=g)
    check_loss(s, logits, rules, targets, weights)
    check_loss(s, logits, rules, targets.clamp(0, vocabulary - 1), None)


@pytest.mark.gpu
@pytest.mark.parametrize("vocabulary", [1, 32, 255, 256, 257, 288, 289, 512, 513, 1024, 1025, 8192, 8193])
def test_loss_at_every_width(native_lib, vocabulary):
    """Both sides of every border between forms of the kernel."""
    s = make(vocabulary, 11, vocabulary, torch.float32, 0, 3, None)
    logits, rules = to_gpu(s, 2)
    g = torch.Generator().manual_seed(vocabulary)
    targets = torch.randint(-1, vocabulary, (11,), generator=g, dtype=torch.int32)
    targets[0], targets[1] = vocabulary - 1, vocabulary
    check_loss(s, logits, rules, targets, torch.rand(11, generator=g))


@pytest.mark.gpu
def test_loss_of_odd_rows(native_lib):
    """-inf logits, a certain symbol, huge and equal logits, a NaN where it counts."""
    from leo_b200.logits import masked_cross_entropy

    for vocabulary in (3, 257, 5000):
        x = torch.randn(6, vocabulary, generator=torch.Generator().manual_seed(1))
        x[0] = -math.inf
        x[1] = -math.inf
        x[1, 1] = 2.0
        x[2] = 3e38
        x[3] = -3e38
        x[4, 0] = 100.0
        s = {"logits": x, "rules": {}}
        check_loss(s, x.cuda(), {}, torch.tensor([0, 1, 2, 1, 0, 2], dtype=torch.int32), None)
        x[5, 2] = math.nan
        losses, gradient = masked_cross_entropy(x.cuda(), torch.full((6,), 1, dtype=torch.int32, device="cuda"))
        assert bool(losses[5].isnan()) and bool(gradient[5].isnan().any()) and not bool(gradient[:5].isnan().any())
    losses, gradient = masked_cross_entropy(x.cuda()[:0], torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert losses.shape == (0,) and gradient.shape == (0, 5000)


@pytest.mark.gpu
def test_loss_gradient_matches_differences(native_lib):
    """The gradient along a direction against the loss's central difference in 64 bits."""
    from leo_b200.logits import masked_cross_entropy, pack_allowed

    rows, vocabulary = 8, 257
    g = torch.Generator().manual_seed(2)
    x = torch.randn(rows, vocabulary, generator=g)
    ok = torch.rand(1, vocabulary, generator=g) < 0.6
    ok[:, :rows] = True
    targets = torch.arange(rows, dtype=torch.int32)
    weights = torch.rand(rows, generator=g)
    _, gradient = masked_cross_entropy(x.cuda(), targets.cuda(), allowed=pack_allowed(ok).cuda(), weights=weights.cuda())
    v = torch.randn(rows, vocabulary, generator=g, dtype=torch.float64)

    def value(z):
        z = torch.where(ok, z, -math.inf)
        return float((weights.double() * (torch.logsumexp(z, 1) - z[torch.arange(rows), targets.long()])).sum())

    slope = (value(x.double() + 1e-6 * v) - value(x.double() - 1e-6 * v)) / 2e-6
    mine = float((gradient.cpu().double() * v).sum())
    # every element is within 100 half steps of its parts, the difference within 1e-8
    tolerance = 100 * U * float((weights.double()[:, None] * v.abs()).sum()) + 1e-8
    assert abs(mine - slope) <= tolerance


# ---------------------------------------------------------------- GPU: calls


@pytest.mark.gpu
def test_captured_and_replayed(native_lib):
    from leo_b200.logits import adjust_logits, masked_cross_entropy, pick_symbols

    s = make(1, 20, 257, torch.bfloat16, history=30, states=4, bias="shared")
    logits, rules = to_gpu(s)
    targets = torch.randint(0, 257, (20,), dtype=torch.int32, device="cuda")
    uniforms = torch.rand(20, dtype=torch.float64, device="cuda")
    mask = {k: rules[k] for k in ("allowed", "state")}

    def everything():
        return (adjust_logits(logits, **rules), *pick_symbols(logits, temperature=0.9, uniforms=uniforms, **rules),
                *masked_cross_entropy(logits, targets, **mask))

    everything()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = everything()
    for seed in range(3):
        logits.copy_(torch.randn(20, 257, generator=torch.Generator().manual_seed(seed)))
        uniforms.uniform_()
        graph.replay()
        want = everything()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.gpu
def test_other_streams(native_lib):
    from leo_b200.logits import adjust_logits, masked_cross_entropy, pick_symbols

    s = make(2, 50, 9001, torch.float32, history=30, states=4, bias="rows")
    logits, rules = to_gpu(s)
    targets = torch.zeros(50, dtype=torch.int32, device="cuda")
    mask = {k: rules[k] for k in ("allowed", "state")}
    torch.cuda.synchronize()
    want = (adjust_logits(logits, **rules), *pick_symbols(logits, **rules), *masked_cross_entropy(logits, targets, **mask))
    torch.cuda.synchronize()
    for stream in [torch.cuda.Stream() for _ in range(3)]:
        got = (adjust_logits(logits, stream=stream, **rules), *pick_symbols(logits, stream=stream, **rules),
               *masked_cross_entropy(logits, targets, stream=stream, **mask))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.gpu
def test_refusals(native_lib):
    from leo_b200.logits import adjust_logits, masked_cross_entropy, pick_symbols
    from leo_b200.native import LeoError

    x = torch.zeros(4, 40, device="cuda")
    ints = torch.zeros(4, 6, dtype=torch.int32, device="cuda")
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    rows = torch.zeros(4, dtype=torch.int32, device="cuda")
    floats = torch.ones(4, device="cuda")

    def refused(call, match):
        with pytest.raises((ValueError, LeoError), match=match):
            call()

    refused(lambda: adjust_logits(x.double()), "float32, bfloat16 or float16")
    refused(lambda: adjust_logits(x[0]), "two dimensions")
    refused(lambda: adjust_logits(x[:, :0]), "at least one symbol")
    refused(lambda: adjust_logits(x.t()), "adjacent")
    refused(lambda: adjust_logits(x, history=ints.long()), "history must be")
    refused(lambda: adjust_logits(x, history=ints[:3]), "history must have 4 rows")
    refused(lambda: adjust_logits(x, lengths=rows), "needs a history")
    refused(lambda: adjust_logits(x, history=ints, lengths=rows[:3]), "lengths must have shape")
    refused(lambda: adjust_logits(x, history=ints, repetition=0.0), "positive and finite")
    refused(lambda: adjust_logits(x, history=ints, repetition=floats[:2]), "repetition must have shape")
    refused(lambda: adjust_logits(x, history=ints, presence=floats.double()), "presence must be")
    refused(lambda: adjust_logits(x, frequency=math.nan), "finite")
    refused(lambda: adjust_logits(x, bias=x[:3]), "bias must have shape")
    refused(lambda: adjust_logits(x, bias=x[0, :39]), "adjacent elements")
    refused(lambda: adjust_logits(x, bias=x.bfloat16()), "bias must be")
    refused(lambda: adjust_logits(x, allowed=table[:, :1]), "2 words")
    refused(lambda: adjust_logits(x, allowed=table), "1 or 4 rows")
    refused(lambda: adjust_logits(x, allowed=table[:0], state=rows), "at least one state")
    refused(lambda: adjust_logits(x, allowed=table.bool(), state=rows), "allowed must be")
    refused(lambda: adjust_logits(x, state=rows), "needs a mask table")
    refused(lambda: adjust_logits(x, allowed=table, state=rows.long()), "state must be")
    refused(lambda: adjust_logits(x, allowed=table.cpu(), state=rows), "CUDA tensor")
    refused(lambda: adjust_logits(x, out=x[:3]), "out must have shape")
    refused(lambda: adjust_logits(x, out=x[:1].expand(4, 40)), "overlap")
    refused(lambda: adjust_logits(x.clone().requires_grad_()), "detach")
    refused(lambda: pick_symbols(x, temperature=1.0), "needs uniforms")
    refused(lambda: pick_symbols(x, temperature=-1.0), "not be negative")
    refused(lambda: pick_symbols(x, temperature=1.0, uniforms=floats), "uniforms must be")
    refused(lambda: masked_cross_entropy(x, rows.long()), "targets must be")
    refused(lambda: masked_cross_entropy(x, rows[:2]), "targets must have shape")
    refused(lambda: masked_cross_entropy(x, rows, weights=floats[:2]), "weights must have shape")
    refused(lambda: masked_cross_entropy(x, rows, allowed=table), "1 or 4 rows")

"""The operators in use: a recurrent readout trained over packed stories (scan,
masked loss, their gradients) and served a byte at a time (step, pick), and
the backend's own pick of the next symbol.

The tolerance of the training step counts, in float32 half steps u = 2^-24 of
the norm: 64 for a product over 32 channels and its sums, 3 / (1 - 0.95) = 60
for a scan with gates up to 0.95, 2 x 10 x (64 + 60) for what an error of logits
up to 10 does to a softmax, 50 for the loss's sums, 257 for the product over
the classes on the way back, 60 for the scan back: 2000 in all.
"""

import numpy as np
import pytest
import torch

U = 2.0**-24
LENGTHS = [37, 0, 150, 1, 300]
WIDTH, CLASSES = 32, 257


def offsets():
    return [0] + np.cumsum(LENGTHS).tolist()


def make():
    g = torch.Generator().manual_seed(7)
    tokens = sum(LENGTHS)
    return {"byte": torch.randint(0, 256, (tokens,), generator=g),
            "embedding": torch.randn(256, WIDTH, generator=g),
            "readout": torch.randn(CLASSES, WIDTH, generator=g) / 4,
            "decay": 0.95 * torch.rand(tokens, WIDTH, generator=g),
            "initial": torch.randn(len(LENGTHS), WIDTH, generator=g),
            "target": torch.randint(0, 128, (tokens,), generator=g, dtype=torch.int32),
            # two grammar states: ASCII, and everything but control bytes
            "table": torch.stack([torch.arange(CLASSES) < 128,
                                  (torch.arange(CLASSES) >= 32) | (torch.arange(CLASSES) < 128)]),
            "state": torch.randint(-1, 2, (tokens,), generator=g, dtype=torch.int32),
            "weight": 0.5 + torch.rand(tokens, generator=g)}


def reference(m):
    """Losses and gradients in 64 bits by autograd, a token at a time."""
    leaf = {k: m[k].double().requires_grad_() for k in ("embedding", "readout", "decay", "initial")}
    states = []
    for s, begin in enumerate(offsets()[:-1]):
        h = leaf["initial"][s]
        for t in range(begin, begin + LENGTHS[s]):
            h = leaf["decay"][t] * h + leaf["embedding"][m["byte"][t]]
            states.append(h)
    logits = torch.stack(states) @ leaf["readout"].T
    ok = torch.where((m["state"] < 0)[:, None], True, m["table"][m["state"].clamp(min=0).long()])
    z = torch.where(ok, logits, -torch.inf)
    losses = torch.logsumexp(z, 1) - logits.gather(1, m["target"].long()[:, None])[:, 0]
    (losses * m["weight"].double()).sum().backward()
    return losses.detach(), {k: v.grad for k, v in leaf.items()}


@pytest.mark.gpu
def test_a_readout_is_trained(native_lib):
    from leo_b200.gated_scan import StoryLayout, gated_scan, gated_scan_backward
    from leo_b200.logits import masked_cross_entropy, pack_allowed

    m = make()
    want, want_grad = reference(m)
    d = {k: v.cuda() for k, v in m.items()}
    layout = StoryLayout(offsets(), "cuda:0")
    scan = gated_scan(d["embedding"][d["byte"]], d["decay"], layout, d["initial"], keep_carries=True)
    with torch.no_grad():  # float32 products are float32 by default
        logits = scan.states @ d["readout"].T
        losses, slope = masked_cross_entropy(logits, d["target"], allowed=pack_allowed(d["table"]), state=d["state"],
                                             weights=d["weight"])
        grad = gated_scan_backward(slope @ d["readout"], d["embedding"][d["byte"]], d["decay"], layout, scan.carries,
                                   initial=d["initial"])
        got = {"readout": slope.T @ scan.states, "decay": grad.decay, "initial": grad.initial,
               "embedding": torch.zeros_like(d["embedding"]).index_add_(0, d["byte"], grad.drive)}
    assert float((losses.cpu().double() - want).norm() / want.norm()) <= 2000 * U
    for name, g in want_grad.items():
        off = float((got[name].cpu().double() - g).norm() / g.norm())
        assert off <= 2000 * U, (name, off)


@pytest.mark.gpu
def test_the_readout_is_served_a_byte_at_a_time(native_lib):
    """Lanes that step through their stories reach the scan's states and pick what its logits say."""
    from leo_b200.gated_scan import StoryLayout, gated_scan, gated_step
    from leo_b200.logits import adjust_logits, pack_allowed, pick_symbols

    m = make()
    d = {k: v.cuda() for k, v in m.items()}
    lanes, tokens = 6, 40
    byte, decay = d["byte"][: lanes * tokens], d["decay"][: lanes * tokens]
    drive = d["embedding"][byte]
    start = torch.randn(lanes, WIDTH, device="cuda")
    scan = gated_scan(drive, decay, StoryLayout([i * tokens for i in range(lanes + 1)], "cuda:0"), start)
    state = start.clone()
    table = pack_allowed(d["table"])
    grammar = torch.arange(lanes, dtype=torch.int32, device="cuda") % 3 - 1
    history = byte.view(lanes, tokens).to(torch.int32)
    for t in range(tokens):
        out = gated_step(drive.view(lanes, tokens, WIDTH)[:, t], decay.view(lanes, tokens, WIDTH)[:, t], state)
        logits = out @ d["readout"].T
        rules = {"allowed": table, "state": grammar, "history": history, "presence": 0.75, "repetition": 1.5,
                 "lengths": torch.full((lanes,), t, dtype=torch.int32, device="cuda")}
        symbols, chance = pick_symbols(logits, **rules)
        adjusted = adjust_logits(logits, **rules)
        # two roundings of the adjusted logits at most lie between the pick's 64 bits and these
        top = adjusted.amax(1)
        mine = adjusted.gather(1, symbols.long()[:, None])[:, 0]
        assert bool((top - mine <= 4 * U * (top.abs() + 8.0)).all())
        assert bool((chance <= 0).all()) and bool((symbols >= 0).all())
    # 3 roundings a token of values that the gates keep below 20 x the largest drive
    bound = 3 * 20 * U * float(drive.abs().max() + start.abs().max()) * 20
    assert float((state - scan.final).abs().max()) <= bound
    assert float((scan.states.view(lanes, tokens, WIDTH)[:, -1] - scan.final).abs().max()) == 0.0


@pytest.mark.gpu
def test_backend_picks_the_next_symbol(native_lib):
    from leo_b200.backend import GpuBackend
    from leo_b200.configs import WORKLOADS
    from leo_b200.ctypes_types import BEGIN_DOCUMENT, END_DOCUMENT, TRAINING
    from leo_b200.model import HostModel
    from leo_b200.native import LeoError
    from leo_b200.synthetic import story_stream

    wl = WORKLOADS["test"]
    with GpuBackend(HostModel.initialize(wl.config, wl.topology), device=0, max_lanes=4) as gpu:
        gpu.train_story_batch(story_stream(1, 4, 16, 48), TRAINING)
        digest, statistics = gpu.state_digest(), bytes(gpu.synchronize_model().statistics)

        def probabilities():
            return gpu.lane_array(gpu.CANONICAL_LANE, "probabilities", capacity=4 * 257)

        def document(steps, **rules):
            gpu.begin_document()
            gpu.advance_frozen_batch([(BEGIN_DOCUMENT, None)] + [(b, None) for b in b"once "])
            symbol, said = ord("u"), []
            for _ in range(steps):
                symbol, chance = gpu.next_symbol(symbol, **rules)
                said.append((symbol, chance))
                if symbol == END_DOCUMENT:
                    break
            return said

        tick = gpu.canonical_tick
        first = document(12)
        gpu.canonical_tick = tick
        assert document(12) == first  # nothing was learned, and nothing is left of the pick
        gpu.canonical_tick = tick
        document(1)
        p = probabilities().astype(np.float64)
        assert first[0][0] in (int(p.argmax()), END_DOCUMENT) and abs(np.exp(first[0][1]) - p.max()) <= 1e-5
        # a mask, a bias that forces a symbol, and one drawn at the end of the distribution
        gpu.canonical_tick = tick
        assert document(1, allowed=[c == 65 for c in range(257)])[0] == (65, 0.0)
        gpu.canonical_tick = tick
        force = np.zeros(257, np.float32)
        force[256] = 1e4
        assert document(3, bias=force)[0][0] == END_DOCUMENT
        gpu.canonical_tick = tick
        greedy = document(1)[0][0]
        gpu.canonical_tick = tick
        other = document(1, history=[greedy, greedy], presence=50.0)[0][0]
        assert other != greedy
        gpu.canonical_tick = tick
        drawn = document(1, temperature=1.0, uniform=1.0 - 2.0**-53)[0][0]
        assert drawn == END_DOCUMENT or p[drawn] > 0
        with pytest.raises(LeoError, match="no symbol is left"):
            gpu.next_symbol(65, allowed=[False] * 257)
        before = gpu.lane_array(gpu.CANONICAL_LANE, "probabilities", capacity=4 * 257).copy()
        for refused in ({"temperature": -1.0}, {"repetition": 0.0}, {"presence": float("nan")}):
            with pytest.raises(ValueError, match="must"):
                gpu.next_symbol(66, **refused)  # no step is taken
        assert np.array_equal(before, gpu.lane_array(gpu.CANONICAL_LANE, "probabilities", capacity=4 * 257))
        with pytest.raises(ValueError, match="uniform"):
            gpu.next_symbol(65, uniform=1.0)
        with pytest.raises(ValueError, match="257 entries"):
            gpu.next_symbol(65, bias=[0.0])
        assert gpu.state_digest() == digest
        assert bytes(gpu.synchronize_model().statistics) == statistics


REFUSED = [{"repetition": 1e-50}, {"repetition": 1e300}, {"presence": 1e300}, {"presence": -1e39}, {"frequency": 1e39},
           {"frequency": float("inf")}, {"bias": np.zeros((257, 1))}, {"bias": [0.0] * 256}, {"bias": 1.0},
           {"allowed": np.ones((257, 2), bool)}, {"temperature": float("nan")}, {"uniform": float("nan")}]


@pytest.mark.parametrize("arguments", REFUSED, ids=[next(iter(r)) for r in REFUSED])
def test_next_symbol_refuses_before_the_step(arguments):
    """What 32 bits make 0 or infinite, and what has another shape, is refused while the document stands."""
    from leo_b200.backend import GpuBackend

    class Standing:
        device, CANONICAL_LANE = 0, 0

        def training_step_batch(self, *_):
            pytest.fail("the step was taken")

    with pytest.raises(ValueError):
        GpuBackend.next_symbol(Standing(), 65, **arguments)


@pytest.mark.gpu
def test_the_greedy_pick_is_the_most_likely_class(native_lib):
    """Without rules next_symbol gives the arg-max of the step's probabilities, the end only where it is that."""
    from leo_b200.backend import GpuBackend
    from leo_b200.configs import WORKLOADS
    from leo_b200.ctypes_types import BEGIN_DOCUMENT, END_DOCUMENT, TRAINING
    from leo_b200.model import HostModel
    from leo_b200.synthetic import story_stream

    wl = WORKLOADS["test"]
    with GpuBackend(HostModel.initialize(wl.config, wl.topology), device=0, max_lanes=4) as gpu:
        gpu.train_story_batch(story_stream(1, 4, 16, 48), TRAINING)
        gpu.begin_document()
        gpu.advance_frozen_batch([(BEGIN_DOCUMENT, None)])
        for byte in b"once upon a time, ":
            symbol, chance = gpu.next_symbol(byte)
            p = gpu.lane_array(gpu.CANONICAL_LANE, "probabilities", capacity=4 * 257).astype(np.float64)
            # the logarithms are floats: classes a rounding of theirs apart may be taken for equal
            taken = 256 if symbol == END_DOCUMENT else symbol
            assert np.log(p[taken]) >= np.log(p.max()) * (1 + 2 * U)
            assert abs(chance - np.log(p[taken] / p.sum())) <= 1e-5

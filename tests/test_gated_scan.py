"""The gated recurrence over packed stories, its gradients and its one-token step.

The oracle is the recurrence itself in 64 bits, token by token.  Tolerances
count roundings: with u = 2^-24, a state that is formed from at most three
float32 roundings a token (of the running state, of a product of gates, of a
partial state) is off by at most E, E[t] = |a[t]| E[t-1] + 3 u B[t], where B is
the recurrence of the absolute values; the last rounding to the output's type
adds half a step, finfo.eps / 2, of the value.
"""

import ctypes as C

import numpy as np
import pytest
import torch

U = 2.0**-24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def offsets_of(lengths):
    return [0] + np.cumsum(lengths).tolist()


def make(seed, lengths, channels, dtype, decay, initial=True, device="cpu"):
    """Inputs in their own types; gates around the configurations' decays."""
    g = torch.Generator().manual_seed(seed)
    tokens, stories = sum(lengths), len(lengths)
    base = torch.tensor([0.0, 0.5, 0.85, 0.97, 0.999, 1.0, -0.9])[torch.randint(7, (channels,), generator=g)]
    if decay == "channel":
        a = base
    else:
        a = (base * (0.9 + 0.1 * torch.rand(tokens, channels, generator=g)))
        a = a.to(torch.float32 if decay == "f32" else dtype)
    s = {"x": torch.randn(tokens, channels, generator=g).to(dtype), "a": a,
         "g": torch.randn(tokens, channels, generator=g).to(dtype),
         "h0": torch.randn(stories, channels, generator=g) if initial else None,
         "gf": torch.randn(stories, channels, generator=g)}
    return {k: v.to(device) if v is not None else None for k, v in s.items()}


def oracle(lengths, x, a, g=None, h0=None, gf=None):
    """States, gradients and their error bounds (before the last rounding), in 64 bits on the CPU."""
    f = lambda v: None if v is None else v.detach().cpu().double()  # noqa: E731
    x, a, g, h0, gf = f(x), f(a), f(g), f(h0), f(gf)
    tokens, channels = x.shape
    full = a.expand(tokens, channels)
    out = {k: torch.zeros(tokens, channels, dtype=torch.float64) for k in ("h", "eh", "dx", "edx", "da", "eda")}
    stories = len(lengths)
    zero = torch.zeros(channels, dtype=torch.float64)
    out |= {k: torch.zeros(stories, channels, dtype=torch.float64) for k in ("final", "efinal", "dh0", "edh0")}
    for s, begin in enumerate(offsets_of(lengths)[:-1]):
        h = h0[s] if h0 is not None else zero
        b, e = h.abs(), zero
        previous = []
        for t in range(begin, begin + lengths[s]):
            previous.append((h, e))
            h, b = full[t] * h + x[t], full[t].abs() * b + x[t].abs()
            e = full[t].abs() * e + 3 * U * b
            out["h"][t], out["eh"][t] = h, e
        out["final"][s], out["efinal"][s] = h, e
        if g is None:
            continue
        m = gf[s] if gf is not None else zero
        b, e = m.abs(), zero
        for t in reversed(range(begin, begin + lengths[s])):
            lam, bl = g[t] + m, g[t].abs() + b
            el = e + 2 * U * bl
            out["dx"][t], out["edx"][t] = lam, el
            hp, ehp = previous[t - begin]
            ehp = ehp + 2 * U * hp.abs()  # carried through memory in 32 bits
            out["da"][t] = lam * hp
            out["eda"][t] = el * hp.abs() + ehp * lam.abs() + el * ehp + U * (lam * hp).abs()
            m, b = full[t] * lam, full[t].abs() * bl
            e = full[t].abs() * el + 2 * U * b
        out["dh0"][s], out["edh0"][s] = m, e + 2 * U * m.abs()
    if a.dim() == 1:
        # sums of at most 64 terms in 32 bits, the partial sums in 64
        out["eda"] = out["eda"].sum(0) + 64 * U * out["da"].abs().sum(0)
        out["da"] = out["da"].sum(0)
    return out


def close(got, want, error, what):
    eps = torch.finfo(got.dtype).eps
    got = got.detach().cpu().double()
    tiny = 2.0**-24 if eps == 2.0**-10 else 2.0**-126  # half a step among float16's subnormals
    tolerance = error + eps / 2 * (want.abs() + error) * (1 + 2.0**-20) + tiny
    off = (got - want).abs() - tolerance
    assert got.shape == want.shape, what
    assert bool((off <= 0).all()), (what, float(off.max()), int(off.argmax()))


# ---------------------------------------------------------------- CPU


def table_of(native_lib, offsets):
    """(bytes, tables) of a story table, its pointers offsets from 0."""
    from leo_b200.ctypes_types import LeoB200StoryTables
    from leo_b200.native import check

    off = np.array(offsets, dtype=np.uint64)
    size = native_lib.leo_b200_story_table_bytes(off.ctypes.data, len(offsets) - 1)
    check(0 if size else -1)
    host, tables = torch.empty(size, dtype=torch.uint8), LeoB200StoryTables()
    check(native_lib.leo_b200_story_table(off.ctypes.data, len(offsets) - 1, host.data_ptr(), size, None,
                                          C.byref(tables)))
    return host.numpy().tobytes(), tables


@pytest.mark.parametrize("lengths", [[1], [0], [0, 0, 7, 0], [32, 32], [31, 1, 33], [5] * 40, [100, 0, 1, 64, 0, 3],
                                     [128, 1], [129, 0, 300], [40, 2000, 7, 700, 128, 65, 64, 1], [5000]])
def test_story_table(native_lib, lengths):
    """Starts and ranks of the tokens; tiles that cover them once; every tile behind those that it reads from."""
    from leo_b200.ctypes_types import LeoB200StoryTile

    offsets = offsets_of(lengths)
    tokens = offsets[-1]
    raw, t = table_of(native_lib, offsets)
    with_tokens = [s for s, n in enumerate(lengths) if n]
    assert (t.tokens, t.stories, t.full) == (tokens, len(lengths), len(with_tokens))
    order = np.frombuffer(raw, np.uint32, len(lengths), t.order or 0)
    assert order.tolist() == with_tokens + [s for s, n in enumerate(lengths) if not n]
    words = np.frombuffer(raw, np.uint32, 2 * (tokens // 32 + 2), t.words or 0).reshape(-1, 2)
    begins = [offsets[s] for s in with_tokens] + [tokens]
    for w, (starts, rank) in enumerate(words.tolist()):
        assert starts == sum(1 << (b - 32 * w) for b in begins if b // 32 == w)
        assert rank == sum(1 for b in begins if b < 32 * w)
    for k, longest in enumerate((128, 64)):
        tiles = []
        for d in reversed(range(2)):
            listed = [LeoB200StoryTile.from_buffer_copy(raw, (t.schedule[k][d] or 0) + 32 * i)
                      for i in range(t.tiles[k])]
            turn = {x.tile: i for i, x in enumerate(listed)}
            tiles = sorted(listed, key=lambda x: x.tile)
            assert [x.tile for x in tiles] == list(range(t.tiles[k]))
            assert [x.first for x in tiles] == [0] + np.cumsum([x.count for x in tiles]).tolist()[:-1]
            assert sum(x.count for x in tiles) == tokens and max(x.count for x in tiles) <= longest
            story = [i for i in range(len(begins) - 1) for _ in range(begins[i], begins[i + 1])]
            for x in tiles if tokens else []:
                last = x.first + x.count - 1
                into = story[x.first] if d == 0 else story[last]
                out = story[last] if d == 0 else story[x.first]
                where = begins[into] if d == 0 else begins[into + 1] - 1
                holder = next(y.tile for y in tiles if y.first <= where < y.first + y.count)
                assert x.holder == holder
                far = begins[out + 1] - 1 if d == 0 else begins[out]
                assert x.onward == int(not x.first <= far <= last)
                step = 1 if holder <= x.tile else -1
                assert all(turn[y] < turn[x.tile] for y in range(holder, x.tile, step))
        rank = [0] * t.tiles[k]
        for x in tiles if tokens else []:
            rank[x.tile] = rank[x.tile - 1] + 1 if x.tile and x.first not in begins else 0
        assert t.longest[k] == max(rank) + 1
    halves = {x.tile: x for x in (LeoB200StoryTile.from_buffer_copy(raw, (t.schedule[1][0] or 0) + 32 * i)
                                  for i in range(t.tiles[1]))}
    for i in range(t.tiles[0]):
        x = LeoB200StoryTile.from_buffer_copy(raw, (t.schedule[0][0] or 0) + 32 * i)
        assert halves[x.kept].first == x.first and halves[x.kept].kept == x.kept
        if x.count > 64:
            assert halves[x.kept + 1].first == x.first + 64


@pytest.mark.parametrize("offsets", [[1, 2], [0, 5, 3], [0, 2**31], [0]])
def test_story_table_refuses(native_lib, offsets):
    from leo_b200.native import LeoError

    with pytest.raises(LeoError):
        table_of(native_lib, offsets)


def test_story_table_refuses_bad_memory(native_lib):
    from leo_b200.ctypes_types import LeoB200StoryTables

    off = np.array([0, 500], dtype=np.uint64)
    size = native_lib.leo_b200_story_table_bytes(off.ctypes.data, 1)
    host, tables = torch.empty(size + 16, dtype=torch.uint8), C.byref(LeoB200StoryTables())
    call = native_lib.leo_b200_story_table
    assert call(off.ctypes.data, 1, host.data_ptr(), size - 1, None, tables) == -1
    assert call(off.ctypes.data, 1, host.data_ptr() + 4, size, None, tables) == -1
    assert call(off.ctypes.data, 1, host.data_ptr(), size, 8, tables) == -1
    assert call(off.ctypes.data, 1, None, size, None, tables) == -1
    assert call(off.ctypes.data, 1, host.data_ptr(), size, None, None) == -1


@pytest.mark.parametrize("offsets", [[], [0], [[0, 1]], [0.0, 1.0], [0, -1], [1, 2], [0, 2, 1]])
def test_layout_refuses_bad_offsets(native_lib, offsets):
    from leo_b200.gated_scan import StoryLayout
    from leo_b200.native import LeoError

    with pytest.raises((ValueError, LeoError)):
        StoryLayout(offsets, "cuda:0")


def test_layout_refuses_the_cpu(native_lib):
    from leo_b200.gated_scan import StoryLayout

    with pytest.raises(ValueError, match="CUDA device"):
        StoryLayout([0, 3], "cpu")


def test_cpu_tensors_are_refused(native_lib):
    from leo_b200.gated_scan import gated_scan, gated_scan_backward, gated_step

    x = torch.zeros(3, 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        gated_scan(x, x, None)
    with pytest.raises(ValueError, match="CUDA tensor"):
        gated_scan_backward(x, x, x, None, None)
    with pytest.raises(ValueError, match="CUDA tensor"):
        gated_step(x, x, x)


@pytest.mark.parametrize("bad", ["stories", "tokens", "channels", "dtype", "decay", "null", "final", "workspace"])
def test_entry_point_refuses_before_device_work(native_lib, bad):
    from leo_b200.ctypes_types import LeoB200StoryTables

    p = 256
    t = LeoB200StoryTables(p, p, ((p, p), (p, p)), (8, 16), (3, 6), 1000, 3, 3)
    args = dict(channels=70, dtype=1, decay_dtype=0, drive=p, final=p)  # and no workspace
    if bad == "stories":
        t.stories = 0
    elif bad == "tokens":
        t.tokens = 1 << 31
    elif bad == "channels":
        args["channels"] = 0
    elif bad == "dtype":
        args["dtype"] = 7
    elif bad == "decay":
        args.update(dtype=0, decay_dtype=1)
    elif bad == "null":
        args["drive"] = None
    elif bad == "final":
        args["final"] = None
    rc = native_lib.leo_b200_gated_scan(0, C.byref(t), args["channels"], args["dtype"], args["drive"], 70,
                                        args["decay_dtype"], p, 70, 0, None, p, args["final"], None,
                                        None, 0, None)
    assert rc == -1 and native_lib.leo_b200_last_error()
    rc = native_lib.leo_b200_gated_scan_backward(0, C.byref(t), args["channels"], args["dtype"], p, 70,
                                                 args["drive"], 70, args["decay_dtype"], p, 70, 0, None, None,
                                                 None if bad == "final" else p, p, p, None, None,
                                                 0, None)
    assert rc == -1


def test_oracle_gradients_match_differences():
    """The oracle's gradients against central differences of its own states."""
    lengths, channels = [3, 0, 5], 2
    s = make(3, lengths, channels, torch.float32, "f32")
    v = {k: s[k].double() for k in s}

    def value(x, a, h0):
        r = oracle(lengths, x, a, h0=h0)
        return float((r["h"] * v["g"]).sum() + (r["final"] * v["gf"]).sum())

    r = oracle(lengths, v["x"], v["a"], v["g"], v["h0"], v["gf"])
    for name, grad in (("x", r["dx"]), ("a", r["da"]), ("h0", r["dh0"])):
        for i in range(v[name].numel()):
            step = torch.zeros(v[name].numel(), dtype=torch.float64)
            step[i] = 1e-5
            at = {k: v[k] for k in ("x", "a", "h0")}
            up = value(**{**at, name: v[name] + step.view_as(v[name])})
            down = value(**{**at, name: v[name] - step.view_as(v[name])})
            assert abs((up - down) / 2e-5 - float(grad.reshape(-1)[i])) < 1e-8


# ---------------------------------------------------------------- GPU

SHAPES = [
    # lengths, channels
    ([1], 1),
    ([0, 1, 0], 3),
    ([0, 0], 5),
    ([15, 17, 16], 64),
    ([127, 1, 129], 65),
    ([128, 256, 128], 130),
    ([1] * 70 + [0, 3], 31),
    ([700, 0, 1300, 33], 66),
    ([2049], 257),
    ([6000, 1, 2500], 10),
]


def layout_of(lengths):
    from leo_b200.gated_scan import StoryLayout

    return StoryLayout(offsets_of(lengths), "cuda:0")


def run_all(s, lengths, layout=None, stream=None):
    from leo_b200.gated_scan import gated_scan, gated_scan_backward

    layout = layout or layout_of(lengths)
    scan = gated_scan(s["x"], s["a"], layout, s["h0"], keep_carries=True, stream=stream)
    grad = gated_scan_backward(s["g"], s["x"], s["a"], layout, scan.carries, initial=s["h0"], grad_final=s["gf"],
                               stream=stream)
    return scan, grad


def check_all(s, lengths, scan, grad):
    r = oracle(lengths, s["x"], s["a"], s["g"], s["h0"], s["gf"])
    close(scan.states, r["h"], r["eh"], "states")
    close(scan.final, r["final"], r["efinal"], "final")
    close(grad.drive, r["dx"], r["edx"], "grad_drive")
    close(grad.decay, r["da"], r["eda"], "grad_decay")
    if s["h0"] is not None:
        close(grad.initial, r["dh0"], r["edh0"], "grad_initial")
    else:
        assert grad.initial is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,decay", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"),
                                         ("f16", "f32"), ("f32", "channel"), ("bf16", "channel")])
@pytest.mark.parametrize("lengths,channels", SHAPES, ids=[f"{sum(n)}t-{len(n)}s-{c}c" for n, c in SHAPES])
def test_scan_and_gradients(native_lib, lengths, channels, dtype, decay):
    for initial in (True, False):
        s = make(len(lengths) + channels, lengths, channels, DTYPES[dtype], decay, initial, "cuda")
        scan, grad = run_all(s, lengths)
        check_all(s, lengths, scan, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [1, 66, 136])
@pytest.mark.parametrize("dtype,decay", [("f32", "f32"), ("f32", "channel"), ("bf16", "bf16"), ("bf16", "f32"),
                                         ("bf16", "channel"), ("f16", "f16"), ("f16", "channel")])
def test_long_stories_of_few_channels(native_lib, channels, dtype, decay):
    """Tiles mapped ahead, with short, empty and long stories around one another."""
    lengths = [300, 2600, 0, 1, 5, 130, 2200, 64]
    s = make(41, lengths, channels, DTYPES[dtype], decay, channels != 66, "cuda")
    scan, grad = run_all(s, lengths)
    check_all(s, lengths, scan, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,channels,dtype,decay", [
    ([3000, 600], 1600, "bf16", "f32"), ([2300], 1537, "f32", "f32"), ([5000], 768, "f16", "channel"),
    ([40, 3500, 100, 2700], 648, "f32", "channel"), ([2500, 7], 1282, "bf16", "bf16")])
def test_long_stories_of_many_channels(native_lib, lengths, channels, dtype, decay):
    """States handed from tile to tile in one pass, over more tiles than a tile looks back."""
    s = make(31, lengths, channels, DTYPES[dtype], decay, True, "cuda")
    scan, grad = run_all(s, lengths)
    check_all(s, lengths, scan, grad)


@pytest.mark.gpu
def test_one_story_over_many_blocks(native_lib):
    """A story long enough that partial states of distant blocks meet, gates near 1."""
    lengths = [20_011]
    s = make(5, lengths, 70, torch.float32, "f32", True, "cuda")
    s["a"] = (1.0 - 1e-3 * torch.rand(20_011, 70, device="cuda"))
    scan, grad = run_all(s, lengths)
    check_all(s, lengths, scan, grad)
    again, grad2 = run_all(s, lengths)
    assert torch.equal(scan.states, again.states) and torch.equal(grad.decay, grad2.decay)


@pytest.mark.gpu
def test_gradients_match_differences(native_lib):
    """The kernel's gradient along a direction against the oracle's central difference."""
    lengths = [40, 0, 150]
    s = make(9, lengths, 6, torch.float32, "f32", True, "cuda")
    _, grad = run_all(s, lengths)
    r = oracle(lengths, s["x"], s["a"], s["g"], s["h0"], s["gf"])
    gen = torch.Generator().manual_seed(1)
    for name, got, error in (("x", grad.drive, r["edx"]), ("a", grad.decay, r["eda"]), ("h0", grad.initial, r["edh0"])):
        v = torch.randn(got.shape, generator=gen, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = {k: s[k].cpu().double() for k in ("x", "a", "h0")}
            moved[name] = moved[name] + sign * 1e-6 * v
            q = oracle(lengths, moved["x"], moved["a"], h0=moved["h0"])
            ends.append(float((q["h"] * s["g"].cpu().double()).sum() + (q["final"] * s["gf"].cpu().double()).sum()))
        slope = (ends[0] - ends[1]) / 2e-6
        mine = float((got.cpu().double() * v).sum())
        tolerance = float(((error + U * got.cpu().double().abs()) * v.abs()).sum()) + 1e-6 * (1 + abs(slope))
        assert abs(mine - slope) <= tolerance, (name, mine, slope, tolerance)


@pytest.mark.gpu
def test_rows_of_wider_tensors(native_lib):
    """Slices of one projection, a broadcast gate row, and rows that no vector load reaches aligned."""
    lengths, channels = [200, 313], 70
    for dtype, extra in ((torch.bfloat16, 1), (torch.float32, 0), (torch.float16, 2)):
        s = make(11, lengths, channels, dtype, "same", True, "cuda")
        wide = torch.zeros(sum(lengths), 3 * channels + extra, dtype=dtype, device="cuda")
        wide[:, extra:channels + extra] = s["x"]
        wide[:, channels + extra:2 * channels + extra] = s["a"]
        wide[:, 2 * channels + extra:] = s["g"]
        t = dict(s, x=wide[:, extra:channels + extra], a=wide[:, channels + extra:2 * channels + extra],
                 g=wide[:, 2 * channels + extra:])
        scan, grad = run_all(t, lengths)
        check_all(t, lengths, scan, grad)
        t = dict(s, a=s["a"][:1].expand(sum(lengths), channels))
        scan, grad = run_all(t, lengths)
        check_all(t, lengths, scan, grad)


@pytest.mark.gpu
def test_a_story_never_reaches_another(native_lib):
    """NaN and infinities of one story stay in it, in both directions: in one
    tile, over many tiles mapped ahead, and over many in one pass."""
    for lengths, channels in (([90, 200, 61], 64), ([90, 200, 2600, 61], 64), ([90, 200, 2600, 61], 1540)):
        check_isolation(lengths, channels)


def check_isolation(lengths, channels):
    s = make(13, lengths, channels, torch.float32, "f32", True, "cuda")
    clean, clean_grad = run_all(s, lengths)
    for bad in (float("nan"), float("inf")):
        t = {k: v.clone() for k, v in s.items()}
        t["x"][100], t["a"][250], t["g"][120] = bad, bad, bad
        t["h0"][1], t["gf"][1] = bad, bad
        scan, grad = run_all(t, lengths)
        for a, b in ((scan.states, clean.states), (grad.drive, clean_grad.drive), (grad.decay, clean_grad.decay)):
            assert torch.equal(a[:90], b[:90]) and torch.equal(a[290:], b[290:])
            assert not torch.isfinite(a[90:290]).all()
        for a, b in ((scan.final, clean.final), (grad.initial, clean_grad.initial)):
            assert torch.equal(a[0], b[0]) and torch.equal(a[2:], b[2:])


@pytest.mark.gpu
def test_steps_equal_the_scan(native_lib):
    """A story fed a token at a time to every lane ends in the scan's states."""
    from leo_b200.gated_scan import gated_scan, gated_step

    lanes, tokens, channels = 5, 37, 71
    s = make(17, [tokens] * lanes, channels, torch.bfloat16, "f32", True, "cuda")
    scan = gated_scan(s["x"], s["a"], layout_of([tokens] * lanes), s["h0"])
    r = oracle([tokens] * lanes, s["x"], s["a"], h0=s["h0"])
    state = s["h0"].clone()
    x, a = s["x"].view(lanes, tokens, channels), s["a"].view(lanes, tokens, channels)
    for t in range(tokens):
        out = gated_step(x[:, t], a[:, t], state)
        close(out, r["h"].view(lanes, tokens, channels)[:, t], r["eh"].view(lanes, tokens, channels)[:, t], t)
    close(state, r["final"], r["efinal"], "state")
    close(scan.final, r["final"], r["efinal"], "final")


@pytest.mark.gpu
@pytest.mark.parametrize("lanes,channels,dtype,decay", [(1, 1, "f32", "f32"), (3, 257, "bf16", "bf16"),
                                                        (64, 1024, "f16", "channel"), (70_000, 3, "f32", "channel"),
                                                        (7, 70, "bf16", "f32"), (0, 4, "f32", "f32")])
def test_step(native_lib, lanes, channels, dtype, decay):
    from leo_b200.gated_scan import gated_step

    s = make(19, [lanes], channels, DTYPES[dtype], decay, False, "cuda")
    wide = torch.randn(lanes, channels + 3, device="cuda")
    state = wide[:, 1:channels + 1]
    before = wide.clone()
    out = gated_step(s["x"], s["a"], state)
    want = s["a"].cpu().double() * before[:, 1:channels + 1].cpu().double() + s["x"].cpu().double()
    # one fused or two separate roundings in 32 bits
    error = 2 * U * (want.abs() + s["x"].cpu().double().abs())
    close(state, want, error, "state")
    close(out, want, error, "output")
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, channels + 1:], before[:, channels + 1:])


@pytest.mark.gpu
def test_captured_and_replayed(native_lib):
    """Two graphs that share a layout, replayed in turn on new inputs, and eager calls between them."""
    from leo_b200.gated_scan import gated_step

    lengths, channels = [300, 0, 500], 70
    layout = layout_of(lengths)
    graphs = []
    for seed in (1, 2):
        s = make(seed, lengths, channels, torch.bfloat16, "f32", True, "cuda")
        state = torch.zeros(4, channels, device="cuda")
        run_all(s, lengths, layout)
        gated_step(s["x"][:4], s["a"][:4], state)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run_all(s, lengths, layout)
            gated_step(s["x"][:4], s["a"][:4], state)
        graphs.append((graph, s, state, out))
    for turn in range(3):
        for k, (graph, s, state, (scan, grad)) in enumerate(graphs):
            new = make(100 + 10 * turn + k, lengths, channels, torch.bfloat16, "f32", True, "cuda")
            for name in s:
                s[name].copy_(new[name])
            state.zero_()
            graph.replay()
        eager = run_all(graphs[0][1], lengths, layout)
        torch.cuda.synchronize()
        for graph, s, state, (scan, grad) in graphs:
            check_all(s, lengths, scan, grad)
            assert torch.equal(state, s["x"][:4].float())
        assert torch.equal(eager[0].states, graphs[0][3][0].states)


@pytest.mark.gpu
def test_other_streams(native_lib):
    """Calls on several streams at once with one layout, and `stream=` beside a busy current stream."""
    lengths, channels = [3000, 1000], 130
    layout = layout_of(lengths)
    s = make(23, lengths, channels, torch.float32, "f32", True, "cuda")
    want, want_grad = run_all(s, lengths, layout)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for turn in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(run_all(s, lengths, layout))
            got.append(run_all(s, lengths, layout, stream=st))
    torch.cuda.synchronize()
    for scan, grad in got:
        assert torch.equal(scan.states, want.states) and torch.equal(scan.final, want.final)
        assert torch.equal(grad.drive, want_grad.drive) and torch.equal(grad.decay, want_grad.decay)
    # a layout that goes away while another stream still reads it
    for st in streams:
        with torch.cuda.stream(st):
            torch.cuda._sleep(2_000_000)
            got = run_all(s, lengths, layout_of(lengths))
        torch.full((1 << 16,), 7, dtype=torch.uint8, device="cuda")
        st.synchronize()
        assert torch.equal(got[0].states, want.states)


@pytest.mark.gpu
def test_no_wait_gave_up(native_lib):
    from leo_b200.gated_scan import gated_scan_gave_up

    assert gated_scan_gave_up(0) is False


@pytest.mark.gpu
def test_refusals(native_lib):
    from leo_b200.gated_scan import gated_scan, gated_scan_backward, gated_step

    layout = layout_of([4, 6])
    x = torch.zeros(10, 8, device="cuda")
    h0 = torch.zeros(2, 8, device="cuda")
    scan = gated_scan(x, x, layout, h0, keep_carries=True)

    def refused(call, match):
        with pytest.raises(ValueError, match=match):
            call()

    refused(lambda: gated_scan(x.double(), x, layout), "float32, bfloat16 or float16")
    refused(lambda: gated_scan(x[:9], x[:9], layout), "10 tokens")
    refused(lambda: gated_scan(x[:, :0], x[:, :0], layout), "at least one channel")
    refused(lambda: gated_scan(x.view(10, 2, 4), x, layout), "two dimensions")
    refused(lambda: gated_scan(x.t().contiguous().t(), x, layout), "adjacent")
    refused(lambda: gated_scan(x, x.bfloat16(), layout), "drive's type or float32")
    refused(lambda: gated_scan(x, x[:, :7], layout), "decay must have shape")
    refused(lambda: gated_scan(x, x[0, :7], layout), "one row")
    refused(lambda: gated_scan(x, x.cpu(), layout), "CUDA tensor")
    refused(lambda: gated_scan(x, x, layout, h0[:1]), "initial must have shape")
    refused(lambda: gated_scan(x, x, layout, h0.bfloat16()), "initial must be")
    refused(lambda: gated_scan(x, x, layout, torch.zeros(8, 2, device="cuda").t()), "contiguous")
    refused(lambda: gated_scan(x.clone().requires_grad_(), x, layout), "detach")
    refused(lambda: gated_scan_backward(x[:9], x, x, layout, scan.carries), "grad_states must have shape")
    refused(lambda: gated_scan_backward(x, x, x, layout, None), "needs the carries")
    refused(lambda: gated_scan_backward(x, x, x, layout, scan.carries[:-1]), "carries must have shape")
    refused(lambda: gated_scan_backward(x, x, x, layout, scan.carries, grad_final=h0[:1]), "grad_final must have")
    refused(lambda: gated_step(x, x, x.bfloat16()), "state must be")
    refused(lambda: gated_step(x, x, x[:1].expand(10, 8)), "overlap")
    refused(lambda: gated_step(x, x, h0), "state must have shape")
    with torch.no_grad():
        gated_scan(x.clone().requires_grad_(), x, layout)


# ---------------------------------------------------------------- infinite states


def token_by_token(lengths, s):
    """States and gradients in 64 bits, a token at a time; infinities and NaN as the recurrence makes them."""
    x, a, g, h0, gf = (s[k].cpu().double() for k in ("x", "a", "g", "h0", "gf"))
    a = a.expand_as(x)
    h, dx, da = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    final, dh0 = h0.clone(), gf.clone()
    for i, begin in enumerate(offsets_of(lengths)[:-1]):
        for t in range(begin, begin + lengths[i]):
            final[i] = h[t] = a[t] * (h[t - 1] if t > begin else h0[i]) + x[t]
        for t in reversed(range(begin, begin + lengths[i])):
            dx[t] = g[t] + dh0[i]
            da[t] = dx[t] * (h[t - 1] if t > begin else h0[i])
            dh0[i] = a[t] * dx[t]
    return h, final, dx, da, dh0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,decay", [("f32", "f32"), ("f32", "channel"), ("bf16", "f32")])
@pytest.mark.parametrize("lengths,channels", [([1500, 700], 72), ([5000], 10), ([3000, 0, 90, 40], 71),
                                              ([2500, 130, 2100], 1540)],
                         ids=["tiles", "runs", "unaligned", "one pass"])
def test_infinite_states_stay_infinite(native_lib, lengths, channels, dtype, decay):
    """Products of many gates that underflow: an infinite state times one is infinite, with the sign that
    the gates give it, and NaN only after a gate of 0; on the way back as well.  Finite channels keep to
    their bounds, however small their products of gates.  (Eight gates in a row of product 0 in float
    may do what one of 0 does, which 1e-4 does not reach.)"""
    s = make(3, lengths, channels, DTYPES[dtype], decay, True)
    fast = torch.tensor([0.3, 0.05, -0.4, 1e-4, 0.9, -0.01])[torch.arange(channels) % 6]
    s["a"] = (fast if decay == "channel" else fast.expand(sum(lengths), channels)).clone()
    bad = torch.arange(channels) // 6 % 2 == 0  # channels with infinities
    s["h0"][0, bad] = float("inf")
    s["gf"][0, bad] = -float("inf")
    if decay != "channel":  # a gate of 0 far behind the infinity, in some of them
        s["a"][lengths[0] - 2, bad & (torch.arange(channels) % 4 == 0)] = 0.0
        if len(lengths) == 3:  # and an infinite drive in the middle of the last story
            s["x"][sum(lengths) - lengths[-1] // 2, bad] = -float("inf")
    s = {k: v.cuda() for k, v in s.items()}
    scan, grad = run_all(s, lengths)
    h, final, dx, da, dh0 = token_by_token(lengths, s)
    assert bool(torch.isinf(h[:, bad]).any())
    if decay == "channel":
        da = da.sum(0)
    for got, want, what in ((scan.states, h, "states"), (scan.final, final, "final"), (grad.drive, dx, "drive"),
                            (grad.decay, da, "decay"), (grad.initial, dh0, "initial")):
        want = want.to(torch.float32)
        rest = torch.isfinite(want)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want)), what
        assert torch.equal(torch.isfinite(got.cpu()), rest), what
        there = ~rest & ~torch.isnan(want)
        assert torch.equal(got.cpu().float()[there], want[there]), what
    clean = {k: v[..., ~bad.cuda()].contiguous() for k, v in s.items()}
    part = lambda t: t[..., ~bad.cuda()]  # noqa: E731
    r = oracle(lengths, clean["x"], clean["a"], clean["g"], clean["h0"], clean["gf"])
    close(part(scan.states), r["h"], r["eh"], "states")
    close(part(grad.drive), r["dx"], r["edx"], "grad_drive")
    close(part(grad.decay), r["da"], r["eda"], "grad_decay")

"""Cases and plain forms of the story-scan and logit operators.

``run`` passes once through one operator: with ``own`` false in elementary
torch operations (32 bits; 64 where a whole-number answer hangs on a border),
with ``own`` true through ``leo_b200.gated_scan`` and ``leo_b200.logits``.
``exact`` gives the same outputs in 64 bits, written separately from the plain
form: the recurrence step by step, the logit operators from their definitions.

Kinds of case:

* ``scan``   h_t = a_t h_{t-1} + x_t over packed stories, forward only;
* ``train``  the same with its backward pass;
* ``step``   one token for every lane, the 32-bit state updated in place;
* ``adjust`` penalties, biases and a grammar mask on logits;
* ``pick``   the same, then the next symbol (greedy or at a given uniform);
* ``loss``   the cross entropy over the allowed symbols, with its gradient.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

# Decays of the framework's own configurations (branch, membrane, eligibility,
# fatigue, the three adaptations): what a channel's gate is drawn around.
DECAYS = (0.85, 0.90, 0.95, 0.97, 0.99, 0.999)


def listed():
    return [
        # A handful of short texts, as an interactive caller sends them; latency counts.
        {"name": "scan-short-stories", "kind": "scan", "tokens": 137, "stories": 4, "channels": 192,
         "dtype": "float32", "decay": "steps", "initial": True, "empty": 0},
        # The 64-worker story batch (512-2048 bytes a story) over the 1,024 winners of a step, inference.
        {"name": "scan-64-stories", "kind": "scan", "tokens": 81920, "stories": 64, "channels": 1024,
         "dtype": "bfloat16", "decay": "float32", "initial": False, "empty": 0},
        # The 32-worker story batch (256-1024 bytes a story) over the probe model's 4,096 neurons, training.
        {"name": "train-32-stories", "kind": "train", "tokens": 20480, "stories": 32, "channels": 4096,
         "dtype": "bfloat16", "decay": "float32", "initial": True, "empty": 1},
        # One long document, one fixed decay a channel (as the configurations have), an odd number of channels.
        {"name": "train-one-document", "kind": "train", "tokens": 65537, "stories": 1, "channels": 257,
         "dtype": "float32", "decay": "channel", "initial": True, "empty": 0},
        # One byte for each of 64 lanes: the serving step.
        {"name": "step-64-lanes", "kind": "step", "lanes": 64, "channels": 1024, "dtype": "float32", "decay": "steps"},
        # A large serving batch.
        {"name": "step-4096-lanes", "kind": "step", "lanes": 4096, "channels": 4096, "dtype": "bfloat16",
         "decay": "float32"},
        # 64 lanes of byte logits, each with the story so far as its history.
        {"name": "adjust-bytes", "kind": "adjust", "rows": 64, "vocabulary": 257, "history": 2048, "states": 8,
         "dtype": "float32", "bias": "shared"},
        # A subword vocabulary of odd size, one bias row for each request.
        {"name": "adjust-wide", "kind": "adjust", "rows": 256, "vocabulary": 50001, "history": 1000, "states": 0,
         "dtype": "bfloat16", "bias": "rows"},
        # The next byte of 64 lanes, drawn under a grammar mask.
        {"name": "pick-bytes", "kind": "pick", "rows": 64, "vocabulary": 257, "history": 512, "states": 8,
         "dtype": "float32", "bias": "none", "greedy": False},
        # The next token of 64 requests from a large vocabulary.
        {"name": "pick-wide", "kind": "pick", "rows": 64, "vocabulary": 131072, "history": 2048, "states": 0,
         "dtype": "bfloat16", "bias": "shared", "greedy": False},
        # Every target of the 64-worker story batch: byte logits, a grammar state a row.
        {"name": "loss-bytes", "kind": "loss", "rows": 81984, "vocabulary": 257, "states": 8, "dtype": "float32"},
        # A training step's rows over a subword vocabulary.
        {"name": "loss-wide", "kind": "loss", "rows": 2048, "vocabulary": 32001, "states": 0, "dtype": "bfloat16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "train", "train", "step", "adjust", "pick", "pick", "loss", "loss"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if kind in ("scan", "train"):
        channels = _log(rng, 16, 4096)
        tokens = _log(rng, 1, min(131072, 60_000_000 // channels))
        return {"kind": kind, "tokens": tokens, "stories": _log(rng, 1, max(1, min(256, tokens))),
                "channels": channels, "dtype": dtype,
                "decay": rng.choice(["steps", "float32", "channel"]), "initial": rng.random() < 0.5,
                "empty": rng.choice([0, 0, 1, 3])}
    if kind == "step":
        return {"kind": kind, "lanes": _log(rng, 1, 4096), "channels": _log(rng, 16, 4096), "dtype": dtype,
                "decay": rng.choice(["steps", "float32", "channel"])}
    if rng.random() < 0.5:  # the byte model's own classes
        vocabulary = 257
        rows = _log(rng, 1, 81984 if kind == "loss" else 4096)
    else:
        vocabulary = _log(rng, 258, 131072)
        rows = _log(rng, 1, max(1, min(4096, 8_000_000 // vocabulary)))
    case = {"kind": kind, "rows": rows, "vocabulary": vocabulary, "states": rng.choice([0, 1, 8, 40]),
            "dtype": dtype}
    if kind != "loss":
        case["history"] = _log(rng, 1, 2048)
        case["bias"] = rng.choice(["none", "shared", "rows"])
    if kind == "pick":
        case["greedy"] = rng.random() < 0.4
    return case


# ---------------------------------------------------------------- inputs


def _offsets(case, generator):
    """Story boundaries: lengths within a factor of four of one another, `empty` of them zero."""
    stories, empty = case["stories"], min(case["empty"], case["stories"] - 1)
    weights = 0.4 + 1.2 * torch.rand(stories, generator=generator, dtype=torch.float64)
    weights[torch.randperm(stories, generator=generator)[:empty]] = 0.0
    ends = torch.round(torch.cumsum(weights, 0) / weights.sum() * case["tokens"]).to(torch.int64)
    ends[-1] = case["tokens"]
    return [0] + ends.tolist()


def _gates(shape, case, g):
    base = torch.tensor(DECAYS, device=DEVICE)[torch.randint(len(DECAYS), shape[-1:], generator=g, device=DEVICE)]
    if case["decay"] == "channel":
        return base.to(torch.float32)
    speed = 2.0 * torch.rand(shape, generator=g, device=DEVICE)
    return torch.exp(torch.log(base) * speed).to(torch.float32 if case["decay"] == "float32"
                                                 else DTYPES[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    s = {"kind": kind}
    if kind in ("scan", "train"):
        tokens, stories, channels = case["tokens"], case["stories"], case["channels"]
        offsets = _offsets(case, cpu)
        s["drive"] = torch.randn(tokens, channels, generator=g, device=DEVICE).to(dtype)
        s["decay"] = _gates((tokens, channels), case, g)
        s["initial"] = torch.randn(stories, channels, generator=g, device=DEVICE) if case["initial"] else None
        if kind == "train":
            s["grad_states"] = torch.randn(tokens, channels, generator=g, device=DEVICE).to(dtype)
            s["grad_final"] = torch.randn(stories, channels, generator=g, device=DEVICE)
        s["offsets"] = torch.tensor(offsets, device=DEVICE)
        s["longest"] = max(b - a for a, b in zip(offsets, offsets[1:]))
        if own:
            from leo_b200.gated_scan import StoryLayout

            s["layout"] = StoryLayout(offsets, torch.device(DEVICE, torch.cuda.current_device()))
    elif kind == "step":
        shape = (case["lanes"], case["channels"])
        s["drive"] = torch.randn(shape, generator=g, device=DEVICE).to(dtype)
        s["decay"] = _gates(shape, case, g)
        s["state"] = torch.randn(shape, generator=g, device=DEVICE)
    else:
        rows, vocabulary = case["rows"], case["vocabulary"]
        # A peaked distribution: a few likely symbols a row over a wide tail, as a trained model's logits are.
        s["logits"] = (3.0 * torch.randn(rows, vocabulary, generator=g, device=DEVICE)).to(dtype)
        s["allowed"] = s["state"] = None
        if case["states"]:
            words = (vocabulary + 31) // 32
            bits = torch.rand(case["states"], words * 32, generator=g, device=DEVICE) < 0.7
            bits[:, 0] = True  # a grammar always leaves something to say
            weight = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], device=DEVICE)
            s["allowed"] = (bits.view(-1, words, 32) * weight).sum(2).to(torch.int32)
            # -1: a row that no grammar constrains
            s["state"] = torch.randint(-1, case["states"], (rows,), generator=g, device=DEVICE, dtype=torch.int32)
        if kind == "loss":
            s["targets"] = torch.randint(0, vocabulary, (rows,), generator=g, device=DEVICE, dtype=torch.int32)
            if case["states"]:  # a target is a symbol that its grammar state allows
                ok = _allowed(s["allowed"], s["state"], rows, vocabulary).gather(1, s["targets"].long()[:, None])[:, 0]
                s["targets"] = torch.where(ok, s["targets"], 0)
            quiet = torch.rand(rows, generator=g, device=DEVICE) < 0.05  # rows without a target
            s["targets"] = torch.where(quiet, -1, s["targets"]).to(torch.int32)
            # the end of a document weighs four times as much, as the configurations have it
            s["weights"] = torch.where(s["targets"] == vocabulary - 1, 4.0, 1.0)
        else:
            # A text so far: symbols of very different frequency, its length another one in each row.
            u = torch.rand(rows, case["history"], generator=g, device=DEVICE)
            s["history"] = torch.clamp((vocabulary * u ** 3).to(torch.int32), max=vocabulary - 1)
            s["lengths"] = torch.randint(0, case["history"] + 1, (rows,), generator=g, device=DEVICE,
                                         dtype=torch.int32)
            s["bias"] = None
            if case["bias"] != "none":
                shape = (vocabulary,) if case["bias"] == "shared" else (rows, vocabulary)
                s["bias"] = torch.randn(shape, generator=g, device=DEVICE)
            s["repetition"] = 1.0 + 0.5 * torch.rand(rows, generator=g, device=DEVICE)
            s["presence"] = 0.5 * torch.rand(rows, generator=g, device=DEVICE)
            s["frequency"] = 0.1 * torch.rand(rows, generator=g, device=DEVICE)
        if kind == "pick":
            warm = 0.5 + torch.rand(rows, generator=g, device=DEVICE)
            s["temperature"] = torch.zeros_like(warm) if case["greedy"] else warm
            s["uniforms"] = torch.rand(rows, generator=g, device=DEVICE, dtype=torch.float64)
    return s


# ---------------------------------------------------------------- the operators' plain forms


def _allowed(table, state, rows, vocabulary):
    bits = (table[:, :, None] >> torch.arange(32, device=table.device)) & 1
    bits = bits.reshape(table.shape[0], -1)[:, :vocabulary].bool()
    return bits[state.clamp(min=0).long()] | (state < 0)[:, None]


def _doubling(gate, value, backwards=False):
    """All states of value_t + gate_t * previous, by combining spans of doubling length."""
    span, tokens = 1, value.shape[0]
    while span < tokens:
        if backwards:
            near, far = slice(0, tokens - span), slice(span, tokens)
        else:
            near, far = slice(span, tokens), slice(0, tokens - span)
        value_next, gate_next = value.clone(), gate.clone()
        value_next[near] = value[near] + gate[near] * value[far]
        gate_next[near] = gate[near] * gate[far]
        value, gate = value_next, gate_next
        span *= 2
    return value


def _plain_scan(s):
    offsets, drive = s["offsets"], s["drive"]
    tokens, channels = drive.shape
    # Squaring a slow gate over and over doubles its relative error each time: 64 bits for long stories.
    wide = torch.float64 if s["longest"] > 4096 else torch.float32
    decay = s["decay"].to(wide).expand(tokens, channels)
    x = drive.to(wide)
    full = offsets[1:] > offsets[:-1]  # stories with a token
    first, last = offsets[:-1][full], offsets[1:][full] - 1
    start = torch.zeros(len(offsets) - 1, channels, device=DEVICE, dtype=wide)
    if s["initial"] is not None:
        start += s["initial"]
    value, gate = x.clone(), decay.clone()
    value[first] = decay[first] * start[full] + x[first]
    gate[first] = 0.0
    states = _doubling(gate, value)
    final = start.clone()
    final[full] = states[last]
    out = {"states": states.to(drive.dtype), "final": final.float()}
    if s["kind"] == "scan":
        return out
    previous = torch.cat([states[:1], states[:-1]])
    previous[first] = start[full]
    value = s["grad_states"].to(wide, copy=True)
    value[last] += s["grad_final"][full]
    gate = torch.cat([decay[1:], decay[:1]])
    gate[last] = 0.0
    slope = _doubling(gate, value, backwards=True)
    grad_decay = slope * previous
    out["grad_drive"] = slope.to(drive.dtype)
    out["grad_decay"] = (grad_decay.sum(0, dtype=torch.float64) if s["decay"].dim() == 1 else grad_decay).to(s["decay"].dtype)
    if s["initial"] is not None:
        grad_initial = s["grad_final"].clone()
        grad_initial[full] = (decay[first] * slope[first]).float()
        out["grad_initial"] = grad_initial
    return out


def _plain_step(s):
    state = s["decay"].float() * s["state"] + s["drive"].float()
    s["state"].copy_(state)
    return {"states": state.to(s["drive"].dtype), "state": s["state"]}


def _adjusted(s, dtype):
    rows, vocabulary = s["logits"].shape
    z = s["logits"].to(dtype)
    columns = torch.arange(s["history"].shape[1], device=DEVICE)
    symbol = torch.where(columns < s["lengths"][:, None], s["history"], vocabulary).long()
    count = torch.zeros(rows, vocabulary + 1, device=DEVICE, dtype=dtype)
    count.scatter_add_(1, symbol, torch.ones((), device=DEVICE, dtype=dtype).expand(symbol.shape))
    count = count[:, :vocabulary]
    repetition = s["repetition"].to(dtype)[:, None]
    seen = count > 0
    z = torch.where(seen, torch.where(z > 0, z / repetition, z * repetition), z)
    z = z - torch.where(seen, s["presence"].to(dtype)[:, None] + s["frequency"].to(dtype)[:, None] * count, 0.0)
    if s["bias"] is not None:
        z = z + s["bias"].to(dtype)
    if s["allowed"] is not None:
        z = torch.where(_allowed(s["allowed"], s["state"], rows, vocabulary), z, -math.inf)
    return z


def _plain_pick(s):
    z = _adjusted(s, torch.float64)
    rows, vocabulary = z.shape
    top = z.amax(1, keepdim=True)
    index = torch.arange(vocabulary, device=DEVICE)
    best = torch.where(z == top, index, vocabulary).amin(1)
    temperature = s["temperature"].double()[:, None]
    greedy = temperature == 0
    weight = torch.exp((z - top) / torch.where(greedy, 1.0, temperature))
    sums = torch.cumsum(weight, 1)
    drawn = (sums <= s["uniforms"][:, None] * sums[:, -1:]).sum(1)
    drawn = torch.minimum(drawn, torch.where(weight > 0, index, 0).amax(1))
    symbol = torch.where(greedy[:, 0], best, drawn)
    chance = weight.gather(1, symbol[:, None])[:, 0] / sums[:, -1]
    return {"symbols": symbol.to(torch.int32), "log_probability": torch.log(chance).float()}


def _plain_loss(s):
    logits, targets = s["logits"], s["targets"]
    rows, vocabulary = logits.shape
    z = logits.float()
    if s["allowed"] is not None:
        z = torch.where(_allowed(s["allowed"], s["state"], rows, vocabulary), z, -math.inf)
    top = z.amax(1, keepdim=True)
    weight = torch.exp(z - top)
    total = weight.sum(1, keepdim=True)
    has = targets >= 0
    at = targets.clamp(min=0).long()[:, None]
    loss = torch.log(total[:, 0]) + top[:, 0] - z.gather(1, at)[:, 0]
    gradient = weight / total
    gradient.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    gradient = torch.where(has[:, None], s["weights"][:, None] * gradient, 0.0)
    return {"losses": torch.where(has, loss, 0.0), "gradient": gradient.to(logits.dtype)}


# ---------------------------------------------------------------- one pass


def _run_own(s):
    kind = s["kind"]
    if kind in ("scan", "train"):
        from leo_b200.gated_scan import gated_scan, gated_scan_backward

        scan = gated_scan(s["drive"], s["decay"], s["layout"], s["initial"], keep_carries=kind == "train")
        out = {"states": scan.states, "final": scan.final}
        if kind == "train":
            grad = gated_scan_backward(s["grad_states"], s["drive"], s["decay"], s["layout"], scan.carries,
                                       initial=s["initial"], grad_final=s["grad_final"])
            out["grad_drive"], out["grad_decay"] = grad.drive, grad.decay
            if s["initial"] is not None:
                out["grad_initial"] = grad.initial
        return out
    if kind == "step":
        from leo_b200.gated_scan import gated_step

        return {"states": gated_step(s["drive"], s["decay"], s["state"]), "state": s["state"]}
    from leo_b200.logits import adjust_logits, masked_cross_entropy, pick_symbols

    if kind == "loss":
        losses, gradient = masked_cross_entropy(s["logits"], s["targets"], allowed=s["allowed"], state=s["state"],
                                                weights=s["weights"])
        return {"losses": losses, "gradient": gradient}
    penalties = {"history": s["history"], "lengths": s["lengths"], "repetition": s["repetition"],
                 "presence": s["presence"], "frequency": s["frequency"], "bias": s["bias"],
                 "allowed": s["allowed"], "state": s["state"]}
    if kind == "adjust":
        return {"logits": adjust_logits(s["logits"], **penalties)}
    symbols, log_probability = pick_symbols(s["logits"], temperature=s["temperature"], uniforms=s["uniforms"],
                                            **penalties)
    return {"symbols": symbols, "log_probability": log_probability}


def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if kind in ("scan", "train"):
        return _plain_scan(s)
    if kind == "step":
        return _plain_step(s)
    if kind == "adjust":
        return {"logits": _adjusted(s, torch.float32).to(s["logits"].dtype)}
    return _plain_pick(s) if kind == "pick" else _plain_loss(s)


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "float32" else 2
    if kind in ("scan", "train", "step"):
        elements = case.get("tokens", case.get("lanes")) * case["channels"]
        gate = {"steps": size * elements, "float32": 4 * elements, "channel": 4 * case["channels"]}[case["decay"]]
        if kind == "step":
            return {"bytes": elements * (2 * size + 8) + gate, "flops": 2 * elements}
        ends = 4 * case["stories"] * case["channels"]
        moved = elements * 2 * size + gate + ends * (2 if case["initial"] else 1)
        if kind == "train":
            moved += elements * 2 * size + gate + ends * (2 if case["initial"] else 1)
        return {"bytes": moved, "flops": elements * (2 if kind == "scan" else 5)}
    rows, vocabulary = case["rows"], case["vocabulary"]
    elements = rows * vocabulary
    mask = case["states"] * ((vocabulary + 31) // 32) * 4 + (4 * rows if case["states"] else 0)
    if kind == "loss":
        return {"bytes": 2 * size * elements + 12 * rows + mask, "flops": 6 * elements}
    moved = size * elements + mask + 4 * rows * (case["history"] // 2 + 4)
    moved += {"none": 0, "shared": 4 * vocabulary, "rows": 4 * elements}[case["bias"]]
    if kind == "adjust":
        return {"bytes": moved + size * elements, "flops": 3 * elements}
    return {"bytes": moved + 20 * rows, "flops": 8 * elements}


# ---------------------------------------------------------------- 64 bits, from the definitions


def _exact_scan(case, s):
    offsets = s["offsets"].tolist()
    tokens, channels = s["drive"].shape
    stories = case["stories"]
    lengths = [offsets[i + 1] - offsets[i] for i in range(stories)]
    x = s["drive"].double()
    a = s["decay"].double()
    at = lambda rows: a[rows] if a.dim() == 2 else a  # noqa: E731
    start = s["initial"].double() if s["initial"] is not None else torch.zeros(stories, channels, device=DEVICE,
                                                                              dtype=torch.float64)
    # Stories from the longest to the shortest: at every step the first `live` of them still have a token.
    order = sorted(range(stories), key=lambda i: -lengths[i])
    begin = torch.tensor([offsets[i] for i in order], device=DEVICE)
    h = start[torch.tensor(order, device=DEVICE)]
    states = torch.empty(tokens, channels, device=DEVICE, dtype=torch.float64)
    live, alive = stories, []
    for t in range(max(lengths)):
        while lengths[order[live - 1]] <= t:
            live -= 1
        alive.append(live)
        rows = begin[:live] + t
        h[:live] = at(rows) * h[:live] + x[rows]
        states[rows] = h[:live]
    back = torch.empty_like(h)
    back[torch.tensor(order, device=DEVICE)] = h
    out = {"states": states, "final": back}
    if case["kind"] == "scan":
        return out
    g = s["grad_states"].double()
    m = s["grad_final"].double()[torch.tensor(order, device=DEVICE)]
    s0 = start[torch.tensor(order, device=DEVICE)]
    slope = torch.empty_like(states)
    grad_decay = torch.empty_like(states) if a.dim() == 2 else torch.zeros(channels, device=DEVICE,
                                                                           dtype=torch.float64)
    for t in reversed(range(len(alive))):
        live = alive[t]
        rows = begin[:live] + t
        lam = g[rows] + m[:live]
        slope[rows] = lam
        term = lam * (states[rows - 1] if t else s0[:live])
        if a.dim() == 2:
            grad_decay[rows] = term
        else:
            grad_decay += term.sum(0)
        m[:live] = at(rows) * lam
    out["grad_drive"], out["grad_decay"] = slope, grad_decay
    if s["initial"] is not None:
        out["grad_initial"] = torch.empty_like(m)
        out["grad_initial"][torch.tensor(order, device=DEVICE)] = m
    return out


def _exact_mask(s, r, vocabulary):
    if s["allowed"] is None or int(s["state"][r]) < 0:
        return None
    words = s["allowed"][int(s["state"][r])].long() & 0xFFFFFFFF
    v = torch.arange(vocabulary, device=DEVICE)
    return (words[v // 32] >> (v % 32)) % 2 == 1


def _exact_adjusted(s, r):
    z = s["logits"][r].double()
    spoken = s["history"][r, : int(s["lengths"][r])].long()
    count = torch.bincount(spoken, minlength=z.numel()).double()
    rho, presence, frequency = (s[k][r].double() for k in ("repetition", "presence", "frequency"))
    penalised = torch.where(z > 0, z / rho, z * rho) - (presence + frequency * count)
    z = torch.where(count > 0, penalised, z)
    if s["bias"] is not None:
        z = z + (s["bias"] if s["bias"].dim() == 1 else s["bias"][r]).double()
    ok = _exact_mask(s, r, z.numel())
    return z if ok is None else z.masked_fill(~ok, -math.inf)


def _exact_loss(s):
    """Every row at once, one grammar state after another."""
    logits, targets = s["logits"], s["targets"].long()
    rows, vocabulary = logits.shape
    losses = torch.zeros(rows, device=DEVICE, dtype=torch.float64)
    gradient = torch.zeros(rows, vocabulary, device=DEVICE, dtype=torch.float64)
    states = [-1] if s["allowed"] is None else range(-1, s["allowed"].shape[0])
    for k in states:
        rows_k = torch.nonzero((targets >= 0) if s["allowed"] is None else (targets >= 0) & (s["state"] == k))[:, 0]
        if not len(rows_k):
            continue
        ok = None if k < 0 else _exact_mask(s, int(rows_k[0]), vocabulary)
        at = torch.arange(vocabulary, device=DEVICE) if ok is None else torch.nonzero(ok)[:, 0]
        log_p = torch.log_softmax(logits[rows_k][:, at].double(), 1)
        place = torch.full((vocabulary,), -1, device=DEVICE)
        place[at] = torch.arange(len(at), device=DEVICE)
        hit = place[targets[rows_k]]
        line = torch.arange(len(rows_k), device=DEVICE)
        losses[rows_k] = -log_p[line, hit]
        p = torch.exp(log_p)
        p[line, hit] -= 1.0
        gradient[rows_k[:, None], at] = p * s["weights"][rows_k].double()[:, None]
    return {"losses": losses, "gradient": gradient}


def exact(case, seed):
    kind = case["kind"]
    if kind in ("scan", "train") and case["tokens"] > 70_000 * case["stories"]:
        return None  # a step at a time takes too long
    s = prepare(case, seed)
    if kind in ("scan", "train"):
        return _exact_scan(case, s)
    if kind == "step":
        h = s["decay"].double() * s["state"].double() + s["drive"].double()
        return {"states": h, "state": h}
    if kind == "loss":
        return _exact_loss(s)
    rows = case["rows"]
    if kind == "adjust":
        return {"logits": torch.stack([_exact_adjusted(s, r) for r in range(rows)])}
    symbols, chances = [], []
    for r in range(rows):
        z = _exact_adjusted(s, r)
        heat = float(s["temperature"][r])
        log_p = torch.log_softmax(z / heat if heat else z, 0)
        if heat:
            u = float(s["uniforms"][r])
            symbol = int(torch.searchsorted(torch.cumsum(torch.exp(log_p), 0), u, right=True))
            symbol = min(symbol, z.numel() - 1)
        else:
            symbol = int(torch.nonzero(z == z.max())[0, 0])
        symbols.append(symbol)
        chances.append(log_p[symbol])
    return {"symbols": torch.tensor(symbols, device=DEVICE, dtype=torch.int32),
            "log_probability": torch.stack(chances)}

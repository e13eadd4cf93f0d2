"""The measured calls of the selective state space layer's operators.

The selective scan over prompts and training batches, the short causal
convolution before it, both as steps of single tokens, and the root-mean-square
norm with the residual's addition and an 8-bit form of its result.  Each case is
one pass at sizes that programs use: the 125M model's training batch (B16 T1024,
width 768, inner width 1536), the decode configuration's 2,048 requests, and
ragged, narrow or long ones.  Training cases run forward and backward and return
the outputs and every gradient.  ``draw`` gives further cases of the same kinds.

With ``own`` false the operators run in their plain form: products, sums and
indexing of torch in float32, rounded once at the end (the recurrence by
doubling: log2(T) rounds over all tokens at once).  ``exact`` restates them in
float64 from their definitions, the recurrence token by token both ways.
"""

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
E4M3_MAX = 448.0
OTHER = 64  # what a projection's rows hold beside the part that is used


def listed():
    return [
        # One request's prompt at the 125M layer's inner width: few sequences.
        dict(name="scan_prompt", kind="scan", train=False, batch=1, time=2000, channels=1536,
             groups=1, states=16, dtype="bfloat16", gate=True, softplus=True, skip=True,
             initial=False, ragged=False),
        # One long document's prompt: the largest forward pass.
        dict(name="scan_long", kind="scan", train=False, batch=1, time=32768, channels=2048,
             groups=1, states=16, dtype="bfloat16", gate=True, softplus=True, skip=True,
             initial=False, ragged=False),
        # The 125M bfloat16 model's layer, trained.
        dict(name="scan_train_bf16", kind="scan", train=True, batch=16, time=1024, channels=1536,
             groups=1, states=16, dtype="bfloat16", gate=True, softplus=True, skip=True,
             initial=False, ragged=False),
        # A float32 training step over padded sequences of odd lengths that carry
        # a state from the step before, four groups of input and output weights.
        dict(name="scan_train_f32", kind="scan", train=True, batch=8, time=1000, channels=768,
             groups=4, states=16, dtype="float32", gate=True, softplus=True, skip=True,
             initial=True, ragged=True),
        # One token for a handful of requests, the state returned as a new one.
        dict(name="scan_step_small", kind="scan_step", in_place=False, batch=4, channels=1536,
             groups=1, states=16, dtype="bfloat16", gate=True, softplus=True, skip=True,
             idle=False),
        # One token for 2,048 resident requests, some of them idle, in place.
        dict(name="scan_step_large", kind="scan_step", in_place=True, batch=2048, channels=1536,
             groups=1, states=16, dtype="bfloat16", gate=True, softplus=True, skip=True,
             idle=True),
        # The convolution before the trained layer's scan.
        dict(name="conv_train_bf16", kind="conv", train=True, batch=16, time=1024, channels=1536,
             width=4, dtype="bfloat16", bias=True, activation="silu", initial=False,
             ragged=False),
        # The same of the float32 step over padded sequences that are continued.
        dict(name="conv_train_f32", kind="conv", train=True, batch=8, time=1000, channels=768,
             width=4, dtype="float32", bias=True, activation="silu", initial=True, ragged=True),
        # One token for 2,048 resident requests, the last tokens shifted in place.
        dict(name="conv_step_large", kind="conv_step", in_place=True, batch=2048, channels=1536,
             width=4, dtype="bfloat16", bias=True, activation="silu", idle=True),
        # The norm of a decode step of four requests: latency only.
        dict(name="norm_small", kind="norm", train=False, rows=4, channels=768, dtype="bfloat16",
             residual="bfloat16", weight=True),
        # The norm before a trained layer, over a float32 residual stream.
        dict(name="norm_train_bf16", kind="norm", train=True, rows=16384, channels=768,
             dtype="bfloat16", residual="float32", weight=True),
        # The norm of a large prompt batch before a product in 8 bits, a scale for
        # each 128 channels: the largest rows.
        dict(name="norm_8bit", kind="norm_8bit", rows=16384, channels=4096, dtype="bfloat16",
             residual="bfloat16", weight=True, block=128),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def _channels(rng):
    return rng.choice([768, 1536, 2048, rng.randint(1, 64), rng.randint(65, 2048)])


def _grouped(rng):
    """Channels, and the groups of them that share their weights."""
    groups = rng.choice([1, 1, 1, 2, 4, rng.randint(2, 12)])
    return max(1, _channels(rng) // groups) * groups, groups


def draw(rng):
    kind = rng.choice(["scan"] * 5 + ["scan_step", "conv", "conv", "conv_step", "norm", "norm",
                                      "norm_8bit"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16"])
    if kind in ("scan", "scan_step"):
        channels, groups = _grouped(rng)
        states = rng.choice([16, 16, 16, 8, rng.randint(1, 64)])
        some = dict(channels=channels, groups=groups, states=states, dtype=dtype,
                    gate=rng.random() < 0.7, softplus=rng.random() < 0.7,
                    skip=rng.random() < 0.7)
        if kind == "scan_step":
            limit = 2048 * 1536 * 16 // (channels * states)
            return dict(kind=kind, in_place=rng.random() < 0.5,
                        batch=_log(rng, 1, min(2048, limit)), idle=rng.random() < 0.4, **some)
        train = rng.random() < 0.6
        # State updates of the listed training step and of the long prompt.
        limit = (16 * 1024 * 1536 * 16 if train else 32768 * 2048 * 16) // (channels * states)
        time = _log(rng, 1, min(limit, 8192 if train else 32768))
        return dict(kind=kind, train=train, batch=_log(rng, 1, min(64, limit // time)), time=time,
                    initial=rng.random() < 0.4, ragged=rng.random() < 0.3, **some)
    if kind in ("conv", "conv_step"):
        channels = _channels(rng)
        some = dict(channels=channels, width=rng.choice([4, 4, 3, 2, rng.randint(1, 8)]),
                    dtype=dtype, bias=rng.random() < 0.8,
                    activation=rng.choice(["silu", "silu", "none"]))
        if kind == "conv_step":
            return dict(kind=kind, in_place=rng.random() < 0.5, batch=_log(rng, 1, 2048),
                        idle=rng.random() < 0.4, **some)
        limit = 16 * 1024 * 1536 // channels
        time = _log(rng, 1, min(limit, 32768))
        return dict(kind=kind, train=rng.random() < 0.7, batch=_log(rng, 1, min(64, limit // time)),
                    time=time, initial=rng.random() < 0.4, ragged=rng.random() < 0.3, **some)
    channels = rng.choice([768, 1536, 2048, 4096, rng.randint(1, 300), rng.randint(301, 8192)])
    rows = _log(rng, 1, min(16384, 16384 * 4096 // channels))
    some = dict(rows=rows, channels=channels, dtype=dtype, weight=rng.random() < 0.8,
                residual=rng.choice(["none", "float32", "bfloat16", dtype]))
    if kind == "norm_8bit":
        return dict(kind=kind, block=rng.choice([0, 32, 64, 128, 128, 256]), **some)
    return dict(kind=kind, train=rng.random() < 0.7, **some)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


class _Draw:
    """Seeded device tensors in a fixed order."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(int(seed))

    def normal(self, *shape, mean=0.0, scale=1.0):
        return torch.randn(*shape, device=DEVICE, generator=self.gen) * scale + mean

    def uniform(self, low, high, *shape):
        return torch.rand(*shape, device=DEVICE, generator=self.gen) * (high - low) + low

    def integers(self, low, high, *shape):
        return torch.randint(low, high, shape, device=DEVICE, generator=self.gen)


def _dtype(name):
    return torch.bfloat16 if name == "bfloat16" else torch.float32


def _lengths(g, batch, time):
    """Every length from an empty row to a full one; at least one is full."""
    lengths = g.integers(0, time + 1, batch)
    lengths[g.integers(0, batch, 1)] = time
    return lengths.to(torch.int32)


def _scan_inputs(case, seed):
    """The scan's inputs over sequences, or of one token each for a step."""
    g = _Draw(seed)
    lead = (case["batch"],) if case["kind"] == "scan_step" else (case["batch"], case["time"])
    d, groups, n = case["channels"], case["groups"], case["states"]
    dt = _dtype(case["dtype"])
    # The gate, and B and C, are parts of the rows of wider projections.
    inner = g.normal(*lead, OTHER + d).to(dt)
    small = g.normal(*lead, OTHER + 2 * groups * n).to(dt)
    b, c = (t.unflatten(-1, (groups, n)) for t in small[..., OTHER:].split(groups * n, -1))
    steps = torch.exp(g.uniform(math.log(1e-3), math.log(1e-1), d))
    if case["softplus"]:
        delta = g.normal(*lead, d, scale=0.5).to(dt)
    else:
        delta = (steps * torch.exp(g.normal(*lead, d, scale=0.5))).to(dt)
    ladder = torch.arange(1, n + 1, device=DEVICE, dtype=torch.float32)
    x = dict(x=g.normal(*lead, d).to(dt), delta=delta, a=-ladder * g.uniform(0.8, 1.2, d, n),
             b=b, c=c)
    if case["skip"]:
        x["skip"] = g.normal(d, mean=1.0, scale=0.2)
    if case["gate"]:
        x["gate"] = inner[..., OTHER:]
    if case["softplus"]:
        # The inverse of softplus at steps between 0.001 and 0.1.
        x["delta_bias"] = steps + torch.log(-torch.expm1(-steps))
    fixed, cot = {}, {}
    if case["kind"] == "scan_step":
        x["state"] = g.normal(*lead, d, n, scale=0.3)
        if case["idle"]:
            fixed["active"] = g.uniform(0.0, 1.0, *lead) < 0.9
        return x, fixed, cot
    if case["initial"]:
        x["initial"] = g.normal(case["batch"], d, n, scale=0.3)
    if case["ragged"]:
        fixed["lengths"] = _lengths(g, *lead)
    if case["train"]:
        cot["output"] = g.normal(*lead, d).to(dt)
        if case["initial"]:
            cot["state"] = g.normal(case["batch"], d, n, scale=0.3)
    return x, fixed, cot


def _conv_inputs(case, seed):
    g = _Draw(seed)
    lead = (case["batch"],) if case["kind"] == "conv_step" else (case["batch"], case["time"])
    d, w = case["channels"], case["width"]
    dt = _dtype(case["dtype"])
    # A part of the rows of a wider projection.
    x = dict(x=g.normal(*lead, d + OTHER).to(dt)[..., :d],
             weight=g.uniform(-1.0, 1.0, d, w) * w**-0.5)
    if case["bias"]:
        x["bias"] = g.uniform(-1.0, 1.0, d) * w**-0.5
    fixed, cot = {}, {}
    if case["kind"] == "conv_step":
        x["state"] = g.normal(case["batch"], w - 1, d).to(dt)
        if case["idle"]:
            fixed["active"] = g.uniform(0.0, 1.0, *lead) < 0.9
        return x, fixed, cot
    if case["initial"]:
        x["initial"] = g.normal(case["batch"], w - 1, d).to(dt)
    if case["ragged"]:
        fixed["lengths"] = _lengths(g, *lead)
    if case["train"]:
        cot["output"] = g.normal(*lead, d).to(dt)
    return x, fixed, cot


def _norm_inputs(case, seed):
    g = _Draw(seed)
    m, c = case["rows"], case["channels"]
    dt = _dtype(case["dtype"])
    x = dict(x=g.normal(m, c).to(dt))
    if case["weight"]:
        x["weight"] = g.uniform(0.5, 1.5, c)
    cot = {}
    if case["residual"] != "none":
        x["residual"] = g.normal(m, c, scale=2.0).to(_dtype(case["residual"]))
    if case.get("train"):
        cot["output"] = g.normal(m, c).to(dt)
        if "residual" in x:
            cot["sum"] = g.normal(m, c).to(x["residual"].dtype)
    return x, {}, cot


def _inputs(case, seed):
    if case["kind"].startswith("scan"):
        return _scan_inputs(case, seed)
    if case["kind"].startswith("conv"):
        return _conv_inputs(case, seed)
    return _norm_inputs(case, seed)


def prepare(case, seed):
    x, fixed, cot = _inputs(case, seed)
    if case.get("train"):
        for t in x.values():
            t.requires_grad_(True)
    return dict(case=case, x=x, fixed=fixed, cot=cot)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _plain_silu(z):
    return z / (1.0 + torch.exp(-z))


def _plain_silu_slope(z):
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain_softplus(z):
    return torch.clamp(z, min=0.0) + torch.log1p(torch.exp(-z.abs()))


def _doubling(a, u):
    """h_t = a_t h_{t-1} + u_t along axis 1, in place: after a round, the a and u of
    a token hold what its last 2, 4, ... tokens do."""
    gap = 1
    while gap < a.shape[1]:
        u[:, gap:] += a[:, gap:] * u[:, :-gap]
        a[:, gap:] = a[:, gap:] * a[:, :-gap]
        gap *= 2
    return u


def _over_channels(t, groups, channels):
    """[B,T,G,N] -> [B,T,channels,N]: what each channel of the groups given reads."""
    return t[:, :, groups] if t.shape[2] > 1 else t.expand(-1, -1, channels, -1)


def _plain_scan_part(case, x, present, cot, span, groups):
    """Some channels' outputs, and of all channels the gradients too."""
    here = {n: (t[..., span] if n in ("x", "delta", "gate", "skip", "delta_bias") else t)
            for n, t in x.items()}
    xs, delta = here["x"].float(), here["delta"].float()
    a = here["a"][span].float()
    d = a.shape[0]
    b, c = (_over_channels(here[n].float(), groups, d) for n in ("b", "c"))
    raw = delta + here["delta_bias"] if case["softplus"] else delta
    step = _plain_softplus(raw) if case["softplus"] else raw
    if present is not None:
        zero = torch.zeros_like(step)
        step, xs = torch.where(present, step, zero), torch.where(present, xs, zero)
        b, c = (torch.where(present[..., None], t, torch.zeros_like(t)) for t in (b, c))
    keep = torch.exp(step[..., None] * a)
    u = (step * xs)[..., None] * b
    start = here["initial"][:, span] if "initial" in here else None
    if start is not None:
        u[:, 0] += keep[:, 0] * start
    h = _doubling(keep.clone(), u)
    y = (h * c).sum(-1)
    if "skip" in here:
        y = y + here["skip"] * xs
    gate = here["gate"].float() if "gate" in here else None
    out = y if gate is None else y * _plain_silu(gate)
    if present is not None:
        out = torch.where(present, out, torch.zeros_like(out))
    dt = x["x"].dtype
    r = dict(output=out.to(dt), state=h[:, -1].clone())
    if not cot:
        return r
    dout = cot["output"][..., span].float()
    if present is not None:
        dout = torch.where(present, dout, torch.zeros_like(dout))
    dy = dout if gate is None else dout * _plain_silu(gate)
    if gate is not None:
        d_gate = dout * y * _plain_silu_slope(gate)
        r["d_gate"] = (d_gate if present is None
                       else torch.where(present, d_gate, torch.zeros_like(d_gate))).to(dt)
    # The recurrence of the states' cotangents, in reversed time.
    g = (dy[..., None] * c).flip(1)
    if "state" in cot:
        g[:, 0] += cot["state"][:, span]
    back = torch.cat([torch.ones_like(keep[:, :1]), keep[:, 1:].flip(1)], dim=1)
    g = _doubling(back, g).flip(1)
    before = torch.empty_like(h)
    before[:, 1:] = h[:, :-1]
    before[:, 0] = 0.0 if start is None else start
    shape = (case["groups"], -1)
    r["d_c"] = (h * dy[..., None]).unflatten(2, shape).sum(3).to(dt)
    r["d_b"] = (g * (step * xs)[..., None]).unflatten(2, shape).sum(3).to(dt)
    into = (g * b).sum(-1)
    rate = g * keep * before
    d_step = xs * into + (rate * a).sum(-1)
    d_x = step * into + (here["skip"] * dy if "skip" in here else 0.0)
    r["d_x"] = d_x.to(dt)
    r["d_a"] = (rate * step[..., None]).sum((0, 1))
    if "skip" in here:
        r["d_skip"] = (dy * xs).sum((0, 1))
    if case["softplus"]:
        d_step = d_step / (1.0 + torch.exp(-raw))
        if present is not None:
            d_step = torch.where(present, d_step, torch.zeros_like(d_step))
        r["d_delta_bias"] = d_step.sum((0, 1))
    elif present is not None:
        d_step = torch.where(present, d_step, torch.zeros_like(d_step))
    r["d_delta"] = d_step.to(dt)
    if start is not None:
        r["d_initial"] = keep[:, 0] * g[:, 0]
    return r


def _plain_scan(case, x, lengths, cot):
    batch, time, d = x["x"].shape
    groups, each = case["groups"], case["channels"] // case["groups"]
    present = None
    if lengths is not None:
        present = (torch.arange(time, device=DEVICE) < lengths[:, None])[..., None]
    of = torch.arange(d, device=DEVICE) // each
    # As many channels at once as keep an array of all states within 4 GiB (all of
    # them in training).
    most = d if cot else max(1, (1 << 30) // (batch * time * case["states"]))
    parts = [_plain_scan_part(case, x, present, cot, slice(i, i + most), of[i:i + most])
             for i in range(0, d, most)]
    if len(parts) == 1:
        return parts[0]
    return dict(output=torch.cat([r["output"] for r in parts], dim=2),
                state=torch.cat([r["state"] for r in parts], dim=1))


def _plain_scan_step(case, x, active):
    of = torch.arange(case["channels"], device=DEVICE) // (case["channels"] // case["groups"])
    xs, delta = x["x"].float(), x["delta"].float()
    b, c = (x[n].float()[:, of] for n in ("b", "c"))
    step = _plain_softplus(delta + x["delta_bias"]) if case["softplus"] else delta
    state = torch.exp(step[..., None] * x["a"]) * x["state"] + (step * xs)[..., None] * b
    y = (state * c).sum(-1)
    if "skip" in x:
        y = y + x["skip"] * xs
    if "gate" in x:
        y = y * _plain_silu(x["gate"].float())
    if active is not None:
        y = torch.where(active[:, None], y, torch.zeros_like(y))
        state = torch.where(active[:, None, None], state, x["state"])
    if case["in_place"]:
        state = x["state"].copy_(state)
    return dict(output=y.to(x["x"].dtype), state=state)


def _plain_conv(case, x, lengths):
    xs, w = x["x"].float(), x["weight"].float()
    batch, time, d = xs.shape
    width = case["width"]
    before = x["initial"].float() if "initial" in x else xs.new_zeros(batch, width - 1, d)
    rows = torch.cat([before, xs], dim=1)
    z = rows[:, :time] * w[:, 0]
    for j in range(1, width):
        z = z + rows[:, j:j + time] * w[:, j]
    if "bias" in x:
        z = z + x["bias"]
    y = _plain_silu(z) if case["activation"] == "silu" else z
    if lengths is None:
        state = rows[:, time:]
    else:
        present = (torch.arange(time, device=DEVICE) < lengths[:, None])[..., None]
        y = torch.where(present, y, torch.zeros_like(y))
        last = lengths.long()[:, None] + torch.arange(width - 1, device=DEVICE)
        state = torch.gather(rows, 1, last[..., None].expand(-1, -1, d))
    return dict(output=y.to(x["x"].dtype), state=state.to(x["x"].dtype))


def _plain_conv_step(case, x, active):
    rows = torch.cat([x["state"], x["x"][:, None]], dim=1)
    z = (rows.float() * x["weight"].float().t()).sum(1)
    if "bias" in x:
        z = z + x["bias"]
    y = _plain_silu(z) if case["activation"] == "silu" else z
    state = rows[:, 1:]
    if active is not None:
        y = torch.where(active[:, None], y, torch.zeros_like(y))
        state = torch.where(active[:, None, None], state, x["state"])
    if case["in_place"]:
        state = x["state"].copy_(state)
    return dict(output=y.to(x["x"].dtype), state=state)


def _plain_norm(x):
    total = x["x"].float()
    if "residual" in x:
        total = (total + x["residual"].float()).to(x["residual"].dtype)
    s = total.float()
    y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS)
    if "weight" in x:
        y = y * x["weight"]
    return y, total


def _plain_norm_8bit(case, x):
    y, total = _plain_norm(x)
    m, c = y.shape
    block = case["block"] or c
    blocks = -(-c // block)
    parts = torch.cat([y, y.new_zeros(m, blocks * block - c)], -1).reshape(m, blocks, block)
    scale = torch.clamp(parts.abs().amax(-1) / E4M3_MAX, min=2.0**-126)
    q = (parts / scale[..., None]).to(torch.float8_e4m3fn).reshape(m, -1)[:, :c]
    r = dict(output=q, scale=scale)
    if "residual" in x:
        r["sum"] = total
    return r


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

_OPTIONS = ("skip", "gate", "delta_bias")


def _scan(case, x, fixed):
    from mamba4_amd import selective_scan

    r = selective_scan(x["x"], x["delta"], x["a"], x["b"], x["c"],
                       **{n: x.get(n) for n in _OPTIONS}, softplus=case["softplus"],
                       initial=x.get("initial"), lengths=fixed.get("lengths"))
    return dict(output=r.output, state=r.state)


def _scan_step(case, x, fixed):
    if not own:
        return _plain_scan_step(case, x, fixed.get("active"))
    from mamba4_amd import selective_scan_step, selective_scan_step_

    step = selective_scan_step_ if case["in_place"] else selective_scan_step
    r = step(x["state"], x["x"], x["delta"], x["a"], x["b"], x["c"],
             **{n: x.get(n) for n in _OPTIONS}, softplus=case["softplus"],
             active=fixed.get("active"))
    return dict(output=r.output, state=r.state)


def _conv(case, x, fixed):
    if not own:
        return _plain_conv(case, x, fixed.get("lengths"))
    from mamba4_amd import causal_conv

    r = causal_conv(x["x"], x["weight"], x.get("bias"), activation=case["activation"],
                    initial=x.get("initial"), lengths=fixed.get("lengths"))
    return dict(output=r.output, state=r.state)


def _conv_step(case, x, fixed):
    if not own:
        return _plain_conv_step(case, x, fixed.get("active"))
    from mamba4_amd import causal_conv_step, causal_conv_step_

    step = causal_conv_step_ if case["in_place"] else causal_conv_step
    r = step(x["state"], x["x"], x["weight"], x.get("bias"), activation=case["activation"],
             active=fixed.get("active"))
    return dict(output=r.output, state=r.state)


def _norm(case, x, fixed):
    if not own:
        y, total = _plain_norm(x)
        r = dict(output=y.to(x["x"].dtype))
    else:
        from mamba4_amd import rms_norm

        y, total = rms_norm(x["x"], x.get("weight"), residual=x.get("residual"), eps=EPS)
        r = dict(output=y)
    if "residual" in x:
        r["sum"] = total
    return r


def _norm_8bit(case, x, fixed):
    if not own:
        return _plain_norm_8bit(case, x)
    from mamba4_amd import rms_norm_e4m3

    q, scale, total = rms_norm_e4m3(x["x"], x.get("weight"), residual=x.get("residual"), eps=EPS,
                                    block=case["block"] or None)
    r = dict(output=q, scale=scale)
    if "residual" in x:
        r["sum"] = total
    return r


_CALLS = dict(scan=_scan, scan_step=_scan_step, conv=_conv, conv_step=_conv_step, norm=_norm,
              norm_8bit=_norm_8bit)


def _differentiate(call, x, cot):
    """The call's outputs and the gradient of every input from the cotangents."""
    out = call(x)
    grads = torch.autograd.grad([out[n] for n in cot], list(x.values()), list(cot.values()))
    out = {n: t.detach() for n, t in out.items()}
    out.update({"d_" + n: g for n, g in zip(x, grads)})
    return out


def run(state):
    case, x, fixed, cot = state["case"], state["x"], state["fixed"], state["cot"]
    if case["kind"] == "scan" and not own:
        with torch.no_grad():
            return _plain_scan(case, x, fixed.get("lengths"), cot)
    call = _CALLS[case["kind"]]
    if case.get("train"):
        return _differentiate(lambda y: call(case, y, fixed), x, cot)
    with torch.no_grad():
        return call(case, x, fixed)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    """Inputs read once, outputs written once, and the operators' own arithmetic
    (a state's update and its part of the result: 7 operations forward, 17 back)."""
    kind, row = case["kind"], (2 if case["dtype"] == "bfloat16" else 4)
    if kind.startswith("norm"):
        m, c = case["rows"], case["channels"]
        other = dict(none=0, float32=4, bfloat16=2)[case["residual"]]
        if kind == "norm_8bit":
            blocks = -(-c // (case["block"] or c))
            return dict(bytes=m * (c * (row + 2 * other + 1) + 4 * blocks) + 4 * c, flops=7 * m * c)
        moved, flops = m * c * (2 * row + 2 * other) + 4 * c, 6 * m * c
        if case["train"]:
            # Back: the sum (or x), the cotangents read, the gradients written.
            moved += m * c * (2 * row + 3 * other if other else 3 * row) + 8 * c
            flops += 12 * m * c
        return dict(bytes=moved, flops=flops)
    tokens = case["batch"] * case.get("time", 1)
    d = case["channels"]
    rows = tokens * d * row
    if kind.startswith("conv"):
        w = case["width"]
        parameters = 4 * d * (w + 1)
        state = case["batch"] * (w - 1) * d * row
        if kind == "conv_step":
            return dict(bytes=2 * rows + 2 * state + parameters, flops=tokens * d * (2 * w + 4))
        start = state if case["initial"] else 0
        moved, flops = 2 * rows + state + start + parameters, tokens * d * (2 * w + 4)
        if case["train"]:
            moved += 3 * rows + 2 * start + 2 * parameters
            flops += tokens * d * (6 * w + 8)
        return dict(bytes=moved, flops=flops)
    n = case["states"]
    arrays = 3 + (1 if case["gate"] else 0)
    parameters = 4 * d * (n + (1 if case["skip"] else 0) + (1 if case["softplus"] else 0))
    weights = 2 * tokens * case["groups"] * n * row
    state = 4 * case["batch"] * d * n
    updates = tokens * d * n
    if kind == "scan_step":
        return dict(bytes=arrays * rows + weights + parameters + 2 * state, flops=7 * updates)
    moved = arrays * rows + weights + parameters + state * (2 if case["initial"] else 1)
    if not case["train"]:
        return dict(bytes=moved, flops=7 * updates)
    # Back: the inputs and the output's cotangent read, the gradients written.
    moved += (2 * arrays - 1) * rows + 2 * weights + 2 * parameters
    moved += 3 * state if case["initial"] else 0
    return dict(bytes=moved, flops=24 * updates)


# ---------------------------------------------------------------------------
# The operators in float64
# ---------------------------------------------------------------------------


def _double(x):
    return {n: t.detach().double() for n, t in x.items()}


def _silu64(z):
    return z * torch.sigmoid(z)


def _token64(case, x, t):
    """Token t's step, decay and inflow, and its b and c, of every channel."""
    each = case["channels"] // case["groups"]
    raw = x["delta"][:, t]
    if case["softplus"]:
        raw = raw + x["delta_bias"]
        step = torch.logaddexp(raw, torch.zeros_like(raw))
    else:
        step = raw
    b, c = (x[n][:, t].repeat_interleave(each, dim=1) for n in ("b", "c"))
    return raw, step, torch.exp(step[..., None] * x["a"]), b, c


def _scan64(case, x, lengths, cot):
    """Token by token, and back again."""
    batch, time, d = x["x"].shape
    n = case["states"]
    h = x["initial"] if "initial" in x else x["x"].new_zeros(batch, d, n)
    out = torch.zeros_like(x["x"])
    here = None if lengths is None else torch.arange(time, device=DEVICE)[:, None] < lengths
    kept = h.new_empty(time, batch, d, n) if cot else None
    inner = torch.zeros_like(out) if cot else None
    for t in range(time):
        if cot:
            kept[t] = h
        _, step, keep, b, c = _token64(case, x, t)
        new = torch.addcmul(keep * h, (step * x["x"][:, t])[..., None], b)
        y = torch.matmul(new[..., None, :], c[..., None])[..., 0, 0]
        if "skip" in x:
            y = torch.addcmul(y, x["skip"], x["x"][:, t])
        if here is not None:
            new = torch.where(here[t][:, None, None], new, h)
            y = y * here[t][:, None]
        h = new
        if cot:
            inner[:, t] = y
        out[:, t] = y * _silu64(x["gate"][:, t]) if "gate" in x else y
    r = dict(output=out, state=h)
    if not cot:
        return r
    grads = {m: torch.zeros_like(t) for m, t in x.items()}
    g = cot["state"].clone() if "state" in cot else torch.zeros_like(h)
    groups = (batch, case["groups"], d // case["groups"], n)
    for t in reversed(range(time)):
        raw, step, keep, b, c = _token64(case, x, t)
        on = torch.ones(batch, 1, device=DEVICE, dtype=torch.double) if here is None \
            else here[t].double()[:, None]
        dy = cot["output"][:, t] * on
        if "gate" in x:
            z = x["gate"][:, t]
            s = torch.sigmoid(z)
            grads["gate"][:, t] = dy * inner[:, t] * (s + z * s * (1.0 - s))
            dy = dy * z * s
        if "skip" in x:
            grads["skip"] += (dy * x["x"][:, t]).sum(0)
        here_h = keep * kept[t] + (step * x["x"][:, t])[..., None] * b
        grads["c"][:, t] = (dy[..., None] * here_h).reshape(groups).sum(2)
        full = g + dy[..., None] * c
        flow = (full * b).sum(-1)
        on2 = on[..., None]
        grads["b"][:, t] = (on2 * full * (step * x["x"][:, t])[..., None]).reshape(groups).sum(2)
        rate = full * keep * kept[t] * on2
        grads["a"] += (rate * step[..., None]).sum(0)
        d_step = (flow * x["x"][:, t]) * on + (rate * x["a"]).sum(-1)
        grads["x"][:, t] = flow * step * on + (dy * x["skip"] if "skip" in x else 0.0)
        if case["softplus"]:
            d_step = d_step * torch.sigmoid(raw)
            grads["delta_bias"] += d_step.sum(0)
        grads["delta"][:, t] = d_step
        g = torch.where(on2 > 0, full * keep, g)
    if "initial" in x:
        grads["initial"] = g
    r.update({"d_" + m: t for m, t in grads.items()})
    return r


def _scan_step64(case, x, active):
    one = {n: (t if n in ("a", "skip", "delta_bias") else t[:, None])
           for n, t in x.items() if n != "state"}
    one["initial"] = x["state"]
    lengths = None if active is None else active.long()
    r = _scan64(dict(case, time=1), one, lengths, {})
    return dict(output=r["output"][:, 0], state=r["state"])


def _conv64(case, x, lengths):
    batch, time, d = x["x"].shape
    width = case["width"]
    start = x["initial"] if "initial" in x else x["x"].new_zeros(batch, width - 1, d)
    rows = torch.cat([start, x["x"]], dim=1)
    z = torch.matmul(rows.unfold(1, width, 1)[..., None, :], x["weight"][..., None])[..., 0, 0]
    if "bias" in x:
        z = z + x["bias"]
    y = _silu64(z) if case["activation"] == "silu" else z
    ends = torch.full((batch,), time, device=DEVICE) if lengths is None else lengths.long()
    y = y * (torch.arange(time, device=DEVICE)[None] < ends[:, None])[..., None]
    state = torch.stack([rows[i, e:e + width - 1] for i, e in enumerate(ends.tolist())])
    return dict(output=y, state=state)


def _conv_step64(case, x, active):
    z = torch.einsum("bwd,dw->bd", torch.cat([x["state"], x["x"][:, None]], 1), x["weight"])
    if "bias" in x:
        z = z + x["bias"]
    y = _silu64(z) if case["activation"] == "silu" else z
    state = torch.cat([x["state"], x["x"][:, None]], 1)[:, 1:]
    if active is not None:
        y = y * active[:, None]
        state = torch.where(active[:, None, None], state, x["state"])
    return dict(output=y, state=state)


def _norm64(case, x, dtype):
    """``dtype``: what the sum is rounded to before it is normalised."""
    total = x["x"] if "residual" not in x else x["x"] + x["residual"]
    rounded = total + (total.detach().to(dtype).double() - total.detach())
    y = rounded / torch.sqrt(rounded.square().sum(-1, keepdim=True) / case["channels"] + EPS)
    if "weight" in x:
        y = y * x["weight"]
    r = dict(output=y)
    if "residual" in x:
        r["sum"] = rounded
    return r


def _norm_8bit64(case, x, dtype):
    r = _norm64(case, x, dtype)
    y, c = r["output"], case["channels"]
    parts = torch.split(y, case["block"] or c, -1)
    scale = torch.stack([p.abs().max(-1).values for p in parts], -1) / E4M3_MAX
    scale = torch.clamp(scale, min=2.0**-126)
    r["output"] = torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(parts)], -1)
    r["scale"] = scale
    return r


def exact(case, seed):
    kind = case["kind"]
    x, fixed, cot = _inputs(case, seed)
    dtype = x["residual"].dtype if "residual" in x else torch.float64
    x, cot = _double(x), _double(cot)
    if kind == "scan":
        return _scan64(case, x, fixed.get("lengths"), cot)
    if kind == "scan_step":
        return _scan_step64(case, x, fixed.get("active"))
    if kind == "conv_step":
        return _conv_step64(case, x, fixed.get("active"))
    if kind == "norm_8bit":
        return _norm_8bit64(case, x, dtype)
    if kind == "conv":
        def call(y):
            return _conv64(case, y, fixed.get("lengths"))
    else:
        def call(y):
            return _norm64(case, y, dtype)
    if not case["train"]:
        return call(x)
    return _differentiate(call, {n: t.requires_grad_(True) for n, t in x.items()}, cot)

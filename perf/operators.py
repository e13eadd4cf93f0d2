"""The measured calls of the retention layer's operators.

Decayed linear attention over prompts and training batches, its step for
single tokens, group normalisation with an activation or a gate, and the scaled
embedding lookup with its gradient.  Each case is one pass at sizes that
programs use: the 125M model's layer shapes (B16 T1024, 12 heads of N64 P128),
the decode configuration of 2,048 requests by 8 heads, and ragged, narrow or
long ones.  Training cases run forward and backward and return the outputs and
every gradient.  ``draw`` gives further cases of the same kinds.

With ``own`` false the operators run in their plain form: chunked products,
sums and indexing of torch in float32, rounded once at the end.  ``exact`` restates
them in float64 from their definitions (the recurrence token by token, the
sums over all pairs of tokens).
"""

import math

import torch

own = False

DEVICE = "cuda"
CHUNK = 64


def listed():
    return [
        # One request's prompt at the 125M layer's shape: few sequences.
        dict(name="attention_prompt", kind="attention", train=False, batch=1, time=2000, heads=12,
             query_heads=12, key_heads=12, value_heads=12, key_dim=64, value_dim=128,
             dtype="bfloat16", decay="token", initial=False, ragged=False),
        # One long document's prompt with wide keys shared by four heads each:
        # the largest forward pass.
        dict(name="attention_long", kind="attention", train=False, batch=1, time=32768, heads=16,
             query_heads=16, key_heads=4, value_heads=16, key_dim=128, value_dim=128,
             dtype="bfloat16", decay="head", initial=False, ragged=False),
        # The 125M bfloat16 model's layer, trained, a decay for every token.
        dict(name="attention_train_bf16", kind="attention", train=True, batch=16, time=1024,
             heads=12, query_heads=12, key_heads=12, value_heads=12, key_dim=64, value_dim=128,
             dtype="bfloat16", decay="token", initial=False, ragged=False),
        # A float32 training step over padded sequences of odd lengths that
        # carry a state from the step before.
        dict(name="attention_train_f32", kind="attention", train=True, batch=8, time=1000, heads=8,
             query_heads=8, key_heads=8, value_heads=8, key_dim=64, value_dim=64,
             dtype="float32", decay="head", initial=True, ragged=True),
        # One token for a handful of requests, the state returned as a new one.
        dict(name="step_small", kind="step", in_place=False, batch=4, heads=12, query_heads=12,
             key_heads=12, value_heads=12, key_dim=64, value_dim=128, dtype="bfloat16",
             decay="token", idle=False),
        # One token for 2,048 resident requests, updated in place.
        dict(name="step_large", kind="step", in_place=True, batch=2048, heads=8, query_heads=8,
             key_heads=8, value_heads=8, key_dim=64, value_dim=64, dtype="float32",
             decay="token", idle=True),
        # The norm of a decode step's heads under its gate: latency only.
        dict(name="norm_small", kind="norm", train=False, samples=4, positions=1, channels=1536,
             groups=12, dtype="bfloat16", gate=True, affine=True, activation="silu"),
        # The norm of every token's heads under its gate, trained (B16 T1024,
        # 12 heads of 128).
        dict(name="norm_train_bf16", kind="norm", train=True, samples=16384, positions=1,
             channels=1536, groups=12, dtype="bfloat16", gate=True, affine=True,
             activation="silu"),
        # Frames of features normalised over their positions, trained.
        dict(name="norm_train_positions", kind="norm", train=True, samples=8, positions=4000,
             channels=512, groups=32, dtype="float32", gate=False, affine=True,
             activation="silu"),
        # The tokens of a decode step of 2,048 requests.
        dict(name="embedding_small", kind="embedding", train=False, tokens=2048, rows=32000,
             width=768, table="bfloat16", out="bfloat16", padded=False),
        # A training batch (B16 T1024), a float32 table under a bfloat16 model.
        dict(name="embedding_train", kind="embedding", train=True, tokens=16384, rows=32000,
             width=768, table="float32", out="bfloat16", padded=False),
        # A large batch of padded sequences over an odd vocabulary.
        dict(name="embedding_train_large", kind="embedding", train=True, tokens=131071,
             rows=50257, width=1024, table="bfloat16", out="bfloat16", padded=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def _heads(rng):
    """Heads, and the heads that the queries, keys and values have."""
    shared = rng.randint(1, 4)
    groups = rng.randint(1, 4)
    heads = shared * groups
    kind = rng.choice(["own", "own", "keys and values", "queries and keys"])
    if kind == "own":
        return heads, heads, heads, heads
    if kind == "keys and values":
        return heads, heads, groups, groups
    return heads, groups, groups, heads


def draw(rng):
    kind = rng.choice(["attention"] * 4 + ["step"] * 2 + ["norm"] * 3 + ["embedding"] * 2)
    if kind == "attention":
        train = rng.random() < 0.6
        heads, query_heads, key_heads, value_heads = _heads(rng)
        key_dim = rng.choice([64, 64, 128, rng.randint(16, 127)])
        value_dim = rng.choice([64, 64, 128, rng.randint(16, 127)])
        # Elements of the widest listed training step and of the long prompt.
        limit = (75_000_000 if train else 250_000_000) // (2 * heads * (key_dim + value_dim))
        time = _log(rng, 1, min(limit, 4096 if train else 32768))
        return dict(kind=kind, train=train, batch=_log(rng, 1, min(64, limit // time)), time=time,
                    heads=heads, query_heads=query_heads, key_heads=key_heads,
                    value_heads=value_heads, key_dim=key_dim, value_dim=value_dim,
                    dtype=rng.choice(["float32", "bfloat16", "bfloat16"]),
                    decay=rng.choice(["token", "head"]), initial=rng.random() < 0.4,
                    ragged=rng.random() < 0.3)
    if kind == "step":
        heads, query_heads, key_heads, value_heads = _heads(rng)
        key_dim = rng.choice([64, 64, 128, rng.randint(16, 127)])
        value_dim = rng.choice([64, 64, 128, rng.randint(16, 127)])
        limit = 2048 * 8 * 64 * 64 // (heads * key_dim * value_dim)
        return dict(kind=kind, in_place=rng.random() < 0.5, batch=_log(rng, 1, min(2048, limit)),
                    heads=heads, query_heads=query_heads, key_heads=key_heads,
                    value_heads=value_heads, key_dim=key_dim, value_dim=value_dim,
                    dtype=rng.choice(["float32", "bfloat16"]),
                    decay=rng.choice(["token", "head"]), idle=rng.random() < 0.3)
    if kind == "norm":
        groups = rng.choice([1, 12, 32, rng.randint(2, 24)])
        width = rng.choice([8, 16, 64, 64, 128, rng.randint(3, 130)])
        channels = groups * width
        limit = 16384 * 1536 // channels
        positions = rng.choice([1, 1, _log(rng, 2, min(limit, 8192))])
        return dict(kind=kind, train=rng.random() < 0.7,
                    samples=_log(rng, 1, min(16384, limit // positions)), positions=positions,
                    channels=channels, groups=groups,
                    dtype=rng.choice(["float32", "bfloat16", "bfloat16"]),
                    gate=rng.random() < 0.5, affine=rng.random() < 0.8,
                    activation=rng.choice(["none", "silu", "silu", "gelu"]))
    width = rng.choice([512, 768, 1024, rng.randint(30, 1100)])
    return dict(kind=kind, train=rng.random() < 0.7, tokens=_log(rng, 1, 131071),
                rows=_log(rng, 256, 50257), width=width,
                table=rng.choice(["float32", "bfloat16"]),
                out=rng.choice(["float32", "bfloat16"]), padded=rng.random() < 0.4)


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

    def unit(self, *shape):
        x = self.normal(*shape)
        return x / x.norm(dim=-1, keepdim=True)

    def integers(self, low, high, *shape):
        return torch.randint(low, high, shape, device=DEVICE, generator=self.gen)


def _dtype(name):
    return torch.bfloat16 if name == "bfloat16" else torch.float32


def _decay(g, case, *token_shape):
    """Log decays: a ladder of half-lives over the heads, or gates of every
    token and head around sigmoid(3)."""
    h = case["heads"]
    if case["decay"] == "head":
        ladder = torch.arange(h, device=DEVICE, dtype=torch.float32)
        rate = torch.exp2(-3.0 - 5.0 * ladder / max(1, h - 1)) * g.uniform(0.8, 1.2, h)
        return torch.log1p(-rate)
    logits = g.normal(*token_shape, h, mean=3.0)
    return torch.minimum(logits, torch.zeros_like(logits)) - torch.log1p(torch.exp(-logits.abs()))


def _attention_inputs(case, seed):
    g = _Draw(seed)
    b, t, h, n, p = (case[k] for k in ("batch", "time", "heads", "key_dim", "value_dim"))
    dt = _dtype(case["dtype"])
    x = dict(queries=g.unit(b, t, case["query_heads"], n).to(dt),
             keys=g.unit(b, t, case["key_heads"], n).to(dt),
             values=g.normal(b, t, case["value_heads"], p).to(dt),
             log_decay=_decay(g, case, b, t))
    if case["initial"]:
        x["initial"] = g.normal(b, h, n, p, scale=0.3)
    fixed = {}
    if case["ragged"]:
        # Every length from an empty row to a full one; at least one is full.
        lengths = g.integers(0, t + 1, b)
        lengths[g.integers(0, b, 1)] = t
        fixed["lengths"] = lengths.to(torch.int32)
    cot = {}
    if case["train"]:
        cot["output"] = g.normal(b, t, h, p).to(dt)
        if case["initial"]:
            cot["state"] = g.normal(b, h, n, p, scale=0.3)
    return x, fixed, cot


def _step_inputs(case, seed):
    g = _Draw(seed)
    b, h, n, p = (case[k] for k in ("batch", "heads", "key_dim", "value_dim"))
    dt = _dtype(case["dtype"])
    x = dict(state=g.normal(b, h, n, p, scale=0.3),
             query=g.unit(b, case["query_heads"], n).to(dt),
             key=g.unit(b, case["key_heads"], n).to(dt),
             value=g.normal(b, case["value_heads"], p).to(dt), log_decay=_decay(g, case, b))
    if case["idle"]:
        x["active"] = g.uniform(0.0, 1.0, b) < 0.9
    return x


def _norm_inputs(case, seed):
    g = _Draw(seed)
    m, s, c = case["samples"], case["positions"], case["channels"]
    shape = (m, c) if s == 1 else (m, s, c)
    dt = _dtype(case["dtype"])
    x = dict(x=g.normal(*shape, mean=0.3, scale=1.5).to(dt))
    if case["affine"]:
        x["weight"] = g.uniform(0.5, 1.5, c)
        x["bias"] = g.normal(c, scale=0.2)
    if case["gate"]:
        x["gate"] = g.normal(*shape).to(dt)
    return x, (dict(output=g.normal(*shape).to(dt)) if case["train"] else {})


def _embedding_inputs(case, seed):
    g = _Draw(seed)
    n, rows, c = case["tokens"], case["rows"], case["width"]
    table = g.normal(rows, c, scale=0.02).to(_dtype(case["table"]))
    # Text's frequencies: the rank r about proportionally to 1 / r.
    ranks = torch.exp(g.uniform(0.0, math.log(rows + 1.0), n)).long() - 1
    ids = torch.clamp(ranks, 0, rows - 1) * 48271 % rows
    if case["padded"]:
        ids = torch.where(g.uniform(0.0, 1.0, n) < 0.1, torch.full_like(ids, -1), ids)
    cot = dict(output=g.normal(n, c).to(_dtype(case["out"]))) if case["train"] else {}
    return dict(table=table), dict(ids=ids), cot


def prepare(case, seed):
    kind = case["kind"]
    fixed, cot = {}, {}
    if kind == "attention":
        x, fixed, cot = _attention_inputs(case, seed)
    elif kind == "step":
        x = _step_inputs(case, seed)
    elif kind == "norm":
        x, cot = _norm_inputs(case, seed)
    else:
        x, fixed, cot = _embedding_inputs(case, seed)
    if case.get("train"):
        for t in x.values():
            t.requires_grad_(True)
    return dict(case=case, x=x, fixed=fixed, cot=cot)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _spread(t, heads):
    """[..., h, W] -> [..., heads, W], each head repeated for those that share it."""
    return t if t.shape[-2] == heads else t.repeat_interleave(heads // t.shape[-2], dim=-2)


def _chunks(t, chunks):
    """[B,T,H,W] -> [B*H,chunks,64,W], zeros after the last token."""
    b, time, h, w = t.shape
    t = t.transpose(1, 2).reshape(b * h, time, w)
    if time < chunks * CHUNK:
        t = torch.cat([t, t.new_zeros(b * h, chunks * CHUNK - time, w)], dim=1)
    return t.reshape(b * h, chunks, CHUNK, w)


def _plain_attention(x, lengths):
    dtype = x["values"].dtype
    b, time = x["queries"].shape[:2]
    h = max(x[n].shape[2] for n in ("queries", "keys", "values"))
    n, p = x["keys"].shape[-1], x["values"].shape[-1]
    q, k, v = (_spread(x[m].float(), h) for m in ("queries", "keys", "values"))
    g = x["log_decay"].float().expand(b, time, h)[..., None]
    present = None
    if lengths is not None:
        present = (torch.arange(time, device=q.device) < lengths[:, None])[..., None, None]
        k, v, g = (torch.where(present, t, torch.zeros_like(t)) for t in (k, v, g))
    chunks = -(-time // CHUNK)
    q, k, v, g = (_chunks(t, chunks) for t in (q, k, v, g))
    prefix = torch.cumsum(g, dim=2)
    last = prefix[:, :, -1:]
    gap = prefix - prefix.transpose(2, 3)
    causal = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp(gap.masked_fill(~causal, -math.inf))
    out = torch.matmul(torch.matmul(q, k.transpose(2, 3)) * decay, v)
    local = torch.matmul((k * torch.exp(last - prefix)).transpose(2, 3), v)
    state = x["initial"].float().reshape(b * h, n, p) if "initial" in x \
        else q.new_zeros(b * h, n, p)
    carry = torch.exp(last)
    starts = []
    for c in range(chunks):
        starts.append(state)
        state = carry[:, c] * state + local[:, c]
    out = out + torch.exp(prefix) * torch.matmul(q, torch.stack(starts, dim=1))
    out = out.reshape(b, h, chunks * CHUNK, p)[:, :, :time].transpose(1, 2)
    out = out * _scale(n)
    if present is not None:
        out = torch.where(present, out, torch.zeros_like(out))
    return dict(output=out.to(dtype), state=state.reshape(b, h, n, p))


def _scale(key_dim):
    return key_dim ** -0.5


def _plain_step(case, x):
    h = case["heads"]
    q, k, v = (_spread(x[m].float(), h) for m in ("query", "key", "value"))
    lam = torch.exp(x["log_decay"].float()).expand(case["batch"], h)[..., None, None]
    state = lam * x["state"] + k[..., :, None] * v[..., None, :]
    out = (q[..., :, None] * state).sum(dim=-2) * _scale(case["key_dim"])
    if "active" in x:
        active = x["active"][:, None, None]
        out = torch.where(active, out, torch.zeros_like(out))
        state = torch.where(active[..., None], state, x["state"])
    if case["in_place"]:
        state = x["state"].copy_(state)
    return dict(output=out.to(x["value"].dtype), state=state)


def _plain_activation(z, name):
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _plain_norm(case, x):
    m, s, c, groups = (case[k] for k in ("samples", "positions", "channels", "groups"))
    t = x["x"].float().reshape(m, s, groups, c // groups)
    mean = t.mean(dim=(1, 3), keepdim=True)
    centred = t - mean
    variance = (centred * centred).mean(dim=(1, 3), keepdim=True)
    z = (centred * torch.rsqrt(variance + 1e-5)).reshape(x["x"].shape)
    if "weight" in x:
        z = z * x["weight"] + x["bias"]
    if "gate" in x:
        z = z * _plain_activation(x["gate"].float(), case["activation"])
    else:
        z = _plain_activation(z, case["activation"])
    return dict(output=z.to(x["x"].dtype))


def _plain_embedding(case, table, ids, cot):
    known = (ids >= 0) & (ids < case["rows"])
    safe = torch.where(known, ids, torch.zeros_like(ids))
    scale = math.sqrt(case["width"])
    rows = table[safe].float() * scale
    out = dict(output=torch.where(known[:, None], rows, torch.zeros_like(rows))
               .to(_dtype(case["out"])))
    if cot:
        d = cot["output"].float() * (known[:, None] * scale)
        grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
        out["d_table"] = grad.index_add_(0, safe, d).to(table.dtype)
    return out


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _attention(case, x, fixed):
    if not own:
        return _plain_attention(x, fixed.get("lengths"))
    from mamba4_amd import linear_attention

    r = linear_attention(x["queries"], x["keys"], x["values"], x["log_decay"],
                         initial=x.get("initial"), lengths=fixed.get("lengths"),
                         scale=_scale(case["key_dim"]))
    return dict(output=r.output, state=r.state)


def _step(case, x):
    if not own:
        return _plain_step(case, x)
    from mamba4_amd import linear_attention_step, linear_attention_step_

    step = linear_attention_step_ if case["in_place"] else linear_attention_step
    r = step(x["state"], x["query"], x["key"], x["value"], x["log_decay"],
             active=x.get("active"), scale=_scale(case["key_dim"]))
    return dict(output=r.output, state=r.state)


def _norm(case, x):
    if not own:
        return _plain_norm(case, x)
    from mamba4_amd import group_norm

    return dict(output=group_norm(x["x"], case["groups"], x.get("weight"), x.get("bias"),
                                  gate=x.get("gate"), activation=case["activation"], eps=1e-5))


def _embedding(case, x, fixed):
    from mamba4_amd import embedding

    return dict(output=embedding(fixed["ids"], x["table"], scale=math.sqrt(case["width"]),
                                 dtype=_dtype(case["out"])))


def _differentiate(call, x, cot):
    """The call's outputs and the gradient of every input from the cotangents."""
    out = call(x)
    grads = torch.autograd.grad([out[n] for n in cot], list(x.values()), list(cot.values()))
    out = {n: t.detach() for n, t in out.items()}
    out.update({"d_" + n: g for n, g in zip(x, grads)})
    return out


def run(state):
    case, x, fixed, cot = state["case"], state["x"], state["fixed"], state["cot"]
    kind = case["kind"]
    if kind == "step":
        return _step(case, x)
    if kind == "embedding" and not own:
        with torch.no_grad():
            return _plain_embedding(case, x["table"], fixed["ids"], cot)
    calls = dict(attention=lambda y: _attention(case, y, fixed), norm=lambda y: _norm(case, y),
                 embedding=lambda y: _embedding(case, y, fixed))
    if case["train"]:
        return _differentiate(calls[kind], x, cot)
    with torch.no_grad():
        return calls[kind](x)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    """Inputs read once, outputs written once, and the operators' own
    multiply-adds (the causal products of 64-token chunks and their states)."""
    kind = case["kind"]
    if kind in ("attention", "step"):
        b, t, h = case["batch"], case.get("time", 1), case["heads"]
        n, p = case["key_dim"], case["value_dim"]
        row = 2 if case["dtype"] == "bfloat16" else 4
        rows = b * t * ((case["query_heads"] + case["key_heads"]) * n
                        + case["value_heads"] * p) * row
        out = b * t * h * p * row
        decay = 4 * (h if case["decay"] == "head" else b * t * h)
        state = 4 * b * h * n * p
        if kind == "step":
            return dict(bytes=rows + out + decay + 2 * state, flops=5 * b * h * n * p)
        moved = rows + out + decay + state * (2 if case["initial"] else 1)
        flops = b * t * h * (min(t, CHUNK) * (n + p) + 4 * n * p)
        if case["train"]:
            # Back: the inputs and the cotangents read, the gradients written.
            moved += 2 * (rows + decay) + out + (2 * state if case["initial"] else 0)
            flops *= 4
        return dict(bytes=moved, flops=flops)
    if kind == "norm":
        count = case["samples"] * case["positions"] * case["channels"]
        row = 2 if case["dtype"] == "bfloat16" else 4
        arrays = 2 + (1 if case["gate"] else 0)
        flops = 12 * count
        if case["train"]:
            arrays += 3 + (2 if case["gate"] else 0)
            flops += 24 * count
        return dict(bytes=arrays * count * row, flops=flops)
    n, c = case["tokens"], case["width"]
    row = 2 if case["table"] == "bfloat16" else 4
    out = 2 if case["out"] == "bfloat16" else 4
    # Rows drawn more than once are read once.
    read = min(n, case["rows"]) * c * row + 8 * n
    moved, flops = read + n * c * out, n * c
    if case["train"]:
        moved += 8 * n + n * c * out + case["rows"] * c * row
        flops += 2 * n * c
    return dict(bytes=moved, flops=flops)


# ---------------------------------------------------------------------------
# The operators in float64
# ---------------------------------------------------------------------------


def _recurrence64(q, k, v, g, state):
    """The definition, token by token: q, k [B,T,H,N], v [B,T,H,P], g [B,T,H]."""
    out = torch.empty_like(v)
    lam = torch.exp(g)[..., None, None]
    for t in range(q.shape[1]):
        state = state * lam[:, t]
        state = torch.addcmul(state, k[:, t, :, :, None], v[:, t, :, None, :])
        out[:, t] = torch.matmul(q[:, t, :, None, :], state)[:, :, 0]
    return out, state


def _pairs64(q, k, v, g, state):
    """The same as sums over every pair of tokens, for automatic gradients."""
    time = q.shape[1]
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    total = torch.cumsum(g.transpose(1, 2), dim=2)
    gap = total[..., :, None] - total[..., None, :]
    later = torch.ones(time, time, dtype=torch.bool, device=q.device).triu(1)
    weight = torch.exp(gap.masked_fill(later, -math.inf))
    out = torch.matmul(torch.matmul(q, k.transpose(2, 3)) * weight, v) \
        + torch.exp(total)[..., None] * torch.matmul(q, state)
    tail = weight[..., -1, :, None]
    final = torch.exp(total[..., -1])[..., None, None] * state \
        + torch.matmul((k * tail).transpose(2, 3), v)
    return out.transpose(1, 2), final


def _attention64(case, x, lengths, form):
    h, n, p = case["heads"], case["key_dim"], case["value_dim"]
    b, time = x["queries"].shape[:2]
    q, k, v = (x[m].repeat_interleave(h // x[m].shape[2], dim=2)
               for m in ("queries", "keys", "values"))
    g = x["log_decay"] + x["queries"].new_zeros(b, time, h)
    if lengths is not None:
        here = (torch.arange(time, device=q.device)[None] < lengths[:, None]).double()
        q, k, v = (t * here[..., None, None] for t in (q, k, v))
        g = g * here[..., None]
    start = x["initial"] if "initial" in x else q.new_zeros(b, h, n, p)
    out, final = form(q, k, v, g, start)
    return dict(output=out * n ** -0.5, state=final)


def _double(x):
    return {n: t.detach().double() for n, t in x.items()}


def _attention_exact(case, seed):
    x, fixed, cot = _attention_inputs(case, seed)
    x, cot, lengths = _double(x), _double(cot), fixed.get("lengths")
    if not case["train"]:
        with torch.no_grad():
            return _attention64(case, x, lengths, _recurrence64)
    # Slices of batch rows, so that the matrices of pairs stay within a few GB.
    step = max(1, (1 << 27) // (case["heads"] * case["time"] ** 2))
    shared = ("log_decay",) if case["decay"] == "head" else ()
    parts = []
    for first in range(0, case["batch"], step):
        rows = slice(first, first + step)
        part = {n: (t if n in shared else t[rows]).clone().requires_grad_(True)
                for n, t in x.items()}
        here = None if lengths is None else lengths[rows]
        parts.append(_differentiate(lambda y: _attention64(case, y, here, _pairs64), part,
                                    {n: t[rows] for n, t in cot.items()}))
    return {n: sum(r[n] for r in parts) if n[2:] in shared and n.startswith("d_")
            else torch.cat([r[n] for r in parts]) for n in parts[0]}


def _step_exact(case, seed):
    x = _step_inputs(case, seed)
    active = x.pop("active", None)
    x = _double(x)
    h = case["heads"]
    q, k, v = (x[m].repeat_interleave(h // x[m].shape[1], dim=1)
               for m in ("query", "key", "value"))
    lam = torch.exp(x["log_decay"] + q.new_zeros(case["batch"], h))
    state = lam[..., None, None] * x["state"] + torch.matmul(k[..., None], v[..., None, :])
    out = torch.matmul(q[..., None, :], state)[..., 0, :] * case["key_dim"] ** -0.5
    if active is not None:
        out = out * active[:, None, None]
        state = torch.where(active[:, None, None, None], state, x["state"])
    return dict(output=out, state=state)


def _norm64(case, x):
    m, groups = case["samples"], case["groups"]
    t = x["x"].reshape(m, case["positions"], groups, -1)
    count = t.shape[1] * t.shape[3]
    mean = t.sum(dim=(1, 3), keepdim=True) / count
    variance = ((t - mean) ** 2).sum(dim=(1, 3), keepdim=True) / count
    z = ((t - mean) / torch.sqrt(variance + 1e-5)).reshape(x["x"].shape)
    if "weight" in x:
        z = z * x["weight"] + x["bias"]
    u = x["gate"] if "gate" in x else z
    if case["activation"] == "silu":
        u = u * torch.sigmoid(u)
    elif case["activation"] == "gelu":
        u = u * 0.5 * torch.erfc(-u / math.sqrt(2.0))
    return dict(output=z * u if "gate" in x else u)


def exact(case, seed):
    kind = case["kind"]
    if kind == "attention":
        return _attention_exact(case, seed)
    if kind == "step":
        return _step_exact(case, seed)
    if kind == "norm":
        x, cot = _norm_inputs(case, seed)
        x, cot = _double(x), _double(cot)
        if not case["train"]:
            return _norm64(case, x)
        x = {n: t.requires_grad_(True) for n, t in x.items()}
        return _differentiate(lambda y: _norm64(case, y), x, cot)
    x, fixed, cot = _embedding_inputs(case, seed)
    rows = torch.cat([x["table"].double(), x["table"].new_zeros(1, case["width"]).double()])
    ids = fixed["ids"]
    ids = torch.where(ids < 0, torch.full_like(ids, case["rows"]), ids)
    root = case["width"] ** 0.5
    out = dict(output=rows[ids] * root)
    if cot:
        grad = torch.zeros_like(rows)
        grad.index_put_((ids,), cot["output"].double() * root, accumulate=True)
        out["d_table"] = grad[:-1]
    return out

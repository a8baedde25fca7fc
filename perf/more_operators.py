"""Cases of the causal mixer's operators: linear attention with a decay per head, its single-token step, rotary positions.

``run`` computes a case with elementary torch operations in FP32 (``own``
false) or through the package's operators (``own`` true); ``exact`` evaluates
the definition in 64 bits.

Definitions, per sample and head, over the valid tokens t = 1, 2, .. in order
(a masked token is as though absent: it changes no state and its output is zero):

* decay attention: ``S_t = e^l S_{t-1} + k_t v_t^T``, ``y_t = scale * S_t^T q_t`` from a given ``S_0`` or zero,
  ``l`` the head's log decay; the last state is an output when a state is carried.  A training pass
  also returns the gradients of q, k, v and the given state, the last state's gradient being an input.
* its step: one token per sample, the new state and the output; an inactive sample keeps its state.
* rotary positions: of the first ``2 f`` features of a head, pair i (features ``2i, 2i + 1``, or ``i, i + f``)
  is turned by the angle ``position * frequency_i`` and multiplied by ``magnitude``; a training pass also
  returns the gradient of x.
"""

import functools
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MOST_VALUES = 8 * 8192 * 16 * 128


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # Prompts of a small served batch at the vision width and length (8 samples of 65 tokens, width 192): latency.
        dict(name="decay_prompt_8x65", op="decay", batch=8, length=65, heads=6, key=32, value=32, type="fp16", mask="none", state=False, train=False),
        # A continued prompt of one long document: few heads, so the token axis is what there is to work on.
        dict(name="decay_prompt_65536", op="decay", batch=1, length=65536, heads=8, key=64, value=64, type="bf16", mask="none", state=True, train=False),
        # Training step at the mixer's benchmark shape: 64 x 4096 tokens, width 256, 8 heads.
        dict(name="decay_train_64x4096", op="decay", batch=64, length=4096, heads=8, key=32, value=32, type="bf16", mask="none", state=False, train=True),
        # Padded samples of an odd length at width 512 in FP16, one of them empty.
        dict(name="decay_train_padded", op="decay", batch=32, length=2047, heads=8, key=64, value=64, type="fp16", mask="prefix", state=False, train=True),
        # A wide model's step: 128 features per head.
        dict(name="decay_train_wide", op="decay", batch=8, length=8192, heads=16, key=128, value=128, type="bf16", mask="none", state=False, train=True),
        # Truncated back-propagation at sizes that divide nothing: states in and out, tokens masked anywhere.
        dict(name="decay_train_odd", op="decay", batch=3, length=1361, heads=5, key=40, value=72, type="fp16", mask="holes", state=True, train=True),
        # One sample's next token at the mixer's width: latency.
        dict(name="step_one", op="step", batch=1, heads=8, key=32, value=32, type="bf16", masked=False),
        # The next tokens of a full served batch of a wide model: every state read and written once.
        dict(name="step_256_wide", op="step", batch=256, heads=16, key=128, value=128, type="bf16", masked=False),
        # Odd sizes, some samples finished.
        dict(name="step_odd", op="step", batch=37, heads=5, key=40, value=72, type="fp16", masked=True),
        # Queries and keys of the next token of 16 samples, far into their texts: latency.
        dict(name="rotary_next_tokens", op="rotary", batch=16, length=1, heads=16, dim=64, rotary=64, type="bf16", interleaved=False, scaling="none", positions="far", train=False),
        # Queries and keys of a training step at the mixer's benchmark shape.
        dict(name="rotary_train_64x4096", op="rotary", batch=64, length=4096, heads=16, dim=32, rotary=32, type="bf16", interleaved=False, scaling="none", positions="range", train=True),
        # Part of the head, interleaved pairs, a context stretched eightfold, every sample at its own positions, odd length.
        dict(name="rotary_train_stretched", op="rotary", batch=3, length=20011, heads=10, dim=80, rotary=48, type="fp32", interleaved=True, scaling="blend", positions="sample", train=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("decay", "decay", "step", "rotary"))
    batch = _log(rng, 1, 64)
    if op == "rotary":
        heads, dim = _log(rng, 1, 32), 8 * _log(rng, 2, 16)
        most = max(1, min(65536, _MOST_VALUES // (batch * heads * dim)))
        return dict(op=op, batch=batch, length=_log(rng, 1, most), heads=heads, dim=dim, rotary=2 * rng.randint(1, dim // 2) if rng.random() < 0.4 else dim,
                    type=rng.choice(("bf16", "fp16", "fp32")), interleaved=rng.random() < 0.5, scaling=rng.choice(("none", "linear", "base", "blend")),
                    positions=rng.choice(("range", "sample", "far")), train=rng.random() < 0.5)
    heads, key, value = _log(rng, 1, 16), 8 * _log(rng, 2, 16), 8 * _log(rng, 2, 16)
    if op == "step":
        return dict(op=op, batch=_log(rng, 1, 256), heads=heads, key=key, value=value, type=rng.choice(("bf16", "fp16", "fp32")), masked=rng.random() < 0.4)
    most = max(1, min(65536, _MOST_VALUES // (batch * heads * max(key, value))))
    return dict(op=op, batch=batch, length=_log(rng, 1, most), heads=heads, key=key, value=value, type=rng.choice(("bf16", "fp16")),
                mask=rng.choice(("none", "none", "prefix", "holes")), state=rng.random() < 0.4, train=rng.random() < 0.6)


# ---------------------------------------------------------------------------- inputs
def _mask(case, g):
    shape = (case["batch"], case["length"])
    if case["mask"] == "none":
        return None
    if case["mask"] == "prefix":  # padded at the end, one sample of a batch without a token
        valid = torch.randint(max(1, shape[1] // 4), shape[1] + 1, (shape[0], 1), device="cuda", generator=g)
        valid[1:2] = 0
        return torch.arange(shape[1], device="cuda") < valid
    return torch.rand(shape, device="cuda", generator=g) < 0.8


def _frequencies(case):
    """``rotary / 2`` angles per position in 64 bits, and the magnitude."""
    half, factor, original, base = case["rotary"] // 2, 8.0, 4096, 10000.0
    i = torch.arange(half, dtype=torch.float64) / half
    if case["scaling"] == "base":  # a larger base: the slowest pair eight times slower, the fastest as it was
        base *= factor ** (half / max(1, half - 1))
    f = base ** -i
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "blend":  # by the number of turns within the original context: below one as linear, above 32 as it was
        keep = ((original * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        return f / factor * (1 - keep) + f * keep, 0.1 * math.log(factor) + 1
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    kind, b, h = _TYPES[case["type"]], case["batch"], case["heads"]
    if case["op"] == "rotary":
        n = case["length"]
        frequencies, magnitude = _frequencies(case)
        state = dict(case=case, x=normal(b, n, h, case["dim"]).to(kind), frequencies=frequencies.cuda(), magnitude=magnitude, positions=None)
        if case["positions"] != "range":
            most = 2 ** 20 if case["positions"] == "far" else 32768
            state["positions"] = torch.randint(0, most, (b, 1), device="cuda", generator=g) + torch.arange(n, device="cuda")
        if case["train"]:
            state |= dict(x=state["x"].requires_grad_(), dy=normal(b, n, h, case["dim"]).to(kind))
        return state
    dk, dv = case["key"], case["value"]
    # windows from 8 to 512 tokens, the heads spread evenly over their logarithm
    log_decay = torch.log1p(-2.0 ** -(3 + 6 * torch.arange(h, device="cuda") / max(1, h - 1)))
    state = dict(case=case, log_decay=log_decay, scale=dk ** -0.5)
    carried = 4 * normal(b, h, dk, dv)
    if case["op"] == "step":
        active = torch.rand(b, device="cuda", generator=g) < 0.7 if case["masked"] else None
        return state | dict(q=normal(b, h, dk).to(kind), k=normal(b, h, dk).to(kind), v=normal(b, h, dv).to(kind), state=carried,
                            mask=active, new_state=torch.empty_like(carried))
    n = case["length"]
    state |= dict(q=normal(b, n, h, dk).to(kind), k=normal(b, n, h, dk).to(kind), v=normal(b, n, h, dv).to(kind), mask=_mask(case, g),
                  state=carried if case["state"] else None)
    if case["train"]:
        state |= {name: state[name].requires_grad_() for name in ("q", "k", "v", "state") if state[name] is not None}
        state |= dict(dy=normal(b, n, h, dv).to(kind), dlast=normal(b, h, dk, dv) if case["state"] else None)
    return state


# ---------------------------------------------------------------------------- plain forms
_CHUNK = 64


def _chunks(x):
    """[B, N, H, d] -> [chunks, B H, 64, d], zeros behind the last token."""
    b, n, h, d = x.shape
    x = torch.nn.functional.pad(x.transpose(1, 2), (0, 0, 0, -n % _CHUNK))
    return x.reshape(b * h, -1, _CHUNK, d).transpose(0, 1).contiguous()


def _scan_plain(x, y, z, log_decay, mask, state, late):
    """``w_t = x_t . (sum of e^(l (t - s)) y_s z_s over s <= t, and the state)``, and the state after the last token.

    x, y, z [B, N, H, d] with zeros in masked rows, mask [B, N]; the state is
    decayed before a token joins it (``late`` false) or after (true).
    """
    b, n, h, _ = x.shape
    live = torch.nn.functional.pad(mask.float(), (0, -n % _CHUNK)).reshape(b, -1, _CHUNK)
    live = live.repeat_interleave(h, 0).transpose(0, 1)  # [chunks, B H, 64]
    rate = log_decay.repeat(b)[None, :, None]
    rank = live.cumsum(-1)  # counts the token itself
    count = rank[..., -1:]
    apart = rate[..., None] * (rank[..., :, None] - rank[..., None, :])
    lower = torch.ones(_CHUNK, _CHUNK, device=x.device).tril()
    weight = torch.exp(torch.where(lower.bool(), apart, 0.0)) * lower
    x, y, z = _chunks(x), _chunks(y), _chunks(z)
    inside = (x @ y.mT * weight) @ z
    into = torch.exp(rate * (rank - late)) * live
    from_each = torch.exp(rate * (count - rank + late)) * live
    whole = torch.exp(rate * count)[..., None]
    added = (y * from_each[..., None]).mT @ z
    states = []
    state = torch.zeros_like(added[0]) if state is None else state.reshape(added[0].shape)
    for c in range(len(added)):
        states.append(state)
        state = state * whole[c] + added[c]
    w = inside + (x @ torch.stack(states)) * into[..., None]
    w = w.transpose(0, 1).reshape(b, h, -1, w.shape[-1])[:, :, :n].transpose(1, 2)
    return w, state.reshape(b, h, *state.shape[1:])


def _decay_plain(s):
    c, l, a = s["case"], s["log_decay"], s["scale"]
    mask = torch.ones(c["batch"], c["length"], dtype=torch.bool, device=l.device) if s["mask"] is None else s["mask"]
    clear = lambda t: torch.where(mask[..., None, None], t.detach().float(), 0.0)  # noqa: E731
    q, k, v = clear(s["q"]) * a, clear(s["k"]), clear(s["v"])
    s0 = None if s["state"] is None else s["state"].detach()
    kind = s["q"].dtype
    y, last = _scan_plain(q, k, v, l, mask, s0, 0)
    out = dict(y=y.to(kind))
    if c["state"]:
        out["last"] = last
    if not c["train"]:
        return out
    dy = clear(s["dy"])
    dq, _ = _scan_plain(dy, v, k, l, mask, None if s0 is None else s0.mT.contiguous(), 0)
    back = lambda t: t.flip(1)  # noqa: E731
    dlast = s["dlast"]
    dk, _ = _scan_plain(back(v), back(dy), back(q), l, back(mask), None if dlast is None else dlast.mT.contiguous(), 1)
    dv, dstate = _scan_plain(back(k), back(q), back(dy), l, back(mask), dlast, 1)
    out |= dict(dq=(dq * a).to(kind), dk=back(dk).to(kind), dv=back(dv).to(kind))
    if c["state"]:
        out["dstate"] = dstate
    return out


def _step_plain(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    new = s["state"] * torch.exp(s["log_decay"])[:, None, None] + k[..., None] * v[..., None, :]
    y = (q[..., None] * new).sum(-2) * s["scale"]
    if s["mask"] is not None:
        new = torch.where(s["mask"][:, None, None, None], new, s["state"])
        y = torch.where(s["mask"][:, None, None], y, 0.0)
    return dict(y=y.to(s["q"].dtype), new_state=new)


def _turn_plain(x, s, sign):
    c = s["case"]
    half = c["rotary"] // 2
    positions = torch.arange(c["length"], device=x.device)[None] if s["positions"] is None else s["positions"]
    angle = positions.double()[..., None] * s["frequencies"]
    cos, sin = (torch.cos(angle) * s["magnitude"]).float()[:, :, None], (torch.sin(angle) * (s["magnitude"] * sign)).float()[:, :, None]
    part, rest = x[..., : 2 * half].float(), x[..., 2 * half:]
    if c["interleaved"]:
        first, second = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((first * cos - second * sin, second * cos + first * sin), dim=-1).flatten(-2)
    else:
        first, second = part[..., :half], part[..., half:]
        turned = torch.cat((first * cos - second * sin, second * cos + first * sin), dim=-1)
    return torch.cat((turned.to(x.dtype), rest), dim=-1)


def _rotary_plain(s):
    y = _turn_plain(s["x"].detach(), s, 1)
    return dict(y=y, dx=_turn_plain(s["dy"], s, -1)) if s["case"]["train"] else y


# ---------------------------------------------------------------------------- the package's operators
@functools.cache
def _package():
    from lsso_b200.ball import cuda, decay, rotary

    cuda.load()
    return decay.decay_attention, decay.decay_attention_step, rotary.rotary


def _decay_own(s):
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        y = _package()[0](s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], state=s["state"], valid_mask=s["mask"], return_state=c["state"])
    y, last = y if c["state"] else (y, None)
    out = dict(y=y, last=last) if c["state"] else dict(y=y)
    if not c["train"]:
        return out
    inputs, ends, upstream = [s["q"], s["k"], s["v"]], [y], [s["dy"]]
    if c["state"]:
        inputs, ends, upstream = inputs + [s["state"]], ends + [last], upstream + [s["dlast"]]
    return out | dict(zip(("dq", "dk", "dv", "dstate"), torch.autograd.grad(ends, inputs, upstream)))


def _step_own(s):
    y = _package()[1](s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"], valid_mask=s["mask"], new_state=s["new_state"])
    return dict(y=y, new_state=s["new_state"])


def _rotary_own(s):
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        y = _package()[2](s["x"], s["frequencies"], s["positions"], interleaved=c["interleaved"], magnitude=s["magnitude"])
    return dict(y=y, dx=torch.autograd.grad(y, s["x"], s["dy"])[0]) if c["train"] else y


_RUN = {"decay": (_decay_plain, _decay_own), "step": (_step_plain, _step_own), "rotary": (_rotary_plain, _rotary_own)}


def run(state):
    return _RUN[state["case"]["op"]][bool(own)](state)


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["type"]]
    b, h = case["batch"], case["heads"]
    if case["op"] == "rotary":
        t = b * case["length"]
        tables = 4 * case["rotary"] + (0 if case["positions"] == "range" else 8 * t)
        passes = 2 if case["train"] else 1
        return {"bytes": 2 * passes * t * h * case["dim"] * size + tables, "flops": 3 * passes * t * h * case["rotary"]}
    dk, dv = case["key"], case["value"]
    if case["op"] == "step":  # the state in and out; update and readout
        return {"bytes": b * h * (8 * dk * dv + size * (2 * dk + 2 * dv)), "flops": 5 * b * h * dk * dv}
    t = b * case["length"]
    moved = t * h * size * (2 * dk + 2 * dv) + (t if case["mask"] != "none" else 0) + (8 * b * h * dk * dv if case["state"] else 0)
    flops = 4 * t * h * dk * dv  # update and readout
    if case["train"]:  # dy in, three gradients out; both states again, three readouts
        moved += t * h * size * (2 * dk + 2 * dv) + (8 * b * h * dk * dv if case["state"] else 0)
        flops += 10 * t * h * dk * dv
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------- 64 bits
def _by_token(x, live):
    """[B, N, H, d] -> [N, B H, d] in 64 bits, zeros in masked rows."""
    x = torch.where(live[..., None, None], x.detach().double(), 0.0)
    return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[-1])


def _decay_exact(s):
    c = s["case"]
    b, n, h, dk, dv = (c[x] for x in ("batch", "length", "heads", "key", "value"))
    live = torch.ones(b, n, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    gamma = torch.exp(s["log_decay"].double()).repeat(b)
    keep = torch.where(live.T[..., None], gamma.reshape(b, h), 1.0).reshape(n, b * h, 1, 1)
    q, k, v = (_by_token(s[x], live) for x in ("q", "k", "v"))
    shape = lambda t: t.reshape(n, b, h, -1).transpose(0, 1)  # noqa: E731
    a = s["scale"]
    train = c["train"]
    memory = torch.zeros(b * h, dk, dv, dtype=torch.float64, device="cuda") if s["state"] is None else s["state"].detach().double().reshape(b * h, dk, dv)
    y = torch.empty(n, b * h, dv, dtype=torch.float64, device="cuda")
    if train:
        dy = _by_token(s["dy"], live)
        dq, dkey, dvalue = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for t in range(n):
        memory = torch.baddbmm(memory * keep[t], k[t].unsqueeze(2), v[t].unsqueeze(1))
        torch.bmm(q[t].unsqueeze(1), memory, out=y[t].unsqueeze(1))
        if train:
            torch.bmm(memory, dy[t].unsqueeze(2), out=dq[t].unsqueeze(2))
    out = dict(y=shape(y * a))
    if c["state"]:
        out["last"] = memory.reshape(b, h, dk, dv)
    if not train:
        return out
    upstream = torch.zeros_like(memory) if s["dlast"] is None else s["dlast"].double().reshape(b * h, dk, dv)
    for t in reversed(range(n)):
        upstream = torch.baddbmm(upstream, q[t].unsqueeze(2), dy[t].unsqueeze(1), alpha=a)
        torch.bmm(upstream, v[t].unsqueeze(2), out=dkey[t].unsqueeze(2))
        torch.bmm(k[t].unsqueeze(1), upstream, out=dvalue[t].unsqueeze(1))
        upstream = upstream * keep[t]
    hidden = lambda t: torch.where(live[..., None, None], shape(t), 0.0)  # noqa: E731
    out |= dict(dq=shape(dq * a), dk=hidden(dkey), dv=hidden(dvalue))
    if c["state"]:
        out["dstate"] = upstream.reshape(b, h, dk, dv)
    return out


def _step_exact(s):
    active = torch.ones(s["q"].shape[0], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    old = s["state"].double()
    new = torch.einsum("h,bhkv->bhkv", torch.exp(s["log_decay"].double()), old) + torch.einsum("bhk,bhv->bhkv", s["k"].double(), s["v"].double())
    y = torch.einsum("bhk,bhkv->bhv", s["q"].double() * s["scale"], new)
    return dict(y=y * active[:, None, None], new_state=torch.where(active[:, None, None, None], new, old))


def _rotary_exact(s):
    c = s["case"]
    half = c["rotary"] // 2
    positions = torch.arange(c["length"], device="cuda").expand(c["batch"], -1) if s["positions"] is None else s["positions"]
    turn = torch.polar(torch.tensor(s["magnitude"], dtype=torch.float64, device="cuda"), torch.einsum("bn,f->bnf", positions.double(), s["frequencies"]))
    first = torch.arange(half, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else half)

    def apply(x, by):
        x = x.detach().double()
        z = torch.complex(x[..., first], x[..., second]) * by[:, :, None]
        out = x.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    y = apply(s["x"], turn)
    return dict(y=y, dx=apply(s["dy"], turn.conj())) if c["train"] else y


def exact(case, seed):
    return {"decay": _decay_exact, "step": _step_exact, "rotary": _rotary_exact}[case["op"]](prepare(case, seed))

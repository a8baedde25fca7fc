"""Cases of the token shell's operators: gated feed-forward, token embedding, dropout with the residual sum.

``run`` computes a case with elementary torch operations in FP32 (``own``
false) or through the package's operators (``own`` true); ``exact`` evaluates
the definition in 64 bits.

Definitions.  ``act`` is SiLU, ``g / (1 + e^-g)``, or GELU, ``g (1 + erf(g / sqrt 2)) / 2``.

* gated feed-forward: ``[g | u] = x W_in^T + b_in``, ``y = (act(g) * u) W_out^T + b_out``;
  a training pass also returns the gradients of x, the weights and the biases.
* token embedding: ``y[t] = scale * W[id[t]]``, zero where the mask is unset; a training pass also
  returns ``dW[v] = scale * sum of dy[t] over valid t with id[t] = v`` (the padding row zero).
* dropout with the residual sum: ``y = residual + branch * keep / (1 - p)``, zero in masked rows;
  ``keep`` of element 4j + i is ``word i >= round(p 2^32)`` of Philox4x32-10 (Salmon et al., SC 2011)
  at counter ``(j mod 2^32, j div 2^32, site, step mod 2^32)`` and key ``(seed mod 2^32, seed div 2^32)``;
  a training pass also returns the gradients of the branch and the residual.
"""

import functools
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_LARGEST_FLOPS = 18 * 32768 * 1024 * 4096


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # One token of a served model of the mixer's width 256: weight traffic and launch latency.
        dict(name="ffn_one_token", op="ffn", tokens=1, dim=256, hidden=688, act="silu", type="bf16", bias=False, train=False),
        # A served batch of short prompts at width 512, below one 128-row tile.
        dict(name="ffn_short_batch", op="ffn", tokens=97, dim=512, hidden=1368, act="silu", type="fp16", bias=False, train=False),
        # Training step at the mixer's benchmark shape: 64 x 4096 tokens, width 256.
        dict(name="ffn_train_64x4096", op="ffn", tokens=64 * 4096, dim=256, hidden=688, act="silu", type="bf16", bias=False, train=True),
        # Vision width 192, an odd number of tokens, biases and GELU, in FP16.
        dict(name="ffn_train_ragged_gelu", op="ffn", tokens=20011, dim=192, hidden=520, act="gelu", type="fp16", bias=True, train=True),
        # A wide model's step: tensor-core bound in all six products.
        dict(name="ffn_train_wide", op="ffn", tokens=32768, dim=1024, hidden=4096, act="silu", type="bf16", bias=False, train=True),
        # Lookup for 8 samples of 65 tokens (the vision sequence length): latency.
        dict(name="embed_lookup_8x65", op="embedding", batch=8, length=65, vocab=8192, dim=192, out="bf16", ids="uniform", masked=False, padding=False, train=False),
        # The four-layer shell's embedding: 64 x 4096 tokens over a vocabulary of 8, so every row sums 32 thousand tokens.
        dict(name="embed_train_vocab8", op="embedding", batch=64, length=4096, vocab=8, dim=128, out="bf16", ids="uniform", masked=False, padding=False, train=True),
        # A text vocabulary with its skewed use, padded samples, a padding row, odd vocabulary size.
        dict(name="embed_train_text", op="embedding", batch=32, length=2048, vocab=50021, dim=512, out="bf16", ids="skewed", masked=True, padding=True, train=True),
        # A small FP32 step at sizes that divide nothing.
        dict(name="embed_train_odd", op="embedding", batch=3, length=1361, vocab=1013, dim=100, out="fp32", ids="skewed", masked=True, padding=False, train=True),
        # One residual branch of a served or small step: latency.
        dict(name="dropout_8x65", op="dropout", batch=8, length=65, dim=192, branch="bf16", residual="fp32", p=0.1, masked=False, train=False),
        # The residual branch at the mixer's benchmark shape under mixed precision: FP16 branch, FP32 residual.
        dict(name="dropout_train_64x4096", op="dropout", batch=64, length=4096, dim=256, branch="fp16", residual="fp32", p=0.1, masked=False, train=True),
        # Padded samples of odd width in BF16, a high rate.
        dict(name="dropout_train_masked", op="dropout", batch=32, length=2047, dim=250, branch="bf16", residual="bf16", p=0.35, masked=True, train=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("ffn", "embedding", "dropout"))
    if op == "ffn":
        train = rng.random() < 0.6
        dim, hidden = 8 * _log(rng, 8, 128), 8 * _log(rng, 8, 512)
        most = min(262144, _LARGEST_FLOPS // ((18 if train else 6) * dim * hidden), 2 ** 30 // (dim + 3 * hidden))
        return dict(op=op, tokens=_log(rng, 1, most), dim=dim, hidden=hidden, act=rng.choice(("silu", "gelu")),
                    type=rng.choice(("bf16", "fp16")), bias=rng.random() < 0.5, train=train)
    batch = _log(rng, 1, 64)
    if op == "embedding":
        dim = _log(rng, 8, 1024)
        vocab = min(_log(rng, 2, 65536), 2 ** 25 // dim)
        return dict(op=op, batch=batch, length=_log(rng, 1, min(4096, max(1, 2 ** 26 // (dim * batch)))), vocab=vocab, dim=dim,
                    out=rng.choice(("bf16", "fp16", "fp32")), ids=rng.choice(("uniform", "skewed")),
                    masked=rng.random() < 0.5, padding=rng.random() < 0.3, train=rng.random() < 0.7)
    dim = _log(rng, 16, 1024)
    branch, residual = rng.choice((("bf16", "fp32"), ("fp16", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32")))
    return dict(op=op, batch=batch, length=_log(rng, 1, min(4096, max(1, 2 ** 26 // (dim * batch)))), dim=dim, branch=branch,
                residual=residual, p=rng.choice((0.05, 0.1, 0.2, 0.5)), masked=rng.random() < 0.5, train=rng.random() < 0.7)


# ---------------------------------------------------------------------------- inputs
def _mask(case, generator):
    """Padded samples: a valid prefix of a quarter to all of the length."""
    if not case["masked"]:
        return None
    length = case["length"]
    valid = torch.randint(max(1, length // 4), length + 1, (case["batch"], 1), device="cuda", generator=generator)
    return torch.arange(length, device="cuda") < valid


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "ffn":
        t, d, h, kind = case["tokens"], case["dim"], case["hidden"], _TYPES[case["type"]]
        train = case["train"]
        state = dict(case=case, x=normal(t, d).to(kind), w_in=(normal(2 * h, d) / d ** 0.5).to(kind),
                     w_out=(normal(d, h) / h ** 0.5).to(kind), b_in=None, b_out=None)
        if case["bias"]:
            state |= dict(b_in=(0.2 * normal(2 * h)).to(kind), b_out=(0.2 * normal(d)).to(kind))
        if train:
            state["dy"] = normal(t, d).to(kind)
            state |= {k: state[k].requires_grad_() for k in ("x", "w_in", "w_out", "b_in", "b_out") if state[k] is not None}
        return state
    shape = (case["batch"], case["length"])
    if case["op"] == "embedding":
        vocab, dim = case["vocab"], case["dim"]
        if case["ids"] == "uniform":
            ids = torch.randint(0, vocab, shape, device="cuda", generator=g)
        else:  # frequency falls as 1 / rank, over a fixed shuffle of the rows
            rank = ((torch.rand(shape, device="cuda", generator=g) * math.log(vocab + 1)).exp().long() - 1).clamp(0, vocab - 1)
            ids = torch.randperm(vocab, device="cuda", generator=g)[rank]
        mask = _mask(case, g)
        weight = normal(vocab, dim)
        state = dict(case=case, ids=ids, weight=weight, scale=dim ** 0.5, mask=mask, padding=vocab // 2 if case["padding"] else None)
        if case["train"]:
            state |= dict(weight=weight.requires_grad_(), dy=normal(*shape, dim).to(_TYPES[case["out"]]))
        return state
    state = dict(case=case, branch=normal(*shape, case["dim"]).to(_TYPES[case["branch"]]),
                 residual=(2 * normal(*shape, case["dim"])).to(_TYPES[case["residual"]]), mask=_mask(case, g),
                 rng=torch.randint(0, 2 ** 40, (2,), device="cuda", generator=g), site=3)
    if case["train"]:
        state |= {k: state[k].requires_grad_() for k in ("branch", "residual")}
        state["dy"] = normal(*shape, case["dim"]).to(_TYPES[case["residual"]])
    return state


# ---------------------------------------------------------------------------- plain forms
def _ffn_plain(s):
    c = s["case"]
    kind = s["x"].dtype
    x, w_in, w_out = s["x"].detach().float(), s["w_in"].detach().float(), s["w_out"].detach().float()
    gu = x @ w_in.T
    if c["bias"]:
        gu = gu + s["b_in"].detach().float()
    g, u = gu[:, : c["hidden"]], gu[:, c["hidden"]:]
    if c["act"] == "silu":
        cdf = 1 / (1 + torch.exp(-g))
    else:
        cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    a = g * cdf
    h = a * u
    y = h @ w_out.T
    if c["bias"]:
        y = y + s["b_out"].detach().float()
    if not c["train"]:
        return y.to(kind)
    dy = s["dy"].float()
    dh = dy @ w_out
    slope = cdf * (1 + g * (1 - cdf)) if c["act"] == "silu" else cdf + g * torch.exp(-0.5 * g * g) * (0.5 / math.pi) ** 0.5
    dgu = torch.cat((dh * u * slope, dh * a), dim=1)
    out = dict(y=y.to(kind), dx=(dgu @ w_in).to(kind), dw_in=(dgu.T @ x).to(kind), dw_out=(dy.T @ h).to(kind))
    if c["bias"]:
        out |= dict(db_in=dgu.sum(0).to(kind), db_out=dy.sum(0).to(kind))
    return out


def _embedding_plain(s):
    c, weight, ids = s["case"], s["weight"].detach(), s["ids"]
    y = weight[ids] * s["scale"]
    if s["mask"] is not None:
        y = torch.where(s["mask"][..., None], y, 0.0)
    y = y.to(_TYPES[c["out"]])
    if not c["train"]:
        return y
    dy = s["dy"].float().reshape(-1, c["dim"])
    if s["mask"] is not None:
        dy = torch.where(s["mask"].reshape(-1, 1), dy, 0.0)
    dw = torch.zeros_like(weight).index_add_(0, ids.reshape(-1), dy) * s["scale"]
    if s["padding"] is not None:
        dw[s["padding"]] = 0
    return dict(y=y, dw=dw)


def _round(state, _):
    """One Philox round on int64 tensors that hold 32-bit words (products wrap at 64 bits, which keeps all of their bits)."""
    c0, c1, c2, c3, k0, k1 = state
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    m = 0xFFFFFFFF
    return ((b >> 32) & m) ^ c1 ^ k0, b & m, ((a >> 32) & m) ^ c3 ^ k1, a & m, (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m


def _keep_plain(s):
    """0 / 1 of every element, as FP32."""
    like, m = s["branch"], 0xFFFFFFFF
    j = torch.arange((like.numel() + 3) // 4, device=like.device)
    seed, step = s["rng"][0], s["rng"][1]
    start = (j & m, j >> 32, torch.full_like(j, s["site"]), (step & m).expand_as(j), seed & m, (seed >> 32) & m)
    words = torch.stack(functools.reduce(_round, range(10), start)[:4], dim=1).reshape(-1)[: like.numel()]
    return (words >= round(s["case"]["p"] * 2 ** 32)).float().reshape(like.shape)


def _dropout_plain(s):
    c, branch, residual = s["case"], s["branch"].detach(), s["residual"].detach()
    factor = _keep_plain(s) * (1 / (1 - c["p"]))
    if s["mask"] is not None:
        factor = torch.where(s["mask"][..., None], factor, 0.0)
    y = residual.float() + branch.float() * factor
    if s["mask"] is not None:
        y = torch.where(s["mask"][..., None], y, 0.0)
    y = y.to(residual.dtype)
    if not c["train"]:
        return y
    dy = s["dy"].float()
    dr = dy if s["mask"] is None else torch.where(s["mask"][..., None], dy, 0.0)
    return dict(y=y, dbranch=(dy * factor).to(branch.dtype), dresidual=dr.to(residual.dtype))


# ---------------------------------------------------------------------------- the package's operators
@functools.cache
def _package():
    from lsso_b200.ball import cuda, dropout, embedding, feedforward

    cuda.load()
    return feedforward.gated_feed_forward, embedding.token_embedding, dropout.dropout_add


def _ffn_own(s):
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        y = _package()[0](s["x"], s["w_in"], s["w_out"], s["b_in"], s["b_out"], activation=c["act"])
    if not c["train"]:
        return y
    names = [n for n in ("x", "w_in", "w_out", "b_in", "b_out") if s[n] is not None]
    return dict(zip(["y"] + ["d" + n for n in names], (y, *torch.autograd.grad(y, [s[n] for n in names], s["dy"]))))


def _embedding_own(s):
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        y = _package()[1](s["ids"], s["weight"], scale=s["scale"], valid_mask=s["mask"], padding_idx=s["padding"], dtype=_TYPES[c["out"]])
    return dict(y=y, dw=torch.autograd.grad(y, s["weight"], s["dy"])[0]) if c["train"] else y


def _dropout_own(s):
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        y = _package()[2](s["branch"], s["residual"], p=c["p"], state=s["rng"], site=s["site"], valid_mask=s["mask"])
    if not c["train"]:
        return y
    return dict(zip(("y", "dbranch", "dresidual"), (y, *torch.autograd.grad(y, (s["branch"], s["residual"]), s["dy"]))))


_RUN = {"ffn": (_ffn_plain, _ffn_own), "embedding": (_embedding_plain, _embedding_own), "dropout": (_dropout_plain, _dropout_own)}


def run(state):
    return _RUN[state["case"]["op"]][bool(own)](state)


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "ffn":
        t, d, h = case["tokens"], case["dim"], case["hidden"]
        weights = 3 * d * h + (2 * h + d if case["bias"] else 0)
        if case["train"]:  # x, dy in; y, dx out; weights in and their gradients out
            return {"bytes": 2 * (4 * t * d + 2 * weights), "flops": 18 * t * d * h}
        return {"bytes": 2 * (2 * t * d + weights), "flops": 6 * t * d * h}
    t, d = case["batch"] * case["length"], case["dim"]
    mask = t if case["masked"] else 0
    if case["op"] == "embedding":
        out, rows = size[case["out"]], min(case["vocab"], t)
        forward = 8 * t + mask + 4 * rows * d + out * t * d
        if case["train"]:  # the upstream gradient in, the whole weight gradient out
            return {"bytes": forward + out * t * d + 4 * case["vocab"] * d, "flops": 2 * t * d}
        return {"bytes": forward, "flops": t * d}
    b, r = size[case["branch"]], size[case["residual"]]
    forward = t * d * (b + 2 * r) + mask
    if case["train"]:  # the upstream gradient in, the branch's out; the residual's is the upstream one unless rows are masked
        return {"bytes": forward + t * d * (r + b + (r if case["masked"] else 0)), "flops": 4 * t * d}
    return {"bytes": forward, "flops": 2 * t * d}


# ---------------------------------------------------------------------------- 64 bits
def _ffn_exact(s):
    c = s["case"]
    names = [n for n in ("x", "w_in", "w_out", "b_in", "b_out") if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_(c["train"]) for n in names}
    gate, up = v["w_in"].split(c["hidden"])
    g, u = torch.nn.functional.linear(v["x"], gate), torch.nn.functional.linear(v["x"], up)
    if c["bias"]:
        b_gate, b_up = v["b_in"].split(c["hidden"])
        g, u = g + b_gate, u + b_up
    act = g * torch.sigmoid(g) if c["act"] == "silu" else 0.5 * g * torch.erfc(-g / math.sqrt(2))
    y = torch.nn.functional.linear(act * u, v["w_out"], v.get("b_out"))
    if not c["train"]:
        return y
    grads = torch.autograd.grad(y, [v[n] for n in names], s["dy"].double())
    return dict(zip(["y"] + ["d" + n for n in names], (y.detach(), *grads)))


def _embedding_exact(s):
    c = s["case"]
    live = torch.ones_like(s["ids"], dtype=torch.bool) if s["mask"] is None else s["mask"]
    weight, ids = s["weight"].detach().double(), s["ids"]
    y = weight.index_select(0, ids.flatten()).reshape(*ids.shape, c["dim"]) * s["scale"] * live[..., None]
    if not c["train"]:
        return y
    counted = live if s["padding"] is None else live & (ids != s["padding"])
    dw = torch.zeros_like(weight).index_put_((ids[counted],), s["dy"][counted].double() * s["scale"], accumulate=True)
    return dict(y=y, dw=dw)


def _high(a, b):
    """High 32 bits of the product of 32-bit words, from 16-bit halves (nothing wraps)."""
    a1, a0, b1, b0 = a >> 16, a & 0xFFFF, b >> 16, b & 0xFFFF
    cross = a1 * b0 + (a0 * b0 >> 16)
    return a1 * b1 + (cross >> 16) + ((cross & 0xFFFF) + a0 * b1 >> 16)


def _dropout_exact(s):
    c, n = s["case"], s["branch"].numel()
    seed, step = (int(v) for v in s["rng"].tolist())
    key = [seed % 2 ** 32, seed // 2 ** 32]
    group = torch.arange((n + 3) // 4, device=s["branch"].device)
    word = [group % 2 ** 32, group // 2 ** 32, torch.full_like(group, s["site"]), torch.full_like(group, step % 2 ** 32)]
    for i in range(10):
        k = [(key[0] + i * 0x9E3779B9) % 2 ** 32, (key[1] + i * 0xBB67AE85) % 2 ** 32]
        low = [word[q] * (m & 0xFFFF) + ((word[q] * (m >> 16) & 0xFFFF) << 16) & 0xFFFFFFFF for q, m in ((0, 0xD2511F53), (2, 0xCD9E8D57))]
        word = [_high(word[2], 0xCD9E8D57) ^ word[1] ^ k[0], low[1], _high(word[0], 0xD2511F53) ^ word[3] ^ k[1], low[0]]
    dropped = torch.stack(word, dim=-1).flatten()[:n].reshape(s["branch"].shape) < round(c["p"] * 2 ** 32)
    live = torch.ones_like(dropped) if s["mask"] is None else s["mask"][..., None].expand_as(dropped)
    branch = (s["branch"].detach().double() / (1 - c["p"])).masked_fill(dropped, 0.0)
    y = (s["residual"].detach().double() + branch) * live
    if not c["train"]:
        return y
    dy = s["dy"].double() * live
    return dict(y=y, dbranch=(dy / (1 - c["p"])).masked_fill(dropped, 0.0), dresidual=dy)


def exact(case, seed):
    return {"ffn": _ffn_exact, "embedding": _embedding_exact, "dropout": _dropout_exact}[case["op"]](prepare(case, seed))

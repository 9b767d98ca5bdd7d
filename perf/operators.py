"""The operators of a state space block as cases that can be timed: the short causal convolution, the selective state space
scan behind it, and the norms around the block with its gate and its residual.

A case is a dict of plain values.  `listed()` gives the fixed ones, `draw(rng)` one more of the same ranges, `prepare` makes
what a program has in hand before the call (on the GPU, from a seed), `run` is one pass: in the operators' plain form, or
(`own`) through the public entry points of the package.  `exact` gives the same outputs from the definitions in 64 bits, `work`
says what a pass cannot do without.

Kinds of cases ("kind"), d channels, S states a channel:
  conv_step, scan_step      one token for each of `batch` sequences, the state taken and the next one given
  conv_prompt, scan_prompt  a forward pass without gradients that gives the final state
  conv_train, scan_train    forward and backward pass, every gradient
  norm                      norm behind the block, gate, residual scale, sum with the stream, norm before the next block: forward
  norm_train                the same with the backward pass

A block's input projection gives x and z side by side, and a second one the step sizes' inner activations, B and C: where
"views" is set the operators get them as the views that they are.  "lens": lengths of packed sequences ("" = `batch` sequences of T
tokens).
"""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp32": 4}


def _package():
    # the package lives below a folder whose name is no identifier, relative to the root the process works in
    path = os.path.join(os.getcwd(), "hdla-impl_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import hdla_hip
    return hdla_hip


def _conv(kind, name=None, *, batch, T=1, d, W=4, dtype="bf16", act="silu", lens="", state=True, views=False):
    c = dict(kind=kind, batch=batch, T=T, d=d, W=W, dtype=dtype, act=act, lens=lens, state=state, views=views)
    return dict(c, name=name) if name else c


def _scan(kind, name=None, *, batch, T=1, d, S=16, groups=1, dtype="bf16", gate=True, lens="", state=True, views=False):
    c = dict(kind=kind, batch=batch, T=T, d=d, S=S, groups=groups, dtype=dtype, gate=gate, lens=lens, state=state, views=views)
    return dict(c, name=name) if name else c


def _norm(kind, name=None, *, rows, d, dtype="bf16", stream="bf16", post=True, gate=True, scale=True):
    c = dict(kind=kind, rows=rows, d=d, dtype=dtype, stream=stream, post=post, gate=gate, scale=scale)
    return dict(c, name=name) if name else c


def listed():
    return [
        # interactive generation: one token of one sequence, where the call itself is the cost
        _conv("conv_step", "conv_step_one", batch=1, d=2048),
        # a long prompt of one sequence, x being half of the input projection's output
        _conv("conv_prompt", "conv_prompt", batch=1, T=16384, d=4096, state=False, views=True),
        # a training step of the repository's own batch (4 x 2048 tokens, 1024 channels, twice as many in the block)
        _conv("conv_train", "conv_train", batch=4, T=2048, d=2048, state=False, views=True),
        # full precision, packed texts of unequal, odd lengths that continue earlier ones: numerics work and checks
        _conv("conv_train", "conv_train_fp32", batch=1, T=5003, d=1000, W=3, dtype="fp32", lens="1731,37,2204,1031"),
        # interactive generation
        _scan("scan_step", "scan_step_one", batch=1, d=2048),
        # a serving batch: one token each for 256 sequences, the states stream through
        _scan("scan_step", "scan_step_batch", batch=256, d=4096),
        # a long prompt of one sequence
        _scan("scan_prompt", "scan_prompt", batch=1, T=8192, d=4096, state=False, views=True),
        # a training step of the repository's own batch
        _scan("scan_train", "scan_train", batch=4, T=2048, d=2048, state=False, views=True),
        # full precision, packed sequences with states, two groups of channels with inputs of their own, more states
        _scan("scan_train", "scan_train_fp32", batch=1, T=2503, d=520, S=32, groups=2, dtype="fp32", lens="731,37,1204,531"),
        # the norms around the block: a decode step
        _norm("norm", "norm_step", rows=16, d=2048),
        # a long prompt, the residual stream in 32 bits
        _norm("norm", "norm_prompt", rows=16384, d=4096, stream="fp32", scale=False),
        # a training step
        _norm("norm_train", "norm_train", rows=8192, d=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, total, n):
    """n lengths (at least one token each) that add up to total, in any order."""
    cuts = sorted(rng.sample(range(1, total), n - 1))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    kind = rng.choice(["conv_step", "conv_prompt", "conv_train", "scan_step", "scan_prompt", "scan_train", "scan_train", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind.startswith("norm"):
        d = rng.choice([8 * _log(rng, 16, 512), 2 ** rng.randint(8, 12), _log(rng, 65, 4096)])
        most = 8192 * 2048 if kind == "norm_train" else 16384 * 4096
        return _norm(kind, rows=_log(rng, 1, min(20000, most // d // (2 if dtype == "fp32" else 1))), d=d, dtype=dtype,
                     stream=rng.choice([dtype, "fp32"]), post=rng.random() < 0.7, gate=rng.random() < 0.7, scale=rng.random() < 0.6)
    d = rng.choice([16 * _log(rng, 8, 256), 2 ** rng.randint(9, 12), _log(rng, 65, 4096)])
    W, S = rng.choice([2, 3, 4, 4]), rng.choice([8, 16, 16, 32, 12])
    if kind == "conv_step":
        return _conv(kind, batch=_log(rng, 1, 256), d=d, W=W, dtype=dtype, act=rng.choice(["silu", "none"]))
    if kind == "scan_step":
        return _scan(kind, batch=_log(rng, 1, max(1, min(256, 256 * 4096 * 16 // (d * S)))), d=d, S=S, dtype=dtype, gate=rng.random() < 0.8)
    state, views = rng.random() < 0.5, rng.random() < 0.5
    if kind.startswith("conv"):
        most = min(16384, (4 * 2048 * 2048 if kind == "conv_train" else 16384 * 4096) // d // (2 if dtype == "fp32" else 1))
    else:
        most = (4 * 2048 * 2048 * 16 if kind == "scan_train" else 8192 * 4096 * 16) // (d * S) // (4 if dtype == "fp32" else 1)
        # (the plain form is one pass after another: not more tokens than the longest listed case)
        most = min(2048 if kind == "scan_train" else 8192, most)
    total = _log(rng, 20, most)
    groups = rng.choice([1, 1, 2, 4]) if d % 4 == 0 else 1
    make = (lambda **k: _conv(kind, d=d, W=W, dtype=dtype, act=rng.choice(["silu", "none"]), state=state, views=views, **k)) if kind.startswith("conv") else \
        (lambda **k: _scan(kind, d=d, S=S, groups=groups, dtype=dtype, gate=rng.random() < 0.8, state=state, views=views, **k))
    if rng.random() < 0.4:
        return make(batch=1, T=total, lens=_split(rng, total, min(rng.randint(2, 12), total // 8)))
    B = rng.choice([1, 1, 2, 3, 4, 8])
    return make(batch=B, T=max(1, total // B))


# ---- inputs --------------------------------------------------------------------------------------------------------
def _lens(c):
    return [int(x) for x in c["lens"].split(",")] if c["lens"] else []


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    ru = lambda *s: torch.rand(*s, generator=g, device="cuda")
    dt, kind, d = _DT[c["dtype"]], c["kind"], c["d"]
    train = kind.endswith("train")
    leaf = lambda t: t.detach().requires_grad_(train)
    s = {"c": c}
    if kind.startswith("norm"):
        rows, sd = c["rows"], _DT[c["stream"]]
        s["x"], s["residual"] = leaf(rn(rows, d).to(dt)), leaf((2.0 * rn(rows, d)).to(sd))
        s["weight"] = leaf(1.0 + 0.1 * rn(d))
        s["post"] = leaf(1.0 + 0.1 * rn(d)) if c["post"] else None
        s["gate"] = leaf(rn(rows, d).to(dt)) if c["gate"] else None
        s["scale"] = leaf(0.5 + 0.1 * rn(d)) if c["scale"] else None
        if train:
            s["dy"], s["dr"] = rn(rows, d).to(dt), rn(rows, d).to(sd)
        return s
    B, T, lens = c["batch"], c["T"], _lens(c)
    N = len(lens) if lens else B
    s["cu"] = torch.tensor([sum(lens[:i]) for i in range(N + 1)], device="cuda") if lens else None
    if kind.startswith("conv"):
        W = c["W"]
        lead = (B,) if kind == "conv_step" else (B, T)
        x = rn(*lead, 2 * d if c["views"] else d).to(dt)
        s["x"] = leaf(x[..., :d])
        s["weight"], s["bias"] = leaf((rn(d, W) / math.sqrt(W)).to(dt)), leaf((0.1 * rn(d)).to(dt))
        s["state"] = leaf(rn(N, W - 1, d).to(dt)) if c["state"] else None
        if train:
            s["dy"], s["dstate"] = rn(B, T, d).to(dt), rn(N, W - 1, d).to(dt) if c["state"] else None
        return s
    S, G = c["S"], c["groups"]
    lead = (B,) if kind == "scan_step" else (B, T)
    # step sizes between a thousandth and a tenth about which the input moves them; decays from one to S, as they begin
    bias = torch.exp(math.log(1e-3) + (math.log(0.1) - math.log(1e-3)) * ru(d))
    s["dt_bias"] = leaf(bias + torch.log(-torch.expm1(-bias)))
    s["A"] = leaf(-torch.arange(1, S + 1, device="cuda").float() * torch.exp(0.1 * rn(d, S)))
    s["D"] = leaf(1.0 + 0.1 * rn(d))
    s["dt"] = leaf((0.5 * rn(*lead, d)).to(dt))
    xz = rn(*lead, 2 * d).to(dt)
    x, z = (xz[..., :d], xz[..., d:]) if c["views"] else (xz[..., :d].contiguous(), xz[..., d:].contiguous())
    s["x"], s["z"] = leaf(x), leaf(z) if c["gate"] else None
    inner = max(1, d // 32)
    proj = rn(*lead, inner + 2 * G * S).to(dt)
    b, cc = (proj[..., inner + i * G * S:inner + (i + 1) * G * S] for i in range(2))
    if not c["views"]:
        b, cc = b.contiguous(), cc.contiguous()
    s["B"], s["C"] = leaf(b.unflatten(-1, (G, S))), leaf(cc.unflatten(-1, (G, S)))
    s["h0"] = leaf(0.3 * rn(N, d, S)) if c["state"] else None
    if train:
        s["dy"], s["dh"] = rn(B, T, d).to(dt), rn(N, d, S) if c["state"] else None
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _f(t):
    return None if t is None else t.detach().float()


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _pieces(c):
    """(batch index or slice of it, first token, one behind the last, state index) of each group of sequences of one length."""
    if not c["lens"]:
        return [(slice(0, c["batch"]), 0, c["T"], slice(0, c["batch"]))]
    out, at = [], 0
    for i, n in enumerate(_lens(c)):
        out.append((slice(0, 1), at, at + n, slice(i, i + 1)))
        at += n
    return out


def _plain_conv(s, train):
    c, W, T = s["c"], s["c"]["W"], s["c"]["T"]
    x, w, b, st, dy, dst = (_f(s.get(k)) for k in ("x", "weight", "bias", "state", "dy", "dstate"))
    y = torch.empty_like(x)
    N = len(_lens(c)) if c["lens"] else c["batch"]
    last = x.new_zeros(N, W - 1, c["d"])
    dx, dw, db, dfirst = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b), torch.zeros_like(last)
    for bs, t0, t1, ns in _pieces(c):
        n = t1 - t0
        ext = torch.cat([st[ns] if st is not None else last[ns] * 0.0, x[bs, t0:t1]], dim=1)       # what the taps meet
        p = b + sum(w[:, j] * ext[:, j:j + n] for j in range(W))
        sg = _sigmoid(p)
        y[bs, t0:t1] = p * sg if c["act"] == "silu" else p
        last[ns] = ext[:, n:]
        if train:
            g = dy[bs, t0:t1] * (sg * (1.0 + p * (1.0 - sg))) if c["act"] == "silu" else dy[bs, t0:t1]
            de = torch.zeros_like(ext)
            if dst is not None:
                de[:, n:] += dst[ns]
            for j in range(W):
                de[:, j:j + n] += w[:, j] * g
                dw[:, j] += (g * ext[:, j:j + n]).sum((0, 1))
            db += g.sum((0, 1))
            dx[bs, t0:t1], dfirst[ns] = de[:, W - 1:], de[:, :W - 1]
    t = s["x"].dtype
    out = [y.to(t), last.to(t)]
    if train:
        out += [dx.to(t), dw.to(t), db.to(t)] + ([dfirst.to(t)] if st is not None else [])
    return out


def _plain_conv_step(s):
    x, w, b, st = (_f(s[k]) for k in ("x", "weight", "bias", "state"))
    ext = torch.cat([st, x[:, None]], dim=1)
    p = b + (ext * w.t()).sum(1)
    t = s["x"].dtype
    return [(p * _sigmoid(p) if s["c"]["act"] == "silu" else p).to(t), ext[:, 1:].to(t)]


def _step_size(dt, bias):
    v = dt + bias
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))


def _plain_scan(s, train):
    c, S, G, d = s["c"], s["c"]["S"], s["c"]["groups"], s["c"]["d"]
    x, dt, A, B, C, D, z, bias, h0, dy, dh = (_f(s.get(k)) for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "h0", "dy", "dh"))
    N = len(_lens(c)) if c["lens"] else c["batch"]
    wide = lambda t: t.repeat_interleave(d // G, dim=2)                     # [., T, G, S] for every channel
    y, last = torch.empty_like(x), x.new_zeros(N, d, S)
    gr = {k: torch.zeros_like(t) for k, t in (("x", x), ("dt", dt), ("A", A), ("B", B), ("C", C), ("D", D), ("bias", bias), ("h0", last))}
    gr["z"] = torch.zeros_like(x)
    for bs, t0, t1, ns in _pieces(c):
        n = t1 - t0
        cut = lambda t: t[bs, t0:t1]
        X, B_, C_ = cut(x), wide(cut(B)), wide(cut(C))
        step = _step_size(cut(dt), bias)
        decay = torch.exp(step[..., None] * A)
        add = (step * X)[..., None] * B_
        h = h0[ns] if h0 is not None else last[ns] * 0.0
        hs = torch.empty_like(add)
        for t in range(n):
            h = torch.addcmul(add[:, t], decay[:, t], h)
            hs[:, t] = h
        last[ns] = h
        del add
        inner = (hs * C_).sum(-1) + D * X
        sg = _sigmoid(cut(z)) if z is not None else None
        gate = cut(z) * sg if z is not None else 1.0
        y[bs, t0:t1] = inner * gate
        if not train:
            continue
        e = cut(dy) * gate
        if z is not None:
            gr["z"][bs, t0:t1] = cut(dy) * inner * (sg * (1.0 + cut(z) * (1.0 - sg)))
        first = h0[ns] if h0 is not None else last[ns] * 0.0
        back = dh[ns] if dh is not None else last[ns] * 0.0
        gs = C_ * e[..., None]                                              # what reaches each state from its own output
        gr["C"][bs, t0:t1] = (e[..., None] * hs).unflatten(2, (G, d // G)).sum(3)
        for t in range(n - 1, -1, -1):
            gs[:, t] += back
            back = decay[:, t] * gs[:, t]
        gr["h0"][ns] = back
        u = decay
        u[:, 1:] *= hs[:, :-1]
        u[:, 0] *= first
        del hs
        through = gs * u
        gr["A"] += (through * step[..., None]).sum((0, 1))
        dstep = (through * A).sum(-1)
        del through
        dadd = (gs * B_).sum(-1)
        gr["B"][bs, t0:t1] = (gs * (step * X)[..., None]).unflatten(2, (G, d // G)).sum(3)
        gr["x"][bs, t0:t1] = dadd * step + D * e
        raw = (dstep + dadd * X) * _sigmoid(cut(dt) + bias)
        gr["dt"][bs, t0:t1] = raw
        gr["bias"] += raw.sum((0, 1))
        gr["D"] += (e * X).sum((0, 1))
    t = s["x"].dtype
    out = [y.to(t), last]
    if train:
        out += [gr["x"].to(t), gr["dt"].to(t), gr["A"], gr["B"].to(t), gr["C"].to(t), gr["D"], gr["bias"]]
        out += ([gr["z"].to(t)] if z is not None else []) + ([gr["h0"]] if h0 is not None else [])
    return out


def _plain_scan_step(s):
    c = s["c"]
    x, dt, A, B, C, D, z, bias, h = (_f(s.get(k)) for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "h0"))
    wide = lambda t: t.repeat_interleave(c["d"] // c["groups"], dim=1)
    step = _step_size(dt, bias)
    h = torch.exp(step[..., None] * A) * h + (step * x)[..., None] * wide(B)
    y = (h * wide(C)).sum(-1) + D * x
    if z is not None:
        y = y * (z * _sigmoid(z))
    return [y.to(s["x"].dtype), h]


_EPS = 1e-5


def _plain_norm(s, train):
    x, res, w, post, gate, scale, dy, dr = (_f(s.get(k)) for k in ("x", "residual", "weight", "post", "gate", "scale", "dy", "dr"))
    inv = lambda t: 1.0 / torch.sqrt((t * t).mean(-1, keepdim=True) + _EPS)
    ix = inv(x) if post is not None else None
    p = x * ix * post if post is not None else x
    sg = _sigmoid(gate) if gate is not None else 1.0
    u = p * sg
    r = res + (u * scale if scale is not None else u)
    ir = inv(r)
    y = r * ir * w
    t, sd = s["x"].dtype, s["residual"].dtype
    out = [y.to(t), r.to(sd)]
    if not train:
        return out
    rn = r * ir
    m = dy * w
    dr = dr + ir * (m - rn * (m * rn).mean(-1, keepdim=True))
    du = dr * scale if scale is not None else dr
    dp = du * sg
    dx = dp
    if post is not None:
        xn = x * ix
        q = dp * post
        dx = ix * (q - xn * (q * xn).mean(-1, keepdim=True))
    out += [dx.to(t), dr.to(sd), (dy * rn).sum(0)]
    out += [(dp * xn).sum(0)] if post is not None else []
    out += [(du * p * sg * (1.0 - sg)).to(t)] if gate is not None else []
    return out + ([(dr * u).sum(0)] if scale is not None else [])


# ---- one pass ------------------------------------------------------------------------------------------------------
def _leaves(s):
    """What gradients are asked of, in the order of the outputs."""
    names = {"c": ("x", "weight", "bias", "state"), "s": ("x", "dt", "A", "B", "C", "D", "dt_bias", "z", "h0"),
             "n": ("x", "residual", "weight", "post", "gate", "scale")}[s["c"]["kind"][0]]
    return [s[k] for k in names if s[k] is not None]


def _with_gradients(s, outs, gos):
    pairs = [(o, g) for o, g in zip(outs, gos) if g is not None]
    return [o.detach() for o in outs] + list(torch.autograd.grad([o for o, _ in pairs], _leaves(s), [g for _, g in pairs]))


def _own_call(s):
    lib, c, kind = _package(), s["c"], s["c"]["kind"]
    if kind == "conv_step":
        return lib.short_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation=_act(c))
    if kind.startswith("conv"):
        return lib.short_conv(s["x"], s["weight"], s["bias"], activation=_act(c), initial_state=s["state"], output_final_state=True, cu_seqlens=s["cu"])
    if kind == "scan_step":
        return lib.state_space_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["h0"], s["D"], s["z"], dt_bias=s["dt_bias"], dt_softplus=True)
    if kind.startswith("scan"):
        return lib.state_space_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], dt_bias=s["dt_bias"], dt_softplus=True,
                                    initial_state=s["h0"], output_final_state=True, cu_seqlens=s["cu"])
    return lib.block_norm(s["x"], s["residual"], s["weight"], post_weight=s["post"], gate=s["gate"], gate_act="sigmoid",
                          residual_scale=1.0 if s["scale"] is None else s["scale"], eps=_EPS)


def _act(c):
    return "silu" if c["act"] == "silu" else None


def run(state):
    s, kind = state, state["c"]["kind"]
    train = kind.endswith("train")
    if own:
        if not train:
            with torch.no_grad():
                return list(_own_call(s))
        return _with_gradients(s, _own_call(s), (s["dy"], s["dr"] if kind[0] == "n" else s["dstate"] if kind[0] == "c" else s["dh"]))
    with torch.no_grad():
        if kind == "conv_step":
            return _plain_conv_step(s)
        if kind == "scan_step":
            return _plain_scan_step(s)
        return (_plain_conv if kind[0] == "c" else _plain_scan if kind[0] == "s" else _plain_norm)(s, train)


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    """Token after token from the definitions, gradients by differentiating them."""
    s = prepare(case, seed)
    kind = case["kind"]
    train = kind.endswith("train")
    for k, v in list(s.items()):
        if torch.is_tensor(v) and v.is_floating_point():
            s[k] = v.detach().double().requires_grad_(train)
    with torch.set_grad_enabled(train):
        outs = {"c": _exact_conv, "s": _exact_scan, "n": _exact_norm}[kind[0]](s)
    if not train:
        return outs
    return _with_gradients(s, outs, (s["dy"], s["dr"] if kind[0] == "n" else s["dstate"] if kind[0] == "c" else s["dh"]))


def _spans(c):
    """(batch row, first token, one behind the last) of each sequence."""
    if c["lens"]:
        ends = [sum(_lens(c)[:i]) for i in range(len(_lens(c)) + 1)]
        return [(0, a, b) for a, b in zip(ends, ends[1:])]
    return [(b, 0, c["T"]) for b in range(c["batch"])]


def _exact_conv(s):
    c, W = s["c"], s["c"]["W"]
    one = c["kind"] == "conv_step"
    x = s["x"][:, None] if one else s["x"]
    ys, lasts = [], []
    for i, (b, t0, t1) in enumerate(_spans(dict(c, T=1))) if one else enumerate(_spans(c)):
        before = s["state"][i] if s["state"] is not None else x.new_zeros(W - 1, c["d"])
        seen = torch.cat([before, x[b, t0:t1]])
        p = (seen.unfold(0, W, 1) * s["weight"]).sum(-1) + s["bias"]
        ys.append(torch.nn.functional.silu(p) if c["act"] == "silu" else p)
        lasts.append(seen[len(seen) - (W - 1):])
    y = torch.cat(ys).reshape(x.shape)
    return [y[:, 0] if one else y, torch.stack(lasts)]


def _exact_scan(s):
    c, G, d = s["c"], s["c"]["groups"], s["c"]["d"]
    one = c["kind"] == "scan_step"
    tok = (lambda t: t[:, None]) if one else (lambda t: t)
    step = torch.nn.functional.softplus(tok(s["dt"]) + s["dt_bias"], threshold=1e4)
    # sequences of one length side by side, each group token after token
    spans = _spans(dict(c, T=1) if one else c)
    batched = not c["lens"]
    ys, lasts = [], []
    for i, (b, t0, t1) in enumerate(spans[:1] if batched else spans):
        rows, ns = (slice(0, c["batch"]), slice(0, c["batch"])) if batched else (slice(0, 1), slice(i, i + 1))
        h = s["h0"][ns] if s["h0"] is not None else step.new_zeros(c["batch"] if batched else 1, d, c["S"])
        h = h.unflatten(1, (G, d // G))
        X, E, Bs, Cs = (tok(s[k])[rows, t0:t1].unbind(1) if k else step[rows, t0:t1].unbind(1) for k in ("x", None, "B", "C"))
        A = s["A"].unflatten(0, (G, d // G))
        out = []
        for xt, et, Bt, Ct in zip(X, E, Bs, Cs):
            et, xt = et.unflatten(1, (G, d // G)), xt.unflatten(1, (G, d // G))
            h = torch.exp(et[..., None] * A) * h + (et * xt)[..., None] * Bt[:, :, None]
            out.append((h * Ct[:, :, None]).sum(-1).flatten(1))
        ys.append(torch.stack(out, 1))
        lasts.append(h.flatten(1, 2))
    y = torch.cat(ys, 1) + s["D"] * tok(s["x"])
    if s["z"] is not None:
        y = y * torch.nn.functional.silu(tok(s["z"]))
    return [y[:, 0] if one else y, torch.cat(lasts)]


def _exact_norm(s):
    rms = lambda t: torch.sqrt(t.pow(2).mean(-1, keepdim=True) + _EPS)
    p = s["x"] / rms(s["x"]) * s["post"] if s["post"] is not None else s["x"]
    if s["gate"] is not None:
        p = p * torch.sigmoid(s["gate"])
    r = s["residual"] + (p if s["scale"] is None else s["scale"] * p)
    return [r / rms(r) * s["weight"], r]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    """Bytes: every input once, every output once.  Operations: of the formulas themselves, an exponential counted as one."""
    c = case
    d, es = c["d"], _ES[c["dtype"]]
    if c["kind"].startswith("norm"):
        n, sb = c["rows"] * d, _ES[c["stream"]]
        vectors = 1 + c["post"] + c["scale"]
        fwd = n * (es * (2 + c["gate"]) + 2 * sb) + 4 * d * vectors
        ops = n * (6 + 5 * c["post"] + 5 * c["gate"])
        if c["kind"] == "norm":
            return {"bytes": fwd, "flops": ops}
        return {"bytes": fwd + n * (es * (2 + c["gate"]) + 2 * sb) + 4 * d * vectors, "flops": 3 * ops}
    N = len(_lens(c)) if c["lens"] else c["batch"]
    n = c["batch"] * c["T"] * d
    if c["kind"].startswith("conv"):
        W = c["W"]
        states = N * (W - 1) * d * es
        fwd = 2 * n * es + (W + 1) * d * es + states * (1 + c["state"])
        ops = n * (2 * W + 1 + 5 * (c["act"] == "silu"))
        if c["kind"] != "conv_train":
            return {"bytes": fwd, "flops": ops}
        return {"bytes": fwd + 2 * n * es + (W + 1) * d * es + 2 * states * c["state"], "flops": 3 * ops}
    S, groups = c["S"], c["groups"]
    states, inner = N * d * S * 4, c["batch"] * c["T"] * groups * S * es
    fwd = n * es * (3 + c["gate"]) + 2 * inner + states * (1 + c["state"]) + 4 * d * (S + 2)
    ops = n * (7 * S + 10)
    if c["kind"] != "scan_train":
        return {"bytes": fwd, "flops": ops}
    return {"bytes": fwd + n * es * (3 + c["gate"]) + 2 * inner + 2 * states * c["state"] + 4 * d * (S + 2), "flops": 3 * ops}

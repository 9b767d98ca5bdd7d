"""The operators of a state space block from their definitions, in float64 on the CPU, token after token; gradients by autograd.

Beside each result stands how large the terms are that it is a sum of (`*_magnitudes`): what a 32-bit evaluation may be off by is a number of roundings
times 2^-24 times that."""
import torch


def spans(B, T, cu=None):
    """(batch row, first token, one behind the last) of each sequence."""
    if cu is None:
        return [(b, 0, T) for b in range(B)]
    cu = [int(c) for c in cu]
    return [(0, a, b) for a, b in zip(cu, cu[1:])]


def silu(x):
    return x * torch.sigmoid(x)


def short_conv(x, w, bias=None, state=None, act=False, cu=None):
    """x [B, T, D], w [D, W], state [N, W-1, D]; returns y (rows of no sequence zero) and the final states."""
    B, T, D = x.shape
    W = w.shape[1]
    y, last = torch.zeros_like(x), []
    parts = []
    for n, (b, t0, t1) in enumerate(spans(B, T, cu)):
        before = x.new_zeros(W - 1, D) if state is None else state[n]
        seen = torch.cat([before, x[b, t0:t1]])
        if t1 > t0:
            p = (seen.unfold(0, W, 1) * w).sum(-1)
            p = p if bias is None else p + bias
            parts.append((b, t0, t1, silu(p) if act else p))
        last.append(seen[seen.shape[0] - (W - 1):])
    for b, t0, t1, p in parts:
        y = y.index_put((torch.full((t1 - t0,), b), torch.arange(t0, t1)), p)
    return y, torch.stack(last)


def step_sizes(dt, bias, softplus):
    v = dt if bias is None else dt + bias
    return torch.nn.functional.softplus(v, threshold=1e4) if softplus else v


def scan(x, dt, A, B, C, D=None, z=None, bias=None, softplus=False, h0=None, cu=None):
    """x, dt, z [B, T, D], A [D, S], B, C [B, T, G, S], h0 [N, D, S]; returns y (rows of no sequence zero) and the final states."""
    nb, T, d = x.shape
    G = B.shape[2]
    delta = step_sizes(dt, bias, softplus)
    y, last = torch.zeros_like(x), []
    for n, (b, t0, t1) in enumerate(spans(nb, T, cu)):
        h = x.new_zeros(A.shape) if h0 is None else h0[n]
        out = []
        for t in range(t0, t1):
            Bt, Ct = (v[b, t].repeat_interleave(d // G, 0) for v in (B, C))
            h = torch.exp(delta[b, t][:, None] * A) * h + (delta[b, t] * x[b, t])[:, None] * Bt
            out.append((h * Ct).sum(-1))
        if out:
            o = torch.stack(out)
            o = o if D is None else o + D * x[b, t0:t1]
            o = o if z is None else o * silu(z[b, t0:t1])
            y = y.index_put((torch.full((t1 - t0,), b), torch.arange(t0, t1)), o)
        last.append(h)
    return y, torch.stack(last)


def scan_magnitudes(x, dt, A, B, C, D=None, z=None, bias=None, softplus=False, h0=None, cu=None, dy=None, dht=None):
    """Every output of the scan and of its backward pass with each term taken by its absolute value, and the sum of the roundings that a path of
    such terms passes through, in units of 2^-24: (dict of magnitudes, count)."""
    nb, T, d = x.shape
    G, S = B.shape[2], A.shape[1]
    f = lambda t: None if t is None else t.detach().double().abs()
    v = (dt if bias is None else dt + bias).detach().double()
    delta = (torch.nn.functional.softplus(v, threshold=1e4) if softplus else v).abs()
    decay = torch.exp(step_sizes(dt, bias, softplus).detach()[..., None] * A.detach())        # [B, T, D, S]
    X, Ab, Bb, Cb, Dd, zz, H0, dY, dH = (f(t) for t in (x, A, B, C, D, z, h0, dy, dht))
    zd = None if z is None else z.detach().double()
    gate = torch.ones_like(X) if z is None else silu(zd).abs()
    sl = None if z is None else (torch.sigmoid(zd) * (1 + zd * (1 - torch.sigmoid(zd)))).abs() + 0.1
    wide = lambda t: t.repeat_interleave(d // G, 2)
    Bw, Cw = wide(Bb), wide(Cb)
    seqs = spans(nb, T, cu)
    m = {k: torch.zeros_like(t) for k, t in (("y", X), ("x", X), ("dt", X), ("z", X), ("A", Ab), ("B", Bb), ("C", Cb))}
    m["D"], m["bias"] = torch.zeros(d, dtype=torch.float64), torch.zeros(d, dtype=torch.float64)
    m["ht"], m["h0"] = torch.zeros(len(seqs), d, S, dtype=torch.float64), torch.zeros(len(seqs), d, S, dtype=torch.float64)
    group = lambda t: t.unflatten(0, (G, d // G)).sum(1)
    for n, (b, t0, t1) in enumerate(seqs):
        h = torch.zeros(d, S, dtype=torch.float64) if H0 is None else H0[n]
        hs = [h]
        for t in range(t0, t1):
            h = decay[b, t] * h + (delta[b, t] * X[b, t])[:, None] * Bw[b, t]
            hs.append(h)
            inner = (h * Cw[b, t]).sum(-1) + (0 if Dd is None else Dd * X[b, t])
            m["y"][b, t] = inner * gate[b, t]
            if dY is not None and z is not None:
                m["z"][b, t] = dY[b, t] * inner * sl[b, t]
        m["ht"][n] = h
        if dY is None:
            continue
        g = torch.zeros(d, S, dtype=torch.float64) if dH is None else dH[n]
        for t in range(t1 - 1, t0 - 1, -1):
            e = dY[b, t] * gate[b, t]
            g = g + Cw[b, t] * e[:, None]
            before = decay[b, t] * hs[t - t0]
            m["C"][b, t] = group(e[:, None] * hs[t - t0 + 1])
            m["B"][b, t] = group(g * (delta[b, t] * X[b, t])[:, None])
            m["x"][b, t] = delta[b, t] * (g * Bw[b, t]).sum(-1) + (0 if Dd is None else Dd * e)
            raw = (g * (Ab * before + X[b, t][:, None] * Bw[b, t])).sum(-1)
            m["dt"][b, t] = raw
            m["bias"] += raw
            m["A"] += g * delta[b, t][:, None] * before
            m["D"] += e * X[b, t]
            g = decay[b, t] * g
        m["h0"][n] = g
    longest = max([t1 - t0 for _, t0, t1 in seqs] + [1])
    # a step's decay: two roundings of its exponent (times the exponent) and the exponential's; delta's own; the product, the sum
    step = 3 * float((delta[..., None] * Ab).max() if T else 0) + 2 * float(v.abs().max() if T else 0) + 10
    return m, 2 * longest * step + T * nb + d + 64


def scan_bounds(x, dt, A, B, C, D=None, z=None, bias=None, softplus=False, h0=None, cu=None, dy=None, dht=None):
    """How far each output and gradient of the scan may be off in 32 bits, element by element: errors go through the recurrences as the values do and fade with them.

    u = 2^-24 is half a step.  To first order, with every term by its absolute value:
      v = dt + bias            u |v|
      delta = softplus(v)      sigmoid(v) u |v| from v; e = exp(-|v|) is off by 2 |v| + 2 (its exponent's product and constant, the exponential's last place), the rest of log(1 + e) by 8;
                               the sum by one:  u (sigmoid(v) |v| + 10 delta + 2 |v| log(1 + e))
      a = exp(delta A)         relative: |A| err(delta) from delta; of the exponent's own 3 u |delta A|, and 8 more where a piece's decay comes from a sum of eight steps; 2 u of the
                               exponential, 2 u of products of pieces' decays:  rho = |A| err(delta) + u (11 |delta A| + 4); what underflows is off by 2^-125
      b = delta x B            |x B| err(delta) + 2 u |b|
      h' = a h + b             a err(h) + (a rho) |h| + err(b) + 3 u |h'|: the walk from zero, the chain over the pieces, the walk from what enters
      sums over states         four in a lane, at most four exchanges, a product: 10 u
      sigmoid                  relative: (2 |z| + 2) (1 - s) of its exponential, 4 of sum and reciprocal
      sums over channels       a lane's exchanges and a block after the other, at least four channels each: u (8 + channels / 4)
    The gradients g of h go back by the same recurrence.  Sums over all n tokens (dA, dD, d bias) are off by no more than the sum of their terms' bounds and u (n + 16) of the sum of the
    terms.  Where n is large that is far: roundings do not all fall to one side.  Of errors that are as likely up as down, each within its own bound, the sum's standard deviation is the
    root of the bounds' squares over 1.7; a rounding that stays in a state for w tokens is w times in the sum, and its tokens' bounds are w times as large.  Four times that root is seven
    standard deviations, and the smaller of the two is taken."""
    u, tiny = 2.0 ** -24, 2.0 ** -125
    nb, T, d = x.shape
    G, S = B.shape[2], A.shape[1]
    f = lambda t: None if t is None else t.detach().double()
    x, dt, A, B, C, D, z, bias, h0, dy, dht = (f(t) for t in (x, dt, A, B, C, D, z, bias, h0, dy, dht))
    v = dt if bias is None else dt + bias
    if softplus:
        s, log = torch.sigmoid(v), torch.log1p(torch.exp(-v.abs()))
        delta = v.clamp(min=0) + log
        ed = u * (s * v.abs() + 10 * delta + 2 * v.abs() * log)
        slope, eslope = s, u * s * (4 + 2 * (3 * v.abs() + 2) * torch.sigmoid(-v))
    else:
        delta, ed, slope, eslope = v, u * v.abs(), torch.ones_like(v), torch.zeros_like(v)
    X, size = x.abs(), delta.abs()
    if z is None:
        gate, egate, sl, SL, esl = torch.ones_like(x), torch.zeros_like(x), None, None, None
    else:
        s, r = torch.sigmoid(z), torch.sigmoid(-z)
        es = u * s * ((2 * z.abs() + 2) * r + 4)
        gate, egate = z.abs() * s, z.abs() * es
        sl, SL = (s * (1 + z * r)).abs(), s * (1 + z.abs() * r)
        esl = es * (1 + z * r).abs() + s * z.abs() * es + 3 * u * SL
    wide = lambda t: t.abs().repeat_interleave(d // G, 0)                    # [G, S] for every channel
    group = lambda t: t.unflatten(0, (G, d // G)).sum(1)
    seqs = spans(nb, T, cu)
    out = {k: torch.zeros_like(t) for k, t in (("y", x), ("x", x), ("dt", x), ("z", x), ("A", A), ("B", B), ("C", C))}
    zeros = lambda *n: x.new_zeros(*n)
    out["D"], out["bias"], out["ht"], out["h0"] = zeros(d), zeros(d), zeros(len(seqs), d, S), zeros(len(seqs), d, S)
    sums = {k: [torch.zeros_like(out[k]) for _ in range(3)] for k in ("A", "D", "bias")}      # over tokens: of bounds, of their squares, of terms

    def token(k, bound, term):
        for to, t in zip(sums[k], (bound, bound * bound, term)):
            to += t

    Aa = A.abs()

    def decay(b, t):
        a = torch.exp(delta[b, t][:, None] * A)
        rho = Aa * ed[b, t][:, None] + u * (11 * size[b, t][:, None] * Aa + 4)
        return a, torch.where(a > 0, a * rho, 0 * a) + tiny * ((a > 0) & (a < 2.0 ** -100))

    for n, (b, t0, t1) in enumerate(seqs):
        h = zeros(d, S) if h0 is None else h0[n].abs()
        eh = torch.zeros_like(h)
        hs, ehs = [h], [eh]
        I, eI = [], []
        for t in range(t0, t1):
            a, ea = decay(b, t)
            Bt, Ct = wide(B[b, t]), wide(C[b, t])
            add = (size[b, t] * X[b, t])[:, None] * Bt
            eb = (X[b, t] * ed[b, t])[:, None] * Bt + 2 * u * add
            eh = a * eh + ea * h + eb
            h = a * h + add
            eh = eh + 3 * u * h
            hs.append(h)
            ehs.append(eh)
            inner = (h * Ct).sum(-1) + (0 if D is None else (D * x[b, t]).abs())
            ei = (eh * Ct).sum(-1) + 10 * u * inner
            I.append(inner)
            eI.append(ei)
            out["y"][b, t] = gate[b, t] * ei + inner * egate[b, t] + 2 * u * inner * gate[b, t]
        out["ht"][n] = eh
        if dy is None:
            continue
        g = zeros(d, S) if dht is None else dht[n].abs()
        eg = torch.zeros_like(g)
        channels = u * (8 + d // G / 4)
        for t in range(t1 - 1, t0 - 1, -1):
            i = t - t0
            a, ea = decay(b, t)
            Bt, Ct = wide(B[b, t]), wide(C[b, t])
            Y, Dl, Ed, Xt = dy[b, t].abs(), size[b, t], ed[b, t], X[b, t]
            e = Y * gate[b, t]
            ee = Y * egate[b, t] + 2 * u * e
            g = g + Ct * e[:, None]
            eg = eg + Ct * ee[:, None] + 3 * u * g
            out["C"][b, t] = group(hs[i + 1] * ee[:, None] + ehs[i + 1] * e[:, None] + channels * hs[i + 1] * e[:, None])
            add, eadd = Dl * Xt, Xt * Ed + u * Dl * Xt
            out["B"][b, t] = group(eg * add[:, None] + g * eadd[:, None] + channels * g * add[:, None])
            gb = (g * Bt).sum(-1)
            egb = (eg * Bt).sum(-1) + 10 * u * gb
            th = a * g * hs[i]
            eth = a * eg * hs[i] + ea * g * hs[i] + a * g * ehs[i] + 3 * u * th
            ga = (Aa * th).sum(-1)
            ega = (Aa * eth).sum(-1) + 14 * u * ga
            De = 0 if D is None else D.abs() * e
            out["x"][b, t] = Dl * egb + gb * Ed + (0 if D is None else D.abs() * ee) + 3 * u * (gb * Dl + De)
            raw, eraw = gb * Xt + ga, Xt * egb + ega + 2 * u * (gb * Xt + ga)
            out["dt"][b, t] = slope[b, t] * eraw + raw * eslope[b, t] + u * raw * slope[b, t]
            token("A", Dl[:, None] * eth + th * Ed[:, None], Dl[:, None] * th)
            token("D", Xt * ee, e * Xt)
            token("bias", out["dt"][b, t], raw * slope[b, t])
            if z is not None:
                out["z"][b, t] = Y * (eI[i] * sl[b, t] + I[i] * esl[b, t] + 2 * u * I[i] * SL[b, t])
            eg = a * eg + ea * g
            g = a * g
        out["h0"][n] = eg + u * g
    count = nb * T + 16
    for k, (bound, squares, term) in sums.items():
        out[k] = torch.minimum(bound + count * u * term, 4 * squares.sqrt() + 4 * count ** 0.5 * u * term)
    return out


def gate_sigmoid(g):
    """The sigmoid with the derivative s sigmoid(-g): torch.sigmoid's s (1 - s) is zero above 37 in float64."""
    return torch.exp(torch.nn.functional.logsigmoid(g))


def block_norm(x, residual=None, weight=None, post_norm=False, post_weight=None, gate=None, act="sigmoid", scale=1.0, eps=1e-5):
    rms = lambda t: torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps)
    p = x / rms(x) if post_norm or post_weight is not None else x
    p = p if post_weight is None else p * post_weight
    if gate is not None:
        p = p * (gate_sigmoid(gate) if act == "sigmoid" else silu(gate) if act == "silu" else gate)
    r = scale * p if residual is None else residual + scale * p
    y = r / rms(r)
    return (y if weight is None else y * weight), r


def block_norm_magnitudes(x, residual=None, weight=None, post_norm=False, post_weight=None, gate=None, act="sigmoid", scale=1.0, eps=1e-5, dy=None, dr=None):
    """As scan_magnitudes, for block_norm: (dict, count)."""
    f = lambda t: t.detach().double() if isinstance(t, torch.Tensor) else t
    x, residual, weight, post_weight, gate, scale, dy, dr = (f(t) for t in (x, residual, weight, post_weight, gate, scale, dy, dr))
    E = x.shape[-1]
    inv = lambda t: 1 / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps)
    one = torch.ones(E, dtype=torch.float64)
    w, pw = (one if t is None else t.abs() for t in (weight, post_weight))
    sc = scale.abs() if isinstance(scale, torch.Tensor) else abs(scale) * one
    normed = post_norm or post_weight is not None
    ix = inv(x) if normed else 1.0
    xh = (x * ix).abs()
    p = xh * (pw if normed else 1)
    if gate is None:
        a, da = torch.ones_like(x), torch.zeros_like(x)
    else:
        s = torch.sigmoid(gate)
        a, da = {"sigmoid": (s, s * torch.sigmoid(-gate)), "silu": ((gate * s).abs(), (s * (1 + gate * (1 - s))).abs() + 0.1)}.get(act, (gate.abs(), torch.ones_like(x)))
    u = p * a
    r = sc * u + (0 if residual is None else residual.abs())
    _, true = block_norm(x, residual, weight, post_norm, post_weight, gate, act, scale, eps)
    ir = inv(true)
    rh = r * ir
    m = {"y": rh * w, "r": r}
    dy = torch.zeros_like(x) if dy is None else dy.abs()
    dr = torch.zeros_like(x) if dr is None else dr.abs()
    k = dy * w
    t = dr + ir * (k + rh * (k * rh).mean(-1, keepdim=True))
    m["residual"] = t
    m["weight"], m["scale"] = (dy * rh).flatten(0, -2).sum(0), (t * u).flatten(0, -2).sum(0)
    du = t * sc
    m["gate"] = du * p * da
    dp = du * a
    m["post_weight"] = (dp * xh).flatten(0, -2).sum(0)
    q = dp * pw
    m["x"] = ix * (q + xh * (q * xh).mean(-1, keepdim=True)) if normed else dp
    # a row's sums: a lane's, then across lanes; each 1 / rms a division and a root; two norms one behind the other, forwards and back
    rows = x.numel() // E
    return m, 4 * (E // 64 + 24) + rows + 64

"""Plain float64 implementations of the sequence operators, token by token, with the scale of every output's terms.

Each function returns {name: (value, scale)}: ``scale`` is the same sum with the absolute value of every term, so that a computation
whose every product and partial sum is off by k roundings of fp32 is within k * 2^-24 * scale of ``value``."""
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, ref, k, dtype, what=""):
    """|got - value| <= k fp32 roundings of the terms' scale + one rounding to the output type (and its smallest step)."""
    value, scale = ref
    assert tuple(got.shape) == tuple(value.shape), (what, got.shape, value.shape)
    out = got.detach().double().cpu()
    bound = k * U32 * scale + half_step(got.dtype) * (value.abs() + k * U32 * scale) + torch.finfo(got.dtype).tiny * half_step(got.dtype) * 2
    assert torch.isfinite(out).all(), f"{what}: not finite"
    off = (out - value).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound (largest error {off.max().item():.3g})"
    assert got.dtype == dtype, (what, got.dtype)


def lengths_or_full(lengths, B, L):
    return [L] * B if lengths is None else [min(max(int(n), 0), L) for n in lengths]


# ---- selective scan ----------------------------------------------------------------------------------------------------------
def softplus64(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _scan(step, decay, u, A, B, C, D, gate, dgate, sig, dy, h0, dh_end, ns):
    """All tensors (batch, L, ...) float64, B and C already per channel.  The recurrence and its gradients, written out."""
    Bt, L, dim = u.shape
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)      # noqa: E731
    N = A.shape[1]
    y, hT = z(Bt, L, dim), z(Bt, dim, N)
    g = {k: z(Bt, L, dim) for k in ("du", "ddelta", "dz")}
    gB, gC, dA, dD, dh0 = z(Bt, L, dim, N), z(Bt, L, dim, N), z(dim, N), z(dim), z(Bt, dim, N)
    dbias = z(dim)
    for b in range(Bt):
        h = [h0[b]]
        for t in range(ns[b]):
            h.append(decay[b, t] * h[-1] + (step[b, t] * u[b, t])[:, None] * B[b, t])
            inner = (C[b, t] * h[-1]).sum(-1) + D * u[b, t]
            y[b, t] = inner * gate[b, t]
            g["dz"][b, t] = dy[b, t] * inner * dgate[b, t]
        hT[b] = h[-1]
        carry = dh_end[b]
        for t in reversed(range(ns[b])):
            d = dy[b, t] * gate[b, t]
            k = C[b, t] * d[:, None] + carry
            w = k * decay[b, t] * h[t]
            SG = (k * B[b, t]).sum(-1)
            dstep = (w * A).sum(-1) + SG * u[b, t]
            g["ddelta"][b, t] = dstep * sig[b, t]
            g["du"][b, t] = SG * step[b, t] + d * D
            gB[b, t] = k * (step[b, t] * u[b, t])[:, None]
            gC[b, t] = h[t + 1] * d[:, None]
            dA += w * step[b, t][:, None]
            dD += d * u[b, t]
            dbias += g["ddelta"][b, t]
            carry = decay[b, t] * k
        dh0[b] = carry
    return {"y": y, "state": hT, **g, "dB": gB, "dC": gC, "dA": dA, "dD": dD, "ddelta_bias": dbias, "dstate": dh0}


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=True, state=None, lengths=None, dout=None, dstate_out=None):
    """{name: (value, scale)} of y, state and, with dout, every gradient."""
    f = lambda t: None if t is None else t.detach().double().cpu()       # noqa: E731
    u, delta, A, B, C, D, z, delta_bias, state, dout, dstate_out = map(f, (u, delta, A, B, C, D, z, delta_bias, state, dout, dstate_out))
    Bt, L, dim = u.shape
    N = A.shape[1]
    ns = lengths_or_full(lengths, Bt, L)
    if B.dim() == 3:
        B = B[:, :, None]
    if C.dim() == 3:
        C = C[:, :, None]
    G = B.shape[2]
    live = torch.zeros(Bt, L, dtype=torch.bool)
    for b, n in enumerate(ns):
        live[b, :n] = True
    keep = lambda t: torch.where(live.view(Bt, L, *[1] * (t.dim() - 2)), t, torch.zeros((), dtype=torch.float64))    # noqa: E731
    u, delta, B, C = keep(u), keep(delta), keep(B), keep(C)
    z = keep(z) if z is not None else None
    dy = keep(dout) if dout is not None else torch.zeros_like(u)
    raw = delta + (delta_bias if delta_bias is not None else 0.0)
    step = softplus64(raw) if softplus else raw
    sig = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    gate = torch.ones_like(u) if z is None else z * torch.sigmoid(z)
    dgate = torch.zeros_like(u) if z is None else torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))
    Dv = torch.zeros(dim, dtype=torch.float64) if D is None else D
    h0 = torch.zeros(Bt, dim, N, dtype=torch.float64) if state is None else state
    dhe = torch.zeros(Bt, dim, N, dtype=torch.float64) if dstate_out is None else dstate_out
    decay = torch.exp(step[..., None] * A)
    per = lambda t: t.repeat_interleave(dim // G, 2)                    # noqa: E731
    args = (u, A, per(B), per(C), Dv, gate, dgate, sig, dy, h0, dhe)
    val = _scan(step, decay, *args, ns)
    sca = _scan(step.abs(), decay, *[a.abs() for a in args], ns)
    # the gate's derivative is a sum of terms of both signs: its scale is that of the terms
    if z is not None:
        sg = torch.sigmoid(z)
        sca["dz"] = _scan(step.abs(), decay, *[a.abs() for a in args[:6]], sg * (1 + z.abs() * (1 - sg)), *[a.abs() for a in args[7:]], ns)["dz"]
    for k in ("dB", "dC"):
        for r in (val, sca):
            r[k] = r[k].view(Bt, L, G, dim // G, N).sum(3)
    return {k: (val[k], sca[k]) for k in val}


def scan_roundings(A, delta, delta_bias, softplus, L, N):
    """Roundings per term: a state passes at most L tokens; a decay exp(step A) is off by |step A| (8 u: softplus' 6, the product's and
    log2 e's) + 2 u (the exponential), a product with step or a gate by at most 16 u; sums over states, channels and tokens add at most
    N / 4 + 64 (a quad's lanes, then trees) and 64 per tile of a chain."""
    raw = delta.double().cpu() + (delta_bias.double().cpu() if delta_bias is not None else 0.0)
    raw = raw[torch.isfinite(raw)]
    step = softplus64(raw) if softplus else raw.abs()
    reach = min(float(step.max()) * float(A.abs().max()), 30.0)      # where |step A| is larger, the term has died out
    return (8 * reach + 12) * min(L, 64) + L + N + 96


# ---- causal convolution ----------------------------------------------------------------------------------------------------------
def _conv(x, w, bias, state, ns, silu, dout, dstate_out, absolute):
    a = (lambda t: t.abs()) if absolute else (lambda t: t)
    Bt, L, D = x.shape
    K = w.shape[1]
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)      # noqa: E731
    y, last, dx, dst, dw, db = z(Bt, L, D), z(Bt, K - 1, D), z(Bt, L, D), z(Bt, K - 1, D), z(D, K), z(D)
    for b in range(Bt):
        n = ns[b]
        line = torch.cat([state[b], x[b, :n]], 0)
        last[b] = line[n:n + K - 1]
        dline = z(n + K - 1, D)
        dline[n:] += a(dstate_out[b])
        for t in range(n):
            p = bias.clone()
            pa = bias.abs()
            for k in range(K):
                p = p + w[:, k] * line[t + k]
                pa = pa + (w[:, k] * line[t + k]).abs()
            s = torch.sigmoid(p)
            # |act'| <= 1.1 and |act''| <= 0.5: an error of the sum p moves the value by at most 1.1 of it and the slope by 0.5 of it
            if silu:
                y[b, t] = 1.1 * pa if absolute else p * s
                slope = s * (1 + p.abs() * (1 - s)) + 0.5 * pa if absolute else s * (1 + p * (1 - s))
            else:
                y[b, t], slope = (pa if absolute else p), torch.ones_like(p)
            dp = a(dout[b, t]) * slope
            db += dp
            for k in range(K):
                dline[t + k] += a(w[:, k]) * dp
                dw[:, k] += a(line[t + k]) * dp
        dx[b, :n] = dline[K - 1:]
        dst[b] = dline[:K - 1]
    return {"y": y, "state": last, "dx": dx, "dstate": dst, "dweight": dw, "dbias": db}


def causal_conv(x, weight, bias=None, state=None, lengths=None, silu=True, dout=None, dstate_out=None):
    f = lambda t: None if t is None else t.detach().double().cpu()       # noqa: E731
    x, weight, bias, state, dout, dstate_out = map(f, (x, weight, bias, state, dout, dstate_out))
    Bt, L, D = x.shape
    K = weight.shape[1]
    zeros = torch.zeros(Bt, K - 1, D, dtype=torch.float64)
    ns = lengths_or_full(lengths, Bt, L)
    args = (x, weight, torch.zeros(D, dtype=torch.float64) if bias is None else bias, zeros if state is None else state, ns, silu,
            torch.zeros_like(x) if dout is None else dout, zeros if dstate_out is None else dstate_out)
    val, sca = _conv(*args, False), _conv(*args, True)
    return {k: (val[k], sca[k]) for k in val}


# ---- the norms around a block ----------------------------------------------------------------------------------------------------
def norm_residual(y, pre_w, residual=None, post_w=None, gate=None, scale=None, gate_act="silu", eps=1e-5, dnormed=None, dresidual_out=None):
    f = lambda t: None if t is None else t.detach().double().cpu()       # noqa: E731
    y, v, r0, w, g, s, dn, dr0 = map(f, (y, pre_w, residual, post_w, gate, scale, dnormed, dresidual_out))
    D = y.shape[-1]
    one = torch.ones(D, dtype=torch.float64)
    y = y.reshape(-1, D)
    flat = lambda t: torch.zeros_like(y) if t is None else t.reshape(-1, D)      # noqa: E731
    r0, dn, dr0 = flat(r0), flat(dn), flat(dr0)
    first = w is not None
    w = one if w is None else w
    s = one if s is None else s
    mean = lambda t: t.mean(-1, keepdim=True)      # noqa: E731
    ry = torch.rsqrt(mean(y * y) + eps) if first else torch.ones(y.shape[0], 1, dtype=torch.float64)
    if g is None:
        a, da, daa = torch.ones_like(y), torch.zeros_like(y), torch.zeros_like(y)
    else:
        g = g.reshape(-1, D)
        sg = torch.sigmoid(g)
        if gate_act == "none":
            a, da = g, torch.ones_like(g)
            daa = da
        elif gate_act == "sigmoid":
            a, da = sg, sg * (1 - sg)
            daa = da
        else:
            a, da = g * sg, sg * (1 + g * (1 - sg))
            daa = sg * (1 + g.abs() * (1 - sg))
    yh = y * ry
    p = a * yh * w
    r = r0 + s * p
    rsc = r0.abs() + (s * p).abs()
    rr = torch.rsqrt(mean(r * r) + eps)
    # r's error is relative to its terms; the norm divides by rms(r), whose own error is at most the mean of r's
    hat = r * rr
    hsc = rr * rsc + hat.abs() * (rr * torch.sqrt(mean(rsc * rsc)))
    normed, nsc = hat * v, hsc * v.abs()
    t = dn * v
    m1, m1s = mean(t * hat), mean(t.abs() * hsc)
    amp = 1 + rr * torch.sqrt(mean(rsc * rsc))
    dr = dr0 + rr * (t - hat * m1)
    drs = dr0.abs() + rr * amp * (t.abs() + hsc * m1s)
    dp, dps = dr * s, drs * s.abs()
    q, qs = dp * a * w, dps * (a * w).abs()
    m2 = mean(q * yh) if first else torch.zeros_like(ry)
    m2s = mean(qs * yh.abs()) if first else torch.zeros_like(ry)
    dy, dys = ry * (q - yh * m2), ry * (qs + yh.abs() * m2s)
    out = {"normed": (normed, nsc), "residual": (r, rsc), "dy": (dy, dys), "dresidual": (dr, drs),
           "dgate": (dp * yh * w * da, dps * (yh * w).abs() * daa.abs()), "dpre_w": ((dn * hat).sum(0), (dn.abs() * hsc).sum(0)),
           "dpost_w": ((dp * a * yh).sum(0), (dps * (a * yh).abs()).sum(0)), "dscale": ((dr * p).sum(0), (drs * p.abs()).sum(0))}
    return out

"""The selective scan in float64 with a running error bound, batched over sequences and channels on the tensors' own device.

``seq_ref`` charges every term of a result with one number of roundings.  Here the error of a state is carried along the tokens as the
kernels make it, E_t = a_t E_(t-1) + a_t H_(t-1) eps_t + |step u B| delta_t + ..., with H the same recurrence over absolute values: a token
with a large |step A| is charged for it once, and its term dies out with the state.  u = 2^-24 is one rounding of fp32 to nearest; the
hardware's exponential and reciprocal are good to one unit in the last place, 2 u.  H, not |h|, stands in every term, so that the bound
also holds where a chunk's state is put together from the state that a chunk leaves from zero and the decayed one before it."""
import torch

from seq_ref import U32 as U, half_step, lengths_or_full, softplus64


def check(got, ref, dtype, what=""):
    """|got - value| <= the bound (and a hundredth of it for products of two errors) + one rounding to the output's type."""
    value, err = ref
    assert tuple(got.shape) == tuple(value.shape), (what, got.shape, value.shape)
    assert got.dtype == dtype, (what, got.dtype)
    out, err = got.detach().double(), 1.01 * err
    assert torch.isfinite(out).all(), f"{what}: not finite"
    bound = err + half_step(got.dtype) * (value.abs() + err) + torch.finfo(got.dtype).tiny * 64
    off = (out - value).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound (largest error {off.max().item():.3g})"
    return worst


def _sigmoid(x, raw_err=0.0):
    """sigmoid and its relative error: 1 / (1 + exp(-x)); the exponential's argument is off by 2 u |x| (log2 e and the product) + raw_err."""
    s = torch.sigmoid(x)
    return s, ((2 * x.abs() + 2) * U + raw_err) * (1 - s) + 3 * U


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=True, state=None, lengths=None, dout=None, dstate_out=None,
                   reach=0, chain=0):
    """{name: (value, bound)} of y, state and, with dout, every gradient.  reach: the tokens of a chunk (a chunk's decay is taken from the
    fp32 sum of its steps); chain: how many tokens of one channel one accumulator adds for dA, dD and ddelta_bias."""
    f = lambda t: None if t is None else t.detach().double()       # noqa: E731
    u, delta, A, B, C, D, z, delta_bias, state, dout, dstate_out = map(f, (u, delta, A, B, C, D, z, delta_bias, state, dout, dstate_out))
    Bt, L, dim = u.shape
    N, dev = A.shape[1], u.device
    if B.dim() == 3:
        B, C = B[:, :, None], C[:, :, None]
    G = B.shape[2]
    ns = torch.tensor(lengths_or_full(lengths, Bt, L), device=dev)
    live = torch.arange(L, device=dev)[None] < ns[:, None]
    zero = torch.zeros((), dtype=torch.float64, device=dev)
    keep = lambda t: torch.where(live.view(Bt, L, *[1] * (t.dim() - 2)), t, zero)    # noqa: E731
    u, delta, B, C = keep(u), keep(delta), keep(B), keep(C)
    raw = delta + (0.0 if delta_bias is None else delta_bias)
    eraw = raw.abs() * U                                           # the sum of delta and its bias is rounded
    if softplus:
        # log1p(e) from e = exp(-|raw|): (2 |raw| + 2) u of the exponential, 4 u of e / (2 + e), which the series takes 1.09 times, and 4 u
        step, tail = softplus64(raw), torch.log1p(torch.exp(-raw.abs()))
        estep = tail * (2.2 * raw.abs() + 11) * U + step * U + torch.sigmoid(raw) * eraw
        sig, esig = _sigmoid(raw, eraw)
    else:
        step, estep, sig, esig = raw, eraw, torch.ones_like(raw), torch.zeros_like(raw)
    step, estep = keep(step), keep(estep)
    su = step * u
    esu = estep * u.abs() + su.abs() * U
    Dv = torch.zeros(dim, dtype=torch.float64, device=dev) if D is None else D
    if z is None:
        gate, egate = torch.ones_like(u), torch.zeros_like(u)
    else:
        z = keep(z)
        sg, esg = _sigmoid(z)
        gate = z * sg
        egate = gate.abs() * (esg + U)
        slope = sg * (1 + z * (1 - sg))
        eslope = sg * (z.abs() * (sg * esg + U) + U * (1 + z.abs() * (1 - sg))) + slope.abs() * (esg + 2 * U)
    per = lambda t, at: t[:, at].repeat_interleave(dim // G, 1)    # noqa: E731   (Bt, dim, N) rows of a token

    def decay_at(t):
        x = step[:, t, :, None] * A
        return torch.exp(x), A.abs() * estep[:, t, :, None] + x.abs() * (4 + reach) * U + 3 * U

    n3 = lambda: torch.zeros(Bt, dim, N, dtype=torch.float64, device=dev)      # noqa: E731
    h = n3() if state is None else state
    H, E = h.abs(), n3()
    before = []                                                    # h, H, E before every token
    y, ey = torch.zeros_like(u), torch.zeros_like(u)
    inner = torch.zeros_like(u)
    for t in range(L):
        before.append((h, H, E) if dout is not None else None)
        a, eps = decay_at(t)
        Bv, Cv, m = per(B, t), per(C, t), live[:, t, None, None]
        term, Ah = su[:, t, :, None] * Bv, a * H
        H2 = Ah + term.abs()
        E2 = a * E + Ah * (eps + U) + Bv.abs() * esu[:, t, :, None] + U * term.abs() + U * H2
        h, H, E = torch.where(m, a * h + term, h), torch.where(m, H2, H), torch.where(m, E2, E)
        inner[:, t] = (Cv * h).sum(-1) + Dv * u[:, t]
        yabs = (Cv.abs() * H).sum(-1) + (Dv * u[:, t]).abs()
        ein = (Cv.abs() * E).sum(-1) + (N / 2 + 5) * U * yabs
        y[:, t] = inner[:, t] * gate[:, t]
        ey[:, t] = ein * gate[:, t].abs() + yabs * (egate[:, t] + 2 * U * gate[:, t].abs())
    out = {"y": (keep(y), keep(ey)), "state": (h, E)}
    if dout is None:
        return out
    dout = keep(dout)
    d = dout * gate
    ed = dout.abs() * egate + 2 * U * d.abs()
    names = ("du", "ddelta", "dz")
    g, e = ({k: torch.zeros_like(u) for k in names} for _ in range(2))
    gB, eB, gC, eC = (torch.zeros(Bt, L, G, N, dtype=torch.float64, device=dev) for _ in range(4))
    dA, eA = (torch.zeros(dim, N, dtype=torch.float64, device=dev) for _ in range(2))
    sd = torch.zeros_like(u)                                       # the absolute terms of ddelta
    carry = n3() if dstate_out is None else dstate_out
    K, Ek = carry.abs(), n3()
    chan = (24 + dim // G // 16) * U                               # a sum over the channels of a group: lanes, waves, blocks
    fold = lambda t: t.view(Bt, G, dim // G, N).sum(2)             # noqa: E731
    for t in reversed(range(L)):
        a, eps = decay_at(t)
        Bv, Cv, m = per(B, t), per(C, t), live[:, t, None, None]
        hb, Hb, Eb = before[t]
        at = lambda v: v[:, t, :, None]                            # noqa: E731
        k = Cv * at(d) + carry
        kabs = Cv.abs() * at(d).abs() + K
        ek = Ek + Cv.abs() * at(ed) + 2 * U * kabs
        ah, AH = a * hb, a * Hb
        eah = a * Eb + AH * (eps + U)
        sua, ud, dd = at(su).abs(), u[:, t], d[:, t]
        tB = kabs * sua
        gB[:, t] = fold(k * at(su))
        eB[:, t] = fold(ek * sua + kabs * at(esu) + chan * tB)
        tC = at(d).abs() * AH + Bv.abs() * at(d).abs() * sua
        gC[:, t] = fold((ah + at(su) * Bv) * at(d))
        eC[:, t] = fold(at(d).abs() * eah + AH * at(ed) + Bv.abs() * (at(d).abs() * at(esu) + sua * at(ed)) + chan * tC)
        w, wabs = k * ah, kabs * AH
        ew = ek * AH + kabs * eah + U * wabs
        sa = at(step).abs()
        dA += torch.where(m, w * at(step), zero).sum(0)
        eA += torch.where(m, ew * sa + wabs * at(estep) + (chain + 6) * U * wabs * sa, zero).sum(0)
        SW, SWa = (w * A).sum(-1), (wabs * A.abs()).sum(-1)
        eSW = (ew * A.abs()).sum(-1) + (N / 4 + 8) * U * SWa
        SG, SGa = (k * Bv).sum(-1), (kabs * Bv.abs()).sum(-1)
        eSG = (ek * Bv.abs()).sum(-1) + (N / 4 + 5) * U * SGa
        ds, dsa = SW + SG * ud, SWa + SGa * ud.abs()
        eds = eSW + ud.abs() * eSG + 2 * U * dsa
        g["ddelta"][:, t] = ds * sig[:, t]
        sd[:, t] = dsa * sig[:, t]
        e["ddelta"][:, t] = eds * sig[:, t] + dsa * sig[:, t] * (esig[:, t] + U)
        g["du"][:, t] = SG * step[:, t] + dd * Dv
        e["du"][:, t] = eSG * step[:, t].abs() + SGa * estep[:, t] + Dv.abs() * ed[:, t] + 3 * U * (SGa * step[:, t].abs() + (dd * Dv).abs())
        if z is not None:
            cb = (Cv.abs() * Bv.abs()).sum(-1)
            SY = (Cv.abs() * AH).sum(-1)
            tot = SY + (step[:, t].abs() * cb + Dv.abs()) * ud.abs()
            ein = (Cv.abs() * eah).sum(-1) + ud.abs() * cb * estep[:, t] + (N / 4 + 12) * U * tot
            g["dz"][:, t] = dout[:, t] * inner[:, t] * slope[:, t]
            e["dz"][:, t] = dout[:, t].abs() * (ein * slope[:, t].abs() + tot * (eslope[:, t] + 4 * U * slope[:, t].abs()))
        carry = torch.where(m, a * k, carry)
        Ek = torch.where(m, a * ek + a * kabs * (eps + U), Ek)
        K = torch.where(m, a * kabs, K)
    out.update({k: (keep(g[k]), keep(e[k])) for k in names})
    out.update(dB=(keep(gB), keep(eB)), dC=(keep(gC), keep(eC)), dA=(dA, eA), dstate=(carry, Ek))
    both = lambda v, er, t: (keep(v).sum((0, 1)), keep(er + (chain + 6) * U * t).sum((0, 1)))      # noqa: E731
    out["dD"] = both(d * u, ed * u.abs(), (d * u).abs())
    out["ddelta_bias"] = both(g["ddelta"], e["ddelta"], sd)
    return out

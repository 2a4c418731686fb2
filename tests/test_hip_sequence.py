"""The sequence operators (short causal convolution, selective state space scan, norms around a block) against plain float64
implementations (seq_ref.py), at the sizes and masks where they can go wrong.  A bound is k roundings of fp32 times the scale of a
result's terms, plus one rounding to the output's type; k is counted at each operator.  Refusals run on the CPU."""
import pytest
import torch

import seq_ref
from urnn_amd import ops, train_ops

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def make(gen, *shape, scale=1.0, dtype=torch.float32, dev="cuda"):
    return (scale * torch.randn(*shape, generator=gen)).to(dtype).to(dev)


def rng(seed):
    return torch.Generator().manual_seed(seed)


def poison(t, lengths):
    """NaN and infinities in every padded place of (B, L, ...)."""
    for b, n in enumerate(lengths):
        t[b, n:] = float("nan")
        if n < t.shape[1]:
            t[b, -1] = float("inf")
    return t


# ---- causal convolution ----------------------------------------------------------------------------------------------------------
# k: K + 1 fused terms, the activation's exponential, reciprocal and products (8), the derivative's (8); sums over tokens: at most 64
# tokens of a lane's chunk x the chunks it walks (one here), 32 lanes, then double
CONV_K = 160


def conv_case(B, L, D, K, dtype, seed, carried=True, lengths=None, bias=True):
    g = rng(seed)
    x = make(g, B, L, D, dtype=dtype)
    n = None
    if lengths is not None:
        n = torch.tensor(lengths, dtype=torch.int32)
        poison(x, [min(max(v, 0), L) for v in lengths])
    c = {"x": x, "weight": make(g, D, K, scale=0.5), "bias": make(g, D, scale=0.3) if bias else None,
         "state": make(g, B, K - 1, D, dtype=dtype) if carried else None}
    return c, n


CONV = [  # B, L, D, K, carried, lengths
    (1, 1, 1, 4, False, None),
    (1, 1, 8, 2, True, None),
    (2, 2, 24, 4, True, None),                    # fewer tokens than taps
    (3, 5, 33, 3, True, [5, 0, 1]),
    (2, 70, 64, 4, True, [70, 37]),
    (4, 33, 40, 2, False, [33, 2, -3, 99]),       # lengths out of range are clamped
    (1, 257, 520, 4, False, None),
    (9, 12, 96, 4, True, None),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,L,D,K,carried,lengths", CONV)
def test_causal_conv(B, L, D, K, carried, lengths, dtype):
    c, n = conv_case(B, L, D, K, dtype, 7 * L + D, carried, lengths)
    for silu in (True, False):
        ref = seq_ref.causal_conv(**c, lengths=lengths, silu=silu)
        nd = None if n is None else n.cuda()
        y, st = ops.causal_conv(c["x"], c["weight"], bias=c["bias"], state=c["state"], lengths=nd, silu=silu, want_state=True)
        seq_ref.check(y, ref["y"], CONV_K, dtype, "y")
        seq_ref.check(st, ref["state"], 0, dtype, "state")
        assert torch.equal(st.double().cpu(), ref["state"][0])
        y2 = ops.causal_conv(c["x"], c["weight"], bias=c["bias"], state=c["state"], lengths=nd, silu=silu)
        assert torch.equal(y, y2)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,L,D,K,carried,lengths", CONV)
def test_causal_conv_backward(B, L, D, K, carried, lengths, dtype):
    c, n = conv_case(B, L, D, K, dtype, 11 * L + D, carried, lengths)
    g = rng(5)
    dout, dso = make(g, B, L, D, dtype=dtype), make(g, B, K - 1, D, dtype=dtype)
    if lengths is not None:
        poison(dout, [min(max(v, 0), L) for v in lengths])
    nd = None if n is None else n.cuda()
    for silu in (True, False):
        ref = seq_ref.causal_conv(**c, lengths=lengths, silu=silu, dout=dout, dstate_out=dso)
        got = train_ops.causal_conv_backward(c["x"], c["weight"], dout, bias=c["bias"], state=c["state"], lengths=nd, silu=silu, dstate_out=dso)
        for k in ("dx", "dstate", "dweight", "dbias"):
            if k == "dstate" and not carried:
                assert got[k] is None
                continue
            seq_ref.check(got[k], ref[k], CONV_K, torch.float32 if k in ("dweight", "dbias") else dtype, k)
        more = train_ops.causal_conv_backward(c["x"], c["weight"], dout, bias=c["bias"], state=c["state"], lengths=nd, silu=silu, dstate_out=dso,
                                              grads={"dweight": got["dweight"].clone(), "dbias": got["dbias"].clone()}, accumulate=True)
        assert torch.equal(more["dweight"], 2 * got["dweight"]) and torch.equal(more["dbias"], 2 * got["dbias"])
        assert torch.equal(more["dx"], got["dx"])


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,D,K", [(1, 1, 2), (3, 33, 3), (5, 64, 4), (1, 1000, 4)])
def test_causal_conv_step_continues_a_prompt(B, D, K, dtype):
    c, _ = conv_case(B, 9, D, K, dtype, D, True)
    ref = seq_ref.causal_conv(**c)
    whole = ops.causal_conv(c["x"], c["weight"], bias=c["bias"], state=c["state"])
    _, st = ops.causal_conv(c["x"][:, :4], c["weight"], bias=c["bias"], state=c["state"], want_state=True)
    for t in range(4, 9):
        y, new = ops.causal_conv_step(c["x"][:, t], st, c["weight"], bias=c["bias"])
        held = st.clone()
        y2, st2 = ops.causal_conv_step(c["x"][:, t], st, c["weight"], bias=c["bias"], state_out=st)      # in place
        assert st2 is st and torch.equal(st, new) and torch.equal(y, y2) and not torch.equal(held, new)
        seq_ref.check(y, (ref["y"][0][:, t], ref["y"][1][:, t]), CONV_K, dtype, "y")
        assert torch.equal(y, whole[:, t])
    assert torch.equal(st.double().cpu(), ref["state"][0])


@gpu
def test_causal_conv_strides():
    """Slices of a wider projection, a transposed batch and a broadcast batch, with rows on and off 16 bytes."""
    g = rng(3)
    for D, off, dtype in ((32, 8, torch.bfloat16), (32, 3, torch.bfloat16), (12, 4, torch.float32), (7, 1, torch.float16)):
        wide = make(g, 4, 10, 3 * D + 8, dtype=dtype)
        w, b = make(g, D, 4), make(g, D)
        for x in (wide[..., off:off + D], wide.transpose(0, 1)[..., off:off + D], wide[:1, :, off:off + D].expand(4, -1, -1)):
            dout = make(g, *x.shape, dtype=dtype)
            assert torch.equal(ops.causal_conv(x, w, bias=b), ops.causal_conv(x.contiguous(), w, bias=b))
            a, e = train_ops.causal_conv_backward(x, w, dout, bias=b), train_ops.causal_conv_backward(x.contiguous(), w, dout, bias=b)
            for k in ("dx", "dbias", "dweight"):
                ref = seq_ref.causal_conv(x, w, b, dout=dout)
                seq_ref.check(a[k], ref[k], CONV_K, a[k].dtype, k)
                seq_ref.check(e[k], ref[k], CONV_K, a[k].dtype, k)


# ---- selective scan ----------------------------------------------------------------------------------------------------------
def scan_case(B, L, dim, N, G, dtype, seed, carried=True, lengths=None, gate=True, bias=True, skip=True, softplus=True, train=True, dev="cuda"):
    g = rng(seed)
    step = torch.exp(torch.empty(dim).uniform_(-6.0, -0.7, generator=g))
    c = {"u": make(g, B, L, dim, dtype=dtype, dev=dev), "delta": make(g, B, L, dim, scale=0.7, dtype=dtype, dev=dev),
         "A": -torch.arange(1, N + 1).float().repeat(dim, 1).mul(torch.empty(dim, N).uniform_(0.7, 1.3, generator=g)).to(dev),
         "B": make(g, B, L, G, N, dtype=dtype, dev=dev), "C": make(g, B, L, G, N, dtype=dtype, dev=dev), "D": make(g, dim, dev=dev) if skip else None,
         "z": make(g, B, L, dim, dtype=dtype, dev=dev) if gate else None,
         "delta_bias": (step + torch.log(-torch.expm1(-step))).to(dev) if bias else None,
         "state": make(g, B, dim, N, dev=dev) if carried else None, "softplus": softplus}
    if not softplus:
        c["delta"] = c["delta"].abs() * 0.1
        c["delta_bias"] = step.to(dev) if bias else None
    n = None
    if lengths is not None:
        n = torch.tensor(lengths, dtype=torch.int32, device=dev)
        for k in ("u", "delta", "B", "C", "z"):
            if c[k] is not None:
                poison(c[k], [min(max(v, 0), L) for v in lengths])
    return c, n


def scan_k(c):
    return seq_ref.scan_roundings(c["A"], c["delta"], c["delta_bias"], c["softplus"], c["u"].shape[1], c["A"].shape[1])


SCAN = [  # B, L, dim, N, G, lengths, options
    (1, 1, 1, 1, 1, None, {}),
    (2, 1, 96, 16, 1, [0, 1], {}),
    (1, 7, 64, 16, 1, None, {"carried": False}),
    (3, 33, 65, 16, 1, [33, 0, 8], {}),
    (2, 40, 24, 3, 4, None, {"gate": False}),
    (2, 64, 60, 5, 3, [64, 31], {"softplus": False}),
    (1, 129, 130, 8, 1, None, {"skip": False, "bias": False}),
    (2, 75, 16, 32, 2, [75, 74], {}),
    (1, 50, 10, 64, 1, None, {"gate": False, "carried": False}),
    (1, 300, 128, 16, 1, None, {}),                            # cut into chunks
    (2, 333, 100, 16, 2, [333, 65], {}),                       # ... with whole chunks behind a sequence's end
    (2, 200, 48, 12, 1, [-1, 500], {"carried": False}),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,L,dim,N,G,lengths,opts", SCAN)
def test_selective_scan(B, L, dim, N, G, lengths, opts, dtype):
    c, n = scan_case(B, L, dim, N, G, dtype, L + dim, lengths=lengths, **opts)
    ref = seq_ref.selective_scan(**c, lengths=lengths)
    y, st = ops.selective_scan(**c, lengths=n, want_state=True)
    k = scan_k(c)
    seq_ref.check(y, ref["y"], k, dtype, "y")
    seq_ref.check(st, ref["state"], k, torch.float32, "state")
    ws = ops.selective_scan_workspace(c["u"], c["A"])
    y2 = ops.selective_scan(**c, lengths=n, ws=ws)             # a training forward gives the same
    assert torch.equal(y, y2)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,dim,N,G", [(1, 1, 1, 1), (3, 65, 16, 1), (2, 24, 3, 4), (2, 30, 8, 3), (5, 16, 64, 1), (2, 40, 12, 2), (1, 7, 32, 1)])
def test_selective_scan_step_continues_a_prompt(B, dim, N, G, dtype):
    c, _ = scan_case(B, 8, dim, N, G, dtype, dim)
    ref = seq_ref.selective_scan(**c)
    k = scan_k(c)
    cut = {key: v[:, :3] for key, v in c.items() if key in ("u", "delta", "B", "C", "z")}
    _, st = ops.selective_scan(**{**c, **cut}, want_state=True)
    for t in range(3, 8):
        tok = {key: c[key][:, t] for key in ("u", "delta", "B", "C", "z")}
        y, new = ops.selective_scan_step(**{**c, **tok, "state": st})
        y2, st2 = ops.selective_scan_step(**{**c, **tok, "state": st}, state_out=st)
        assert st2 is st and torch.equal(st, new) and torch.equal(y, y2)
        seq_ref.check(y, (ref["y"][0][:, t], ref["y"][1][:, t]), k, dtype, "y")
    seq_ref.check(st, ref["state"], k, torch.float32, "state")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,L,dim,N,G,lengths,opts", SCAN)
def test_selective_scan_backward(B, L, dim, N, G, lengths, opts, dtype):
    c, n = scan_case(B, L, dim, N, G, dtype, 3 * L + dim, lengths=lengths, **opts)
    g = rng(17)
    dout, dso = make(g, B, L, dim, dtype=dtype), make(g, B, dim, N)
    if lengths is not None:
        poison(dout, [min(max(v, 0), L) for v in lengths])
    ref = seq_ref.selective_scan(**c, lengths=lengths, dout=dout, dstate_out=dso)
    ws = ops.selective_scan_workspace(c["u"], c["A"])
    ops.selective_scan(**c, lengths=n, ws=ws)
    held = ws.clone()
    args = {k: v for k, v in c.items() if k != "state"}
    got = train_ops.selective_scan_backward(**args, dout=dout, fwd_ws=ws, lengths=n, dstate_out=dso, want_dstate=True)
    k = 2 * scan_k(c)
    wide = {"dA", "dD", "ddelta_bias", "dstate"}
    for name in ("dz", "dC", "du", "dB", "ddelta", "dA", "dD", "ddelta_bias", "dstate"):
        if {"dz": c["z"], "dD": c["D"], "ddelta_bias": c["delta_bias"]}.get(name, 0) is None:
            assert got[name] is None
            continue
        seq_ref.check(got[name], ref[name], k + (B * L if name in wide else 0), torch.float32 if name in wide else dtype, name)
    assert torch.equal(ws, held)                                # the record is only read: a second backward gives the same bits
    grads = {name: got[name].clone() for name in ("dA", "dD", "ddelta_bias") if got[name] is not None}
    more = train_ops.selective_scan_backward(**args, dout=dout, fwd_ws=ws, lengths=n, dstate_out=dso, grads=grads, accumulate=True)
    for name in ("du", "ddelta", "dB", "dC"):
        assert torch.equal(more[name], got[name]), name
    for name in ("dA", "dD", "ddelta_bias"):
        assert got[name] is None or torch.equal(more[name], 2 * got[name]), name
    assert more["dstate"] is None


@gpu
def test_selective_scan_backward_many_sequences():
    """More sequences than blocks along the batch: one block sums several."""
    c, n = scan_case(1100, 3, 130, 4, 1, torch.float32, 8, lengths=[3, 0, 1, 2] * 275)
    dout = make(rng(4), 1100, 3, 130)
    ref = seq_ref.selective_scan(**c, lengths=n.tolist(), dout=dout)
    ws = ops.selective_scan_workspace(c["u"], c["A"])
    ops.selective_scan(**c, lengths=n, ws=ws)
    got = train_ops.selective_scan_backward(**{k: v for k, v in c.items() if k != "state"}, dout=dout, fwd_ws=ws, lengths=n)
    for name in ("du", "dB", "dC", "ddelta", "dz"):
        seq_ref.check(got[name], ref[name], 2 * scan_k(c), torch.float32, name)
    for name in ("dA", "dD", "ddelta_bias"):                    # a block's chain of 3 x 2 tokens, then double
        seq_ref.check(got[name], ref[name], 2 * scan_k(c), torch.float32, name)


@gpu
def test_selective_scan_gradients_against_differences():
    """The sum of every gradient along a direction, against central differences of the float64 forward.  h = 1e-5: the forward's values
    are O(10), so that rounding leaves 1e-15 * 10 / 1e-5 = 1e-9 and the third derivative about h^2; the kernels add 1e-5 of the scale."""
    c, _ = scan_case(2, 37, 20, 8, 2, torch.float32, 21)
    g = rng(2)
    dout, dso = make(g, 2, 37, 20), make(g, 2, 20, 8)
    ws = ops.selective_scan_workspace(c["u"], c["A"])
    ops.selective_scan(**c, ws=ws)
    got = train_ops.selective_scan_backward(**{k: v for k, v in c.items() if k != "state"}, dout=dout, fwd_ws=ws, dstate_out=dso, want_dstate=True)
    names = {"u": "du", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "delta_bias": "ddelta_bias", "state": "dstate"}

    def f(shift):
        moved = {k: (v.double().cpu() + shift.get(k, 0.0)) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
        r = seq_ref.selective_scan(**moved)
        return ((r["y"][0] * dout.double().cpu()).sum() + (r["state"][0] * dso.double().cpu()).sum()).item()

    h = 1e-5
    for k, dk in names.items():
        v = torch.randn(c[k].shape, generator=g, dtype=torch.float64)
        want = (f({k: h * v}) - f({k: -h * v})) / (2 * h)
        have = (got[dk].double().cpu() * v).sum().item()
        scale = (got[dk].double().cpu() * v).abs().sum().item()
        assert abs(have - want) <= 1e-5 * scale, (k, have, want)


@gpu
def test_selective_scan_strides_and_ungrouped_rows():
    """u and z as halves of one projection, delta, B and C as parts of another, (batch, L, N) B and C."""
    g = rng(1)
    B, L, dim, N = 2, 21, 48, 16
    xz, dbc = make(g, B, L, 2 * dim, dtype=torch.bfloat16), make(g, B, L, dim + 2 * N + 3, dtype=torch.bfloat16)
    c, _ = scan_case(B, L, dim, N, 1, torch.bfloat16, 2)
    c.update(u=xz[..., :dim], z=xz[..., dim:], delta=dbc[..., :dim], B=dbc[..., dim:dim + N], C=dbc[..., dim + N:dim + 2 * N])
    y, st = ops.selective_scan(**c, want_state=True)
    flat = {k: v.contiguous() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    y2, st2 = ops.selective_scan(**flat, want_state=True)
    assert torch.equal(y, y2) and torch.equal(st, st2)
    ref = seq_ref.selective_scan(**c)
    seq_ref.check(y, ref["y"], scan_k(c), torch.bfloat16, "y")
    dout = make(g, B, L, dim + 5, dtype=torch.bfloat16)[..., 5:]
    ws = ops.selective_scan_workspace(c["u"], c["A"])
    ops.selective_scan(**c, ws=ws)
    ref = seq_ref.selective_scan(**c, dout=dout)
    a = train_ops.selective_scan_backward(**{k: v for k, v in c.items() if k != "state"}, dout=dout, fwd_ws=ws)
    b = train_ops.selective_scan_backward(**{k: v for k, v in flat.items() if k != "state"}, dout=dout.contiguous(), fwd_ws=ws)
    assert a["dB"].shape == (B, L, N)
    for k in ("du", "ddelta", "dz", "dB", "dC", "dA", "dD"):
        assert torch.equal(a[k], b[k]), k
    seq_ref.check(a["du"], ref["du"], 2 * scan_k(c), torch.bfloat16, "du")
    one = {k: c[k][:, 0] for k in ("u", "delta", "B", "C", "z")}
    a, ha = ops.selective_scan_step(**{**c, **one})
    b, hb = ops.selective_scan_step(**{**c, **{k: v.contiguous() for k, v in one.items()}})
    assert torch.equal(a, b) and torch.equal(ha, hb)


@gpu
def test_selective_scan_extremes():
    """A decay that dies at once (A = -inf), one that never does (A = 0), steps of zero, and large raw steps."""
    c, _ = scan_case(1, 70, 20, 4, 1, torch.float32, 4)
    c["A"][:, 0], c["A"][:, 1] = float("-inf"), 0.0
    c["delta"][0, ::3] = 60.0                                  # softplus(60) = 60
    c["delta"][0, 1::3] = -60.0                                # exp(-60)
    y, st = ops.selective_scan(**c, want_state=True)
    A = c["A"].clone()
    A[:, 0] = -1e30
    ref = seq_ref.selective_scan(**{**c, "A": A})
    seq_ref.check(y, ref["y"], scan_k(c), torch.float32, "y")
    seq_ref.check(st, ref["state"], scan_k(c), torch.float32, "state")


@gpu
def test_selective_scan_growing_states_across_chunks():
    """A > 0: the product of a chunk's factors overflows (e^(3 * 32)); states and gradients that are zero stay zero."""
    c, _ = scan_case(1, 200, 20, 4, 1, torch.float32, 6, carried=False, softplus=False, bias=False)
    c["A"] = torch.full_like(c["A"], 3.0)
    c["delta"] = torch.ones_like(c["delta"])
    c["u"][:, :197] = 0
    dout = torch.zeros_like(c["u"])
    dout[:, :2] = 1.0
    ref = seq_ref.selective_scan(**c, dout=dout)
    ws = ops.selective_scan_workspace(c["u"], c["A"])
    y, st = ops.selective_scan(**c, ws=ws, want_state=True)
    k = scan_k(c)
    seq_ref.check(y, ref["y"], k, torch.float32, "y")
    seq_ref.check(st, ref["state"], k, torch.float32, "state")
    got = train_ops.selective_scan_backward(**{n: v for n, v in c.items() if n != "state"}, dout=dout, fwd_ws=ws)
    for name in ("du", "ddelta", "dz", "dB", "dC", "dA", "dD"):
        seq_ref.check(got[name], ref[name], 2 * k + 200, torch.float32, name)


# ---- the norms around a block ----------------------------------------------------------------------------------------------------
# k: a thread's chain of 16 squares and a tree over at most 1024 threads (10 + 16), rsqrt and its argument (4), gate (8) and products;
# the backward's means pass through the forward's once more; column sums: the rows a block walks (at most 4 here) and the fold
NORM_K = 128
NORM = [(1, 1), (1, 7), (5, 38), (3, 96), (17, 128), (4, 129), (9, 512), (3, 1001), (2, 2048), (3, 2049), (2, 4096), (2, 5000), (2, 8192), (1, 16384), (1, 16383)]


def norm_case(M, D, dtype, seed, post=True, gate=True, residual=True, scale=True):
    g = rng(seed)
    return {"y": make(g, M, D, dtype=dtype), "pre_w": make(g, D), "residual": make(g, M, D, scale=2.0, dtype=dtype) if residual else None,
            "post_w": make(g, D) if post else None, "gate": make(g, M, D, dtype=dtype) if gate else None, "scale": make(g, D, scale=0.3) if scale else None}


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,D", NORM)
def test_norm_residual(M, D, dtype):
    c = norm_case(M, D, dtype, M + D)
    g = rng(9)
    dn, dr = make(g, M, D, dtype=dtype), make(g, M, D, dtype=dtype)
    ref = seq_ref.norm_residual(**c, dnormed=dn, dresidual_out=dr)
    n, r = ops.norm_residual(**c)
    seq_ref.check(n, ref["normed"], NORM_K, dtype, "normed")
    seq_ref.check(r, ref["residual"], NORM_K, dtype, "residual")
    got = train_ops.norm_residual_backward(dnormed=dn, dresidual_out=dr, **c)
    for k in ("dy", "dgate", "dresidual", "dpre_w", "dpost_w", "dscale"):
        seq_ref.check(got[k], ref[k], 4 * NORM_K, torch.float32 if k in ("dpre_w", "dpost_w", "dscale") else dtype, k)


@gpu
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("post,gate,residual,scale", [(True, True, True, True), (False, True, True, True), (True, False, True, False),
                                                      (True, True, False, True), (False, False, True, False), (False, False, False, False)])
def test_norm_residual_parts(post, gate, residual, scale, act):
    for M, D in ((6, 100), (70, 260), (1500, 24)):
        c = norm_case(M, D, torch.float32, 3, post, gate, residual, scale)
        g = rng(9)
        dn, dr = make(g, M, D), make(g, M, D)
        ref = seq_ref.norm_residual(**c, gate_act=act, eps=1e-3, dnormed=dn, dresidual_out=dr)
        n, r = ops.norm_residual(**c, gate_act=act, eps=1e-3)
        seq_ref.check(n, ref["normed"], NORM_K, torch.float32, "normed")
        seq_ref.check(r, ref["residual"], NORM_K, torch.float32, "residual")
        got = train_ops.norm_residual_backward(dnormed=dn, dresidual_out=dr, gate_act=act, eps=1e-3, **c)
        have = {"dy": True, "dgate": gate, "dresidual": residual, "dpre_w": True, "dpost_w": post, "dscale": scale}
        for k, there in have.items():
            if not there:
                assert got[k] is None
            else:
                seq_ref.check(got[k], ref[k], 4 * NORM_K, torch.float32, k)
        again = train_ops.norm_residual_backward(dnormed=dn, dresidual_out=dr, gate_act=act, eps=1e-3, accumulate=True,
                                                 grads={k: got[k].clone() for k in ("dpre_w", "dpost_w", "dscale") if got[k] is not None}, **c)
        assert torch.equal(again["dpre_w"], 2 * got["dpre_w"]) and torch.equal(again["dy"], got["dy"])
        # one gradient only: the other counts as zeros
        half = train_ops.norm_residual_backward(dnormed=dn, gate_act=act, eps=1e-3, **c)
        full = train_ops.norm_residual_backward(dnormed=dn, dresidual_out=torch.zeros_like(dr), gate_act=act, eps=1e-3, **c)
        assert torch.equal(half["dy"], full["dy"]) and torch.equal(half["dpre_w"], full["dpre_w"])


@gpu
def test_norm_residual_strides_and_in_place():
    g = rng(2)
    for D, off, dtype in ((64, 8, torch.bfloat16), (64, 5, torch.bfloat16), (10, 2, torch.float32)):
        both = make(g, 2, 9, 2 * D + 8, dtype=dtype)
        c = norm_case(18, D, dtype, 4)
        y, gate = both[..., off - off % 2:][..., :D], both[..., D + off:][..., :D]
        res = c["residual"].view(2, 9, D)
        kw = dict(pre_w=c["pre_w"], post_w=c["post_w"], scale=c["scale"])
        n, r = ops.norm_residual(y, residual=res, gate=gate, **kw)
        ref = seq_ref.norm_residual(y, residual=res, gate=gate, **kw)
        seq_ref.check(n.view(18, D), ref["normed"], NORM_K, dtype, "normed")
        held = res.clone()
        n2, r2 = ops.norm_residual(y, residual=held, gate=gate, residual_out=held, **kw)
        assert r2 is held and torch.equal(n, n2) and torch.equal(r, held)
        dn = make(g, 2, 9, D, dtype=dtype)
        a = train_ops.norm_residual_backward(y, dnormed=dn, residual=res, gate=gate, **kw)
        b = train_ops.norm_residual_backward(y.contiguous(), dnormed=dn, residual=res, gate=gate.contiguous(), **kw)
        assert a["dy"].shape == (2, 9, D)
        for k in a:
            assert torch.allclose(a[k].float(), b[k].float(), rtol=2 * seq_ref.half_step(dtype), atol=1e-5), k


# ---- refusals (no GPU) ----------------------------------------------------------------------------------------------------------
def refused(match, fn, *a, **kw):
    with pytest.raises(RuntimeError, match=match):
        fn(*a, **kw)


def test_refusals_causal_conv():
    x, w, b, st = torch.zeros(2, 5, 8), torch.zeros(8, 4), torch.zeros(8), torch.zeros(2, 3, 8)
    refused("no CPU path", ops.causal_conv, x, w)
    refused("no CPU path", ops.causal_conv_step, x[:, 0], st, w)
    refused("float32, bfloat16 or float16", ops.causal_conv, x.double(), w)
    refused(r"expected \(B, L, D\)", ops.causal_conv, x[0], w)
    refused(r"expected \(8, 2..4\)", ops.causal_conv, x, torch.zeros(8, 5))
    refused(r"expected \(8, 2..4\)", ops.causal_conv, x, torch.zeros(8, 1))
    refused(r"expected \(8, 2..4\)", ops.causal_conv, x, torch.zeros(7, 4))
    refused("weight is torch.bfloat16", ops.causal_conv, x, w.bfloat16())
    refused("bias has shape", ops.causal_conv, x, w, bias=b[:4])
    refused("state has shape", ops.causal_conv, x, w, state=torch.zeros(2, 4, 8))
    refused("state is torch.float32", ops.causal_conv, x.bfloat16(), w, state=st)
    refused("state is None", ops.causal_conv_step, x[:, 0], None, w)
    refused("channels of x must be adjacent", ops.causal_conv, torch.zeros(2, 8, 5).transpose(1, 2), w)
    refused("lengths has shape", ops.causal_conv, x, w, lengths=torch.zeros(3, dtype=torch.int32))
    refused("lengths is torch.int64", ops.causal_conv, x, w, lengths=torch.zeros(2, dtype=torch.int64))
    refused("empty input", ops.causal_conv, torch.zeros(2, 0, 8), w)
    refused("out has shape", ops.causal_conv, x, w, out=torch.zeros(2, 5, 7))
    refused("out overlaps an input", ops.causal_conv, x, w, out=x)
    refused("state_out overlaps an input", ops.causal_conv, x, w, state=st, want_state=True, state_out=st)
    both = torch.zeros(3, 3, 8)
    refused("state_out overlaps an input", ops.causal_conv_step, x[:, 0], both[:2], w, state_out=both[1:])
    refused("dout has shape", train_ops.causal_conv_backward, x, w, x[:, :4])
    refused("dstate_out has shape", train_ops.causal_conv_backward, x, w, x, dstate_out=torch.zeros(2, 2, 8))


def test_refusals_selective_scan():
    c, _ = scan_case(2, 5, 8, 4, 2, torch.float32, 0, dev="cpu")
    step = {**c, **{k: c[k][:, 0] for k in ("u", "delta", "B", "C", "z")}}
    refused("no CPU path", ops.selective_scan, **c)
    refused("no CPU path", ops.selective_scan_step, **step)
    refused("float32, bfloat16 or float16", ops.selective_scan, **{**c, "u": c["u"].double()})
    refused(r"expected \(batch, L, dim\)", ops.selective_scan, **{**c, "u": c["u"][0]})
    refused("delta has shape", ops.selective_scan, **{**c, "delta": c["delta"][:, :3]})
    refused("delta is torch.bfloat16", ops.selective_scan, **{**c, "delta": c["delta"].bfloat16()})
    refused("A has shape", ops.selective_scan, **{**c, "A": torch.zeros(8, 65)})
    refused("A has shape", ops.selective_scan, **{**c, "A": torch.zeros(7, 4)})
    refused("A is torch.bfloat16", ops.selective_scan, **{**c, "A": c["A"].bfloat16()})
    refused("groups must divide 8", ops.selective_scan, **{**c, "B": torch.zeros(2, 5, 3, 4)})
    refused("C has shape", ops.selective_scan, **{**c, "C": torch.zeros(2, 5, 1, 4)})
    refused("B has shape", ops.selective_scan, **{**c, "B": torch.zeros(2, 5, 2, 3)})
    refused("groups of B must be adjacent", ops.selective_scan, **{**c, "B": torch.zeros(2, 5, 2, 8)[..., :4]})
    refused("D has shape", ops.selective_scan, **{**c, "D": torch.zeros(4)})
    refused("delta_bias is torch.float16", ops.selective_scan, **{**c, "delta_bias": torch.zeros(8).half()})
    refused("state has shape", ops.selective_scan, **{**c, "state": torch.zeros(2, 8, 5)})
    refused("state is torch.bfloat16", ops.selective_scan, **{**c, "state": c["state"].bfloat16()})
    refused("lengths must be contiguous", ops.selective_scan, **c, lengths=torch.zeros(4, dtype=torch.int32)[::2])
    refused("out overlaps an input", ops.selective_scan, **c, out=c["u"])
    refused("out must be contiguous", ops.selective_scan, **c, out=torch.zeros(2, 8, 5).transpose(1, 2))
    refused("state_out overlaps an input", ops.selective_scan, **c, want_state=True, state_out=c["state"])
    back = {k: v for k, v in c.items() if k != "state"}
    ws = torch.zeros(1 << 16, dtype=torch.uint8)
    refused("no CPU path", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws)
    refused("fwd_ws is None", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=None)
    refused("dout has shape", train_ops.selective_scan_backward, **back, dout=c["u"][:, :2], fwd_ws=ws)
    refused("dstate_out is torch.bfloat16", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, dstate_out=c["state"].bfloat16())
    refused("accumulate needs", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, accumulate=True, grads={"dA": c["A"]})
    refused("dA has shape", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, grads={"dA": c["A"][:4]})
    refused("state is None", ops.selective_scan_step, **{**step, "state": None})
    refused("state_out is torch.bfloat16", ops.selective_scan_step, **step, state_out=c["state"].bfloat16())


def test_refusals_norm_residual():
    c = {k: v.cpu() if v is not None else None for k, v in
         {"y": torch.zeros(4, 8), "pre_w": torch.zeros(8), "residual": torch.zeros(4, 8), "post_w": torch.zeros(8), "gate": torch.zeros(4, 8),
          "scale": torch.zeros(8)}.items()}
    refused("no CPU path", ops.norm_residual, **c)
    refused("gate_act 'tanh' is none of", ops.norm_residual, **c, gate_act="tanh")
    refused("float32, bfloat16 or float16", ops.norm_residual, **{**c, "y": c["y"].double()})
    refused("pre_w has shape", ops.norm_residual, **{**c, "pre_w": torch.zeros(7)})
    refused("scale is torch.bfloat16", ops.norm_residual, **{**c, "scale": torch.zeros(8).bfloat16()})
    refused("gate has shape", ops.norm_residual, **{**c, "gate": torch.zeros(1, 8)})
    refused("residual is torch.bfloat16", ops.norm_residual, **{**c, "residual": c["residual"].bfloat16()})
    refused("16384", ops.norm_residual, torch.zeros(1, 16385), torch.zeros(16385))
    refused("not evenly spaced", ops.norm_residual, torch.zeros(3, 4, 16, 8)[:, :, ::3], c["pre_w"])      # (B, L, D) may be spaced in any way
    buf = torch.zeros(5, 8)
    refused("out overlaps an input", ops.norm_residual, **{**c, "y": buf[:4]}, out=buf[1:])
    refused("out overlaps an input", ops.norm_residual, **c, out=buf[1:], residual_out=buf[:4])
    refused("empty input", ops.norm_residual, torch.zeros(0, 8), c["pre_w"])
    refused("dnormed has shape", train_ops.norm_residual_backward, dnormed=torch.zeros(4, 7), **c)
    refused("accumulate needs", train_ops.norm_residual_backward, dnormed=c["y"], accumulate=True, **c)


def test_refusals_of_buffers():
    """Workspaces, records and gradient buffers: plain bytes of their own, no buffer for two things at once."""
    c, _ = scan_case(2, 5, 8, 4, 2, torch.float32, 0, dev="cpu")
    back = {k: v for k, v in c.items() if k != "state"}
    ws = torch.zeros(1 << 16, dtype=torch.uint8)
    refused("contiguous uint8", ops.selective_scan, **c, ws=ops.Arena("cpu"))            # the next call would get the same record
    refused("contiguous uint8", ops.selective_scan, **c, ws=ws[::2])
    refused("contiguous uint8", ops.selective_scan, **c, ws=torch.zeros(1, dtype=torch.uint8).expand(1 << 16))
    refused("contiguous uint8", ops.selective_scan, **c, ws=torch.zeros(1 << 16))
    refused("of 64 bytes given", ops.selective_scan, **c, ws=ws[:64])
    both = torch.zeros(1 << 16, dtype=torch.uint8)
    refused("ws overlaps", ops.selective_scan, **c, ws=both, out=both[:2 * 5 * 8 * 4].view(torch.float32).view(2, 5, 8))
    refused("contiguous uint8", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ops.Arena("cpu"))
    refused("fwd_ws of 64 bytes", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws[:64])
    refused("expected .batch, L, dim. and .dim, N.", ops.selective_scan_workspace, c["u"][0], c["A"])
    d = torch.zeros(8)
    refused("overlaps", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, grads={"dD": d, "ddelta_bias": d.view(8)})
    refused("one buffer", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, grads={"dD": d, "ddelta_bias": d})
    refused("dA overlaps", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, grads={"dA": c["A"]})
    x, w, b = torch.zeros(2, 5, 8), torch.zeros(8, 4), torch.zeros(8)
    refused("dbias overlaps", train_ops.causal_conv_backward, x, w, x, bias=b, grads={"dbias": b})
    y, v = torch.zeros(3, 8), torch.zeros(8)
    refused("one buffer", train_ops.norm_residual_backward, y, v, y, post_w=v, grads={"dpre_w": d, "dpost_w": d})


def test_c_entries_refuse_what_no_launch_holds():
    from urnn_amd._lib import lib
    L = lib()
    strides = (__import__("ctypes").c_long * 12)()
    assert L.urnn_causal_conv_backward(16, 0, 0, 16, 0, 0, 0, 32, 0, 0, 0, 64, 0, 16, 0, 16, 1 << 40, 0, 1, 1, 1 << 24, 4, 1, 0, 0) == -1
    assert b"one launch" in L.urnn_last_error()
    big = (16, 16, 16, 16, 0, 16, strides, 16, 0, 0, 0, 0, 16, 1 << 60, 16, 16, 16, 16, 0, 16, 0, 0, 0, 16, 1 << 60, 0)
    assert L.urnn_selective_scan_backward(*big, 1, 1, 1 << 21, 1, 64, 1, 0, 0) == -1 and b"one launch" in L.urnn_last_error()
    assert L.urnn_norm_residual(16, 0, 0, strides, 16, 0, 0, 32, 0, 0, 4194304, 4194304, 4097, 0, 1e-5, 0) == -1 and b"one launch" in L.urnn_last_error()
    assert L.urnn_norm_residual(16, 0, 0, strides, 16, 0, 0, 32, 0, 0, 8388608, 8388608, 2049, 0, 1e-5, 0) == -1 and b"one launch" in L.urnn_last_error()


def test_c_entries_refuse_without_a_gpu():
    """Argument errors come before any HIP call, as codes with a message."""
    from urnn_amd._lib import lib
    L = lib()
    assert L.urnn_causal_conv(0, 0, 0, 16, 0, 0, 0, 16, 0, 0, 1, 1, 8, 4, 1, 0) == -2 and b"NULL" in L.urnn_last_error()
    assert L.urnn_causal_conv(16, 0, 0, 16, 0, 0, 0, 16, 0, 3, 1, 1, 8, 4, 1, 0) == -1 and b"dtype=3" in L.urnn_last_error()
    assert L.urnn_causal_conv(16, 0, 0, 16, 0, 0, 0, 16, 0, 0, 1, 1, 8, 5, 1, 0) == -1 and b"taps" in L.urnn_last_error()
    assert L.urnn_causal_conv(16, 0, 0, 16, 0, 32, 0, 16, 32, 0, 1, 1, 8, 4, 1, 0) == -1 and b"state_out" in L.urnn_last_error()
    assert L.urnn_causal_conv_backward(16, 0, 0, 16, 0, 0, 0, 32, 0, 0, 0, 64, 0, 16, 0, 16, 0, 0, 1, 64, 8, 4, 1, 0, 0) == -3
    strides = (__import__("ctypes").c_long * 10)()
    args = (16, 16, 16, 16, 0, strides, 16, 0, 0, 0, 0, 16, 0)
    assert L.urnn_selective_scan(*args, 0, 0, 0, 0, 1, 300, 8, 3, 4, 1, 0) == -1 and b"groups" in L.urnn_last_error()
    assert L.urnn_selective_scan(*args, 0, 0, 0, 0, 1, 300, 8, 1, 65, 1, 0) == -1 and b"N=65" in L.urnn_last_error()
    assert L.urnn_selective_scan(*args, 0, 0, 0, 0, 1, 300, 8, 1, 4, 1, 0) == -2 and b"workspace" in L.urnn_last_error()
    assert L.urnn_selective_scan(*args, 16, 16, 0, 0, 1, 300, 8, 1, 4, 1, 0) == -3
    assert L.urnn_selective_scan(*args, 8, 1 << 30, 0, 0, 1, 300, 8, 1, 4, 1, 0) == -4
    assert L.urnn_selective_scan_workspace_bytes(1, 300, 8, 4, 1) > L.urnn_selective_scan_workspace_bytes(1, 300, 8, 4, 0) > 0
    assert L.urnn_norm_residual(16, 0, 0, strides, 16, 0, 0, 32, 32, 0, 1, 1, 8, 0, 1e-5, 0) == -1 and b"same buffer" in L.urnn_last_error()
    assert L.urnn_norm_residual(16, 0, 0, strides, 16, 0, 0, 32, 0, 0, 1, 1, 16385, 0, 1e-5, 0) == -1
    assert L.urnn_norm_residual(16, 0, 0, strides, 16, 0, 0, 32, 0, 0, 6, 4, 8, 0, 1e-5, 0) == -1 and b"rows" in L.urnn_last_error()


# ---- a run of them together -------------------------------------------------------------------------------------------------------
class Block:
    """norm -> projection -> convolution -> projection -> scan -> projection -> norm, as a model's layer: the projections are plain
    products, everything between them is this library's."""

    def __init__(self, width, dim, N, K, rank, dtype, seed):
        g = rng(seed)
        self.dim, self.N, self.rank, self.dtype = dim, N, rank, dtype
        self.w_in = make(g, width, 2 * dim, scale=width ** -0.5, dtype=dtype)
        self.w_x = make(g, dim, rank + 2 * N, scale=dim ** -0.5, dtype=dtype)
        self.w_dt = make(g, rank, dim, scale=rank ** -0.5, dtype=dtype)
        self.w_out = make(g, dim, width, scale=dim ** -0.5, dtype=dtype)
        self.conv_w, self.conv_b = make(g, dim, K, scale=0.5), make(g, dim, scale=0.1)
        self.A = -torch.arange(1, N + 1).float().repeat(dim, 1).cuda()
        self.D, self.dt_b = make(g, dim), make(g, dim, scale=0.3) - 2.0
        self.pre_w, self.post_w, self.scale = 1 + make(g, width, scale=0.1), 1 + make(g, width, scale=0.1), make(g, width, scale=0.3)

    def first(self, x):
        return ops.norm_residual(x, self.pre_w)[0]

    def split(self, u):
        p = u @ self.w_x
        return (p[..., :self.rank] @ self.w_dt), p[..., self.rank:self.rank + self.N], p[..., self.rank + self.N:]

    def inner(self, x, n, conv_state=None, state=None, lengths=None):
        """-> (residual, normed, conv state, state) of a (B, L, width) run."""
        xz = n @ self.w_in
        u, cs = ops.causal_conv(xz[..., :self.dim], self.conv_w, bias=self.conv_b, state=conv_state, lengths=lengths, want_state=True)
        dt, B, C = self.split(u)
        y, st = ops.selective_scan(u, dt, self.A, B, C, D=self.D, z=xz[..., self.dim:], delta_bias=self.dt_b, state=state, lengths=lengths,
                                   want_state=True)
        normed, res = ops.norm_residual(y @ self.w_out, self.pre_w, residual=x, post_w=self.post_w, scale=self.scale)
        return res, normed, cs, st

    def token(self, x, n, conv_state, state):
        """One token, states in place."""
        xz = n @ self.w_in
        u, _ = ops.causal_conv_step(xz[:, :self.dim], conv_state, self.conv_w, bias=self.conv_b, state_out=conv_state)
        dt, B, C = self.split(u)
        y, _ = ops.selective_scan_step(u, dt, self.A, B, C, state, D=self.D, z=xz[:, self.dim:], delta_bias=self.dt_b, state_out=state)
        return ops.norm_residual(y @ self.w_out, self.pre_w, residual=x, post_w=self.post_w, scale=self.scale)


@gpu
def test_block_prompt_then_tokens():
    """A prompt in two pieces and then token by token gives what the whole sequence gives at once, and a padded batch what its rows give
    alone.  float32; the two ways add the same terms in different orders: 2^-24 x 400 roundings along 40 tokens and three products."""
    blk = Block(24, 48, 8, 4, 6, torch.float32, 5)
    x = make(rng(6), 3, 40, 24)
    res, normed, cs, st = blk.inner(x, blk.first(x))
    tol = dict(rtol=400 * seq_ref.U32, atol=400 * seq_ref.U32 * 8)
    r1, n1, c1, s1 = blk.inner(x[:, :17], blk.first(x[:, :17]))
    r2, n2, c2, s2 = blk.inner(x[:, 17:33], blk.first(x[:, 17:33]), c1, s1)
    assert torch.allclose(torch.cat([r1, r2], 1), res[:, :33], **tol) and torch.allclose(torch.cat([n1, n2], 1), normed[:, :33], **tol)
    for t in range(33, 40):
        n, r = blk.token(x[:, t], blk.first(x[:, t]), c2, s2)
        assert torch.allclose(r, res[:, t], **tol) and torch.allclose(n, normed[:, t], **tol)
    assert torch.allclose(c2, cs, **tol) and torch.allclose(s2, st, **tol)
    lens = [40, 9, 0]
    _, _, cp, sp = blk.inner(x, blk.first(x), lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    rp, _, _, _ = blk.inner(x, blk.first(x), lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for b, n in enumerate(lens):
        if n:
            ra, _, ca, sa = blk.inner(x[b:b + 1, :n], blk.first(x[b:b + 1, :n]))
            assert torch.allclose(rp[b, :n], ra[0], **tol) and torch.allclose(cp[b], ca[0], **tol) and torch.allclose(sp[b], sa[0], **tol)
    assert torch.equal(sp[2], torch.zeros_like(sp[2])) and torch.equal(rp[1, 9:], x[1, 9:])      # a block of zeros adds nothing


@gpu
def test_block_training_window_against_autograd():
    """The chain's gradients -- norm, convolution, scan, norm, with plain products between -- against autograd through the float64 formulas.
    400 roundings of float32 on every path, relative to the largest gradient of a tensor (sums of both signs)."""
    B, L, W, dim, N, K, R = 2, 23, 12, 20, 4, 3, 5
    blk = Block(W, dim, N, K, R, torch.float32, 9)
    x = make(rng(10), B, L, W)
    dn, dr = make(rng(11), B, L, W), make(rng(12), B, L, W)
    cs0, st0 = make(rng(13), B, K - 1, dim), make(rng(14), B, dim, N)

    # the library's kernels, the products' gradients written out
    n0, _ = ops.norm_residual(x, blk.pre_w)
    xz = n0 @ blk.w_in
    xc, z = xz[..., :dim], xz[..., dim:]
    u = ops.causal_conv(xc, blk.conv_w, bias=blk.conv_b, state=cs0)
    dt, Bm, Cm = blk.split(u)
    ws = ops.selective_scan_workspace(u, blk.A)
    scan = dict(A=blk.A, B=Bm, C=Cm, D=blk.D, z=z, delta_bias=blk.dt_b)
    y = ops.selective_scan(u, dt, state=st0, ws=ws, **scan)
    o = y @ blk.w_out
    gn = train_ops.norm_residual_backward(o, blk.pre_w, dn, dresidual_out=dr, residual=x, post_w=blk.post_w, scale=blk.scale)
    gs = train_ops.selective_scan_backward(u, dt, dout=gn["dy"] @ blk.w_out.t(), fwd_ws=ws, want_dstate=True, **scan)
    dp = torch.cat([gs["ddelta"] @ blk.w_dt.t(), gs["dB"], gs["dC"]], -1)
    gc = train_ops.causal_conv_backward(xc, blk.conv_w, gs["du"] + dp @ blk.w_x.t(), bias=blk.conv_b, state=cs0)
    gp = train_ops.norm_residual_backward(x, blk.pre_w, torch.cat([gc["dx"], gs["dz"]], -1) @ blk.w_in.t(), grads={"dpre_w": gn["dpre_w"]},
                                          accumulate=True)
    got = {"x": gn["dresidual"] + gp["dy"], "pre_w": gp["dpre_w"], "post_w": gn["dpost_w"], "scale": gn["dscale"], "conv_w": gc["dweight"],
           "conv_b": gc["dbias"], "A": gs["dA"], "D": gs["dD"], "dt_b": gs["ddelta_bias"], "cs0": gc["dstate"], "st0": gs["dstate"]}

    f = lambda t: t.double().cpu().requires_grad_(True)      # noqa: E731
    P = {k: f(v) for k, v in {"x": x, "pre_w": blk.pre_w, "post_w": blk.post_w, "scale": blk.scale, "conv_w": blk.conv_w, "conv_b": blk.conv_b,
                              "A": blk.A, "D": blk.D, "dt_b": blk.dt_b, "cs0": cs0, "st0": st0}.items()}
    wi, wx, wd, wo = (t.double().cpu() for t in (blk.w_in, blk.w_x, blk.w_dt, blk.w_out))
    rms = lambda t: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5)      # noqa: E731
    pz = rms(P["x"]) * P["pre_w"] @ wi
    line = torch.cat([P["cs0"], pz[..., :dim]], 1)
    uu = torch.nn.functional.silu(sum(line[:, k:k + L] * P["conv_w"][:, k] for k in range(K)) + P["conv_b"])
    pr = uu @ wx
    step = seq_ref.softplus64(pr[..., :R] @ wd + P["dt_b"])
    h, rows = P["st0"], []
    for t in range(L):
        h = torch.exp(step[:, t, :, None] * P["A"]) * h + (step[:, t] * uu[:, t])[..., None] * pr[:, t, None, R:R + N]
        rows.append((h * pr[:, t, None, R + N:]).sum(-1) + P["D"] * uu[:, t])
    yy = torch.stack(rows, 1) * torch.nn.functional.silu(pz[..., dim:])
    res = P["x"] + P["scale"] * rms(yy @ wo) * P["post_w"]
    want = torch.autograd.grad([rms(res) * P["pre_w"], res], list(P.values()), [dn.double().cpu(), dr.double().cpu()])
    for (k, w) in zip(P, want):
        off = (got[k].double().cpu() - w).abs().max().item()
        assert off <= 400 * seq_ref.U32 * w.abs().max().item() + 1e-7, (k, off, w.abs().max().item())


@gpu
def test_calls_are_bit_reproducible_on_any_stream_and_in_graphs():
    """Two calls at once on two streams, and graphs replayed several times with eager work between, give the eager bits; two captured graphs
    with one Arena's buffers between them replay in turn."""
    c, n = scan_case(2, 210, 48, 16, 2, torch.bfloat16, 31, lengths=[210, 77])
    cc, _ = conv_case(2, 210, 48, 4, torch.bfloat16, 32)
    nc = norm_case(300, 96, torch.bfloat16, 33)
    dout, dn = make(rng(34), 2, 210, 48, dtype=torch.bfloat16), make(rng(35), 300, 96, dtype=torch.bfloat16)
    arena = ops.Arena("cuda")
    back = {k: v for k, v in c.items() if k != "state"}

    def work(ar=None):
        y = ops.causal_conv(cc["x"], cc["weight"], bias=cc["bias"], state=cc["state"])
        gc = train_ops.causal_conv_backward(cc["x"], cc["weight"], dout, bias=cc["bias"], state=cc["state"], scratch=ar)
        ws = ops.selective_scan_workspace(c["u"], c["A"])
        s = ops.selective_scan(**c, lengths=n, ws=ws)
        gs = train_ops.selective_scan_backward(**back, dout=dout, fwd_ws=ws, lengths=n, scratch=ar)
        m, r = ops.norm_residual(**nc)
        gn = train_ops.norm_residual_backward(dnormed=dn, scratch=ar, **nc)
        h = ops.selective_scan_step(**{**c, **{k: c[k][:, 0] for k in ("u", "delta", "B", "C", "z")}})
        return [y, s, m, r, *h] + [v for g in (gc, gs, gn) for k, v in sorted(g.items()) if v is not None]

    eager = [t.clone() for t in work()]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    s1.wait_stream(torch.cuda.current_stream())
    s2.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        a = work()
    with torch.cuda.stream(s2):
        b = work()
    torch.cuda.synchronize()
    for x, y, z in zip(eager, a, b):
        assert torch.equal(x, y) and torch.equal(x, z)
    work(arena)                                                # sizes the arena
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(arena))
        graphs.append(g)
    for turn in range(4):
        for g, out in zip(graphs, outs):
            for t in out:
                t.fill_(7)
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(eager, out):
                assert torch.equal(x, y), turn
            assert torch.equal(work()[1], eager[1])


@gpu
def test_tensors_of_another_device_are_refused():
    class Elsewhere:                                           # a box has one GPU: a tensor that says it is on another one
        shape, dtype, device = (1, 2), torch.float32, torch.device("cuda:1")
        is_cuda = True

        def get_device(self):
            return 1
    with pytest.raises(RuntimeError, match="current device"):
        ops._seq_device("op", Elsewhere())
    with pytest.raises(RuntimeError, match="tensors on"):
        ops._seq_device("op", torch.zeros(1, device="cuda"), Elsewhere())


@gpu
def test_large_offsets():
    """A sequence whose tokens lie beyond 2^31 elements of the first: strides of 64 bits."""
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    L, D, N = 66, 64, 4
    stride = (1 << 32) // 128 + 64                             # elements between tokens: 64 tokens are 2^31
    big = torch.empty(stride * L + 2 * D, dtype=torch.bfloat16, device="cuda")
    x, z = big.as_strided((1, L, D), (stride * L, stride, 1)), big.as_strided((1, L, D), (stride * L, stride, 1), D)
    small, zs = make(rng(1), 1, L, D, dtype=torch.bfloat16), make(rng(2), 1, L, D, dtype=torch.bfloat16)
    x.copy_(small)
    z.copy_(zs)
    c, _ = scan_case(1, L, D, N, 1, torch.bfloat16, 3)
    assert torch.equal(ops.selective_scan(**{**c, "u": x, "z": z}), ops.selective_scan(**{**c, "u": small, "z": zs}))
    w = make(rng(4), D, 4)
    assert torch.equal(ops.causal_conv(x, w), ops.causal_conv(small, w))
    a, b = train_ops.causal_conv_backward(x, w, z), train_ops.causal_conv_backward(small, w, zs)
    assert torch.equal(a["dx"], b["dx"]) and torch.equal(a["dweight"], b["dweight"])
    g = {}
    for u_, z_, d_ in ((x, z, x), (small, zs, small)):
        ws = ops.selective_scan_workspace(u_, c["A"])
        ops.selective_scan(**{**c, "u": u_, "z": z_}, ws=ws)
        g[u_.stride(1)] = train_ops.selective_scan_backward(**{**{k: v for k, v in c.items() if k != "state"}, "u": u_, "z": z_}, dout=d_, fwd_ws=ws)
    a, b = g.values()
    for k in ("du", "ddelta", "dz", "dA", "dB", "dC", "dD"):
        assert torch.equal(a[k], b[k]), k
    n1 = ops.norm_residual(x[0], w[:, 0].contiguous())
    n2 = ops.norm_residual(small[0], w[:, 0].contiguous())
    assert torch.equal(n1[0], n2[0])

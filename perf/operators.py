"""The sequence operators' measured cases: short causal convolution, selective state space scan, and the norms around a block.

``run`` computes a case either in elementary torch operations (``own`` false) or through this repository's operators
(``own`` true).  Widths 96 and 192, planes of 125 x 125 pixels and windows of 12 frames are the network's own; the others
are generic."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST = {"conv": 2 * 4096 * 4096, "scan": 32768 * 2048 * 16, "scan_train": 4 * 2048 * 2048 * 16, "norm": 8192 * 4096}


def listed():
    return [
        # one row of a small decoder, one frame after the other: the smallest call there is, all latency
        {"name": "scan_step_one", "op": "scan_step", "dtype": "fp32", "batch": 1, "channels": 192, "states": 16, "groups": 1, "gate": True},
        # a full serving batch, one token each: the states are read and written once
        {"name": "scan_step_batch", "op": "scan_step", "dtype": "bf16", "batch": 256, "channels": 4096, "states": 16, "groups": 1, "gate": True},
        # one long prompt: nothing but the time axis to spread over the chip
        {"name": "scan_prompt_long", "op": "scan", "dtype": "bf16", "batch": 1, "length": 32768, "channels": 2048, "states": 16, "groups": 1,
         "gate": True, "ragged": False, "carried": False, "train": False},
        # a padded batch of prompts that continue earlier ones, at sizes that fit no tile, with two groups of B and C
        {"name": "scan_prompt_ragged", "op": "scan", "dtype": "fp16", "batch": 7, "length": 1021, "channels": 1000, "states": 16, "groups": 2,
         "gate": True, "ragged": True, "carried": True, "train": False},
        # an ordinary training step: forward and every gradient
        {"name": "scan_train", "op": "scan", "dtype": "bf16", "batch": 4, "length": 2048, "channels": 2048, "states": 16, "groups": 1,
         "gate": True, "ragged": False, "carried": False, "train": True},
        # a training window of 12 frames over the pixels of the quarter-resolution plane: very many, very short sequences
        {"name": "scan_train_frames", "op": "scan", "dtype": "fp32", "batch": 15625, "length": 12, "channels": 96, "states": 8, "groups": 1,
         "gate": False, "ragged": False, "carried": True, "train": True},
        # the convolution of a serving batch, one token each
        {"name": "conv_step", "op": "conv_step", "dtype": "bf16", "batch": 64, "channels": 2048, "taps": 4},
        # the convolution of two long prompts
        {"name": "conv_prompt", "op": "conv", "dtype": "bf16", "batch": 2, "length": 4096, "channels": 4096, "taps": 4, "ragged": False,
         "carried": False, "train": False},
        # forward and gradients, padded, of odd sizes
        {"name": "conv_train_ragged", "op": "conv", "dtype": "fp32", "batch": 6, "length": 1531, "channels": 1001, "taps": 3, "ragged": True,
         "carried": True, "train": True},
        # the norms around a block for a handful of tokens
        {"name": "norm_step", "op": "norm", "dtype": "bf16", "rows": 8, "channels": 2048, "gate": True, "train": False},
        # ... for a prompt
        {"name": "norm_prompt", "op": "norm", "dtype": "bf16", "rows": 8192, "channels": 4096, "gate": True, "train": False},
        # ... and for a training step, forward and gradients, at an odd width
        {"name": "norm_train", "op": "norm", "dtype": "fp32", "rows": 12345, "channels": 1001, "gate": True, "train": True},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["scan_step", "scan", "scan", "scan", "conv_step", "conv", "conv", "norm", "norm"])
    case = {"op": op, "dtype": rng.choice(["fp32", "bf16", "bf16", "fp16"])}
    groups = rng.choice([1, 1, 1, 2, 4])
    channels = _log(rng, 24, 4096)
    if op == "norm":
        return {**case, "rows": _log(rng, 1, LARGEST["norm"] // channels), "channels": channels, "gate": rng.random() < 0.7, "train": rng.random() < 0.5}
    if op.startswith("scan"):
        channels = groups * max(1, channels // groups)
        case.update(channels=channels, states=rng.choice([4, 8, 12, 16, 16, 16, 32]), groups=groups, gate=rng.random() < 0.6)
    else:
        case.update(channels=channels, taps=rng.choice([2, 3, 4, 4]))
    if op.endswith("step"):
        return {**case, "batch": _log(rng, 1, 256)}
    train = rng.random() < 0.5
    most = LARGEST["conv"] // channels if op == "conv" else LARGEST["scan_train" if train else "scan"] // (channels * case["states"])
    most = max(4, most // 2 if train and op == "conv" else most)
    length = _log(rng, 1, min(32768, most))
    batch = _log(rng, 1, max(1, most // length))
    return {**case, "batch": batch, "length": length, "ragged": rng.random() < 0.4, "carried": rng.random() < 0.5, "train": train}


def _lengths(case, r):
    """Lengths of a padded batch: one full, one empty where there is room, the others anywhere."""
    if not case.get("ragged"):
        return None
    n = torch.randint(0, case["length"] + 1, (case["batch"],), generator=r, device="cuda", dtype=torch.int32)
    n[0] = case["length"]
    if case["batch"] > 2:
        n[1] = 0
    return n


def prepare(case, seed):
    r = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    D = case["channels"]

    def normal(*shape, scale=1.0, dtype=dt):
        return (scale * torch.randn(*shape, generator=r, device="cuda")).to(dtype)

    def uniform(low, high, *shape):
        return low + (high - low) * torch.rand(*shape, generator=r, device="cuda")

    s = {"case": dict(case)}
    if case["op"] == "norm":
        M = case["rows"]
        s.update(y=normal(M, D), residual=normal(M, D, scale=2.0), pre_w=uniform(0.5, 1.5, D), post_w=uniform(0.5, 1.5, D),
                 scale=uniform(0.05, 0.4, D), gate=normal(M, D) if case["gate"] else None)
        if case["train"]:
            s.update(dnormed=normal(M, D), dresidual=normal(M, D))
        return s
    Bt = case["batch"]
    s["lengths"] = _lengths(case, r)
    lead = (Bt,) if case["op"].endswith("step") else (Bt, case["length"])
    if case["op"].startswith("conv"):
        K = case["taps"]
        s.update(x=normal(*lead, D), weight=uniform(-0.6, 0.6, D, K), bias=uniform(-0.3, 0.3, D),
                 state=normal(Bt, K - 1, D) if case["op"] == "conv_step" or case["carried"] else None)
    else:
        N, G = case["states"], case["groups"]
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), D))
        s.update(u=normal(*lead, D), delta=normal(*lead, D, scale=0.5), B=normal(*lead, G, N), C=normal(*lead, G, N),
                 A=-torch.arange(1, N + 1, device="cuda") * uniform(0.8, 1.25, D, N), D=uniform(0.5, 1.5, D),
                 delta_bias=step + torch.log(-torch.expm1(-step)), z=normal(*lead, D) if case["gate"] else None,
                 state=normal(Bt, D, N, dtype=torch.float32) if case["op"] == "scan_step" or case["carried"] else None)
    if case.get("train"):
        s["dout"] = normal(*lead, D)
    return s


def run(state):
    op, train = state["case"]["op"], state["case"].get("train", False)
    if own:
        return _own(op, train, state)
    return {"scan_step": _plain_scan_step, "scan": _plain_scan, "conv_step": _plain_conv_step, "conv": _plain_conv, "norm": _plain_norm}[op](state)


def _own(op, train, s):
    from urnn_amd import ops, train_ops
    if op == "scan_step":
        y, h = ops.selective_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"])
        return {"y": y, "state": h}
    if op == "conv_step":
        y, h = ops.causal_conv_step(s["x"], s["state"], s["weight"], bias=s["bias"])
        return {"y": y, "state": h}
    if op == "scan":
        if not train:
            y, h = ops.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"], state=s["state"],
                                      lengths=s["lengths"], want_state=True)
            return {"y": y, "state": h}
        ws = ops.selective_scan_workspace(s["u"], s["A"])
        y = ops.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"], state=s["state"],
                               lengths=s["lengths"], ws=ws)
        g = train_ops.selective_scan_backward(s["u"], s["delta"], s["A"], s["B"], s["C"], s["dout"], ws, D=s["D"], z=s["z"],
                                              delta_bias=s["delta_bias"], lengths=s["lengths"], want_dstate=s["state"] is not None)
        return {"y": y, **{k: v for k, v in g.items() if v is not None}}
    if op == "conv":
        if not train:
            y, h = ops.causal_conv(s["x"], s["weight"], bias=s["bias"], state=s["state"], lengths=s["lengths"], want_state=True)
            return {"y": y, "state": h}
        y = ops.causal_conv(s["x"], s["weight"], bias=s["bias"], state=s["state"], lengths=s["lengths"])
        g = train_ops.causal_conv_backward(s["x"], s["weight"], s["dout"], bias=s["bias"], state=s["state"], lengths=s["lengths"])
        return {"y": y, **{k: v for k, v in g.items() if v is not None}}
    normed, res = ops.norm_residual(s["y"], s["pre_w"], residual=s["residual"], post_w=s["post_w"], gate=s["gate"], scale=s["scale"])
    if not train:
        return {"normed": normed, "residual": res}
    g = train_ops.norm_residual_backward(s["y"], s["pre_w"], s["dnormed"], dresidual_out=s["dresidual"], residual=s["residual"],
                                         post_w=s["post_w"], gate=s["gate"], scale=s["scale"])
    return {"normed": normed, "residual": res, **{k: v for k, v in g.items() if v is not None}}


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _valid(s):
    """(batch, length, 1): which tokens are within their sequence."""
    x = s["u"] if "u" in s else s["x"]
    if s["lengths"] is None:
        return torch.ones(x.shape[0], x.shape[1], 1, dtype=torch.bool, device="cuda")
    return (torch.arange(x.shape[1], device="cuda")[None, :] < s["lengths"][:, None])[..., None]


def _linear_recurrence(a, b):
    """h_t = a_t h_(t-1) + b_t along dim 1 with h_(-1) = 0, by doubling the reach of each entry."""
    a, h, reach = a.clone(), b.clone(), 1
    while reach < a.shape[1]:
        h = torch.cat([h[:, :reach], a[:, reach:] * h[:, :-reach] + h[:, reach:]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return h


def _per_channel(x, D):
    """(..., groups, states) -> (..., channels, states)."""
    return x.float().repeat_interleave(D // x.shape[-2], -2)


def _plain_scan_step(s):
    D = s["u"].shape[-1]
    u, step = s["u"].float(), _softplus(s["delta"].float() + s["delta_bias"])
    h = torch.exp(step[..., None] * s["A"]) * s["state"] + (step * u)[..., None] * _per_channel(s["B"], D)
    y = (h * _per_channel(s["C"], D)).sum(-1) + s["D"] * u
    if s["z"] is not None:
        y = y * s["z"].float() * torch.sigmoid(s["z"].float())
    return {"y": y.to(s["u"].dtype), "state": h}


def _plain_scan(s):
    D, valid, dt = s["u"].shape[-1], _valid(s), s["u"].dtype
    zero = torch.zeros((), device="cuda")
    u = torch.where(valid, s["u"].float(), zero)
    raw = s["delta"].float() + s["delta_bias"]
    step = torch.where(valid, _softplus(raw), zero)
    Bf = torch.where(valid[..., None], s["B"].float(), zero)
    Cf = torch.where(valid[..., None], s["C"].float(), zero)
    Bc, Cc = _per_channel(Bf, D), _per_channel(Cf, D)
    first = torch.zeros(u.shape[0], D, s["A"].shape[1], device="cuda") if s["state"] is None else s["state"]
    a = torch.exp(step[..., None] * s["A"])
    b = (step * u)[..., None] * Bc
    b[:, 0] += a[:, 0] * first
    h = _linear_recurrence(a, b)
    inner = (h * Cc).sum(-1) + s["D"] * u
    y = inner
    if s["z"] is not None:
        z = torch.where(valid, s["z"].float(), zero)
        sg = torch.sigmoid(z)
        y = inner * z * sg
    out = {"y": torch.where(valid, y, zero).to(dt)}
    if not s["case"]["train"]:
        return {**out, "state": h[:, -1].clone()}
    dy = torch.where(valid, s["dout"].float(), zero)
    if s["z"] is not None:
        out["dz"] = (dy * inner * sg * (1 + z * (1 - sg))).to(dt)
        dy = dy * z * sg
    # g_t = C_t dy_t + a_(t+1) g_(t+1): the same recurrence, backwards
    ahead = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    g = _linear_recurrence(ahead.flip(1), (dy[..., None] * Cc).flip(1)).flip(1)
    before = torch.cat([first[:, None], h[:, :-1]], 1)
    through = g * before * a
    gB = (g * Bc).sum(-1)
    dstep = torch.where(valid, (through * s["A"]).sum(-1) + gB * u, zero)
    ddelta = dstep * torch.sigmoid(raw)
    grouped = Bf.shape[:3] + (D // Bf.shape[2], Bf.shape[3])
    out.update(du=(gB * step + dy * s["D"]).to(dt), ddelta=ddelta.to(dt),
               dA=(through * step[..., None]).sum((0, 1), dtype=torch.float64).float(),
               dB=(g * (step * u)[..., None]).view(grouped).sum(3).to(dt), dC=(h * dy[..., None]).view(grouped).sum(3).to(dt),
               dD=(dy * u).sum((0, 1), dtype=torch.float64).float(), ddelta_bias=ddelta.sum((0, 1), dtype=torch.float64).float())
    if s["state"] is not None:
        out["dstate"] = a[:, 0] * g[:, 0]
    return out


def _plain_conv_step(s):
    window = torch.cat([s["state"], s["x"][:, None]], 1)
    p = (window.float() * s["weight"].t()).sum(1) + s["bias"]
    return {"y": (p * torch.sigmoid(p)).to(s["x"].dtype), "state": window[:, 1:].clone()}


def _plain_conv(s):
    x, w, K = s["x"], s["weight"], s["weight"].shape[1]
    Bt, L, D = x.shape
    valid = _valid(s)
    zero = torch.zeros((), device="cuda")
    before = torch.zeros(Bt, K - 1, D, dtype=x.dtype, device="cuda") if s["state"] is None else s["state"]
    line = torch.cat([before.float(), torch.where(valid, x.float(), zero)], 1)
    p = (line.unfold(1, K, 1) * w).sum(-1) + s["bias"]
    sg = torch.sigmoid(p)
    out = {"y": torch.where(valid, p * sg, zero).to(x.dtype)}
    if not s["case"]["train"]:
        n = torch.full((Bt,), L, device="cuda") if s["lengths"] is None else s["lengths"].long()
        at = n[:, None] + torch.arange(K - 1, device="cuda")[None]
        return {**out, "state": line.gather(1, at[..., None].expand(-1, -1, D)).to(x.dtype)}
    dp = torch.where(valid, s["dout"].float() * sg * (1 + p * (1 - sg)), zero)
    padded = torch.cat([torch.zeros(Bt, K - 1, D, device="cuda"), dp, torch.zeros(Bt, K - 1, D, device="cuda")], 1)
    dline = (padded.unfold(1, K, 1) * w.flip(1)).sum(-1)
    out.update(dx=torch.where(valid, dline[:, K - 1:], zero).to(x.dtype),
               dweight=(line.unfold(1, K, 1) * dp[..., None]).sum((0, 1), dtype=torch.float64).float(),
               dbias=dp.sum((0, 1), dtype=torch.float64).float())
    if s["state"] is not None:
        out["dstate"] = dline[:, :K - 1].to(x.dtype)
    return out


EPS = 1e-5


def _plain_norm(s):
    dt = s["y"].dtype
    y, w, v = s["y"].float(), s["post_w"], s["pre_w"]
    ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    act, sg, g = 1.0, None, None
    if s["gate"] is not None:
        g = s["gate"].float()
        sg = torch.sigmoid(g)
        act = g * sg
    p = act * (y * ry) * w
    r = s["residual"].float() + s["scale"] * p
    rr = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
    hat = r * rr
    out = {"normed": (hat * v).to(dt), "residual": r.to(dt)}
    if not s["case"]["train"]:
        return out
    dn = s["dnormed"].float()
    t = dn * v
    dr = s["dresidual"].float() + rr * (t - hat * (t * hat).mean(-1, keepdim=True))
    dp = dr * s["scale"]
    yh = y * ry
    q = dp * act * w
    out.update(dy=(ry * (q - yh * (q * yh).mean(-1, keepdim=True))).to(dt), dresidual=dr.to(dt),
               dpre_w=(dn * hat).sum(0, dtype=torch.float64).float(), dpost_w=(dp * act * yh).sum(0, dtype=torch.float64).float(),
               dscale=(dr * p).sum(0, dtype=torch.float64).float())
    if g is not None:
        out["dgate"] = (dp * yh * w * sg * (1 + g * (1 - sg))).to(dt)
    return out


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    if case["op"] == "norm":
        return _exact_norm(case, s)
    if case["op"].endswith("step"):      # a step is a sequence of one token
        for k in ("x", "u", "delta", "B", "C", "z"):
            if s.get(k) is not None:
                s[k] = s[k][:, None]
    train = case.get("train", False)
    if train and case["op"] == "scan" and case["length"] > 12000:
        return None                      # a graph of that many nodes takes its time
    leaves = {}
    names = {"x": "dx", "weight": "dweight", "bias": "dbias"} if case["op"].startswith("conv") else {
        "u": "du", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "delta_bias": "ddelta_bias"}
    if train:
        leaves = {k: v for k, v in {**names, "state": "dstate"}.items() if s[k] is not None}
        for k in leaves:
            s[k].requires_grad_(True)
    with torch.set_grad_enabled(train):
        y, last = _exact_conv(case, s) if case["op"].startswith("conv") else _exact_scan(case, s)
    if train:
        grads = torch.autograd.grad(y, [s[k] for k in leaves], s["dout"], allow_unused=True)
        return {"y": y.detach(), **{leaves[k]: torch.zeros_like(s[k]) if g is None else g for k, g in zip(leaves, grads)}}
    return {"y": y[:, 0] if case["op"].endswith("step") else y, "state": last}


def _inside(case, s, t):
    """(batch,) truth values: token t is within its sequence; None where all are."""
    return None if s["lengths"] is None else t < s["lengths"]


def _exact_scan(case, s):
    Bt, L, D = s["u"].shape
    G, N = s["B"].shape[2:]
    h = torch.zeros(Bt, G, D // G, N, dtype=torch.float64, device="cuda") if s["state"] is None else s["state"].view(Bt, G, D // G, N)
    A = s["A"].view(1, G, D // G, N)
    step = torch.nn.functional.softplus(s["delta"] + s["delta_bias"], threshold=700.0)
    rows = []
    for t in range(L):
        dt, ut = step[:, t].view(Bt, G, D // G, 1), s["u"][:, t].view(Bt, G, D // G, 1)
        new = torch.exp(dt * A) * h + dt * ut * s["B"][:, t].view(Bt, G, 1, N)
        at = (new @ s["C"][:, t].view(Bt, G, N, 1)).view(Bt, D) + s["D"] * s["u"][:, t]
        if s["z"] is not None:
            at = at * torch.nn.functional.silu(s["z"][:, t])
        m = _inside(case, s, t)
        h = new if m is None else torch.where(m.view(Bt, 1, 1, 1), new, h)
        rows.append(at if m is None else torch.where(m.view(Bt, 1), at, torch.zeros_like(at)))
    return torch.stack(rows, 1), h.reshape(Bt, D, N)


def _exact_conv(case, s):
    x, K = s["x"], s["weight"].shape[1]
    Bt, L, D = x.shape
    state = torch.zeros(Bt, K - 1, D, dtype=torch.float64, device="cuda") if s["state"] is None else s["state"]
    line = torch.cat([state, x], 1)
    p = sum(line[:, k:k + L] * s["weight"][:, k] for k in range(K)) + s["bias"]
    y = torch.nn.functional.silu(p)
    if s["lengths"] is None:
        return y, line[:, L:]
    keep = torch.arange(L, device="cuda")[None, :, None] < s["lengths"][:, None, None]
    last = torch.stack([line[b, n:n + K - 1] for b, n in enumerate(s["lengths"].tolist())])
    return torch.where(keep, y, torch.zeros_like(y)), last


def _exact_norm(case, s):
    leaves = [k for k in ("y", "residual", "pre_w", "post_w", "scale", "gate") if s[k] is not None]
    for k in leaves:
        s[k].requires_grad_(case["train"])
    with torch.set_grad_enabled(case["train"]):
        def rms(x):
            return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
        p = rms(s["y"]) * s["post_w"]
        if s["gate"] is not None:
            p = p * torch.nn.functional.silu(s["gate"])
        r = s["residual"] + p * s["scale"]
        n = rms(r) * s["pre_w"]
    if not case["train"]:
        return {"normed": n, "residual": r}
    grads = torch.autograd.grad([n, r], [s[k] for k in leaves], [s["dnormed"], s["dresidual"]])
    return {"normed": n.detach(), "residual": r.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    D, train = case["channels"], case.get("train", False)
    if case["op"] == "norm":
        wide = (2 + case["gate"] + 2) + (2 + 2 + case["gate"] if train else 0)     # each of y, r, g (and the gradients' two) once
        return {"bytes": wide * e * case["rows"] * D + 4 * D * (6 if train else 3), "flops": case["rows"] * D * (45 if train else 15)}
    Bt, L = case["batch"], case.get("length", 1)
    if case["op"].startswith("conv"):
        K = case["taps"]
        n = Bt * L * D
        carried = e * Bt * (K - 1) * D
        state = 2 * carried if not train else carried * (2 if case["carried"] else 0)
        if not train and case["op"] == "conv" and not case["carried"]:
            state = carried
        return {"bytes": (4 if train else 2) * e * n + state + 4 * D * (K + 1) * (2 if train else 1), "flops": n * (2 * K + 5) * (3 if train else 1)}
    N, G = case["states"], case["groups"]
    n, z = Bt * L * D, int(case["gate"])
    state = 4 * Bt * D * N
    params = 4 * D * (N + 2)
    if not train:
        carried = 1 if case["op"] == "scan" and not case["carried"] else 2
        return {"bytes": (3 + z) * e * n + 2 * e * Bt * L * G * N + carried * state + params, "flops": n * (7 * N + 12)}
    # u, delta, z, dout, B, C in; y, du, ddelta, dz, dB, dC out
    return {"bytes": (6 + 2 * z) * e * n + 4 * e * Bt * L * G * N + (2 * state if case["carried"] else 0) + 2 * params, "flops": n * (22 * N + 40)}

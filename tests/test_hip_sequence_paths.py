"""The parts of the sequence operators that only larger calls reach, each shape shown to reach its part by the sizes that the library's own
workspace queries give: batches of chunks in the carries, summaries in several pieces, several tokens or chunks to a thread, several rows
to a block.  And the fp32 scan held to a running error bound (seq_bounds)."""
import pytest
import torch

import seq_bounds
import seq_ref
from test_hip_sequence import CONV_K, NORM_K, SCAN, make, poison, rng, scan_case
from test_hip_sequence_edges import GRADS, WIDE, scan_gradients
from urnn_amd import ops, train_ops
from urnn_amd._lib import lib

gpu = pytest.mark.gpu
up = lambda n: (n + 255) // 256 * 256      # noqa: E731


# ---- selective scan ----------------------------------------------------------------------------------------------------------
def states(N):
    return next(n for n in (4, 8, 16, 32, 64) if N <= n)


def forward_chunks(B, L, D, N):
    """Chunks of a forward, from the size of its scratch: sums [B][chunks][D] and states [B][chunks][D][NP], none for one chunk."""
    n = lib().urnn_selective_scan_workspace_bytes(B, L, D, N, 0)
    if n == 0:
        return 1
    c = next(c for c in range(2, L + 1) if up(4 * B * c * D) + up(4 * B * c * D * states(N)) >= n)
    assert up(4 * B * c * D) + up(4 * B * c * D * states(N)) == n
    return c


def backward_split(B, L, D, G, N):
    """(chunks, pieces, slots, blocks of a group), written down from the launcher's rule and checked against the size of its scratch."""
    npad = states(N)
    cw = 32 if npad <= 16 else 16
    w = -(-(D // G) // cw)
    waves = -(-w // -(-w // 4))
    gcbs = -(-(D // G) // (waves * cw))
    blocks = B * G * gcbs
    want = max(1, min(1 if blocks >= 512 else -(-512 // blocks), -(-L // 64)))
    cl = -(--(-L // want) // 64) * 64
    chunks, m = -(-L // cl), 1
    while m < 8 and cl % (32 * m) == 0 and cl // (2 * m) >= 64 and blocks * chunks * m < 2048:
        m *= 2
    slots = min(B, max(1, (768 if npad <= 8 else 512) // (G * gcbs * chunks)))
    cross = chunks * m if chunks > 1 else 0
    rows = up(4 * gcbs * B * L * G * N) if gcbs > 1 else 0
    total = up(4 * B * cross * D) + up(4 * B * cross * D * npad) + 2 * rows + up(4 * slots * chunks * D * (N + 2))
    assert lib().urnn_selective_scan_backward_workspace_bytes(B, L, D, G, N) == total
    return {"chunks": chunks, "pieces": m, "slots": slots, "blocks": gcbs, "cl": cl}


def check_scan(c, n, lengths, dtype, seed, dso=True):
    """Forward and every gradient against the running bound."""
    B, L, D = c["u"].shape
    G, N = c["B"].shape[2:]
    g = rng(seed)
    dout, dso = make(g, B, L, D, dtype=dtype), make(g, B, D, N) if dso else None
    if lengths is not None:
        poison(dout, [min(max(v, 0), L) for v in lengths])
    s = backward_split(B, L, D, G, N)
    reach = max(-(-L // forward_chunks(B, L, D, N)) + 16, s["cl"]) if max(s["chunks"], forward_chunks(B, L, D, N)) > 1 else 0
    ref = seq_bounds.selective_scan(**c, lengths=lengths, dout=dout, dstate_out=dso, reach=reach, chain=min(L, s["cl"]) * -(-B // s["slots"]))
    got = scan_gradients(c, dout, n, dso)
    worst = {}
    for k in ("y", "state", *GRADS):
        if {"dz": c["z"], "dD": c["D"], "ddelta_bias": c["delta_bias"]}.get(k, 0) is None:
            assert got[k] is None
        else:
            worst[k] = seq_bounds.check(got[k], ref[k], torch.float32 if k in WIDE or k == "state" else dtype, k)
    return worst


@gpu
@pytest.mark.parametrize("B,L,dim,N,G,lengths,opts", SCAN)
def test_scan_within_the_running_bound(B, L, dim, N, G, lengths, opts):
    c, n = scan_case(B, L, dim, N, G, torch.float32, 5 * L + dim, lengths=lengths, **opts)
    check_scan(c, n, lengths, torch.float32, 18)


def test_the_running_bound_binds():
    """float64 results rounded to fp32 pass, and one row of B (of 300) rounded to 16 bits does not (CPU)."""
    c, _ = scan_case(1, 300, 16, 16, 1, torch.float32, 3, dev="cpu")
    ref = seq_bounds.selective_scan(**c, reach=32)
    assert seq_bounds.check(ref["y"][0].float(), ref["y"], torch.float32) < 0.5
    row = c["B"].clone()
    row[:, 200] = row[:, 200].bfloat16().float()
    off = seq_bounds.selective_scan(**{**c, "B": row})["y"][0].float()
    with pytest.raises(AssertionError, match="times the bound"):
        seq_bounds.check(off, ref["y"], torch.float32)


SPLITS = [  # B, L, dim, N, G, lengths, options, what is reached
    (3, 1100, 8, 4, 1, [1100, 0, 70], {}, dict(forward=35, chunks=18, pieces=1)),              # three and two batches of 16 in the carries
    (1, 1100, 130, 16, 1, None, {"gate": False}, dict(forward=35, chunks=18, pieces=1, blocks=2)),
    (2, 1217, 24, 12, 3, [1217, 600], {"carried": False}, dict(forward=39, chunks=20, pieces=1)),
    (256, 256, 8, 4, 1, "any", {}, dict(chunks=2, pieces=2)),
    (256, 512, 8, 4, 1, "any", {}, dict(chunks=2, pieces=4)),
    (26, 8980, 8, 4, 1, "any", {}, dict(chunks=18, pieces=8)),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,L,dim,N,G,lengths,opts,reached", SPLITS)
def test_scan_in_many_chunks(B, L, dim, N, G, lengths, opts, reached, dtype):
    if dtype != torch.float32 and L > 2000:
        pytest.skip("one type is enough for the longest")
    if lengths == "any":
        lengths = torch.randint(0, L + 1, (B,), generator=rng(L)).tolist()
        lengths[:5] = [L, 0, 1, 64, L - 1]
    have = {"forward": forward_chunks(B, L, dim, N), **backward_split(B, L, dim, G, N)}
    assert {k: have[k] for k in reached} == reached
    c, n = scan_case(B, L, dim, N, G, dtype, L, lengths=lengths, **opts)
    check_scan(c, n, lengths, dtype, 19)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,dim,N,G", [(257, 2048, 16, 1), (1026, 520, 8, 2), (4099, 128, 3, 1), (259, 2100, 32, 1)])
def test_scan_step_of_a_large_batch(B, dim, N, G, dtype):
    """Four sequences to a thread (524 288 channels and up; one from 32 states on), a batch that four does not divide; in place as well."""
    assert B * dim >= 4 * 64 * 2048 and B % 4
    c, _ = scan_case(B, 1, dim, N, G, dtype, dim)
    ref = seq_bounds.selective_scan(**c)
    tok = {**c, **{k: c[k][:, 0] for k in ("u", "delta", "B", "C", "z")}}
    y, st = ops.selective_scan_step(**tok)
    seq_bounds.check(y, tuple(v[:, 0] for v in ref["y"]), dtype, "y")
    seq_bounds.check(st, ref["state"], torch.float32, "state")
    held = c["state"].clone()
    y2, st2 = ops.selective_scan_step(**{**tok, "state": held}, state_out=held)
    assert st2 is held and torch.equal(held, st) and torch.equal(y2, y)


# ---- causal convolution ----------------------------------------------------------------------------------------------------------
def conv_reference(x, weight, bias, state, lengths, silu, dout=None, dstate_out=None):
    """seq_ref.causal_conv, batched, on the tensors' device: {name: (value, scale)}."""
    x, w, bias, state, dout, dstate_out = (None if t is None else t.detach().double() for t in (x, weight, bias, state, dout, dstate_out))
    B, L, D = x.shape
    K = w.shape[1]
    n = torch.tensor(seq_ref.lengths_or_full(lengths, B, L), device=x.device)
    live = (torch.arange(L, device=x.device)[None] < n[:, None])[..., None]
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    line = torch.cat([state, torch.where(live, x, zero)], 1)
    p = bias + sum(line[:, k:k + L] * w[:, k] for k in range(K))
    pa = bias.abs() + sum((line[:, k:k + L] * w[:, k]).abs() for k in range(K))
    s = torch.sigmoid(p)
    y, ya = (p * s, 1.1 * pa) if silu else (p, pa)
    at = n[:, None] + torch.arange(K - 1, device=x.device)
    last = line.gather(1, at[..., None].expand(-1, -1, D))
    out = {"y": (torch.where(live, y, zero), torch.where(live, ya, zero)), "state": (last, torch.zeros_like(last))}
    if dout is not None:
        slope, sa = (s * (1 + p * (1 - s)), s * (1 + p.abs() * (1 - s)) + 0.5 * pa) if silu else (torch.ones_like(p), torch.ones_like(p))
        both = []
        for a, sl in ((lambda t: t, slope), (lambda t: t.abs(), sa)):
            dp = torch.where(live, a(dout) * sl, zero)
            dline = torch.zeros_like(line)
            for k in range(K):
                dline[:, k:k + L] += a(w[:, k]) * dp
            dline.scatter_add_(1, at[..., None].expand(-1, -1, D), a(dstate_out))
            both.append({"dx": torch.where(live, dline[:, K - 1:], zero), "dstate": dline[:, :K - 1],
                         "dweight": torch.stack([(a(line[:, k:k + L]) * dp).sum((0, 1)) for k in range(K)], 1), "dbias": dp.sum((0, 1))})
        out.update({k: (both[0][k], both[1][k]) for k in both[0]})
    return {k: tuple(t.cpu() for t in v) for k, v in out.items()}


def conv_forward_tokens(B, L, D, elem):
    """Tokens of a forward thread, from the launcher's rule (rows that 16 bytes divide: a thread has that many channels)."""
    nv, T = D * elem // 16 if D * elem % 16 == 0 else D, 32
    while T > 4 and B * nv * -(-L // T) < 1 << 17:
        T //= 2
    return T


def conv_backward_walk(B, L, D, K):
    """(tokens of a chunk, chunks that a lane walks at most), the parts from the size of the scratch."""
    parts = next(p for p in range(1, 1025) if up(4 * p * (K + 1) * D) == lib().urnn_causal_conv_backward_workspace_bytes(B, L, D, K))
    nv, xb = -(-D // 2), 8
    while xb < 64 and xb < nv:
        xb *= 2
    lanes = parts * (256 // xb)
    T = min(L, max(8, min(64, -(-B * L // lanes))))
    return T, -(-B * -(-L // T) // lanes)


CONVS = [  # B, L, D, K, dtype, tokens of a forward thread, tokens of a backward chunk, chunks to a backward lane
    (64, 64, 257, 4, torch.float32, 8, 8, 1),
    (130, 61, 520, 3, torch.float16, 4, 10, 2),
    (65, 64, 1001, 4, torch.bfloat16, 16, 9, 2),
    (128, 67, 515, 2, torch.float32, 32, 11, 2),
    (65, 65, 2000, 4, torch.bfloat16, 8, 17, 2),
    (70, 2000, 24, 4, torch.bfloat16, 4, 9, 1),
    (130, 64, 1028, 3, torch.float32, 16, 19, 2),
]


@gpu
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("B,L,D,K,dtype,tokens,back,walks", CONVS)
def test_conv_of_many_tokens(B, L, D, K, dtype, tokens, back, walks, silu):
    """A thread's walk along several groups of tokens, and lanes of the backward that walk several chunks: their sums grow by as many
    tokens (64 a chunk are in CONV_K)."""
    assert conv_forward_tokens(B, L, D, 4 if dtype == torch.float32 else 2) == tokens
    assert conv_backward_walk(B, L, D, K) == (back, walks)
    g = rng(D)
    lengths = torch.randint(0, L + 1, (B,), generator=g).tolist()
    lengths[:7] = [L, 0, 1, 2, tokens, tokens + 1, L - 1]
    x, dout = make(g, B, L, D, dtype=dtype), make(g, B, L, D, dtype=dtype)
    poison(x, lengths)
    poison(dout, lengths)
    state, dso = make(g, B, K - 1, D, dtype=dtype), make(g, B, K - 1, D, dtype=dtype)
    w, b = make(g, D, K, scale=0.5), make(g, D, scale=0.3)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ref = conv_reference(x, w, b, state, lengths, silu, dout, dso)
    y, st = ops.causal_conv(x, w, bias=b, state=state, lengths=n, silu=silu, want_state=True)
    got = {"y": y, "state": st, **train_ops.causal_conv_backward(x, w, dout, bias=b, state=state, lengths=n, silu=silu, dstate_out=dso)}
    for k in ("y", "state", "dx", "dstate", "dweight", "dbias"):
        seq_ref.check(got[k], ref[k], CONV_K + 64 * (walks - 1), torch.float32 if k in ("dweight", "dbias") else dtype, k)


# ---- the norms around a block ----------------------------------------------------------------------------------------------------
def norm_turns(M, D):
    """Rows that a thread group of the backward walks, from the number of its blocks' partial sums (the size of the scratch)."""
    threads = next(t for t, most in ((16, 128), (64, 512), (128, 1024), (256, 2048), (512, 4096), (1024, 16384)) if D <= most)
    rb = max(1, 256 // threads)
    parts = next(p for p in range(1, 769) if up(12 * p * D) == lib().urnn_norm_residual_backward_workspace_bytes(M, D))
    return -(-M // (rb * parts))


NORMS = [  # M, D, rows that a thread group walks
    (12299, 24, 2), (24600, 8, 3), (3091, 260, 2), (1550, 1001, 2), (2307, 520, 2), (779, 2048, 2), (1600, 1100, 3), (259, 2049, 2), (513, 4096, 3), (270, 5000, 2),
    (262, 16384, 2), (261, 16383, 2),
]


@gpu
@pytest.mark.parametrize("M,D,turns", NORMS)
def test_norm_backward_of_many_rows(M, D, turns):
    """A block of the backward walks several rows, the last turn not whole.  Column sums: `turns` rows more in a chain (at most three
    here, of the sixteen that NORM_K has for them four times over)."""
    assert norm_turns(M, D) == turns
    dtype = (torch.float32, torch.bfloat16, torch.float16)[M % 3]
    g = rng(D)
    c = {"y": make(g, M, D, dtype=dtype), "pre_w": make(g, D), "residual": make(g, M, D, scale=2.0, dtype=dtype), "post_w": make(g, D),
         "gate": make(g, M, D, dtype=dtype), "scale": make(g, D, scale=0.3)}
    dn, dr = make(g, M, D, dtype=dtype), make(g, M, D, dtype=dtype)
    ref = seq_ref.norm_residual(**c, dnormed=dn, dresidual_out=dr)
    got = train_ops.norm_residual_backward(dnormed=dn, dresidual_out=dr, **c)
    for k in ("dy", "dgate", "dresidual", "dpre_w", "dpost_w", "dscale"):
        seq_ref.check(got[k], ref[k], 4 * NORM_K, torch.float32 if k in ("dpre_w", "dpost_w", "dscale") else dtype, k)

"""The sequence operators at the edges of what their documentation allows: parameters at the ends of float32, buffers in unusual places,
sizes near the limits of a launch.  Bounds on errors are those of seq_bounds."""
import pytest
import torch

import seq_bounds
from test_hip_sequence import make, refused, rng, scan_case
from urnn_amd import ops, train_ops

gpu = pytest.mark.gpu
GRADS = ("du", "ddelta", "dz", "dB", "dC", "dA", "dD", "ddelta_bias", "dstate")
WIDE = ("dA", "dD", "ddelta_bias", "dstate")


def scan_gradients(c, dout, lengths=None, dstate_out=None):
    ws = ops.selective_scan_workspace(c["u"], c["A"])
    y, st = ops.selective_scan(**c, lengths=lengths, ws=ws, want_state=True)
    got = train_ops.selective_scan_backward(**{k: v for k, v in c.items() if k != "state"}, dout=dout, fwd_ws=ws, lengths=lengths,
                                            dstate_out=dstate_out, want_dstate=True)
    return {"y": y, "state": st, **got}


# ---- the scan's A at the ends of float32 -----------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("L,dim,N,G", [(70, 20, 4, 1), (9, 20, 16, 1), (130, 10, 32, 1), (5, 7, 64, 1), (40, 24, 8, 4)])
def test_selective_scan_backward_where_states_die_at_once(L, dim, N, G, dtype):
    """A = -inf in one state of every channel, in blocks that their channels do not fill: every gradient is finite, that of the other
    states as well.  The reference takes -1e30, whose decay is zero too (steps are above 1e-4 here)."""
    c, _ = scan_case(2, L, dim, N, G, dtype, L + N)
    dout, dso = make(rng(3), 2, L, dim, dtype=dtype), make(rng(4), 2, dim, N)
    finite = c["A"].clone()
    finite[:, 1] = -1e30
    ref = seq_bounds.selective_scan(**{**c, "A": finite}, dout=dout, dstate_out=dso, reach=64, chain=2 * L)
    c["A"][:, 1] = float("-inf")
    got = scan_gradients(c, dout, dstate_out=dso)
    for k in ("y", "state", *GRADS):
        seq_bounds.check(got[k], ref[k], torch.float32 if k in WIDE or k == "state" else dtype, k)


@gpu
@pytest.mark.parametrize("N", [4, 16, 32])
def test_selective_scan_largest_decay_rate_at_steps_of_zero(N):
    """A = -(largest float32) and steps that are exactly zero (softplus(-200)) between others: exp(0 A) = 1, the state stays.  Its gradients
    likewise; those of the steps are a product of |A| with sums that float32 does not hold, and are not looked at."""
    c, _ = scan_case(2, 70, 20, N, 1, torch.float32, N, bias=False)
    c["A"][:, 0] = -torch.finfo(torch.float32).max
    c["delta"][:, 1:40] = -200.0                               # one token of decay first; whole chunks of zero steps behind it
    c["delta"][1] = -200.0                                     # no step at all in the second sequence
    dout, dso = make(rng(3), 2, 70, 20), make(rng(4), 2, 20, N)
    ref = seq_bounds.selective_scan(**c, dout=dout, dstate_out=dso, reach=64, chain=140)
    got = scan_gradients(c, dout, dstate_out=dso)
    for k in ("y", "state", "du", "dz", "dB", "dC", "dD", "dstate"):
        seq_bounds.check(got[k], ref[k], torch.float32, k)
    h = c["state"]                                             # and token by token
    for t in range(3):
        y, h = ops.selective_scan_step(**{**c, **{k: c[k][:, t] for k in ("u", "delta", "B", "C", "z")}, "state": h})
        seq_bounds.check(y, tuple(v[:, t] for v in ref["y"]), torch.float32, "step y")


# ---- refusals (no GPU) ----------------------------------------------------------------------------------------------------------
def test_conv_gradients_without_a_bias_take_no_buffer_for_one():
    """A dbias in grads (of another layer, of any size) is neither written nor handed back as a gradient."""
    x, w = torch.zeros(2, 5, 8), torch.zeros(8, 4)
    for buf in (torch.zeros(8), torch.zeros(3), torch.zeros(8, dtype=torch.bfloat16)):
        refused("dbias in grads, but there is no bias", train_ops.causal_conv_backward, x, w, x, grads={"dbias": buf})
    refused("no CPU path", train_ops.causal_conv_backward, x, w, x, grads={"dbias": None})     # what a call without one leaves


def test_gradients_of_absent_parameters_are_not_handed_back():
    """grads of a call with more parameters: what they hold is no gradient of this call."""
    c, _ = scan_case(2, 5, 8, 4, 2, torch.float32, 0, bias=False, skip=False, dev="cpu")
    back = {k: v for k, v in c.items() if k != "state"}
    ws, v, y = torch.zeros(1 << 16, dtype=torch.uint8), torch.zeros(8), torch.zeros(3, 8)
    refused("dD in grads, but there is no D", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, grads={"dD": v})
    refused("ddelta_bias in grads, but there is no delta_bias", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, grads={"ddelta_bias": v})
    refused("no CPU path", train_ops.selective_scan_backward, **back, dout=c["u"], fwd_ws=ws, grads={"dD": None, "ddelta_bias": None})
    refused("dpost_w in grads, but there is no post_w", train_ops.norm_residual_backward, y, v, y, scale=v, grads={"dpost_w": v})
    refused("dscale in grads, but there is no scale", train_ops.norm_residual_backward, y, v, y, post_w=v, grads={"dscale": v})
    refused("no CPU path", train_ops.norm_residual_backward, y, v, y, grads={"dscale": None, "dpost_w": None})


def test_norm_outputs_apart_from_the_parameters():
    """An output over a weight would be read by rows that are not done yet."""
    y, both = torch.zeros(4, 8), torch.zeros(6, 8)
    for name in ("pre_w", "post_w", "scale"):
        par = {"pre_w": torch.ones(8), name: both[4]}
        refused("out overlaps an input", ops.norm_residual, y, out=both[2:], **par)
        refused("residual_out overlaps an input", ops.norm_residual, y, residual_out=both[1:5], **par)
        refused("no CPU path", ops.norm_residual, y, out=both[:4], **par)


def test_outputs_apart_from_the_lengths():
    """lengths are read by every block until the last one is done."""
    c, _ = scan_case(2, 5, 8, 4, 2, torch.float32, 0, dev="cpu")
    out, st = torch.zeros(2, 5, 8), torch.zeros(2, 8, 4)
    n, m = out.view(torch.int32)[0, 0, :2], st.view(torch.int32)[1, 7, 2:]
    refused("out overlaps an input", ops.selective_scan, **c, lengths=n, out=out)
    refused("state_out overlaps an input", ops.selective_scan, **c, lengths=m, want_state=True, state_out=st)
    x, w, cs = torch.zeros(2, 5, 8), torch.zeros(8, 4), torch.zeros(2, 3, 8)
    refused("out overlaps an input", ops.causal_conv, x, w, lengths=n, out=out)
    refused("state_out overlaps an input", ops.causal_conv, x, w, lengths=cs.view(torch.int32)[0, 0, :2], want_state=True, state_out=cs)
    refused("no CPU path", ops.causal_conv, x, w, lengths=n, out=torch.zeros(2, 5, 8))


def test_an_arena_of_another_device_is_refused(monkeypatch):
    """A backward's scratch from an Arena is looked at like a buffer of the caller's."""
    class Input:                                               # stands for a tensor on the current device
        is_cuda, device = True, torch.device("cuda:0")

        def get_device(self):
            return 0
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    refused("op: .* GPU", train_ops._seq_scratch, "op", ops.Arena("cpu"), 64, torch.device("cuda:0"), (Input(),))


# ---- sizes near the limits of a launch -------------------------------------------------------------------------------------------
def test_scan_limits_are_those_of_its_launches():
    """Waves of 64 channels of a group: fewer than 2^26 (2^32 threads); a token: four threads to a channel.  Sizes that pass go on to the
    NULL check (-2), the others are refused (-1)."""
    from urnn_amd._lib import lib
    L = lib()

    def prompt(B, D, G=1):
        return L.urnn_selective_scan(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, B, 2, D, G, 4, 1, 0)

    def token(B, D, G=1):
        return L.urnn_selective_scan_step(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, B, D, G, 4, 1, 0)

    for inside, outside in (((4194305, 24), (1 << 26, 24)), (((1 << 26) - 1, 1), (1 << 26, 1)), (((1 << 25) - 1, 65), (1 << 25, 65)),
                            ((63, 1 << 20, 1 << 20), (64, 1 << 20, 1 << 20)), ((1, (1 << 30) - 64), (1, (1 << 30) - 63))):
        assert prompt(*inside) == -2, inside
        assert prompt(*outside) == -1 and b"one launch" in L.urnn_last_error(), outside
    for inside, outside in (((4194305, 24), (1 << 26, 24)), (((1 << 30) - 64, 1), ((1 << 30) - 63, 1)), ((1, (1 << 30) - 64), (1, (1 << 30) - 63))):
        assert token(*inside) == -2, inside
        assert token(*outside) == -1 and b"one launch" in L.urnn_last_error(), outside


def test_lengths_that_a_rounding_up_would_overflow_are_refused():
    """Tokens are counted in int and rounded up to whole chunks: close to 2^31 of them the sum would be negative.  Sizes that pass go on to
    the NULL check (-2)."""
    from urnn_amd._lib import lib
    L = lib()
    for n, code in (((1 << 31) - 256, -2), ((1 << 31) - 255, -1), ((1 << 31) - 1, -1)):
        assert L.urnn_causal_conv(16, 1, 1, 16, 0, 0, 0, 0, 0, 1, 1, n, 1, 4, 1, 0) == code
        assert L.urnn_causal_conv_backward(16, 1, 1, 16, 0, 0, 0, 0, 1, 1, 0, 0, 0, 0, 0, 0, 0, 1, 1, n, 1, 4, 1, 0, 0) == code
        assert L.urnn_selective_scan(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1, n, 1, 1, 4, 1, 0) == code
        assert L.urnn_selective_scan_backward(*[0] * 13, 0, *[0] * 10, 0, 1, 1, n, 1, 1, 4, 1, 0, 0) == code


@gpu
def test_scan_of_four_million_short_sequences():
    """As many waves as sequences: the results are those of the batch's parts, bit for bit."""
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    B, L, D, N = 4194305, 2, 24, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    t = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)      # noqa: E731
    c = {"u": t(B, L, D), "delta": t(B, L, D), "B": t(B, L, N), "C": t(B, L, N), "z": t(B, L, D)}
    par = {"A": -torch.rand(D, N, generator=g, device="cuda"), "D": torch.ones(D, device="cuda")}
    state, dout = torch.randn(B, D, N, generator=g, device="cuda"), t(B, L, D)
    got = scan_gradients({**c, **par, "state": state}, dout)
    y, st = ops.selective_scan_step(**{k: v[:, 0] for k, v in c.items()}, **par, state=state)
    for lo in range(0, B, 1 << 20):
        cut = slice(lo, min(lo + (1 << 20), B))
        part = {k: v[cut] for k, v in c.items()}
        want = scan_gradients({**part, **par, "state": state[cut]}, dout[cut])
        for k in ("y", "state", "du", "ddelta", "dz", "dB", "dC", "dstate"):
            assert torch.equal(got[k][cut], want[k]), (k, lo)
        yw, sw = ops.selective_scan_step(**{k: v[:, 0] for k, v in part.items()}, **par, state=state[cut])
        assert torch.equal(y[cut], yw) and torch.equal(st[cut], sw), lo
    assert all(torch.isfinite(got[k]).all() for k in ("dA", "dD"))


def test_norm_limits_are_those_of_its_launches():
    """Blocks of 256 threads and up, a row to 16 .. 1024 of them by its width: fewer than 2^32 threads.  Sizes that pass go on to the NULL
    check of the outputs (-2)."""
    from urnn_amd._lib import lib
    L = lib()
    strides = (__import__("ctypes").c_long * 10)()
    for D, rows in ((1, (1 << 28) - 16), (128, (1 << 28) - 16), (129, (1 << 26) - 4), (512, (1 << 26) - 4), (513, (1 << 25) - 2), (1025, (1 << 24) - 1),
                    (2048, (1 << 24) - 1), (2049, (1 << 23) - 1), (4096, (1 << 23) - 1), (4097, (1 << 22) - 1), (16384, (1 << 22) - 1)):
        for n, code in ((rows, -2), (rows + 1, -1)):
            assert L.urnn_norm_residual(16, 0, 0, strides, 16, 0, 0, 0, 0, 0, n, n, D, 0, 1e-5, 0) == code, (D, n)
            assert L.urnn_norm_residual_backward(16, 0, 0, 0, 0, strides, 16, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, n, n, D, 0, 1e-5, 0, 0) == code, (D, n)
        assert b"one launch" in L.urnn_last_error()


@gpu
def test_norms_of_nine_million_rows():
    """The results are those of the rows' parts, bit for bit."""
    M, D = 9000001, 24
    g = torch.Generator(device="cuda").manual_seed(3)
    t = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)      # noqa: E731
    c, w = {"y": t(M, D), "residual": t(M, D), "gate": t(M, D)}, torch.rand(3, D, generator=g, device="cuda")
    par, dn = {"pre_w": w[0], "post_w": w[1], "scale": w[2]}, t(M, D)
    n, r = ops.norm_residual(**c, **par)
    got = train_ops.norm_residual_backward(dnormed=dn, **c, **par)
    for lo in range(0, M, 1 << 22):
        cut = slice(lo, min(lo + (1 << 22), M))
        part = {k: v[cut] for k, v in c.items()}
        nw, rw = ops.norm_residual(**part, **par)
        want = train_ops.norm_residual_backward(dnormed=dn[cut], **part, **par)
        assert torch.equal(n[cut], nw) and torch.equal(r[cut], rw), lo
        for k in ("dy", "dgate", "dresidual"):
            assert torch.equal(got[k][cut], want[k]), (k, lo)
    assert all(torch.isfinite(got[k]).all() for k in ("dpre_w", "dpost_w", "dscale"))

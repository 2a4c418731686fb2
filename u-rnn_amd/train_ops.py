"""ctypes wrappers of the training entry points of the C ABI: backward of the ConvGRU / Skip-ConvGRU cell, the
stage convs, the transposed convs and the head; the loss; the clipped Adam step.  ``urnn_amd.training`` assembles them into SWP
windows and the training loop.  A backward call reads the scratch buffer its forward ran on (``fwd_ws``)."""
import ctypes

import torch

from . import ops
from ._lib import check, lib


def _bwd_scratch(scratch, nbytes, dev):
    """Backward scratch: ``scratch`` is the owner's ``ops.Arena`` (buffer "bwd", shared by all backward calls of a stream) or None
    (a fresh buffer for this call)."""
    return ops._scratch(scratch, nbytes, dev, key="bwd")


def gru_cell_backward(x, e, h, W1, W2, gn1_w, gn2_w, dh_out, I, fwd_ws, grads=None, accumulate=False, packed=None, dh_out2=None,
                      scratch=None, dh_out3=None, dh_out4=None, split_dh=False):
    """Gradients of one cell step.  ``fwd_ws`` is the scratch buffer the forward ``ops.gru_cell(x, e, h, ..., ws=fwd_ws)`` of the
    SAME inputs ran on (untouched since): it holds the raw gates / candidate and the GroupNorm statistics.
    W1 (2F,K[,1,1]) / W2 (F,K[,1,1]): conv weights in the reference layout.  Returns a dict with dx, de (when given), dh and
    dW1, db1, dg1, dbe1, dW2, db2, dg2, dbe2; pass ``grads`` (the dict of a previous call) with ``accumulate=True`` to add
    the parameter gradients of another timestep.  ``packed``: a one-element list the caller keeps per cell for the packed
    weights of the input-gradient GEMMs -- filled on the first call, reused until the caller empties it (after an optimizer
    step); None: packed on every call.  ``dh_out2`` .. ``dh_out4``: optional further terms of dL/dh' (added on the fly).  ``split_dh``:
    dL/dh is returned as two terms, ``dh`` + ``dh2`` (the second straight out of its GEMM), for a consumer that sums its terms itself --
    the previous timestep's call."""
    ops._dev_check(x, e, h, W1, W2, gn1_w, gn2_w, dh_out, dh_out2, dh_out3, dh_out4)
    B, F, H, W = h.shape
    K = I + (F if e is not None else 0) + F
    if W1.numel() != 2 * F * K or W2.numel() != F * K:
        raise RuntimeError(f"gru_cell_backward: weights do not match I={I}, F={F}, skip={e is not None}")
    L = lib()
    dev = h.device
    fwd = ops._scratch(fwd_ws, L.urnn_gru_cell_workspace_bytes(B, F, H, W), dev)
    ws = _bwd_scratch(scratch, L.urnn_gru_cell_backward_workspace_bytes(B, I, F, int(e is not None), H, W), dev)
    f32 = dict(dtype=torch.float32, device=dev)
    g = grads if grads is not None else {}
    if "dW1" not in g:          # caller-provided buffers (e.g. views of a flat gradient buffer) are written in place
        g.update(dW1=torch.empty(2 * F, K, **f32), db1=torch.empty(2 * F, **f32), dg1=torch.empty(2 * F, **f32),
                 dbe1=torch.empty(2 * F, **f32), dW2=torch.empty(F, K, **f32), db2=torch.empty(F, **f32),
                 dg2=torch.empty(F, **f32), dbe2=torch.empty(F, **f32))
        accumulate = False
    g["dh"] = torch.empty_like(h)
    g["dh2"] = torch.empty_like(h) if split_dh else None
    if x is not None and e is not None and B == 1:        # one block: a single GEMM writes dx | de in place
        dxe = torch.empty((1, I + F, H, W), **f32)
        g["dx"], g["de"] = dxe[:, :I], dxe[:, I:]
    else:
        g["dx"] = torch.empty_like(x) if x is not None else None
        g["de"] = torch.empty_like(e) if e is not None else None
    repack = packed is None or not packed
    if repack:
        pk = torch.empty(L.urnn_gru_cell_backward_packed_floats(I, F, int(e is not None)), **f32)
        if packed is not None:
            packed.append(pk)
    else:
        pk = packed[0]
    p = ops._ptr
    check(L.urnn_gru_cell_backward_f32(p(x), p(e), p(h), p(W1), p(W2), p(gn1_w), p(gn2_w), p(fwd), p(dh_out), p(dh_out2), p(dh_out3),
                                       p(dh_out4), p(g["dx"]), p(g["de"]),
                                       p(g["dh"]), p(g["dh2"]), p(g["dW1"]), p(g["db1"]), p(g["dg1"]), p(g["dbe1"]), p(g["dW2"]), p(g["db2"]),
                                       p(g["dg2"]), p(g["dbe2"]), p(pk), int(repack), p(ws), ws.numel(), B, I, F, H, W,
                                       int(bool(accumulate)), ops._stream()), "urnn_gru_cell_backward_f32")
    return g


def weight_gradient(dy, segs, dW=None, db=None, accumulate=False, scratch=None):
    """dW (N,K) = sum over pixels of dy (B,N,H,W) x cat(segs) (B,K,H,W) (1x1-conv weight gradient), db (N) likewise; segs: one to
    three (B,C_i,H,W) tensors."""
    L = lib()
    B, N, H, W = dy.shape
    Cs = [int(t.shape[1]) for t in segs] + [0] * (3 - len(segs))
    K = sum(Cs)
    dev = dy.device
    dW = torch.empty(N, K, device=dev) if dW is None else dW
    db = torch.empty(N, device=dev) if db is None else db
    ws = _bwd_scratch(scratch, L.urnn_weight_gradient_workspace_bytes(B, N, K, H, W), dev)
    p = ops._ptr
    ptrs = [p(t) for t in segs] + [None] * (3 - len(segs))
    check(L.urnn_weight_gradient_f32(p(dy), ptrs[0], Cs[0], ptrs[1], Cs[1], ptrs[2], Cs[2], p(dW), p(db), p(ws), ws.numel(), B, N,
                                     H, W, int(accumulate), ops._stream()), "urnn_weight_gradient_f32")
    return dW, db


def _layer_packs(packed, nfloats, dev):
    """Caller-kept packed weights of a layer's backward GEMMs: ``packed`` is None (pack per call) or a list that receives the
    buffer on first use and hands it back afterwards (the caller clears it when the parameters change).  -> (buffer, repack)"""
    if packed is None:
        return None, 1
    if not packed:
        packed.append(torch.empty(nfloats, dtype=torch.float32, device=dev))
        return packed[0], 1
    return packed[0], 0


def stage_conv_backward(x, weight, bias, dout, pool, dweight=None, dbias=None, accumulate=False, slope=ops.LRELU_SLOPE, scratch=None,
                        packed=None):
    """Backward of ``ops.stage_conv`` (conv1x1 + LeakyReLU [+ AvgPool2]).  weight (Cout,Cin[,1,1]), bias (Cout).
    Returns (dx, dweight, dbias)."""
    ops._dev_check(x, weight, bias, dout)
    B, Cin, H, W = x.shape
    Cout = weight.shape[0]
    L = lib()
    ws = _bwd_scratch(scratch, L.urnn_stage_conv_backward_workspace_bytes(B, Cin, Cout, H, W), x.device)
    if dweight is None:
        dweight, dbias, accumulate = torch.empty_like(weight), torch.empty_like(bias), False
    dx = torch.empty_like(x)
    p = ops._ptr
    pk, repack = _layer_packs(packed, L.urnn_stage_conv_backward_packed_floats(Cin, Cout), x.device)
    check(L.urnn_stage_conv_backward_f32(p(x), p(weight), p(bias), p(dout), p(dx), p(dweight), p(dbias), p(pk), repack, p(ws), ws.numel(),
                                         B, Cin, Cout, H, W, int(bool(pool)), slope, int(bool(accumulate)), ops._stream()),
          "urnn_stage_conv_backward_f32")
    return dx, dweight, dbias


def deconv2x2_backward(x, weight, out, dout, dweight=None, dbias=None, accumulate=False, slope=ops.LRELU_SLOPE, scratch=None,
                       packed=None):
    """Backward of ``ops.deconv2x2``.  weight (Cin,Cout,2,2); ``out`` is the forward output.  Returns (dx, dweight, dbias)."""
    ops._dev_check(x, weight, out, dout)
    B, Cin, H, W = x.shape
    Cout = weight.shape[1]
    L = lib()
    ws = _bwd_scratch(scratch, L.urnn_deconv2x2_backward_workspace_bytes(B, Cin, Cout, H, W), x.device)
    if dweight is None:
        dweight, dbias, accumulate = torch.empty_like(weight), torch.empty(Cout, dtype=torch.float32, device=x.device), False
    dx = torch.empty_like(x)
    p = ops._ptr
    pk, repack = _layer_packs(packed, L.urnn_deconv2x2_backward_packed_floats(Cin, Cout), x.device)
    check(L.urnn_deconv2x2_backward_f32(p(x), p(weight), p(out), p(dout), p(dx), p(dweight), p(dbias), p(pk), repack, p(ws), ws.numel(), B,
                                        Cin, Cout, H, W, slope, int(bool(accumulate)), ops._stream()), "urnn_deconv2x2_backward_f32")
    return dx, dweight, dbias


def head_backward(feat, conv_w, ln_w, ln_b, reg_w, out_raw, out_cls, dout, cls_thred, fwd_ws, grads=None, accumulate=False,
                  slope=ops.LRELU_SLOPE, scratch=None):
    """Backward of ``ops.head`` w.r.t. the masked depth.  ``fwd_ws``: the scratch the forward on the same ``feat`` ran on
    (``ops.head(..., want_raw=True, ws=fwd_ws)``, untouched since: it holds the five LayerNorm statistics).  conv_w (5,C,C), ln_w / ln_b (5,C,H,W), reg_w (C).
    Returns a dict: dfeat, dconv_w, dln_w, dln_b, dreg_w, dreg_b."""
    ops._dev_check(feat, conv_w, ln_w, ln_b, reg_w, out_raw, out_cls, dout)
    B, C, H, W = feat.shape
    L = lib()
    fwd = ops._scratch(fwd_ws, L.urnn_head_workspace_bytes(B, C, H, W), feat.device)
    ws = _bwd_scratch(scratch, L.urnn_head_backward_workspace_bytes(B, H, W), feat.device)
    f32 = dict(dtype=torch.float32, device=feat.device)
    g = grads if grads is not None else {}
    if grads is None or not accumulate:
        g.update(dconv_w=torch.empty_like(conv_w), dln_w=torch.empty_like(ln_w), dln_b=torch.empty_like(ln_b),
                 dreg_w=torch.empty(C, **f32), dreg_b=torch.empty(1, **f32))
    g["dfeat"] = torch.empty_like(feat)
    p = ops._ptr
    check(L.urnn_head_backward_f32(p(feat), p(conv_w), p(ln_w), p(ln_b), p(reg_w), p(fwd), p(out_raw), p(out_cls), p(dout), p(g["dfeat"]),
                                   p(g["dconv_w"]), p(g["dln_w"]), p(g["dln_b"]), p(g["dreg_w"]), p(g["dreg_b"]), p(ws), ws.numel(),
                                   B, C, H, W, float(cls_thred), slope, int(bool(accumulate)), ops._stream()), "urnn_head_backward_f32")
    return g


def loss(reg, target, cls_thred=0.0, want_grad=True, scratch=None):
    """FocalBCE_and_WMSE on a window's outputs.  Returns (components: 5-float device tensor [loss, loss_reg, wet MSE, dry MSE,
    loss_cls], dreg or None)."""
    ops._dev_check(reg, target)
    n = reg.numel()
    if target.numel() != n:
        raise RuntimeError("loss: reg and target differ in size")
    L = lib()
    ws = _bwd_scratch(scratch, L.urnn_loss_workspace_bytes(n), reg.device)
    comps = torch.empty(5, dtype=torch.float32, device=reg.device)
    dreg = torch.empty_like(reg) if want_grad else None
    check(L.urnn_loss_f32(ops._ptr(reg), ops._ptr(target), float(cls_thred), ops._ptr(comps), ops._ptr(dreg), ops._ptr(ws), ws.numel(), n,
                          ops._stream()), "urnn_loss_f32")
    return comps, dreg


def adam_step(params, grads, exp_avg, exp_avg_sq, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, max_grad_norm=0.0, step_dev=None,
              scratch=None):
    """In-place Adam step on flat float32 buffers (with optional global-norm clipping).  ``step_dev`` (int32 device scalar)
    overrides ``step`` for graph replay.  Returns a 2-float device tensor: (clip coefficient, gradient norm)."""
    ops._dev_check(params, grads, exp_avg, exp_avg_sq)
    if step_dev is not None and (not step_dev.is_cuda or step_dev.dtype != torch.int32):
        raise RuntimeError("adam_step: step_dev must be an int32 device scalar")
    n = params.numel()
    L = lib()
    ws = _bwd_scratch(scratch, L.urnn_adam_workspace_bytes(n), params.device)
    out = torch.empty(2, dtype=torch.float32, device=params.device)
    p = ops._ptr
    check(L.urnn_adam_step_f32(p(params), p(grads), p(exp_avg), p(exp_avg_sq), n, float(lr), float(betas[0]), float(betas[1]), float(eps),
                               int(step), p(step_dev), float(max_grad_norm), p(out), p(ws), ws.numel(), ops._stream()), "urnn_adam_step_f32")
    return out


# ---- sequence operators (ops.causal_conv, ops.selective_scan, ops.norm_residual) --------------------------------------------
def _param_grads_check(what, grads, accumulate, params, inputs, absent=()):
    """-> (the dict that receives the gradients, the buffers in it that the caller gave: apart from the inputs and from one another).
    ``absent``: gradients of parameters that this call does not have; a buffer for one would come back as if it were a gradient."""
    g = {} if grads is None else grads
    for k in absent:
        if g.get(k) is not None:
            raise RuntimeError(f"{what}: {k} in grads, but there is no {k[1:]}")
    if accumulate and any(g.get(k) is None for k in params):
        raise RuntimeError(f"{what}: accumulate needs the gradients {sorted(params)} in grads")
    given = [g[k] for k in params if g.get(k) is not None]
    if not given:
        return g, given
    for k, w in params.items():
        if g.get(k) is not None:
            ops._seq_check(what, k, g[k], tuple(w.shape), torch.float32, contiguous=True)
            ops._apart(what, k, g[k], (*inputs, *(t for t in given if t is not g[k])))
    if len({t.data_ptr() for t in given}) < len(given):
        raise RuntimeError(f"{what}: one buffer for several of the gradients {sorted(params)}")
    return g, given


def _param_grads(grads, params):
    """Buffers of the parameters' gradients: those of a former call's dict or the caller's own views, and new ones."""
    for k, w in params.items():
        if grads.get(k) is None:
            grads[k] = torch.empty_like(w)
    return grads


def causal_conv_backward(x, weight, dout, bias=None, state=None, lengths=None, silu=True, dstate_out=None, grads=None, accumulate=False,
                         scratch=None):
    """Backward of ``ops.causal_conv`` given dout (B,L,D) and, where the returned state was used further, ``dstate_out`` (B,K-1,D).
    Returns a dict: dx, dstate (None without state), dweight, dbias (None without bias); parameter gradients are float32, into the buffers
    of ``grads`` if given, added to them with ``accumulate``; a buffer for a parameter that the call does not have is refused."""
    what = "causal_conv_backward"
    dt = ops._seq_dtype(what, x)
    if x.dim() != 3:
        raise RuntimeError(f"{what}: x has shape {tuple(x.shape)}, expected (B, L, D)")
    B, L = x.shape[0], x.shape[1]
    D, K = ops._conv_seq_check(what, x, weight, bias, state, (B, L))
    ops._seq_check(what, "dout", dout, (B, L, D), x.dtype)
    ops._lengths_check(what, lengths, B)
    if dstate_out is not None:
        ops._seq_check(what, "dstate_out", dstate_out, (B, K - 1, D), x.dtype, contiguous=True)
    params = {"dweight": weight, **({"dbias": bias} if bias is not None else {})}
    inputs = (x, weight, dout, bias, state, lengths, dstate_out)
    g, given = _param_grads_check(what, grads, accumulate, params, inputs, absent=("dbias",) if bias is None else ())
    stream = ops._seq_device(what, *inputs, *given)
    L_ = lib()
    _param_grads(g, params)
    g.setdefault("dbias", None)
    g["dx"] = ops._empty_as(x)
    g["dstate"] = torch.empty_like(state) if state is not None else None
    ws = _seq_scratch(what, scratch, L_.urnn_causal_conv_backward_workspace_bytes(B, L, D, K), x.device, (*inputs, *given))
    p = ops._ptr
    check(L_.urnn_causal_conv_backward(p(x), *x.stride()[:2], p(weight), p(bias), p(state), p(lengths), p(dout), *dout.stride()[:2], p(dstate_out),
                                       p(g["dx"]), p(g["dstate"]), p(g["dweight"]), p(g["dbias"]), p(ws), ws.numel(), dt, B, L, D, K,
                                       int(bool(silu)), int(bool(accumulate)), stream), "urnn_causal_conv_backward")
    return g


def _seq_scratch(what, scratch, nbytes, dev, others):
    """Scratch of a sequence operator's backward (no status words: nothing in it needs to start at zero)."""
    if scratch is None:
        return torch.empty(int(nbytes), dtype=torch.uint8, device=dev)
    if isinstance(scratch, ops.Arena):
        scratch = _bwd_scratch(scratch, nbytes, dev)
    else:
        ops._seq_buffer(what, "scratch", scratch, nbytes, others)
    ops._seq_device(what, others[0], scratch)
    return scratch


def norm_residual_backward(y, pre_w, dnormed, dresidual_out=None, residual=None, post_w=None, gate=None, scale=None, gate_act="silu",
                           eps=ops.NORM_EPS, grads=None, accumulate=False, scratch=None):
    """Backward of ``ops.norm_residual`` given the gradients of its two outputs (either may be None).  Returns a dict: dy, dgate, dresidual
    (None without them), dpre_w, dpost_w, dscale (float32; None without them), as ``causal_conv_backward``."""
    what = "norm_residual_backward"
    dt = ops._seq_dtype(what, y)
    strides = ops._norm_check(what, y, pre_w, residual, post_w, gate, scale, gate_act)
    shape, D = tuple(y.shape), y.shape[-1]
    strides += ops._row_strides(what, y, (("dnormed", dnormed), ("dresidual_out", dresidual_out)))
    every = {"dpre_w": pre_w, "dpost_w": post_w, "dscale": scale}
    params = {k: w for k, w in every.items() if w is not None}
    inputs = (y, pre_w, dnormed, dresidual_out, residual, post_w, gate, scale)
    g, given = _param_grads_check(what, grads, accumulate, params, inputs, absent=every.keys() - params)
    stream = ops._seq_device(what, *inputs, *given)
    L_ = lib()
    _param_grads(g, params)
    new = lambda t: None if t is None else ops._empty_as(t)      # noqa: E731
    g["dy"], g["dgate"], g["dresidual"] = new(y), new(gate), new(residual)
    rows = y.numel() // D
    ws = _seq_scratch(what, scratch, L_.urnn_norm_residual_backward_workspace_bytes(rows, D), y.device, (*inputs, *given))
    p = ops._ptr
    out = [p(g[k]) if w is not None else 0 for k, w in every.items()]
    for k in every:
        g.setdefault(k, None)
    check(L_.urnn_norm_residual_backward(p(y), p(gate), p(residual), p(dnormed), p(dresidual_out), (ctypes.c_long * 10)(*strides), p(pre_w), p(post_w),
                                         p(scale), p(g["dy"]), p(g["dgate"]), p(g["dresidual"]), *out, p(ws), ws.numel(), dt, rows, ops._inner_rows(shape, rows), D,
                                         ops.GATE_ACTS[gate_act], float(eps), int(bool(accumulate)), stream), "urnn_norm_residual_backward")
    return g


def selective_scan_backward(u, delta, A, B, C, dout, fwd_ws, D=None, z=None, delta_bias=None, softplus=True, lengths=None, dstate_out=None,
                            want_dstate=False, grads=None, accumulate=False, scratch=None):
    """Backward of ``ops.selective_scan`` given dout (batch,L,dim) and, where the returned state was used further, ``dstate_out``
    (batch,dim,N).  ``fwd_ws``: the buffer that the forward of the SAME inputs ran with (``ws=``, untouched since): it holds the
    states the gradients need, the initial one among them.  Returns a dict: du, ddelta, dB, dC, dz in the
    activations' type and B's shape, dA, dD, ddelta_bias float32 (into the buffers of ``grads`` if given, added to them with ``accumulate``),
    dstate float32 with ``want_dstate``; None where there is no such input."""
    what = "selective_scan_backward"
    dt = ops._seq_dtype(what, u)
    if u.dim() != 3:
        raise RuntimeError(f"{what}: u has shape {tuple(u.shape)}, expected (batch, L, dim)")
    nb, L = u.shape[0], u.shape[1]
    B_given, C_given = B, C
    dim, G, N, B, C = ops._scan_check(what, u, delta, A, B, C, D, z, delta_bias, (nb, L))
    ops._seq_check(what, "dout", dout, (nb, L, dim), u.dtype)
    ops._lengths_check(what, lengths, nb)
    if dstate_out is not None:
        ops._seq_check(what, "dstate_out", dstate_out, (nb, dim, N), torch.float32, contiguous=True)
    if fwd_ws is None:
        raise RuntimeError(f"{what}: fwd_ws is None: run the forward with ws=ops.selective_scan_workspace(u, A)")
    every = {"dA": A, "dD": D, "ddelta_bias": delta_bias}
    params = {k: w for k, w in every.items() if w is not None}
    inputs = (u, delta, A, B, C, D, z, delta_bias, dout, lengths, dstate_out)
    g, given = _param_grads_check(what, grads, accumulate, params, inputs, absent=every.keys() - params)
    L_ = lib()
    record = ops._seq_buffer(what, "fwd_ws", fwd_ws, L_.urnn_selective_scan_workspace_bytes(nb, L, dim, N, 1), given)
    stream = ops._seq_device(what, *inputs, *given, record)
    _param_grads(g, params)
    g.setdefault("dD", None)
    g.setdefault("ddelta_bias", None)
    new = ops._empty_as
    g["du"], g["ddelta"], g["dB"], g["dC"] = new(u), new(delta), new(B_given), new(C_given)
    g["dz"] = new(z) if z is not None else None
    g["dstate"] = torch.empty((nb, dim, N), dtype=torch.float32, device=u.device) if want_dstate else None
    ws = _seq_scratch(what, scratch, L_.urnn_selective_scan_backward_workspace_bytes(nb, L, dim, G, N), u.device, (*inputs, *given, record))
    p = ops._ptr
    strides = (ctypes.c_long * 12)(*u.stride()[:2], *delta.stride()[:2], *B.stride()[:2], *C.stride()[:2], *(z.stride()[:2] if z is not None else (0, 0)),
                                   *dout.stride()[:2])
    check(L_.urnn_selective_scan_backward(p(u), p(delta), p(B), p(C), p(z), p(dout), strides, p(A), p(D), p(delta_bias), p(lengths), p(dstate_out),
                                          p(record), record.numel(), p(g["du"]), p(g["ddelta"]), p(g["dB"]), p(g["dC"]), p(g["dz"]), p(g["dA"]),
                                          p(g["dD"]) if D is not None else 0, p(g["ddelta_bias"]) if delta_bias is not None else 0, p(g["dstate"]),
                                          p(ws), ws.numel(), dt, nb, L, dim, G, N, int(bool(softplus)), int(bool(accumulate)), stream),
          "urnn_selective_scan_backward")
    return g

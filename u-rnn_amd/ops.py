"""Tensor-level wrappers over the C ABI: torch owns memory and streams, HIP kernels do the arithmetic.

Every function takes contiguous float32 CUDA(=HIP) tensors, passes ``data_ptr()`` + dims + the current
stream across the ABI and returns torch tensors.  No op has a PyTorch fallback.
"""
import ctypes
import os

import torch

from ._lib import check, lib

LRELU_SLOPE = 0.2   # get_activation("lrelu"), utils.py:63
NORM_EPS = 1e-5     # nn.GroupNorm / nn.LayerNorm default eps


MATRIX_MODES = {"fp32": 0, "bf16": 1, "fp32_mfma": 2, "fp32_cand": 3}


class matrix_mode:
    """``with ops.matrix_mode("bf16"):`` -- GEMM arithmetic of the launches enqueued inside (include/urnn_hip.h
    urnn_set_matrix_mode): "fp32" = the reference's semantics on the 16-bit matrix pipe (default), "bf16" = bf16 compute with fp32
    accumulation, "fp32_mfma" = the exact fp32 matrix instructions everywhere (slower), "fp32_cand" = the default except for the
    full-resolution cells' candidate GEMM on the fp32 instruction (a few per cent slower; plain-fp32 torch's long-rollout error)."""

    def __init__(self, mode):
        self.mode = MATRIX_MODES[mode]

    def __enter__(self):
        self.prev = lib().urnn_get_matrix_mode()
        check(lib().urnn_set_matrix_mode(self.mode), "urnn_set_matrix_mode")
        return self

    def __exit__(self, *exc):
        lib().urnn_set_matrix_mode(self.prev)
        return False


class _NoGuard:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


class _ExactGuard:
    """The launches inside run with URNN_MATRIX_FP32_MFMA when the process is in one of the f16-piece modes."""

    def __enter__(self):
        self.prev = lib().urnn_get_matrix_mode()
        if self.prev in (MATRIX_MODES["fp32"], MATRIX_MODES["fp32_cand"]):
            check(lib().urnn_set_matrix_mode(MATRIX_MODES["fp32_mfma"]), "urnn_set_matrix_mode")
        return self

    def __exit__(self, *exc):
        lib().urnn_set_matrix_mode(self.prev)
        return False


def exact_matrix_if(flag):
    """``with ops.exact_matrix_if(layer_has_a_weight_beyond_f16_range): launch(...)`` -- the f16 x 3 forward arithmetic is finite for
    |weight| < 64 (include/urnn_hip.h); a layer outside that range takes the exact fp32 matrix instruction instead of NaN."""
    return _ExactGuard() if flag else _NO_GUARD


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dev_check(*tensors):
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("urnn_amd ops need tensors on the GPU (cuda:N / HIP device); there is no CPU path")
        if t.dtype != torch.float32:
            raise RuntimeError(f"urnn_amd ops are float32 only (got {t.dtype})")
        if not t.is_contiguous():
            raise RuntimeError("urnn_amd ops need contiguous tensors")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def tuning_env(name, default):
    """Development knobs (URNN_TUNE_*: A/B switches of the schedules) are read ONLY when URNN_TUNING=1 is set -- the product path
    takes every default whatever else the environment holds (the library's own knobs exist in -DURNN_TUNING builds only)."""
    if os.environ.get("URNN_TUNING") != "1":
        return default
    return os.environ.get(name, default)


def workspace(nbytes, device):
    """A scratch buffer of ``nbytes`` bytes (caller-owned, as the C ABI requires)."""
    # the first 16 KB of a cell / head workspace are STATUS words that kernels only ever OR into and the cooperative launches' barrier
    # words (include/urnn_hip.h URNN_STATUS_AREA_BYTES): only those need to start at zero -- the rest is scratch every kernel writes
    # before it reads (tens of MB per full-resolution cell)
    buf = torch.empty(int(nbytes), dtype=torch.uint8, device=device)
    buf[:min(STATUS_AREA_BYTES, int(nbytes))].zero_()
    return buf


class Arena:
    """Scratch buffers OWNED BY ONE engine / trainer, keyed by name (GroupNorm / LayerNorm partials, raw gates, backward
    scratch).  There is deliberately no process-wide pool: a captured hipGraph holds raw pointers into its scratch, so the
    buffers must live exactly as long as the owner's graphs.  Grow-only; growing a buffer bumps ``generation`` (an owner that
    captured graphs compares it and re-captures) and is refused while a capture is running."""

    def __init__(self, device):
        self.device = torch.device(device)
        self._buf = {}
        self.generation = 0

    def get(self, key, nbytes):
        buf = self._buf.get(key)
        if buf is None or buf.numel() < nbytes:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("scratch buffer %r must be sized before graph capture (run the path once eagerly)" % (key,))
            buf = workspace(nbytes, self.device)
            self._buf[key] = buf
            self.generation += 1
        return buf


def _scratch(ws, nbytes, device, key="ws"):
    """ws: None (a fresh buffer for this call), an Arena (its buffer ``key``) or a uint8 tensor of at least nbytes."""
    if ws is None:
        return workspace(nbytes, device)
    if isinstance(ws, Arena):
        return ws.get(key, nbytes)
    if ws.numel() < nbytes:
        raise RuntimeError(f"workspace of {ws.numel()} bytes given, {nbytes} needed")
    return ws


def gru_cell_workspace_bytes(B, F, H, W):
    return lib().urnn_gru_cell_workspace_bytes(B, F, H, W)


def _counter_check(*counters):
    for c in counters:
        if c is None or not c.is_cuda or c.dtype != torch.int32 or c.numel() != 1:
            raise RuntimeError("frame counters are int32 device scalars")


def head_workspace_bytes(B, C, H, W):
    return lib().urnn_head_workspace_bytes(B, C, H, W)


STATUS_AREA_BYTES = 16384                                               # include/urnn_hip.h URNN_STATUS_AREA_BYTES
STATUS_GATES, STATUS_CAND, STATUS_HEAD, STATUS_BARRIER = 1, 2, 4, 8     # include/urnn_hip.h: word 0 of a cell / head workspace
STATUS_NAMES = {STATUS_GATES: "GroupNorm sums of a cell's gates", STATUS_CAND: "GroupNorm sums of a cell's candidate",
                STATUS_HEAD: "LayerNorm sums of the head",
                STATUS_BARRIER: "a cooperative launch's grid barrier gave up (its blocks were not all resident: the GPU is shared, "
                                "partitioned or masked)"}


def workspace_status(ws):
    """Word 0 of a workspace's status area (0 = every norm's statistics were finite).  Reads the device: synchronises."""
    return int(ws[:4].view(torch.int32).item())


def max_abs(values):
    """max |v| of a float32 device tensor as a python float (urnn_max_abs_f32; NaN if any element is NaN)."""
    _dev_check(values)
    out = torch.empty(1, dtype=torch.float32, device=values.device)
    check(lib().urnn_max_abs_f32(_ptr(values), values.numel(), _ptr(out), _stream()), "urnn_max_abs_f32")
    return float(out.item())


# ---- weight packing ----------------------------------------------------------------------------------
def pack_conv(weight, bias):
    """nn.Conv2d (Cout,Cin,1,1) [+ bias] -> packed buffer for stage_conv."""
    _dev_check(weight, bias)
    Cout, Cin = weight.shape[0], weight.shape[1]
    L = lib()
    out = torch.empty(L.urnn_packed_conv_floats(Cin, Cout), dtype=torch.float32, device=weight.device)
    check(L.urnn_pack_conv_f32(_ptr(weight), _ptr(bias), _ptr(out), Cin, Cout, _stream()), "urnn_pack_conv_f32")
    return out


def pack_gru(W1, b1, W2, b2, I, F, skip):
    _dev_check(W1, b1, W2, b2)
    L = lib()
    out = torch.empty(L.urnn_packed_gru_floats(I, F, int(skip)), dtype=torch.float32, device=W1.device)
    check(L.urnn_pack_gru_f32(_ptr(W1), _ptr(b1), _ptr(W2), _ptr(b2), _ptr(out), I, F, int(skip), _stream()),
          "urnn_pack_gru_f32")
    return out


def pack_deconv(weight, bias):
    """nn.ConvTranspose2d (Cin,Cout,2,2) + bias -> packed buffer for deconv2x2."""
    _dev_check(weight, bias)
    Cin, Cout = weight.shape[0], weight.shape[1]
    L = lib()
    out = torch.empty(L.urnn_packed_deconv_floats(Cin, Cout), dtype=torch.float32, device=weight.device)
    check(L.urnn_pack_deconv_f32(_ptr(weight), _ptr(bias), _ptr(out), Cin, Cout, _stream()), "urnn_pack_deconv_f32")
    return out


# ---- forwards ----------------------------------------------------------------------------------------
def stage_conv_stem_applies(B, Cin, Cout, H, W):
    """Can the flat conv to the head's 16 channels take the head's first LayerNorm statistics in its epilogue (urnn_stage_conv_stem_f32)?"""
    return bool(lib().urnn_stage_conv_stem_applies(B, Cin, Cout, H, W))


def stage_conv(x, packed, Cout, pool, out=None, slope=LRELU_SLOPE, head_w=None, head_partial0=None):
    """[AvgPool2](LeakyReLU(conv1x1(x))): x (B,Cin,H,W) -> (B,Cout,H[/2],W[/2]).  ``head_w`` (the head's conv_w) + ``head_partial0``
    (``head_tail_partial``): the decoder's last conv also leaves the head's first LayerNorm partials there (``stage_conv_stem_applies``)."""
    _dev_check(x, packed, out)
    B, Cin, H, W = x.shape
    if out is None:
        out = torch.empty((B, Cout, H // 2, W // 2) if pool else (B, Cout, H, W), dtype=torch.float32, device=x.device)
    if head_w is not None:
        if pool or head_partial0 is None:
            raise ValueError("the head's statistics go with the flat conv and need their partial buffer")
        check(lib().urnn_stage_conv_stem_f32(_ptr(x), _ptr(packed), _ptr(out), B, Cin, Cout, H, W, slope, _ptr(head_w), _ptr(head_partial0),
                                             _stream()), "urnn_stage_conv_stem_f32")
        return out
    check(lib().urnn_stage_conv_f32(_ptr(x), _ptr(packed), _ptr(out), B, Cin, Cout, H, W, 1 if pool else 0, slope,
                                    _stream()), "urnn_stage_conv_f32")
    return out


PHASE_GATES, PHASE_GN1, PHASE_CAND, PHASE_GN2, PHASE_BLEND, PHASE_ALL = 1, 2, 4, 8, 16, 31
PHASE_COOP = 64        # modifier: the whole cell of a small plane as one cooperative launch (include/urnn_hip.h URNN_PHASE_COOP)
PHASE_FUSED_R = 32     # modifier: reset gate recomputed inside the candidate kernel (include/urnn_hip.h URNN_PHASE_FUSED_R)


def gru_cell(x, e, h, packed, gn1_w, gn1_b, gn2_w, gn2_b, I, out=None, eps=NORM_EPS, phases=PHASE_ALL, ws=None):
    """ConvGRU (e None) / Skip-ConvGRU step.  x may be None (zeros, I channels).  out may be h (in place).
    ``phases`` enqueues a subset of the cell's five kernels (profiling only).  ``ws``: the cell's scratch (``_scratch``); the
    backward pass reads the forward's scratch, so training passes the same buffer to both."""
    _dev_check(x, e, h, packed, gn1_w, gn1_b, gn2_w, gn2_b, out)
    B, F, H, W = h.shape
    if x is not None and tuple(x.shape) != (B, I, H, W):
        raise RuntimeError(f"gru_cell: x has shape {tuple(x.shape)}, expected {(B, I, H, W)}")
    if e is not None and tuple(e.shape) != (B, F, H, W):
        raise RuntimeError(f"gru_cell: e has shape {tuple(e.shape)}, expected {(B, F, H, W)}")
    L = lib()
    ws = _scratch(ws, L.urnn_gru_cell_workspace_bytes(B, F, H, W), h.device)
    if out is None:
        out = torch.empty_like(h)
    check(L.urnn_gru_cell_phases_f32(_ptr(x), _ptr(e), _ptr(h), _ptr(packed), _ptr(gn1_w), _ptr(gn1_b), _ptr(gn2_w),
                                     _ptr(gn2_b), _ptr(out), _ptr(ws), ws.numel(), B, I, F, H, W, eps, int(phases),
                                     _stream()), "urnn_gru_cell_f32")
    return out


def gru_cell_tail_applies(B, F, H, W, Cout, pool):
    """Can the end of a cell on (B, F, H, W) be fused with its consumer, a 1x1 conv F -> Cout (pool: + AvgPool2)?"""
    return bool(lib().urnn_gru_cell_tail_applies(B, F, H, W, Cout, 1 if pool else 0))


def head_tail_partial(B, H, W, device):
    """Buffer for the head's first LayerNorm statistics when the kernel that produces the feature map takes them (gru_cell_tail)."""
    return torch.zeros(lib().urnn_head_tail_partial_floats(B, H, W), dtype=torch.float32, device=device)


def gru_cell_tail(x, e, h, packed, gn1_w, gn1_b, gn2_w, gn2_b, I, conv_packed, Cout, pool, conv_out=None, out=None, eps=NORM_EPS,
                  phases=PHASE_ALL, ws=None, head_w=None, head_partial0=None, slope=LRELU_SLOPE):
    """``gru_cell`` whose last kernel (GroupNorm finalize + blend) also runs the 1x1 conv that consumes the new state:
    returns (h', [AvgPool2](LeakyReLU(conv(h')))).  ``head_w`` (the head's stem conv (16,16)) + ``head_partial0``: the launch also
    takes the head's first LayerNorm statistics (``head(..., partial0=head_partial0)`` then skips its first pass)."""
    _dev_check(x, e, h, packed, gn1_w, gn1_b, gn2_w, gn2_b, out, conv_packed, conv_out, head_w, head_partial0)
    B, F, H, W = h.shape
    L = lib()
    ws = _scratch(ws, L.urnn_gru_cell_workspace_bytes(B, F, H, W), h.device)
    if out is None:
        out = torch.empty_like(h)
    if conv_out is None:
        conv_out = torch.empty((B, Cout, H // 2, W // 2) if pool else (B, Cout, H, W), dtype=torch.float32, device=h.device)
    check(L.urnn_gru_cell_tail_f32(_ptr(x), _ptr(e), _ptr(h), _ptr(packed), _ptr(gn1_w), _ptr(gn1_b), _ptr(gn2_w), _ptr(gn2_b), _ptr(out),
                                   _ptr(ws), ws.numel(), B, I, F, H, W, eps, int(phases), _ptr(conv_packed), int(Cout), 1 if pool else 0,
                                   slope, _ptr(conv_out), _ptr(head_w), _ptr(head_partial0), _stream()), "urnn_gru_cell_tail_f32")
    return out, conv_out


def gru_cell_strip(x, e, h, packed, gn1_w, gn1_b, gn2_w, gn2_b, I, global_pixels, exchange, out=None, eps=NORM_EPS, ws=None):
    """One horizontal strip of a cell step whose plane of ``global_pixels`` pixels is split over ranks (include/urnn_hip.h,
    "Spatial strips").  ``exchange(sums)`` must all-reduce (sum) the float64 device tensor in place; it is called twice."""
    _dev_check(x, e, h, packed, gn1_w, gn1_b, gn2_w, gn2_b, out)
    B, F, H, W = h.shape
    L = lib()
    ws = _scratch(ws, L.urnn_gru_cell_workspace_bytes(B, F, H, W), h.device)
    if out is None:
        out = torch.empty_like(h)

    def phase(mask):
        check(L.urnn_gru_cell_strip_f32(_ptr(x), _ptr(e), _ptr(h), _ptr(packed), _ptr(gn1_w), _ptr(gn1_b), _ptr(gn2_w), _ptr(gn2_b),
                                        _ptr(out), _ptr(ws), ws.numel(), B, I, F, H, W, eps, mask, int(global_pixels), _stream()),
              "urnn_gru_cell_strip_f32")

    def swap(which, groups):
        sums = torch.empty((B, groups, 2), dtype=torch.float64, device=h.device)
        for direction in (0, 1):
            check(L.urnn_gru_cell_strip_stats_f32(_ptr(ws), ws.numel(), B, F, H, W, which, direction, _ptr(sums), _stream()),
                  "urnn_gru_cell_strip_stats_f32")
            if direction == 0:
                exchange(sums)

    phase(PHASE_GATES)
    swap(1, 2 * F // 32)
    phase(PHASE_CAND)
    swap(2, F // 32)
    phase(PHASE_GN2 | PHASE_BLEND)
    return out


def head_strip(feat, conv_w, ln_w, ln_b, cls_w, cls_b, reg_w, reg_b, cls_thred, global_pixels, exchange, want_raw=False, eps=NORM_EPS,
               slope=LRELU_SLOPE, ws=None):
    """One strip of the head: ln_w / ln_b are the strip's rows (5,C,H,W); three statistics exchanges (LayerNorm levels)."""
    _dev_check(feat, conv_w, ln_w, ln_b, cls_w, cls_b, reg_w, reg_b)
    B, C, H, W = feat.shape
    L = lib()
    ws = _scratch(ws, L.urnn_head_workspace_bytes(B, C, H, W), feat.device)
    f32 = dict(dtype=torch.float32, device=feat.device)
    masked, cls = torch.empty((B, H, W), **f32), torch.empty((B, H, W), **f32)
    raw = torch.empty((B, H, W), **f32) if want_raw else None

    def phase(mask):
        check(L.urnn_head_strip_f32(_ptr(feat), _ptr(conv_w), _ptr(ln_w), _ptr(ln_b), _ptr(cls_w), _ptr(cls_b), _ptr(reg_w), _ptr(reg_b),
                                    _ptr(masked), _ptr(cls), _ptr(raw), None, _ptr(ws), ws.numel(), B, C, H, W, float(cls_thred), eps,
                                    slope, mask, int(global_pixels), _stream()), "urnn_head_strip_f32")

    for level in range(3):
        phase(1 << (2 * level))                                   # K1 / K2 / K3: convs + partial sums of the level's norms
        sums = torch.empty((1 if level == 0 else 2, B, 2), dtype=torch.float64, device=feat.device)
        for direction in (0, 1):
            check(L.urnn_head_strip_stats_f32(_ptr(ws), ws.numel(), B, C, H, W, level, direction, _ptr(sums), _stream()),
                  "urnn_head_strip_stats_f32")
            if direction == 0:
                exchange(sums)
        phase(2 << (2 * level))                                   # F1 / F2 / F3
    phase(64)                                                     # K4
    return masked, cls, raw


def deconv2x2(x, packed, Cout, out=None, slope=LRELU_SLOPE):
    """LeakyReLU(ConvTranspose2d(k=2,s=2)(x)): (B,Cin,H,W) -> (B,Cout,2H,2W)."""
    _dev_check(x, packed, out)
    B, Cin, H, W = x.shape
    if out is None:
        out = torch.empty((B, Cout, 2 * H, 2 * W), dtype=torch.float32, device=x.device)
    check(lib().urnn_deconv2x2_f32(_ptr(x), _ptr(packed), _ptr(out), B, Cin, Cout, H, W, slope, _stream()),
          "urnn_deconv2x2_f32")
    return out


def head(feat, conv_w, ln_w, ln_b, cls_w, cls_b, reg_w, reg_b, cls_thred, out_masked=None, out_cls=None, out_raw=None,
         frame_index=None, want_raw=False, eps=NORM_EPS, slope=LRELU_SLOPE, ws=None, partial0=None, coop=False, frame_next=None):
    """Dual head + mask.  Returns (masked, cls, raw|None), each (B,H,W) unless preallocated (T,B,H,W) buffers
    plus a device ``frame_index`` are given.  ``frame_next`` (captured frame loops): the int32 device word that receives
    ``frame_index + 1`` -- the next head's ``frame_index``; two words used alternately are a frame counter without a kernel of its own
    (urnn_head_rollout_f32)."""
    _dev_check(feat, conv_w, ln_w, ln_b, cls_w, cls_b, reg_w, reg_b, out_masked, out_cls, out_raw)
    B, C, H, W = feat.shape
    L = lib()
    ws = _scratch(ws, L.urnn_head_workspace_bytes(B, C, H, W), feat.device)
    if out_masked is None:
        out_masked = torch.empty((B, H, W), dtype=torch.float32, device=feat.device)
    if out_cls is None:
        out_cls = torch.empty((B, H, W), dtype=torch.float32, device=feat.device)
    if out_raw is None and want_raw:
        out_raw = torch.empty((B, H, W), dtype=torch.float32, device=feat.device)
    if frame_next is not None:
        _dev_check(partial0)
        _counter_check(frame_index, frame_next)
        check(L.urnn_head_rollout_f32(_ptr(feat), _ptr(conv_w), _ptr(ln_w), _ptr(ln_b), _ptr(cls_w), _ptr(cls_b), _ptr(reg_w),
                                      _ptr(reg_b), _ptr(out_masked), _ptr(out_cls), _ptr(out_raw), _ptr(frame_index), _ptr(ws),
                                      ws.numel(), B, C, H, W, float(cls_thred), eps, slope, int(bool(coop) and partial0 is None),
                                      _ptr(partial0), _ptr(frame_next), _stream()), "urnn_head_rollout_f32")
        return out_masked, out_cls, out_raw
    if partial0 is not None:      # the first LayerNorm's statistics were taken by the kernel that produced feat (gru_cell_tail)
        _dev_check(partial0)
        check(L.urnn_head_after_tail_f32(_ptr(feat), _ptr(conv_w), _ptr(ln_w), _ptr(ln_b), _ptr(cls_w), _ptr(cls_b), _ptr(reg_w),
                                         _ptr(reg_b), _ptr(out_masked), _ptr(out_cls), _ptr(out_raw), _ptr(frame_index), _ptr(ws),
                                         ws.numel(), B, C, H, W, float(cls_thred), eps, slope, _ptr(partial0), _stream()),
              "urnn_head_after_tail_f32")
        return out_masked, out_cls, out_raw
    fn, what = (L.urnn_head_coop_f32, "urnn_head_coop_f32") if coop else (L.urnn_head_f32, "urnn_head_f32")   # coop: one cooperative launch
    check(fn(_ptr(feat), _ptr(conv_w), _ptr(ln_w), _ptr(ln_b), _ptr(cls_w), _ptr(cls_b), _ptr(reg_w),
             _ptr(reg_b), _ptr(out_masked), _ptr(out_cls), _ptr(out_raw), _ptr(frame_index), _ptr(ws),
             ws.numel(), B, C, H, W, float(cls_thred), eps, slope, _stream()), what)
    return out_masked, out_cls, out_raw


def preprocess(rain, cumsum, dem, imperv, manhole, dem_min, dem_max, t, nums, rain_max, cumsum_max, out=None, t_dev=None, t_next=None):
    """Per-frame input assembly: returns (B, 2*nums+3, H, W).  rain/cumsum (B,T) scalar or (B,T,H,W) spatial;
    dem/imperv/manhole (B,H,W).  ``t_dev`` (int32 device scalar) overrides ``t`` for graph replay; ``t_next``: the device word that
    receives ``t_dev + 1``, the next frame's ``t_dev`` (urnn_preprocess_rollout_f32)."""
    _dev_check(rain, cumsum, dem, imperv, manhole, out)
    B, H, W = dem.shape
    T = rain.shape[1]
    spatial = 1 if rain.dim() == 4 else 0
    C = 2 * nums + 3
    if out is None:
        out = torch.empty((B, C, H, W), dtype=torch.float32, device=dem.device)
    if t_next is not None:
        _counter_check(t_dev, t_next)
        check(lib().urnn_preprocess_rollout_f32(_ptr(rain), _ptr(cumsum), _ptr(dem), _ptr(imperv), _ptr(manhole), float(dem_min),
                                                float(dem_max), _ptr(out), _ptr(t_dev), _ptr(t_next), B, T, nums, H, W, spatial,
                                                float(rain_max), float(cumsum_max), _stream()), "urnn_preprocess_rollout_f32")
        return out
    check(lib().urnn_preprocess_f32(_ptr(rain), _ptr(cumsum), _ptr(dem), _ptr(imperv), _ptr(manhole), float(dem_min),
                                    float(dem_max), _ptr(out), int(t), _ptr(t_dev), B, T, nums, H, W, spatial,
                                    float(rain_max), float(cumsum_max), _stream()), "urnn_preprocess_f32")
    return out


def stage1_static(dem, imperv, manhole, dem_min, dem_max, weight, nums, out=None):
    """Static part of encoder stage 1 for scalar-rain events: S (B,Cout,H,W), once per event."""
    _dev_check(dem, imperv, manhole, weight, out)
    B, H, W = dem.shape
    Cout = weight.shape[0]
    if out is None:
        out = torch.empty((B, Cout, H, W), dtype=torch.float32, device=dem.device)
    check(lib().urnn_stage1_static_f32(_ptr(dem), _ptr(imperv), _ptr(manhole), float(dem_min), float(dem_max), _ptr(weight),
                                       _ptr(out), B, int(nums), Cout, H, W, _stream()), "urnn_stage1_static_f32")
    return out


def stage1_scalar_rain(S, rain, cumsum, weight, bias, t, nums, rain_max, cumsum_max, out=None, t_dev=None, slope=LRELU_SLOPE,
                       t_next=None):
    """preprocess_inputs + Encoder.stage1 for scalar rain: LeakyReLU(S + v_t) -> (B,Cout,H,W).  ``t_next`` as in preprocess."""
    _dev_check(S, rain, cumsum, weight, bias, out)
    B, Cout, H, W = S.shape
    if out is None:
        out = torch.empty_like(S)
    if t_next is not None:
        _counter_check(t_dev, t_next)
        check(lib().urnn_stage1_scalar_rain_rollout_f32(_ptr(S), _ptr(rain), _ptr(cumsum), _ptr(weight), _ptr(bias), _ptr(out),
                                                        _ptr(t_dev), _ptr(t_next), B, rain.shape[1], int(nums), Cout, H, W,
                                                        float(rain_max), float(cumsum_max), slope, _stream()),
              "urnn_stage1_scalar_rain_rollout_f32")
        return out
    check(lib().urnn_stage1_scalar_rain_f32(_ptr(S), _ptr(rain), _ptr(cumsum), _ptr(weight), _ptr(bias), _ptr(out), int(t),
                                            _ptr(t_dev), B, rain.shape[1], int(nums), Cout, H, W, float(rain_max),
                                            float(cumsum_max), slope, _stream()), "urnn_stage1_scalar_rain_f32")
    return out


def advance_counter(counter, delta=1):
    check(lib().urnn_advance_counter(_ptr(counter), int(delta), _stream()), "urnn_advance_counter")


# ---- sequence operators --------------------------------------------------------------------------------------------------
# Short causal convolution, selective state space scan and the norms around a block, over (batch, length, channels) tensors.  They take
# float32, bfloat16 or float16 activations (parameters, states of the scan and parameter gradients are float32) whose channels are
# adjacent: a slice of a wider projection goes in as it is.  Their gradients are in train_ops.
SEQ_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # include/urnn_hip.h URNN_F32 / URNN_BF16 / URNN_F16
GATE_ACTS = {"none": 0, "sigmoid": 1, "silu": 2}                         # include/urnn_hip.h URNN_GATE_*


def _seq_dtype(what, t):
    code = SEQ_DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"{what}: activations are float32, bfloat16 or float16 (got {t.dtype})")
    return code


def _seq_check(what, name, t, shape, dtype, contiguous=False):
    """Shape, type and layout of an argument (no device is needed to refuse a wrong one)."""
    if t.shape == shape and t.dtype is dtype and (t.is_contiguous() if contiguous else t.stride(-1) == 1):
        return
    if tuple(t.shape) != shape:
        raise RuntimeError(f"{what}: {name} has shape {tuple(t.shape)}, expected {shape}")
    if t.dtype != dtype:
        raise RuntimeError(f"{what}: {name} is {t.dtype}, expected {dtype}")
    if contiguous:
        if not t.is_contiguous():
            raise RuntimeError(f"{what}: {name} must be contiguous")
    elif t.stride(-1) != 1 and t.shape[-1] != 1:
        raise RuntimeError(f"{what}: the channels of {name} must be adjacent (stride {t.stride(-1)})")


# The current stream as the C ABI takes it, without the stream object that torch.cuda.current_stream() builds (2.7 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _seq_device(what, *tensors):
    """All on the current device: kernels are enqueued on its current stream.  Returns that stream."""
    cur = tensors[0].get_device()                        # -1: a CPU tensor
    if cur >= 0 and cur == torch.cuda.current_device():
        for t in tensors:
            if t is not None and t.get_device() != cur:
                break
        else:
            return _raw_stream(cur)
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{what}: urnn_amd ops need tensors on the GPU (cuda:N / HIP device); there is no CPU path")
        if dev is None:
            dev = t.device
            if dev.index != torch.cuda.current_device():
                raise RuntimeError(f"{what}: tensors are on {dev}, the current device is cuda:{torch.cuda.current_device()}")
        elif t.device != dev:
            raise RuntimeError(f"{what}: tensors on {dev} and {t.device}")


# A single-token call is bound by its way here (11 to 15 us against 3 to 4 on the device): array types made once, and an output
# from the input it looks like.
_Long5, _Long6 = ctypes.c_long * 5, ctypes.c_long * 6


def _empty_as(t):
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _span(t):
    if t.is_contiguous():
        return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
    return t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _seq_out(what, name, t, shape, dtype, inputs, same=()):
    """A given output buffer: contiguous, of the result's shape, and apart from every input (``same``: inputs it may be exactly)."""
    _seq_check(what, name, t, shape, dtype, contiguous=True)
    lo = t.data_ptr()
    hi = lo + t.numel() * t.element_size()
    for x in inputs:
        if x is None:
            continue
        a = x.data_ptr()
        if a >= hi or (a < lo and _span(x)[1] <= lo) or x.numel() == 0:
            continue
        if a != lo or not any(x is s for s in same) or not x.is_contiguous():
            raise RuntimeError(f"{what}: {name} overlaps an input")


def _seq_buffer(what, name, buf, nbytes, others):
    """A workspace or record that the caller gives: nbytes of plain bytes, apart from every tensor of the call."""
    if not isinstance(buf, torch.Tensor) or buf.dtype != torch.uint8 or not buf.is_contiguous():
        raise RuntimeError(f"{what}: {name} is a contiguous uint8 tensor")
    if buf.numel() < nbytes:
        raise RuntimeError(f"{what}: {name} of {buf.numel()} bytes given, {nbytes} needed")
    _apart(what, name, buf, others)
    return buf


def _apart(what, name, t, others):
    lo, hi = _span(t)
    for x in others:
        if x is None:
            continue
        a = x.data_ptr()
        if a < hi and (a >= lo or _span(x)[1] > lo) and x.numel():
            raise RuntimeError(f"{what}: {name} overlaps another tensor of the call")


def _lengths_check(what, lengths, B):
    if lengths is not None:
        _seq_check(what, "lengths", lengths, (B,), torch.int32, contiguous=True)


def _no_empty(what, t):
    if t.numel() == 0:
        raise RuntimeError(f"{what}: empty input of shape {tuple(t.shape)}")


def _conv_seq_check(what, x, weight, bias, state, lead):
    _no_empty(what, x)
    D = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != D or not 2 <= weight.shape[1] <= 4:
        raise RuntimeError(f"{what}: weight has shape {tuple(weight.shape)}, expected ({D}, 2..4)")
    K = weight.shape[1]
    if (x.shape == lead + (D,) and x.stride(-1) == 1 and weight.dtype is torch.float32 and weight.is_contiguous()      # the usual call, in one go
            and (bias is None or (bias.shape == (D,) and bias.dtype is torch.float32 and bias.is_contiguous()))
            and (state is None or (state.shape == (lead[0], K - 1, D) and state.dtype is x.dtype and state.is_contiguous()))):
        return D, K
    _seq_check(what, "x", x, lead + (D,), x.dtype)
    _seq_check(what, "weight", weight, (D, K), torch.float32, contiguous=True)
    if bias is not None:
        _seq_check(what, "bias", bias, (D,), torch.float32, contiguous=True)
    if state is not None:
        _seq_check(what, "state", state, (lead[0], K - 1, D), x.dtype, contiguous=True)
    return D, K


def causal_conv(x, weight, bias=None, state=None, lengths=None, silu=True, out=None, want_state=False, state_out=None):
    """Short causal depthwise convolution along time: y[:, t] = silu(bias + sum_k weight[:, k] * line[:, t + k]), line = [state | x].

    x (B,L,D); weight (D,K), K = 2..4; bias (D); ``state`` (B,K-1,D): the inputs before the first token, oldest first (None: zeros);
    ``lengths`` (B) int32: tokens of each sequence of a padded batch -- later ones are not read and give zeros.  ``silu`` False: no
    activation.  Returns y (B,L,D), or (y, state (B,K-1,D)) with ``want_state``: the last K-1 inputs of every sequence, what the next
    call or ``causal_conv_step`` goes on from."""
    what = "causal_conv"
    dt = _seq_dtype(what, x)
    if x.dim() != 3:
        raise RuntimeError(f"{what}: x has shape {tuple(x.shape)}, expected (B, L, D)")
    B, L = x.shape[0], x.shape[1]
    D, K = _conv_seq_check(what, x, weight, bias, state, (B, L))
    _lengths_check(what, lengths, B)
    if out is not None:
        _seq_out(what, "out", out, (B, L, D), x.dtype, (x, weight, bias, state, lengths, state_out))
    if state_out is not None:
        _seq_out(what, "state_out", state_out, (B, K - 1, D), x.dtype, (x, weight, bias, state, lengths))
    stream = _seq_device(what, x, weight, bias, state, lengths, out, state_out)
    if out is None:
        out = _empty_as(x)
    if want_state and state_out is None:
        state_out = torch.empty((B, K - 1, D), dtype=x.dtype, device=x.device)
    sb, st, _ = x.stride()
    check(lib().urnn_causal_conv(_ptr(x), sb, st, _ptr(weight), _ptr(bias), _ptr(state), _ptr(lengths), _ptr(out), _ptr(state_out), dt, B, L,
                                 D, K, 1 if silu else 0, stream), "urnn_causal_conv")
    return (out, state_out) if want_state else out


def causal_conv_step(x, state, weight, bias=None, silu=True, out=None, state_out=None):
    """``causal_conv`` for one token: x (B,D), state (B,K-1,D) -> (y (B,D), new state).  ``state_out`` may be ``state``: in place."""
    what = "causal_conv_step"
    dt = _seq_dtype(what, x)
    if x.dim() != 2:
        raise RuntimeError(f"{what}: x has shape {tuple(x.shape)}, expected (B, D)")
    if state is None:
        raise RuntimeError(f"{what}: state is None")
    B = x.shape[0]
    D, K = _conv_seq_check(what, x, weight, bias, state, (B,))
    if out is not None:
        _seq_out(what, "out", out, (B, D), x.dtype, (x, weight, bias, state, state_out))
    if state_out is not None:
        _seq_out(what, "state_out", state_out, (B, K - 1, D), x.dtype, (x, weight, bias, state), same=(state,))
    stream = _seq_device(what, x, weight, bias, state, out, state_out)
    if out is None:
        out = _empty_as(x)
    if state_out is None:
        state_out = torch.empty_like(state)
    check(lib().urnn_causal_conv_step(x.data_ptr(), x.stride(0), weight.data_ptr(), _ptr(bias), state.data_ptr(), out.data_ptr(), state_out.data_ptr(), dt, B, D, K,
                                      1 if silu else 0, stream), "urnn_causal_conv_step")
    return out, state_out


def _scan_check(what, u, delta, A, B, C, D, z, delta_bias, lead):
    """-> (channels, groups, states, B, C) with B and C as (..., groups, states)."""
    _no_empty(what, u)
    dim = u.shape[-1]
    if A.dim() != 2 or A.shape[0] != dim or not 1 <= A.shape[1] <= 64:
        raise RuntimeError(f"{what}: A has shape {tuple(A.shape)}, expected ({dim}, 1..64)")
    N = A.shape[1]
    dt, f32, shape = u.dtype, torch.float32, u.shape
    if B.dim() == len(lead) + 2 and shape == lead + (dim,) and delta.shape == shape and delta.dtype is dt and A.dtype is f32 and A.is_contiguous():
        G = B.shape[-2]                                  # the usual call, in one go; whatever it does not settle goes through the list below
        rows, par = lead + (G, N), (dim,)
        if (G >= 1 and dim % G == 0 and B.shape == rows and C.shape == rows and B.dtype is dt and C.dtype is dt
                and u.stride(-1) == delta.stride(-1) == B.stride(-1) == C.stride(-1) == 1
                and (G == 1 or B.stride(-2) == C.stride(-2) == N)
                and (z is None or (z.shape == shape and z.dtype is dt and z.stride(-1) == 1))
                and (D is None or (D.shape == par and D.dtype is f32 and D.is_contiguous()))
                and (delta_bias is None or (delta_bias.shape == par and delta_bias.dtype is f32 and delta_bias.is_contiguous()))):
            return dim, G, N, B, C
    _seq_check(what, "u", u, lead + (dim,), u.dtype)
    _seq_check(what, "delta", delta, lead + (dim,), u.dtype)
    if z is not None:
        _seq_check(what, "z", z, lead + (dim,), u.dtype)
    _seq_check(what, "A", A, (dim, N), torch.float32, contiguous=True)
    for name, t in (("D", D), ("delta_bias", delta_bias)):
        if t is not None:
            _seq_check(what, name, t, (dim,), torch.float32, contiguous=True)
    if B.dim() == len(lead) + 1:
        B = B.unsqueeze(-2)
    if C.dim() == len(lead) + 1:
        C = C.unsqueeze(-2)
    G = B.shape[-2] if B.dim() == len(lead) + 2 else 0
    if G < 1 or dim % G:
        raise RuntimeError(f"{what}: B has shape {tuple(B.shape)}; its groups must divide {dim} channels")
    for name, t in (("B", B), ("C", C)):
        _seq_check(what, name, t, lead + (G, N), u.dtype)
        if G > 1 and t.stride(-2) != N:
            raise RuntimeError(f"{what}: the groups of {name} must be adjacent (stride {t.stride(-2)}, {N} states)")
    return dim, G, N, B, C


def selective_scan_workspace(u, A):
    """The record that a training forward leaves for ``train_ops.selective_scan_backward``: a buffer for ``selective_scan(..., ws=)``."""
    if u.dim() != 3 or A.dim() != 2:
        raise RuntimeError(f"selective_scan_workspace: u {tuple(u.shape)} and A {tuple(A.shape)}, expected (batch, L, dim) and (dim, N)")
    B, L, dim = u.shape
    n = lib().urnn_selective_scan_workspace_bytes(B, L, dim, A.shape[1], 1)
    return torch.empty(int(n), dtype=torch.uint8, device=u.device)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=True, state=None, lengths=None, out=None, want_state=False,
                   state_out=None, ws=None):
    """Selective state space scan: step = softplus(delta + delta_bias), h_t = exp(step A) h_(t-1) + step u B_t,
    y = (C_t . h_t + D u) * silu(z).

    u, delta, z (batch,L,dim); A (dim,N), N = 1..64; B, C (batch,L,N) or (batch,L,G,N) with dim / G channels to a group; D, delta_bias
    (dim).  ``softplus`` False: step = delta + delta_bias.  ``state`` (batch,dim,N) float32: the state before the first token (None: zeros);
    ``lengths`` (batch) int32: tokens of each sequence of a padded batch -- later ones are not read and give zeros.  ``ws``: a buffer of
    ``selective_scan_workspace(u, A)`` that the backward will read: a training forward, with a buffer for every call whose backward is still
    to come (an Arena, which hands out the same one again, is refused); None: scratch for this call.
    Returns y, or (y, state after each sequence's last token) with ``want_state``."""
    what = "selective_scan"
    dt = _seq_dtype(what, u)
    if u.dim() != 3:
        raise RuntimeError(f"{what}: u has shape {tuple(u.shape)}, expected (batch, L, dim)")
    nb, L = u.shape[0], u.shape[1]
    dim, G, N, B, C = _scan_check(what, u, delta, A, B, C, D, z, delta_bias, (nb, L))
    if state is not None:
        _seq_check(what, "state", state, (nb, dim, N), torch.float32, contiguous=True)
    _lengths_check(what, lengths, nb)
    inputs = (u, delta, A, B, C, D, z, delta_bias, state, lengths)
    if out is not None:
        _seq_out(what, "out", out, (nb, L, dim), u.dtype, inputs + (state_out,))
    if state_out is not None:
        _seq_out(what, "state_out", state_out, (nb, dim, N), torch.float32, inputs)
    Lb = lib()
    keep = ws is not None
    nbytes = Lb.urnn_selective_scan_workspace_bytes(nb, L, dim, N, 1 if keep else 0)
    if keep:
        _seq_buffer(what, "ws", ws, nbytes, inputs + (out, state_out))
    stream = _seq_device(what, *inputs, out, state_out, ws)
    if nbytes and not keep:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=u.device)
    if out is None:
        out = _empty_as(u)
    if want_state and state_out is None:
        state_out = torch.empty((nb, dim, N), dtype=torch.float32, device=u.device)
    strides = (ctypes.c_long * 10)(*u.stride()[:2], *delta.stride()[:2], *B.stride()[:2], *C.stride()[:2], *(z.stride()[:2] if z is not None else (0, 0)))
    check(Lb.urnn_selective_scan(_ptr(u), _ptr(delta), _ptr(B), _ptr(C), _ptr(z), strides, _ptr(A), _ptr(D), _ptr(delta_bias), _ptr(state),
                                 _ptr(lengths), _ptr(out), _ptr(state_out), _ptr(ws), nbytes if not keep else ws.numel(), 1 if keep else 0, dt, nb, L,
                                 dim, G, N, 1 if softplus else 0, stream), "urnn_selective_scan")
    return (out, state_out) if want_state else out


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, softplus=True, out=None, state_out=None):
    """``selective_scan`` for one token: u, delta, z (batch,dim), B, C (batch,N) or (batch,G,N), state (batch,dim,N) float32 -> (y, new state).
    ``state_out`` may be ``state``: in place."""
    what = "selective_scan_step"
    dt = _seq_dtype(what, u)
    if u.dim() != 2:
        raise RuntimeError(f"{what}: u has shape {tuple(u.shape)}, expected (batch, dim)")
    if state is None:
        raise RuntimeError(f"{what}: state is None")
    nb = u.shape[0]
    dim, G, N, B, C = _scan_check(what, u, delta, A, B, C, D, z, delta_bias, (nb,))
    _seq_check(what, "state", state, (nb, dim, N), torch.float32, contiguous=True)
    inputs = (u, delta, A, B, C, D, z, delta_bias, state)
    if out is not None:
        _seq_out(what, "out", out, (nb, dim), u.dtype, inputs + (state_out,))
    if state_out is not None:
        _seq_out(what, "state_out", state_out, (nb, dim, N), torch.float32, inputs, same=(state,))
    stream = _seq_device(what, *inputs, out, state_out)
    if out is None:
        out = _empty_as(u)
    if state_out is None:
        state_out = torch.empty_like(state)
    strides = _Long5(u.stride(0), delta.stride(0), B.stride(0), C.stride(0), z.stride(0) if z is not None else 0)
    check(lib().urnn_selective_scan_step(u.data_ptr(), delta.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(z), strides, A.data_ptr(), _ptr(D), _ptr(delta_bias),
                                         state.data_ptr(), out.data_ptr(), state_out.data_ptr(), dt, nb, dim, G, N, 1 if softplus else 0, stream),
          "urnn_selective_scan_step")
    return out, state_out


def _rows(what, name, t, shape, dtype):
    """(..., D): strides of the rows, as (outer, inner) of a (B, L, D) tensor or (anything, row) of evenly spaced rows."""
    if len(shape) == 2:
        inner, channel = t.stride()[-2:] if t.shape == shape else (0, 0)
        if channel != 1 or t.dtype is not dtype:
            _seq_check(what, name, t, shape, dtype)
        return 0, inner if shape[0] > 1 else shape[1]
    _seq_check(what, name, t, shape, dtype)
    if len(shape) == 3:
        return t.stride()[:2]
    stride, n = None, 1
    for size, s in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride = s
        elif s != stride * n:
            raise RuntimeError(f"{what}: the rows of {name} are not evenly spaced (strides {t.stride()})")
        n *= size
    return 0, shape[-1] if stride is None else stride


def _norm_check(what, y, pre_w, residual, post_w, gate, scale, gate_act):
    _no_empty(what, y)
    D = y.shape[-1]
    if gate_act not in GATE_ACTS:
        raise RuntimeError(f"{what}: gate_act {gate_act!r} is none of {sorted(GATE_ACTS)}")
    if D > 16384:
        raise RuntimeError(f"{what}: {D} channels (at most 16384)")
    for name, t in (("pre_w", pre_w), ("post_w", post_w), ("scale", scale)):
        if t is not None and not (t.shape == (D,) and t.dtype is torch.float32 and t.is_contiguous()):
            _seq_check(what, name, t, (D,), torch.float32, contiguous=True)
    return _row_strides(what, y, (("y", y), ("gate", gate), ("residual", residual)))


def _row_strides(what, y, named):
    """[outer, inner] of every tensor, one after the other (zeros for None)."""
    shape, out = tuple(y.shape), []
    for name, t in named:
        out += _rows(what, name, t, shape, y.dtype) if t is not None else (0, 0)
    return out


def _inner_rows(shape, rows):
    return shape[1] if len(shape) == 3 else rows


def norm_residual(y, pre_w, residual=None, post_w=None, gate=None, scale=None, gate_act="silu", eps=NORM_EPS, out=None, residual_out=None):
    """The norms around a block in one pass over (..., D) rows: the norm after it (``post_w``) with its gate, the residual with its
    scale, and the norm before the next one (``pre_w``):

        r' = residual + scale * act(gate) * post_w * y / rms(y),    normed = pre_w * r' / rms(r'),    rms(x) = sqrt(mean(x^2) + eps).

    post_w None: y enters as it is; residual, gate or scale None: left out.  ``gate_act``: "silu", "sigmoid" or "none" (the gate itself).
    Parameters (D) float32.  Returns (normed, r'), both contiguous.  ``residual_out`` may be ``residual`` (in place)."""
    what = "norm_residual"
    dt = _seq_dtype(what, y)
    strides = _norm_check(what, y, pre_w, residual, post_w, gate, scale, gate_act)
    shape, rows_in, inputs = tuple(y.shape), (y, residual, gate), (y, residual, gate, pre_w, post_w, scale)
    if out is not None:
        _seq_out(what, "out", out, shape, y.dtype, inputs + (residual_out,), same=rows_in)
    if residual_out is not None:
        _seq_out(what, "residual_out", residual_out, shape, y.dtype, inputs, same=rows_in)
    stream = _seq_device(what, y, pre_w, residual, post_w, gate, scale, out, residual_out)
    if out is None:
        out = _empty_as(y)
    if residual_out is None:
        residual_out = _empty_as(y)
    D = shape[-1]
    rows = y.numel() // D
    check(lib().urnn_norm_residual(y.data_ptr(), _ptr(gate), _ptr(residual), _Long6(*strides), pre_w.data_ptr(), _ptr(post_w), _ptr(scale),
                                   out.data_ptr(), residual_out.data_ptr(), dt, rows, _inner_rows(shape, rows), D, GATE_ACTS[gate_act], float(eps), stream),
          "urnn_norm_residual")
    return out, residual_out

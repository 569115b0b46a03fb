"""Typed wrappers of the sequence-layer entry points of libslamhip.so: root-mean-square
norm, 8-bit operands and their product, short causal convolution, selective scan
(csrc/rms_norm.hip, gemm_fp8.hip, causal_conv.hip, selective_scan.hip).

As in encoder_ops the caller brings GPU tensors for inputs and outputs, every call is
checked on the host and launches on the current stream (of the tensors' device), and
there is no autograd: a backward pass is a call of its own.  A refused call raises
ValueError (what the tensors show) or RuntimeError (the library's limits of sizes and
combinations) and launches nothing.  Outputs share no memory with each other or with
inputs where a call does not say so.  Activations are float32 or bfloat16, parameters,
statistics and states float32.  Workspaces are torch allocations of the call.
"""
import struct

import torch

from .. import capi
from .encoder_ops import BF16, F32

FP8 = torch.float8_e4m3fn
_DTYPE = {F32: 0, BF16: 1}


# A call for single frames is bound by the host: the scan's takes 11 us, 8 of them for the checks below and 3 for the launch, its
# kernel 6.  So they spare objects and calls: torch.cuda.current_stream() alone would cost 2 us, an attribute of a tensor 0.05 us.
def _launch(device, name, *args):
    fn = getattr(capi.load(), name)
    stream = torch._C._cuda_getCurrentRawStream(device)
    if device != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    else:
        rc = fn(*args, stream)
    if rc:
        capi.check(rc, name)


def _bad(what, t, want):
    got = "None" if t is None else "%s %s on %s, strides %s" % (t.dtype, tuple(t.shape), t.device, t.stride())
    raise ValueError("%s: expected %s, got %s" % (what, want, got))


def _opt(t, dtype, shape, device, what):
    """The address of a contiguous tensor of this type and shape on GPU `device`, None without one."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        _bad(what, t, "a contiguous %s tensor %s on cuda:%d" % (dtype, shape, device))
    return t.data_ptr()


def _flat(t, dtype, shape, device, what):
    if t is None:
        _bad(what, t, "a contiguous %s tensor %s on cuda:%d" % (dtype, shape, device))
    return _opt(t, dtype, shape, device, what)


def _matrix(t, what):
    """(rows, columns, type code, device index) of a contiguous float32 or bfloat16 GPU matrix."""
    if t.dim() != 2 or t.dtype not in _DTYPE or not t.is_cuda or not t.is_contiguous() or t.shape[1] == 0:
        _bad(what, t, "a contiguous float32 or bfloat16 GPU matrix with columns")
    return *t.shape, _DTYPE[t.dtype], t.get_device()


def _sequence(t, what):
    """(B, T, C, type, device index) of a float32 or bfloat16 GPU tensor [B, T, C]."""
    if t.dim() != 3 or t.dtype not in _DTYPE or not t.is_cuda or t.shape[2] == 0:
        _bad(what, t, "a float32 or bfloat16 GPU tensor [B, T, C] with channels")
    return *t.shape, t.dtype, t.get_device()


def _sequences(dtype, device, inputs, outputs):
    """The addresses of sequences [B, T, C] of this type with unit stride over C, and their strides over B and T as an array of 64-bit
    integers.  inputs, outputs: (name, tensor, shape); None, where the shape is too, has no address.  An output's rows may not
    overlap, and no output begins where an input or another output does (steps of a sequence are worked on at once)."""
    ptrs, strides = [], []
    for what, t, shape in inputs + outputs:
        if t is None and shape is None:
            strides += (0, 0)
            ptrs.append(None)
            continue
        if t is None or t.dtype is not dtype or t.shape != shape or t.get_device() != device:
            _bad(what, t, "a %s tensor %s on cuda:%d" % (dtype, shape, device))
        sb, st, sc = t.stride()
        if sc != 1 and shape[2] > 1:
            _bad(what, t, "unit stride over the last axis")
        strides += (sb, st)
        ptrs.append(t.data_ptr())
    for i, (what, t, _) in enumerate(outputs, len(inputs)):
        if t is None:
            continue
        if not t.is_contiguous():
            (B, T, C), (sb, st, _) = t.shape, t.stride()
            if (T > 1 and st < C) or (B > 1 and sb < C) or (B > 1 and T > 1 and sb < (T - 1) * st + C and st < (B - 1) * sb + C):
                _bad(what, t, "rows that do not overlap")
        if ptrs[i] and ptrs[i] in ptrs[:i]:
            raise ValueError("%s is one of the inputs or another output" % what)
    return ptrs, _PACK[len(strides)](*strides)


_PACK = {n: struct.Struct("%dq" % n).pack for n in (4, 6, 12, 22)}


def _apart(ptr, ptrs, what):
    if ptr and ptr in ptrs:
        raise ValueError("%s is one of the sequences" % what)


def rms_norm_fwd(x, weight, eps, y=None, residual=None, sum_out=None, y8=None, scales=None, rstd=None):
    """s = x + residual (rounded to x's type, written to sum_out), y = s * (mean(s^2) + eps)^-1/2 * weight over the rows
    of x [rows, C], C <= 16384.  Any of y, sum_out and the pair y8 (e4m3) / scales (float32 [rows, ceil(C / 128)]) may be asked
    for; the 8-bit values are those of the unrounded y / scale, scale = max(max|y| / 448, 2^-100) of 128 values.  rstd
    (float32 [rows]) is kept for rms_norm_bwd.  y and sum_out may be x or residual itself."""
    rows, C, dt, dev = _matrix(x, "x")
    _launch(dev, "slamhip_rms_norm_fwd", x.data_ptr(), _opt(residual, x.dtype, (rows, C), dev, "residual"),
            _flat(weight, F32, (C,), dev, "weight"), eps, rows, C, dt, _opt(sum_out, x.dtype, (rows, C), dev, "sum_out"),
            _opt(y, x.dtype, (rows, C), dev, "y"), _opt(y8, FP8, (rows, C), dev, "y8"),
            _opt(scales, F32, (rows, (C + 127) // 128), dev, "scales"), _opt(rstd, F32, (rows,), dev, "rstd"))


def rms_norm_bwd(dy, sum_, weight, rstd, dx, dweight, d_sum=None):
    """Gradients of rms_norm_fwd: dx (of x and of residual alike) and dweight from dy, from sum_ (sum_out of the forward
    pass, or its x when it had no residual) and from d_sum, the gradient that arrives at sum_out.  dx may be dy or d_sum."""
    rows, C, dt, dev = _matrix(sum_, "sum")
    lib = capi.load()
    nbytes = lib.slamhip_rms_norm_bwd_workspace_bytes(rows, C)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(dev, "slamhip_rms_norm_bwd", _flat(dy, sum_.dtype, (rows, C), dev, "dy"), sum_.data_ptr(),
            _flat(weight, F32, (C,), dev, "weight"), _flat(rstd, F32, (rows,), dev, "rstd"),
            _opt(d_sum, sum_.dtype, (rows, C), dev, "d_sum"), rows, C, dt, _flat(dx, sum_.dtype, (rows, C), dev, "dx"),
            _flat(dweight, F32, (C,), dev, "dweight"), ws.data_ptr(), nbytes)


def quantize_fp8(x, q, scales):
    """x [rows, C] -> e4m3 q and a float32 scale for each 128 consecutive values of a row, scales [rows, ceil(C / 128)]."""
    rows, C, dt, dev = _matrix(x, "x")
    _launch(dev, "slamhip_quantize_fp8", x.data_ptr(), rows, C, dt, _flat(q, FP8, (rows, C), dev, "q"),
            _flat(scales, F32, (rows, (C + 127) // 128), dev, "scales"))


def quantize_fp8_blocks(x, q, scales):
    """quantize_fp8 with a scale for each 128 x 128 block: scales [ceil(R / 128), ceil(C / 128)] (the product's weights)."""
    R, C, dt, dev = _matrix(x, "x")
    _launch(dev, "slamhip_quantize_fp8_blocks", x.data_ptr(), R, C, dt, _flat(q, FP8, (R, C), dev, "q"),
            _flat(scales, F32, ((R + 127) // 128, (C + 127) // 128), dev, "scales"))


def gemm_nt_fp8(a8, a_scales, b8, b_scales, out):
    """out [M, N] (bfloat16) = a8 . b8^T of e4m3 operands a8 [M, K], b8 [N, K], where each 128 values of an a8 row have
    a scale, a_scales [M, ceil(K / 128)], and each 128 x 128 block of b8 one, b_scales [ceil(N / 128), ceil(K / 128)]: what
    quantize_fp8 (or rms_norm_fwd) and quantize_fp8_blocks write.  K a multiple of 16."""
    if out.dim() != 2 or not out.is_cuda or a8.dim() != 2 or a8.shape[1] == 0:
        _bad("out", out, "a bfloat16 GPU matrix and operands with columns")
    (M, N), K, dev = out.shape, a8.shape[1], out.get_device()
    kb = (K + 127) // 128
    if K % 16 or a8.data_ptr() % 16 or b8.data_ptr() % 16:
        raise ValueError("gemm_nt_fp8: K must be a multiple of 16 and the operands 16-byte aligned, got K = %d" % K)
    nbytes = capi.load().slamhip_gemm_nt_fp8_workspace_bytes(M, N, K)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _launch(dev, "slamhip_gemm_nt_fp8", _flat(a8, FP8, (M, K), dev, "a8"), _flat(a_scales, F32, (M, kb), dev, "a_scales"),
            _flat(b8, FP8, (N, K), dev, "b8"), _flat(b_scales, F32, ((N + 127) // 128, kb), dev, "b_scales"), M, N, K,
            _flat(out, BF16, (M, N), dev, "out"), capi.ptr(ws), nbytes)


def _taps(weight, C, device):
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= 4:
        _bad("weight", weight, "[%d, K] with 2 <= K <= 4" % C)
    return _flat(weight, F32, (C, weight.shape[1]), device, "weight"), weight.shape[1]


def causal_conv_fwd(x, weight, bias, y, state_in=None, state_out=None, lengths=None, silu=True):
    """Convolution over time of x [B, T, C] with one filter a channel, weight [C, K], 2 <= K <= 4:
    pre[t] = bias + sum_k weight[:, k] xp[t + k] with xp = state_in [B, K - 1, C] (None: zeros) followed by x, and
    y = pre * sigmoid(pre) (pre with silu=False).  state_out receives the last K - 1 rows of xp, to be state_in of the call that
    continues the sequences (one frame at a time: T = 1); it may be state_in itself.  lengths (int32 [B]) bounds each sequence:
    rows behind it are not used and are zero in y.  x and y may be views with any strides over B and T."""
    B, T, C, dt, dev = _sequence(x, "x")
    (xp, yp), strides = _sequences(dt, dev, (("x", x, (B, T, C)),), (("y", y, (B, T, C)),))
    w, K = _taps(weight, C, dev)
    sp, op = _opt(state_in, dt, (B, K - 1, C), dev, "state_in"), _opt(state_out, dt, (B, K - 1, C), dev, "state_out")
    _apart(sp, (yp,), "state_in")
    _apart(op, (xp, yp), "state_out")
    _launch(dev, "slamhip_causal_conv_fwd", xp, strides, w, _opt(bias, F32, (C,), dev, "bias"), sp,
            _opt(lengths, torch.int32, (B,), dev, "lengths"), B, T, C, K, int(silu), _DTYPE[dt], yp, op)


def causal_conv_bwd(dy, x, weight, bias, dx, dweight, dbias=None, state_in=None, d_state_in=None, d_state_out=None, lengths=None,
                    silu=True):
    """Gradients of causal_conv_fwd (same x, weight, bias, state_in, lengths, silu): dx, dweight, dbias and d_state_in from dy
    and from d_state_out, the gradient that arrives at state_out."""
    B, T, C, dt, dev = _sequence(x, "x")
    shape = (B, T, C)
    (yp, xp, dp), strides = _sequences(dt, dev, (("dy", dy, shape), ("x", x, shape)), (("dx", dx, shape),))
    w, K = _taps(weight, C, dev)
    ip, op = _opt(state_in, dt, (B, K - 1, C), dev, "state_in"), _opt(d_state_out, dt, (B, K - 1, C), dev, "d_state_out")
    gp = _opt(d_state_in, dt, (B, K - 1, C), dev, "d_state_in")
    _apart(dp, (ip, op), "dx")
    _apart(gp, (yp, xp, dp, ip, op), "d_state_in")
    nbytes = capi.load().slamhip_causal_conv_bwd_workspace_bytes(B, T, C, K)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(dev, "slamhip_causal_conv_bwd", yp, xp, strides, w, _opt(bias, F32, (C,), dev, "bias"), ip, op,
            _opt(lengths, torch.int32, (B,), dev, "lengths"), B, T, C, K, int(silu), _DTYPE[dt], dp,
            _flat(dweight, F32, (C, K), dev, "dweight"), _opt(dbias, F32, (C,), dev, "dbias"), gp, ws.data_ptr(), nbytes)


def selective_scan_kept_states(B, T, C, N, device):
    """The buffer in which selective_scan_fwd keeps states for selective_scan_bwd (every 16 steps, 8 for N > 8)."""
    return torch.empty(capi.load().slamhip_selective_scan_kept_floats(B, T, C, N), dtype=F32, device=device)


def _scan_inputs(u, delta, A, Bm, Cm, z):
    """The sizes, and the input sequences as _sequences() takes them."""
    B, T, C, dt, dev = _sequence(u, "u")
    if A.dim() != 2 or not 1 <= A.shape[1] <= 32:
        _bad("A", A, "[%d, N] with 1 <= N <= 32" % C)
    N = A.shape[1]
    shape, states = (B, T, C), (B, T, N)
    return B, T, C, N, dt, dev, (("u", u, shape), ("delta", delta, shape), ("z", z, None if z is None else shape), ("Bm", Bm, states),
                                 ("Cm", Cm, states))


def selective_scan_fwd(u, delta, A, Bm, Cm, y, D=None, z=None, delta_bias=None, softplus=True, state_in=None, state_out=None,
                       kept_states=None, lengths=None):
    """dt = softplus(delta + delta_bias), h_t = exp(dt A) h_{t-1} + dt u Bm, y = (Cm . h_t + D u) z / (1 + e^-z) over the steps of
    u, delta, z, y [B, T, C], A [C, N], Bm, Cm [B, T, N], N <= 32.  D and delta_bias [C] and the gate z are optional; softplus=False
    takes delta + delta_bias as it is.  state_in [B, C, N] (None: zeros) is h before the first step and state_out h after the last,
    to be state_in of the call that continues the sequences (one frame at a time: T = 1); it may be state_in itself.  lengths
    (int32 [B]) bounds each sequence: rows behind it are not used and are zero in y.  kept_states (selective_scan_kept_states)
    is what selective_scan_bwd needs.  Sequences may be views with any strides over B and T."""
    B, T, C, N, dt, dev, inputs = _scan_inputs(u, delta, A, Bm, Cm, z)
    (*ptrs, yp), strides = _sequences(dt, dev, inputs, (("y", y, (B, T, C)),))
    lib = capi.load()
    kp = ws = None
    if kept_states is not None:
        kp = _flat(kept_states, F32, (lib.slamhip_selective_scan_kept_floats(B, T, C, N),), dev, "kept_states")
    nbytes = lib.slamhip_selective_scan_fwd_workspace_bytes(B, T, C, N)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(dev, "slamhip_selective_scan_fwd", *ptrs, strides, _flat(A, F32, (C, N), dev, "A"),
            _opt(D, F32, (C,), dev, "D"), _opt(delta_bias, F32, (C,), dev, "delta_bias"), _opt(state_in, F32, (B, C, N), dev, "state_in"),
            _opt(lengths, torch.int32, (B,), dev, "lengths"), B, T, C, N, int(softplus), _DTYPE[dt], yp,
            _opt(state_out, F32, (B, C, N), dev, "state_out"), kp, capi.ptr(ws), nbytes)


def selective_scan_bwd(dy, u, delta, A, Bm, Cm, kept_states, du, ddelta, dA, dB, dC, D=None, z=None, delta_bias=None, softplus=True,
                       dD=None, dz=None, d_delta_bias=None, d_state_in=None, d_state_out=None, lengths=None):
    """Gradients of selective_scan_fwd at the same inputs, with the states that it kept, from dy and from d_state_out, the
    gradient that arrives at state_out: du, ddelta, dz (given when z is), dB, dC, dA, dD, d_delta_bias and d_state_in."""
    if (z is None) != (dz is None):
        raise ValueError("selective_scan_bwd: dz is wanted exactly when there is z")
    B, T, C, N, dt, dev, inputs = _scan_inputs(u, delta, A, Bm, Cm, z)
    shape, states = (B, T, C), (B, T, N)
    ptrs, strides = _sequences(dt, dev, (("dy", dy, shape),) + inputs, (
        ("du", du, shape), ("ddelta", ddelta, shape), ("dz", dz, None if dz is None else shape), ("dB", dB, states), ("dC", dC, states)))
    gp, op = _opt(d_state_in, F32, (B, C, N), dev, "d_state_in"), _opt(d_state_out, F32, (B, C, N), dev, "d_state_out")
    _apart(gp, ptrs + [op], "d_state_in")
    _apart(op, ptrs[6:], "d_state_out")
    lib = capi.load()
    kp = _flat(kept_states, F32, (lib.slamhip_selective_scan_kept_floats(B, T, C, N),), dev, "kept_states")
    nbytes = lib.slamhip_selective_scan_bwd_workspace_bytes(B, T, C, N)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(dev, "slamhip_selective_scan_bwd", *ptrs[:6], strides, _flat(A, F32, (C, N), dev, "A"), _opt(D, F32, (C,), dev, "D"),
            _opt(delta_bias, F32, (C,), dev, "delta_bias"), kp, op,
            _opt(lengths, torch.int32, (B,), dev, "lengths"), B, T, C, N, int(softplus), _DTYPE[dt], *ptrs[6:],
            _flat(dA, F32, (C, N), dev, "dA"), _opt(dD, F32, (C,), dev, "dD"), _opt(d_delta_bias, F32, (C,), dev, "d_delta_bias"),
            gp, ws.data_ptr(), nbytes)

"""The sequence-layer entry points of libslamhip.so on torch tensors: root-mean-square
norm, 8-bit operands and their product, short causal convolution, selective scan
(csrc/rms_norm.hip, gemm_fp8.hip, causal_conv.hip, selective_scan.hip).

As in encoder_ops the caller brings GPU tensors for inputs and outputs, every call is
checked on the host and launches on the current stream (of the tensors' device), and
there is no autograd: a backward pass is a call of its own.  The checks are native
(csrc/sequence_binding.cpp): in Python they would take longer than a single frame's kernel.  A refused call raises
ValueError (what the tensors show) or RuntimeError (the library's limits of sizes and
combinations) and launches nothing.  Outputs share no memory with each other or with
inputs where a call does not say so.  Activations are float32 or bfloat16, parameters,
statistics and states float32.  Workspaces are torch allocations of the call.  Limits:
sequences B <= 65535, T and C <= 2^20; norms of fewer than 2^24 rows; operands of the
product with (rows + 256) K < 2^31.  In a padded batch a sequence of length 0 may have anything in its
state: it passes through and takes no part in the parameters' gradients.
"""
import ctypes
import sys

import torch

from .. import capi
from .encoder_ops import BF16, F32  # noqa: F401  (the activations' types)

try:
    from .._lib import _sequence
except ImportError as e:
    raise RuntimeError("slam_amd: _lib/_sequence.so cannot be loaded (%s) - build it with `make -C slam_amd/csrc binding PYTHON=%s`; there is no fallback"
                       % (e, sys.executable))

FP8 = torch.float8_e4m3fn

_lib = capi.load()
_sequence.bind({name: ctypes.cast(getattr(_lib, name), ctypes.c_void_p).value for name in capi.SIGNATURES})


def rms_norm_fwd(x, weight, eps, y=None, residual=None, sum_out=None, y8=None, scales=None, rstd=None):
    """s = x + residual (rounded to x's type, written to sum_out), y = s * (mean(s^2) + eps)^-1/2 * weight over the rows
    of x [rows, C], C <= 16384.  Any of y, sum_out and the pair y8 (e4m3) / scales (float32 [rows, ceil(C / 128)]) may be asked
    for; the 8-bit values are those of the unrounded y / scale, scale = max(max|y| / 448, 2^-100) of 128 values.  rstd
    (float32 [rows]) is kept for rms_norm_bwd.  y and sum_out may be x or residual itself."""
    _sequence.rms_norm_fwd(x, weight, eps, y, residual, sum_out, y8, scales, rstd)


def rms_norm_bwd(dy, sum_, weight, rstd, dx, dweight, d_sum=None):
    """Gradients of rms_norm_fwd: dx (of x and of residual alike) and dweight from dy, from sum_ (sum_out of the forward
    pass, or its x when it had no residual) and from d_sum, the gradient that arrives at sum_out.  dx may be dy or d_sum."""
    _sequence.rms_norm_bwd(dy, sum_, weight, rstd, dx, dweight, d_sum)


def quantize_fp8(x, q, scales):
    """x [rows, C] -> e4m3 q and a float32 scale for each 128 consecutive values of a row, scales [rows, ceil(C / 128)]."""
    _sequence.quantize_fp8(x, q, scales)


def quantize_fp8_blocks(x, q, scales):
    """quantize_fp8 with a scale for each 128 x 128 block: scales [ceil(R / 128), ceil(C / 128)] (the product's weights)."""
    _sequence.quantize_fp8_blocks(x, q, scales)


def gemm_nt_fp8(a8, a_scales, b8, b_scales, out):
    """out [M, N] (bfloat16) = a8 . b8^T of e4m3 operands a8 [M, K], b8 [N, K], where each 128 values of an a8 row have
    a scale, a_scales [M, ceil(K / 128)], and each 128 x 128 block of b8 one, b_scales [ceil(N / 128), ceil(K / 128)]: what
    quantize_fp8 (or rms_norm_fwd) and quantize_fp8_blocks write.  K a multiple of 16, a8 and b8 16-byte aligned."""
    _sequence.gemm_nt_fp8(a8, a_scales, b8, b_scales, out)


def causal_conv_fwd(x, weight, bias, y, state_in=None, state_out=None, lengths=None, silu=True):
    """Convolution over time of x [B, T, C] with one filter a channel, weight [C, K], 2 <= K <= 4:
    pre[t] = bias + sum_k weight[:, k] xp[t + k] with xp = state_in [B, K - 1, C] (None: zeros) followed by x, and
    y = pre * sigmoid(pre) (pre with silu=False).  state_out receives the last K - 1 rows of xp, to be state_in of the call that
    continues the sequences (one frame at a time: T = 1); it may be state_in itself.  lengths (int32 [B], taken into [0, T]) bounds each
    sequence: rows behind it are not used and are zero in y.  x and y may be views with any strides over B and T."""
    _sequence.causal_conv_fwd(x, weight, bias, y, state_in, state_out, lengths, silu)


def causal_conv_bwd(dy, x, weight, bias, dx, dweight, dbias=None, state_in=None, d_state_in=None, d_state_out=None, lengths=None,
                    silu=True):
    """Gradients of causal_conv_fwd (same x, weight, bias, state_in, lengths, silu): dx, dweight, dbias and d_state_in from dy
    and from d_state_out, the gradient that arrives at state_out."""
    _sequence.causal_conv_bwd(dy, x, weight, bias, dx, dweight, dbias, state_in, d_state_in, d_state_out, lengths, silu)


def selective_scan_kept_states(B, T, C, N, device):
    """The buffer in which selective_scan_fwd keeps states for selective_scan_bwd (every 16 steps, 8 for N > 8)."""
    return torch.empty(_lib.slamhip_selective_scan_kept_floats(B, T, C, N), dtype=F32, device=device)


def selective_scan_fwd(u, delta, A, Bm, Cm, y, D=None, z=None, delta_bias=None, softplus=True, state_in=None, state_out=None,
                       kept_states=None, lengths=None):
    """dt = softplus(delta + delta_bias), h_t = exp(dt A) h_{t-1} + dt u Bm, y = (Cm . h_t + D u) z / (1 + e^-z) over the steps of
    u, delta, z, y [B, T, C], A [C, N], Bm, Cm [B, T, N], N <= 32.  D and delta_bias [C] and the gate z are optional; softplus=False
    takes delta + delta_bias as it is.  state_in [B, C, N] (None: zeros) is h before the first step and state_out h after the last,
    to be state_in of the call that continues the sequences (one frame at a time: T = 1); it may be state_in itself.  lengths
    (int32 [B], taken into [0, T]) bounds each sequence: rows behind it are not used and are zero in y.  kept_states (selective_scan_kept_states)
    is what selective_scan_bwd needs.  Sequences may be views with any strides over B and T.  States grow where A dt is
    positive (positive A; with softplus=False negative steps too): exp(A sum dt) over any stretch of a sequence has to be a float32."""
    _sequence.selective_scan_fwd(u, delta, A, Bm, Cm, y, D, z, delta_bias, softplus, state_in, state_out, kept_states, lengths)


def selective_scan_bwd(dy, u, delta, A, Bm, Cm, kept_states, du, ddelta, dA, dB, dC, D=None, z=None, delta_bias=None, softplus=True,
                       dD=None, dz=None, d_delta_bias=None, d_state_in=None, d_state_out=None, lengths=None):
    """Gradients of selective_scan_fwd at the same inputs, with the states that it kept, from dy and from d_state_out, the
    gradient that arrives at state_out: du, ddelta, dz (given when z is), dB, dC, dA, dD, d_delta_bias and d_state_in."""
    _sequence.selective_scan_bwd(dy, u, delta, A, Bm, Cm, kept_states, du, ddelta, dA, dB, dC, D, z, delta_bias, softplus, dD, dz,
                                  d_delta_bias, d_state_in, d_state_out, lengths)

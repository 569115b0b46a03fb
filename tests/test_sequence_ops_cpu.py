"""CPU checks of the sequence-layer operators: refused calls launch nothing, workspace sizes, and the float64 restatement that the
GPU tests compare with (its gradients against differences)."""
import ctypes

import pytest
import torch

from oracle import sequence_oracle as so
from slam_amd import capi
from slam_amd.network import sequence_ops as ops

P = ctypes.c_void_p(4096)     # an address that a refused call never reads
S = (ctypes.c_longlong * 22)()
E_ARG, E_SIZE = -1, -3
F32, BF16 = 0, 1


def refused(code, word, name, *args):
    lib = capi.load()
    assert getattr(lib, name)(*args) == code, name
    assert word.encode() in lib.slamhip_last_error(), lib.slamhip_last_error()


def test_rms_norm_refusals():
    f, b = "slamhip_rms_norm_fwd", "slamhip_rms_norm_bwd"
    refused(E_ARG, "known type", f, P, None, P, 1e-5, 1, 8, 2, None, P, None, None, None, None)
    refused(E_ARG, "rows", f, P, None, P, 1e-5, -1, 8, F32, None, P, None, None, None, None)
    refused(E_ARG, "C >= 1", f, P, None, P, 1e-5, 1, 0, F32, None, P, None, None, None, None)
    refused(E_SIZE, "16384", f, P, None, P, 1e-5, 1, 16385, F32, None, P, None, None, None, None)
    refused(E_SIZE, "rows", f, P, None, P, 1e-5, 1 << 24, 8, F32, None, P, None, None, None, None)
    refused(E_ARG, "null", f, None, None, P, 1e-5, 1, 8, F32, None, P, None, None, None, None)
    refused(E_ARG, "null", f, P, None, P, 1e-5, 1, 8, F32, None, None, None, None, None, None)
    refused(E_ARG, "scales", f, P, None, P, 1e-5, 1, 8, F32, None, None, P, None, None, None)
    refused(E_ARG, "residual", f, P, None, P, 1e-5, 1, 8, F32, P, P, None, None, None, None)
    refused(E_ARG, "null", b, P, P, P, None, None, 1, 8, F32, P, P, P, 1 << 20, None)
    refused(E_ARG, "workspace", b, P, P, P, P, None, 100, 8, F32, P, P, P, 16, None)
    lib = capi.load()
    assert lib.slamhip_rms_norm_fwd(None, None, None, 1e-5, 0, 8, F32, None, None, None, None, None, None) == 0
    assert lib.slamhip_rms_norm_bwd_workspace_bytes(0, 8) == 0


def test_quantize_and_product_refusals():
    refused(E_ARG, "known type", "slamhip_quantize_fp8", P, 1, 8, 7, P, P, None)
    refused(E_ARG, "null", "slamhip_quantize_fp8", P, 1, 8, F32, None, P, None)
    refused(E_SIZE, "blocks", "slamhip_quantize_fp8", P, 1 << 28, 128, F32, P, P, None)
    refused(E_SIZE, "rows", "slamhip_quantize_fp8_blocks", P, 65535 * 128 + 1, 128, F32, P, P, None)
    refused(E_ARG, "null", "slamhip_quantize_fp8_blocks", P, 1, 8, F32, P, None, None)
    g = "slamhip_gemm_nt_fp8"
    refused(E_ARG, "K >= 1", g, P, P, P, P, 1, 1, 0, P, None, 0, None)
    refused(E_SIZE, "multiple of 16", g, P, P, P, P, 1, 1, 24, P, None, 0, None)
    refused(E_SIZE, "2 GB", g, P, P, P, P, 1 << 20, 1, 4096, P, None, 0, None)
    refused(E_ARG, "null", g, P, None, P, P, 1, 1, 16, P, None, 0, None)
    refused(E_ARG, "aligned", g, ctypes.c_void_p(4104), P, P, P, 1, 1, 16, P, None, 0, None)
    need = capi.load().slamhip_gemm_nt_fp8_workspace_bytes(100, 64, 8192)      # two tiles: cut along k
    assert need > 0 and capi.load().slamhip_gemm_nt_fp8_workspace_bytes(8192, 8192, 4096) == 0
    refused(E_ARG, "workspace", g, P, P, P, P, 100, 64, 8192, P, P, need - 1, None)
    refused(E_ARG, "workspace", g, P, P, P, P, 100, 64, 8192, P, None, need, None)
    assert capi.load().slamhip_gemm_nt_fp8(None, None, None, None, 0, 8, 16, None, None, 0, None) == 0


def test_causal_conv_refusals():
    f, b = "slamhip_causal_conv_fwd", "slamhip_causal_conv_bwd"
    ok = [P, S, P, P, None, None, 1, 4, 8, 4, 1, F32, P, None, None]

    def changed(i, v):
        return ok[:i] + [v] + ok[i + 1:]
    for K in (1, 5):
        refused(E_ARG, "K <= 4", f, *changed(9, K))
    refused(E_ARG, "known type", f, *changed(11, 2))
    refused(E_ARG, "C >= 1", f, *changed(8, 0))
    refused(E_SIZE, "65535", f, *changed(6, 65536))
    refused(E_SIZE, "2^20", f, *changed(7, (1 << 20) + 1))
    for i in (0, 1, 2, 12):
        refused(E_ARG, "null", f, *changed(i, None))
    lib = capi.load()
    assert lib.slamhip_causal_conv_fwd(*changed(6, 0)) == 0
    need = lib.slamhip_causal_conv_bwd_workspace_bytes(1, 4, 8, 4)
    assert need >= 5 * 8 * 4
    refused(E_ARG, "workspace", b, P, P, S, P, P, None, None, None, 1, 4, 8, 4, 1, F32, P, P, P, None, P, need - 1, None)
    refused(E_ARG, "null", b, P, P, S, P, P, None, None, None, 1, 4, 8, 4, 1, F32, P, None, P, None, P, need, None)


def test_selective_scan_refusals():
    f, b = "slamhip_selective_scan_fwd", "slamhip_selective_scan_bwd"
    lib = capi.load()
    ok = [P, P, P, P, P, S, P, P, P, None, None, 1, 4, 8, 16, 1, F32, P, None, None, None, 0, None]

    def changed(i, v):
        return ok[:i] + [v] + ok[i + 1:]
    for N in (0, 33):
        refused(E_ARG, "N <= 32", f, *changed(14, N))
    refused(E_ARG, "known type", f, *changed(16, 5))
    refused(E_SIZE, "65535", f, *changed(11, 65536))
    for i in (0, 1, 3, 4, 5, 6, 17):
        refused(E_ARG, "null", f, *changed(i, None))
    need = lib.slamhip_selective_scan_fwd_workspace_bytes(1, 4096, 8, 16)     # few channels: cut into chunks
    assert need > 0 and lib.slamhip_selective_scan_fwd_workspace_bytes(64, 1, 4096, 16) == 0
    refused(E_ARG, "workspace", f, *changed(12, 4096)[:20], P, need - 1, None)
    bwd = [P, P, P, P, P, P, S, P, P, P, P, None, None, 1, 4, 8, 16, 1, F32, P, P, P, P, P, P, P, P, None, P, 1 << 30, None]

    def other(i, v):
        return bwd[:i] + [v] + bwd[i + 1:]
    refused(E_ARG, "dz", b, *other(3, None))
    refused(E_ARG, "null", b, *other(10, None))
    refused(E_ARG, "workspace", b, *other(29, 0))
    assert lib.slamhip_selective_scan_kept_floats(2, 33, 5, 8) == 2 * 3 * 5 * 8
    assert lib.slamhip_selective_scan_kept_floats(2, 33, 5, 32) == 2 * 5 * 5 * 32


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 16), torch.ones(16)
    with pytest.raises(ValueError, match="GPU matrix"):
        ops.rms_norm_fwd(x, w, 1e-5, y=x)
    with pytest.raises(ValueError, match="GPU matrix"):
        ops.quantize_fp8(x, x.to(ops.FP8), torch.ones(4, 1))
    with pytest.raises(ValueError, match="GPU matrix"):
        ops.gemm_nt_fp8(x.to(ops.FP8), torch.ones(4, 1), x.to(ops.FP8), torch.ones(1, 1), torch.zeros(4, 4))
    s = torch.zeros(2, 3, 16)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.causal_conv_fwd(s, torch.ones(16, 4), None, s)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.selective_scan_fwd(s, s, torch.ones(16, 4), torch.zeros(2, 3, 4), torch.zeros(2, 3, 4), s)


def test_restatement_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)  # noqa: E731
    lengths = [4, 0, 2]
    assert torch.autograd.gradcheck(lambda x, w, b, s: so.causal_conv(x, w, b, s, lengths), (r(3, 4, 2), r(2, 3), r(2), r(3, 2, 2)))
    A = (-torch.rand(2, 3, generator=g, dtype=torch.float64)).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda u, d, a, Bm, Cm, D, z, bias, s: so.selective_scan(u, d, a, Bm, Cm, D, z, bias, True, s, lengths),
                                    (r(3, 4, 2), r(3, 4, 2), A, r(3, 4, 3), r(3, 4, 3), r(2), r(3, 4, 2), r(2), r(3, 2, 3)))
    assert torch.autograd.gradcheck(lambda x, w: so.rms_norm(x, w, 1e-5)[1], (r(3, 5), r(5)))


def test_restatement_rounds_to_e4m3_like_torch():
    v = torch.cat((torch.linspace(-500, 500, 4001, dtype=torch.float64), torch.logspace(-5, 0, 2001, dtype=torch.float64)))
    want = v.float().clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(so.round_e4m3(v.float().double()), want)


def test_workspaces_of_empty_calls():
    """No sequences or no steps."""
    lib = capi.load()
    for B, T in ((0, 0), (0, 7), (3, 0)):
        assert lib.slamhip_selective_scan_kept_floats(B, T, 5, 16) == 0
        assert lib.slamhip_selective_scan_fwd_workspace_bytes(B, T, 5, 16) == 0
        # the state's gradient passes through and the parameters' are zero: a sum for each sequence
        assert lib.slamhip_selective_scan_bwd_workspace_bytes(B, T, 5, 16) == (0 if B == 0 else B * 5 * 18 * 4)


def test_the_binding_refuses_what_is_no_gpu_tensor():
    m, w = torch.zeros(2, 8), torch.zeros(8)
    s = torch.zeros(1, 3, 8)
    with pytest.raises(ValueError, match="x: expected .*GPU matrix.*got float"):
        ops.rms_norm_fwd(m, w, 1e-5, y=m)
    with pytest.raises(ValueError, match="x: expected a tensor, got list"):
        ops.rms_norm_fwd([1.0], w, 1e-5)
    with pytest.raises(ValueError, match="sum: expected .* got None"):
        ops.rms_norm_bwd(m, None, w, w, m, w)
    for call in (lambda: ops.quantize_fp8(m, m, m), lambda: ops.quantize_fp8_blocks(m, m, m), lambda: ops.gemm_nt_fp8(m, m, m, m, m),
                 lambda: ops.causal_conv_fwd(s, m, w, s), lambda: ops.causal_conv_bwd(s, s, m, w, s, m),
                 lambda: ops.selective_scan_fwd(s, s, m, s, s, s), lambda: ops.selective_scan_bwd(s, s, s, m, s, s, w, s, s, m, s, s)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError, match="takes 3 arguments"):
        ops._sequence.quantize_fp8(m)

"""Sizes beyond the sequence layer's limits: their calls are refused, so their workspaces are nothing (and no sum of sizes overflows on the way)."""
import ctypes

import pytest

from slam_amd import capi

MOST = 2 ** 31 - 1
P, S = ctypes.c_void_p(4096), (ctypes.c_longlong * 22)()
E_SIZE, F32 = -3, 0


@pytest.mark.parametrize("B,T,C", [(65536, 4096, 64), (1, (1 << 20) + 1, 8), (1, 64, (1 << 20) + 1), (1, 64, MOST), (1, MOST, 64), (MOST, 4, 4), (MOST, MOST, MOST)])
def test_sequences(B, T, C):
    lib = capi.load()
    for N in (1, 16, 32):
        assert lib.slamhip_selective_scan_kept_floats(B, T, C, N) == 0
        assert lib.slamhip_selective_scan_fwd_workspace_bytes(B, T, C, N) == 0
        assert lib.slamhip_selective_scan_bwd_workspace_bytes(B, T, C, N) == 0
    for K in (2, 4):
        assert lib.slamhip_causal_conv_bwd_workspace_bytes(B, T, C, K) == 0
    assert lib.slamhip_selective_scan_fwd(P, P, P, P, P, S, P, P, P, None, None, B, T, C, 16, 1, F32, P, None, None, None, 0, None) == E_SIZE
    assert lib.slamhip_selective_scan_bwd(P, P, P, P, P, P, S, P, P, P, P, None, None, B, T, C, 16, 1, F32, P, P, P, P, P, P, P, P, None, P, 0, None) == E_SIZE
    assert lib.slamhip_causal_conv_fwd(P, S, P, P, None, None, B, T, C, 4, 1, F32, P, None, None) == E_SIZE
    assert lib.slamhip_causal_conv_bwd(P, P, S, P, P, None, None, None, B, T, C, 4, 1, F32, P, P, P, None, P, 0, None) == E_SIZE


@pytest.mark.parametrize("rows,C", [(1 << 24, 8), (100, 16385), (MOST, MOST), (1 << 40, 64)])
def test_norm(rows, C):
    lib = capi.load()
    assert lib.slamhip_rms_norm_bwd_workspace_bytes(rows, C) == 0
    assert lib.slamhip_rms_norm_bwd(P, P, P, P, None, rows, C, F32, P, P, P, 0, None) == E_SIZE


@pytest.mark.parametrize("M,N,K", [(MOST, 64, 16), (16, MOST, 16), (100, 64, MOST // 16 * 16), (MOST, MOST, MOST // 16 * 16), (1, 1, 1 << 24)])
def test_product(M, N, K):
    lib = capi.load()
    assert lib.slamhip_gemm_nt_fp8_workspace_bytes(M, N, K) == 0
    assert lib.slamhip_gemm_nt_fp8(P, P, P, P, M, N, K, P, None, 0, None) == E_SIZE


def test_the_limits_themselves_have_workspaces():
    lib = capi.load()
    assert lib.slamhip_selective_scan_bwd_workspace_bytes(1, 1 << 20, 64, 4) > 0 and lib.slamhip_selective_scan_bwd_workspace_bytes(1, 64, 1 << 20, 4) > 0
    assert lib.slamhip_causal_conv_bwd_workspace_bytes(65535, 4, 8, 4) > 0
    assert lib.slamhip_rms_norm_bwd_workspace_bytes((1 << 24) - 1, 16384) > 0

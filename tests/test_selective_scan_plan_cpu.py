"""How the selective scan is cut: the number of chunks, read off the workspaces' sizes, is what the rule beside scan_shape() says."""
import pytest

from slam_amd import capi


def forward_chunks(B, T, C, N):
    floats = capi.load().slamhip_selective_scan_fwd_workspace_bytes(B, T, C, N) // 4
    if floats == 0:
        return 1
    n, rest = divmod(floats - B * C * N, B * C * (N + 1))      # states [B][chunks + 1][C][N], sums [B][chunks][C]
    assert rest == 0 and n > 1
    return n


def backward_chunks(B, T, C, N):
    P = 1 if N <= 4 else 2 if N <= 8 else 4 if N <= 16 else 8
    floats = capi.load().slamhip_selective_scan_bwd_workspace_bytes(B, T, C, N) // 4 - B * T * -(-C // 64) * 8 * P
    if floats == B * C * (N + 2):
        return 1
    n, rest = divmod(floats, B * C * (2 * N + 3))              # carries and sums of dt, parts of dA, dD and the bias's gradient
    assert rest == 0 and n > 1
    return n


def shortest(T):
    s = 16
    while s * s < T:
        s += 16
    return s


@pytest.mark.parametrize("T", [32, 33, 47, 100, 200, 256, 257, 333, 1000, 1024, 1030, 1454, 3000, 4000, 4096])
def test_few_channels_take_the_shortest_chunks(T):
    """One sequence of 64 channels: four waves, so that the shortest chunks are asked for at every length."""
    assert forward_chunks(1, T, 64, 16) == -(-T // shortest(T))
    assert backward_chunks(1, T, 64, 16) == -(-T // shortest(T))


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31])
def test_short_sequences_stay_whole(T):
    assert forward_chunks(1, T, 64, 16) == 1 and backward_chunks(1, T, 64, 16) == 1


def test_the_cuts_that_the_measurements_name():
    assert forward_chunks(1, 200, 512, 16) == 13 and backward_chunks(1, 200, 512, 16) == 13
    assert forward_chunks(5, 200, 1000, 8) == 13 and backward_chunks(5, 200, 1000, 8) == 7
    assert forward_chunks(4, 333, 1024, 16) == 11 and backward_chunks(4, 333, 1024, 16) == 7
    assert forward_chunks(8, 2048, 2048, 16) == 8 and backward_chunks(8, 2048, 2048, 16) == 8
    assert forward_chunks(1, 8192, 4096, 16) == 32
    assert forward_chunks(32, 130, 700, 4) == 1 and forward_chunks(8, 60, 4090, 4) == 1

"""The norm on tensors that are input and output at once, where its documentation allows it: the bits of the call with separate ones.  Rows of
every number of lanes, and rows whose last octet is loaded by another wave than the octet in front of it (C = 1025, 1541, 2049)."""
import pytest
import torch

from slam_amd.network import sequence_ops as ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
COLUMNS = [7, 100, 131, 200, 300, 513, 1000, 1025, 1541, 2049, 4096, 5001, 16383]


def operands(rows, C, dtype, n):
    g = torch.Generator(device="cuda").manual_seed(C)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return [new(rows, C).to(dtype) for _ in range(n)] + [new(C)]


@pytest.mark.parametrize("C", COLUMNS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [5, 700])
def test_forward_over_its_inputs(rows, C, dtype):
    x, r, w = operands(rows, C, dtype, 2)
    y, s, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device="cuda")
    ops.rms_norm_fwd(x, w, 1e-5, y=y, residual=r, sum_out=s, rstd=rstd)
    for y_over, s_over in ((0, 1), (1, 0), (0, None), (1, None), (None, 0), (None, 1)):
        ins = [x.clone(), r.clone()]
        got_y = torch.empty_like(x) if y_over is None else ins[y_over]
        got_s = torch.empty_like(x) if s_over is None else ins[s_over]
        got_r = torch.empty_like(rstd)
        ops.rms_norm_fwd(ins[0], w, 1e-5, y=got_y, residual=ins[1], sum_out=got_s, rstd=got_r)
        assert torch.equal(got_y, y) and torch.equal(got_s, s) and torch.equal(got_r, rstd), (y_over, s_over)
    ops.rms_norm_fwd(x, w, 1e-5, y=y)
    ops.rms_norm_fwd(x, w, 1e-5, y=x)
    assert torch.equal(x, y)


@pytest.mark.parametrize("C", COLUMNS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [2, 5, 700])
def test_backward_over_its_gradients(rows, C, dtype):
    s, dy, d_sum, w = operands(rows, C, dtype, 3)
    y, rstd = torch.empty_like(s), torch.empty(rows, device="cuda")
    ops.rms_norm_fwd(s, w, 1e-5, y=y, rstd=rstd)
    for with_sum in (False, True):
        want, want_w = torch.empty_like(s), torch.empty_like(w)
        ops.rms_norm_bwd(dy, s, w, rstd, want, want_w, d_sum=d_sum if with_sum else None)
        for over in ("dy", "d_sum") if with_sum else ("dy",):
            a, b, dw = dy.clone(), d_sum.clone(), torch.empty_like(w)
            dx = a if over == "dy" else b
            ops.rms_norm_bwd(a, s, w, rstd, dx, dw, d_sum=b if with_sum else None)
            assert torch.equal(dx, want) and torch.equal(dw, want_w), (over, with_sum)

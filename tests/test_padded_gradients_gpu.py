"""Padded batches: what a sequence does not use takes no part in the gradients of the parameters, also where it is no number.  A sequence of
length zero may have anything in its state (a slot that no stream uses), and rows behind a sequence's end meet its last rows in no product."""
import pytest
import torch

from oracle import sequence_oracle as so
from slam_amd.network import sequence_ops as ops
from test_sequence_ops_gpu import BF16, DEV, F32, NAN, close, rand, scan_case, scan_run, scan_want

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("T,C,K", [(9, 6, 4), (40, 130, 3), (70, 67, 2)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("silu", [True, False])
def test_convolution_with_an_unused_slot(T, C, K, dtype, silu):
    """Sequence 1 has no rows and NaN in its state and in the gradient that arrives there: the weights' gradients are those of the others."""
    g = torch.Generator().manual_seed(T)
    B, lengths = 3, torch.tensor([T, 0, T // 2], dtype=torch.int32)
    x, dy, st, dst = rand(g, B, T, C, dtype=dtype), rand(g, B, T, C, dtype=dtype), rand(g, B, K - 1, C, dtype=dtype), rand(g, B, K - 1, C, dtype=dtype)
    w, b = rand(g, C, K, scale=K ** -0.5), rand(g, C, scale=0.3)
    run = dict(x=x.clone(), dy=dy.clone(), st=st.clone(), dst=dst.clone())
    for i in range(B):
        run["x"][i, int(lengths[i]):] = NAN
        run["dy"][i, int(lengths[i]):] = NAN
    run["st"][1], run["dst"][1] = NAN, INF
    c = {k: v.to(DEV) for k, v in run.items()}
    e = torch.empty_like
    y, left, dx, dw, db, din = e(c["x"]), e(c["st"]), e(c["x"]), torch.empty(C, K, device=DEV), torch.empty(C, device=DEV), e(c["st"])
    n, wd, bd = lengths.to(DEV), w.to(DEV), b.to(DEV)
    ops.causal_conv_fwd(c["x"], wd, bd, y, state_in=c["st"], state_out=left, lengths=n, silu=silu)
    ops.causal_conv_bwd(c["dy"], c["x"], wd, bd, dx, dw, db, state_in=c["st"], d_state_in=din, d_state_out=c["dst"], lengths=n, silu=silu)
    wl, bl = w.double().requires_grad_(True), b.double().requires_grad_(True)
    keep = [0, 2]
    want, _ = so.causal_conv(x[keep].double(), wl, bl, st[keep].double(), lengths[keep], silu)
    (want * dy[keep].double()).sum().backward()
    bound = so.causal_conv_error(x[keep].double(), wl.detach(), bl.detach(), dy[keep].double(), st[keep].double(), None, lengths[keep], silu)
    close(dw, wl.grad, bound["dweight"], "dweight")
    close(db, bl.grad, bound["dbias"], "dbias")
    close(y[keep], want, bound["y"], "y")
    assert not bool(y[1].any()) and not bool(dx[1].any())
    assert bool(left[1].isnan().all()) and bool(din[1].isinf().all())       # the state and its gradient pass through


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("len0", [1, 2, 5, 9])
def test_convolution_of_an_infinite_last_row(dtype, len0):
    """The last row of a sequence is infinite: only the products that it is part of are, the same with rows of padding behind it as without."""
    K, C, T = 4, 5, 20
    g = torch.Generator().manual_seed(len0)
    x, dy, w = rand(g, 1, T, C, dtype=dtype).to(DEV), rand(g, 1, T, C, dtype=dtype).to(DEV), rand(g, C, K).to(DEV)
    x[0, len0 - 1, 2] = INF
    out = []
    for n in (len0, T):
        xs, dys = x[:, :n].contiguous(), dy[:, :n].contiguous()
        dx, dw = torch.empty_like(xs), torch.empty(C, K, device=DEV)
        ops.causal_conv_bwd(dys, xs, w, None, dx, dw, lengths=torch.tensor([len0], dtype=torch.int32, device=DEV), silu=False)
        out.append(dw)
    # the last tap alone meets the last row
    assert bool(out[0][2, K - 1].isinf()) and int(out[0].isfinite().sum()) == C * K - 1
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize("T,C,N", [(1, 5, 4), (20, 70, 3), (40, 9, 8), (150, 64, 16), (70, 30, 20)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_with_unused_slots(T, C, N, dtype):
    """Sequences 1 and 3 have no rows; one has NaN in its state, the other an infinity in its state and NaN in the gradient that arrives
    there: the gradients of all parameters and of the other sequences are those without them."""
    g = torch.Generator().manual_seed(T + C)
    B, keep = 4, [0, 2]
    t = scan_case(g, B, T, C, N, dtype, state=True)
    t["lengths"] = torch.tensor([T, 0, T // 2 + 1, 0], dtype=torch.int32)
    few = {k: v if v is None or k in ("A", "D", "delta_bias") else v[keep] for k, v in t.items()}
    want, bound = scan_want(few)
    for i in range(B):
        for name in ("u", "delta", "dy", "z", "Bm", "Cm"):
            t[name][i, int(t["lengths"][i]):] = NAN
    t["state_in"][1], t["state_in"][3], t["d_state_out"][3] = NAN, INF, NAN
    got = scan_run(t, dtype)
    for k, v in got.items():
        close(v if k in ("dA", "dD", "d_delta_bias") else v[keep], want[k], bound[k], k)
    for k in ("y", "du", "ddelta", "dz", "dB", "dC"):
        assert not bool(got[k][1].any()) and not bool(got[k][3].any()), k
    # states and their gradients pass through
    assert bool(got["state_out"][1].isnan().all()) and bool(got["state_out"][3].isinf().all()) and bool(got["d_state_in"][3].isnan().all())
    assert torch.equal(got["d_state_in"][1].cpu(), t["d_state_out"][1])

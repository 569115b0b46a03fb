"""Sequence-layer operators on the GPU against their float64 restatement (oracle/sequence_oracle.py).

Tolerances: half a step of the output's type relative to the value (torch.finfo(t).eps / 2), plus the float32 error bound that
the oracle states for the operator (units of 2^-24 of the magnitudes that pass through its sums)."""
import itertools

import numpy as np
import pytest
import torch

from oracle import sequence_oracle as so
from slam_amd.network import sequence_ops as ops

pytestmark = pytest.mark.gpu
BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
DEV = torch.device("cuda")
NAN = float("nan")


def close(got, want, bound, what):
    """bound: float64 like want, the float32 part in units of U; the output's own rounding comes on top."""
    got, half = got.detach().cpu(), torch.finfo(got.dtype).eps / 2
    want = want.detach()
    tol = want.abs() * half * (1 + 2.0 ** -10) + torch.as_tensor(bound, dtype=torch.float64) * so.U * 1.01 + 1e-37
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g where %.3g is allowed" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(tol[bad][off[bad].argmax()]))


def rand(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------------------ rms norm
NORM_SHAPES = [(1, 1), (3, 7), (5, 64), (2, 512), (7, 513), (4, 1000), (3, 2048), (2, 2049), (3, 4096), (2, 5001), (1, 8192), (2, 16384), (1500, 96),
               # lanes for narrow rows, and more rows than the backward pass has places for
               (40, 130), (701, 200), (5, 256), (9000, 24), (2100, 300), (1100, 1100), (600, 2100), (300, 9001)]


@pytest.mark.parametrize("rows,C", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_forward_and_gradients(rows, C, dtype, residual):
    g = torch.Generator().manual_seed(rows * 31 + C)
    x, dy, d_sum = rand(g, rows, C, dtype=dtype), rand(g, rows, C, dtype=dtype), rand(g, rows, C, dtype=dtype)
    r = rand(g, rows, C, dtype=dtype, scale=3.0) if residual else None
    w, eps = 1.0 + rand(g, C, scale=0.1), 1e-5
    new = lambda t: torch.full(t.shape, NAN, dtype=t.dtype, device=DEV)  # noqa: E731
    dx, dw, s, y, rstd = new(x), new(w), new(x), new(x), torch.full((rows,), NAN, device=DEV)
    c = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    ops.rms_norm_fwd(c(x), c(w), eps, y=y, residual=c(r), sum_out=s if residual else None, rstd=rstd)
    total = s if residual else c(x)
    ops.rms_norm_bwd(c(dy), total, c(w), rstd, dx, dw, d_sum=c(d_sum) if residual else None)

    xl, wl = x.double().requires_grad_(True), w.double().requires_grad_(True)
    want_s, want_y, want_r = so.rms_norm(xl, wl, eps, None if r is None else r.double(), dtype)
    if residual:
        assert torch.equal(s.cpu().double(), want_s.detach())
        (want_y * dy.double()).sum().add((want_s * d_sum.double()).sum()).backward()
    else:
        (want_y * dy.double()).sum().backward()
    # the mean of squares: a thread adds at most 64 of them, then 8 levels; root, quotient and two products
    n = 64 + 8 + 8
    close(rstd, want_r, n * want_r, "rstd")
    close(y, want_y, n * want_y.abs(), "y")
    hat = (want_s * want_r[:, None]).detach().abs()
    wdy = (wl.detach() * dy.double()).abs()
    dot = (wdy * hat).mean(1, keepdim=True)
    close(dx, xl.grad, want_r.detach()[:, None] * (3 * n * wdy + 6 * n * hat * dot) + (2 * d_sum.double().abs() if residual else 0), "dx")
    # columns: rows of a slot in sequence, then 32 chains of slots
    close(dw, wl.grad, ((dy.double().abs() * hat).sum(0)) * (n + rows / 1024 + 2 + 64), "dweight")


@pytest.mark.parametrize("rows,C", [(1, 1), (3, 130), (5, 257), (2, 513), (4, 4096), (3, 6000), (2, 16384)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rms_norm_8bit_output(rows, C, dtype):
    g = torch.Generator().manual_seed(C)
    x, r, w = rand(g, rows, C, dtype=dtype), rand(g, rows, C, dtype=dtype), rand(g, C)
    w[:min(C, 128)] = 0.0                      # a block of zeros has the smallest scale
    q = torch.zeros(rows, C, dtype=FP8, device=DEV)
    scales = torch.zeros(rows, -(-C // 128), device=DEV)
    s = torch.empty(rows, C, dtype=dtype, device=DEV)
    ops.rms_norm_fwd(x.to(DEV), w.to(DEV), 1e-5, residual=r.to(DEV), sum_out=s, y8=q, scales=scales)
    _, want, _ = so.rms_norm(x.double(), w.double(), 1e-5, r.double(), dtype)
    want_scales = so.row_scales(want)
    np.testing.assert_allclose(scales.cpu().double().numpy(), want_scales.numpy(), rtol=82 * so.U)
    sc = so.spread_scales(scales.cpu().double(), C)
    off = (q.cpu().double() * sc - want).abs()
    # half a step of 3 mantissa bits, or half the smallest subnormal (2^-9), and the norm's own error
    tol = torch.maximum(want.abs() * 2.0 ** -4, sc * 2.0 ** -10) + want.abs() * 90 * so.U
    assert bool((off <= tol).all()), float((off / tol).max())
    assert float(q.float().abs().max()) <= 448.0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rms_norm_in_place_and_special_rows(dtype):
    """A row of zeros has rstd eps^-1/2; a NaN and an infinity stay in their own rows; outputs may be the inputs."""
    rows, C = 4, 300
    g = torch.Generator().manual_seed(1)
    x, r, w = rand(g, rows, C, dtype=dtype), rand(g, rows, C, dtype=dtype), rand(g, C)
    x[0], r[0] = 0, 0
    x[1, 7] = NAN
    x[2, 9] = float("inf")
    a, b, rstd = x.to(DEV), r.to(DEV), torch.empty(rows, device=DEV)
    q, scales = torch.zeros(rows, C, dtype=FP8, device=DEV), torch.empty(rows, 3, device=DEV)
    ops.rms_norm_fwd(a, w.to(DEV), 1e-4, y=a, residual=b, sum_out=b, y8=q, scales=scales, rstd=rstd)
    assert torch.equal(a[0].float(), torch.zeros(C, device=DEV)) and abs(float(rstd[0]) - 100.0) < 1e-3
    assert torch.equal(q[0].float(), torch.zeros(C, device=DEV)) and float(scales[0, 0]) == 2.0 ** -100
    assert bool(a[1].isnan().all()) and bool(q[1].float().isnan().all()) and bool(scales[1].isnan().all())
    assert float(rstd[2]) == 0.0 and bool(a[2, 9].isnan()) and float(a[2, 8]) == 0.0
    s, y, _ = so.rms_norm(x[3:].double(), w.double(), 1e-4, r[3:].double(), dtype)
    close(a[3:], y, 80 * y.abs(), "y")
    assert torch.equal(b[3:].cpu().double(), s)


# ------------------------------------------------------------------------------------------------------ 8-bit operands
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 16), (3, 128), (17, 129), (5, 1000), (300, 4096)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_rows_equal_the_rule_exactly(rows, C, dtype):
    """Scales and values are IEEE quotients rounded to even: bit for bit what torch's elementary operations give."""
    g = torch.Generator().manual_seed(C)
    x = rand(g, rows, C, dtype=dtype) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g).float()).to(dtype)
    x[0, :128] = 0
    q, scales = torch.zeros(rows, C, dtype=FP8, device=DEV), torch.empty(rows, -(-C // 128), device=DEV)
    ops.quantize_fp8(x.to(DEV), q, scales)
    want_scales = so.row_scales(x.float())
    want = (x.float() / so.spread_scales(want_scales, C)).clamp(-448, 448).to(FP8)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(q.cpu().float(), want.float())


@pytest.mark.parametrize("R,C", [(1, 16), (128, 128), (130, 272), (257, 1000), (1024, 512)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_blocks_equal_the_rule_exactly(R, C, dtype):
    g = torch.Generator().manual_seed(R + C)
    x = rand(g, R, C, dtype=dtype)
    x[:128, :128] = 0
    q, scales = torch.zeros(R, C, dtype=FP8, device=DEV), torch.empty(-(-R // 128), -(-C // 128), device=DEV)
    ops.quantize_fp8_blocks(x.to(DEV), q, scales)
    nb, kb = scales.shape
    p = torch.nn.functional.pad(x.float(), (0, kb * 128 - C, 0, nb * 128 - R)).view(nb, 128, kb, 128)
    want_scales = (p.abs().amax((1, 3)) / 448.0).clamp_min(2.0 ** -100)
    want = (x.float() / so.spread_scales(want_scales.repeat_interleave(128, 0)[:R], C)).clamp(-448, 448).to(FP8)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(q.cpu().float(), want.float())


def test_quantize_values_around_halfway():
    """Values whose quotient is halfway between two of the format, and their neighbours, over the range of scales."""
    g = torch.Generator().manual_seed(3)
    rows = 2048
    scale = (1 + torch.randint(0, 4096, (rows, 1), generator=g) / 4096.0) * torch.exp2(torch.randint(-100, 110, (rows, 1), generator=g).float())
    half = (2 * torch.randint(8, 16, (rows, 128), generator=g) + 1) / 16.0 * torch.exp2(torch.randint(-6, 8, (rows, 128), generator=g).float())
    x = half * scale
    x = torch.where(torch.rand(x.shape, generator=g) < 0.5, x, torch.nextafter(x, torch.where(torch.rand(x.shape, generator=g) < 0.5, 0.0, 3e38)))
    x = x.minimum(447 * scale) * torch.where(torch.rand(x.shape, generator=g) < 0.5, -1.0, 1.0)
    x[:, :1] = 448 * scale
    q, scales = torch.zeros(rows, 128, dtype=FP8, device=DEV), torch.empty(rows, 1, device=DEV)
    ops.quantize_fp8(x.to(DEV), q, scales)
    assert torch.equal(scales.cpu(), scale)
    assert torch.equal(q.cpu().float(), (x / scale).to(FP8).float())


def test_quantize_special_values():
    """The largest value becomes 448; a NaN takes its block with it and no other; an infinity's block has an infinite scale."""
    x = torch.ones(4, 256, device=DEV)
    x[0, 3] = -57.0
    x[1, 5] = NAN
    x[2, 200] = float("inf")
    x[3] = 1e-38                                  # 1e-38 / 448 is below the smallest scale
    q, scales = torch.zeros(4, 256, dtype=FP8, device=DEV), torch.empty(4, 2, device=DEV)
    ops.quantize_fp8(x, q, scales)
    v = q.float()
    assert float(v[0, 3]) == -448.0 and float(v[0, 200]) == 448.0
    assert bool(v[1, :128].isnan().all()) and bool(scales[1, 0].isnan()) and float(v[1, 128]) == 448.0
    assert float(v[2, 0]) == 448.0 and bool(v[2, 200].isnan()) and float(v[2, 201]) == 0.0 and bool(scales[2, 1].isinf())
    assert float(scales[3, 0]) == 2.0 ** -100 and float(v[3].abs().max()) == 0.0


# ---------------------------------------------------------------------------------------------------------- the product
GEMM_SHAPES = [(1, 1, 16), (1, 16, 128), (3, 130, 272), (16, 64, 4096), (17, 48, 640), (33, 200, 144), (64, 16, 128), (65, 1, 16), (65, 129, 400),
               (128, 128, 128), (200, 300, 1040), (257, 513, 384), (300, 64, 2048), (777, 520, 1024),
               # one for each tile shape, with odd edges: 64 x 128, 128 x 128, 256 x 256; 3, 5 and 9 blocks of k; 128 x 128 in two groups
               (700, 1500, 384), (1500, 1400, 272), (2100, 2050, 640), (3500, 3400, 1152), (1500, 1400, 2192),
               # few tiles and much k: parts of k, of which the last is short
               (5, 40, 8336), (100, 70, 9232), (300, 200, 12304), (40, 478, 7328), (112, 1300, 2576)]


def gemm_bound(av, bv):
    """The matrix unit cuts each of eight consecutive products to 2^-13 of the largest one's power of two: at most seven of them
    lose up to 2^-13 of the largest.  The sums of eight, and the blocks, are added in float32: K / 8 additions and a multiply-add
    a block.  In units of U."""
    M, K = av.shape
    pad = -K % 8
    a, b = (torch.nn.functional.pad(t.abs(), (0, pad)).view(t.shape[0], -1, 8) for t in (av, bv))
    largest = torch.zeros(M, bv.shape[0], dtype=torch.float64)
    for i in range(a.shape[1]):
        largest += (a[:, None, i] * b[None, :, i]).amax(2)
    return 7 * 2.0 ** -13 / so.U * largest + (K / 8 + 16) * (av.abs() @ bv.abs().t())


@pytest.mark.parametrize("M,N,K", GEMM_SHAPES)
def test_gemm_nt_fp8(M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    a, b = rand(g, M, K), rand(g, N, K)
    b[:, : K // 2] *= 8.0                         # the blocks' scales differ
    kb, nb = -(-K // 128), -(-N // 128)
    a8, sa = torch.empty(M, K, dtype=FP8, device=DEV), torch.empty(M, kb, device=DEV)
    b8, sb = torch.empty(N, K, dtype=FP8, device=DEV), torch.empty(nb, kb, device=DEV)
    ops.quantize_fp8(a.to(DEV), a8, sa)
    ops.quantize_fp8_blocks(b.to(DEV), b8, sb)
    out = torch.full((M, N), NAN, dtype=BF16, device=DEV)
    ops.gemm_nt_fp8(a8, sa, b8, sb, out)
    av = a8.cpu().double() * so.spread_scales(sa.cpu().double(), K)
    bv = b8.cpu().double() * so.spread_scales(sb.cpu().double().repeat_interleave(128, 0)[:N], K)
    close(out, av @ bv.t(), gemm_bound(av, bv), "out")


def test_gemm_nt_fp8_special_values():
    """NaN and infinity reach exactly the rows and columns that they belong to."""
    M, N, K = 70, 140, 256
    g = torch.Generator().manual_seed(3)
    a8, b8 = rand(g, M, K).to(FP8).to(DEV), rand(g, N, K).to(FP8).to(DEV)
    sa, sb = torch.ones(M, 2, device=DEV), torch.ones(2, 2, device=DEV)
    a8.view(torch.uint8)[5, 200] = 0x7F
    sa[9, 0] = float("inf")
    out = torch.empty(M, N, dtype=BF16, device=DEV)
    ops.gemm_nt_fp8(a8, sa, b8, sb, out)
    assert bool(out[5].isnan().all()) and not bool(out[9].isfinite().any())
    keep = [i for i in range(M) if i not in (5, 9)]
    assert bool(out[keep].isfinite().all())
    # few rows take another kernel
    few = torch.empty(4, N, dtype=BF16, device=DEV)
    ops.gemm_nt_fp8(a8[:4], sa[:4], b8, sb, few)
    av, bv = a8[:4].cpu().double(), b8.cpu().double()
    close(few, av @ bv.t(), gemm_bound(av, bv), "few")
    close(out[:4], av @ bv.t(), gemm_bound(av, bv), "out")


# --------------------------------------------------------------------------------------------------------- convolution
def padded(g, B, T, C, dtype, kind, fill=NAN):
    """A sequence tensor on the GPU and its float64 values; kind 1: the middle of wider rows, kind 2: steps before sequences."""
    v = rand(g, B, T, C, dtype=dtype)
    if kind == 0:
        return v.to(DEV), v.double()
    if kind == 1:
        wide = torch.full((B, T, 2 * C + 3), fill, dtype=dtype, device=DEV)
        view = wide[:, :, 1:C + 1]
    else:
        view = torch.full((T, B, C), fill, dtype=dtype, device=DEV).transpose(0, 1)
    view.copy_(v)
    return view, v.double()


CONV_CASES = [(1, 1, 1, 2, 0), (2, 1, 8, 4, 0), (3, 2, 5, 3, 1), (1, 3, 64, 4, 0), (2, 17, 9, 4, 2), (4, 40, 33, 3, 1), (1, 200, 136, 4, 0), (3, 65, 512, 2, 2),
              (2, 131, 1000, 4, 1), (2, 70, 6, 3, 1), (2, 21, 1027, 4, 0), (3, 19, 270, 3, 1), (1, 9, 3, 4, 1)]


@pytest.mark.parametrize("B,T,C,K,kind", CONV_CASES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("state,ragged,silu", [(False, False, True), (True, True, True), (True, False, False), (False, True, False)])
def test_causal_conv_forward_and_gradients(B, T, C, K, kind, dtype, state, ragged, silu):
    g = torch.Generator().manual_seed(B * 1000 + T + C)
    x, xd = padded(g, B, T, C, dtype, kind)
    dy, dyd = padded(g, B, T, C, dtype, (kind + 1) % 3)
    w, b = rand(g, C, K, scale=K ** -0.5), rand(g, C, scale=0.3) if silu else None
    st, dst = (rand(g, B, K - 1, C, dtype=dtype), rand(g, B, K - 1, C, dtype=dtype)) if state else (None, None)
    lengths = torch.tensor([(0, T, 1, T // 2)[i % 4] for i in range(B)], dtype=torch.int32) if ragged else None
    if ragged:       # what lies behind a sequence is not used
        for i in range(B):
            x[i, int(lengths[i]):] = NAN
            dy[i, int(lengths[i]):] = NAN
    c = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    y, _ = padded(g, B, T, C, dtype, (kind + 2) % 3)
    dx, _ = padded(g, B, T, C, dtype, kind)
    new = lambda *s, dt=dtype: torch.full(s, NAN, dtype=dt, device=DEV)  # noqa: E731
    out_state, din = new(B, K - 1, C), new(B, K - 1, C)
    dw, db = new(C, K, dt=F32), new(C, dt=F32)
    ops.causal_conv_fwd(x, c(w), c(b), y, state_in=c(st), state_out=out_state, lengths=c(lengths), silu=silu)
    ops.causal_conv_bwd(dy, x, c(w), c(b), dx, dw, db, state_in=c(st), d_state_in=din, d_state_out=c(dst), lengths=c(lengths), silu=silu)

    leaf = lambda t: None if t is None else t.double().clone().requires_grad_(True)  # noqa: E731
    xl, wl, bl, sl = leaf(xd), leaf(w), leaf(b), leaf(st if state else torch.zeros(B, K - 1, C))
    want, want_state = so.causal_conv(xl, wl, bl, sl, lengths, silu)
    loss = (want * dyd).sum() + ((want_state * dst.double()).sum() if state else 0)
    loss.backward()
    zero = lambda l, ref: torch.zeros_like(ref) if l is None else l  # noqa: E731
    bound = so.causal_conv_error(xd, w.double(), None if b is None else b.double(), dyd, sl.detach(), None if dst is None else dst.double(),
                                 lengths, silu)
    close(y, want, bound["y"], "y")
    assert torch.equal(out_state.cpu().double(), want_state.detach())
    close(dx, zero(xl.grad, xd), bound["dx"], "dx")
    close(din, zero(sl.grad, sl), bound["d_state_in"], "d_state_in")
    close(dw, zero(wl.grad, wl), bound["dweight"], "dweight")
    if b is not None:
        close(db, zero(bl.grad, bl), bound["dbias"], "dbias")


@pytest.mark.parametrize("C", [72, 73, 75, 2])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_causal_conv_continues_sequences(dtype, C):
    """One call over all steps, and calls over pieces (one step at a time at the end) with the state kept in place."""
    B, T, K = 3, 37, 4
    g = torch.Generator().manual_seed(5)
    x, w, b = rand(g, B, T, C, dtype=dtype).to(DEV), rand(g, C, K).to(DEV), rand(g, C).to(DEV)
    whole = torch.empty_like(x)
    ops.causal_conv_fwd(x, w, b, whole)
    state = torch.zeros(B, K - 1, C, dtype=dtype, device=DEV)
    got = torch.empty_like(x)
    for t0, t1 in [(0, 20), (20, 22), (22, 33)] + [(t, t + 1) for t in range(33, T)]:
        ops.causal_conv_fwd(x[:, t0:t1], w, b, got[:, t0:t1], state_in=state, state_out=state)
    assert torch.equal(whole, got)
    assert torch.equal(state, x[:, -3:])


# ---------------------------------------------------------------------------------------------------------------- scan
def scan_case(g, B, T, C, N, dtype, kind=0, use_z=True, use_D=True, use_bias=True, softplus=True, state=True, ragged=False):
    t = {}
    for i, name in enumerate(("u", "delta", "dy", "z")):
        t[name], t[name + "_"] = padded(g, B, T, C, dtype, (kind + i) % 3)
    for i, name in enumerate(("Bm", "Cm")):
        t[name], t[name + "_"] = padded(g, B, T, N, dtype, (kind + i) % 3)
    if not softplus:
        t["delta"].copy_((t["delta_"].abs() * 0.1).to(dtype))
        t["delta_"] = (t["delta_"].abs() * 0.1).to(dtype).double()
    if not use_z:
        t["z"] = t["z_"] = None
    t["A"] = -torch.exp(rand(g, C, N, scale=0.7))
    t["D"] = rand(g, C) if use_D else None
    t["delta_bias"] = rand(g, C) - 2.0 if use_bias and softplus else None
    t["state_in"], t["d_state_out"] = (rand(g, B, C, N), rand(g, B, C, N)) if state else (None, None)
    t["lengths"] = torch.tensor([(T, 0, 1, T // 2)[i % 4] for i in range(B)], dtype=torch.int32) if ragged else None
    if ragged:
        for i in range(B):
            for name in ("u", "delta", "dy", "z", "Bm", "Cm"):
                if t[name] is not None:
                    t[name][i, int(t["lengths"][i]):] = NAN
    return t


def scan_run(t, dtype, softplus=True):
    B, T, C = t["u"].shape
    N = t["A"].shape[1]
    c = lambda k: None if t[k] is None else t[k].to(DEV)  # noqa: E731
    new = lambda *s, dt=dtype: torch.full(s, NAN, dtype=dt, device=DEV)  # noqa: E731
    out = dict(y=new(B, T, C), state_out=new(B, C, N, dt=F32))
    kept = ops.selective_scan_kept_states(B, T, C, N, DEV)
    ops.selective_scan_fwd(t["u"], t["delta"], c("A"), t["Bm"], t["Cm"], out["y"], D=c("D"), z=t["z"], delta_bias=c("delta_bias"),
                           softplus=softplus, state_in=c("state_in"), state_out=out["state_out"], kept_states=kept, lengths=c("lengths"))
    out |= dict(du=new(B, T, C), ddelta=new(B, T, C), dB=new(B, T, N), dC=new(B, T, N), dA=new(C, N, dt=F32), dD=new(C, dt=F32),
                d_delta_bias=new(C, dt=F32), d_state_in=new(B, C, N, dt=F32))
    if t["z"] is not None:
        out["dz"] = new(B, T, C)
    ops.selective_scan_bwd(t["dy"], t["u"], t["delta"], c("A"), t["Bm"], t["Cm"], kept, out["du"], out["ddelta"], out["dA"], out["dB"],
                           out["dC"], D=c("D"), z=t["z"], delta_bias=c("delta_bias"), softplus=softplus, dD=out["dD"], dz=out.get("dz"),
                           d_delta_bias=out["d_delta_bias"], d_state_in=out["d_state_in"], d_state_out=c("d_state_out"),
                           lengths=c("lengths"))
    return out


def scan_want(t, softplus=True):
    leaf = lambda v: None if v is None else v.double().clone().requires_grad_(True)  # noqa: E731
    v = {k: leaf(t[k + "_"]) for k in ("u", "delta", "z", "Bm", "Cm")}
    v |= {k: leaf(t[k]) for k in ("A", "D", "delta_bias")}
    B, T, C = t["u"].shape
    v["state_in"] = leaf(t["state_in"] if t["state_in"] is not None else torch.zeros(B, C, t["A"].shape[1]))
    y, state = so.selective_scan(v["u"], v["delta"], v["A"], v["Bm"], v["Cm"], v["D"], v["z"], v["delta_bias"], softplus, v["state_in"],
                                 t["lengths"])
    loss = (y * t["dy_"]).sum()
    if t["d_state_out"] is not None:
        loss = loss + (state * t["d_state_out"].double()).sum()
    if loss.requires_grad:
        loss.backward()
    grad = lambda k: None if v[k] is None else (torch.zeros_like(v[k]) if v[k].grad is None else v[k].grad)  # noqa: E731
    want = dict(y=y, state_out=state, du=grad("u"), ddelta=grad("delta"), dz=grad("z"), dB=grad("Bm"), dC=grad("Cm"), dA=grad("A"),
                dD=grad("D"), d_delta_bias=grad("delta_bias"), d_state_in=grad("state_in"))
    d = lambda k: None if v[k] is None else v[k].detach()  # noqa: E731
    bound = so.selective_scan_error(d("u"), d("delta"), d("A"), d("Bm"), d("Cm"), t["dy_"], d("D"), d("z"), d("delta_bias"), softplus,
                                    d("state_in"), None if t["d_state_out"] is None else t["d_state_out"].double(), t["lengths"])
    return want, bound


SCAN_CASES = [(1, 1, 1, 1, 0), (2, 1, 16, 16, 0), (3, 2, 5, 4, 1), (1, 15, 17, 3, 2), (2, 16, 64, 8, 0), (4, 17, 65, 5, 1), (2, 33, 40, 16, 2),
              (1, 130, 70, 16, 0), (4, 150, 20, 32, 1), (2, 200, 130, 17, 0), (1, 260, 8, 12, 2)]


@pytest.mark.parametrize("B,T,C,N,kind", SCAN_CASES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("state,ragged", [(False, False), (True, True)])
def test_selective_scan_forward_and_gradients(B, T, C, N, kind, dtype, state, ragged):
    g = torch.Generator().manual_seed(B * 1000 + T + C + N)
    t = scan_case(g, B, T, C, N, dtype, kind, state=state, ragged=ragged)
    got = scan_run(t, dtype)
    want, bound = scan_want(t)
    for k, v in got.items():
        close(v, want[k], bound[k], k)


@pytest.mark.parametrize("use_z,use_D,use_bias,softplus", [o for o in itertools.product((False, True), repeat=4) if not all(o)])
def test_selective_scan_options(use_z, use_D, use_bias, softplus):
    g = torch.Generator().manual_seed(11)
    t = scan_case(g, 2, 140, 24, 16, F32, 1, use_z, use_D, use_bias, softplus, state=True, ragged=True)
    got = scan_run(t, F32, softplus)
    want, bound = scan_want(t, softplus)
    for k, v in got.items():
        if k == "dD" and not use_D:
            continue                     # without D its gradient is that of D = 0
        if k == "d_delta_bias" and t["delta_bias"] is None:
            want[k] = want["ddelta"].sum((0, 1))
        close(v, want[k], bound[k], k)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_selective_scan_continues_sequences(dtype):
    """Pieces of a sequence with the state kept in place (cut into chunks or not, then one step at a time) against the whole."""
    B, T, C, N = 2, 300, 24, 16
    g = torch.Generator().manual_seed(5)
    t = scan_case(g, B, T, C, N, dtype, state=False)
    c = lambda k: t[k].to(DEV)  # noqa: E731
    state, got = torch.zeros(B, C, N, device=DEV), torch.full((B, T, C), NAN, dtype=dtype, device=DEV)
    for t0, t1 in [(0, 200), (200, 291), (291, 293)] + [(i, i + 1) for i in range(293, T)]:
        cutout = lambda k: t[k][:, t0:t1]  # noqa: E731
        ops.selective_scan_fwd(cutout("u"), cutout("delta"), c("A"), cutout("Bm"), cutout("Cm"), got[:, t0:t1], D=c("D"), z=cutout("z"),
                               delta_bias=c("delta_bias"), state_in=state, state_out=state)
    want, bound = scan_want(t)
    close(got, want["y"], bound["y"], "y")
    close(state, want["state_out"], bound["state_out"], "state_out")


def test_selective_scan_far_steps_and_decays():
    """Time steps of 1e-4 keep their relative precision, decays of e^-400 vanish, growing states stay finite where they are."""
    B, T, C, N = 1, 20, 16, 4
    g = torch.Generator().manual_seed(9)
    t = scan_case(g, B, T, C, N, F32, state=True)
    t["delta_bias"] = torch.linspace(-9.0, 6.0, C)
    t["A"] = -torch.logspace(-2, 2, N).repeat(C, 1)
    t["A"][:, 0] = 0.01
    got = scan_run(t, F32)
    want, bound = scan_want(t)
    for k, v in got.items():
        close(v, want[k], bound[k], k)


@pytest.mark.parametrize("T", [0, 5])
def test_empty_sequences(T):
    B, C, N, K = 2, 8, 4, 3
    z = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    g = torch.Generator().manual_seed(2)
    state = rand(g, B, C, N).to(DEV)
    out = torch.full_like(state, NAN)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    y = torch.full((B, T, C), NAN, device=DEV)
    ops.selective_scan_fwd(z(B, T, C), z(B, T, C), -torch.ones(C, N, device=DEV), z(B, T, N), z(B, T, N), y, state_in=state, state_out=out,
                           lengths=lengths)
    assert torch.equal(out, state) and not bool(y.any())
    rows = rand(g, B, K - 1, C).to(DEV)
    left = torch.full_like(rows, NAN)
    ops.causal_conv_fwd(z(B, T, C), torch.ones(C, K, device=DEV), None, y, state_in=rows, state_out=left, lengths=lengths)
    assert torch.equal(left, rows)
    dw, din = torch.full((C, K), NAN, device=DEV), torch.full_like(rows, NAN)
    ops.causal_conv_bwd(z(B, T, C), z(B, T, C), torch.ones(C, K, device=DEV), None, y, dw, state_in=rows, d_state_in=din, d_state_out=left,
                        lengths=lengths)
    assert torch.equal(din, left) and not bool(dw.any())
    # the scan back: the gradient of the state passes through, nothing else gets any
    kept = ops.selective_scan_kept_states(B, T, C, N, DEV)
    ops.selective_scan_fwd(z(B, T, C), z(B, T, C), -torch.ones(C, N, device=DEV), z(B, T, N), z(B, T, N), y, kept_states=kept, lengths=lengths)
    full = lambda *s: torch.full(s, NAN, device=DEV)  # noqa: E731
    du, dd, dB, dC, dA, dstate = full(B, T, C), full(B, T, C), full(B, T, N), full(B, T, N), full(C, N), full(B, C, N)
    ops.selective_scan_bwd(full(B, T, C), full(B, T, C), full(B, T, C), -torch.ones(C, N, device=DEV), full(B, T, N), full(B, T, N), kept,
                           du, dd, dA, dB, dC, d_state_in=dstate, d_state_out=state, lengths=lengths)
    assert torch.equal(dstate, state) and not any(bool(t.any()) for t in (du, dd, dB, dC, dA))
    # no sequences, no rows
    e = torch.empty(0, 3, C, device=DEV)
    ops.causal_conv_fwd(e, torch.ones(C, K, device=DEV), None, torch.empty_like(e))
    ops.causal_conv_bwd(e, e, torch.ones(C, K, device=DEV), None, torch.empty_like(e), dw)
    assert not bool(dw.any())
    none, bc = torch.empty(0, 3, C, device=DEV), torch.empty(0, 3, N, device=DEV)
    kept, dA = ops.selective_scan_kept_states(0, 3, C, N, DEV), full(C, N)
    ops.selective_scan_fwd(none, none, -torch.ones(C, N, device=DEV), bc, bc, none, kept_states=kept)
    ops.selective_scan_bwd(none, none, none, -torch.ones(C, N, device=DEV), bc, bc, kept, none, none, dA, bc, bc)
    assert not bool(dA.any())
    m = torch.empty(0, C, device=DEV)
    dweight = torch.full((C,), NAN, device=DEV)
    ops.rms_norm_fwd(m, torch.ones(C, device=DEV), 1e-5, y=torch.empty_like(m))
    ops.rms_norm_bwd(m, m, torch.ones(C, device=DEV), torch.empty(0, device=DEV), torch.empty_like(m), dweight)
    assert not bool(dweight.any())


# --------------------------------------------------------------------------------------------------- one step at a time
@pytest.mark.parametrize("B,C,N", [(1, 1, 1), (3, 5, 3), (2, 64, 8), (5, 70, 16), (2, 130, 20), (33, 16, 32)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("use_z,use_D,use_bias,softplus,ragged", [(True, True, True, True, False), (False, False, False, True, True), (True, False, True, False, False)])
def test_selective_scan_one_step(B, C, N, dtype, use_z, use_D, use_bias, softplus, ragged):
    g = torch.Generator().manual_seed(B + C + N)
    t = scan_case(g, B, 1, C, N, dtype, 1, use_z, use_D, use_bias, softplus, state=True, ragged=ragged)
    c = lambda k: None if t[k] is None else t[k].to(DEV)  # noqa: E731
    y, state = torch.full((B, 1, C), NAN, dtype=dtype, device=DEV), c("state_in")
    ops.selective_scan_fwd(t["u"], t["delta"], c("A"), t["Bm"], t["Cm"], y, D=c("D"), z=t["z"], delta_bias=c("delta_bias"), softplus=softplus,
                           state_in=state, state_out=state, lengths=c("lengths"))
    want, bound = scan_want(t, softplus)
    close(y, want["y"], bound["y"], "y")
    close(state, want["state_out"], bound["state_out"], "state_out")


# ----------------------------------------------------------------------------------------- the layer that they are part of
def layer_parameters(g, width, inner, N, K=4):
    p = dict(norm=1.0 + rand(g, width, scale=0.1), w_in=rand(g, 2 * inner, width, scale=width ** -0.5), w_out=rand(g, width, inner, scale=inner ** -0.5),
             conv=rand(g, inner, K, scale=K ** -0.5), conv_bias=rand(g, inner, scale=0.1), A=-torch.exp(rand(g, inner, N, scale=0.5)),
             D=rand(g, inner), delta_bias=rand(g, inner) - 3.0, w_b=rand(g, N, inner, scale=inner ** -0.5), w_c=rand(g, N, inner, scale=inner ** -0.5),
             w_d=rand(g, inner, inner, scale=0.3 * inner ** -0.5))
    return p


def layer_training(p, x, dy, use_ops):
    """Forward and backward of a float32 sequence layer (norm, projection, convolution, scan with its gate, projection) with the
    residual added behind it.  The projections are torch products; use_ops False: all in float64 through autograd."""
    B, T, width = x.shape
    inner, N = p["A"].shape
    if not use_ops:
        q = {k: v.double().requires_grad_(True) for k, v in p.items()}
        xl = x.double().requires_grad_(True)
        _, y, _ = so.rms_norm(xl.reshape(-1, width), q["norm"], 1e-5)
        h = (y @ q["w_in"].t()).reshape(B, T, 2 * inner)
        u, _ = so.causal_conv(h[..., :inner], q["conv"], q["conv_bias"])
        s, _ = so.selective_scan(u, u @ q["w_d"].t(), q["A"], u @ q["w_b"].t(), u @ q["w_c"].t(), q["D"], h[..., inner:], q["delta_bias"])
        out = xl + s @ q["w_out"].t()
        (out * dy.double()).sum().backward()
        return out.detach(), xl.grad, {k: v.grad for k, v in q.items()}
    q = {k: v.to(DEV) for k, v in p.items()}
    xg, dyg = x.to(DEV), dy.to(DEV)
    new = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    flat = xg.reshape(-1, width)
    y, rstd = new(B * T, width), new(B * T)
    ops.rms_norm_fwd(flat, q["norm"], 1e-5, y=y, rstd=rstd)
    h = (y @ q["w_in"].t()).reshape(B, T, 2 * inner)
    cx, z = h[..., :inner], h[..., inner:]
    u, s = new(B, T, inner), new(B, T, inner)
    ops.causal_conv_fwd(cx, q["conv"], q["conv_bias"], u)
    delta, Bm, Cm = u @ q["w_d"].t(), u @ q["w_b"].t(), u @ q["w_c"].t()
    kept = ops.selective_scan_kept_states(B, T, inner, N, DEV)
    ops.selective_scan_fwd(u, delta, q["A"], Bm, Cm, s, D=q["D"], z=z, delta_bias=q["delta_bias"], kept_states=kept)
    out = xg + s @ q["w_out"].t()
    g = {}
    ds = dyg @ q["w_out"]
    g["w_out"] = dyg.reshape(-1, width).t() @ s.reshape(-1, inner)
    dh = new(B, T, 2 * inner)                      # the gradients of both halves side by side, as the halves are
    du, dd, dB, dC = new(B, T, inner), new(B, T, inner), new(B, T, N), new(B, T, N)
    for k in ("A", "D", "delta_bias", "conv", "conv_bias", "norm"):
        g[k] = torch.empty_like(q[k])
    ops.selective_scan_bwd(ds, u, delta, q["A"], Bm, Cm, kept, du, dd, g["A"], dB, dC, D=q["D"], z=z, delta_bias=q["delta_bias"], dD=g["D"],
                           dz=dh[..., inner:], d_delta_bias=g["delta_bias"])
    rows = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    g["w_d"], g["w_b"], g["w_c"] = rows(dd).t() @ rows(u), rows(dB).t() @ rows(u), rows(dC).t() @ rows(u)
    du += dd @ q["w_d"] + dB @ q["w_b"] + dC @ q["w_c"]
    ops.causal_conv_bwd(du, cx, q["conv"], q["conv_bias"], dh[..., :inner], g["conv"], g["conv_bias"])
    g["w_in"] = rows(dh).t() @ y
    dx = new(B * T, width)
    ops.rms_norm_bwd(rows(dh) @ q["w_in"], flat, q["norm"], rstd, dx, g["norm"])
    return out, dyg + dx.reshape(B, T, width), g


def test_a_layer_trains():
    """All operators in the order of a training step.  Every gradient within 1e-4 of its largest value: a chain of about ten float32
    sums of up to 512 terms (512 x 2^-24 = 3e-5 each at worst, their usual error a thirtieth of that)."""
    g = torch.Generator().manual_seed(8)
    B, T, width, inner, N = 2, 150, 48, 96, 16
    p = layer_parameters(g, width, inner, N)
    x, dy = rand(g, B, T, width), rand(g, B, T, width)
    want, want_dx, want_g = layer_training(p, x, dy, False)
    out, dx, grads = layer_training(p, x, dy, True)
    for name, a, b in [("out", out, want), ("dx", dx, want_dx)] + [(k, grads[k], want_g[k]) for k in want_g]:
        off = float((a.cpu().double() - b).abs().max() / b.abs().max())
        assert off < 1e-4, (name, off)


def serve(p, q, x, state):
    """A frame of each stream through the layer with 8-bit projections; state: convolution's and scan's, kept in place."""
    B, width = x.shape
    inner, N = p["A"].shape
    new = lambda *s, dt=BF16: torch.empty(*s, dtype=dt, device=DEV)  # noqa: E731
    a8, sa = new(B, width, dt=FP8), new(B, -(-width // 128), dt=F32)
    ops.rms_norm_fwd(x, p["norm"], 1e-5, y8=a8, scales=sa)
    h = new(B, 2 * inner)
    ops.gemm_nt_fp8(a8, sa, *q["w_in"], h)
    h = h.reshape(B, 1, 2 * inner)
    u, s = new(B, 1, inner), new(B, 1, inner)
    ops.causal_conv_fwd(h[..., :inner], p["conv"], p["conv_bias"], u, state_in=state[0], state_out=state[0])
    u8, su, dbc = new(B, inner, dt=FP8), new(B, -(-inner // 128), dt=F32), new(B, inner + 2 * N)
    ops.quantize_fp8(u.reshape(B, inner), u8, su)
    ops.gemm_nt_fp8(u8, su, *q["w_dbc"], dbc)
    delta, Bm, Cm = dbc.reshape(B, 1, inner + 2 * N).split((inner, N, N), dim=2)
    ops.selective_scan_fwd(u, delta, p["A"], Bm, Cm, s, D=p["D"], z=h[..., inner:], delta_bias=p["delta_bias"], state_in=state[1], state_out=state[1])
    s8, ss = new(B, inner, dt=FP8), new(B, -(-inner // 128), dt=F32)
    ops.quantize_fp8(s.reshape(B, inner), s8, ss)
    out = new(B, width)
    ops.gemm_nt_fp8(s8, ss, *q["w_out"], out)
    return x + out


def serving_setup():
    g = torch.Generator().manual_seed(4)
    B, width, inner, N = 3, 256, 512, 16
    p = {k: v.to(DEV) for k, v in layer_parameters(g, width, inner, N).items()}
    q = {}
    p["w_dbc"] = torch.cat((p["w_d"], p["w_b"], p["w_c"]))
    for k in ("w_in", "w_out", "w_dbc"):
        R, C = p[k].shape
        w8, s = torch.empty(R, C, dtype=FP8, device=DEV), torch.empty(-(-R // 128), -(-C // 128), device=DEV)
        ops.quantize_fp8_blocks(p[k], w8, s)
        q[k] = (w8, s)
    fresh = lambda: [torch.zeros(B, 3, inner, dtype=BF16, device=DEV), torch.zeros(B, inner, N, device=DEV)]  # noqa: E731
    frames = [rand(g, B, width, dtype=BF16).to(DEV) for _ in range(12)]
    return p, q, fresh, frames


def test_a_layer_serves_frames_one_by_one_from_a_graph():
    """The layer's step recorded once and replayed for every frame, with eager work and synchronisations in between, against eager
    steps; a second graph of the same step has workspaces of its own and is replayed in turn with the first."""
    p, q, fresh, frames = serving_setup()
    state = fresh()
    want = [serve(p, q, x, state).clone() for x in frames]
    end = [t.clone() for t in state]
    assert all(bool(w.isfinite().all()) for w in want) and not torch.equal(want[0], want[1])
    x = torch.empty_like(frames[0])
    state = fresh()
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        for t in state:
            t.zero_()
        x.copy_(frames[0])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            serve(p, q, x, state)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = serve(p, q, x, state)
        graphs.append((graph, out))
    for t in state:
        t.zero_()
    for i, f in enumerate(frames):
        x.copy_(f)
        graph, out = graphs[i % 2]
        graph.replay()
        if i % 3 == 0:
            torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        torch.randn(1000, device=DEV).sum()
    assert torch.equal(state[0], end[0]) and torch.equal(state[1], end[1])


def test_a_training_step_replays():
    """Forward and backward of convolution, scan and norm recorded in one graph, replayed on new inputs: bits of the eager calls."""
    g = torch.Generator().manual_seed(6)
    B, T, C, N, K = 2, 300, 80, 16, 4
    x, dy = torch.empty(B, T, C, device=DEV), torch.empty(B, T, C, device=DEV)
    w, b = rand(g, C, K).to(DEV), rand(g, C).to(DEV)
    A, nw = (-torch.exp(rand(g, C, N))).to(DEV), rand(g, C).to(DEV)
    Bm, Cm = rand(g, B, T, N).to(DEV), rand(g, B, T, N).to(DEV)

    def body():
        new = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
        u, y, n, rstd = new(B, T, C), new(B, T, C), new(B * T, C), new(B * T)
        kept = ops.selective_scan_kept_states(B, T, C, N, DEV)
        ops.causal_conv_fwd(x, w, b, u)
        ops.selective_scan_fwd(u, u, A, Bm, Cm, y, kept_states=kept)
        ops.rms_norm_fwd(y.reshape(-1, C), nw, 1e-5, y=n, rstd=rstd)
        dn, dnw, du, dd, dA, dB, dC = new(B * T, C), new(C), new(B, T, C), new(B, T, C), new(C, N), new(B, T, N), new(B, T, N)
        ops.rms_norm_bwd(dy.reshape(-1, C), y.reshape(-1, C), nw, rstd, dn, dnw)
        ops.selective_scan_bwd(dn.reshape(B, T, C), u, u, A, Bm, Cm, kept, du, dd, dA, dB, dC)
        du += dd
        dx, dw, db = new(B, T, C), new(C, K), new(C)
        ops.causal_conv_bwd(du, x, w, b, dx, dw, db)
        return [n, dnw, dA, dB, dC, dx, dw, db]

    x.normal_(), dy.normal_()
    body()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = body()
    for i in range(4):
        x.normal_(), dy.normal_()
        want = body()
        for t in outs:
            t.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(outs, want):
            assert torch.equal(a, c), i


def test_calls_on_two_streams_at_once():
    """Two streams, each with its own operands and workspaces, many calls in flight: bits of the calls one by one."""
    g = torch.Generator().manual_seed(12)
    B, T, C, N = 2, 400, 64, 16
    sets = []
    for _ in range(2):
        t = scan_case(g, B, T, C, N, F32, state=True)
        sets.append((t, scan_run(t, F32)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(scan_run(sets[i][0], F32))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for k, v in sets[i][1].items():
                assert torch.equal(r[k], v), (i, k)


def test_gradients_against_differences():
    """Directional differences of the kernels' own float32 forward pass: d loss = loss(v + h d) - loss(v - h d) over 2 h with h = 2^-8.
    The difference's error is h^2 / 6 of the third derivative (of order one: 3e-6) and the rounding of the outputs, 1e-6 / h of
    their sum's usual error = 3e-4 relative to the sum of magnitudes; 5e-3 of the derivative's size is asked for."""
    g = torch.Generator().manual_seed(21)
    B, T, C, N = 2, 70, 24, 8
    t = scan_case(g, B, T, C, N, F32, state=True)
    got = scan_run(t, F32)
    names = dict(u="du", delta="ddelta", z="dz", Bm="dB", Cm="dC", A="dA", D="dD", delta_bias="d_delta_bias", state_in="d_state_in")

    def loss(v):
        y, state = torch.empty(B, T, C, device=DEV), torch.empty(B, C, N, device=DEV)
        c = lambda k: v[k].to(DEV)  # noqa: E731
        ops.selective_scan_fwd(v["u"], v["delta"], c("A"), v["Bm"], v["Cm"], y, D=c("D"), z=v["z"], delta_bias=c("delta_bias"),
                               state_in=c("state_in"), state_out=state)
        return float((y.double() * t["dy"].double()).sum() + (state.double() * t["d_state_out"].to(DEV).double()).sum())

    h = 2.0 ** -8
    for name, grad in names.items():
        d = torch.randn(t[name].shape, generator=g).to(t[name].device)
        if name == "A":
            d *= t["A"].abs()
        plus, minus = dict(t), dict(t)
        plus[name], minus[name] = t[name] + h * d, t[name] - h * d
        slope = (loss(plus) - loss(minus)) / (2 * h)
        want = float((got[grad].double().to(d.device) * d.double()).sum())
        size = float((got[grad].double().to(d.device) * d.double()).square().sum().sqrt())
        assert abs(slope - want) < 5e-3 * max(size, abs(want)) + 1e-3, (name, slope, want)


# ------------------------------------------------------------------------------------------------------------ refusals
def test_refused_calls_leave_the_outputs_alone():
    B, T, C, N, K = 2, 5, 16, 8, 4
    z = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    x, y, w, A, bc = z(B, T, C), torch.full((B, T, C), 3.0, device=DEV), z(C, K), -torch.ones(C, N, device=DEV), z(B, T, N)
    conv = lambda **k: ops.causal_conv_fwd(**{**dict(x=x, weight=w, bias=None, y=y), **k})  # noqa: E731
    scan = lambda **k: ops.selective_scan_fwd(**{**dict(u=x, delta=x, A=A, Bm=bc, Cm=bc, y=y), **k})  # noqa: E731
    for bad in (dict(weight=z(C, 5)), dict(weight=z(C, 1)), dict(weight=z(C + 1, K)), dict(weight=w.double()), dict(y=z(B, T, C, dt=BF16)),
                dict(y=z(B, T + 1, C)), dict(y=x), dict(bias=z(C + 1)), dict(state_in=z(B, K, C)), dict(state_out=x[:, :3]),
                dict(lengths=z(B)), dict(lengths=z(B + 1, dt=torch.int32)), dict(x=z(B, C, T).transpose(1, 2)), dict(x=x.half()), dict(x=x[0]),
                dict(x=x.cpu()), dict(y=z(1, T, C).expand(B, T, C)), dict(y=z(B, 1, C).expand(B, T, C))):
        with pytest.raises(ValueError):
            conv(**bad)
    for bad in (dict(A=z(C, 33)), dict(A=z(C, 0)), dict(A=z(N, C)), dict(delta=z(B, T, C, dt=BF16)), dict(Bm=z(B, T, N + 1)), dict(Cm=z(B, T + 1, N)),
                dict(y=x), dict(z=z(B, T, C + 1)), dict(D=z(N)), dict(delta_bias=z(C, dt=BF16)), dict(state_in=z(B, N, C)),
                dict(state_out=z(B, C, N, dt=BF16)), dict(kept_states=z(7)), dict(lengths=z(B, dt=torch.int64)), dict(u=x.transpose(1, 2))):
        with pytest.raises(ValueError):
            scan(**bad)
    kept = ops.selective_scan_kept_states(B, T, C, N, DEV)
    new = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    back = lambda **k: ops.selective_scan_bwd(**{**dict(dy=x, u=new(B, T, C), delta=new(B, T, C), A=A, Bm=bc, Cm=bc, kept_states=kept, du=y,  # noqa: E731
                                                        ddelta=new(B, T, C), dA=new(C, N), dB=new(B, T, N), dC=new(B, T, N)), **k})
    both = new(B, T, C)
    for bad in (dict(du=x), dict(du=both, ddelta=both), dict(dz=new(B, T, C)), dict(z=new(B, T, C)), dict(kept_states=kept[1:]), dict(dA=new(N, C)), dict(du=None), dict(dB=bc),
                dict(d_state_in=new(B, C, N + 1))):
        with pytest.raises(ValueError):
            back(**bad)
    m, nw, q, s = z(4, 300), z(300), z(4, 300, dt=FP8), z(4, 3)
    keep = torch.full((4, 300), 3.0, device=DEV)
    for call in (lambda: ops.rms_norm_fwd(m, nw, 1e-5, y=keep[:, :299]), lambda: ops.rms_norm_fwd(m, nw[1:], 1e-5, y=keep),
                 lambda: ops.rms_norm_fwd(m.t(), nw, 1e-5, y=keep), lambda: ops.rms_norm_fwd(m, nw, 1e-5, y8=q, scales=z(4, 2)),
                 lambda: ops.rms_norm_fwd(m, nw, 1e-5, y=keep, rstd=z(3)), lambda: ops.rms_norm_bwd(m, m, nw, z(4), keep, z(299)),
                 lambda: ops.quantize_fp8(m, q, z(4, 2)), lambda: ops.quantize_fp8(m, m, s), lambda: ops.quantize_fp8_blocks(m, q, z(1, 2))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.rms_norm_fwd(m, nw, 1e-5), lambda: ops.rms_norm_fwd(m, nw, 1e-5, y8=q),
                 lambda: ops.rms_norm_fwd(m, nw, 1e-5, y=keep, sum_out=z(4, 300)), lambda: ops.rms_norm_fwd(z(1, 16400), z(16400), 1e-5, y=z(1, 16400))):
        with pytest.raises(RuntimeError):
            call()
    a8, b8, out = z(4, 304, dt=FP8), z(8, 304, dt=FP8), torch.full((4, 8), 3.0, dtype=BF16, device=DEV)
    gemm = lambda **k: ops.gemm_nt_fp8(**{**dict(a8=a8, a_scales=z(4, 3), b8=b8, b_scales=z(1, 3), out=out), **k})  # noqa: E731
    for bad in (dict(a8=q, a_scales=s), dict(a_scales=z(4, 2)), dict(b8=z(8, 320, dt=FP8)), dict(b_scales=z(8, 3)), dict(out=z(4, 8)),
                dict(out=z(4, 9, dt=BF16)), dict(a8=z(4 * 304 + 8, dt=FP8)[8:].view(4, 304)), dict(out=z(8, 4, dt=BF16).t())):
        with pytest.raises(ValueError):
            gemm(**bad)
    torch.cuda.synchronize()
    assert bool((y == 3.0).all()) and bool((keep == 3.0).all()) and bool((out == 3.0).all())


# --------------------------------------------------------------------------------------------------- far places in memory
def test_offsets_beyond_32_bits():
    """Sequences and steps more than 2^31 elements apart, outputs of more than 2^31 elements: the same bits as close together."""
    g = torch.Generator().manual_seed(31)
    B, T, C, N, K = 2, 40, 24, 16, 4
    t = scan_case(g, B, T, C, N, BF16, state=True)
    far = torch.empty(2 ** 31 + 10 * T * C, dtype=BF16, device=DEV)

    def spread(v, at):
        out = torch.as_strided(far, v.shape, (2 ** 31 + 64, v.shape[2], 1), at)
        return out.copy_(v)

    near = scan_run(t, BF16)
    moved = dict(t)
    for i, k in enumerate(("u", "delta", "z", "dy", "Bm", "Cm")):
        moved[k] = spread(t[k], i * T * C)
    got = scan_run(moved, BF16)
    for k, v in near.items():
        assert torch.equal(got[k], v), k
    # an output whose sequences are far apart, and an input whose steps are (2^26 elements, 40 of them)
    y = torch.as_strided(far, (B, T, C), (2 ** 31 + 64, C, 1), 8 * T * C)
    args = lambda v, out: ops.selective_scan_fwd(v["u"], v["delta"], t["A"].to(DEV), v["Bm"], v["Cm"], out, D=t["D"].to(DEV), z=v["z"],  # noqa: E731
                                                 delta_bias=t["delta_bias"].to(DEV), state_in=t["state_in"].to(DEV))
    args(moved, y)
    assert torch.equal(y, near["y"])
    w, b = rand(g, C, K).to(DEV), rand(g, C).to(DEV)
    want, got = torch.empty(B, T, C, dtype=BF16, device=DEV), torch.as_strided(far, (B, T, C), (C, 2 ** 31 // T, 1), 8 * T * C)
    x = t["u"].contiguous()
    ops.causal_conv_fwd(x, w, b, want)
    ops.causal_conv_fwd(moved["u"], w, b, got)
    assert torch.equal(got, want)
    got.copy_(x)
    again, want_d, got_d = torch.empty_like(want), [torch.empty_like(v) for v in (x, w, b)], [torch.empty_like(v) for v in (x, w, b)]
    ops.causal_conv_fwd(got, w, b, again)
    assert torch.equal(again, want)
    ops.causal_conv_bwd(t["dy"].contiguous(), x, w, b, *want_d)
    ops.causal_conv_bwd(moved["dy"], got, w, b, *got_d)
    assert all(torch.equal(p, q) for p, q in zip(got_d, want_d))
    del far, y, moved, got
    # more than 2^31 values of a norm, of 8-bit operands and of a product
    rows, C = 2 ** 17 + 3, 16384
    x, nw = torch.zeros(rows, C, dtype=BF16, device=DEV), rand(g, C).to(DEV)
    x[-3:] = rand(g, 3, C, dtype=BF16).to(DEV)
    y, x8, s = torch.empty_like(x), torch.empty(rows, C, dtype=FP8, device=DEV), torch.empty(rows, C // 128, device=DEV)
    rstd, dx, dw = torch.empty(rows, device=DEV), torch.empty_like(x), torch.empty_like(nw)
    ops.rms_norm_fwd(x, nw, 1e-5, y=y, y8=x8, scales=s, rstd=rstd)
    ops.rms_norm_bwd(x, x, nw, rstd, dx, dw)
    y3, x3, s3, r3, dx3, dw3 = torch.empty(3, C, dtype=BF16, device=DEV), torch.empty(3, C, dtype=FP8, device=DEV), s[:3].clone(), rstd[:3].clone(), dx[:3].clone(), dw.clone()
    ops.rms_norm_fwd(x[-3:].clone(), nw, 1e-5, y=y3, y8=x3, scales=s3, rstd=r3)
    ops.rms_norm_bwd(x[-3:].clone(), x[-3:].clone(), nw, r3, dx3, dw3)
    b8 = lambda v: v.view(torch.uint8)  # noqa: E731
    assert torch.equal(y[-3:], y3) and torch.equal(b8(x8[-3:]), b8(x3)) and torch.equal(s[-3:], s3) and torch.equal(rstd[-3:], r3)
    assert torch.equal(dx[-3:], dx3) and bool((dw - dw3).abs().max() <= 1e-5 * dw3.abs().max())    # zero rows add nothing; another order
    ops.quantize_fp8(x, x8, s)
    ops.quantize_fp8(x[-3:].clone(), x3, s3)
    assert torch.equal(b8(x8[-3:]), b8(x3)) and torch.equal(s[-3:], s3)
    del x, y, x8, s, rstd, dx
    M = N = 46400
    a8, sa = (rand(g, M, 16) * 2).to(FP8).to(DEV), torch.ones(M, 1, device=DEV)
    out, last = torch.empty(M, N, dtype=BF16, device=DEV), torch.empty(64, N, dtype=BF16, device=DEV)
    sb = torch.ones(-(-N // 128), 1, device=DEV)
    ops.gemm_nt_fp8(a8, sa, a8, sb, out)
    ops.gemm_nt_fp8(a8[-64:].contiguous(), sa[-64:].contiguous(), a8, sb, last)
    assert torch.equal(out[-64:], last)


# ------------------------------------------------------------------------------------------------- views and other threads
def test_broadcast_inputs_and_their_gradients():
    """Inputs expanded over sequences and steps (strides of zero): the gradients are those of their copies, each element's own."""
    g = torch.Generator().manual_seed(77)
    B, T, C, N, K = 3, 50, 70, 16, 4
    t = scan_case(g, B, T, C, N, F32, use_z=False, state=True)
    flat = dict(t)
    for k, shape in (("u", (1, 1, C)), ("delta", (1, T, C)), ("Bm", (B, 1, N)), ("Cm", (1, 1, N)), ("dy", (1, T, C))):
        one = rand(g, *shape).to(DEV)
        t[k] = one.expand(B, T, shape[2])
        flat[k] = t[k].contiguous()
    want, got = scan_run(flat, F32), scan_run(t, F32)
    for k, v in want.items():
        assert torch.equal(got[k], v), k
    w, b = rand(g, C, K).to(DEV), rand(g, C).to(DEV)
    new = lambda *s: torch.full(s, NAN, device=DEV)  # noqa: E731
    outs = []
    for v in (flat, t):
        y, dx, dw, db = new(B, T, C), new(B, T, C), new(C, K), new(C)
        ops.causal_conv_fwd(v["u"], w, b, y)
        ops.causal_conv_bwd(v["dy"], v["u"], w, b, dx, dw, db)
        outs.append((y, dx, dw, db))
    assert all(torch.equal(p, q) for p, q in zip(*outs))


@pytest.mark.parametrize("C,N", [(5, 3), (70, 16), (67, 20)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_lies_beside_the_outputs_stays(C, N, dtype):
    g = torch.Generator().manual_seed(C)
    B, T, K = 2, 37, 3
    t = scan_case(g, B, T, C, N, dtype, state=True, ragged=True)
    c = lambda k: t[k].to(DEV)  # noqa: E731

    def beside(W):
        wide = torch.full((B + 1, T + 2, W + 5), 7.0, dtype=dtype, device=DEV)
        return wide, wide[:B, 1:T + 1, 2:W + 2]

    def untouched(wide, W):
        wide = wide.clone()
        inner = wide[:B, 1:T + 1, 2:W + 2]
        assert not bool((inner == 7.0).all())
        inner.fill_(7.0)
        assert bool((wide == 7.0).all())

    made = {k: beside(W) for k, W in (("y", C), ("du", C), ("ddelta", C), ("dz", C), ("dB", N), ("dC", N), ("cy", C), ("cdx", C))}
    out = {k: v[1] for k, v in made.items()}
    kept = ops.selective_scan_kept_states(B, T, C, N, DEV)
    ops.selective_scan_fwd(t["u"], t["delta"], c("A"), t["Bm"], t["Cm"], out["y"], D=c("D"), z=t["z"], delta_bias=c("delta_bias"),
                           kept_states=kept, lengths=c("lengths"))
    dA = torch.empty(C, N, device=DEV)
    ops.selective_scan_bwd(t["dy"], t["u"], t["delta"], c("A"), t["Bm"], t["Cm"], kept, out["du"], out["ddelta"], dA, out["dB"], out["dC"],
                           D=c("D"), z=t["z"], delta_bias=c("delta_bias"), dz=out["dz"], lengths=c("lengths"))
    w = rand(g, C, K).to(DEV)
    dw = torch.empty_like(w)
    ops.causal_conv_fwd(t["u"], w, None, out["cy"], lengths=c("lengths"))
    ops.causal_conv_bwd(t["dy"], t["u"], w, None, out["cdx"], dw, lengths=c("lengths"))
    for k, (wide, view) in made.items():
        untouched(wide, view.shape[2])
        for i in range(B):
            assert not bool(view[i, int(t["lengths"][i]):].any()), k


def test_calls_from_two_threads():
    """Two threads, each with its own stream and operands, without waiting for each other: bits of the calls one by one."""
    import threading
    g = torch.Generator().manual_seed(13)
    sets = [scan_case(g, 2, 300, 48, 16, F32, state=True) for _ in range(2)]
    want = [scan_run(t, F32) for t in sets]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = scan_run(sets[i], F32)
                    stream.synchronize()
                    assert all(torch.equal(got[k], v) for k, v in want[i].items())
        except BaseException as e:  # noqa: B902
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed

"""Calls at the edges of what the sequence layer's documentation allows: lengths outside [0, T], contiguous tensors at the alignment of an
element, as many sequences and rows as there may be, the deepest products, the product's parts inside a graph."""
import pytest
import torch

from oracle import sequence_oracle as so
from slam_amd.network import sequence_ops as ops
from test_sequence_ops_gpu import BF16, DEV, F32, FP8, NAN, rand, scan_case, scan_run

pytestmark = pytest.mark.gpu


def shifted(t, by=1):
    """A contiguous copy whose first element lies `by` elements behind an aligned address."""
    flat = torch.empty(t.numel() + by, dtype=t.dtype, device=DEV)
    out = flat[by:].view(t.shape)
    out.copy_(t)
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 40, 150])
def test_lengths_outside_the_sequence(dtype, T):
    """Taken as the nearest of 0 and T: the bits of the call with those, forward and back."""
    g = torch.Generator().manual_seed(T)
    B, C, N, K = 4, 21, 16, 4
    t = scan_case(g, B, T, C, N, dtype, state=True)
    raw, near = torch.tensor([T + 9, -3, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32), torch.tensor([T, 0, T, 0], dtype=torch.int32)
    results = []
    for n in (near, raw):
        t["lengths"] = n
        out = scan_run(t, dtype)
        x, w, dy, st = t["u"], rand(torch.Generator().manual_seed(1), C, K).to(DEV), t["dy"], t["z"][:, :1].expand(B, K - 1, C).contiguous()
        new = lambda *s, dt=dtype: torch.full(s, NAN, dtype=dt, device=DEV)  # noqa: E731
        out |= dict(cy=new(B, T, C), cs=new(B, K - 1, C), cdx=new(B, T, C), cdw=new(C, K, dt=F32), cdb=new(C, dt=F32), cds=new(B, K - 1, C))
        ops.causal_conv_fwd(x, w, None, out["cy"], state_in=st, state_out=out["cs"], lengths=n.to(DEV))
        ops.causal_conv_bwd(dy, x, w, None, out["cdx"], out["cdw"], out["cdb"], state_in=st, d_state_in=out["cds"], d_state_out=st, lengths=n.to(DEV))
        y = new(B, 1, C)
        first = [t[k][:, :1] for k in ("u", "delta", "Bm", "Cm", "z")]
        state = t["state_in"].to(DEV)
        ops.selective_scan_fwd(first[0], first[1], t["A"].to(DEV), first[2], first[3], y, z=first[4], state_in=state, state_out=state, lengths=n.to(DEV))
        out |= dict(step_y=y, step_state=state)
        results.append(out)
    for k, v in results[0].items():
        assert torch.equal(v, results[1][k]), k
    assert bool(results[0]["y"][0].any()) and not bool(results[0]["y"][1].any())


@pytest.mark.parametrize("C", [3, 24, 130, 1000, 1029, 4096])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_and_8bit_rows_at_any_alignment(C, dtype):
    g = torch.Generator().manual_seed(C)
    rows = 5
    x, r, dy, w = (rand(g, *s, dtype=t).to(DEV) for s, t in (((rows, C), dtype), ((rows, C), dtype), ((rows, C), dtype), ((C,), F32)))
    outs = []
    for move in (lambda t: t, shifted):
        new = lambda *s, dt=dtype: move(torch.zeros(*s, dtype=dt, device=DEV))  # noqa: E731
        a, b, d, v = move(x), move(r), move(dy), move(w)
        kb = -(-C // 128)
        y, s, q, sc, rs, dx, dw = new(rows, C), new(rows, C), new(rows, C, dt=FP8), new(rows, kb, dt=F32), new(rows, dt=F32), new(rows, C), new(C, dt=F32)
        ops.rms_norm_fwd(a, v, 1e-5, y=y, residual=b, sum_out=s, y8=q, scales=sc, rstd=rs)
        ops.rms_norm_bwd(d, s, v, rs, dx, dw, d_sum=b)
        q2, s2, q3, s3 = new(rows, C, dt=FP8), new(rows, kb, dt=F32), new(rows, C, dt=FP8), new(1, kb, dt=F32)
        ops.quantize_fp8(a, q2, s2)
        ops.quantize_fp8_blocks(a, q3, s3)
        outs.append([t.view(torch.uint8) if t.dtype == FP8 else t for t in (y, s, q, sc, rs, dx, dw, q2, s2, q3, s3)])
    assert all(torch.equal(p, q) for p, q in zip(*outs))


@pytest.mark.parametrize("M,N,K", [(3, 21, 400), (70, 131, 400), (300, 1031, 1040)])
def test_product_at_any_alignment_of_scales_and_output(M, N, K):
    g = torch.Generator().manual_seed(M)
    a8, b8 = rand(g, M, K).to(FP8).to(DEV), rand(g, N, K).to(FP8).to(DEV)
    sa, sb = rand(g, M, -(-K // 128)).abs().to(DEV), rand(g, -(-N // 128), -(-K // 128)).abs().to(DEV)
    want, got = torch.empty(M, N, dtype=BF16, device=DEV), shifted(torch.zeros(M, N, dtype=BF16))
    ops.gemm_nt_fp8(a8, sa, b8, sb, want)
    ops.gemm_nt_fp8(a8, shifted(sa), b8, shifted(sb), got)
    assert torch.equal(want, got)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_and_convolution_at_any_alignment(dtype):
    g = torch.Generator().manual_seed(3)
    B, T, C, N, K = 2, 50, 37, 16, 4
    t = scan_case(g, B, T, C, N, dtype, state=True)
    for k in ("u", "delta", "z", "dy", "Bm", "Cm"):
        t[k] = t[k].contiguous()
    want = scan_run(t, dtype)
    moved = {k: shifted(v) if isinstance(v, torch.Tensor) and not k.endswith("_") and k != "lengths" else v for k, v in t.items()}
    got = scan_run(moved, dtype)
    for k, v in want.items():
        assert torch.equal(got[k], v), k
    w, b = rand(g, C, K).to(DEV), rand(g, C).to(DEV)
    outs = []
    for move in (lambda v: v, shifted):
        y, dx, dw, db = (move(torch.zeros_like(v)) for v in (t["u"], t["u"], w, b))
        ops.causal_conv_fwd(move(t["u"]), move(w), move(b), y)
        ops.causal_conv_bwd(move(t["dy"]), move(t["u"]), move(w), move(b), dx, dw, db)
        outs.append((y, dx, dw, db))
    assert all(torch.equal(p, q) for p, q in zip(*outs))


@pytest.mark.parametrize("T", [1, 3])
def test_the_most_sequences(T):
    """65535 of them: each has the bits of a call by itself; gradients of parameters against sums of the halves."""
    B, C, N, K = 65535, 5, 3, 3
    dg = torch.Generator(device=DEV).manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=dg, device=DEV)  # noqa: E731
    u, delta, z, dy, Bm, Cm, A, h = r(B, T, C), r(B, T, C), r(B, T, C), r(B, T, C), r(B, T, N), r(B, T, N), -r(C, N).exp(), r(B, C, N)
    w, st = r(C, K), r(B, K - 1, C)

    def run(s):
        n = s.stop - s.start
        e = lambda *v: torch.full(v, NAN, device=DEV)  # noqa: E731
        o = dict(y=e(n, T, C), h=e(n, C, N), du=e(n, T, C), dd=e(n, T, C), dz=e(n, T, C), dB=e(n, T, N), dC=e(n, T, N), dh=e(n, C, N), cy=e(n, T, C), cs=e(n, K - 1, C),
                 cdx=e(n, T, C), dA=e(C, N), dw=e(C, K))
        kept = ops.selective_scan_kept_states(n, T, C, N, DEV)
        ops.selective_scan_fwd(u[s], delta[s], A, Bm[s], Cm[s], o["y"], z=z[s], state_in=h[s], state_out=o["h"], kept_states=kept)
        ops.selective_scan_bwd(dy[s], u[s], delta[s], A, Bm[s], Cm[s], kept, o["du"], o["dd"], o["dA"], o["dB"], o["dC"], z=z[s], dz=o["dz"], d_state_in=o["dh"],
                               d_state_out=h[s])
        ops.causal_conv_fwd(u[s], w, None, o["cy"], state_in=st[s], state_out=o["cs"])
        ops.causal_conv_bwd(dy[s], u[s], w, None, o["cdx"], o["dw"], state_in=st[s])
        return o

    whole = run(slice(0, B))
    halves = [run(slice(0, 30000)), run(slice(30000, B))]
    for k, v in whole.items():
        if k in ("dA", "dw"):
            # two orders of the same float32 sum of 65535 T terms; their usual error is sqrt of it, a thousandth of what is asked for
            parts = halves[0][k].double() + halves[1][k].double()
            assert bool(((v.double() - parts).abs() <= 65535 * T * 2.0 ** -24 * v.abs().max()).all()), k
        else:
            assert torch.equal(v, torch.cat([q[k] for q in halves])), k


def test_the_most_rows_of_a_norm():
    rows, C = (1 << 24) - 1, 3
    dg = torch.Generator(device=DEV).manual_seed(1)
    x, dy, w = torch.randn(rows, C, generator=dg, device=DEV), torch.randn(rows, C, generator=dg, device=DEV), torch.randn(C, generator=dg, device=DEV)
    y, rstd, dx, dw = torch.empty_like(x), torch.empty(rows, device=DEV), torch.empty_like(x), torch.empty_like(w)
    ops.rms_norm_fwd(x, w, 1e-5, y=y, rstd=rstd)
    ops.rms_norm_bwd(dy, x, w, rstd, dx, dw)
    tail = slice(rows - 1000, rows)
    y2, r2, dx2, dw2 = torch.empty(1000, C, device=DEV), torch.empty(1000, device=DEV), torch.empty(1000, C, device=DEV), torch.empty_like(w)
    ops.rms_norm_fwd(x[tail], w, 1e-5, y=y2, rstd=r2)
    ops.rms_norm_bwd(dy[tail], x[tail], w, r2, dx2, dw2)
    assert torch.equal(y[tail], y2) and torch.equal(rstd[tail], r2) and torch.equal(dx[tail], dx2)
    hat = x.double() * rstd.double()[:, None]
    # a slot's rows in sequence (2^24 / (512 x 16) of them), then slots and parts: under 2200 float32 additions
    assert bool(((dw.double() - (dy.double() * hat).sum(0)).abs() <= (2200 + 8) * so.U * (dy.double() * hat).abs().sum(0)).all())


@pytest.mark.parametrize("M,N,K", [(1, 20, 7000000), (17, 40, 1000016), (70, 64, 300016)])
def test_the_deepest_products(M, N, K):
    """Operands of small whole numbers in a scale of one: at most eight of a block's products are cut to 2^-13 of the largest, all of them
    whole numbers below 2^13 times the least; sums stay below 2^24, so the float32 sums are exact and the output is the rounded whole number."""
    dg = torch.Generator(device=DEV).manual_seed(K)
    a, b = (torch.randint(-1, 2, s, generator=dg, device=DEV).to(F32) for s in ((M, K), (N, K)))
    out = torch.full((M, N), NAN, dtype=BF16, device=DEV)
    kb = -(-K // 128)
    ops.gemm_nt_fp8(a.to(FP8), torch.ones(M, kb, device=DEV), b.to(FP8), torch.ones(-(-N // 128), kb, device=DEV), out)
    want = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    for k in range(0, K, 1 << 18):
        want += torch.mm(a[:, k:k + (1 << 18)].double(), b[:, k:k + (1 << 18)].double().t().contiguous())
    assert torch.equal(out, want.to(BF16))


def test_parts_of_a_product_in_two_graphs():
    """Products that are cut along k have a workspace each: two graphs of two products, replayed in turn with eager work in between."""
    g = torch.Generator().manual_seed(5)
    shapes = [(100, 70, 9232), (5, 40, 8336)]
    sets = []
    for M, N, K in shapes:
        kb = -(-K // 128)
        sets.append((torch.empty(M, K, dtype=FP8, device=DEV), rand(g, M, kb).abs().to(DEV), rand(g, N, K).to(FP8).to(DEV), rand(g, -(-N // 128), kb).abs().to(DEV)))
    side = torch.cuda.Stream()

    def body():
        outs = []
        for (a8, sa, b8, sb), (M, N, K) in zip(sets, shapes):
            outs.append(torch.empty(M, N, dtype=BF16, device=DEV))
            ops.gemm_nt_fp8(a8, sa, b8, sb, outs[-1])
        return outs

    def fill(seed):
        dg = torch.Generator(device=DEV).manual_seed(seed)
        for a8, *_ in sets:
            a8.copy_(torch.randn(a8.shape, generator=dg, device=DEV))

    fill(0)
    body()
    graphs = []
    for _ in range(2):
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = body()
        graphs.append((graph, outs))
    for i in range(6):
        fill(i)
        want = body()
        graph, outs = graphs[i % 2]
        for t in outs:
            t.fill_(7.0)
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, want)), i

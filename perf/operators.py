"""The sequence-layer operators as cases that can be timed and compared: RMS norm with the residual's addition,
matrix product of 8-bit operands, short causal convolution, selective scan.

`run` computes a case either in elementary torch operations (`own` false) or through slam_amd.network.sequence_ops
(`own` true); `exact` computes it in 64 bits.  Layouts: sequences [B, T, C], channels innermost; a padded batch has
`lengths` [B], rows at and after a sequence's length are zero in every output.
"""
import math

import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
MIN_SCALE = 2.0 ** -100     # a block of zeros gets this scale
EPS = 1e-5


def listed():
    return [
        # one frame of each of 32 streams enters the convolution of a 4096-wide layer (the fully connected width here)
        dict(name="conv_token", op="conv", B=32, T=1, C=4096, K=4, dtype="bf16", train=False, state=True, ragged=False),
        # a batch of recorded sequences of up to 200 frames (the configured sequence length), of unequal length
        dict(name="conv_frames", op="conv", B=16, T=200, C=2048, K=4, dtype="bf16", train=False, state=True, ragged=True),
        # a training step's forward and backward over long sequences
        dict(name="conv_train", op="conv", B=8, T=2048, C=4096, K=4, dtype="bf16", train=True, state=False, ragged=False),
        # the scan's update for one frame of each of 32 streams
        dict(name="scan_token", op="scan", B=32, T=1, C=4096, N=16, dtype="bf16", train=False, state=True, ragged=False),
        # one long recording taken in at once
        dict(name="scan_prompt", op="scan", B=1, T=8192, C=4096, N=16, dtype="bf16", train=False, state=True, ragged=False),
        # a training step over recorded sequences of unequal length, float32, an odd width
        dict(name="scan_train_ragged", op="scan", B=5, T=200, C=1000, N=8, dtype="f32", train=True, state=True, ragged=True),
        # a training step over long sequences
        dict(name="scan_train", op="scan", B=8, T=2048, C=2048, N=16, dtype="bf16", train=True, state=False, ragged=False),
        # the norm in front of an 8-bit projection, one frame of each of 4 streams
        dict(name="norm_token", op="norm", rows=4, C=4096, dtype="bf16", residual=True, fp8=True, train=False),
        # the norm of a training step, with the gradient that arrives at the sum
        dict(name="norm_train", op="norm", rows=16384, C=4096, dtype="bf16", residual=True, fp8=False, train=True),
        # the projection of one frame of each of 4 streams: the weights are read once
        dict(name="gemm_token", op="gemm", M=4, N=8192, K=4096, quantize=False),
        # the projection behind a scan: activations are put in 8 bits within the call; an odd number of rows
        dict(name="gemm_frames", op="gemm", M=777, N=2056, K=4096, quantize=True),
        # the projection of a long batch
        dict(name="gemm_prompt", op="gemm", M=8192, N=8192, K=4096, quantize=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("conv", "scan", "norm", "gemm"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    train = rng.random() < 0.5
    while True:
        if op == "conv":
            c = dict(op=op, B=_spread(rng, 1, 64), T=_spread(rng, 1, 8192), C=_spread(rng, 8, 8192), K=rng.choice((2, 3, 4)),
                     dtype=dtype, train=train, state=rng.random() < 0.5, ragged=rng.random() < 0.5)
            ok = c["B"] * c["T"] * c["C"] <= 1 << 25
        elif op == "scan":
            c = dict(op=op, B=_spread(rng, 1, 64), T=_spread(rng, 1, 8192), C=_spread(rng, 8, 8192), N=rng.choice((4, 8, 12, 16, 16, 16, 32)),
                     dtype=dtype, train=train, state=rng.random() < 0.5, ragged=rng.random() < 0.5)
            ok = c["B"] * c["T"] * c["C"] * c["N"] <= 1 << 28
        elif op == "norm":
            c = dict(op=op, rows=_spread(rng, 1, 32768), C=_spread(rng, 8, 16384), dtype=dtype, residual=rng.random() < 0.7,
                     fp8=not train and rng.random() < 0.6, train=train)
            ok = c["rows"] * c["C"] <= 1 << 26
        else:
            c = dict(op=op, M=_spread(rng, 1, 8192), N=_spread(rng, 16, 16384), K=16 * _spread(rng, 4, 1024),
                     quantize=rng.random() < 0.5)
            ok = c["M"] * c["N"] * c["K"] <= 1 << 37
        if ok:
            return c


def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _lengths(case, g):
    """Lengths of a padded batch: the longest sequence fills it."""
    if not case["ragged"]:
        return None
    n = torch.randint((case["T"] + 1) // 2, case["T"] + 1, (case["B"],), generator=g, device="cuda", dtype=torch.int32)
    n[0] = case["T"]
    return n


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case=dict(case))
    if case["op"] == "conv":
        B, T, C, K, dt = case["B"], case["T"], case["C"], case["K"], _dtype(case["dtype"])
        # the layer's projection holds the convolution's input and the gate side by side
        s["x"] = randn(B, T, 2 * C, dtype=dt)[..., :C]
        s["weight"] = randn(C, K, scale=K ** -0.5)
        s["bias"] = randn(C, scale=0.1)
        s["lengths"] = _lengths(case, g)
        s["state_in"] = randn(B, K - 1, C, dtype=dt) if case["state"] else None
        if case["train"]:
            s["dy"] = randn(B, T, C, dtype=dt)
            s["d_state_out"] = randn(B, K - 1, C, dtype=dt) if case["state"] else None
    elif case["op"] == "scan":
        B, T, C, N, dt = case["B"], case["T"], case["C"], case["N"], _dtype(case["dtype"])
        s["u"] = randn(B, T, C, dtype=dt)
        s["delta"] = randn(B, T, C, dtype=dt, scale=0.5)
        s["z"] = randn(B, T, 2 * C, dtype=dt)[..., C:]
        # time steps of 0.001 to 0.1 at delta = 0, decay rates of 1 to N
        step = torch.exp(torch.rand(C, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
        s["delta_bias"] = torch.log(torch.expm1(step))
        s["A"] = -(torch.arange(1, N + 1, device="cuda").float() * torch.exp(randn(C, N, scale=0.2)))
        s["D"] = 1.0 + randn(C, scale=0.1)
        s["Bm"] = randn(B, T, N, dtype=dt)
        s["Cm"] = randn(B, T, N, dtype=dt)
        s["lengths"] = _lengths(case, g)
        s["state_in"] = randn(B, C, N, scale=0.5) if case["state"] else None
        if case["train"]:
            s["dy"] = randn(B, T, C, dtype=dt)
            s["d_state_out"] = randn(B, C, N, scale=0.5) if case["state"] else None
    elif case["op"] == "norm":
        rows, C, dt = case["rows"], case["C"], _dtype(case["dtype"])
        s["x"] = randn(rows, C, dtype=dt)
        s["weight"] = 1.0 + randn(C, scale=0.1)
        s["residual"] = randn(rows, C, dtype=dt, scale=4.0) if case["residual"] else None
        if case["train"]:
            s["dy"] = randn(rows, C, dtype=dt)
            s["d_sum"] = randn(rows, C, dtype=dt) if case["residual"] else None
    else:
        M, N, K = case["M"], case["N"], case["K"]
        s["b8"], s["b_scales"] = _quantize_blocks(randn(N, K, scale=K ** -0.5))
        a = randn(M, K, dtype=torch.bfloat16)
        if case["quantize"]:
            s["a"] = a
        else:
            s["a8"], s["a_scales"] = _quantize_rows(a.float())
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _silu_slope(v):
    p = _sigmoid(v)
    return p * (1.0 + v * (1.0 - p))


def _inside(lengths, T, like):
    """[B, T, 1] of ones inside the sequences; None where the batch is not padded."""
    if lengths is None:
        return None
    return (torch.arange(T, device=like.device)[None, :] < lengths[:, None])[..., None]


def _masked(v, mask):
    return v if mask is None else torch.where(mask, v, torch.zeros((), dtype=v.dtype, device=v.device))


def _quantize_rows(v):
    """float32 [M, K] -> e4m3 [M, K] and scales [M, ceil(K / 128)]."""
    M, K = v.shape
    kb = -(-K // 128)
    p = torch.nn.functional.pad(v, (0, kb * 128 - K)).view(M, kb, 128)
    scales = (p.abs().amax(2) / FP8_MAX).clamp_min(MIN_SCALE)
    q = (p / scales[..., None]).clamp(-FP8_MAX, FP8_MAX).view(M, kb * 128)[:, :K]
    return q.to(FP8).contiguous(), scales


def _quantize_blocks(w):
    """float32 [N, K] -> e4m3 [N, K] and scales [ceil(N / 128), ceil(K / 128)]."""
    N, K = w.shape
    nb, kb = -(-N // 128), -(-K // 128)
    p = torch.nn.functional.pad(w, (0, kb * 128 - K, 0, nb * 128 - N)).view(nb, 128, kb, 128)
    scales = (p.abs().amax((1, 3)) / FP8_MAX).clamp_min(MIN_SCALE)
    q = (p / scales[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).view(nb * 128, kb * 128)[:N, :K]
    return q.to(FP8).contiguous(), scales


def _plain_gemm(s):
    case = s["case"]
    a8, sa = _quantize_rows(s["a"].float()) if case["quantize"] else (s["a8"], s["a_scales"])
    a = a8.float() * sa.repeat_interleave(128, 1)[:, :case["K"]]
    b = s["b8"].float() * s["b_scales"].repeat_interleave(128, 0)[:case["N"]].repeat_interleave(128, 1)[:, :case["K"]]
    return {"out": (a @ b.t()).to(torch.bfloat16)}


def _plain_norm(s):
    case = s["case"]
    x, w = s["x"], s["weight"]
    total = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    v = total.float()
    rstd = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
    hat = v * rstd
    y = hat * w
    out = {}
    if case["residual"]:
        out["sum"] = total
    if case["fp8"]:
        out["y8"], out["scales"] = _quantize_rows(y)
    else:
        out["y"] = y.to(x.dtype)
    if case["train"]:
        dy = s["dy"].float()
        wdy = w * dy
        dx = rstd * (wdy - hat * (wdy * hat).mean(1, keepdim=True))
        if s["d_sum"] is not None:
            dx = dx + s["d_sum"].float()
        out["dx"] = dx.to(x.dtype)
        out["dweight"] = (dy * hat).sum(0, dtype=torch.float64).float()
    return out


def _plain_conv(s):
    case = s["case"]
    x, w, dt = s["x"], s["weight"], s["x"].dtype
    B, T, C = x.shape
    K = w.shape[1]
    mask = _inside(s["lengths"], T, x)
    before = torch.zeros(B, K - 1, C, dtype=dt, device=x.device) if s["state_in"] is None else s["state_in"]
    padded = torch.cat((before, x), 1)
    window = padded.float().unfold(1, K, 1)                          # [B, T, C, K]
    pre = (window * w).sum(-1) + s["bias"]
    out = {"y": _masked(pre * _sigmoid(pre), mask).to(dt)}
    ends = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device=x.device)
    at = (ends[:, None] + torch.arange(K - 1, device=x.device))[..., None].expand(B, K - 1, C)
    out["state_out"] = padded.gather(1, at)
    if case["train"]:
        dpre = _masked(s["dy"].float() * _silu_slope(pre), mask)
        dpad = torch.nn.functional.pad(dpre, (0, 0, K - 1, K - 1)).unfold(1, K, 1)   # [B, T + K - 1, C, K]
        dx = (dpad * w.flip(1)).sum(-1)
        if s["d_state_out"] is not None:
            dx = dx.scatter_add(1, at, s["d_state_out"].float())
            out["d_state_in"] = dx[:, :K - 1].to(dt)
        out["dx"] = _masked(dx[:, K - 1:], mask).to(dt)
        out["dweight"] = (dpre[..., None] * window).sum((0, 1), dtype=torch.float64).float()
        out["dbias"] = dpre.sum((0, 1), dtype=torch.float64).float()
    return out


def _linear_recurrence(a, x):
    """h_t = a_t h_{t-1} + x_t along axis 1, by doubling; overwrites both operands, returns x."""
    k = 1
    while k < x.shape[1]:
        x[:, k:] += a[:, k:] * x[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return x


def _plain_scan(s):
    case = s["case"]
    dt = s["u"].dtype
    u, z, A, D = s["u"].float(), s["z"].float(), s["A"], s["D"]
    Bm, Cm = s["Bm"].float()[:, :, None, :], s["Cm"].float()[:, :, None, :]
    B, T, C = u.shape
    mask = _inside(s["lengths"], T, u)
    raw = s["delta"].float() + s["delta_bias"]
    step = _masked(torch.clamp_min(raw, 0.0) + torch.log1p(torch.exp(-raw.abs())), mask)
    a = torch.exp(step[..., None] * A)
    x = (step * u)[..., None] * Bm
    if s["state_in"] is not None:
        x[:, 0] += a[:, 0] * s["state_in"]
    h = _linear_recurrence(a.clone() if case["train"] else a, x)
    inner = (h * Cm).sum(-1) + D * u
    gate = z * _sigmoid(z)
    out = {"y": _masked(inner * gate, mask).to(dt)}
    if case["state"]:
        out["state_out"] = h[:, -1].clone()
    if case["train"]:
        dy = _masked(s["dy"].float(), mask)
        out["dz"] = (dy * inner * _silu_slope(z)).to(dt)
        dinner = dy * gate
        g = dinner[..., None] * Cm
        if s["d_state_out"] is not None:
            g[:, -1] += s["d_state_out"]
        after = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1).flip(1)
        g = _linear_recurrence(after, g.flip(1)).flip(1)
        del after
        out["dC"] = (h * dinner[..., None]).sum(2).to(dt)
        out["dB"] = (g * (step * u)[..., None]).sum(2).to(dt)
        first = torch.zeros_like(h[:, :1]) if s["state_in"] is None else s["state_in"][:, None]
        gah = a.mul_(g)                                               # g a h_{t-1}: the gradient at the exponent
        if s["d_state_out"] is not None:
            out["d_state_in"] = gah[:, 0].clone()
        gah = gah.mul_(torch.cat((first, h[:, :-1]), 1))
        gb = (g * Bm).sum(-1)
        out["du"] = _masked(gb * step + D * dinner, mask).to(dt)
        draw_ = _masked((gb * u + (gah * A).sum(-1)) * _sigmoid(raw), mask)
        out["ddelta"] = draw_.to(dt)
        out["dA"] = (gah * step[..., None]).sum((0, 1), dtype=torch.float64).float()
        out["dD"] = (dinner * u).sum((0, 1), dtype=torch.float64).float()
        out["d_delta_bias"] = draw_.sum((0, 1), dtype=torch.float64).float()
    return out


# ------------------------------------------------------------------------------------- the framework's operators
def _own_gemm(s):
    from slam_amd.network import sequence_ops as ops
    case = s["case"]
    M, N, K = case["M"], case["N"], case["K"]
    if case["quantize"]:
        a8 = torch.empty(M, K, dtype=FP8, device="cuda")
        sa = torch.empty(M, -(-K // 128), dtype=torch.float32, device="cuda")
        ops.quantize_fp8(s["a"], a8, sa)
    else:
        a8, sa = s["a8"], s["a_scales"]
    out = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    ops.gemm_nt_fp8(a8, sa, s["b8"], s["b_scales"], out)
    return {"out": out}


def _own_norm(s):
    from slam_amd.network import sequence_ops as ops
    case, x = s["case"], s["x"]
    rows, C = x.shape
    out = {}
    total = x
    if case["residual"]:
        total = out["sum"] = torch.empty_like(x)
    if case["fp8"]:
        out["y8"] = torch.empty(rows, C, dtype=FP8, device=x.device)
        out["scales"] = torch.empty(rows, -(-C // 128), dtype=torch.float32, device=x.device)
    else:
        out["y"] = torch.empty_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if case["train"] else None
    ops.rms_norm_fwd(x, s["weight"], EPS, y=out.get("y"), residual=s["residual"], sum_out=out.get("sum"), y8=out.get("y8"),
                     scales=out.get("scales"), rstd=rstd)
    if case["train"]:
        out["dx"] = torch.empty_like(x)
        out["dweight"] = torch.empty_like(s["weight"])
        ops.rms_norm_bwd(s["dy"], total, s["weight"], rstd, out["dx"], out["dweight"], d_sum=s["d_sum"])
    return out


def _own_conv(s):
    from slam_amd.network import sequence_ops as ops
    case, x = s["case"], s["x"]
    B, T, C = x.shape
    new = lambda *shape: torch.empty(*shape, dtype=x.dtype, device=x.device)  # noqa: E731
    out = {"y": new(B, T, C), "state_out": new(B, case["K"] - 1, C)}
    ops.causal_conv_fwd(x, s["weight"], s["bias"], out["y"], state_in=s["state_in"], state_out=out["state_out"], lengths=s["lengths"])
    if case["train"]:
        out["dx"] = new(B, T, C)
        out["dweight"], out["dbias"] = torch.empty_like(s["weight"]), torch.empty_like(s["bias"])
        if case["state"]:
            out["d_state_in"] = new(B, case["K"] - 1, C)
        ops.causal_conv_bwd(s["dy"], x, s["weight"], s["bias"], out["dx"], out["dweight"], out["dbias"], state_in=s["state_in"],
                            d_state_in=out.get("d_state_in"), d_state_out=s["d_state_out"], lengths=s["lengths"])
    return out


def _own_scan(s):
    from slam_amd.network import sequence_ops as ops
    case, u = s["case"], s["u"]
    B, T, C = u.shape
    N = case["N"]
    new = lambda *shape, dtype=u.dtype: torch.empty(*shape, dtype=dtype, device=u.device)  # noqa: E731
    out = {"y": new(B, T, C)}
    if case["state"]:
        out["state_out"] = new(B, C, N, dtype=torch.float32)
    kept = ops.selective_scan_kept_states(B, T, C, N, u.device) if case["train"] else None
    ops.selective_scan_fwd(u, s["delta"], s["A"], s["Bm"], s["Cm"], out["y"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                           state_in=s["state_in"], state_out=out.get("state_out"), kept_states=kept, lengths=s["lengths"])
    if case["train"]:
        for k in ("du", "ddelta", "dz"):
            out[k] = new(B, T, C)
        for k in ("dB", "dC"):
            out[k] = new(B, T, N)
        for k, p in (("dA", "A"), ("dD", "D"), ("d_delta_bias", "delta_bias")):
            out[k] = torch.empty_like(s[p])
        if case["state"]:
            out["d_state_in"] = new(B, C, N, dtype=torch.float32)
        ops.selective_scan_bwd(s["dy"], u, s["delta"], s["A"], s["Bm"], s["Cm"], kept, out["du"], out["ddelta"], out["dA"], out["dB"],
                               out["dC"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"], dD=out["dD"], dz=out["dz"],
                               d_delta_bias=out["d_delta_bias"], d_state_in=out.get("d_state_in"), d_state_out=s["d_state_out"],
                               lengths=s["lengths"])
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"gemm": _own_gemm, "norm": _own_norm, "conv": _own_conv, "scan": _own_scan}[op](state)
    return {"gemm": _plain_gemm, "norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan}[op](state)


# ------------------------------------------------------------------------------------------------------- the work
def work(case):
    e = 2 if case.get("dtype", "bf16") == "bf16" else 4
    if case["op"] == "conv":
        n, K = case["B"] * case["T"] * case["C"], case["K"]
        carried = case["B"] * case["C"] * (K - 1) * e * (2 if case["state"] else 1)
        size, flops = 2 * n * e + carried + case["C"] * (K + 1) * 4, n * (2 * K + 5)
        if case["train"]:   # x and y, then dy, x and dx
            size += 3 * n * e + case["C"] * (K + 1) * 8
            flops += n * (6 * K + 12)
        return {"bytes": size, "flops": flops}
    if case["op"] == "scan":
        B, T, C, N = case["B"], case["T"], case["C"], case["N"]
        n = B * T * C
        carried = (8 if case["state"] else 0) * B * C * N
        size = 4 * n * e + 2 * B * T * N * e + carried + C * (N + 2) * 4   # u, delta, z, y; B, C
        flops = n * (6 * N + 20)
        if case["train"]:   # dy, u, delta, z, du, ddelta, dz; B, C, dB, dC
            size += 7 * n * e + 4 * B * T * N * e + carried + C * (N + 2) * 8
            flops += n * (20 * N + 40)
        return {"bytes": size, "flops": flops}
    if case["op"] == "norm":
        n = case["rows"] * case["C"]
        size = n * e * (3 if case["residual"] else 1) + case["C"] * 4
        size += n + 4 * case["rows"] * -(-case["C"] // 128) if case["fp8"] else n * e
        flops = 6 * n
        if case["train"]:   # dy, the sum, its gradient, dx
            size += n * e * (4 if case["residual"] else 3) + case["C"] * 8
            flops += 10 * n
        return {"bytes": size, "flops": flops}
    M, N, K = case["M"], case["N"], case["K"]
    kb = -(-K // 128)
    size = M * K * (2 if case["quantize"] else 1) + (0 if case["quantize"] else 4 * M * kb) + N * K + 4 * -(-N // 128) * kb
    return {"bytes": size + M * N * 2, "flops": 2 * M * N * K}


# ------------------------------------------------------------------------------------------------- 64-bit values
def _round_e4m3(v):
    """float64 -> the nearest value of 1 sign, 4 exponent, 3 mantissa bits (ties to even), saturating."""
    _, e = torch.frexp(v)
    quantum = torch.exp2((e.double() - 1.0).clamp_min(-6.0) - 3.0)
    return (torch.round(v / quantum) * quantum).clamp(-FP8_MAX, FP8_MAX)


def _exact_gemm(s):
    K, N = s["case"]["K"], s["case"]["N"]
    col = torch.arange(K, device="cuda") // 128
    if s["case"]["quantize"]:
        v = s["a"].double()
        top = torch.zeros(v.shape[0], -(-K // 128), dtype=torch.float64, device="cuda")
        top = top.scatter_reduce(1, col[None].expand_as(v), v.abs(), "amax")
        # the format's scale is a float32, and so is the quotient that is rounded to 8 bits: quotients halfway between two
        # of its values are common (three or four bits of a bfloat16), and to even is what they round to
        sa = torch.clamp_min(top / FP8_MAX, MIN_SCALE).float().double()[:, col]
        a = _round_e4m3((v / sa).float().double()) * sa
    else:
        a = s["a8"].double() * s["a_scales"].double()[:, col]
    b = s["b8"].double() * s["b_scales"].double()[torch.arange(N, device="cuda") // 128][:, col]
    return {"out": torch.mm(a, b.t().contiguous())}


def _exact_norm(s):
    case = s["case"]
    v = s["x"].double()
    out = {}
    if case["residual"]:
        out["sum"] = v + s["residual"].double()
        v = (s["x"].float() + s["residual"].float()).to(s["x"].dtype).double()   # the norm is that of the rounded sum
    w = s["weight"].double()
    r = (v.square().sum(1) / v.shape[1] + EPS).rsqrt()[:, None]
    y = v * r * w
    if case["fp8"]:
        col = torch.arange(v.shape[1], device="cuda") // 128
        top = torch.zeros(v.shape[0], -(-v.shape[1] // 128), dtype=torch.float64, device="cuda")
        out["scales"] = torch.clamp_min(top.scatter_reduce(1, col[None].expand_as(y), y.abs(), "amax") / FP8_MAX, MIN_SCALE)
        out["y8"] = _round_e4m3(y / out["scales"][:, col])
    else:
        out["y"] = y
    if case["train"]:
        dy = s["dy"].double()
        dot = (dy * w * v).sum(1, keepdim=True)
        out["dx"] = dy * w * r - v * (r ** 3) * dot / v.shape[1]
        if s["d_sum"] is not None:
            out["dx"] = out["dx"] + s["d_sum"].double()
        out["dweight"] = (dy * v * r).sum(0)
    return out


def _exact_conv(s):
    case = s["case"]
    x, w = s["x"].double(), s["weight"].double()
    B, T, C = x.shape
    K = w.shape[1]
    n = s["lengths"].tolist() if s["lengths"] is not None else [T] * B
    z = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out = {"y": z(B, T, C), "state_out": z(B, K - 1, C)}
    if case["train"]:
        out |= {"dx": z(B, T, C), "dweight": z(C, K), "dbias": z(C)}
        if case["state"]:
            out["d_state_in"] = z(B, K - 1, C)
    for b in range(B):
        t = n[b]
        rows = z(K - 1 + t, C)
        if s["state_in"] is not None:
            rows[:K - 1] = s["state_in"][b].double()
        rows[K - 1:] = x[b, :t]
        pre = s["bias"].double().expand(t, C).clone()
        for k in range(K):
            pre += w[:, k] * rows[k:k + t]
        out["y"][b, :t] = pre * torch.sigmoid(pre)
        out["state_out"][b] = rows[t:]
        if case["train"]:
            sig = torch.sigmoid(pre)
            d = s["dy"][b, :t].double() * (sig + pre * sig * (1 - sig))
            drows = z(K - 1 + t, C)
            for k in range(K):
                drows[k:k + t] += w[:, k] * d
                out["dweight"][:, k] += (d * rows[k:k + t]).sum(0)
            out["dbias"] += d.sum(0)
            if s["d_state_out"] is not None:
                drows[t:] += s["d_state_out"][b].double()
                out["d_state_in"][b] = drows[:K - 1]
            out["dx"][b, :t] = drows[K - 1:]
    return out


def _exact_scan(s):
    case = s["case"]
    u, z, A, D = (s[k].double() for k in ("u", "z", "A", "D"))
    Bm, Cm = s["Bm"].double(), s["Cm"].double()
    B, T, C = u.shape
    N = A.shape[1]
    raw = s["delta"].double() + s["delta_bias"].double()
    step = torch.nn.functional.softplus(raw, threshold=40.0)
    live = torch.ones(B, T, dtype=torch.float64, device="cuda")
    if s["lengths"] is not None:
        live = (torch.arange(T, device="cuda")[None] < s["lengths"][:, None]).double()
    step = step * live[..., None]
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    h = new(B, C, N) if s["state_in"] is None else s["state_in"].double()
    kept = new(T + 1, B, C, N) if case["train"] else None
    inner = new(B, T, C)
    for t in range(T):
        if kept is not None:
            kept[t] = h
        h = torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * u[:, t])[..., None] * Bm[:, t, None, :]
        inner[:, t] = torch.matmul(h, Cm[:, t, :, None])[..., 0]
    inner += D * u
    sig = torch.sigmoid(z)
    out = {"y": inner * z * sig * live[..., None]}
    if case["state"]:
        out["state_out"] = h
    if not case["train"]:
        return out
    kept[T] = h
    dy = s["dy"].double() * live[..., None]
    out["dz"] = dy * inner * (sig + z * sig * (1 - sig))
    dinner = dy * z * sig
    g = new(B, C, N) if s["d_state_out"] is None else s["d_state_out"].double()
    out |= {"du": D * dinner, "dB": new(B, T, N), "dC": new(B, T, N), "dA": new(C, N)}
    dstep = new(B, T, C)
    for t in range(T - 1, -1, -1):
        g = g + dinner[:, t, :, None] * Cm[:, t, None, :]
        out["dC"][:, t] = torch.matmul(dinner[:, t, None, :], kept[t + 1])[:, 0]
        out["dB"][:, t] = torch.matmul((step[:, t] * u[:, t])[:, None, :], g)[:, 0]
        gb = torch.matmul(g, Bm[:, t, :, None])[..., 0]
        out["du"][:, t] += gb * step[:, t]
        g = torch.exp(step[:, t, :, None] * A) * g
        q = g * kept[t]
        dstep[:, t] = gb * u[:, t] + (q * A).sum(-1)
        out["dA"] += (q * step[:, t, :, None]).sum(0)
    if s["d_state_out"] is not None:
        out["d_state_in"] = g
    dstep = dstep * torch.sigmoid(raw) * live[..., None]
    out |= {"ddelta": dstep, "dD": (dinner * u).sum((0, 1)), "d_delta_bias": dstep.sum((0, 1))}
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"gemm": _exact_gemm, "norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](s)

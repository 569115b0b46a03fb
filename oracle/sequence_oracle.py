"""Float64 restatement of the sequence-layer operators (test infrastructure only): root-mean-square norm, 8-bit operands and
their product, causal convolution, selective scan.  Gradients come from autograd over these functions.

The second half states how far float32 arithmetic may be off: every *_error function returns, for each output, a bound on the
absolute error in units of u = 2^-24 (half a float32 step, relative), made of the magnitudes that the sums and products pass
through."""
import torch

F64 = torch.float64
FP8_MAX = 448.0
MIN_SCALE = 2.0 ** -100
U = 2.0 ** -24


def rms_norm(x, weight, eps, residual=None, dtype=torch.float32):
    """(s, y, rstd) of float64 operands; s is rounded to `dtype` as a constant shift, so that gradients pass through it."""
    s = x if residual is None else x + residual
    if residual is not None:
        s = s + (s.detach().float().to(dtype).double() - s.detach())
    rstd = 1.0 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, s * rstd * weight, rstd[..., 0]


def round_e4m3(v):
    _, e = torch.frexp(v)
    quantum = torch.exp2((e.double() - 1.0).clamp_min(-6.0) - 3.0)
    return (torch.round(v / quantum) * quantum).clamp(-FP8_MAX, FP8_MAX)


def row_scales(v):
    """Scales [rows, ceil(C / 128)] of float64 rows."""
    rows, C = v.shape
    kb = -(-C // 128)
    p = torch.nn.functional.pad(v, (0, kb * 128 - C)).view(rows, kb, 128)
    return (p.abs().amax(2) / FP8_MAX).clamp_min(MIN_SCALE)


def spread_scales(scales, C):
    return scales.repeat_interleave(128, -1)[..., :C]


def causal_conv(x, weight, bias, state_in=None, lengths=None, silu=True):
    """(y, state_out)."""
    B, T, C = x.shape
    K = weight.shape[1]
    n = [T] * B if lengths is None else [int(v) for v in lengths]
    ys, states = [], []
    for b in range(B):
        before = torch.zeros(K - 1, C, dtype=F64) if state_in is None else state_in[b]
        rows = torch.cat((before, x[b, :n[b]]))
        pre = bias.expand(n[b], C) if bias is not None else torch.zeros(n[b], C, dtype=F64)
        for k in range(K):
            pre = pre + weight[:, k] * rows[k:k + n[b]]
        y = pre * torch.sigmoid(pre) if silu else pre
        ys.append(torch.cat((y, torch.zeros(T - n[b], C, dtype=F64))))
        states.append(rows[n[b]:])
    return torch.stack(ys), torch.stack(states)


def selective_scan(u, delta, A, Bm, Cm, D=None, z=None, delta_bias=None, softplus=True, state_in=None, lengths=None):
    """(y, state_out)."""
    B, T, C = u.shape
    N = A.shape[1]
    n = [T] * B if lengths is None else [int(v) for v in lengths]
    ys, states = [], []
    for b in range(B):
        h = torch.zeros(C, N, dtype=F64) if state_in is None else state_in[b]
        rows = []
        for t in range(n[b]):
            dt = delta[b, t] if delta_bias is None else delta[b, t] + delta_bias
            if softplus:
                dt = torch.clamp_min(dt, 0) + torch.log1p(torch.exp(-dt.abs()))
            h = torch.exp(dt[:, None] * A) * h + (dt * u[b, t])[:, None] * Bm[b, t]
            y = h @ Cm[b, t]
            if D is not None:
                y = y + D * u[b, t]
            if z is not None:
                y = y * z[b, t] * torch.sigmoid(z[b, t])
            rows.append(y)
        rows += [torch.zeros(C, dtype=F64)] * (T - n[b])
        ys.append(torch.stack(rows) if rows else torch.zeros(0, C, dtype=F64))
        states.append(h)
    return torch.stack(ys), torch.stack(states)


# ------------------------------------------------------------------------------------------------------ error bounds
def _silu_parts(pre, silu):
    """(|silu'| bound, silu' error a unit of pre, factor of the function's own evaluation error)."""
    p = torch.sigmoid(pre)
    if not silu:
        one = torch.ones_like(pre)
        return pre, one, one * 0
    return pre * p, p * (1 + pre * (1 - p)), pre.abs()


def causal_conv_error(x, weight, bias, dy, state_in=None, d_state_out=None, lengths=None, silu=True):
    """Bounds in units of U for y, dx, dweight, dbias, d_state_in.

    pre is K + 1 terms summed in float32: (K + 1) U of the terms' magnitudes S.  silu passes that on with a slope of at most 1.1
    and adds its own error: exp2 of a rounded argument is off by (2 |pre| + 4) U relative, the sum, the reciprocal and the product
    by 6 U more.  The slope of silu' is at most 0.5; evaluating silu' (at most 1.1) costs (2 |pre| + 16) U.  Sums over rows are
    sequential over at most 64 rows, then over the runs of a workgroup and the groups: 400 terms in a row is never reached."""
    B, T, C = x.shape
    K = weight.shape[1]
    n = [T] * B if lengths is None else [int(v) for v in lengths]
    out = dict(y=torch.zeros(B, T, C, dtype=F64), dx=torch.zeros(B, T, C, dtype=F64), dweight=torch.zeros(C, K, dtype=F64),
               dbias=torch.zeros(C, dtype=F64), d_state_in=torch.zeros(B, K - 1, C, dtype=F64))
    for b in range(B):
        before = torch.zeros(K - 1, C, dtype=F64) if state_in is None else state_in[b]
        rows = torch.cat((before, x[b, :n[b]]))
        pre = bias.expand(n[b], C) if bias is not None else torch.zeros(n[b], C, dtype=F64)
        S = pre.abs()
        for k in range(K):
            pre = pre + weight[:, k] * rows[k:k + n[b]]
            S = S + (weight[:, k] * rows[k:k + n[b]]).abs()
        value, slope, far = _silu_parts(pre, silu)
        out["y"][b, :n[b]] = 1.1 * (K + 1) * S + value.abs() * (2 * far + 10) * (1 if silu else 0)
        d = (dy[b, :n[b]] * slope).abs()
        err = dy[b, :n[b]].abs() * ((0.5 * (K + 1) * S + 1.1 * (2 * far + 16)) if silu else torch.zeros_like(S)) + d
        drows = torch.zeros(K - 1 + n[b], C, dtype=F64)
        for k in range(K):
            drows[k:k + n[b]] += weight[:, k].abs() * (err + (K + 2) * d)
            out["dweight"][:, k] += ((err + 400 * d) * rows[k:k + n[b]].abs()).sum(0)
        out["dbias"] += (err + 400 * d).sum(0)
        if d_state_out is not None:
            drows[n[b]:] += 2 * d_state_out[b].abs()
        out["d_state_in"][b] = drows[:K - 1]
        out["dx"][b, :n[b]] = drows[K - 1:]
    return out


def selective_scan_error(u, delta, A, Bm, Cm, dy, D=None, z=None, delta_bias=None, softplus=True, state_in=None, d_state_out=None,
                         lengths=None):
    """Bounds in units of U for y, state_out and all gradients.

    A relative error in dt of 16 U (the sum with the bias, exp2 of a rounded argument, log2, the sums of softplus; |delta +
    bias| is below 8 in the tests) plus the bias sum's own U |delta| |slope| / dt, a decay's of |dt A| (that + 3) + 4, an input
    term's of that + 3.  With those a state's error obeys the state's own recurrence over magnitudes, E_t = a E_{t-1} +
    (errors of this step's terms); where a sequence is cut, the joining of chunks forms the same products in another order, which
    the sums of dt (at most T terms, (T / 16 + 24) U) make at most T / 16 + 24 worse: `cut`.  Gradients likewise, from behind."""
    B, T, C = u.shape
    N = A.shape[1]
    n = [T] * B if lengths is None else [int(v) for v in lengths]
    zero = lambda *s: torch.zeros(*s, dtype=F64)  # noqa: E731
    out = dict(y=zero(B, T, C), du=zero(B, T, C), ddelta=zero(B, T, C), dz=zero(B, T, C), dB=zero(B, T, N), dC=zero(B, T, N),
               dA=zero(C, N), dD=zero(C), d_delta_bias=zero(C), d_state_in=zero(B, C, N), state_out=zero(B, C, N))
    Dm = zero(C) if D is None else D.abs()
    cut = T / 16 + 24
    for b in range(B):
        h = zero(C, N) if state_in is None else state_in[b].abs()
        E = zero(C, N)
        hs, Es, steps = [h], [E], []
        for t in range(n[b]):
            raw = delta[b, t] if delta_bias is None else delta[b, t] + delta_bias
            mag = delta[b, t].abs() + (0 if delta_bias is None else delta_bias.abs())
            dt, slope = raw, torch.ones_like(raw)
            if softplus:
                dt, slope = torch.clamp_min(raw, 0) + torch.log1p(torch.exp(-raw.abs())), torch.sigmoid(raw)
            rdt = 16 + (mag * slope / dt.abs().clamp_min(1e-300) if delta_bias is not None else torch.zeros_like(raw))
            decay = torch.exp(dt[:, None] * A)
            ra = (dt[:, None] * A).abs() * (rdt[:, None] + 3 + cut) + 4
            x = (dt * u[b, t]).abs()[:, None] * Bm[b, t].abs()
            rx = rdt[:, None] + 3
            E = decay * E + decay * h * (ra + 2) + x * (rx + 2)
            h = decay * h + x
            hs.append(h), Es.append(E), steps.append((dt, slope, rdt, decay, ra, x, rx))
            Ca = Cm[b, t].abs()
            inner = h @ Ca + Dm * u[b, t].abs()
            ei = E @ Ca + (N + 4) * inner
            gate, rgate = torch.ones(C, dtype=F64), 0.0
            if z is not None:
                zz = z[b, t]
                gate, rgate = (zz * torch.sigmoid(zz)).abs(), 2 * zz.abs() + 10
                slope_z = torch.sigmoid(zz) * (1 + zz * (1 - torch.sigmoid(zz)))
                out["dz"][b, t] = dy[b, t].abs() * (1.1 * (2 * zz.abs() + 16) * inner + slope_z.abs() * ei + 4 * inner)
            out["y"][b, t] = gate * (ei + inner * (rgate + 2))
        out["state_out"][b] = E
        g = zero(C, N) if d_state_out is None else d_state_out[b].abs()
        Eg = zero(C, N)
        for t in range(n[b] - 1, -1, -1):
            dt, slope, rdt, decay, ra, x, rx = steps[t]
            e, re = dy[b, t].abs(), 0.0
            if z is not None:
                zz = z[b, t]
                e, re = e * (zz * torch.sigmoid(zz)).abs(), 2 * zz.abs() + 11
            Ba, Ca, ua = Bm[b, t].abs(), Cm[b, t].abs(), u[b, t].abs()
            c = e[:, None] * Ca
            Eg = Eg + c * (torch.as_tensor(re, dtype=F64).reshape(-1, 1) + 2) + g
            g = g + c
            w = (dt * u[b, t]).abs()
            out["dC"][b, t] = (e[:, None] * (Es[t + 1] + hs[t + 1] * (torch.as_tensor(re, dtype=F64).reshape(-1, 1) + 40 + C / 64))).sum(0)
            out["dB"][b, t] = (w[:, None] * (Eg + g * (rx + 40 + C / 64))).sum(0)
            gb, egb = g @ Ba, Eg @ Ba
            out["du"][b, t] = dt.abs() * (egb + gb * (N + 6 + rdt)) + Dm * e * (re + 4) + dt.abs() * gb
            q = decay * g * hs[t]
            eq = decay * (Eg * hs[t] + g * Es[t]) + q * (ra + 3)
            s, es = (q * A.abs()).sum(1), (eq * A.abs()).sum(1)
            dd = ua * (egb + gb * (N + 4)) + es + s * (N + 6)
            out["ddelta"][b, t] = slope * (dd + (ua * gb + s) * 12) + 0.25 * (ua * gb + s) * (mag_of(delta, delta_bias, b, t))
            out["dA"] += eq * dt.abs()[:, None] + q * dt.abs()[:, None] * (rdt[:, None] + 2 + 400 + T)
            out["dD"] += e * ua * (re + 400 + T)
            out["d_delta_bias"] += out["ddelta"][b, t] + slope * (ua * gb + s) * (400 + T)
            Eg = decay * Eg + decay * g * (ra + 2)
            g = decay * g
        out["d_state_in"][b] = Eg
    return out


def mag_of(delta, delta_bias, b, t):
    return delta[b, t].abs() + (0 if delta_bias is None else delta_bias.abs())

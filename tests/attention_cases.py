"""64-bit forms of the frame norm, rotary positions and attention with element-wise error bounds, shared by their tests.

Bounds.  u is half a step of the result's type (2^-24 fp32, 2^-8 bf16), f = 2^-24 the rounding of the fp32 arithmetic in
between.  A sum of n terms in fp32 is taken to be off by 4 sqrt(n) f of the sum of magnitudes (roundings of either sign), a
handful of dependent operations by 32 f."""
import math

import torch

F = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def frame_norm(x, gamma, beta, eps, dy=None):
    """-> (y, dx, dgamma, dbeta), (their bounds); x, dy (R, C) in their own types, everything else in 64 bits."""
    u = HALF_STEP[x.dtype]
    up = HALF_STEP[gamma.dtype]
    x64, g, b = x.double(), gamma.double(), beta.double()
    R, C = x64.shape
    mean = x64.mean(1, keepdim=True)
    var = ((x64 - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x64 - mean) * rstd
    y = xh * g + b
    # xhat: a difference of values up to max|x| (rounded once after the mean is refined), sums of C terms behind rstd
    lift = (x64.abs().amax(1, keepdim=True) * rstd)
    exh = F * (4 * lift + (32 + 4 * math.sqrt(C)) * xh.abs())
    out, tol = [y], [exh * g.abs() + 4 * F * (xh * g).abs() + 4 * F * b.abs() + u * y.abs()]
    if dy is not None:
        d = dy.double()
        v = d * g
        a, c = v.mean(1, keepdim=True), (v * xh).mean(1, keepdim=True)
        dx = rstd * (v - a - xh * c)
        es = 4 * math.sqrt(C) * F
        ea = es * v.abs().mean(1, keepdim=True)
        ec = (v.abs() * exh).mean(1, keepdim=True) + es * (v * xh).abs().mean(1, keepdim=True)
        edx = rstd * (ea + exh * c.abs() + xh.abs() * ec + 32 * F * (v.abs() + a.abs() + (xh * c).abs()))
        er = 4 * math.sqrt(R) * F + 32 * F
        dg, db = (d * xh).sum(0), d.sum(0)
        out += [dx, dg, db]
        tol += [edx + u * dx.abs(), (d.abs() * exh).sum(0) + er * (d * xh).abs().sum(0) + up * dg.abs(),
                er * d.abs().sum(0) + up * db.abs()]
    return out, tol


def rotate(x, turns, positions, interleaved=False, magnitude=1.0, inverse=False):
    """x (B, T, H, D), positions (T,) or (B, T) -> y, bound."""
    u = HALF_STEP[x.dtype]
    n = turns.numel()
    angle = torch.frac(positions.double()[..., None] * turns.double()) * (2 * math.pi)
    if angle.dim() == 2:
        angle = angle[None]
    c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
    if inverse:
        s = -s
    x64 = x.double()
    ia = torch.arange(n) * 2 if interleaved else torch.arange(n)
    ib = ia + 1 if interleaved else ia + n
    a, b = x64[..., ia], x64[..., ib]
    y, e = x64.clone(), torch.zeros_like(x64)
    y[..., ia], y[..., ib] = magnitude * (a * c - b * s), magnitude * (a * s + b * c)
    # sine and cosine: argument (remainder and its scaling), the sum's rounding, the factor: 8 f; two products and a sum
    w = magnitude * 12 * F * (a.abs() + b.abs())
    e[..., ia], e[..., ib] = w, w
    rotated = torch.zeros_like(x64, dtype=torch.bool)
    rotated[..., ia] = rotated[..., ib] = True
    return y, torch.where(rotated, e + u * y.abs(), e)


def visible(B, Tq, Tk, lengths, causal):
    i, j = torch.arange(Tq)[:, None], torch.arange(Tk)[None, :]
    v = torch.ones((B, Tq, Tk), dtype=torch.bool)
    if causal:
        v &= j <= i + Tk - Tq
    if lengths is not None:
        v &= j < lengths.cpu().long()[:, None, None]
    return v


def attention(q, k, v, lengths=None, causal=False, scale=None, do=None):
    """CPU tensors (B, Tq, H, D), (B, Tk, Hk, D) -> [o, dq, dk, dv], [bounds]."""
    u = HALF_STEP[q.dtype]
    ur = u if q.dtype == torch.bfloat16 else 2.0 ** -22       # probabilities and score gradients on their way into a product
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    G = H // Hk
    see = visible(B, Tq, Tk, lengths, causal)[:, None]
    if lengths is not None:                                   # what lies behind a length is not part of the formula
        dead = torch.arange(Tk)[None, :] >= lengths.cpu().long()[:, None]
        k = k.masked_fill(dead[:, :, None, None], 0)
        v = v.masked_fill(dead[:, :, None, None], 0)
    Q = q.double().transpose(1, 2)
    K = k.double().transpose(1, 2).repeat_interleave(G, 1)
    V = v.double().transpose(1, 2).repeat_interleave(G, 1)
    Kt, Vt = K.transpose(2, 3).contiguous(), V.transpose(2, 3).contiguous()
    s = (Q @ Kt * scale).masked_fill(~see, -math.inf)
    m = s.amax(3, keepdim=True) if Tk else torch.zeros((B, H, Tq, 1), dtype=torch.float64)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    l = p.sum(3, keepdim=True)
    P = p / torch.where(l == 0, torch.ones_like(l), l)
    o = P @ V
    # a score is off by its product's rounding, a probability relatively by the score's error, twice (its own and the sum's)
    es = F * (4 * math.sqrt(D) + 8) * scale * (Q.abs() @ Kt.abs()).masked_fill(~see, 0)
    es = es.amax(3, keepdim=True) if Tk else torch.zeros((B, H, Tq, 1), dtype=torch.float64)
    mag = (s.masked_fill(~see, 0).abs().amax(3, keepdim=True) if Tk else es) * 4 * F
    e = 2 * (es + mag) + F * (4 * math.sqrt(max(Tk, 1)) + 32)
    to = (ur + e) * (P @ V.abs()) + u * o.abs()
    out, tol = [o.transpose(1, 2)], [to.transpose(1, 2)]
    if do is None:
        return out, tol
    dO = do.double().transpose(1, 2)

    def folded(t):                                            # heads of a group add up
        return t.reshape(B, Hk, G, Tk, D).sum(2).transpose(1, 2)

    Pt = P.transpose(2, 3).contiguous()
    dv, tdv = Pt @ dO, (P * (ur + 2 * e)).transpose(2, 3).contiguous() @ dO.abs()
    dP = (dO @ Vt).masked_fill(~see, 0)
    delta = (dO * o).sum(3, keepdim=True)
    ds = P * (dP - delta)
    edp = F * (4 * math.sqrt(D) + 8) * (dO.abs() @ Vt.abs())
    edelta = (dO.abs() * to).sum(3, keepdim=True) + F * (4 * math.sqrt(D) + 8) * (dO * o).abs().sum(3, keepdim=True)
    eds = P * (2 * e * (dP - delta).abs() + edp + edelta) + (ur + 8 * F) * ds.abs()
    acc = F * 4 * math.sqrt(max(Tk, Tq, 1))
    dq, tdq = ds @ K * scale, (eds + acc * ds.abs()) @ K.abs() * scale
    dst, edst = ds.transpose(2, 3).contiguous(), (eds + acc * ds.abs()).transpose(2, 3).contiguous()
    dk, tdk = dst @ Q * scale, edst @ Q.abs() * scale
    tdv = tdv + acc * (Pt @ dO.abs())
    dk, dv, tdk, tdv = folded(dk), folded(dv), folded(tdk), folded(tdv)
    out += [dq.transpose(1, 2), dk, dv]
    tol += [(tdq + u * dq.abs()).transpose(1, 2), tdk + u * dk.abs(), tdv + u * dv.abs()]
    return out, tol


def check(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, "{}: {} for {}".format(what, tuple(got.shape), tuple(want.shape))
    if got.numel() == 0:
        return
    err = (got - want).abs()
    tiny = 2.0 ** -100                                        # zeros have to be zeros, up to nothing a format can hold
    worst = (err / (bound + tiny)).nan_to_num(nan=math.inf).max().item()
    assert worst <= 1.0, "{}: {:.2f} times the bound (largest error {:.3e})".format(what, worst, err.max().item())

"""fp64 restatement of the gated linear recurrence and of the paged cache, and bounds for what fp32 arithmetic may make of them.

The recurrence (per channel; `first` marks a document's first token, where a = 0 and beta = 1):
    L = s sigmoid(ga)    a = exp(-L)    beta = sqrt(1 - a^2)    h_t = a_t h_{t-1} + beta_t sigmoid(gx_t) x_t    y_t = h_t

Bounds.  Every factor and sum of a kernel is off by a few units of fp32 (2^-24 relative, a rounding).  Going through T tokens, a term
passes at most T products, so a result is off by at most (T + 16) d times the same formula with absolute values (a "bar" below),
with d the units of one token: exponential 4, multiply-add 1, and what the decay gets from its exponent L, which is at most about 1
here: sigmoid 5, product 1: 16 units are enough.  The other factors are in the result once: a gate is off by 5 units and by as many
as its argument is large (60 at most here), beta by 20: less than the 16 d that are added.

These bounds grow with T whether or not the decays forget.  scan_errors and gradient_errors follow an error through the recurrence instead,
token by token, and see what is lost in long sequences too.
"""
import math

import torch

UNIT = 2.0 ** -24


def half_step(dtype):
    """The relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def gated_scan(x, gx, ga, s, h0=None, first=None, bar=False):
    """(y, hT) in fp64; bar: of absolute values."""
    B, T, C = x.shape
    h = torch.zeros(B, C, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    x, gx, ga, s = x.double(), gx.double(), ga.double(), s.double()
    if bar:
        x, h = x.abs(), h.abs()
    ys = []
    for t in range(T):
        L = s * sigmoid(ga[:, t])
        u = sigmoid(gx[:, t]) * x[:, t]
        grown = torch.exp(-L) * h + torch.sqrt(-torch.expm1(-2 * L)) * u
        h = grown if first is None else torch.where(first[:, t, None].bool(), u, grown)
        ys.append(h)
    return torch.stack(ys, 1), h


def gated_scan_gradients(x, gx, ga, s, h0, first, dy, dhT):
    """The gradients (dx, dgx, dga, ds, dh0) by their formulas, and the bars of the same."""
    B, T, C = x.shape
    h0 = torch.zeros(B, C, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    doc = torch.zeros(B, T, 1, dtype=torch.bool, device=x.device) if first is None else first.bool()[..., None]
    s = s.double()
    r, i, r_rest, i_rest = sigmoid(ga.double()), sigmoid(gx.double()), sigmoid(-ga.double()), sigmoid(-gx.double())
    L = s * r
    a = torch.exp(-L).masked_fill(doc, 0.0)
    beta = torch.sqrt(-torch.expm1(-2 * L)).masked_fill(doc, 1.0)
    slope = torch.where(doc | (beta == 0), 0.0, a * a / beta)
    out = []
    for bar in (False, True):
        size = torch.abs if bar else lambda v: v
        y, _ = gated_scan(x, gx, ga, s, h0, first, bar)
        before = torch.cat([size(h0)[:, None], y[:, :-1]], 1)
        G, e = torch.empty_like(y), size(dhT.double())
        for t in reversed(range(T)):
            G[:, t] = size(dy[:, t].double()) + e
            e = torch.where(doc[:, t], 0.0, a[:, t] * G[:, t])
        u = size(i * x.double())
        carried = torch.where(doc, 0.0, a * before)
        dL = G * (u * slope + carried if bar else u * slope - carried)
        out.append((G * beta * i, G * beta * u * i_rest, dL * L * r_rest, (dL * r).sum((0, 1)), e))
    return out


def scan_bound(T, bar, value, dtype):
    """What an output of the recurrence (two passes over T tokens for a gradient) may be off by."""
    return half_step(dtype) * value.abs() + (2 * T + 32) * 16 * UNIT * bar + 1e-35


def _units(x, gx, ga, s, first, dtype):
    """The factors of each token in fp64 and what a kernel may have them off by, in units relative to each (the decay: as a value).

    An exponential is off by 4 units (CUDA's expf by 2, the hardware's 2^x by 4) and, where its argument is multiplied by log2 e first (bf16), by as
    many as the argument is large.  A gate is the inverse (2 units; 4 of the product of two) of 1 + that, taken times the other gate's 1 + that: 8 more,
    and so is what it lacks of 1.  L is a product: 1.  Up to L = 1, 1 - a = q is a polynomial (3 units) of L and a its difference from 1 (1 unit of
    a); beyond, a is an exponential.  v = 1 - a^2 = q (2 - q) is off by no more than q and 3, 1 / beta by half of that and 4 for the root, beta = v / beta
    by one more."""
    x, gx, ga, s = (t.double() for t in (x, gx, ga, s))
    doc = torch.zeros(*x.shape[:2], 1, dtype=torch.bool, device=x.device) if first is None else first.bool()[..., None]
    r, i = sigmoid(ga), sigmoid(gx)
    wide = 1.0 if dtype == torch.bfloat16 else 0.0
    er, ei = 14 + wide * ga.abs(), 14 + wide * gx.abs()
    L = s * r
    eL = er + 1
    a, q = torch.exp(-L), -torch.expm1(-L)
    ea = a * L * eL + torch.where(L <= 1, 3 * q + a, a * (L + 5))
    ev = eL + 6
    beta = torch.sqrt(-torch.expm1(-2 * L))
    eb, einv = ev / 2 + 6, ev / 2 + 5
    zero = torch.zeros_like(a)
    a, ea, beta, eb = (torch.where(doc, v, t) for v, t in ((0.0, a), (zero, ea), (1.0, beta), (zero, eb)))
    return doc, x, r, i, er, ei, L, eL, a, ea, beta, eb, einv


def _forward_errors(f, h0):
    """Per token: h before it and behind it, their bars and errors (in units).  A product with the decay and a sum are a unit each, twice: a kernel makes
    the state before a block of tokens from products of decays and walks the block from there."""
    doc, x, r, i, er, ei, L, eL, a, ea, beta, eb, einv = f
    B, T, C = x.shape
    h = torch.zeros(B, C, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    bar, off = h.abs(), torch.zeros_like(h)
    w = beta * i * x
    ew = (eb + ei + 2) * w.abs()
    outs = []
    for t in range(T):
        before = h, bar, off
        h = a[:, t] * h + w[:, t]
        new = a[:, t] * bar + w[:, t].abs()
        off = a[:, t] * off + (ea[:, t] + 2 * a[:, t]) * bar + ew[:, t] + 2 * new
        bar = new
        outs.append((*before, h, bar, off))
    return [torch.stack(o, 1) for o in zip(*outs)]


def scan_errors(x, gx, ga, s, h0=None, first=None, dtype=None):
    """(y, hT) in fp64 and what a kernel for tensors of `dtype` may have each off by."""
    dtype = dtype or x.dtype
    *_, h, _, off = _forward_errors(_units(x, gx, ga, s, first, dtype), h0)
    off = UNIT * off + 1e-35
    return (h, h[:, -1]), (off + half_step(dtype) * h.abs(), off[:, -1])


def gradient_errors(x, gx, ga, s, h0, first, dy, dhT, dtype=None):
    """What a kernel may have (dx, dgx, dga, ds, dh0) off by, with the same meaning: the errors of the gradient that comes into a token
    go back through the recurrence as those of the state go forward, and every product of a gradient is a unit."""
    dtype = dtype or x.dtype
    f = _units(x, gx, ga, s, first, dtype)
    doc, x, r, i, er, ei, L, eL, a, ea, beta, eb, einv = f
    B, T, C = x.shape
    hb, hbar, hoff = _forward_errors(f, h0)[:3]
    dy = dy.double()
    e = dhT.double()
    ebar, eoff = e.abs(), torch.zeros_like(e)
    Gs = []
    for t in reversed(range(T)):
        G, Gbar = dy[:, t] + e, dy[:, t].abs() + ebar
        Goff = eoff + 2 * Gbar
        e, ebar = a[:, t] * G, a[:, t] * Gbar
        eoff = a[:, t] * Goff + (ea[:, t] + 2 * a[:, t]) * Gbar + 2 * ebar
        Gs.append((G, Gbar, Goff, e, ebar, eoff))
    G, Gbar, Goff, eG, eGbar, eGoff = (torch.stack(o[::-1], 1) for o in zip(*Gs))
    i_rest, r_rest = sigmoid(-gx.double()), sigmoid(-ga.double())
    inv = torch.where(beta > 0, 1 / beta, 0.0)
    u = i * x
    dx, dx_off = G * beta * i, beta * i * Goff + (eb + ei + 3) * Gbar * beta * i
    dgx, dgx_off = dx * x * i_rest, (x * i_rest).abs() * dx_off + (ei + 4) * (Gbar * beta * u * i_rest).abs()
    part = (u * a * inv).abs()
    slope, slope_bar = u * a * inv - hb, part + hbar
    slope_off = (ei + einv + 4) * part + ea * (u * inv).abs() + hoff + slope_bar
    dL = torch.where(doc, 0.0, eG * slope)
    dL_bar = torch.where(doc, 0.0, eGbar * slope_bar)
    dL_off = torch.where(doc, 0.0, slope_bar * eGoff + eGbar * slope_off + eGbar * slope_bar)
    dga, dga_off = dL * L * r_rest, L * r_rest * (dL_off + (eL + er + 4) * dL_bar)
    # ds: each of eight warps sums its tokens, then they and the blocks that shared the tokens, then the sequences
    ds, ds_off = (dL * r).sum((0, 1)), (r * dL_off + er * r * dL_bar).sum((0, 1)) + (T / 8 + 8 * B + 40) * (r * dL_bar).sum((0, 1))
    step = half_step(dtype)
    offs = [UNIT * o + step * v.abs() + 1e-35 for o, v in ((dx_off, dx), (dgx_off, dgx), (dga_off, dga))]
    return (dx, dgx, dga, ds, e), (*offs, UNIT * ds_off + 1e-35, UNIT * eoff + 1e-35)


def rotated(x, position, inv_freq, interleaved, factor):
    """x (M, H, N) turned by its tokens' positions, in fp64."""
    R = 2 * inv_freq.numel()
    x = x.double()
    angle = (position.double()[:, None] * inv_freq.double())[:, None]
    c, s = factor * torch.cos(angle), factor * torch.sin(angle)
    out = x.clone()
    at = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    out[..., at[0]] = x[..., at[0]] * c - x[..., at[1]] * s
    out[..., at[1]] = x[..., at[0]] * s + x[..., at[1]] * c
    return out


def attention(q, k, v, scale, cap=0.0, slopes=None, window=0):
    """One query per head over the tokens of one sequence: q (Hq, N), k, v (len, Hkv, N) -> out (Hq, N), lse (Hq), and the bound of
    each for fp32 arithmetic.

    A score is a sum of N products: N + 2 units of the sum of their absolute values (the tensor core drops what does not fit instead
    of rounding: twice that), and 8 units of its own size for the cap and the bias.  A weight is off by as much as its
    exponent, twice (its own and the largest score), and 2^-22 relative where it is kept as three bf16 numbers; the sums over the
    tokens add 2^-20."""
    n, Hkv = k.shape[:2]
    Hq, N = q.shape
    low = max(0, n - window) if window else 0
    q, k, v = q.double(), k[low:].double(), v[low:].double()
    if n - low <= 0:
        zero = torch.zeros(Hq, N, dtype=torch.float64, device=q.device)
        return zero, torch.full((Hq,), -math.inf, dtype=torch.float64, device=q.device), zero, zero[:, 0]
    k, v = k.repeat_interleave(Hq // Hkv, 1), v.repeat_interleave(Hq // Hkv, 1)
    z = torch.einsum("hn,thn->ht", q, k) * scale
    bar = torch.einsum("hn,thn->ht", q.abs(), k.abs()) * abs(scale)
    if 0 < cap < math.inf:
        z = cap * torch.tanh(z / cap)
    off = 2 * (N + 2) * UNIT * bar + 8 * UNIT * z.abs()
    if slopes is not None:
        bias = slopes.double()[:, None] * (torch.arange(low, n, device=q.device) - (n - 1))
        z = z + bias
        off = off + 4 * UNIT * bias.abs()
    off = torch.where(torch.isfinite(off), off, 0.0).amax(-1)
    m = z.amax(-1)
    w = torch.where(z == -math.inf, 0.0, torch.exp(z - m[:, None]))
    total = w.sum(-1)
    empty = (m == -math.inf)[:, None]
    p = torch.where(empty, 0.0, w / total[:, None])
    used = torch.where(w[..., None] == 0, 0.0, v.transpose(0, 1))   # a token without weight counts for nothing, whatever it holds
    out = torch.einsum("ht,htn->hn", p, used)
    lse = torch.where(empty[:, 0], -math.inf, m + torch.log(total))
    sizes = torch.einsum("ht,htn->hn", p, used.abs())
    return out, lse, (2 * off[:, None] + 2.0 ** -22 + 2.0 ** -20) * sizes, off + 2.0 ** -20 + 4 * UNIT * lse.abs()

"""CPU tier of the gated recurrence and the paged cache: the fp64 forms against autograd and torch, refusals that need no GPU, and the
arithmetic of the kernels' page lookup."""
import ctypes
import math
import random

import pytest
import torch

import rwkv_cuda_b200 as R
from oracle import mixer_oracle as M
from rwkv_cuda_b200 import _lib
from tests import helpers as Hh


def test_gradient_formulas_are_autograds():
    g = Hh.gen(1)
    B, T, C = 2, 23, 5
    leaves = [x.double().requires_grad_(True) for x in (Hh.randn(g, B, T, C), Hh.randn(g, B, T, C), Hh.randn(g, B, T, C), Hh.rand(g, C, lo=0.1, hi=2), Hh.randn(g, B, C))]
    first = Hh.rand(g, B, T) < 0.2
    dy, dhT = Hh.randn(g, B, T, C).double(), Hh.randn(g, B, C).double()
    want = torch.autograd.grad(M.gated_scan(*leaves, first), leaves, (dy, dhT))
    got, bars = M.gated_scan_gradients(*(x.detach() for x in leaves), first, dy, dhT)
    for a, b, bar in zip(got, want, bars):
        torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-12)
        assert (bar >= a.abs() * (1 - 1e-12)).all()


def test_bounds_that_follow_the_decays_see_lost_digits():
    """The formulas in fp32 stay within the bounds at any length; the same with one intermediate rounded to bf16, or with results rounded to it, do not."""
    g = Hh.gen(3)
    B, C = 2, 24
    s = -8 * torch.log(Hh.rand(g, C, lo=0.9, hi=0.999))
    for T in (60, 1500):
        x, gx, ga, dy = (Hh.randn(g, B, T, C) for _ in range(4))
        h0, dhT, first = Hh.randn(g, B, C), Hh.randn(g, B, C), Hh.rand(g, B, T) < 0.01
        (y64, hT64), (by, bhT) = M.scan_errors(x, gx, ga, s, h0, first)
        want, bounds = M.gradient_errors(x, gx, ga, s, h0, first, dy, dhT)
        for a, b in zip((y64, *want), (M.gated_scan(x, gx, ga, s, h0, first)[0], *M.gated_scan_gradients(x, gx, ga, s, h0, first, dy, dhT)[0])):
            torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-12)
        same, short = lambda v: v, lambda v: v.bfloat16().float()
        for lossy in (None, "a", "beta", "u", "h", "G"):
            on = lambda name: short if name == lossy else same
            doc = first[..., None]
            r, i = torch.sigmoid(ga), torch.sigmoid(gx)
            L = s * r
            a = on("a")(torch.exp(-L)).masked_fill(doc, 0.0)
            beta = on("beta")(torch.sqrt(-torch.expm1(-2 * L))).masked_fill(doc, 1.0)
            u = on("u")(i * x)
            h, ys = h0, []
            for t in range(T):
                h = on("h")(a[:, t] * h + beta[:, t] * u[:, t])
                ys.append(h)
            y = torch.stack(ys, 1)
            e, Gs = dhT, []
            for t in reversed(range(T)):
                Gs.append(on("G")(dy[:, t] + e))
                e = a[:, t] * Gs[-1]
            G = torch.stack(Gs[::-1], 1)
            before = torch.cat([h0[:, None], y[:, :-1]], 1)
            dL = (G * (u * torch.where(doc, 0.0, a * a / beta) - a * before)).masked_fill(doc, 0.0)
            got = (G * beta * i, G * beta * u * (1 - i), dL * L * (1 - r), (dL * r).sum((0, 1)), e)
            inside = [bool(((v.double() - w).abs() <= b).all()) for v, w, b in zip((y, h, *got), (y64, hT64, *want), (by, bhT, *bounds))]
            if lossy is None:
                assert all(inside), inside
                for v, w, b in zip((y, h, *got), (y64, hT64, *want), (by, bhT, *bounds)):
                    assert ((short(v).double() - w).abs() > b).any()
            else:
                assert not all(inside), lossy


def test_attention_form():
    g = Hh.gen(2)
    q, k, v = Hh.randn(g, 6, 16), Hh.randn(g, 50, 2, 16), Hh.randn(g, 50, 2, 16)
    out, lse, _, _ = M.attention(q, k, v, 0.25)
    want = torch.nn.functional.scaled_dot_product_attention(q.double()[:, None], k.double().transpose(0, 1).repeat_interleave(3, 0),
                                                            v.double().transpose(0, 1).repeat_interleave(3, 0))
    torch.testing.assert_close(out, want[:, 0])
    out, lse, _, _ = M.attention(q, k, v, 0.25, window=1)
    torch.testing.assert_close(out, v[-1].double().repeat_interleave(3, 0))
    out, lse, _, _ = M.attention(q, k[:0], v[:0], 0.25)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_division_by_multiplication():
    """n / d as the kernels take it: the high half of n * mul, plus n, shifted."""
    rng = random.Random(1)
    for d in [1, 2, 3, 5, 7, 16, 48, 255, 256, 257, 2 ** 16 + 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1] + [rng.randrange(1, 2 ** 31) for _ in range(200)]:
        shift = 0
        while (1 << shift) < d:
            shift += 1
        mul = ((((1 << shift) - d) << 32) // d + 1) & 0xffffffff
        for n in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1] + [rng.randrange(2 ** 31) for _ in range(50)]:
            if n < 2 ** 31:
                total = ((n * mul) >> 32) + n
                assert total < 2 ** 32 and total >> shift == n // d, (n, d)


def test_status_codes_without_launch():
    L = _lib.lib()
    one, err = ctypes.c_void_p(16), L.rwkvb200_last_error
    scan = lambda dtype=1, B=1, T=4, C=8, x=one, y=one: L.rwkvb200_gated_scan_forward(dtype, B, T, C, None, x, one, one, one, None, y, None, None, None)
    assert scan(T=0) == -1 and b"must be positive" in err()
    assert scan(dtype=3) == -1 and b"dtype" in err()
    assert scan(x=None) == -2 and b"'x'" in err()
    assert scan(y=None) == -2 and b"'y'" in err()
    assert scan(T=2 ** 31 - 1) == -1 and b"too long" in err()
    assert L.rwkvb200_gated_scan_backward(1, 1, 4, 8, one, one, one, one, None, None, one, None, None, one, one, one, one, one, None) == -2 and b"'saved'" in err()
    assert L.rwkvb200_gated_scan_saved_bytes(2, 65, 10) == 2 * 2 * 10 * 4 and L.rwkvb200_gated_scan_saved_bytes(0, 1, 1) == 0
    update = lambda B=2, pool=2, slots=one: L.rwkvb200_gated_scan_update(1, B, 8, pool, one, slots, one, one, one, one, one, None)
    assert update(pool=1, slots=None) == -1 and b"states for 2 rows" in err()
    assert update(pool=0) == -1 and update(B=70000, pool=70000) == -1
    append = lambda M=2, B=2, Hq=2, Hkv=1, N=64, R=64, pages=4, page=16, width=2, q=one, q_out=one, cu=None, inv=one: L.rwkvb200_paged_append(
        1, M, B, Hq, Hkv, N, R, pages, page, width, q, one, one, q_out, one, one, one, one, cu, inv, 0, 1.0, None)
    assert append(M=3) == -1 and b"need cu_seqlens" in err()
    assert append(N=200) == -4 and b"head size" in err()
    assert append(R=65) == -1 and append(R=66) == -1 and append(R=-2) == -1
    assert append(q_out=None) == -1 and b"come together" in err()
    assert append(inv=None) == -2 and append(Hq=0) == -1 and append(page=0) == -1
    assert append(width=2 ** 30, page=16) == -1 and b"2^31" in err()
    attend = lambda B=2, Hq=4, Hkv=2, N=64, page=16, width=2, cap=0.0, window=0, work=one, lengths=one: L.rwkvb200_paged_attention(
        1, B, Hq, Hkv, N, 4, page, width, one, one, one, one, lengths, 1.0, cap, window, None, one, None, work, None)
    assert attend(Hq=3) == -1 and b"not a multiple" in err()
    assert attend(N=129) == -4 and attend(cap=-1.0) == -1 and attend(window=-1) == -1 and attend(work=None) == -2 and attend(lengths=None) == -2
    assert attend(cap=float("nan")) == -1
    assert attend(width=2 ** 27, page=16) == -1 and b"2^31" in err()


def test_rows_too_wide_are_refused():
    """A row's bytes are counted in 32 bits, its channels in 31 with some to spare."""
    L = _lib.lib()
    one, err = ctypes.c_void_p(16), L.rwkvb200_last_error
    for dtype, C, T, word in ((0, 2 ** 30, 2, b"4 GiB"), (0, 2 ** 31 - 65537, 5, b"4 GiB"), (0, 2 ** 31 - 1, 1, b"too wide"), (1, 2 ** 31 - 1, 2, b"too wide"),
                              (1, 2 ** 31 - 65536, 2, b"too wide")):
        assert L.rwkvb200_gated_scan_forward(dtype, 1, T, C, None, one, one, one, one, None, one, None, None, None) == -1 and word in err()
        assert L.rwkvb200_gated_scan_backward(dtype, 1, T, C, one, one, one, one, None, one, one, None, None, one, one, one, one, one, None) == -1 and word in err()
    assert L.rwkvb200_gated_scan_update(0, 1, 2 ** 31 - 1, 1, one, None, one, one, one, one, one, None) == -1 and b"too wide" in err()


def test_saved_bytes_of_any_length():
    size = _lib.lib().rwkvb200_gated_scan_saved_bytes
    for T in (2 ** 31 - 1, 2 ** 31 - 64, 2 ** 31 - 63):
        assert size(3, T, 5) == 3 * -(-T // 64) * 5 * 4


def test_ops_refuse_cpu_tensors():
    x, s = torch.zeros(1, 4, 8), torch.zeros(8)
    with pytest.raises(RuntimeError, match="CUDA device"):
        R.ops.gated_scan_forward(x, x, x, s, x.clone())
    with pytest.raises(RuntimeError, match="CUDA device"):
        R.functions.GATED_SCAN.apply(x, x, x, s)
    with pytest.raises(RuntimeError, match="CUDA device"):
        R.ops.gated_scan_update(x[0], x[0], x[0], x[0], s, x[0].clone())
    p, i = torch.zeros(2, 1, 16, 8), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device"):
        R.ops.paged_append(x[:, :1], x[:, :1], p, p.clone(), i, i[0])
    with pytest.raises(RuntimeError, match="CUDA device"):
        R.ops.paged_attention(x[:, :1], p, p.clone(), i, i[0], x[:, :1].clone())

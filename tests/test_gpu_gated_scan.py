"""GPU tests of the gated linear recurrence against its fp64 form: lengths around the tokens of a warp (8, 16), of a round (64, 128)
and of several, channels that fill no warp, odd ones, documents, states in and out; gradients against the formulas and against
differences; values that are not finite; the single-token update and its slots."""
import pytest
import torch

from oracle import mixer_oracle as M
from tests import helpers as Hh

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def inputs(B, T, C, dtype, seed, docs=False, h0=True, scale=1.0):
    g = Hh.gen(seed)
    d = dict(x=Hh.randn(g, B, T, C).to(dtype), gx=Hh.randn(g, B, T, C).to(dtype), ga=(scale * Hh.randn(g, B, T, C)).to(dtype),
             s=-8 * torch.log(Hh.rand(g, C, lo=0.9, hi=0.999)), h0=Hh.randn(g, B, C) if h0 else None,
             first=Hh.rand(g, B, T) < 0.1 if docs else None, dy=Hh.randn(g, B, T, C).to(dtype), dhT=Hh.randn(g, B, C))
    return {n: t.cuda() if t is not None else None for n, t in d.items()}


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    assert (off <= bound).all(), f"{what}: off by {(off / bound).nan_to_num(nan=9e9).max().item():.3g} of the bound"


def forward(d):
    import rwkv_cuda_b200 as R
    y = torch.full_like(d["x"], float("nan"))
    hT = torch.full((d["x"].shape[0], d["x"].shape[2]), float("nan"), device="cuda")
    R.ops.gated_scan_forward(d["x"], d["gx"], d["ga"], d["s"], y, h0=d["h0"], hT=hT, first=d["first"])
    return y, hT


LEAVES = ("x", "gx", "ga", "s", "h0")


def train(d, retain=False):
    import rwkv_cuda_b200 as R
    leaves = [d[n].detach().requires_grad_(True) for n in LEAVES if d[n] is not None]
    out = R.functions.GATED_SCAN.apply(*leaves[:4], leaves[4] if d["h0"] is not None else None, d["first"])
    return out, torch.autograd.grad(out, leaves, (d["dy"], d["dhT"]), retain_graph=retain), leaves


def check(d):
    T, dtype = d["x"].shape[1], d["x"].dtype
    ins = [d[n] for n in ("x", "gx", "ga", "s", "h0", "first")]
    y64, hT64 = M.gated_scan(*ins)
    ybar, hbar = M.gated_scan(*ins, bar=True)
    for y, hT in (forward(d), train(d)[0]):
        within(y, y64, M.scan_bound(T, ybar, y64, dtype), "y")
        within(hT, hT64, M.scan_bound(T, hbar, hT64, F32), "hT")
    grads = train(d)[1]
    want, bars = M.gated_scan_gradients(*ins, d["dy"], d["dhT"])
    for got, w, bar, name in zip(grads, want, bars, ("dx", "dgx", "dga", "ds", "dh0")):
        within(got, w, M.scan_bound(T, bar, w, got.dtype), name)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,C", [(1, 1, 64), (2, 7, 64), (1, 8, 2), (1, 9, 66), (2, 16, 1), (1, 17, 63), (2, 63, 130), (3, 64, 64), (1, 65, 31),
                                   (1, 127, 96), (2, 128, 64), (1, 129, 65), (2, 300, 192), (1, 1025, 64)])
def test_lengths_and_channels(dtype, B, T, C):
    check(inputs(B, T, C, dtype, seed=T, docs=T % 2 == 0, h0=T % 3 != 0))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,C,docs", [(8, 300, 2048, False), (5, 129, 2046, True), (4, 200, 1024, True), (3, 333, 1500, False), (1, 2500, 192, True),
                                        (150, 1, 64, False), (160, 70, 8, True)])
def test_blocks_and_clusters(dtype, B, T, C, docs):
    """Launches of a block per channel tile (from 149 of them on) and of clusters of 2, 4 and 8 blocks, over several rounds."""
    check(inputs(B, T, C, dtype, seed=T, docs=docs))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,C,docs", [(1, 900, 1280, True), (1, 1000, 2304, False), (2, 700, 2880, True), (1, 1030, 3456, False), (4, 333, 833, False), (1, 400, 2560, True)])
def test_clusters_of_any_size(dtype, B, T, C, docs):
    """20 to 108 channel tiles: clusters of 2 to 7 blocks, whose last turn has rounds for some of them only."""
    check(inputs(B, T, C, dtype, seed=T, docs=docs))


def check_digits(d):
    """Forward, training forward and gradients within the bounds that follow errors through the decays."""
    ins = [d[n] for n in ("x", "gx", "ga", "s", "h0", "first")]
    want, bounds = M.scan_errors(*ins)
    for out in (forward(d), train(d)[0]):
        for got, w, b, name in zip(out, want, bounds, ("y", "hT")):
            within(got, w, b, name)
    grads = train(d)[1]
    want, bounds = M.gradient_errors(*ins, d["dy"], d["dhT"])
    for got, w, b, name in zip(grads, want, bounds, ("dx", "dgx", "dga", "ds", "dh0")):
        within(got, w, b, name)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,C,docs", [(1, 1, 64, False), (3, 17, 65, True), (2, 130, 192, False), (1, 1040, 768, True), (2, 1000, 130, False), (8, 512, 1024, True),
                                        (1, 1999, 1919, False), (1, 2500, 192, False), (1, 6000, 64, True), (150, 70, 64, False)])
@pytest.mark.parametrize("decays", ["usual", "large"])
def test_digits_in_long_sequences(dtype, B, T, C, docs, decays):
    """The bound does not grow with T where the state forgets: what rounds to fewer digits anywhere is seen after thousands of tokens too."""
    d = inputs(B, T, C, dtype, seed=T, docs=docs)
    if decays == "large":   # from 0 over the border of the two forms of the decay to exp(-30), all in every tile
        few = torch.tensor([0.0, -0.0, 1e-6, 0.1, 1.0 - 2 ** -24, 1.0, 1.0 + 2 ** -23, 1.7, 2.5, 8.0, 30.0], device="cuda")
        d["s"] = few[torch.arange(C, device="cuda") % len(few)].contiguous()
    check_digits(d)


@pytest.mark.parametrize("B,T,C", [(1, 34, 2 ** 26 + 8), (1, 2_200_003, 1000), (3, 1_100_001, 667)])
def test_more_elements_than_32_bits(B, T, C):
    """Tensors of 2.2e9 bf16 elements, wide or long: parts at their ends against fp64.  s of 0.5 and more forgets 1000 tokens to less than 1e-100."""
    import rwkv_cuda_b200 as R
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    g = torch.Generator("cuda").manual_seed(1)
    x, gx, ga, dy = (torch.empty(B, T, C, dtype=BF, device="cuda").normal_(generator=g) for _ in range(4))
    s = 0.5 + torch.rand(C, device="cuda", generator=g)
    leaves = [t.requires_grad_(True) for t in (x, gx, ga, s)]
    y, hT = R.functions.GATED_SCAN.apply(*leaves)
    dx, dgx, dga, _ = torch.autograd.grad(y, leaves, dy)
    n = min(T, 1200)
    for c in (slice(0, 40), slice(C - 40, C)):
        part = lambda t, at: t.detach()[:, at, c].contiguous()
        first, last = slice(0, n), slice(T - n, T)
        w, b = M.scan_errors(*(part(t, last) for t in (x, gx, ga)), s[c].detach())
        kept = slice(max(0, n - 100), n)
        within(part(y, last)[:, kept], w[0][:, kept], b[0][:, kept], "y")
        within(hT.detach()[:, c], w[1], b[1], "hT")
        for at, kept in ((first, slice(0, min(n, 100))), (last, slice(max(0, n - 100), n) if n < T else slice(0, n))):
            h0 = torch.zeros(B, 40, device="cuda")
            w, b = M.gradient_errors(*(part(t, at) for t in (x, gx, ga)), s[c].detach(), h0, None, part(dy, at), h0)
            for got, ww, bb, name in zip((dx, dgx, dga), w, b, ("dx", "dgx", "dga")):
                within(part(got, at)[:, kept], ww[:, kept], bb[:, kept], name)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [0, 1, 2])
def test_clusters_are_there_at_once(dtype, rows):
    """Whatever the rows' alignment (it decides how much shared memory a block takes): no cluster waits for another to end."""
    import ctypes
    from rwkv_cuda_b200 import _lib
    L, n = _lib.lib(), ctypes.c_int()
    sizes = set()
    for backward in (0, 1):
        for tiles in range(1, 301):
            K = L.rwkvb200_test_gated_scan_cluster(1 if dtype == BF else 0, 1, 8192, tiles * 64 - (rows == 2), rows, backward, ctypes.byref(n))
            assert 1 <= K <= 8 and (K == 1 or tiles <= n.value), f"{tiles} clusters of {K}, {n.value} at once"
            sizes.add(K)
    assert {1, 2, 4, 8} <= sizes   # (from one block for every two SMs to more blocks than there is room for)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("C", [64, 2048])
def test_large_decays(dtype, C):
    """s up to 30: beyond L = 1 the decays come from the exponential, down to exp(-30)."""
    d = inputs(1, 100, C, dtype, seed=1, docs=True)
    d["s"] = torch.linspace(0, 30, C, device="cuda")
    d["s"][:2] = 1.0 + torch.tensor([0.0, 1e-6])
    T = 100
    ins = [d[n] for n in ("x", "gx", "ga", "s", "h0", "first")]
    y64, _ = M.gated_scan(*ins)
    ybar, _ = M.gated_scan(*ins, bar=True)
    want, bars = M.gated_scan_gradients(*ins, d["dy"], d["dhT"])
    more = 1 + d["s"].max().item()   # a unit of the exponent counts as often as the exponent is large
    for got, w, bar, name in zip((forward(d)[0], *train(d)[1]), (y64, *want), (ybar, *bars), ("y", "dx", "dgx", "dga", "ds", "dh0")):
        within(got, w, M.scan_bound(T, bar * more, w, got.dtype), name)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("C", [64, 130])
def test_without_decay(dtype, C):
    """s = 0: the state stays, the gradient through beta is taken as 0, and ds is that of the decay alone."""
    d = inputs(1, 70, C, dtype, seed=1)
    d["s"] = torch.zeros(C, device="cuda")
    y, hT = forward(d)
    assert torch.equal(hT, d["h0"]) and torch.equal(y, d["h0"].to(dtype)[:, None].expand_as(y))
    check(d)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("C", [64, 130, 2048])
@pytest.mark.parametrize("beside", [None, 1.0, 1.5, 20.0, "gates"])
def test_without_decay_beside_others(dtype, C, beside):
    """s of -0.0 is s of 0.0, which -8 log(1) and a saturated logsigmoid make: alone, beside channels with larger s, and beside gates out of range; also
    token by token."""
    import rwkv_cuda_b200 as R
    d = inputs(2, 70, C, dtype, seed=3, docs=C == 130)
    none = torch.zeros(C, dtype=torch.bool, device="cuda")
    none[::3] = True
    s = torch.full((C,), 0.3 if beside in (None, "gates") else beside, device="cuda")
    if beside == "gates":
        d["ga"][:, 5:60:9, 1] = -50.0
    if beside is None:
        none[:] = True
    outs = []
    for zero in (0.0, -0.0):
        d["s"] = torch.where(none, zero, s)
        (y, hT), grads, _ = train(d)
        outs.append((y, hT, *grads, *forward(d)))
    assert torch.signbit(d["s"][0])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    if d["first"] is None:
        assert torch.equal(outs[1][1][:, none], d["h0"][:, none])
        assert torch.equal(outs[1][0][..., none], d["h0"].to(dtype)[:, None, none].expand(-1, 70, -1))
    ins = [d[n] for n in ("x", "gx", "ga", "s", "h0", "first")]
    want, bars = M.gated_scan_gradients(*ins, d["dy"], d["dhT"])
    y64, ybar = M.gated_scan(*ins)[0], M.gated_scan(*ins, bar=True)[0]
    more = 1 + s.max().item()   # a unit of the exponent counts as often as the exponent is large
    for got, w, bar, name in zip((outs[1][0], *outs[1][2:7]), (y64, *want), (ybar, *bars), ("y", "dx", "dgx", "dga", "ds", "dh0")):
        within(got, w, M.scan_bound(70, bar * more, w, got.dtype), name)
    state, y = d["h0"].clone(), torch.empty_like(d["x"][:, 0])
    for t in range(5):
        R.ops.gated_scan_update(state, *(d[n][:, t].contiguous() for n in ("x", "gx", "ga")), d["s"], y)
        assert torch.equal(state[:, none], d["h0"][:, none]) and torch.equal(y[:, none], d["h0"].to(dtype)[:, none])


def test_update_without_decay_in_wide_rows():
    """The same where four channels go to a thread."""
    import rwkv_cuda_b200 as R
    for dtype in (BF, F32):
        d = inputs(100, 1, 1024, dtype, seed=3)
        d["s"][::2] = -0.0
        x, gx, ga = (d[n][:, 0].contiguous() for n in ("x", "gx", "ga"))
        state, y = d["h0"].clone(), torch.empty_like(x)
        R.ops.gated_scan_update(state, x, gx, ga, d["s"], y)
        assert torch.equal(state[:, ::2], d["h0"][:, ::2]) and torch.equal(y[:, ::2], d["h0"].to(dtype)[:, ::2])
        assert (state[:, 1::2] != d["h0"][:, 1::2]).any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [8.0, 15.0])
def test_gates_that_saturate(dtype, scale):
    """Gates from sigmoid(-60) to sigmoid(60): decays of 1 - 1e-27 to exp(-s)."""
    d = inputs(2, 70, 64, dtype, seed=5, scale=scale)
    d["gx"] = d["ga"].flip(1).contiguous()
    check(d)


def test_documents_at_every_token_and_none():
    for fill in (0, 1):
        d = inputs(1, 150, 64, F32, seed=2)
        d["first"] = torch.full((1, 150), fill, dtype=torch.uint8, device="cuda")
        check(d)


def test_gradients_against_differences():
    """Central differences of the fp64 form along one direction per input; the third derivative leaves about step^2 = 1e-8 relative."""
    d = inputs(2, 90, 64, F32, seed=7, docs=True)
    grads = train(d)[1]
    ins = {n: d[n].double() for n in LEAVES}
    value = lambda z: sum((a * b.double()).sum() for a, b in zip(M.gated_scan(*(z[n] for n in LEAVES), d["first"]), (d["dy"], d["dhT"])))
    for n, got in zip(LEAVES, grads):
        way = torch.randn(ins[n].shape, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * (0.1 if n == "s" else 1)
        up, down = ({**ins, n: ins[n] + h * way} for h in (1e-4, -1e-4))
        want, have = (value(up) - value(down)) / 2e-4, (got.double() * way).sum()
        size = (got.double() * way).abs().sum()
        assert abs(want - have) <= 1e-5 * size, n   # rounding of the sum's terms to fp32 and the difference's own error are far below


def test_unaligned_and_strided():
    """Tensors that start at an odd element take the one-channel kernels; strided ones are made contiguous by the training class."""
    for dtype in (BF, F32):
        d = inputs(2, 40, 64, dtype, seed=3)
        y, hT = forward(d)
        out, grads, _ = train(d)
        moved = dict(d)
        for n in ("x", "gx", "ga", "dy"):
            base = torch.empty(d[n].numel() + 1, dtype=dtype, device="cuda")
            moved[n] = base[1:].view(d[n].shape).copy_(d[n])
        out2, grads2, _ = train(moved)
        for a, b in zip((*out, *grads), (*out2, *grads2)):
            assert torch.equal(a, b)
        for n in ("x", "gx", "ga", "dy"):
            moved[n] = d[n].transpose(0, 1).contiguous().transpose(0, 1)
        moved["first"] = None
        out3, grads3, _ = train(moved)
        for a, b in zip((*out, *grads), (*out3, *grads3)):
            assert torch.equal(a, b)
        assert torch.equal(out[0], y) and torch.equal(out[1], hT)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,C,docs", [(2, 80, 129, False), (1, 16, 128, False), (3, 37, 65, True), (1, 8, 1, False), (2, 150, 2047, False), (2, 33, 66, True)])
@pytest.mark.parametrize("starts", [(0, 0, 0, 0), (1, 0, 1, 1), (0, 1, 1, 0), (1, 1, 1, 1), (2, 3, 0, 1)])
def test_rows_anywhere(dtype, B, T, C, docs, starts):
    """Each tensor begins at an element of its own behind a 16-byte boundary, with NaN before and behind it, which stays."""
    import rwkv_cuda_b200 as R
    d = inputs(B, T, C, dtype, seed=C, docs=docs)
    n = B * T * C
    wants = [d[m] for m in ("x", "gx", "ga", "dy")]
    room = [torch.full((n + 16,), float("nan"), device="cuda", dtype=dtype) for _ in range(8)]
    where = [r[8 + o:8 + o + n].view(B, T, C) for r, o in zip(room, starts + starts[::-1])]
    for to, want in zip(where, wants):
        to.copy_(want)
    x, gx, ga, dy, y, dx, dgx, dga = where
    f, p = dict(device="cuda"), lambda t: t.data_ptr() if t is not None else 0
    hT, ds, dh0 = torch.empty(B, C, **f), torch.empty(C, **f), torch.empty(B, C, **f)
    lib, e = R._lib.lib(), 1 if dtype == BF else 0
    saved = torch.empty(lib.rwkvb200_gated_scan_saved_bytes(B, T, C), dtype=torch.uint8, **f)
    work = torch.empty(lib.rwkvb200_gated_scan_work_bytes(B, T, C), dtype=torch.uint8, **f)
    first, stream = d["first"], torch.cuda.current_stream().cuda_stream
    assert lib.rwkvb200_gated_scan_forward(e, B, T, C, p(d["h0"]), p(x), p(gx), p(ga), p(d["s"]), p(first), p(y), p(hT), p(saved), stream) == 0
    assert lib.rwkvb200_gated_scan_backward(e, B, T, C, p(x), p(gx), p(ga), p(d["s"]), p(first), p(saved), p(dy), p(d["dhT"]), p(dh0), p(dx), p(dgx), p(dga),
                                            p(ds), p(work), stream) == 0
    for r, o in zip(room, starts + starts[::-1]):
        assert r[:8 + o].isnan().all() and r[8 + o + n:].isnan().all()
    ins = [d[m] for m in ("x", "gx", "ga", "s", "h0", "first")]
    y64, hT64 = M.gated_scan(*ins)
    ybar, hbar = M.gated_scan(*ins, bar=True)
    within(y, y64, M.scan_bound(T, ybar, y64, dtype), "y")
    within(hT, hT64, M.scan_bound(T, hbar, hT64, F32), "hT")
    want, bars = M.gated_scan_gradients(*ins, d["dy"], d["dhT"])
    for got, w, bar, name in zip((dx, dgx, dga, ds, dh0), want, bars, ("dx", "dgx", "dga", "ds", "dh0")):
        within(got, w, M.scan_bound(T, bar, w, got.dtype), name)


def test_pieces_are_the_whole():
    """A prompt in pieces of any length through the state (in place) is the prompt at once, to rounding."""
    d = inputs(2, 333, 64, F32, seed=4, docs=True)
    y, hT = forward(d)
    import rwkv_cuda_b200 as R
    state, at = d["h0"].clone(), 0
    for n in (1, 100, 64, 128, 40):
        cut = {k: d[k][:, at:at + n].contiguous() for k in ("x", "gx", "ga", "first")}
        part = torch.empty_like(cut["x"])
        R.ops.gated_scan_forward(cut["x"], cut["gx"], cut["ga"], d["s"], part, h0=state, hT=state, first=cut["first"])
        torch.testing.assert_close(part, y[:, at:at + n], rtol=1e-5, atol=1e-5)
        at += n
    assert at == 333
    torch.testing.assert_close(state, hT, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite(bad):
    """An infinity stays one as long as its document lasts, and neither it nor a NaN reaches another document, another channel or an earlier token;
    backward, none of dy's reaches later tokens or the document before."""
    d = inputs(1, 400, 64, F32, seed=6)
    first = torch.zeros(1, 400, dtype=torch.bool, device="cuda")
    first[:, 250] = True
    d["first"] = first
    clean = forward(d)
    _, clean_grads, _ = train(d)
    x = d["x"].clone()
    x[0, 77, 5] = bad
    y, hT = forward({**d, "x": x})
    assert torch.equal(y[:, :77], clean[0][:, :77]) and torch.equal(y[:, 250:], clean[0][:, 250:]) and torch.equal(hT, clean[1])
    others = [c for c in range(64) if c != 5]
    assert torch.equal(y[:, :, others], clean[0][:, :, others])
    seen = y[0, 77:250, 5]
    assert (seen.isnan() if bad != bad else seen == bad).all()
    h0 = d["h0"].clone()
    h0[0, 9] = bad
    y, hT = forward({**d, "h0": h0})
    seen = y[0, :250, 9]
    assert (seen.isnan() if bad != bad else seen == bad).all() and torch.equal(y[:, 250:], clean[0][:, 250:])
    dy = d["dy"].clone()
    dy[0, 300, 5] = bad
    grads = train({**d, "dy": dy})[1]
    for g, c in zip(grads[:3], clean_grads[:3]):
        assert torch.equal(g[:, 301:], c[:, 301:]) and torch.equal(g[:, :250], c[:, :250]) and torch.equal(g[:, :, others], c[:, :, others])
    assert not torch.isfinite(grads[0][0, 251:301, 5]).any()
    assert torch.equal(grads[4], clean_grads[4])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("C", [64, 2048])
def test_gates_that_are_not_finite(dtype, C):
    """A NaN in one gate does not go into the other: with gx NaN (or infinite) the decay stays, so that gradients of earlier tokens stay, and with ga NaN
    the gradient comes to nothing before it only.  Infinite gates are 0 and 1."""
    d = inputs(1, 200, C, dtype, seed=6)
    ins = [d[n] for n in ("x", "gx", "ga", "s", "h0", "first")]
    y64, _ = M.gated_scan(*ins)
    ybar, _ = M.gated_scan(*ins, bar=True)
    want, bars = M.gated_scan_gradients(*ins, d["dy"], d["dhT"])
    others = [c for c in range(C) if c != 5]
    for name, bad in (("gx", float("nan")), ("gx", float("inf")), ("gx", float("-inf")), ("ga", float("nan")), ("ga", float("-inf"))):
        g = d[name].clone()
        g[0, 100, 5] = bad
        (y, hT), grads, _ = train({**d, name: g})
        # What the gate does not reach stays within the bound of the inputs without it; a tile that holds it divides for each gate on
        # its own, so that its neighbours are rounded in other places and are not the same bits.
        bound = M.scan_bound(200, ybar, y64, dtype)
        within(y[:, :100], y64[:, :100], bound[:, :100], "y before")
        within(y[..., others], y64[..., others], bound[..., others], "y beside")
        for got, w, bar in list(zip(grads, want, bars))[:3]:
            bound = M.scan_bound(200, bar, w, dtype)
            within(got[..., others], w[..., others], bound[..., others], "gradient beside")
            if name == "gx" and bad != bad:
                within(got[0, :99, 5], w[0, :99, 5], bound[0, :99, 5], "gradient before")
        if bad != bad:
            assert y[0, 100:, 5].isnan().all() and hT[0, 5].isnan()
            if name == "ga":
                assert grads[0][0, :100, 5].isnan().all()
        else:
            same = {**d, name: g.nan_to_num(posinf=300.0, neginf=-300.0)}   # exp(-300) is 0 in fp32, as of an infinity
            check(same)
            y2, hT2 = forward(same)
            assert torch.equal(y, y2) and torch.equal(hT, hT2)


def test_autograd():
    """Walked twice; only one output used; no state; through torch.autograd.Function."""
    import rwkv_cuda_b200 as R
    d = inputs(2, 70, 64, BF, seed=8, docs=True)
    out, grads, leaves = train(d, retain=True)
    again = torch.autograd.grad(out, leaves, (d["dy"], d["dhT"]))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaves, (d["dy"], d["dhT"]))

    class Sub(R.functions.GATED_SCAN):
        pass
    for h0 in (leaves[4], None):
        outs = []
        for cls in (R.functions.GATED_SCAN, Sub):
            y, hT = cls.apply(*leaves[:4], h0, d["first"])
            one = torch.autograd.grad(y, leaves[:4], d["dy"], retain_graph=True)
            two = torch.autograd.grad(hT, leaves[:4], d["dhT"])
            outs.append((y, hT, *one, *two))
        assert all(torch.equal(a, b) for a, b in zip(*outs))
    # first as uint8; s alone wants a gradient
    s = d["s"].clone().requires_grad_(True)
    y, _ = R.functions.GATED_SCAN.apply(d["x"], d["gx"], d["ga"], s, None, d["first"].to(torch.uint8))
    assert torch.equal(torch.autograd.grad(y, s, d["dy"])[0], outs[0][5])
    assert not R.functions.GATED_SCAN.apply(d["x"], d["gx"], d["ga"], d["s"])[0].requires_grad


def test_captured_training_step():
    d = inputs(2, 200, 64, BF, seed=9)
    want_out, want, _ = train(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads, _ = train(d)
    for t in (*out, *grads):
        t.zero_()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*out, *grads), (*want_out, *want)))


def test_capture_beside_a_living_graph():
    """A leaf that a graph of the default stream holds gets its gradient on that stream, which no capture can have: refused.  Once that graph
    is gone the step is captured."""
    import rwkv_cuda_b200 as R
    d = inputs(2, 200, 64, BF, seed=11)
    want_out, want, leaves = train(d)
    run = lambda: R.functions.GATED_SCAN.apply(*leaves, None)
    with torch.cuda.stream(torch.cuda.Stream()):
        run()
    torch.cuda.synchronize()
    alive = run()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="holds the same leaf"):
        with torch.cuda.graph(graph):
            out = run()
            torch.autograd.grad(out, leaves, (d["dy"], d["dhT"]))
    del alive, out, want_out
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
        grads = torch.autograd.grad(out, leaves, (d["dy"], d["dhT"]))
    for g in grads:
        g.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_gradients_that_are_not_contiguous():
    """A sum's gradient is one element in all places."""
    import rwkv_cuda_b200 as R
    d = inputs(2, 70, 64, F32, seed=12)
    d["dy"], d["dhT"] = torch.ones_like(d["dy"]), torch.ones_like(d["dhT"])
    want, leaves = train(d)[1:]
    y, hT = R.functions.GATED_SCAN.apply(*leaves, None)
    (y.sum() + hT.sum()).backward()
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip(leaves, want))


# ---- one token -----------------------------------------------------------------------------------------------------
def step(state, x, gx, ga, s, slots):
    """fp64, row after row"""
    state, out = state.double().clone(), {}
    for b, slot in enumerate(slots):
        if 0 <= slot < state.shape[0]:
            y, h = M.gated_scan(x[b][None, None], gx[b][None, None], ga[b][None, None], s, state[slot][None])
            state[slot] = h[0]
            out[b] = y[0, 0]
    return state, out


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,C,pool", [(1, 64, 1), (3, 33, 3), (5, 130, 9), (200, 65, 300)])
def test_update(dtype, B, C, pool):
    import rwkv_cuda_b200 as R
    d = inputs(B, 1, C, dtype, seed=B)
    x, gx, ga = (d[n][:, 0].contiguous() for n in ("x", "gx", "ga"))
    g = Hh.gen(1)
    state = Hh.randn(g, pool, C).cuda()
    for slots in ([int(i) for i in torch.randperm(pool, generator=g)[:B]], None):
        mine, y = state.clone(), torch.full((B, C), float("nan"), dtype=dtype, device="cuda")
        R.ops.gated_scan_update(mine, x, gx, ga, d["s"], y, slots=torch.tensor(slots, dtype=torch.int32, device="cuda") if slots else None)
        want, rows = step(state, x, gx, ga, d["s"], slots or list(range(B)))
        size = state.abs().double().max() + 8
        within(mine, want, M.scan_bound(1, size, want, F32), "state")
        y64 = torch.stack([rows[b] for b in range(B)])
        within(y, y64, M.scan_bound(1, size, y64, dtype), "y")


def test_update_slots():
    """Padding rows, a slot that is there three times, and one behind the pool."""
    import rwkv_cuda_b200 as R
    from rwkv_cuda_b200 import _lib
    B, C, pool = 300, 70, 40
    d = inputs(B, 1, C, F32, seed=3)
    x, gx, ga = (d[n][:, 0].contiguous() for n in ("x", "gx", "ga"))
    state = Hh.randn(Hh.gen(2), pool, C).cuda()
    slots = [-1] * B
    slots[0], slots[7], slots[150], slots[299], slots[20], slots[21] = 5, 5, 11, 5, 0, pool - 1
    L = _lib.lib()
    L.rwkvb200_device_status_clear()
    mine, y = state.clone(), torch.full((B, C), 7.0, device="cuda")
    R.ops.gated_scan_update(mine, x, gx, ga, d["s"], y, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    assert L.rwkvb200_device_status() == 0
    want, rows = step(state, x, gx, ga, d["s"], slots)
    within(mine, want, M.scan_bound(3, torch.tensor(16.0, device="cuda"), want, F32), "state")
    for b in range(B):
        if b in rows:
            within(y[b], rows[b], M.scan_bound(3, torch.tensor(16.0, device="cuda"), rows[b], F32), "y")
        else:
            assert (y[b] == 7.0).all()
    slots[40], slots[41] = pool, 2 ** 31 - 1
    again, y2 = state.clone(), torch.full((B, C), 7.0, device="cuda")
    R.ops.gated_scan_update(again, x, gx, ga, d["s"], y2, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    assert L.rwkvb200_device_status() == 121
    assert L.rwkvb200_device_status_clear() == 0 and L.rwkvb200_device_status() == 0
    assert y2[40].isnan().all() and y2[41].isnan().all() and torch.equal(again, mine)
    y2[40:42] = 7.0
    assert torch.equal(y, y2)


def test_update_many_channels():
    """Four channels a thread: shared slots, padding rows and a bad slot there too."""
    import rwkv_cuda_b200 as R
    from rwkv_cuda_b200 import _lib
    L = _lib.lib()
    for dtype in (BF, F32):
        B, C, pool = 200, 516, 150
        d = inputs(B, 1, C, dtype, seed=4)
        x, gx, ga = (d[n][:, 0].contiguous() for n in ("x", "gx", "ga"))
        state = Hh.randn(Hh.gen(2), pool, C).cuda()
        slots = [(b * 7) % pool for b in range(B)]   # 50 slots twice
        slots[3], slots[199], slots[100] = -1, -7, pool
        L.rwkvb200_device_status_clear()
        mine, y = state.clone(), torch.full((B, C), 7.0, dtype=dtype, device="cuda")
        R.ops.gated_scan_update(mine, x, gx, ga, d["s"], y, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
        assert L.rwkvb200_device_status() == 121
        L.rwkvb200_device_status_clear()
        want, rows = step(state, x, gx, ga, d["s"], slots)
        size = torch.tensor(16.0, device="cuda")
        within(mine, want, M.scan_bound(2, size, want, F32), "state")
        for b in range(B):
            if b in rows:
                within(y[b], rows[b], M.scan_bound(2, size, rows[b], dtype), "y")
            else:
                assert y[b].isnan().all() if slots[b] == pool else (y[b] == 7.0).all()


def test_update_is_the_scan():
    """Tokens one at a time, bit by bit what the scan makes of them where its sums have the same order (one token a call)."""
    import rwkv_cuda_b200 as R
    d = inputs(2, 9, 64, BF, seed=12)
    a, b = d["h0"].clone(), d["h0"].clone()
    for t in range(9):
        x, gx, ga = (d[n][:, t].contiguous() for n in ("x", "gx", "ga"))
        y, z = torch.empty_like(x), torch.empty_like(x[:, None])
        R.ops.gated_scan_update(a, x, gx, ga, d["s"], y)
        R.ops.gated_scan_forward(x[:, None], gx[:, None], ga[:, None], d["s"], z, h0=b, hT=b)
        torch.testing.assert_close(a, b, rtol=1e-6, atol=1e-6)
        torch.testing.assert_close(y, z[:, 0], rtol=2 ** -7, atol=1e-6)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,C", [(3, 130), (100, 1024)])
def test_update_and_scan_keep_their_digits(dtype, B, C):
    """Tokens one at a time, each element within its own bound, and the scan over the same tokens within the same: channels without decay, at the border of
    its two forms, and far beyond it side by side, gates out of the ordinary range among them."""
    import rwkv_cuda_b200 as R
    T = 9
    d = inputs(B, T, C, dtype, seed=C)
    few = torch.tensor([0.3, -0.0, 0.0, 1.0 - 2 ** -24, 1.0, 1.0 + 2 ** -23, 2.0, 30.0], device="cuda")
    d["s"] = few[torch.arange(C, device="cuda") % len(few)].contiguous()
    d["ga"][:, 4, ::5], d["gx"][:, 6, 1::5] = -45.0, 50.0
    want, bounds = M.scan_errors(*(d[n] for n in ("x", "gx", "ga", "s", "h0")))
    y, hT = forward(d)
    within(y, want[0], bounds[0], "y of the scan")
    within(hT, want[1], bounds[1], "hT of the scan")
    state = d["h0"].clone()
    for t in range(T):
        y = torch.empty(B, C, dtype=dtype, device="cuda")
        R.ops.gated_scan_update(state, *(d[n][:, t].contiguous() for n in ("x", "gx", "ga")), d["s"], y)
        within(y, want[0][:, t], bounds[0][:, t], f"y {t}")
    within(state, want[1], bounds[1], "state")


def test_refusals():
    import rwkv_cuda_b200 as R
    d = inputs(2, 5, 64, F32, seed=1, docs=True)
    y = torch.empty_like(d["x"])
    call = lambda **k: R.ops.gated_scan_forward(**{**dict(x=d["x"], gx=d["gx"], ga=d["ga"], s=d["s"], y=y, h0=d["h0"], first=d["first"]), **k})
    for k, error, word in ((dict(gx=d["gx"][:, :4]), RuntimeError, "gx: expected shape"), (dict(s=d["s"][:5]), RuntimeError, "s: expected shape"),
                           (dict(ga=d["ga"].to(BF)), TypeError, "ga: expected"), (dict(h0=d["h0"][:1]), RuntimeError, "h0: expected shape"),
                           (dict(first=d["first"].int()), TypeError, "first: expected bool"), (dict(y=y.cpu()), RuntimeError, "CUDA device"),
                           (dict(x=d["x"].transpose(0, 1).contiguous().transpose(0, 1)), RuntimeError, "contiguous"),
                           (dict(x=d["x"][0]), ValueError, "expected \\(B,T,C\\)"), (dict(x=d["x"].half()), TypeError, "not supported")):
        with pytest.raises(error, match=word):
            call(**k)
    with pytest.raises(TypeError, match="not supported"):
        R.functions.GATED_SCAN.apply(d["x"].double(), d["gx"], d["ga"], d["s"])
    with pytest.raises(R.RwkvB200Error, match="states for 2 rows"):
        R.ops.gated_scan_update(d["h0"][:1], *(d[n][:, 0].contiguous() for n in ("x", "gx", "ga")), d["s"], y[:, 0].contiguous())

"""GPU tests of the paged cache: the write with rotary positions and the attention of one new token that reads it, against fp64.
Pages lie anywhere; what no token fills holds NaN, and what the table does not use points nowhere."""
import math

import pytest
import torch

from oracle import mixer_oracle as M
from tests import helpers as Hh

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    same = (got.double() == want) | (got.isnan() & want.isnan())
    assert ((off <= bound) | same).all(), f"{what}: off by {(off / bound).nan_to_num(nan=9e9).masked_fill(same, 0).max().item():.3g} of the bound"


def paged(lengths, Hkv, N, page, dtype, seed, extra=1, room=0):
    """Pools, table and, per sequence, its keys and values (len, Hkv, N)."""
    g = Hh.gen(seed)
    need = [-(-(max(n, 0) + room) // page) for n in lengths]
    width, pages = max(need) + extra, sum(need) + 3
    order = torch.randperm(pages, generator=g)
    pools = [torch.full((pages, Hkv, page, N), float("nan"), dtype=dtype) for _ in range(2)]
    table = torch.full((len(lengths), width), 2 ** 31 - 1, dtype=torch.int32)
    kept, at = [], 0
    for b, n in enumerate(lengths):
        ids = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = ids.int()
        kv = [Hh.randn(g, max(n, 0), Hkv, N).to(dtype) for _ in range(2)]
        j = torch.arange(max(n, 0))
        for pool, x in zip(pools, kv):
            pool[ids[j // page], :, j % page] = x
        kept.append([x.cuda() for x in kv])
    return [p.cuda() for p in pools], table.cuda(), kept


def attend(q, pools, table, lengths, **k):
    import rwkv_cuda_b200 as R
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    R.ops.paged_attention(q, *pools, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), out, lse=lse, **k)
    return out, lse


def check(lengths, Hq, Hkv, N, page, dtype, seed=0, scale=None, **k):
    pools, table, kept = paged(lengths, Hkv, N, page, dtype, seed)
    q = Hh.randn(Hh.gen(seed + 1), len(lengths), Hq, N).to(dtype).cuda()
    out, lse = attend(q, pools, table, lengths, scale=scale, **k)
    for b, n in enumerate(lengths):
        if n < 0:
            assert (out[b] == 7.0).all() and (lse[b] == 7.0).all()
            continue
        o, l, ob, lb = M.attention(q[b], *kept[b], N ** -0.5 if scale is None else scale, k.get("cap", 0.0), k.get("slopes"), k.get("window", 0))
        within(out[b], o, ob + M.half_step(dtype) * o.abs(), f"out {b}")
        within(lse[b], l, lb, f"lse {b}")
    return out, lse


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hq,Hkv,N,page", [(4, 4, 64, 16), (8, 2, 64, 16), (8, 1, 128, 16), (12, 2, 128, 64), (10, 2, 128, 7), (3, 3, 33, 5), (6, 2, 80, 48),
                                           (2, 1, 1, 1), (40, 2, 64, 32), (17, 1, 96, 16), (4, 4, 8, 3), (9, 1, 20, 16), (2, 2, 128, 256), (32, 1, 100, 16)])
def test_heads_and_pages(dtype, Hq, Hkv, N, page):
    check([1, 0, 130, -1, 63, 64, 65, 17], Hq, Hkv, N, page, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[1], [0], [-1], [-5, 3], [15], [16], [17], [255], [256], [257], [5000], [40000], [1, 9000, 2, 0, -1, 700], [3] * 300,
                                     [300 + 17 * i for i in range(40)], [-1, -1, 2000, -1]])
def test_lengths(dtype, lengths):
    check(lengths, 8, 2, 64, 16, dtype, seed=len(lengths))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[5000] + [i % 40 - 1 for i in range(299)], [9000, 0, 1, 8999, 4096, 4097, -1, 63], [20000] * 5, [6000, 100] * 40])
@pytest.mark.parametrize("Hq,Hkv,N", [(8, 2, 128), (3, 3, 64), (20, 1, 72)])
def test_shared_work(dtype, lengths, Hq, Hkv, N):
    """Tables of more than 4096 tokens: the work is shared equally and units that lie in several runs are joined; more sequences than a block has threads."""
    check(lengths, Hq, Hkv, N, 16, dtype, seed=7)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hq,N", [(1, 1), (2, 1), (3, 2), (1, 3)])
def test_more_runs_than_elements(dtype, Hq, N):
    """One long sequence of tiny heads: hundreds of runs of which each block joins an element or none."""
    check([60000], Hq, 1, N, 16, dtype, seed=5)
    check([40000, 3], Hq, 1, N, 16, dtype, seed=5, cap=math.inf)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("most,B", [(500, 3), (1000, 40), (2000, 100), (4000, 2), (64, 300), (16, 1)])
@pytest.mark.parametrize("Hq,Hkv,N", [(8, 2, 128), (6, 6, 64), (32, 2, 64)])
def test_lone_sequences(dtype, most, B, Hq, Hkv, N):
    """Short tables: clusters of 1 to 8 blocks with a sequence's head each, for sequences of all lengths."""
    check([(i * 37) % (most + 1) if i else most for i in range(B)], Hq, Hkv, N, 16, dtype, seed=8)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[1, 0, 130, -1, 63, 64, 65, 17], [9000, 5, 300]])
@pytest.mark.parametrize("N", [64, 128])
def test_without_tensor_maps(dtype, lengths, N):
    """Where the driver makes no tensor maps, rows are copied in pieces; results are the same bits (the products see the same tiles)
    but for tables that are then not given to clusters."""
    from rwkv_cuda_b200 import _lib
    L = _lib.lib()
    with_maps = check(lengths, 8, 2, N, 16, dtype, seed=9)
    L.rwkvb200_test_disable_tensor_maps(1)
    try:
        without = check(lengths, 8, 2, N, 16, dtype, seed=9)
    finally:
        L.rwkvb200_test_disable_tensor_maps(0)
    if max(lengths) > 4096:
        assert torch.equal(with_maps[0], without[0]) and torch.equal(with_maps[1], without[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("k", [dict(cap=30.0), dict(cap=0.5), dict(window=1), dict(window=100), dict(window=5000), dict(slopes=True), dict(scale=0.0),
                               dict(scale=-0.3), dict(scale=3.0), dict(cap=20.0, window=700, slopes=True)])
@pytest.mark.parametrize("Hq,Hkv,N", [(8, 2, 128), (3, 1, 40)])
def test_scores(dtype, k, Hq, Hkv, N):
    k = dict(k)
    if k.get("slopes"):
        k["slopes"] = (2.0 ** -torch.arange(1.0, Hq + 1)).cuda()
    check([1, 99, 100, 101, 3001, 0, 1300], Hq, Hkv, N, 16, dtype, seed=3, **k)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [128, 24])
def test_large_and_unequal_scores(dtype, N):
    """Scores of thousands, one token that has all the weight at the front, in the middle or at the end of a long sequence."""
    n = 3000
    for at in (0, 1, 1500, n - 1):
        pools, table, kept = paged([n], 1, N, 16, dtype, seed=at)
        q = (30 * Hh.randn(Hh.gen(5), 1, 4, N)).to(dtype).cuda()
        page = int(table[0, at // 16])
        key = (q[0, 0].float() * 8).to(dtype)
        pools[0][page, 0, at % 16], kept[0][0][at, 0] = key, key
        out, lse = attend(q, pools, table, [n])
        o, l, ob, lb = M.attention(q[0], *kept[0], N ** -0.5)
        within(out[0], o, ob + M.half_step(dtype) * o.abs(), "out")
        within(lse[0], l, lb, "lse")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [64, 20])
def test_values_that_are_not_finite(dtype, N):
    """Values of infinity come out where the token has weight; keys that make scores of -infinity have none (whatever their values hold); a
    sequence of only such scores gives 0; NaN in a key or value reaches the heads that read it and no others."""
    lengths, g = [200, 200, 200, 50, 200], Hh.gen(3)
    pools, table, kept = paged(lengths, 2, N, 16, dtype, seed=1)

    def put(b, j, head, key=None, value=None):
        for pool, keep, x in ((pools[0], kept[b][0], key), (pools[1], kept[b][1], value)):
            if x is not None:
                pool[int(table[b, j // 16]), head, j % 16] = x
                keep[j, head] = x
    q = Hh.rand(g, 5, 4, N, lo=0.5, hi=1.0).to(dtype).cuda()     # positive: a key of -infinity scores -infinity
    put(0, 77, 0, value=torch.full((N,), math.inf, dtype=dtype))
    put(1, 5, 1, key=torch.full((N,), -math.inf, dtype=dtype), value=torch.full((N,), math.nan, dtype=dtype))
    put(2, 9, 0, key=torch.full((N,), math.nan, dtype=dtype))
    for j in range(50):
        put(3, j, 1, key=torch.full((N,), -math.inf, dtype=dtype), value=torch.full((N,), math.inf, dtype=dtype))
    put(4, 100, 1, value=torch.full((N,), math.nan, dtype=dtype))
    out, lse = attend(q, pools, table, lengths)
    for b in range(5):
        o, l, ob, lb = M.attention(q[b], *kept[b], N ** -0.5)
        bound = (ob + M.half_step(dtype) * o.abs()).nan_to_num(0.0, 0.0, 0.0)
        within(out[b], o, bound, f"out {b}")
        within(lse[b], l, lb.nan_to_num(0.0, 0.0, 0.0), f"lse {b}")
    assert (out[0, :2] == math.inf).all() and torch.isfinite(out[0, 2:]).all() and torch.isfinite(out[1]).all()
    assert out[2, :2].isnan().all() and torch.isfinite(out[2, 2:]).all()
    assert (out[3, 2:] == 0).all() and (lse[3, 2:] == -math.inf).all() and torch.isfinite(out[3, :2]).all()
    assert out[4, 2:].isnan().all() and torch.isfinite(out[4, :2]).all() and torch.isfinite(lse[4]).all()


@pytest.mark.parametrize("Hq,Hkv,N,page,extra", [(8, 2, 128, 16, 1), (8, 2, 64, 16, 300), (32, 2, 128, 16, 1), (40, 2, 64, 16, 300), (6, 2, 40, 7, 1), (3, 1, 33, 16, 1)])
def test_weights_keep_their_digits(Hq, Hkv, N, page, extra):
    """bf16, values of +1 and -1 in turn under nearly equal weights: what is left of them is 1e-3 to 1e-5, so that the rounding of the result hides nothing
    of the weights' own.  (Weights of 2^-17 relative are several times the bound off.)"""
    lengths = [2] * 30 + [4, 64, 100]
    pools, table, kept = paged(lengths, Hkv, N, page, BF, seed=6, extra=extra)
    for b, n in enumerate(lengths):
        for j in range(n):
            at = int(table[b, j // page]), slice(None), j % page
            kept[b][0][j] = pools[0][at] = kept[b][0][j] * (j % 2) * 2.0 ** -11   # (an even token's score is 0)
            kept[b][1][j] = pools[1][at] = 1.0 - 2 * (j % 2)
    q = Hh.randn(Hh.gen(7), len(lengths), Hq, N).to(BF).cuda()
    out, lse = attend(q, pools, table, lengths)
    for b, n in enumerate(lengths):
        o, l, ob, lb = M.attention(q[b], *kept[b], N ** -0.5)
        within(out[b], o, ob + M.half_step(BF) * o.abs(), f"out {b}")
        within(lse[b], l, lb, f"lse {b}")


def test_small_weights_of_infinite_values():
    """A weight down to 2^-120 makes an infinite value of the other head's token infinite and not NaN; without weight it is nothing."""
    for N, Hq in ((64, 2), (128, 12), (40, 2)):
        for power in (20, 100, 120):
            pools, table, kept = paged([20], 1, N, 16, BF, seed=2)
            q = torch.zeros(1, Hq, N, dtype=BF, device="cuda")
            q[:, :, 0] = 1.0
            keys, values = (torch.zeros(20, 1, N, dtype=BF, device="cuda") for _ in range(2))
            keys[:, :, 0], keys[3, :, 0] = 1.0, 1.0 - power
            values[:], values[3, :, 5] = 0.5, math.inf
            for j in range(20):
                pools[0][int(table[0, j // 16]), :, j % 16], pools[1][int(table[0, j // 16]), :, j % 16] = keys[j], values[j]
            out, _ = attend(q, pools, table, [20], scale=math.log(2))
            assert (out[0, :, 5] == math.inf).all() and torch.isfinite(out[0, :, :5]).all() and torch.isfinite(out[0, :, 6:]).all()


def test_large_values_without_weight():
    """The largest values there are, under weights that are 0 in fp32 or nearly so, in some heads or all of them: nothing is left of them."""
    for dtype in (BF, F32):
        for N, Hq in ((64, 2), (128, 12), (40, 2)):
            pools, table, kept = paged([70], 1, N, 16, dtype, seed=2)
            top = torch.finfo(BF).max
            q = torch.zeros(1, Hq, N, dtype=dtype, device="cuda")
            q[:, :, 0] = 1.0
            q[:, ::2, 1] = 1.0      # (odd heads give token 9 its full weight)
            keys, values = (torch.zeros(70, 1, N, dtype=dtype, device="cuda") for _ in range(2))
            keys[3, :, 0], values[3, :, 5] = -1000.0, top
            keys[60, :, 0], values[60, :, 6] = -150.0, -top    # 2^-150 top = 2^-22
            keys[9, :, 1], values[9, :, 7] = -500.0, 2.0 ** 100
            for j in range(70):
                at = int(table[0, j // 16]), slice(None), j % 16
                pools[0][at], pools[1][at] = keys[j], values[j]
            out, _ = attend(q, pools, table, [70], scale=math.log(2))
            assert (out[0, :, :5] == 0).all() and (out[0, :, 5] == 0).all() and (out[0, :, 8:] == 0).all()
            assert (out[0, :, 6].abs() <= 2.0 ** -22).all()   # (weights below 2^-126 are 0)
            assert (out[0, ::2, 7] == 0).all()
            torch.testing.assert_close(out[0, 1::2, 7].double(), torch.full((Hq // 2,), 2.0 ** 100 / 68, dtype=torch.float64, device="cuda"), rtol=2 ** -8, atol=0)


def test_unaligned_tensors():
    """Pools, queries and outputs that start at an odd element."""
    import rwkv_cuda_b200 as R
    lengths = [300, 5, 0, 77]
    for dtype in (BF, F32):
        pools, table, kept = paged(lengths, 2, 64, 16, dtype, seed=1)
        q = Hh.randn(Hh.gen(2), 4, 8, 64).to(dtype).cuda()

        def moved(x):
            return torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)
        out = moved(q)
        R.ops.paged_attention(moved(q), *(moved(p) for p in pools), table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), out)
        for only in range(3):
            part = [moved(x) if i == only else x for i, x in enumerate((q, *pools))]
            o2, _ = attend(*part[:1], part[1:], table, lengths)
            for b, n in enumerate(lengths):
                o, l, ob, lb = M.attention(q[b], *kept[b], 1 / 8)
                within(o2[b], o, ob + M.half_step(dtype) * o.abs(), "out")
                within(out[b], o, ob + M.half_step(dtype) * o.abs(), "out")


def test_shared_pages_and_repeated_runs():
    """Sequences that share their first pages; the same call gives the same bits."""
    dtype = BF
    pools, table, kept = paged([1000, 1000], 2, 64, 16, dtype, seed=4)
    table[1, :30] = table[0, :30]
    kept[1] = [torch.cat([a[:480], b[480:]]) for a, b in zip(*kept)]
    q = Hh.randn(Hh.gen(2), 2, 8, 64).to(dtype).cuda()
    out, lse = attend(q, pools, table, [1000, 1000])
    for b in range(2):
        o, l, ob, lb = M.attention(q[b], *kept[b], 1 / 8)
        within(out[b], o, ob + M.half_step(dtype) * o.abs(), "out")
    for _ in range(3):
        again = attend(q, pools, table, [1000, 1000])
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [64, 33])
def test_pages_and_lengths_that_point_nowhere(dtype, N):
    """Tokens on such pages are left out, lengths end where the table does, and the status word says so."""
    from rwkv_cuda_b200 import _lib
    L = _lib.lib()
    L.rwkvb200_device_status_clear()
    lengths = [600, 200, 600]
    pools, table, kept = paged(lengths, 2, N, 16, dtype, seed=2, extra=0)
    q = Hh.randn(Hh.gen(3), 3, 4, N).to(dtype).cuda()
    attend(q, pools, table, lengths)
    assert L.rwkvb200_device_status() == 0
    for bad in (-1, -2 ** 31, pools[0].shape[0], 2 ** 31 - 1):
        broken = table.clone()
        broken[0, 7], broken[1, 0:13] = bad, bad
        out, lse = attend(q, pools, broken, lengths)
        assert L.rwkvb200_device_status() == 141
        L.rwkvb200_device_status_clear()
        left = torch.tensor([j for j in range(600) if j // 16 != 7], device="cuda")
        o, l, ob, lb = M.attention(q[0], kept[0][0][left], kept[0][1][left], N ** -0.5)
        within(out[0], o, ob + M.half_step(dtype) * o.abs(), "out")
        within(lse[0], l, lb, "lse")
        assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    out, lse = attend(q, pools, table, [600, 200, 2 ** 31 - 1])
    assert L.rwkvb200_device_status() == 142
    L.rwkvb200_device_status_clear()
    o, l, ob, lb = M.attention(q[2], *kept[2], N ** -0.5)   # 600 tokens fill 38 pages up to 608: the rest of the last page counts too
    full = [torch.cat([x, torch.full((8, 2, N), math.nan, dtype=dtype, device="cuda")]) for x in kept[2]]
    assert out[2].isnan().all()
    pools[0][table[2, 37].long(), :, 8:], pools[1][table[2, 37].long(), :, 8:] = 1.0, 1.0
    out, lse = attend(q, pools, table, [600, 200, 2 ** 31 - 1])
    L.rwkvb200_device_status_clear()
    for x in full:
        x[600:] = 1.0
    o, l, ob, lb = M.attention(q[2], *full, N ** -0.5)
    within(out[2], o, ob + M.half_step(dtype) * o.abs(), "out")


def test_offsets_beyond_32_bits():
    """A pool of 2.6e9 elements: pages whose elements lie behind 2^31 and 2^32 bytes and 2^31 elements."""
    free = torch.cuda.mem_get_info()[0]
    if free < 14 << 30:
        pytest.skip("needs 14 GB")
    Hkv, page, N = 8, 256, 128
    pages = 10000
    pools = [torch.zeros(pages, Hkv, page, N, dtype=BF, device="cuda") for _ in range(2)]
    table = torch.tensor([[9999, 1, 8500, 5000], [4100, 9000, 0, 9998]], dtype=torch.int32, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    for i in table.flatten().tolist():
        for p in pools:
            p[i].normal_(generator=g)
    lengths = [1000, 1024]
    q = torch.randn(2, 16, N, device="cuda", generator=g).to(BF)
    out, lse = attend(q, pools, table, lengths)
    for b, n in enumerate(lengths):
        k, v = (p[table[b].long()].transpose(1, 2).reshape(-1, Hkv, N)[:n] for p in pools)
        o, l, ob, lb = M.attention(q[b], k, v, N ** -0.5)
        within(out[b], o, ob + M.half_step(BF) * o.abs(), "out")
    import rwkv_cuda_b200 as R
    new = torch.randn(2, Hkv, N, device="cuda", generator=g).to(BF)
    R.ops.paged_append(new, new, *pools, table, torch.tensor([700, 1023], dtype=torch.int32, device="cuda"))
    assert torch.equal(pools[0][8500, :, 700 - 512], new[0]) and torch.equal(pools[1][9998, :, 255], new[1])


# ---- the write -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hq,Hkv,N,R_,interleaved,page", [(4, 2, 64, 64, False, 16), (4, 2, 64, 64, True, 16), (8, 1, 128, 32, False, 5), (8, 1, 128, 32, True, 5),
                                                          (3, 3, 33, 32, False, 7), (3, 3, 33, 10, True, 7), (2, 2, 80, 24, False, 48),
                                                          (2, 2, 80, 20, True, 48), (1, 1, 2, 2, False, 1), (5, 5, 64, 0, False, 16), (0, 2, 64, 64, False, 16),
                                                          (32, 8, 128, 128, False, 16), (3, 2, 66, 12, False, 7), (2, 3, 66, 22, True, 16)])
def test_append(dtype, Hq, Hkv, N, R_, interleaved, page):
    import rwkv_cuda_b200 as R
    g = Hh.gen(N + R_)
    lengths, counts = [0, 15, 16, 100000 if N == 64 else 50, -1, 3], [1, 20, 1, 7, 4, 0]
    inv = (10000.0 ** (-torch.arange(0, R_, 2) / max(R_, 1))).cuda() if R_ else None
    for ragged in (False, True):
        B = len(lengths)
        n = counts if ragged else [1] * B
        lead = 2 if ragged else 0
        M_ = sum(n) + lead + (3 if ragged else 0)
        cu = torch.tensor([lead + sum(n[:i]) for i in range(B + 1)], dtype=torch.int32).cuda() if ragged else None
        need = [-(-(max(a, 0) + c) // page) for a, c in zip(lengths, n)]
        pages = 40 + max(counts) // page * 2
        table = torch.full((B, max(need)), 2 ** 31 - 1, dtype=torch.int32)
        ids = iter(torch.randperm(pages, generator=g).tolist())
        for b in range(B):
            if lengths[b] >= 0 and n[b]:
                for c in range(lengths[b] // page, need[b]):
                    table[b, c] = next(ids)
        k, v = (Hh.randn(g, M_, Hkv, N).to(dtype).cuda() for _ in range(2))
        q = Hh.randn(g, M_, Hq, N).to(dtype).cuda() if Hq else None
        pools = [torch.full((pages, Hkv, page, N), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        outs = []
        for in_place in (False, True):
            mine = [p.clone() for p in pools]
            q_out = None if q is None else q.clone() if in_place else torch.full_like(q, 7.0)
            R.ops.paged_append(k, v, *mine, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), cu_seqlens=cu,
                               q=q_out if in_place else q, q_out=q_out, inv_freq=inv, interleaved=interleaved, rotary_scale=1.25)
            outs.append((q_out, *mine))
        for b in range(B):
            first = lead + sum(n[:b])
            for i in range(n[b]):
                m, pos = first + i, lengths[b] + i
                if lengths[b] < 0:
                    assert q is None or (outs[0][0][m] == 7.0).all() and torch.equal(outs[1][0][m], q[m])
                    continue
                where = (int(table[b, pos // page]), slice(None), pos % page)
                at = torch.tensor([pos], device="cuda")
                for got, x in ((outs[0][1][where], k[m]), (outs[0][0][m] if Hq else None, q[m] if Hq else None)):
                    if got is not None:
                        want = M.rotated(x[None], at, inv, interleaved, 1.25)[0] if R_ else x.double()
                        # an angle is off by a unit of half a turn, sine and cosine by 4 of their own, products and sum by 4
                        size = 1.25 * 2 * x.double().abs().max() if R_ else 0.0
                        within(got, want, M.half_step(dtype) * want.abs() + 16 * M.UNIT * size, "rotated")
                assert torch.equal(outs[0][2][where], v[m])
                pools[0][where] = pools[1][where] = 0.0
        untouched = pools[0] == 7.0
        for a, b2 in zip(outs[0], outs[1]):
            if a is not None and a.dim() == 4:
                assert torch.equal(a, b2) and (a[untouched] == 7.0).all()
        if ragged and q is not None:
            assert (outs[0][0][:lead] == 7.0).all() and (outs[0][0][-3:] == 7.0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hq,Hkv,N,R_,interleaved,page", [(4, 2, 64, 64, False, 16), (33, 5, 64, 32, True, 16), (8, 1, 128, 32, False, 5), (1, 9, 80, 16, True, 48), (0, 2, 128, 0, False, 16),
                                                          (5, 2, 80, 40, False, 16), (3, 1, 66, 10, True, 16), (2, 2, 30, 14, False, 16), (2, 3, 31, 10, True, 7), (2, 1, 33, 16, False, 16)])
def test_append_many(dtype, Hq, Hkv, N, R_, interleaved, page):
    """Thousands of tokens: a warp does a token."""
    import rwkv_cuda_b200 as R
    g = Hh.gen(N)
    counts = torch.tensor([1500, 1, 0, 1203, 700])
    lengths = torch.tensor([10, 0, 5, 1, 4000])
    B, lead, total = len(counts), 3, int(counts.sum()) + 3 + 5
    cu = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]) + lead
    need = -(-(lengths + counts) // page)
    first = torch.cat([torch.zeros(1, dtype=torch.long), need.cumsum(0)])
    pages = int(first[-1])
    order = torch.randperm(pages, generator=g)
    table = torch.full((B, int(need.max())), -1)
    for b in range(B):
        table[b, :need[b]] = order[first[b]:first[b + 1]]
    k, v = (Hh.randn(g, total, Hkv, N).to(dtype).cuda() for _ in range(2))
    q = Hh.randn(g, total, Hq, N).to(dtype).cuda() if Hq else None
    q_out = torch.full_like(q, 7.0) if Hq else None
    pools = [torch.full((pages, Hkv, page, N), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    inv = (10000.0 ** (-torch.arange(0, R_, 2) / max(R_, 1))).cuda() if R_ else None
    R.ops.paged_append(k, v, *pools, table.int().cuda(), lengths.int().cuda(), cu_seqlens=cu.int().cuda(), q=q, q_out=q_out, inv_freq=inv, interleaved=interleaved)
    m = torch.arange(lead, total - 5)
    seq = torch.searchsorted(cu[1:], m, right=True)
    pos = lengths[seq] + m - cu[seq]
    where = (table[seq, pos // page].cuda(), slice(None), (pos % page).cuda())
    m, pos = m.cuda(), pos.cuda()
    for got, x in ((pools[0][where], k[m]), (q_out[m] if Hq else None, q[m] if Hq else None)):
        if got is not None:
            want = M.rotated(x, pos, inv, interleaved, 1.0) if R_ else x.double()
            within(got, want, M.half_step(dtype) * want.abs() + (16 * M.UNIT * 2 * x.double().abs().max() if R_ else 0.0), "rotated")
    assert torch.equal(pools[1][where], v[m])
    for p in pools:
        p[where] = 7.0
        assert (p == 7.0).all()
    assert not Hq or (q_out[:lead] == 7.0).all() and (q_out[-5:] == 7.0).all()


def test_sequences_that_make_no_sense():
    """cu_seqlens and lengths of any values write to no other place than a token's page."""
    import rwkv_cuda_b200 as R
    from rwkv_cuda_b200 import _lib
    x = Hh.randn(Hh.gen(1), 12, 2, 64).cuda()
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for cu in ([0, -5, 12, 12], [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [5, 4, 3, 2], [2 ** 31 - 1] * 4, [-2 ** 31] * 4):
        for lengths in ([0, 0, 0], [2 ** 31 - 1, -2 ** 31, 31]):
            pools = [torch.full((3, 2, 16, 64), 7.0, device="cuda") for _ in range(2)]
            R.ops.paged_append(x, x, *pools, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"))
            torch.cuda.synchronize()
            assert (pools[0][1:] == 7.0).all() and (pools[1][1:] == 7.0).all()
    _lib.lib().rwkvb200_device_status_clear()


def test_far_positions():
    """Position 2 * 10^9: the angle is taken in fp64."""
    import rwkv_cuda_b200 as R
    N, pos = 64, 2 * 10 ** 9
    inv = (10000.0 ** (-torch.arange(0, N, 2) / N)).cuda()
    q = Hh.randn(Hh.gen(1), 1, 2, N).cuda()
    page = 2 ** 20
    table = torch.zeros(1, 2000, dtype=torch.int32, device="cuda")
    pool = torch.zeros(1, 1, page, N, device="cuda")
    out = torch.empty_like(q)
    R.ops.paged_append(q[:, :1].contiguous(), q[:, 1:].contiguous(), pool, pool.clone(), table, torch.tensor([pos], dtype=torch.int32, device="cuda"), q=q, q_out=out, inv_freq=inv)
    want = M.rotated(q, torch.tensor([pos], device="cuda"), inv, False, 1.0)
    within(out, want, 16 * M.UNIT * 2 * q.abs().max().double(), "q")   # (fp64 leaves 2^-53 * 2e9 = 2e-7 of a radian)
    within(pool[0, 0, pos % page], want[0, 0], 16 * M.UNIT * 2 * q.abs().max().double(), "k")


def test_append_of_the_most_tokens():
    """2^31 - 1 rows, of which the last five belong to a sequence: more than an int holds once it is rounded up to whole blocks."""
    import rwkv_cuda_b200 as R
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    M_ = 2 ** 31 - 1
    k = torch.zeros(M_, 1, 1, dtype=BF, device="cuda")
    k[-5:, 0, 0] = torch.arange(1.0, 6.0).to(BF)
    pools = [torch.zeros(2, 1, 4, 1, dtype=BF, device="cuda") for _ in range(2)]
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    R.ops.paged_append(k, k, *pools, ints([0, 0], [1, 0]), ints(-1, 0), cu_seqlens=ints(0, M_ - 5, M_))
    for p in pools:
        assert p.flatten().tolist() == [5.0, 0.0, 0.0, 0.0, 1.0, 2.0, 3.0, 4.0]


def test_append_to_pages_that_are_none():
    import rwkv_cuda_b200 as R
    from rwkv_cuda_b200 import _lib
    L = _lib.lib()
    L.rwkvb200_device_status_clear()
    for N in (64, 33):
        x = Hh.randn(Hh.gen(1), 3, 2, N).cuda()
        pools = [torch.full((4, 2, 16, N), 7.0, device="cuda") for _ in range(2)]
        for bad, lengths, status in ((-1, [0, 5, 31], 131), (4, [0, 5, 31], 131), (2 ** 31 - 1, [0, 5, 31], 131), (2, [2 ** 31 - 1, 5, 31], 132)):
            table = torch.tensor([[bad, bad], [0, bad], [bad, 1]], dtype=torch.int32, device="cuda")
            mine = [p.clone() for p in pools]
            R.ops.paged_append(x, x, *mine, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
            assert L.rwkvb200_device_status() == status
            L.rwkvb200_device_status_clear()
            for p in mine:
                assert torch.equal(p[0, :, 5], x[1]) and torch.equal(p[1, :, 15], x[2])
                p[0, :, 5] = p[1, :, 15] = 7.0
                assert (p == 7.0).all()


def test_refusals():
    import rwkv_cuda_b200 as R
    pools, table, _ = paged([20, 3], 2, 64, 16, BF, seed=1)
    q, out = (torch.zeros(2, 8, 64, dtype=BF, device="cuda") for _ in range(2))
    lengths = torch.tensor([20, 3], dtype=torch.int32, device="cuda")
    base = dict(q=q, k_pages=pools[0], v_pages=pools[1], table=table, lengths=lengths, out=out)
    for k, error, word in ((dict(q=q[:1]), RuntimeError, "q: expected shape"), (dict(q=q.float()), TypeError, "expected Float, got BFloat16"),
                           (dict(table=table.long()), TypeError, "table: expected"), (dict(lengths=lengths.long()), TypeError, "lengths: expected"),
                           (dict(lengths=lengths[:1]), RuntimeError, "lengths: expected shape"), (dict(v_pages=pools[1][:1]), RuntimeError, "v_pages"),
                           (dict(k_pages=pools[0].transpose(1, 2).contiguous().transpose(1, 2)), RuntimeError, "contiguous"),
                           (dict(table=table.cpu()), RuntimeError, "CUDA device"), (dict(window=-1), ValueError, "negative"),
                           (dict(cap=-1.0), R.RwkvB200Error, "negative"), (dict(slopes=torch.zeros(2, device="cuda")), RuntimeError, "slopes: expected"),
                           (dict(q=q[:, :7].contiguous(), out=out[:, :7].contiguous()), R.RwkvB200Error, "not a multiple"),
                           (dict(lse=torch.zeros(2, 8, dtype=BF, device="cuda")), TypeError, "lse: expected"), (dict(q=q.half()), TypeError, "not supported")):
        with pytest.raises(error, match=word):
            R.ops.paged_attention(**{**base, **k})
    big = torch.zeros(2, 2, 16, 256, dtype=BF, device="cuda")
    with pytest.raises(R.RwkvB200Error, match="head size"):
        R.ops.paged_attention(**{**base, "k_pages": big, "v_pages": big, "q": torch.zeros(2, 8, 256, dtype=BF, device="cuda"), "out": torch.zeros(2, 8, 256, dtype=BF, device="cuda")})
    x = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
    base = dict(k=x, v=x, k_pages=pools[0], v_pages=pools[1], table=table, lengths=lengths)
    for k, error, word in ((dict(k=x[:1]), RuntimeError, "v: expected shape"), (dict(k=x[:, :1].contiguous()), RuntimeError, "k: expected shape"),
                           (dict(q=q), ValueError, "come together"), (dict(v=x.float()), TypeError, "v: expected"),
                           (dict(k=x[:1], v=x[:1]), R.RwkvB200Error, "need cu_seqlens"), (dict(inv_freq=torch.zeros(40, device="cuda")), ValueError, "40 pairs"),
                           (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32, device="cuda")), RuntimeError, "cu_seqlens: expected"),
                           (dict(inv_freq=torch.zeros(4, device="cuda", dtype=torch.float64)), TypeError, "inv_freq: expected")):
        with pytest.raises(error, match=word):
            R.ops.paged_append(**{**base, **k})


def test_two_streams_and_graphs():
    """Calls on two streams at once, and two captured graphs replayed side by side, have a workspace each."""
    import rwkv_cuda_b200 as R
    cases = []
    for i, n in enumerate(([30000, 5], [9000, 40000])):
        pools, table, _ = paged(n, 2, 64, 16, BF, seed=i)
        q = Hh.randn(Hh.gen(i), 2, 8, 64).to(BF).cuda()
        cases.append((q, pools, table, torch.tensor(n, dtype=torch.int32, device="cuda"), attend(q, pools, table, n)[0], torch.empty_like(q)))
    call = lambda c: R.ops.paged_attention(c[0], *c[1], c[2], c[3], c[5])
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(50):
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                call(c)
    torch.cuda.synchronize()
    for c in cases:
        assert torch.equal(c[5], c[4])
        c[5].zero_()
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(c)
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(50):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for c in cases:
        assert torch.equal(c[5], c[4])


# ---- together ------------------------------------------------------------------------------------------------------
def test_decoder_of_two_layers():
    """A recurrent layer that feeds an attention layer: prompts of different lengths are read, then tokens are decoded one by one from a captured graph, in a
    batch with a padding row, against both layers over the whole sequences in fp64 on the same rounded inputs."""
    import rwkv_cuda_b200 as R
    g = Hh.gen(3)
    C, Hq, Hkv, N, page, steps = 128, 4, 2, 64, 16, 9
    prompts = [37, 1, 130]
    B, rows = len(prompts), 4
    s = (-8 * torch.log(Hh.rand(g, C, lo=0.9, hi=0.999))).cuda()
    wk, wv, wq = ((Hh.randn(g, C, n * N) / C ** 0.5).cuda() for n in (Hkv, Hkv, Hq))
    inv = (10000.0 ** (-torch.arange(0, N, 2) / N)).cuda()
    seqs = [[Hh.randn(g, n + steps, C).cuda() for _ in range(3)] for n in prompts]
    slots = torch.tensor([4, 0, 2, -1], dtype=torch.int32, device="cuda")
    state = torch.full((5, C), 7.0, device="cuda")
    width = -(-(max(prompts) + steps) // page)
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    table[:B] = torch.randperm(B * width, generator=g).int().view(B, width)
    pools = [torch.full((B * width, Hkv, page, N), math.nan, device="cuda") for _ in range(2)]
    heads = lambda h, w, n: (h @ w).view(-1, n, N)
    # prompts, one after the other through the recurrence, together into the cache
    hs = []
    for b, (n, xs) in enumerate(zip(prompts, seqs)):
        h, hT = torch.empty(1, n, C, device="cuda"), torch.empty(1, C, device="cuda")
        R.ops.gated_scan_forward(*(x[None, :n].contiguous() for x in xs), s, h, hT=hT)
        state[slots[b].long()] = hT[0]
        hs.append(h[0])
    flat = torch.cat(hs)
    cu = torch.tensor([0, 37, 38, 168, 168], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([0, 0, 0, -1], dtype=torch.int32, device="cuda")
    R.ops.paged_append(heads(flat, wk, Hkv), heads(flat, wv, Hkv), *pools, table, lengths, cu_seqlens=cu, inv_freq=inv)
    lengths[:B] = torch.tensor(prompts, dtype=torch.int32)
    # decoding
    x, gx, ga = (torch.zeros(rows, C, device="cuda") for _ in range(3))
    h, out = torch.zeros(rows, C, device="cuda"), torch.zeros(rows, Hq, N, device="cuda")

    def decode():
        R.ops.gated_scan_update(state, x, gx, ga, s, h, slots=slots)
        q = heads(h, wq, Hq)
        R.ops.paged_append(heads(h, wk, Hkv), heads(h, wv, Hkv), *pools, table, lengths, q=q, q_out=q, inv_freq=inv)
        lengths[:B] += 1
        R.ops.paged_attention(q, *pools, table, lengths, out, cap=30.0, window=100)
    kept = state.clone(), lengths.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode()
    torch.cuda.current_stream().wait_stream(side)
    state.copy_(kept[0]), lengths.copy_(kept[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode()
    state.copy_(kept[0]), lengths.copy_(kept[1])
    got = []
    for i in range(steps):
        for buf, k in zip((x, gx, ga), range(3)):
            for b in range(B):
                buf[b] = seqs[b][k][prompts[b] + i]
        graph.replay()
        got.append(out.clone())
    for b, n in enumerate(prompts):
        y, _ = M.gated_scan(*(t[None] for t in seqs[b]), s)
        pos = torch.arange(n + steps, device="cuda")
        k = M.rotated((y[0] @ wk.double()).view(-1, Hkv, N), pos, inv, False, 1.0)
        v = (y[0] @ wv.double()).view(-1, Hkv, N)
        q = M.rotated((y[0] @ wq.double()).view(-1, Hq, N), pos, inv, False, 1.0)
        for i in range(steps):
            o = M.attention(q[n + i], k[:n + i + 1], v[:n + i + 1], N ** -0.5, 30.0, None, 100)[0]
            torch.testing.assert_close(got[i][b].double(), o, rtol=2e-4, atol=2e-4)   # fp32 layers of unit size, sums of 128 terms
    assert (out[3] == 0).all() and (state[[1, 3]] == 7.0).all()

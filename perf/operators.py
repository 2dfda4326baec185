"""What decoders with more than one kind of layer call beside the RWKV operators, and how it is measured: the gated linear
recurrence and the attention over a paged key-value cache, over the sizes that training and serving programs call them at.

A case names an operator ("op"), the activation type and the sizes:

  scan      gated linear recurrence, training step (forward, then the gradients of every input), with a state in and out
  prompt    the same, forward only, as a prompt is read at inference
  update    its step of one new token per sequence, on states that lie in slots of a pool
  append    new tokens go into the cache: q and k rotated by their positions, k and v written into the pages
  attend    attention of one new token per sequence over the pages

`run` computes the plain form (elementary torch operations in fp32) unless `own` is set: then it calls rwkv_cuda_b200.

The recurrence, per channel c and token t:
    L = s[c] sigmoid(ga)    a = exp(-L)    beta = sqrt(1 - a^2)    u = sigmoid(gx) x    h_t = a h_{t-1} + beta u    y_t = h_t
and at tokens that begin a document (`first`) a = 0, beta = 1.  The attention, per head, over the tokens j of a sequence of
`len` tokens (the last `window` of them if window > 0):
    z_j = scale q.k_j    z_j = cap tanh(z_j / cap) if cap > 0    z_j += slope (j - (len - 1))    softmax, then the sum of v_j
"""
import math

import torch

own = False

BF16, F32 = "bf16", "f32"


def listed():
    return [
        # fine-tuning a small model on short sequences, of a length that is no multiple of anything
        dict(name="scan train small", op="scan", dtype=BF16, B=2, T=1040, C=768, docs=False),
        # fp32 training on packed documents
        dict(name="scan train fp32 documents", op="scan", dtype=F32, B=8, T=512, C=1024, docs=True),
        # an ordinary training batch of a large model
        dict(name="scan train B8 T4096", op="scan", dtype=BF16, B=8, T=4096, C=4096, docs=False),
        # one long sequence of packed documents: few channels for the width of the GPU, many tokens
        dict(name="scan train T32768", op="scan", dtype=BF16, B=1, T=32768, C=2048, docs=True),
        # one prompt of a length that nobody padded
        dict(name="scan prompt T1999", op="prompt", dtype=BF16, B=1, T=1999, C=2048, docs=False),
        # one sequence being decoded: launch latency is all there is
        dict(name="scan update B1", op="update", dtype=BF16, B=1, C=768, pool=1),
        # a decoding step of a serving batch that is padded to 256 rows
        dict(name="scan update B256", op="update", dtype=BF16, B=256, C=4096, pool=512),
        # a decoding step writes one token per sequence
        dict(name="append decode B128", op="append", dtype=BF16, B=128, Hq=32, Hkv=8, N=128, R=128, page=16, new=1, most=4096,
             interleaved=False),
        # prompts of different lengths, behind one another, half of each head rotated
        dict(name="append prompts", op="append", dtype=BF16, B=8, Hq=32, Hkv=32, N=64, R=32, page=64, new=2048, most=32768,
             interleaved=True),
        # one short fp32 sequence, a head of its own for every query head
        dict(name="attend B1 fp32", op="attend", dtype=F32, B=1, Hq=12, Hkv=12, N=64, page=16, most=1000, cap=0.0, window=0,
             bias=False),
        # a serving batch of sequences of very different lengths, grouped heads
        dict(name="attend B128", op="attend", dtype=BF16, B=128, Hq=32, Hkv=8, N=128, page=16, most=4096, cap=0.0, window=0,
             bias=False),
        # one long sequence: the length has to be split; capped scores and a bias that depends on the distance
        dict(name="attend T131001", op="attend", dtype=BF16, B=1, Hq=32, Hkv=8, N=128, page=48, most=131001, cap=30.0, window=0,
             bias=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "prompt", "update", "append", "attend", "attend"])
    dtype = rng.choice([BF16, BF16, F32])
    if op in ("scan", "prompt"):
        while True:
            c = dict(op=op, dtype=dtype, B=_log_int(rng, 1, 16), T=_log_int(rng, 1, 32768), C=_log_int(rng, 64, 4096),
                     docs=rng.random() < 0.5)
            if rng.random() < 0.7:
                c["C"] = (c["C"] + 63) // 64 * 64
            if (1 << 16) <= c["B"] * c["T"] * c["C"] <= 8 * 4096 * 4096 // (2 if dtype == F32 else 1):
                return c
    if op == "update":
        B = _log_int(rng, 1, 256)
        return dict(op=op, dtype=dtype, B=B, C=_log_int(rng, 64, 4096), pool=B + rng.randrange(B + 1))
    Hkv, group = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([1, 2, 4, 6, 8, 16])
    heads = dict(Hq=min(64, Hkv * group) // Hkv * Hkv, Hkv=Hkv, N=rng.choice([64, 64, 128, 128, 80, 33]),
                 page=rng.choice([16, 16, 32, 64, 256, 7]))
    if op == "append":
        new = rng.choice([1, _log_int(rng, 2, 1024)])
        N = heads["N"]
        while True:
            c = dict(op=op, dtype=dtype, B=_log_int(rng, 1, 128 if new == 1 else 16), **heads, new=new, most=_log_int(rng, 2048, 32768),
                     R=rng.choice([N, N // 2, N // 4]) // 2 * 2, interleaved=rng.random() < 0.5)
            if c["B"] * c["most"] * c["Hkv"] * N <= 128 * 4096 * 8 * 128:     # (the pool)
                return c
    while True:
        c = dict(op=op, dtype=dtype, B=_log_int(rng, 1, 128), **heads, most=_log_int(rng, 1, 131072),
                 cap=rng.choice([0.0, 0.0, 30.0]), window=rng.choice([0, 0, 1024]), bias=rng.random() < 0.3)
        # (a plain form reads the whole capacity of every sequence)
        if c["B"] * c["most"] * c["Hkv"] * c["N"] <= 128 * 4096 * 8 * 128 // (2 if dtype == F32 else 1):
            return c


def _lengths(case):
    """(tokens in the cache, new tokens) of each sequence: lengths spread evenly up to the most, new tokens up to the most of
    those, in an order that `prepare` shuffles."""
    B, most, new = case["B"], case["most"], case.get("new", 0)
    counts = [max(1, new - new * (b * 5 % B) // B) if new else 0 for b in range(B)]
    return [(max(0, -(-most * (B - b) // B) - c), c) for b, c in enumerate(counts)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, B = case["op"], case["B"]
    dt = torch.bfloat16 if case["dtype"] == BF16 else torch.float32
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    st = dict(case)
    if op in ("scan", "prompt", "update"):
        C = case["C"]
        T = case.get("T", 1)
        # decays of 0.9 to 0.999 to the power 8 sigmoid(ga)
        st["s"] = -8 * torch.log(0.9 + 0.099 * torch.rand(C, device="cuda", generator=g))
        st["x"], st["gx"], st["ga"] = (rn(B, T, C).to(dt) if op != "update" else rn(B, C).to(dt) for _ in range(3))
        if op == "update":
            pool = case["pool"]
            st["state"] = rn(pool, C)
            st["y"] = torch.zeros(B, C, dtype=dt, device="cuda")
            st["slots"] = torch.randperm(pool, device="cuda", generator=g)[:B].int()
            st["slots"][B - B // 16:] = -1          # rows that only pad the batch
            return st
        st["h0"] = rn(B, C)
        # documents of 500 tokens on average
        st["first"] = (torch.rand(B, T, device="cuda", generator=g) < 1 / 500).to(torch.uint8) if case["docs"] else None
        if op == "scan":
            st["dy"], st["dhT"] = rn(B, T, C).to(dt), rn(B, C)
            for n in ("x", "gx", "ga", "s", "h0"):
                st[n].requires_grad_(True)
        return st
    Hq, Hkv, N, page, most = (case[n] for n in ("Hq", "Hkv", "N", "page", "most"))
    width = -(-most // page)
    # sequences of different lengths in any order; the pages of a sequence lie anywhere in the pool
    lengths, count = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[torch.randperm(B, device="cuda", generator=g)].unbind(1)
    st["lengths"] = lengths.contiguous()
    if op == "append":
        st["cu"] = torch.nn.functional.pad(count.cumsum(0), (1, 0)).int()
        M = int(st["cu"][-1])
    used = (lengths + count + page - 1) // page
    at = torch.nn.functional.pad(used.cumsum(0), (1, 0)).long()
    pages = int(at[-1])
    ids = torch.randperm(pages, device="cuda", generator=g)
    cols = torch.arange(width, device="cuda")
    st["table"] = torch.where(cols < used[:, None], ids[(at[:-1, None] + cols).clamp_(max=pages - 1)], 0).int()
    st["k_pages"], st["v_pages"] = (torch.empty(pages, Hkv, page, N, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2))
    if op == "append":
        st["q"], st["k"], st["v"] = rn(M, Hq, N).to(dt), rn(M, Hkv, N).to(dt), rn(M, Hkv, N).to(dt)
        st["inv_freq"] = 10000.0 ** (-torch.arange(0, case["R"], 2, device="cuda") / max(1, case["R"])).float()
        st["q_out"] = torch.empty_like(st["q"])
    else:
        st["q"] = rn(B, Hq, N).to(dt)
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1, device="cuda") / Hq).float() if case["bias"] else None
    return st


# ---- plain forms -------------------------------------------------------------------------------------------------
def _linear_scan(a, b, dim):
    """h_t = a_t h_{t-1} + b_t along `dim`, h_{-1} = 0, by doubling."""
    T, n = a.shape[dim], 1
    while n < T:
        a0, b0 = a.narrow(dim, 0, T - n), b.narrow(dim, 0, T - n)
        a1, b1 = a.narrow(dim, n, T - n), b.narrow(dim, n, T - n)
        b = torch.cat([b.narrow(dim, 0, n), b1 + a1 * b0], dim)
        a = torch.cat([a.narrow(dim, 0, n), a1 * a0], dim)
        n *= 2
    return b


def _gates(st):
    x, gx, ga = (st[n].float() for n in ("x", "gx", "ga"))
    L = st["s"] * torch.sigmoid(ga)
    a, beta = torch.exp(-L), torch.sqrt(-torch.expm1(-2 * L))
    if st.get("first") is not None:
        f = st["first"].bool()[..., None]
        a, beta = a.masked_fill(f, 0.0), beta.masked_fill(f, 1.0)
    return x, torch.sigmoid(gx), torch.sigmoid(ga), L, a, beta


def _scan_forward(st):
    x, i, r, L, a, beta = _gates(st)
    b = beta * i * x
    b = torch.cat([a[:, :1] * st["h0"][:, None] + b[:, :1], b[:, 1:]], 1)
    return _linear_scan(a, b, 1)


@torch.no_grad()
def _plain_scan(st):
    dt = st["x"].dtype
    h = _scan_forward(st)
    x, i, r, L, a, beta = _gates(st)
    before = torch.cat([st["h0"][:, None], h[:, :-1]], 1)
    dy = st["dy"].float()
    dy = torch.cat([dy[:, :-1], dy[:, -1:] + st["dhT"][:, None]], 1)
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    G = _linear_scan(later.flip(1), dy.flip(1), 1).flip(1)
    u = i * x
    # d beta / d L = a^2 / beta; 0 at a document's first token and where L is 0
    slope = torch.where((beta > 0) & (a > 0), a * a / beta, 0.0)
    dL = G * (u * slope - a * before)
    dga, ds = dL * L * (1 - r), (dL * r).sum((0, 1), dtype=torch.float64).float()
    dgx, dx = G * beta * u * (1 - i), G * beta * i
    return h.to(dt), h[:, -1], dx.to(dt), dgx.to(dt), dga.to(dt), ds, a[:, 0] * G[:, 0]


@torch.no_grad()
def _plain_update(st):
    live = st["slots"] >= 0
    slot = st["slots"][live].long()
    x, i, r, L, a, beta = _gates(st)
    h = a[live] * st["state"][slot] + (beta * i * x)[live]
    st["state"][slot] = h
    st["y"][live] = h.to(st["y"].dtype)
    return st["y"], st["state"]


def _rotated(x, cos, sin, interleaved):
    R = 2 * cos.shape[-1]
    f = x.float()
    a, b = (f[..., 0:R:2], f[..., 1:R:2]) if interleaved else (f[..., : R // 2], f[..., R // 2: R])
    c, s = cos[:, None], sin[:, None]
    p, q = a * c - b * s, a * s + b * c
    head = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([head, f[..., R:]], -1).to(x.dtype)


def _places(st):
    """Sequence and position of every new token, and its page and place there."""
    t = torch.arange(st["k"].shape[0], device="cuda")
    seq = torch.searchsorted(st["cu"][1:], t, right=True)
    pos = st["lengths"][seq] + t - st["cu"][seq]
    return pos, st["table"][seq, pos // st["page"]].long(), (pos % st["page"]).long()


def _plain_append(st):
    pos, page, place = _places(st)
    angle = pos.double()[:, None] * st["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    st["k_pages"][page, :, place] = _rotated(st["k"], cos, sin, st["interleaved"])
    st["v_pages"][page, :, place] = st["v"]
    st["q_out"].copy_(_rotated(st["q"], cos, sin, st["interleaved"]))
    return st["q_out"], st["k_pages"], st["v_pages"]


def _plain_attend(st):
    B, Hq, N = st["q"].shape
    Hkv, page = st["k_pages"].shape[1:3]
    at = st["table"].long()
    k = st["k_pages"][at].transpose(2, 3).reshape(B, -1, Hkv, N).float()
    z = torch.einsum("bhgn,bthn->bhgt", st["q"].float().view(B, Hkv, Hq // Hkv, N), k) / math.sqrt(N)
    del k
    if st["cap"] > 0:
        z = st["cap"] * torch.tanh(z / st["cap"])
    j, last = torch.arange(z.shape[-1], device="cuda"), st["lengths"][:, None, None, None] - 1
    if st["slopes"] is not None:
        z = z + st["slopes"].view(Hkv, -1, 1) * (j - last)
    out = (j > last) | (j <= last - st["window"]) if st["window"] > 0 else j > last
    z = z.masked_fill(out, -math.inf)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - m)
    total = p.sum(-1, keepdim=True)
    v = st["v_pages"][at].transpose(2, 3).reshape(B, -1, Hkv, N).float()
    o = torch.einsum("bhgt,bthn->bhgn", p / total, v)
    return o.reshape(B, Hq, N).to(st["q"].dtype), (m + torch.log(total)).reshape(B, Hq)


# ---- the framework's calls ---------------------------------------------------------------------------------------
def _own(st):
    import rwkv_cuda_b200 as R
    op = st["op"]
    if op == "scan":
        ins = [st[n] for n in ("x", "gx", "ga", "s", "h0")]
        out = R.functions.GATED_SCAN.apply(*ins, st["first"])
        return (*out, *torch.autograd.grad(out, ins, (st["dy"], st["dhT"])))
    if op == "prompt":
        y, hT = torch.empty_like(st["x"]), torch.empty_like(st["h0"])
        R.ops.gated_scan_forward(st["x"], st["gx"], st["ga"], st["s"], y, h0=st["h0"], hT=hT, first=st["first"])
        return y, hT
    if op == "update":
        R.ops.gated_scan_update(st["state"], st["x"], st["gx"], st["ga"], st["s"], st["y"], slots=st["slots"])
        return st["y"], st["state"]
    if op == "append":
        R.ops.paged_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], cu_seqlens=st["cu"], q=st["q"],
                           q_out=st["q_out"], inv_freq=st["inv_freq"], interleaved=st["interleaved"])
        return st["q_out"], st["k_pages"], st["v_pages"]
    out, lse = torch.empty_like(st["q"]), torch.empty(st["q"].shape[:2], device="cuda")
    R.ops.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], out, lse=lse, cap=st["cap"],
                          window=st["window"], slopes=st["slopes"])
    return out, lse


def run(st):
    if own:
        return _own(st)
    op = st["op"]
    if op == "scan":
        return _plain_scan(st)
    if op == "prompt":
        h = _scan_forward(st)
        return h.to(st["x"].dtype), h[:, -1].contiguous()
    if op == "update":
        return _plain_update(st)
    return _plain_append(st) if op == "append" else _plain_attend(st)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    """Bytes: each input read once and each output written once; a training step reads the forward's inputs in the backward
    again.  Operations: those of the formulas, a function (exp, sqrt, a division) as one."""
    op, B = case["op"], case["B"]
    e = 2 if case["dtype"] == BF16 else 4
    if op in ("scan", "prompt"):
        n, rows = B * case["T"] * case["C"], B * case["C"]
        docs = B * case["T"] if case["docs"] else 0
        if op == "prompt":
            return dict(bytes=4 * e * n + 8 * rows + 4 * case["C"] + docs, flops=16 * n)
        return dict(bytes=11 * e * n + 20 * rows + 12 * case["C"] + 2 * docs, flops=48 * n)
    if op == "update":
        rows = B - B // 16
        return dict(bytes=rows * case["C"] * (8 + 4 * e) + 4 * case["C"] + 4 * B, flops=16 * rows * case["C"])
    Hq, Hkv, N, R = case["Hq"], case["Hkv"], case["N"], case.get("R", 0)
    if op == "append":
        M = sum(c for _, c in _lengths(case))
        return dict(bytes=2 * e * M * (Hq + 2 * Hkv) * N + 8 * B, flops=3 * M * (Hq + Hkv) * R)
    tokens = sum(min(n, case["window"] or n) for n, _ in _lengths(case))
    return dict(bytes=2 * e * tokens * Hkv * N + 2 * e * B * Hq * N + 4 * B * Hq + 4 * tokens / case["page"],
                flops=4 * tokens * Hq * N + 4 * tokens * Hq)


# ---- 64 bits -------------------------------------------------------------------------------------------------------
def _exact_scan(st, gradients):
    """Token by token."""
    x, gx, ga, s, h0 = (st[n].detach().double() for n in ("x", "gx", "ga", "s", "h0"))
    B, T, C = x.shape
    sig = lambda v: 1 / (1 + torch.exp(-v))
    first = st["first"].bool() if st["first"] is not None else torch.zeros(B, T, dtype=torch.bool, device="cuda")
    decay = lambda t: torch.where(first[:, t, None], 0.0, torch.exp(-s * sig(ga[:, t])))
    width = lambda t: torch.where(first[:, t, None], 1.0, (-torch.expm1(-2 * s * sig(ga[:, t]))).sqrt())
    h, hs = h0, torch.empty(B, T, C, dtype=torch.float64, device="cuda")
    for t in range(T):
        h = decay(t) * h + width(t) * sig(gx[:, t]) * x[:, t]
        hs[:, t] = h
    if not gradients:
        return hs, h
    dx, dgx, dga = (torch.empty_like(hs) for _ in range(3))
    ds, G = torch.zeros_like(s), st["dhT"].double()
    for t in reversed(range(T)):
        G = G + st["dy"][:, t].double()
        r, i, a, w, before = sig(ga[:, t]), sig(gx[:, t]), decay(t), width(t), hs[:, t - 1] if t else h0
        dx[:, t] = G * w * i
        dgx[:, t] = dx[:, t] * x[:, t] * (1 - i)
        dlog = torch.where(first[:, t, None], 0.0, a * a / w * i * x[:, t] - a * before) * G
        dga[:, t] = dlog * s * r * (1 - r)
        ds += (dlog * r).sum(0)
        G = a * G
    return hs, h, dx, dgx, dga, ds, G


def _exact_append(st):
    pos, page, place = _places(st)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double()[:, None] * st["inv_freq"].double())[:, None]
    R = 2 * turn.shape[-1]

    def rotated(x):
        x = x.double()
        pairs = x[..., :R].unflatten(-1, (-1, 2)) if st["interleaved"] else x[..., :R].unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return torch.cat([z.flatten(-2) if st["interleaved"] else z.transpose(-1, -2).flatten(-2), x[..., R:]], -1)

    k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
    k_pages[page, :, place], v_pages[page, :, place] = rotated(st["k"]), st["v"].double()
    return rotated(st["q"]), k_pages, v_pages


def _exact_attend(st):
    B, Hq, N = st["q"].shape
    Hkv, page = st["k_pages"].shape[1:3]
    out, lse = torch.empty(B, Hq, N, dtype=torch.float64, device="cuda"), torch.empty(B, Hq, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lengths"].tolist()):
        start = max(0, n - st["window"]) if st["window"] else 0
        j = torch.arange(start, n, device="cuda")
        at = st["table"][b].long()[j // page]
        k, v = (p[at, :, j % page].double().repeat_interleave(Hq // Hkv, 1) for p in (st["k_pages"], st["v_pages"]))
        z = (k * st["q"][b].double()).sum(-1) * N ** -0.5
        if st["cap"] > 0:
            z = st["cap"] * torch.tanh(z / st["cap"])
        if st["slopes"] is not None:
            z = z + st["slopes"].double() * (j - (n - 1))[:, None]
        lse[b] = torch.logsumexp(z, 0)
        out[b] = (torch.exp(z - lse[b])[..., None] * v).sum(0)
    return out, lse


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op in ("scan", "prompt"):
            return _exact_scan(st, op == "scan")
        if op == "append":
            return _exact_append(st)
        if op == "attend":
            return _exact_attend(st)
        y, state = st["y"].double(), st["state"].double()
        for b, slot in enumerate(st["slots"].tolist()):
            if slot >= 0:
                L = st["s"].double() / (1 + torch.exp(-st["ga"][b].double()))
                u = st["x"][b].double() / (1 + torch.exp(-st["gx"][b].double()))
                state[slot] = torch.exp(-L) * state[slot] + (1 - torch.exp(-2 * L)).sqrt() * u
                y[b] = state[slot]
        return y, state

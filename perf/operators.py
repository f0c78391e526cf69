"""Cases of the attention operators around the LUCID solve: sliding-window attention with visible first tokens
(forward, and a training step), appending to a paged key/value cache with the position rotation, and the two
single-token forms that read that cache (windowed softmax attention; the solve's next row with the attention on it).

``run`` computes a case in plain torch (32 bits, rounded once) or, with ``own`` set, through this package."""
import math

import torch

own = False

D = 128
ROPE_BASE = 10000.0


def listed():
    return [
        # One window layer of the prefill harness (8 query heads, 4 key/value heads, window 1024) at its shortest
        # prompt; q, k, v are slices of one projection.
        dict(name="prefill_2k", op="window", dtype="bf16", B=1, Nq=2048, Nk=2048, Hq=8, Hkv=4, window=1024, sinks=0, ragged=False, fused=True),
        # The same layer at the harness's longest prompt, first four tokens kept visible.
        dict(name="prefill_64k_sinks", op="window", dtype="bf16", B=1, Nq=65536, Nk=65536, Hq=8, Hkv=4, window=1024, sinks=4, ragged=False, fused=True),
        # A right-padded batch of odd length whose last chunk attends to keys of earlier chunks; three queries per key head.
        dict(name="chunk_ragged_fp16", op="window", dtype="fp16", B=3, Nq=777, Nk=1537, Hq=6, Hkv=2, window=300, sinks=5, ragged=True, fused=False),
        # A small training step: odd length, right-padded, window shorter than the sequence.
        dict(name="train_1k_ragged_fp16", op="train", dtype="fp16", B=2, Nq=999, Nk=999, Hq=4, Hkv=2, window=256, sinks=4, ragged=True, fused=False),
        # A long-sequence training step of one window layer.
        dict(name="train_16k_sinks", op="train", dtype="bf16", B=1, Nq=16384, Nk=16384, Hq=8, Hkv=4, window=1024, sinks=4, ragged=False, fused=False),
        # A training step of a global layer (full causality), one key head per query head.
        dict(name="train_4k_causal", op="train", dtype="bf16", B=2, Nq=4096, Nk=4096, Hq=8, Hkv=8, window=-1, sinks=0, ragged=False, fused=False),
        # One new token for each of 8 running sequences: the smallest call, latency counts.
        dict(name="append_token_b8", op="append", dtype="bf16", B=8, new=1, ctx=4000, Hq=8, Hkv=4, page=64, ragged=False),
        # Prompts of several sequences written into the cache at once.
        dict(name="append_prompts", op="append", dtype="bf16", B=5, new=9000, ctx=700, Hq=8, Hkv=4, page=64, ragged=True),
        # One sequence, one token, a window layer: the latency of a step.
        dict(name="decode_window_b1", op="decode", dtype="bf16", B=1, ctx=8192, Hq=8, Hkv=4, page=64, window=1024, sinks=4, ragged=False),
        # A batch of sequences of different lengths, every key visible: bandwidth counts.
        dict(name="decode_full_b32", op="decode", dtype="bf16", B=32, ctx=16384, Hq=8, Hkv=4, page=64, window=-1, sinks=0, ragged=True),
        # A LUCID layer's step of one long sequence.
        dict(name="lucid_step_b1_64k", op="lucid", dtype="bf16", B=1, ctx=65536, Hq=8, Hkv=4, page=128, window=-1, sinks=0, ragged=False),
        # A LUCID layer's step of a small batch of odd lengths, small pages.
        dict(name="lucid_step_b12_ragged", op="lucid", dtype="bf16", B=12, ctx=3001, Hq=8, Hkv=4, page=16, window=-1, sinks=0, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "train", "append", "decode", "lucid"])
    Hkv, group = rng.choice([(1, 4), (2, 1), (2, 3), (4, 2), (4, 2), (8, 1), (2, 4), (1, 8)])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), Hkv=Hkv, Hq=Hkv * group, ragged=rng.random() < 0.4)
    if op in ("window", "train"):
        n = _log_int(rng, 1, 32768 if op == "window" else 12000)
        full = n <= 4096 and rng.random() < 0.3
        c.update(B=rng.choice([1, 1, 2, 3]) if n <= 8192 else 1, Nk=n, Nq=n if op == "train" or rng.random() < 0.6 else rng.randint(1, n),
                 window=-1 if full else _log_int(rng, 1, 1500), sinks=0 if full else rng.choice([0, 1, 4, 5, 64, 128]), fused=False)
        c["fused"] = c["Nq"] == c["Nk"] and rng.random() < 0.5
    elif op == "append":
        c.update(B=_log_int(rng, 1, 48), new=_log_int(rng, 1, 6000), ctx=_log_int(rng, 1, 100000), page=rng.choice([16, 32, 64, 128, 256]))
        c["new"] = max(1, min(c["new"], 45000 // c["B"]))
        c["ctx"] = max(1, min(c["ctx"], 200000 // c["B"]))
    else:
        ctx = _log_int(rng, 1, 65536)
        c.update(B=min(_log_int(rng, 1, 96), max(1, 400000 // ctx)), ctx=ctx, page=rng.choice([16, 32, 64, 128, 256]), window=-1, sinks=0)
        if op == "decode" and rng.random() < 0.6:
            c.update(window=_log_int(rng, 1, 4000), sinks=rng.choice([0, 1, 4, 9, 100]))
    return c


# ------------------------------------------------------------------------------------------------- inputs
def _generators(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    return g, h


def _lengths(h, B, most, ragged):
    """Lengths from 1 to `most`; the longest is `most` itself."""
    n = torch.full((B,), most, dtype=torch.int64)
    if ragged and B > 1:
        n[1:] = torch.randint(1, most + 1, (B - 1,), generator=h)
    elif ragged:
        n[0] = torch.randint(max(1, most // 2), most + 1, (1,), generator=h)[0]
    return n


def _new_tokens(case):
    """How many tokens each sequence appends: fixed for a case, so that a step's packed batch keeps its size."""
    h = torch.Generator()
    h.manual_seed(case["B"] * 1000003 + case["new"])
    return _lengths(h, case["B"], case["new"], case["ragged"])


def _pages(h, B, cap, page):
    """A block table over a shuffled pool with some pages of other sequences in it: (table (B, P), pages in the pool)."""
    per = -(-cap // page)
    pool = B * per + 3
    return torch.randperm(pool, generator=h)[: B * per].reshape(B, per).to(torch.int32), pool


def prepare(case, seed):
    g, h = _generators(seed)
    dt = dict(bf16=torch.bfloat16, fp16=torch.float16)[case["dtype"]]
    dev = "cuda"

    def randn(*shape):
        return torch.randn(*shape, device=dev, dtype=torch.float32, generator=g).to(dt)

    B, Hq, Hkv, op = case["B"], case["Hq"], case["Hkv"], case["op"]
    st = dict(op=op)
    if op in ("window", "train"):
        Nq, Nk = case["Nq"], case["Nk"]
        if case["fused"]:
            qkv = randn(B, Nk, Hq + 2 * Hkv, D)
            q, k, v = qkv.split((Hq, Hkv, Hkv), dim=2)
        else:
            q, k, v = randn(B, Nq, Hq, D), randn(B, Nk, Hkv, D), randn(B, Nk, Hkv, D)
        st.update(q=q, k=k, v=v, window=None if case["window"] < 0 else case["window"], sinks=case["sinks"], scale=D ** -0.5,
                  lengths=_lengths(h, B, Nk, True).to(dev, torch.int32) if case["ragged"] else None)
        if op == "train":
            for n in ("q", "k", "v"):
                st[n] = st[n].detach().requires_grad_(True)
            st["dout"] = randn(B, Nq, Hq, D)
        return st
    if op == "append":
        new = _new_tokens(case)
        before = _lengths(h, B, case["ctx"], True) - 1
        table, pool = _pages(h, B, case["ctx"] + case["new"], case["page"])
        T = int(new.sum())
        q, k, v = randn(T, Hq + 2 * Hkv, D).split((Hq, Hkv, Hkv), dim=1)
        cu = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0)))
        i = torch.arange(D // 2, dtype=torch.float64)
        st.update(q=q, k=k, v=v, k_cache=torch.zeros(pool, case["page"], Hkv, D, device=dev, dtype=dt),
                  v_cache=torch.zeros(pool, case["page"], Hkv, D, device=dev, dtype=dt), table=table.to(dev),
                  cache_lens=before.to(dev, torch.int32), cu=cu.to(dev, torch.int32),
                  inv_freq=(ROPE_BASE ** (-2 * i / D)).to(torch.float32).to(dev))
        return st
    lens = _lengths(h, B, case["ctx"], case["ragged"])
    table, pool = _pages(h, B, case["ctx"], case["page"])
    k_cache, v_cache = randn(pool, case["page"], Hkv, D), randn(pool, case["page"], Hkv, D)
    st.update(q=randn(B, Hq, D), table=table.to(dev), lens=lens.to(dev, torch.int32))
    if op == "lucid":
        # keys of unit variance as the harness makes them (fp16: smaller ones, V' would leave its range); the cached
        # V' have the size the solve gives them, exp(-|k|^2 ks^2) times that of V
        ks = D ** -0.25
        if dt == torch.float16:
            k_cache.mul_(0.6)
        v_cache.mul_(torch.exp(-(k_cache.float() * ks).square().sum(-1, keepdim=True)).to(dt))
        st.update(v=randn(B, Hkv, D), k_scale=ks, scale=ks * D ** -0.5)
    else:
        st.update(window=None if case["window"] < 0 else case["window"], sinks=case["sinks"], scale=D ** -0.5)
    st.update(k_cache=k_cache, v_cache=v_cache)
    return st


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_window(q, k, v, window, sinks, scale, lengths):
    """Attention of 32-bit q (B, Nq, Hq, D) on k, v (B, Nk, Hkv, D): chunks of R queries against the L keys that any of
    them may see, and the first `sinks` keys."""
    B, Nq, Hq, _ = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    G, off, dev = Hq // Hkv, Nk - Nq, q.device
    W = Nk if window is None else min(window, Nk)
    S = 0 if window is None else min(sinks, Nk)
    R = max(256, W)
    if Nq <= R or W + R >= Nk:
        R, first, L = Nq, torch.zeros(1, dtype=torch.int64, device=dev), Nk
    else:
        first = off - W + 1 + R * torch.arange(-(-Nq // R), device=dev)
        L = W + R - 1
    C = first.numel()
    q = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, C * R - Nq))
    p = off + torch.arange(C * R, device=dev).reshape(C, R, 1)
    j = first[:, None] + torch.arange(L, device=dev)                                # (C, L)
    s_j = torch.arange(S, device=dev).expand(C, S)
    cols = torch.cat((j, s_j), dim=1)
    jw = j[:, None, :]
    seen = torch.cat(((jw >= 0) & (jw <= p) & (jw > p - W), (s_j[:, None, :] <= p - W).expand(C, R, S)), dim=2)
    n = torch.full((B,), Nk, device=dev) if lengths is None else lengths.long()
    n = n.reshape(B, 1, 1, 1)
    seen = seen & (cols[:, None, :] < n) & (p < n)                                  # (B, C, R, L + S)
    at = cols.clamp(0, Nk - 1)
    kg, vg = k[:, at].permute(0, 1, 3, 2, 4), v[:, at].permute(0, 1, 3, 2, 4)         # (B, C, Hkv, L + S, D)
    qg = q.reshape(B, C, R, Hkv, G, D).permute(0, 1, 3, 4, 2, 5).reshape(B, C, Hkv, G * R, D)
    s = (qg @ kg.transpose(-1, -2) * scale).reshape(B, C, Hkv, G, R, L + S)
    s = s.masked_fill(~seen[:, :, None, None], -math.inf)
    m = s.detach().amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    e = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    o = (e.reshape(B, C, Hkv, G * R, L + S) @ vg).reshape(B, C, Hkv, G, R, D)
    return o.permute(0, 1, 4, 2, 3, 5).reshape(B, C * R, Hq, D)[:, :Nq]


def _plain_append(st):
    tok = torch.arange(st["k"].shape[0], device=st["k"].device)
    seq = torch.searchsorted(st["cu"].long(), tok, right=True) - 1
    pos = st["cache_lens"].long()[seq] + tok - st["cu"].long()[seq]
    angle = pos.double()[:, None] * st["inv_freq"].double()                          # far positions need 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        a, b = x.float().chunk(2, dim=-1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(x.dtype)

    page = st["k_cache"].shape[1]
    rows = st["table"][seq, pos // page].long(), pos % page
    st["k_cache"][rows] = turn(st["k"])
    st["v_cache"][rows] = st["v"]
    return turn(st["q"]), st["k_cache"], st["v_cache"]


def _read_cache(st, j):
    """Rows at positions j (B, L) of the cached keys and values, in 32 bits: (B, Hkv, L, D)."""
    page = st["k_cache"].shape[1]
    at = torch.gather(st["table"].long(), 1, j // page), j % page
    return st["k_cache"][at].float().transpose(1, 2), st["v_cache"][at].float().transpose(1, 2)


def _softmax_weights(s, seen):
    s = s.masked_fill(~seen, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_decode(st):
    q = st["q"].float()
    B, Hq, _ = q.shape
    Hkv = st["k_cache"].shape[2]
    cap = st["table"].shape[1] * st["k_cache"].shape[1]
    n = st["lens"].long()[:, None]
    W = cap if st["window"] is None else min(st["window"], cap)
    S = 0 if st["window"] is None else min(st["sinks"], cap)
    jw = n - W + torch.arange(W, device=q.device)
    js = torch.arange(S, device=q.device).expand(B, S)
    j = torch.cat((jw, js), dim=1)
    seen = torch.cat((jw >= 0, js < n - W), dim=1)
    kk, vv = _read_cache(st, j.clamp(0, cap - 1))
    s = q.reshape(B, Hkv, Hq // Hkv, D) @ kk.transpose(-1, -2) * st["scale"]
    return (_softmax_weights(s, seen[:, None, None]) @ vv).reshape(B, Hq, D).to(st["q"].dtype)


def _plain_lucid(st):
    q, v = st["q"].float(), st["v"].float()
    B, Hq, _ = q.shape
    Hkv = v.shape[1]
    cap = st["table"].shape[1] * st["k_cache"].shape[1]
    last = (st["lens"].long() - 1)[:, None]
    j = torch.arange(cap, device=q.device).expand(B, cap)
    kk, vv = _read_cache(st, j)
    at = last.reshape(B, 1, 1, 1).expand(B, Hkv, 1, D)
    kn = torch.gather(kk, 2, at)
    t = (kn @ kk.transpose(-1, -2))[:, :, 0] * st["k_scale"] ** 2                     # (B, Hkv, cap)
    tn = torch.gather(t, 2, last[:, :, None].expand(B, Hkv, 1))
    w = torch.exp((t - tn).masked_fill((j >= last)[:, None], -math.inf))
    new = torch.exp(-tn) * v - (w[:, :, None] @ vv)[:, :, 0]
    new = new.to(st["v"].dtype)
    page = st["k_cache"].shape[1]
    st["v_cache"][torch.gather(st["table"].long(), 1, last // page)[:, 0], last[:, 0] % page] = new
    vv = torch.scatter(vv, 2, at, new.float()[:, :, None])
    s = q.reshape(B, Hkv, Hq // Hkv, D) @ kk.transpose(-1, -2) * st["scale"]
    o = (_softmax_weights(s, (j <= last)[:, None, None]) @ vv).reshape(B, Hq, D).to(st["q"].dtype)
    return o, st["v_cache"]


def run(state):
    st = state
    op = st["op"]
    if own:
        import lucid_kernels_b200 as lk

        if op in ("window", "train"):
            o = lk.window_attention(st["q"], st["k"], st["v"], window=st["window"], sinks=st["sinks"], scale=st["scale"], lengths=st["lengths"])
            return o if op == "window" else (o.detach(), *torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["dout"]))
        if op == "append":
            q = lk.paged_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"], st["cache_lens"], cu_seqlens=st["cu"],
                                q=st["q"], inv_freq=st["inv_freq"])
            return q, st["k_cache"], st["v_cache"]
        if op == "decode":
            return lk.paged_window_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"], window=st["window"],
                                             sinks=st["sinks"], scale=st["scale"])
        o = lk.paged_lucid_attention(st["q"], st["v"], st["k_cache"], st["v_cache"], st["table"], st["lens"], k_scale=st["k_scale"],
                                     scale=st["scale"])
        return o, st["v_cache"]
    if op in ("window", "train"):
        leaves = [st[n].detach().float().requires_grad_(op == "train") for n in ("q", "k", "v")]
        o = _plain_window(*leaves, st["window"], st["sinks"], st["scale"], st["lengths"])
        dt = st["q"].dtype
        if op == "window":
            return o.to(dt)
        grads = torch.autograd.grad(o, leaves, st["dout"].float())
        return (o.detach().to(dt), *(x.to(dt) for x in grads))
    return dict(append=_plain_append, decode=_plain_decode, lucid=_plain_lucid)[op](st)


# ------------------------------------------------------------------------------------------------- counts
def _pairs(Nq, Nk, window, sinks, n):
    """Visible (query, key) pairs of one sequence of n valid tokens and one query head."""
    p = torch.arange(Nk - Nq, min(n, Nk), dtype=torch.float64) if n > Nk - Nq else torch.zeros(0, dtype=torch.float64)
    if window < 0:
        return float((p + 1).sum())
    near = torch.clamp(p + 1, max=window)
    return float((near + torch.minimum((p + 1 - near), torch.tensor(float(sinks), dtype=torch.float64))).sum())


def work(case):
    """Unknown lengths (drawn from the seed) count with their mean, half of the longest."""
    B, Hq, Hkv, op = case["B"], case["Hq"], case["Hkv"], case["op"]
    mean = (lambda n: n + (B - 1) * (n + 1) / 2 if case["ragged"] and B > 1 else B * n * (0.75 if case["ragged"] else 1.0))
    row = 2.0 * D
    if op in ("window", "train"):
        Nq, Nk = case["Nq"], case["Nk"]
        one = _pairs(Nq, Nk, case["window"], case["sinks"], Nk)
        if case["ragged"]:
            some = sum(_pairs(Nq, Nk, case["window"], case["sinks"], max(1, Nk * i // 16)) for i in range(1, 17)) / 16
            pairs = one + (B - 1) * some if B > 1 else some
        else:
            pairs = B * one
        io = B * (2.0 * Nq * Hq + 2 * Nk * Hkv) * row
        if op == "window":
            return dict(bytes=io, flops=4.0 * D * pairs * Hq)
        return dict(bytes=io + B * (2.0 * Nq * Hq + 2 * Nk * Hkv) * row, flops=14.0 * D * pairs * Hq)
    if op == "append":
        T = float(_new_tokens(case).sum())
        return dict(bytes=2.0 * T * (Hq + 2 * Hkv) * row, flops=6.0 * T * (Hq + Hkv) * D / 2)
    seen = mean(case["ctx"])
    if case["window"] >= 0:
        seen = min(seen, B * min(case["ctx"], case["window"] + case["sinks"]))
    heads = Hq + (Hkv if op == "lucid" else 0)
    return dict(bytes=seen * Hkv * 2 * row + B * (2.0 * Hq + (2 * Hkv if op == "lucid" else 0)) * row, flops=4.0 * D * seen * heads)


# ------------------------------------------------------------------------------------------------- 64 bits
def _exact_rows(st, b, kh, rows):
    """Block of queries `rows` of batch b against key head kh, in 64 bits: q, dout or None, keys' indices, weights."""
    Nq, Nk = st["q"].shape[1], st["k"].shape[1]
    G = st["q"].shape[2] // st["k"].shape[2]
    W = Nk if st["window"] is None else min(st["window"], Nk)
    n = Nk if st["lengths"] is None else int(st["lengths"][b])
    lo, hi = rows[0] + Nk - Nq, rows[1] - 1 + Nk - Nq
    dev = st["q"].device
    a = max(0, lo - W + 1)
    head = min(st["sinks"], a) if st["window"] is not None else 0
    j = torch.cat((torch.arange(head, device=dev), torch.arange(a, hi + 1, device=dev)))
    p = torch.arange(lo, hi + 1, device=dev)[:, None]
    near = j[None] > p - W
    if st["window"] is not None:
        near = near | (j[None] < st["sinks"])
    ok = near & (j[None] <= p) & (j[None] < n) & (p < n)
    qq = st["q"].detach()[b, rows[0]:rows[1], kh * G:(kh + 1) * G].double().transpose(0, 1)
    kk = st["k"].detach()[b, j, kh].double()
    s = torch.where(ok, torch.einsum("grd,ld->grl", qq, kk) * st["scale"], torch.tensor(-math.inf, dtype=torch.float64, device=dev))
    w = torch.where(ok.any(1, keepdim=True), torch.softmax(s, -1), torch.zeros_like(s))
    return qq, kk, j, w


def _exact_window(st, train):
    q, k = st["q"], st["k"]
    B, Nq, Hq, _ = q.shape
    Hkv, G = k.shape[2], Hq // k.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(o), torch.zeros(k.shape, dtype=torch.float64, device=q.device), torch.zeros(k.shape, dtype=torch.float64, device=q.device)
    for b in range(B):
        for kh in range(Hkv):
            hs = slice(kh * G, (kh + 1) * G)
            for r in range(0, Nq, 1024):
                rows = (r, min(Nq, r + 1024))
                qq, kk, j, w = _exact_rows(st, b, kh, rows)
                vv = st["v"].detach()[b, j, kh].double()
                oo = torch.einsum("grl,ld->grd", w, vv)
                o[b, rows[0]:rows[1], hs] = oo.transpose(0, 1)
                if train:
                    do = st["dout"][b, rows[0]:rows[1], hs].double().transpose(0, 1)
                    ds = w * (torch.einsum("grd,ld->grl", do, vv) - (do * oo).sum(-1, keepdim=True)) * st["scale"]
                    dq[b, rows[0]:rows[1], hs] = torch.einsum("grl,ld->grd", ds, kk).transpose(0, 1)
                    dk[b, :, kh].index_add_(0, j, torch.einsum("grl,grd->ld", ds, qq))
                    dv[b, :, kh].index_add_(0, j, torch.einsum("grl,grd->ld", w, do))
    return (o, dq, dk, dv) if train else o


def _exact_append(st):
    def rotated(x, pos):
        f = st["inv_freq"].double()
        z = torch.complex(x[..., : D // 2].double(), x[..., D // 2:].double())
        z = z * torch.polar(torch.ones_like(f), f * pos[:, None]).unsqueeze(1)
        return torch.cat((z.real, z.imag), dim=-1)

    qs, kc, vc = [], st["k_cache"].double(), st["v_cache"].double()
    page, cu = kc.shape[1], st["cu"].tolist()
    for b in range(len(cu) - 1):
        t = slice(cu[b], cu[b + 1])
        pos = torch.arange(cu[b + 1] - cu[b], device=kc.device, dtype=torch.float64) + float(st["cache_lens"][b])
        i = pos.long()
        pg = st["table"][b].long()[i // page]
        qs.append(rotated(st["q"][t], pos))
        kc[pg, i % page] = rotated(st["k"][t], pos)
        vc[pg, i % page] = st["v"][t].double()
    return torch.cat(qs), kc, vc


def _exact_step(st, lucid):
    q, vc = st["q"], st["v_cache"].double() if lucid else None
    Hkv = st["k_cache"].shape[2]
    G, page = q.shape[1] // Hkv, st["k_cache"].shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b in range(q.shape[0]):
        n = int(st["lens"][b])
        pg = st["table"][b, : -(-n // page)].long()
        kk = st["k_cache"][pg].flatten(0, 1)[:n].double()
        vv = st["v_cache"][pg].flatten(0, 1)[:n].double()
        if lucid:
            t = torch.einsum("hd,lhd->lh", kk[-1], kk) * st["k_scale"] ** 2
            vv[-1] = torch.exp(-t[-1])[:, None] * st["v"][b].double() - torch.einsum("lh,lhd->hd", torch.exp(t[:-1] - t[-1]), vv[:-1])
            vc[pg[-1], (n - 1) % page] = vv[-1]
        elif st["window"] is not None and n > st["window"]:
            keep = torch.arange(n, device=q.device)
            keep = (keep >= n - st["window"]) | (keep < st["sinks"])
            kk, vv = kk[keep], vv[keep]
        s = torch.einsum("hgd,lhd->hgl", q[b].double().reshape(Hkv, G, D), kk) * st["scale"]
        o[b] = torch.einsum("hgl,lhd->hgd", torch.softmax(s, -1), vv).reshape(-1, D)
    return (o, vc) if lucid else o


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("window", "train"):
            return _exact_window(st, case["op"] == "train")
        if case["op"] == "append":
            return _exact_append(st)
        return _exact_step(st, case["op"] == "lucid")

"""Sliding-window attention with visible first keys (forward, backward), the paged cache and its single-token readers,
against plain 64-bit formulas.

Tolerances.  u = finfo(dtype).eps / 2 is the unit roundoff of the 16-bit type.  The kernels keep scores, statistics and
sums in fp32; what they round to 16 bits is (a) the weights P (or dS) before the second product and (b) the result.
(b) is off by at most u |result|.  (a): each weight is off by at most u times itself, so a sum of weights times values is off
by at most u * (the same sum with absolute values).  fp32 parts (2^-24 per operation, at most ~2^12 of them, and ex2.approx
at 2 ulp on arguments off by 2^-24 * |score|) stay below u / 4 of the same bound sums for the sizes here.  So every
comparison is elementwise |got - ref| <= 1.25 u * bound + u |ref|, with `bound` the sum of absolute values that the formula
itself gives, evaluated in 64 bits; for gradients dS itself carries P's and delta's errors, counted where they arise."""
import math
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
D = 128
gpu = pytest.mark.gpu


def unit(dt):
    return torch.finfo(dt).eps / 2


# ------------------------------------------------------------------------------------------------ references
def visible(Nq, Nk, window, sinks, n, device="cpu"):
    p = torch.arange(Nq, device=device)[:, None] + Nk - Nq
    j = torch.arange(Nk, device=device)[None]
    near = (j > p - window) if window is not None else torch.ones(1, 1, dtype=torch.bool, device=device)
    first = (j < sinks) if window is not None else torch.zeros(1, 1, dtype=torch.bool, device=device)
    return (j <= p) & (near | first) & (j < n) & (p < n)


def reference(q, k, v, window, sinks, scale, lengths, dout=None):
    """Output, lse and gradients in 64 bits, each with the sum of absolute values that its rounding errors scale with."""
    B, Nq, Hq, _ = q.shape
    Nk, Hkv = k.shape[1:3]
    G = Hq // Hkv
    out, bound = torch.zeros(B, Nq, Hq, D, dtype=torch.float64, device=q.device), torch.zeros(B, Nq, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq, Nq), -math.inf, dtype=torch.float64, device=q.device)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)] if dout is not None else None
    gb = [torch.zeros_like(g) for g in grads] if dout is not None else None
    for b in range(B):
        n = Nk if lengths is None else int(lengths[b])
        ok = visible(Nq, Nk, window, sinks, n, q.device)
        rows = ok.any(1)
        for h in range(Hq):
            hk = h // G
            qq, kk, vv = (torch.where(torch.isfinite(t), t, torch.zeros_like(t)).double() for t in (q[b, :, h], k[b, :, hk], v[b, :, hk]))
            s = (qq @ kk.T * scale).masked_fill(~ok, -math.inf)
            lse[b, h] = torch.logsumexp(s, -1)
            P = torch.where(ok, torch.exp(s - torch.where(rows, lse[b, h], torch.zeros_like(lse[b, h]))[:, None]), torch.zeros_like(s))
            out[b, :, h] = P @ vv
            bound[b, :, h] = P @ vv.abs()
            if dout is not None:
                do = torch.where(torch.isfinite(dout[b, :, h]), dout[b, :, h], torch.zeros_like(dout[b, :, h])).double()
                dP = do @ vv.T
                delta = (do * out[b, :, h]).sum(-1, keepdim=True)
                dS = P * (dP - delta)
                # delta is formed from the rounded output: off by u * (|do| . |out|), and by what the output's own
                # weights' rounding adds, u * (|do| . bound)
                dd = (do.abs() * (out[b, :, h].abs() + 1.25 * bound[b, :, h])).sum(-1, keepdim=True)
                eS = dS.abs() + P * dd
                grads[0][b, :, h] = scale * dS @ kk
                gb[0][b, :, h] = scale * eS @ kk.abs()
                grads[1][b, :, hk] += scale * dS.T @ qq
                gb[1][b, :, hk] += scale * eS.T @ qq.abs()
                grads[2][b, :, hk] += P.T @ do
                gb[2][b, :, hk] += P.T @ do.abs()
    return out, bound, lse, grads, gb


def close(got, ref, bound, dt, what=""):
    u = unit(dt)
    tiny = torch.finfo(dt).tiny if dt == torch.float16 else 0.0     # fp16 results below its normal range round in steps of 2^-24
    lim = 1.25 * u * bound + u * ref.abs() + u * tiny + 1e-30
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    bad = err > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).max()):.3f} times the bound"


def make(B, Nq, Nk, Hq, Hkv, dt, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)
    return rnd(B, Nq, Hq, D), rnd(B, Nk, Hkv, D), rnd(B, Nk, Hkv, D), rnd(B, Nq, Hq, D)


# ------------------------------------------------------------------------------------------------ host side
def test_positions_a_single_token_query_sees(tmp_path):
    import shutil

    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path / "paged_visible")
    subprocess.run([gxx, "-O2", "-std=c++17", "-I", os.path.join(ROOT, "lucid_kernels_b200", "csrc"), "-o", exe,
                    os.path.join(ROOT, "tests", "host", "paged_visible.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert out.stdout.startswith("ok ")


def test_entries_of_split_lists_are_in_order(tmp_path):
    import shutil

    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path / "attn_entries")
    subprocess.run([gxx, "-O2", "-std=c++17", "-I", os.path.join(ROOT, "lucid_kernels_b200", "csrc"), "-o", exe,
                    os.path.join(ROOT, "tests", "host", "attn_entries.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert out.stdout.startswith("ok ")


def test_tile_lists_cover_every_visible_pair_once(tmp_path):
    import shutil

    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path / "attn_tiles")
    subprocess.run([gxx, "-O2", "-std=c++17", "-I", os.path.join(ROOT, "lucid_kernels_b200", "csrc"), "-o", exe,
                    os.path.join(ROOT, "tests", "host", "attn_tiles.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert out.stdout.startswith("ok ")


def test_refusals_of_the_c_entry_points():
    """Every refused argument is refused on the host, before anything is launched (no device needed)."""
    import ctypes

    from lucid_kernels_b200 import _cabi

    lib = _cabi.load()
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 1023) // 1024 * 1024
    I3, I2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
    st, s2 = I3(512 * 1024, 1024, 128), I2(1024, 128)
    byref = ctypes.byref

    def window(Nq=512, Nk=512, Hq=4, Hkv=2, Dh=128, dt=1, w=128, s=0, scale=0.1, qs=st):
        return byref(_cabi.WindowAttnDesc(1, Nq, Nk, Hq, Hkv, Dh, dt, w, s, scale, qs, *[st] * 7))

    def fwd(q=p, out=p, rest=None, **kw):
        return lib.lucid_window_attn_fwd(window(**kw), q, p, p, out, rest, None, None, None)

    assert fwd(Dh=64) == -1 and fwd(Nq=0) == -1 and fwd(Nq=513) == -1 and fwd(s=129) == -1 and fwd(s=-1) == -1
    assert fwd(Hq=3) == -10 and fwd(dt=2) == -2 and fwd(q=None) == -5 and fwd(out=None) == -5 and fwd(q=p + 2) == -3
    assert fwd(scale=0.0) == -13 and fwd(scale=float("nan")) == -13 and fwd(scale=float("inf")) == -13
    assert fwd(qs=I3(512 * 1024, 1028, 128)) == -3 and fwd(qs=I3(512 * 1024, 0, 128)) == -9
    assert fwd(Nk=1 << 29) == -1 and lib.lucid_window_attn_fwd(None, p, p, p, p, None, None, None, None) == -5
    assert fwd(rest=p) == -5                                   # without lse
    assert lib.lucid_window_attn_rest_bytes(window(Nq=300)) == 4 * 3 * 128 * 128 * 2

    def bwd(ws=p, wsb=1 << 40, dk=p, dv=p, lse=p):
        return lib.lucid_window_attn_bwd(window(s=4), p, p, p, p, p, lse, p, p, dk, dv, None, ws, wsb, None)

    assert bwd(ws=None) == -5 and bwd(ws=p + 4) == -3 and bwd(wsb=100) == -4 and bwd(dk=None) == -5 and bwd(lse=None) == -5
    assert lib.lucid_window_attn_bwd_workspace_bytes(window()) == 4 * 512 * 8
    assert lib.lucid_window_attn_bwd_workspace_bytes(window(Hkv=3)) == 0

    def cache(**kw):
        a = dict(k_strides=I3(64 * 256, 256, 128), v_strides=I3(64 * 256, 256, 128), table_stride=4, table_width=4, pages=8, page_rows=64)
        a.update(kw)
        return _cabi.PagedCacheDesc(**a)

    def app(c=None, T=3, cu=p, rot=128, freq=p, q=None, q_out=None, dt=1, k=p, lens=p, kc=p, table=p):
        d = _cabi.PagedAppendDesc(c or cache(), 2, T, 4, 2, 128, rot, 0, dt, s2, s2, s2)
        return lib.lucid_paged_append(byref(d), k, p, q, q_out, kc, p, table, lens, cu, freq, None)

    assert app(T=0) == -1 and app(cu=None) == -1 and app(rot=120) == -12 and app(rot=144) == -12 and app(dt=5) == -2
    assert app(k=None) == -5 and app(lens=None) == -5 and app(q=p) == -5 and app(q=p, q_out=p, freq=None) == -5 and app(k=p + 4) == -3
    bad_pages = (dict(page_rows=48), dict(page_rows=0), dict(pages=0), dict(table_width=0), dict(page_rows=131072))
    for bad in bad_pages:
        assert app(cache(**bad)) == -11, bad
    assert app(table=None) == -5 and app(cache(table_stride=3)) == -9 and app(kc=p + 8) == -3
    assert app(cache(k_strides=I3(0, 256, 128))) == -9 and app(cache(table_width=1 << 26, table_stride=1 << 26)) == -1

    def step(Hq=4, Hkv=2, scale=0.1, ws=p, wsb=1 << 40, B=2, c=None, lens=p, s=0, w=100):
        d = _cabi.PagedAttnDesc(c or cache(), B, Hq, Hkv, 128, 1, w, s, scale, 1.0, s2, s2)
        return lib.lucid_paged_window_attn(byref(d), p, p, p, p, p, lens, ws, wsb, None)

    assert step(Hq=5) == -10 and step(scale=-1.0) == -13 and step(B=0) == -1 and step(B=70000) == -1 and step(lens=None) == -5
    assert step(s=-1) == -1 and step(ws=p + 4) == -3 and step(c=cache(page_rows=3)) == -11
    long = cache(table_width=4096, table_stride=4096)
    assert step(c=long, w=-1, ws=None) == -5 and step(c=long, w=-1, wsb=8) == -4

    def lucid(Hq=4, ks=1.0, v=p):
        d = _cabi.PagedAttnDesc(cache(), 2, Hq, 2, 128, 1, -1, 0, 0.1, ks, s2, s2)
        return lib.lucid_paged_lucid_attn(byref(d), p, v, p, p, p, p, p, p, 1 << 40, None)

    assert lucid(Hq=32) == -10 and lucid(ks=0.0) == -13 and lucid(v=None) == -5
    for code in (-10, -11, -12, -13, 4):
        assert lib.lucid_status_string(code) != b"unknown"


def test_refusals_of_the_python_layer():
    from lucid_kernels_b200 import paged_append, paged_lucid_attention, paged_window_attention, window_attention

    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)
    ok = (z(1, 8, 2, D), z(1, 8, 2, D), z(1, 8, 2, D))
    for args, kw, text in [
        ((z(1, 8, 2, 64), z(1, 8, 2, 64), z(1, 8, 2, 64)), {}, "head_dim"),
        ((z(1, 8, 3, D), ok[1], ok[2]), {}, "multiple"),
        ((z(1, 9, 2, D), ok[1], ok[2]), {}, "more queries"),
        ((ok[0], ok[1], z(1, 9, 2, D)), {}, "share"),
        ((ok[0].half(), ok[1], ok[2]), {}, "dtype"),
        (tuple(t.float() for t in ok), {}, "float16"),
        (ok, {}, "CUDA"),
        (ok, dict(window=-1), "window"),
        (ok, dict(window=4, sinks=-1), "sinks"),
    ]:
        with pytest.raises(AssertionError, match=text):
            window_attention(*args, **kw)
    pool, table, lens = z(4, 16, 2, D), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA"):
        paged_append(z(1, 2, D), z(1, 2, D), pool, pool, table, lens)
    with pytest.raises(AssertionError, match="CUDA"):
        paged_window_attention(z(1, 4, D), pool, pool, table, lens)
    with pytest.raises(AssertionError, match="share"):
        paged_lucid_attention(z(1, 4, D), z(1, 2, D), pool, z(4, 16, 1, D), table, lens)


@pytest.mark.parametrize("mode", ["dual", "jvp"])
def test_forward_mode_is_refused(mode):
    """A tangent must not vanish: no operator has a forward-mode derivative.  (A dual tensor does not require a gradient.)"""
    from torch.autograd import forward_ad

    from lucid_kernels_b200 import paged_append, paged_lucid_attention, paged_window_attention, window_attention

    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)
    x, pool, new, row = z(1, 8, 2, D), z(4, 16, 2, D), z(1, 2, D), z(1, 4, D)
    table, lens, freq = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), z(64, dt=torch.float32)
    calls = [
        (x, lambda t: window_attention(t, x, x)), (x, lambda t: window_attention(x, t, x)), (x, lambda t: window_attention(x, x, t)),
        (new, lambda t: paged_append(t, new, pool, pool, table, lens)), (new, lambda t: paged_append(new, t, pool, pool, table, lens)),
        (pool, lambda t: paged_append(new, new, t, pool, table, lens)), (pool, lambda t: paged_append(new, new, pool, t, table, lens)),
        (row, lambda t: paged_append(new, new, pool, pool, table, lens, q=t, inv_freq=freq)),
        (freq, lambda t: paged_append(new, new, pool, pool, table, lens, inv_freq=t)),
        (row, lambda t: paged_window_attention(t, pool, pool, table, lens)), (pool, lambda t: paged_window_attention(row, t, pool, table, lens)),
        (pool, lambda t: paged_window_attention(row, pool, t, table, lens)),
        (row, lambda t: paged_lucid_attention(t, new, pool, pool, table, lens)), (new, lambda t: paged_lucid_attention(row, t, pool, pool, table, lens)),
        (pool, lambda t: paged_lucid_attention(row, new, t, pool, table, lens)), (pool, lambda t: paged_lucid_attention(row, new, pool, t, table, lens)),
    ]
    for at, call in calls:
        with pytest.raises(NotImplementedError, match="forward-mode"), torch.no_grad():
            if mode == "jvp":
                torch.func.jvp(call, (at,), (torch.ones_like(at),))
            else:
                with forward_ad.dual_level():
                    call(forward_ad.make_dual(at, torch.ones_like(at)))
    # inside the mode, tensors without a tangent go their usual way (here to the check of the device)
    with forward_ad.dual_level(), pytest.raises(AssertionError, match="CUDA"):
        window_attention(x, x, x)


def test_cache_operators_refuse_gradients_of_every_input(monkeypatch):
    """(What a call's shapes determine is stubbed: the refusal comes before anything is launched.)"""
    import lucid_kernels_b200.attention as A

    monkeypatch.setattr(A, "_append_plan", lambda *a: A._Plan(A._cabi.PagedAppendDesc(), 0, False, True))
    monkeypatch.setattr(A, "_step_plan", lambda *a: A._Plan(A._cabi.PagedAttnDesc(), 0, False, True))
    monkeypatch.setattr(A, "_plans", {})
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)
    pool, new, row, table, lens = z(4, 16, 2, D), z(1, 2, D), z(1, 4, D), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    append = [new, new.clone(), pool, pool.clone(), row, z(64, dt=torch.float32)]
    step = [row, new, pool, pool.clone()]
    calls = [(append, i, lambda k, v, kc, vc, q, f: A.paged_append(k, v, kc, vc, table, lens, q=q, inv_freq=f)) for i in range(6)] + \
        [(step, i, lambda q, v, kc, vc: A.paged_lucid_attention(q, v, kc, vc, table, lens)) for i in range(4)] + \
        [(step, i, lambda q, v, kc, vc: A.paged_window_attention(q, kc, vc, table, lens)) for i in (0, 2, 3)]
    for inputs, i, call in calls:
        args = [t.clone().requires_grad_(True) if x == i else t for x, t in enumerate(inputs)]
        with pytest.raises(AssertionError, match="no backward"):
            call(*args)


# ------------------------------------------------------------------------------------------------ window attention
SHAPES = [
    # B, Nq, Nk, Hq, Hkv, window, sinks
    (1, 1, 1, 1, 1, None, 0),
    (1, 128, 128, 2, 1, None, 0),
    (2, 257, 257, 4, 2, 64, 0),
    (1, 300, 300, 3, 1, 100, 5),
    (1, 1000, 1000, 2, 2, 128, 128),
    (1, 1, 700, 4, 2, 37, 3),
    (2, 130, 901, 6, 2, 300, 4),
    (1, 513, 640, 8, 1, 1, 0),
    (1, 385, 385, 2, 1, 1, 1),
    (1, 400, 400, 5, 5, None, 0),
    (3, 129, 129, 2, 2, 129, 7),
    (1, 2300, 2300, 2, 1, 250, 9),
    (1, 260, 260, 2, 1, 0, 2),        # first keys only
    (1, 200, 200, 2, 1, 0, 0),        # nothing visible
    # more tiles of queries than SMs: two tiles to an item, several items to a CTA
    (3, 500, 500, 16, 4, 130, 5),
    (3, 500, 500, 15, 5, 200, 100),
    (2, 1000, 1100, 10, 10, None, 0),
    (1, 2500, 2500, 24, 8, 600, 4),
    (2, 2500, 2500, 16, 4, 300, 33),
]


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_window_attention_forward_and_backward(shape, dt):
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    B, Nq, Nk, Hq, Hkv, window, sinks = shape
    q, k, v, do = make(B, Nq, Nk, Hq, Hkv, dt, seed=Nq + Nk)
    scale = D ** -0.5
    ref, bound, lse_ref, grads, gb = reference(q, k, v, window, sinks, scale, None, do)
    out, lse, rest = _window_attention_fwd(q, k, v, window, sinks, scale, check=True)
    close(out, ref, bound, dt, "out")
    close(_window_attention_fwd(q, k, v, window, sinks, scale, training=False, check=True)[0], ref, bound, dt, "out, inference")
    some = torch.isfinite(lse_ref)
    assert torch.equal(torch.isneginf(lse), ~some)
    assert float((lse.double() - lse_ref)[some].abs().max() if some.any() else 0) < 1e-5 * 16
    got = _window_attention_bwd(q, k, v, out, lse, rest, do, window, sinks, scale, check=True)
    for name, x, r, b in zip(("dq", "dk", "dv"), got, grads, gb):
        close(x, r, b, dt, name)


def test_backward_refuses_what_another_forward_kept(monkeypatch):
    """(What the shapes determine is stubbed; the refusal comes before anything is launched.)"""
    import lucid_kernels_b200.attention as A

    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)
    q, k = z(1, 8, 2, D), z(1, 8, 2, D)
    plan = A._Plan(A._cabi.WindowAttnDesc(), q.get_device(), False, True)
    plan.lse_shape, plan.rest, plan.workspace = (1, 2, 8), 8 * 2 * D * 2, 64
    monkeypatch.setattr(A, "_window_plan", lambda *a: plan)
    monkeypatch.setattr(A, "_plans", {})
    monkeypatch.setattr(A, "_device_now", lambda: plan.device)
    lse, rest = z(1, 2, 8, dt=torch.float32), z(plan.rest, dt=torch.uint8)
    for bad_lse, bad_rest in [(z(1, 2, 9, dt=torch.float32), rest), (lse.double(), rest), (lse, rest[:-1]), (lse, z(2 * plan.rest, dt=torch.uint8)),
                              (lse, z(2 * plan.rest, dt=torch.uint8)[::2]), (lse, z(plan.rest))]:
        with pytest.raises(AssertionError, match="must be the forward's"):
            A._window_attention_bwd(q, k, k, q, bad_lse, bad_rest, q)
    A._window_attention_bwd(q, k, k, q, lse, rest, q)
    A._window_attention_bwd(q, k, k, q, lse, None, q)


def test_memory_kept_for_the_backward_is_of_the_size_of_the_result():
    import ctypes

    from lucid_kernels_b200 import _cabi

    st = (ctypes.c_int64 * 3)(1 << 20, 1024, 128)
    for Nq in (1, 2, 100, 127, 128, 129, 300, 4096):
        d = _cabi.WindowAttnDesc(2, Nq, 5000, 6, 2, 128, 1, 300, 4, 0.1, *[st] * 8)
        assert _cabi.load().lucid_window_attn_rest_bytes(ctypes.byref(d)) == 2 * 6 * (Nq if Nq < 128 else -(-Nq // 128) * 128) * 128 * 2


@gpu
@pytest.mark.parametrize("Nq", [1, 3, 8, 100, 127, 128, 129])
def test_rest_stays_inside_its_memory(Nq):
    """What the forward keeps for the backward: nothing is written behind it, whatever stood in it is not read, and gradients
    of a few queries are as accurate as of many."""
    import ctypes

    from lucid_kernels_b200 import _cabi
    from lucid_kernels_b200.attention import _window_attention_bwd

    lib, dt, B, Nk, Hq, Hkv, window, sinks, scale = _cabi.load(), torch.bfloat16, 2, 400, 6, 2, 150, 3, 0.3
    q, k, v, do = make(B, Nq, Nk, Hq, Hkv, dt, seed=Nq)
    st = lambda t: (ctypes.c_int64 * 3)(*t.stride()[:3])
    d = _cabi.WindowAttnDesc(B, Nq, Nk, Hq, Hkv, D, 1, window, sinks, scale, st(q), st(k), st(v), st(q), st(q), st(q), st(k), st(v))
    n = lib.lucid_window_attn_rest_bytes(ctypes.byref(d))
    out, lse = torch.empty_like(q), torch.empty(B, Hq, Nq, device="cuda")
    memory = torch.full((n + 65536,), 255, dtype=torch.uint8, device="cuda")          # (16-bit NaNs)
    assert lib.lucid_window_attn_fwd(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), memory.data_ptr(), lse.data_ptr(),
                                     None, torch.cuda.current_stream().cuda_stream) == 0
    assert bool((memory[n:] == 255).all())
    ref, bound, _, grads, gb = reference(q, k, v, window, sinks, scale, None, do)
    close(out, ref, bound, dt, "out")
    got = _window_attention_bwd(q, k, v, out, lse, memory[:n], do, window, sinks, scale, check=True)
    for name, x, r, b in zip(("dq", "dk", "dv"), got, grads, gb):
        close(x, r, b, dt, name)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("Nq,Nk,Hq,Hkv,window,sinks,lens", [
    (1, 5000, 2, 1, None, 0, None),                       # one tile of queries, eight CTAs on its keys
    (1, 65, 1, 1, None, 0, None),                         # too short to share
    (300, 9000, 3, 1, None, 0, None),                     # nine tiles, eight CTAs each
    (100, 4000, 8, 4, 1024, 4, None),
    (130, 3100, 12, 2, 700, 128, None),                   # two CTAs each
    (128, 1300, 1, 1, 900, 40, None),
    (200, 2600, 2, 2, None, 0, [2600, 0, 1, 2400, 2401]), # no query, no key, the last row of a tile
    (257, 3000, 2, 1, 1500, 3, [3000, 2800, 2999]),
])
def test_few_queries_of_long_sequences(Nq, Nk, Hq, Hkv, window, sinks, lens, dt):
    """Inference: the keys of a tile of queries are dealt out to the CTAs of a cluster.  Stale rows hold NaN."""
    from lucid_kernels_b200 import window_attention

    B = len(lens) if lens else 1
    q, k, v, do = make(B, Nq, Nk, Hq, Hkv, dt, seed=Nq + Nk)
    lengths = None
    if lens:
        lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lens):
            k[b, n:] = v[b, n:] = float("nan")
    scale = D ** -0.5
    with torch.no_grad():
        out = window_attention(q, k, v, window, sinks, scale, lengths)
        again = window_attention(q, k, v, window, sinks, scale, lengths)
    ref, bound = reference(q, torch.nan_to_num(k), torch.nan_to_num(v), window, sinks, scale, lens, do)[:2]
    close(out, ref, bound, dt, "out")
    assert torch.equal(out, again)


@gpu
@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (5, 1), (1, 1)])
@pytest.mark.parametrize("window,sinks,Nq", [(200, 4, 600), (None, 0, 600), (64, 128, 350), (0, 3, 600)])
def test_padded_batch_ignores_whatever_stands_behind_the_sequences(window, sinks, Nq, Hq, Hkv):
    """Lengths from nothing to all, NaN and infinities in every padded position of every input."""
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    dt, Nk = torch.bfloat16, 600
    lens = [600, 0, 1, 127, 128, 129, 257, 599, 300]
    B = len(lens)
    q, k, v, do = make(B, Nq, Nk, Hq, Hkv, dt, seed=3)
    for b, n in enumerate(lens):
        for t in (k, v):
            t[b, n:] = float("nan")
            t[b, n::2] = float("inf")
        for t in (q, do):
            t[b, max(0, n - (Nk - Nq)):] = float("nan")
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scale = 0.07
    ref, bound, lse_ref, grads, gb = reference(q, k, v, window, sinks, scale, lengths, do)
    out, lse, rest = _window_attention_fwd(q, k, v, window, sinks, scale, lengths, check=True)
    close(out, ref, bound, dt, "out")
    close(_window_attention_fwd(q, k, v, window, sinks, scale, lengths, training=False, check=True)[0], ref, bound, dt, "out, inference")
    assert torch.equal(torch.isneginf(lse), torch.isneginf(lse_ref))
    for name, x, r, b in zip(("dq", "dk", "dv"), _window_attention_bwd(q, k, v, out, lse, rest, do, window, sinks, scale, lengths, check=True), grads, gb):
        close(x, r, b, dt, name)
        for i, n in enumerate(lens):
            rows = x[i, max(0, n - (Nk - Nq)):] if name == "dq" else x[i, n:]
            assert not rows.any(), name


@gpu
def test_strided_expanded_and_misaligned_inputs():
    from lucid_kernels_b200 import window_attention

    dt = torch.float16
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    qkv = torch.randn(2, 333, 8, D, device="cuda", generator=g).to(dt)
    q, k, v = qkv.split((4, 2, 2), dim=2)
    want = window_attention(q.contiguous(), k.contiguous(), v.contiguous(), window=90, sinks=2)
    assert torch.equal(window_attention(q, k, v, window=90, sinks=2), want)
    # BHSD-backed, an odd base, a transposed last dimension, one key head expanded over the batch
    assert torch.equal(window_attention(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)), window=90, sinks=2), want)
    raw = torch.empty(q.numel() + 3, dtype=dt, device="cuda")[3:].view(q.shape).copy_(q)
    assert torch.equal(window_attention(raw, k, v, window=90, sinks=2), want)
    turned = q.transpose(1, 3).contiguous().transpose(1, 3)
    assert turned.stride(-1) != 1 and torch.equal(window_attention(turned, k, v, window=90, sinks=2), want)
    k1, v1 = (t[:1].clone().requires_grad_(True) for t in (k, v))
    qg = q.clone().requires_grad_(True)
    do = torch.randn(q.shape, device="cuda", generator=g).to(dt)
    window_attention(qg, k1.expand(2, -1, -1, -1), v1.expand(2, -1, -1, -1), window=90, sinks=2).backward(do)
    kf, vf = (t.detach().repeat(2, 1, 1, 1).requires_grad_(True) for t in (k1, v1))
    q2 = q.clone().requires_grad_(True)
    window_attention(q2, kf, vf, window=90, sinks=2).backward(do)
    assert torch.equal(qg.grad, q2.grad)
    assert torch.equal(k1.grad[0], kf.grad.sum(0)) and torch.equal(v1.grad[0], vf.grad.sum(0))


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape,window,sinks,sharp", [((1, 1, 1, 2, 1), None, 0, 1), ((2, 300, 300, 4, 2), 1, 0, 1), ((1, 200, 260, 3, 3), 0, 1, 1),
                                                      ((1, 400, 400, 4, 2), 2, 0, 1), ((1, 400, 400, 4, 2), 5, 1, 1), ((1, 500, 500, 4, 2), 200, 4, 12)])
def test_gradients_of_rows_with_few_or_peaked_weights(shape, window, sinks, sharp, dt):
    """Where one key has (nearly) all the weight, dS is a difference of nearly equal numbers.  One visible key: exactly 0.
    Otherwise in the 2-norm: dS rounded (u / sqrt 3 on average), the result rounded (the same), and delta from weights
    rounded but normalised, whose error is again at most u times dS's own size: sqrt(3) u / sqrt(3) = u together."""
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    q, k, v, do = make(*shape, dt, seed=31)
    scale = sharp * D ** -0.5
    _, _, _, grads, _ = reference(q, k, v, window, sinks, scale, None, do)
    out, lse, rest = _window_attention_fwd(q, k, v, window, sinks, scale, check=True)
    got = _window_attention_bwd(q, k, v, out, lse, rest, do, window, sinks, scale, check=True)
    for name, x, r in zip(("dq", "dk"), got, grads):
        if float(r.abs().max()) < 1e-12:
            assert not x.any(), name
        else:
            assert float((x.double() - r).norm() / r.norm()) <= unit(dt), name


@gpu
def test_gradient_against_differences():
    """Directional derivatives of the kernel's own forward along one perturbed element block: inputs are exact in 16 bits
    (multiples of 1/8), the step 1/4, central differences; the second-order remainder and the outputs' rounding are bounded
    by the 64-bit reference evaluated at the same two points."""
    from lucid_kernels_b200 import window_attention

    dt, N, W, S = torch.float16, 140, 50, 3
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    q, k, v, do = ((torch.randint(-8, 9, (1, N, h, D), device="cuda", generator=g) / 8).to(dt) for h in (2, 1, 1, 2))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    window_attention(*leaves, window=W, sinks=S).backward(do)
    loss = lambda a, b, c: float((window_attention(a, b, c, window=W, sinks=S).double() * do.double()).sum())
    exact = lambda a, b, c: float((reference(a, b, c, W, S, D ** -0.5, None)[0] * do.double()).sum())
    h = 0.25
    for at in range(3):
        d = (torch.randint(0, 3, leaves[at].shape, device="cuda", generator=g) - 1).to(dt)
        plus, minus = ([t + (h * d if i == at else 0) for i, t in enumerate((q, k, v))], [t - (h * d if i == at else 0) for i, t in enumerate((q, k, v))])
        slope = float((leaves[at].grad.double() * d.double()).sum())
        got = (loss(*plus) - loss(*minus)) / (2 * h)
        curve = (exact(*plus) - exact(*minus)) / (2 * h)              # what differences of this width give in 64 bits
        u = unit(dt)
        rounding = 2.25 * u * 2 * float(do.double().abs().sum()) / (2 * h)        # two losses of |out| <= 1, weights and result
        assert abs(got - curve) <= rounding
        ref = reference(q, k, v, W, S, D ** -0.5, None, do)
        assert abs(slope - float((ref[3][at] * d.double()).sum())) <= float(((1.25 * u * ref[4][at] + u * ref[3][at].abs()) * d.double().abs()).sum())


@gpu
def test_extreme_scores_and_growing_maxima():
    """Scores that span +-600 in base 2 and whose running maximum grows from tile to tile, one row at a time."""
    from lucid_kernels_b200.attention import _window_attention_fwd

    dt, N = torch.bfloat16, 900
    q, k, v, _ = make(1, N, N, 2, 1, dt, seed=11)
    ramp = torch.linspace(0.1, 6.0, N, device="cuda")[None, :, None, None]
    k = (k * ramp).to(dt)
    q = (q * torch.linspace(6.0, 0.1, N, device="cuda")[None, :, None, None]).to(dt)
    for window, sinks in ((None, 0), (400, 2)):
        scale = 1.0
        ref, bound, lse_ref, _, _ = reference(q, k, v, window, sinks, scale, None)
        out, lse, _ = _window_attention_fwd(q, k, v, window, sinks, scale, check=True)
        # a score s carries an fp32 error of up to D products' roundings, 128 * 2^-24 * sum |q||k|, and a weight that
        # relative error: e^delta - 1 with delta <= 2^-17 * sum |q||k|
        size = float((q.double().abs().amax() * k.double().abs().amax()) * 0 + (q.double().norm(dim=-1).amax() * k.double().norm(dim=-1).amax()))
        extra = math.expm1(2 * 2.0 ** -17 * size * scale)
        err = (out.double() - ref).abs()
        assert bool((err <= (1.25 * unit(dt) + extra) * bound + unit(dt) * ref.abs()).all())
        assert float((lse.double() - lse_ref).abs().max()) <= 2.0 ** -17 * size * scale + 1e-4


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("N,drop", [(16384, 25.25), (65536, 20), (65536, 25.25), (65536, 28)])
def test_many_small_weights_beside_a_large_one(N, drop, dt):
    """One key outweighs each of the others by 2^drop, all of them together weigh up to 0.2 % of it: they count, although each
    alone is below what 16 bits hold beside 1."""
    from lucid_kernels_b200 import paged_window_attention
    from lucid_kernels_b200.attention import _window_attention_fwd

    Nq, Hq, scale, page = 128, 160, math.log(2.0), 64
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    q, k = torch.zeros(1, Nq, Hq, D, device="cuda", dtype=dt), torch.zeros(1, N, 1, D, device="cuda", dtype=dt)
    v = (torch.randn(1, N, 1, D, device="cuda", generator=g).abs() + 1).to(dt)
    v[:, 0] = -1
    q[..., 0], k[:, 0, 0, 0] = 1, drop
    s = (q[0, :, 0].double() @ k[0, :, 0].double().T * scale).masked_fill(~visible(Nq, N, None, 0, N, "cuda"), -math.inf)
    P, V = torch.softmax(s, -1), v[0, :, 0].double()
    ref, bound = P @ V, P @ V.abs()
    for heads in (1, 2, Hq):              # keys split or not, one tile of queries or two to a CTA
        for training in (True, False):
            out = _window_attention_fwd(q[:, :, :heads], k, v, scale=scale, training=training, check=True)[0]
            for h in (0, heads - 1):
                close(out[0, :, h], ref, bound, dt, f"{heads} heads, training {training}")
    kc, vc = k.view(N // page, page, 1, D), v.view(N // page, page, 1, D)
    table, n = torch.arange(N // page, device="cuda", dtype=torch.int32)[None], torch.tensor([N], device="cuda", dtype=torch.int32)
    close(paged_window_attention(q[:, -1, :4].contiguous(), kc, vc, table, n, scale=scale, check=True)[0], ref[-1].expand(4, D), bound[-1].expand(4, D), dt, "paged")


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("N,window,sinks", [(20000, None, 0), (65536, None, 0), (40000, 30000, 100)])
def test_gradient_of_values_of_small_weights(N, window, sinks, dt):
    """Alike queries on many keys: each weight is some 2^-16, rounded the same way for every query, and its rounding must
    stay relative to it."""
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    Nq, scale = 256, 0.05
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q = rnd(1, 1, 1, D).expand(1, Nq, 1, D).contiguous().to(dt)
    k, v, do = rnd(1, N, 1, D).to(dt), rnd(1, N, 1, D).to(dt), rnd(1, 1, 1, D).expand(1, Nq, 1, D).contiguous().to(dt)
    s = (q[0, :, 0].double() @ k[0, :, 0].double().T * scale).masked_fill(~visible(Nq, N, window, sinks, N, "cuda"), -math.inf)
    P = torch.softmax(s, -1)
    assert float(P.max()) < 2.0 ** -11 and float(P[P > 0].median()) < 2.0 ** -14
    out, lse, rest = _window_attention_fwd(q, k, v, window, sinks, scale, check=True)
    dv = _window_attention_bwd(q, k, v, out, lse, rest, do, window, sinks, scale, check=True)[2]
    close(dv[0, :, 0], P.T @ do[0, :, 0].double(), P.T @ do[0, :, 0].double().abs(), dt, "dv")


@gpu
@pytest.mark.parametrize("size", [300.0, 700.0, 900.0])
@pytest.mark.parametrize("window,sinks", [(None, 0), (300, 4)])
def test_scores_of_millions_in_fp16_stay_finite(window, sinks, size):
    """Scores of up to 10^7, which fp32 holds to within one: weights are what they may be, but results are means of values, and
    neither they nor gradients are infinite."""
    from lucid_kernels_b200 import paged_window_attention
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    B, N, Hq, Hkv, page = 2, 1024, 4, 2, 64
    sign = lambda *s: torch.randint(0, 2, s, device="cuda", generator=g) * 2.0 - 1
    line = sign(1, 1, 1, D)
    jitter = lambda *s: 1 + 0.02 * torch.randn(*s, device="cuda", generator=g)
    # every key lies along one line, growing along the sequence: maxima keep growing, in small and large steps
    grow = torch.linspace(0.2, 1, N, device="cuda").reshape(1, N, 1, 1)
    q, k = (size * line * jitter(B, N, Hq, 1)).half(), (size * line * grow * jitter(B, N, Hkv, D)).half()
    v, do = (torch.randn(B, N, n, D, device="cuda", generator=g).half() for n in (Hkv, Hq))
    out, lse, rest = _window_attention_fwd(q, k, v, window, sinks, check=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert float(lse.max()) > 0.9 * size ** 2 * D ** 0.5 * 0.9
    top = v.float().abs().amax(dim=1).repeat_interleave(Hq // Hkv, dim=1)[:, None]
    assert bool((out.float().abs() <= top * 1.01).all())
    again = _window_attention_fwd(q, k, v, window, sinks, training=False, check=True)[0]
    assert torch.isfinite(again).all() and bool((again.float().abs() <= top * 1.01).all())
    dv = _window_attention_bwd(q, k, v, out, lse, rest, do, window, sinks, check=True)[2]
    assert torch.isfinite(dv).all()
    kc, vc = k.reshape(B * N // page, page, Hkv, D), v.reshape(B * N // page, page, Hkv, D)
    table = torch.arange(B * N // page, device="cuda", dtype=torch.int32).reshape(B, -1)
    step = paged_window_attention(q[:, -1].contiguous(), kc, vc, table, torch.full((B,), N, device="cuda", dtype=torch.int32), window, sinks, check=True)
    assert torch.isfinite(step).all() and bool((step.float().abs() <= top[:, 0] * 1.01).all())


@gpu
def test_runs_are_identical_and_graphs_replay():
    from lucid_kernels_b200 import window_attention

    dt = torch.bfloat16
    q, k, v, do = make(1, 3000, 3000, 4, 2, dt, seed=21)
    kw = dict(window=500, sinks=4)

    def step(leaves):
        o = window_attention(*leaves, **kw)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    a, b = step(leaves), step(leaves)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    gl = [t.detach().clone().requires_grad_(True) for t in leaves]
    graphs = []
    for _ in range(2):                      # two graphs, replayed in turn: they share no scratch memory
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = step(gl)
        graphs.append((g, r))
    with torch.no_grad():
        gl[1].mul_(0.5)
    want = step([t.detach().clone().requires_grad_(True) for t in gl])
    for g, r in graphs * 2:
        for x in r:
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(r, want))


@gpu
def test_calls_from_a_thread_that_has_made_no_cuda_call():
    """A tensor map can only be made with a current context; a new thread has none until some runtime call gives it one."""
    import threading

    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd
    from lucid_kernels_b200.cute import _forward_sub_bwd, _forward_sub_fwd

    q, k, v, do = make(1, 256, 256, 2, 2, torch.bfloat16)
    calls = [lambda: _window_attention_fwd(q, k, v, 64, 2),
             lambda: _window_attention_bwd(q, k, v, out, lse, rest, do, 64, 2),
             lambda: (_forward_sub_fwd(k * 0.3, v),),
             lambda: _forward_sub_bwd(k * 0.3, v, do)]
    out, lse, rest = calls[0]()
    for call in calls:
        want, got = call(), []
        torch.cuda.synchronize()
        th = threading.Thread(target=lambda: got.append(call()))
        th.start()
        th.join()
        torch.cuda.synchronize()
        assert got and all(torch.equal(x, y) for x, y in zip(want, got[0]))


@gpu
def test_a_thread_may_make_its_first_call_while_a_stream_is_captured():
    import threading

    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    q, k, v, do = make(1, 256, 256, 2, 2, torch.bfloat16)
    want = _window_attention_fwd(q, k, v, 64, 2)
    grads = _window_attention_bwd(q, k, v, *want, do, 64, 2)
    got = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream()

        def work():
            with torch.cuda.stream(stream):
                got.append(_window_attention_bwd(q, k, v, *want, do, 64, 2))

        th = threading.Thread(target=work)
        th.start()
        th.join()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got[0], grads))


@gpu
def test_expired_waits_end_and_are_reported():
    """A wait limit of 0 (a wait that is not satisfied at once has run out): every kernel ends, the error is reported,
    and the next call is right."""
    from lucid_kernels_b200 import _cabi
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    lib = _cabi.load()
    q, k, v, do = make(2, 700, 700, 4, 2, torch.bfloat16)
    out, lse, rest = _window_attention_fwd(q, k, v, 200, 4, check=True)
    grads = _window_attention_bwd(q, k, v, out, lse, rest, do, 200, 4, check=True)
    try:
        lib.lucid_set_wait_limit_ns(0)
        with pytest.raises(_cabi.LucidKernelError, match="timed out"):
            _window_attention_fwd(q, k, v, 200, 4, check=True)
        with pytest.raises(_cabi.LucidKernelError, match="timed out"):
            _window_attention_bwd(q, k, v, out, lse, rest, do, 200, 4, check=True)
    finally:
        lib.lucid_set_wait_limit_ns(2_000_000_000)
    again = _window_attention_fwd(q, k, v, 200, 4, check=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert all(torch.equal(x, y) for x, y in zip(grads, _window_attention_bwd(q, k, v, out, lse, rest, do, 200, 4, check=True)))


@gpu
def test_an_expired_wait_in_a_cluster_ends_it():
    from lucid_kernels_b200 import _cabi
    from lucid_kernels_b200.attention import _window_attention_fwd

    lib = _cabi.load()
    q, k, v, _ = make(1, 200, 4000, 2, 1, torch.bfloat16)
    out = _window_attention_fwd(q, k, v, training=False, check=True)[0]
    try:
        lib.lucid_set_wait_limit_ns(0)
        with pytest.raises(_cabi.LucidKernelError, match="timed out"):
            _window_attention_fwd(q, k, v, training=False, check=True)
    finally:
        lib.lucid_set_wait_limit_ns(2_000_000_000)
    assert torch.equal(_window_attention_fwd(q, k, v, training=False, check=True)[0], out)


def attention_failed(lib):
    """Whether an attention kernel has reported an error since the last look."""
    import ctypes

    status = (ctypes.c_int32 * 8)()
    assert lib.lucid_attn_status(torch.cuda.current_stream().cuda_stream, status) == 0
    assert status[0] in (0, 1, 3), list(status)
    return status[0] != 0


@gpu
def test_a_wait_that_runs_out_at_the_very_end_is_reported():
    """One tile of queries on more and more keys: the warps that write results wait for all of them.  With the shortest limit
    above 0 (64 polls pass before the clock is looked at, and 64 more before the limit counts) that wait, and no other, runs
    out from some number of keys on; next to that number it runs out when every other role has just ended.  A call that reports
    nothing has given the right result, bit for bit."""
    from lucid_kernels_b200 import _cabi
    from lucid_kernels_b200.attention import _window_attention_fwd

    lib, most = _cabi.load(), 1500
    q, k, v, _ = make(1, 128, 128 * most, 1, 1, torch.bfloat16)
    call = lambda n: _window_attention_fwd(q, k[:, :128 * n], v[:, :128 * n])[:2]
    right = {}

    def reported(n):
        if n not in right:
            lib.lucid_set_wait_limit_ns(2_000_000_000)
            right[n] = call(n)
            assert not attention_failed(lib)
        lib.lucid_set_wait_limit_ns(1)
        got = call(n)
        bad = attention_failed(lib)
        assert bad or all(torch.equal(x, y) for x, y in zip(got, right[n])), n
        return bad

    try:
        lo, hi = 1, most
        assert reported(hi)
        while hi - lo > 1:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if reported(mid) else (mid, hi)
        for n in range(max(1, hi - 12), min(most, hi + 12) + 1):
            for _ in range(8):
                reported(n)
    finally:
        lib.lucid_set_wait_limit_ns(2_000_000_000)
    assert all(torch.equal(x, y) for x, y in zip(call(hi), right[hi])) and not attention_failed(lib)


@gpu
@pytest.mark.parametrize("shape,window,sinks", [((1, 128, 128, 1, 1), None, 0), ((1, 100, 256, 2, 1), None, 0), ((1, 256, 256, 3, 1), 60, 3),
                                                ((2, 300, 300, 2, 2), 100, 4), ((1, 64, 1536, 1, 1), None, 0), ((4, 256, 256, 80, 80), None, 0)])
def test_with_no_time_to_wait_small_calls_are_right_or_report(shape, window, sinks):
    from lucid_kernels_b200 import _cabi
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    lib = _cabi.load()
    q, k, v, do = make(*shape, torch.bfloat16)
    out, lse, rest = _window_attention_fwd(q, k, v, window, sinks, check=True)
    calls = [lambda: _window_attention_fwd(q, k, v, window, sinks)[:2],
             lambda: _window_attention_fwd(q, k, v, window, sinks, training=False)[:1],
             lambda: _window_attention_bwd(q, k, v, out, lse, rest, do, window, sinks),
             lambda: _window_attention_bwd(q, k, v, out, lse, rest, do, window, sinks, need_dkv=False)[:1],
             lambda: _window_attention_bwd(q, k, v, out, lse, rest, do, window, sinks, need_dq=False)[1:]]
    right = [call() for call in calls]
    assert not attention_failed(lib)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    try:
        lib.lucid_set_wait_limit_ns(0)
        for n in range(10):
            for i, call in enumerate(calls):
                flush.fill_(n)                  # operands from memory: their loads take longest
                got = call()
                assert attention_failed(lib) or all(torch.equal(x, y) for x, y in zip(got, right[i])), i
    finally:
        lib.lucid_set_wait_limit_ns(2_000_000_000)
    for call, ref in zip(calls, right):
        assert all(torch.equal(x, y) for x, y in zip(call(), ref))
    assert not attention_failed(lib)


@gpu
def test_calls_at_once_on_two_streams():
    """Nothing is shared between calls: the same bits as one after another."""
    from lucid_kernels_b200 import paged_lucid_attention
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    a, c = make(1, 300, 3000, 4, 2, torch.bfloat16, seed=1), make(2, 900, 900, 8, 2, torch.bfloat16, seed=2)
    pages, page = 40, 64
    kc = torch.randn(pages, page, 2, D, device="cuda").bfloat16() * 0.1
    vc = torch.randn(pages, page, 2, D, device="cuda").bfloat16()
    table = torch.randperm(pages, device="cuda", dtype=torch.int32).view(1, -1)
    lens = torch.tensor([2500], dtype=torch.int32, device="cuda")

    def work():
        x = _window_attention_fwd(*a[:3], None, 0, training=False)[0]
        out, lse, rest = _window_attention_fwd(*c[:3], 300, 4)
        grads = _window_attention_bwd(*c[:3], out, lse, rest, c[3], 300, 4)
        pools = kc.clone(), vc.clone()
        y = paged_lucid_attention(a[0][:, 0], a[1][:, 0], *pools, table, lens, k_scale=0.3, scale=0.1)
        return [x, out, lse, *grads, y, pools[1]]

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want))
    with pytest.raises(AssertionError, match="query heads"):
        paged_lucid_attention(a[0][:, 0, :0], a[1][:, 0], kc, vc, table, lens)


@gpu
def test_first_keys_of_more_than_65535_heads():
    """One query on its own key and the first one, for 8200 sequences of 8 heads."""
    from lucid_kernels_b200.attention import _window_attention_bwd, _window_attention_fwd

    B, H, Nk, dt = 8200, 8, 129, torch.bfloat16
    q, k, v, do = make(B, 1, Nk, H, H, dt, seed=7)
    out, lse, rest = _window_attention_fwd(q, k, v, 1, 1, 0.1, check=True)
    dk, dv = _window_attention_bwd(q, k, v, out, lse, rest, do, 1, 1, 0.1, check=True)[1:]
    u = torch.finfo(dt).eps / 2
    for lo in range(0, B, 1025):
        part = slice(lo, lo + 1025)
        s = 0.1 * (q[part].double() * k[part, [0, -1]].double()).sum(-1, keepdim=True)
        want = torch.softmax(s, 1) * do[part].double()
        # the weight and the result are rounded (u each); the exponential and the sum of the weights add less than u
        assert ((dv[part, [0, -1]].double() - want).abs() <= 3 * u * want.abs() + 1e-30).all()
        assert torch.isfinite(dk[part]).all() and dk[part, [0, -1]].any()
    assert not dv[:, 1:-1].any() and not dk[:, 1:-1].any()


@gpu
def test_one_tensor_as_queries_keys_and_values():
    from lucid_kernels_b200 import window_attention

    x, _, _, do = make(1, 300, 300, 2, 2, torch.bfloat16, seed=5)
    leaves = [x.clone().requires_grad_() for _ in range(3)]
    window_attention(*leaves, window=70, sinks=2).backward(do)
    one = x.clone().requires_grad_()
    window_attention(one, one, one, window=70, sinks=2).backward(do)
    parts = [t.grad.double() for t in leaves]
    # two additions in 16 bits, in any order: each off by u = 2^-8 of at most |dq| + |dk| + |dv|, and the first's error on top
    u = torch.finfo(x.dtype).eps / 2
    assert ((one.grad.double() - sum(parts)).abs() <= 2 * u * (1 + u) * sum(t.abs() for t in parts)).all()


@gpu
def test_partial_gradients_and_empty_tensors():
    from lucid_kernels_b200 import window_attention

    dt = torch.float16
    q, k, v, do = make(1, 200, 200, 2, 1, dt)
    full = [t.clone().requires_grad_(True) for t in (q, k, v)]
    window_attention(*full, window=70).backward(do)
    for need in range(3):
        leaves = [t.clone().requires_grad_(i == need) for i, t in enumerate((q, k, v))]
        window_attention(*leaves, window=70).backward(do)
        assert torch.equal(leaves[need].grad, full[need].grad)
    for B, Nq in ((0, 4), (1, 0)):
        e = [torch.empty(B, n, h, D, device="cuda", dtype=dt, requires_grad=True) for n, h in ((Nq, 2), (4, 1), (4, 1))]
        o = window_attention(*e, window=3)
        assert o.shape == e[0].shape
        o.sum().backward()
        assert not e[1].grad.any()


# ------------------------------------------------------------------------------------------------ paged cache
def rotated(x, pos, inv_freq, interleaved=False):
    """64 bits: x (T, H, D), pos (T,)."""
    a = pos.double()[:, None, None] * inv_freq.double()
    r = 2 * inv_freq.numel()
    y, out = x[..., :r].double(), x.double().clone()
    if interleaved:
        p, s = y[..., 0::2], y[..., 1::2]
        out[..., 0:r:2], out[..., 1:r:2] = p * a.cos() - s * a.sin(), s * a.cos() + p * a.sin()
    else:
        p, s = y.chunk(2, -1)
        out[..., :r] = torch.cat((p * a.cos() - s * a.sin(), s * a.cos() + p * a.sin()), -1)
    return out


def frequencies(rot=D):
    return (10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)).float().cuda()


def pool_of(B, cap, page, Hkv, dt, seed=0, fill=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    per = -(-cap // page)
    pages = B * per + 2
    table = torch.randperm(pages, device="cuda", generator=g)[: B * per].reshape(B, per).to(torch.int32)
    mk = lambda: torch.randn(pages, page, Hkv, D, device="cuda", generator=g).to(dt) if fill is None else torch.full((pages, page, Hkv, D), fill, device="cuda", dtype=dt)
    return mk(), mk(), table


def close_rotation(got, ref, x, dt):
    """A rotated element is a sum of two fp32 products, rounded once: u |ref| and fp32 errors of the inputs' size (sines to
    2^-21, products and sum)."""
    size = x.double().abs().amax()
    assert bool(((got.double() - ref).abs() <= unit(dt) * ref.abs() + 2.0 ** -19 * size + (2.0 ** -25 if dt == torch.float16 else 0)).all())


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("page,Hq,Hkv,rot,interleaved", [(16, 8, 4, 128, False), (64, 3, 1, 128, True), (1, 2, 2, 32, False),
                                                         (256, 4, 1, 48, True), (128, 16, 16, 16, False)])
def test_append_rotates_and_places(page, Hq, Hkv, rot, interleaved, dt):
    from lucid_kernels_b200 import paged_append

    new, before = [1, 0, 37, 300, 64], [5, 100, 0, 255, 999_000]
    B = len(new)
    per = [-(-(n + m) // page) for n, m in zip(new, before)]
    width = max(per)
    pages = sum(-(-n // page) + 1 for n in new) + 3
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    table = torch.full((B, width), -7, dtype=torch.int32)                 # only the pages that new tokens reach exist
    for b in range(B):
        for i in range(before[b] // page, per[b]):
            if new[b]:
                table[b, i] = free.pop()
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    T = sum(new) + 3                                                      # three rows of padding behind the last sequence
    qkv = torch.randn(T, Hq + 2 * Hkv, D, device="cuda", generator=g).to(dt)
    q, k, v = qkv.split((Hq, Hkv, Hkv), 1)
    kc = torch.full((pages, page, Hkv, D), 3.0, device="cuda", dtype=dt)
    vc = kc.clone()
    f = frequencies(rot)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    lens = torch.tensor(before, dtype=torch.int32, device="cuda")
    ver = kc._version
    got = paged_append(k, v, kc, vc, table.cuda(), lens, cu_seqlens=cu, q=q, inv_freq=f, interleaved=interleaved, check=True)
    assert kc._version > ver
    assert not got[sum(new):].any()
    touched = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b in range(B):
        for i in range(new[b]):
            t, pos = int(cu[b]) + i, before[b] + i
            touched[int(table[b, pos // page]), pos % page] = True
    pos = torch.cat([torch.arange(n) + m for n, m in zip(new, before)]).cuda()
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)])
    pg = table[seq, (pos.cpu() // page)].long().cuda()
    n = sum(new)
    close_rotation(kc[pg, pos % page], rotated(k[:n], pos, f, interleaved), k, dt)
    close_rotation(got[:n], rotated(q[:n], pos, f, interleaved), q, dt)
    assert torch.equal(vc[pg, pos % page], v[:n])
    assert torch.equal(kc[pg, pos % page][..., rot:], k[:n, :, rot:])
    assert bool((kc[~touched] == 3.0).all()) and bool((vc[~touched] == 3.0).all())


@gpu
def test_append_single_tokens_without_rotation_keys_only_and_interleaved_pools():
    from lucid_kernels_b200 import paged_append

    dt, B, page, Hkv = torch.bfloat16, 70, 32, 2
    both = torch.zeros(B * 2, 2, page, Hkv, D, device="cuda", dtype=dt)          # one pool, keys and values side by side
    kc, vc = both[:, 0], both[:, 1]
    table = torch.arange(B * 2, device="cuda", dtype=torch.int32).reshape(B, 2)
    lens = torch.arange(B, device="cuda", dtype=torch.int32) % 64
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    k, v = (torch.randn(B, Hkv, D, device="cuda", generator=g).to(dt) for _ in range(2))
    assert paged_append(k, None, kc, vc, table, lens, check=True) is None
    rows = table.long()[torch.arange(B), (lens // page).long()], (lens % page).long()
    assert torch.equal(kc[rows], k) and not vc.any()
    paged_append(k, v, kc, vc, table, lens, check=True)
    assert torch.equal(vc[rows], v)


@gpu
@pytest.mark.parametrize("Hq,Hkv,B,most", [(16, 16, 3, 4400), (3, 1, 100, 150), (5, 1, 40, 300)])
def test_append_many_tokens(Hq, Hkv, B, most):
    """A warp per token and several rounds of head rows; many sequences, some of them without tokens."""
    from lucid_kernels_b200 import paged_append

    dt, page = torch.bfloat16, 16
    h = torch.Generator().manual_seed(B)
    new = torch.randint(0, most + 1, (B,), generator=h)
    new[torch.randint(0, B, (B // 3,), generator=h)] = 0
    new[B // 2] = most
    T = int(new.sum())
    assert T >= 4096
    before = torch.randint(0, 50, (B,), generator=h)
    per = -(-int((new + before).max()) // page)
    table = torch.randperm(B * per, generator=h).reshape(B, per).to(torch.int32)
    kc = torch.zeros(B * per, page, Hkv, D, device="cuda", dtype=dt)
    vc = torch.zeros_like(kc)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(T, n, D, device="cuda", generator=g).to(dt) for n in (Hq, Hkv, Hkv))
    cu = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0)))
    f = frequencies()
    got = paged_append(k, v, kc, vc, table.cuda(), before.to(torch.int32).cuda(), cu_seqlens=cu.to(torch.int32).cuda(), q=q, inv_freq=f, check=True)
    seq = torch.repeat_interleave(torch.arange(B), new)
    pos = before[seq] + torch.arange(T) - cu[:-1][seq]
    at = table[seq, pos // page].long().cuda(), (pos % page).cuda()
    close_rotation(kc[at], rotated(k, pos.cuda(), f), k, dt)
    close_rotation(got, rotated(q, pos.cuda(), f), q, dt)
    assert torch.equal(vc[at], v)
    assert int((vc != 0).any(-1).any(-1).sum()) == T


@gpu
@pytest.mark.parametrize("Hq,Hkv", [(8, 4), (4, 1), (33, 8), (1, 1)])
def test_append_is_the_same_however_the_tokens_are_dealt_out(Hq, Hkv):
    """One call, around the number of tokens at which a warp takes on a whole token, against many calls of a few tokens."""
    from lucid_kernels_b200 import paged_append

    dt, page = torch.float16, 32
    groups = -(-(Hq + 2 * Hkv) // 4)
    edge = torch.cuda.get_device_properties(0).multi_processor_count * 24 // min(groups, 4)
    f = frequencies()
    for T in (edge - 1, edge, edge + 1, 2 * edge + 5):
        kc, vc, table = pool_of(1, T + 9, page, Hkv, dt, seed=T)
        kd, vd = kc.clone(), vc.clone()
        g = torch.Generator(device="cuda").manual_seed(T)
        q, k, v = (torch.randn(T, n, D, device="cuda", generator=g).to(dt) for n in (Hq, Hkv, Hkv))
        int32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
        got = paged_append(k, v, kc, vc, table, int32(9), cu_seqlens=int32(0, T), q=q, inv_freq=f, check=True)
        parts = [paged_append(k[a:a + 100], v[a:a + 100], kd, vd, table, int32(9 + a), cu_seqlens=int32(0, min(100, T - a)), q=q[a:a + 100],
                              inv_freq=f, check=True) for a in range(0, T, 100)]
        assert torch.equal(got, torch.cat(parts)) and torch.equal(kc, kd) and torch.equal(vc, vd), T


@gpu
def test_offsets_beyond_32_bits():
    """Pools of more than 2^31 elements, the sequence's pages at their end; inputs whose rows lie that far apart."""
    from lucid_kernels_b200 import paged_append, paged_lucid_attention, paged_window_attention, window_attention

    dt, page, Hkv, Hq, n = torch.bfloat16, 64, 4, 8, 300
    pages = 2 ** 31 // (page * Hkv * D) + 40
    kc, vc = (torch.empty(pages, page, Hkv, D, device="cuda", dtype=dt) for _ in range(2))
    per = -(-n // page)
    table = torch.arange(pages - 1, pages - 1 - per, -1, device="cuda", dtype=torch.int32)[None]
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).to(dt) for h in (Hq, Hkv, Hkv))
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    paged_append(k, v, kc, vc, table, zero, cu_seqlens=cu, check=True)
    small_k, small_v = kc[table[0].long()].clone(), vc[table[0].long()].clone()
    small = torch.arange(per, device="cuda", dtype=torch.int32)[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    a = paged_window_attention(q[-1:], kc, vc, table, lens, 100, 4, check=True)
    assert torch.equal(a, paged_window_attention(q[-1:], small_k, small_v, small, lens, 100, 4, check=True))
    small_v.mul_(1e-3)
    vc[table[0].long()] = small_v
    a = paged_lucid_attention(q[-1:], v[-1:], kc, vc, table, lens, k_scale=0.2, check=True)
    assert torch.equal(a, paged_lucid_attention(q[-1:], v[-1:], small_k, small_v, small, lens, k_scale=0.2, check=True))
    assert torch.equal(vc[table[0].long()], small_v)
    del kc, vc
    width = (2 ** 31 // (n - 1) // 8 + 1) * 8
    far = torch.empty(n, width, device="cuda", dtype=dt)[:, : Hq * D]
    far.copy_(q.reshape(n, Hq * D))
    fq = far.unflatten(1, (Hq, D))[None]
    assert fq.stride(1) * (n - 1) >= 2 ** 31
    assert torch.equal(window_attention(fq, k[None], v[None], 100, 4), window_attention(q[None], k[None], v[None], 100, 4))


@gpu
def test_bad_pages_are_skipped_and_reported():
    """No address is formed from a page outside the pool or a position beyond the table: the host's view of the bounds is
    page_of / the append kernel's own check, and the error is reported once."""
    from lucid_kernels_b200 import _cabi, paged_append, paged_lucid_attention, paged_window_attention

    dt, page, Hkv = torch.bfloat16, 16, 1
    kc, vc, table = pool_of(2, 64, page, Hkv, dt, seed=4)
    k0, v0 = kc.clone(), vc.clone()
    x = torch.ones(2, Hkv, D, device="cuda", dtype=dt)
    lens = torch.tensor([64, 3], dtype=torch.int32, device="cuda")               # sequence 0: behind the table
    with pytest.raises(_cabi.LucidKernelError, match="block table"):
        paged_append(x, x, kc, vc, table, lens, check=True)
    changed = (kc != k0).any(-1).any(-1)
    assert int(changed.sum()) == 1 and bool(changed[int(table[1, 0]), 3])
    bad = table.clone()
    bad[1, 1] = kc.shape[0]
    bad[0, 0] = -1
    q = torch.randn(2, 2, D, device="cuda").to(dt)
    n = torch.tensor([20, 40], dtype=torch.int32, device="cuda")
    with pytest.raises(_cabi.LucidKernelError, match="block table"):
        paged_window_attention(q, kc, vc, bad, n, check=True)
    v1 = vc.clone()
    n = torch.tensor([16, 17], dtype=torch.int32, device="cuda")                  # the newest position's page is the bad one
    with pytest.raises(_cabi.LucidKernelError, match="block table"):
        paged_lucid_attention(q, x, kc, vc, bad, n, check=True)
    assert torch.equal(vc, v1)
    paged_window_attention(q, kc, vc, table, n, check=True)                       # reported once, then forgotten
    n = torch.tensor([2 ** 31 - 1, 40], dtype=torch.int32, device="cuda")         # a length far beyond the table ends, too
    with pytest.raises(_cabi.LucidKernelError, match="block table"):
        paged_window_attention(q, kc, vc, table, n, check=True)
    with pytest.raises(_cabi.LucidKernelError, match="block table"):
        paged_lucid_attention(q, x, kc, vc, table, n, check=True)
    n = torch.tensor([-5, 40], dtype=torch.int32, device="cuda")                  # and a negative one is none
    assert not paged_window_attention(q, kc, vc, table, n, check=True)[0].any()


@gpu
@pytest.mark.parametrize("width", [4, 600])                                       # a cluster's chunks, and more (two kernels)
@pytest.mark.parametrize("window,sinks", [(40, 0), (40, 3), (5, 0), (0, 2), (1, 1), (8000, 5000)])
def test_a_length_beyond_the_table_moves_the_window(window, sinks, width):
    """Positions that do not exist are skipped: the query sees the rest of its window and the first keys, and no others."""
    from lucid_kernels_b200 import _cabi, paged_window_attention

    dt, page, Hq, Hkv = torch.bfloat16, 16, 4, 2
    cap = width * page
    over = [1, 20, window - 1, window, window + 1, 5 * cap, 2 ** 31 - 1 - cap]
    lens = [cap] + [cap + max(0, n) for n in over]
    B = len(lens)
    kc, vc, table = pool_of(1, cap, page, Hkv, dt, seed=6)
    table = table.expand(B, width)
    q = torch.randn(B, Hq, D, device="cuda").to(dt)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = paged_window_attention(q, kc, vc, table, n, window=window, sinks=sinks, scale=0.1)
    with pytest.raises(_cabi.LucidKernelError, match="block table"):
        _cabi.raise_on_attention_error(torch.cuda.current_stream().cuda_stream, "step")
    pos = torch.arange(cap, device="cuda")
    pg = table[0].long()[pos // page]
    kk, vv = kc[pg, pos % page].double(), vc[pg, pos % page].double()
    for b, length in enumerate(lens):
        seen = (pos >= length - window) | (pos < sinks)
        for h in range(Hq):
            s = q[b, h].double() @ kk[seen][:, h // 2].T * 0.1
            v = vv[seen][:, h // 2]
            ref, bound = (torch.softmax(s, -1) @ v, torch.softmax(s, -1) @ v.abs()) if int(seen.sum()) else (torch.zeros(D, device="cuda").double(),) * 2
            close(got[b, h], ref, bound, dt, f"length {length}")


def step_reference(q, kc, vc, table, lens, window, sinks, scale, v=None, k_scale=1.0):
    """(out, bound, v', its bound) in 64 bits."""
    B, Hq, _ = q.shape
    page, Hkv = kc.shape[1:3]
    G = Hq // Hkv
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    bound, new, nb = torch.zeros_like(out), torch.zeros(B, Hkv, D, dtype=torch.float64, device=q.device), torch.zeros(B, Hkv, D, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        pos = torch.arange(n, device=q.device)
        if window is not None:
            pos = pos[(pos >= n - window) | (pos < sinks)]
        pg = table[b].long()[pos // page]
        kk, vv = kc[pg, pos % page].double(), vc[pg, pos % page].double()
        for h in range(Hkv):
            K, V = kk[:, h], vv[:, h].clone()
            if v is not None:
                t = K @ K[-1] * k_scale ** 2
                w = torch.exp(t[:-1] - t[-1])
                new[b, h] = torch.exp(-t[-1]) * v[b, h].double() - w @ V[:-1]
                nb[b, h] = w @ V[:-1].abs()
                V[-1] = new[b, h]
            if len(pos):
                P = torch.softmax(q[b, h * G:(h + 1) * G].double() @ K.T * scale, -1)
                out[b, h * G:(h + 1) * G] = P @ V
                bound[b, h * G:(h + 1) * G] = P @ V.abs()
                if v is not None:      # v'_n enters rounded, with its own error
                    bound[b, h * G:(h + 1) * G] += P[:, -1:] * (nb[b, h] + new[b, h].abs())
    return out, bound, new, nb


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("page,Hq,Hkv,window,sinks,lens", [
    (16, 8, 4, None, 0, [1, 0, 17, 64, 500]),
    (64, 4, 4, 100, 4, [1, 99, 100, 101, 104, 105, 700]),
    (1, 2, 1, 1, 0, [1, 2, 3]),
    (32, 6, 2, 5, 300, [4, 5, 6, 250, 305, 306, 1000]),
    (128, 16, 1, None, 0, [1023]),
    (256, 40, 2, 64, 1, [3, 70, 2000]),
    (64, 3, 3, 0, 3, [1, 2, 3, 4, 90]),
    (64, 3, 3, 0, 0, [1, 90]),
    (64, 4, 1, None, 0, [9000]),
])
def test_paged_window_attention(page, Hq, Hkv, window, sinks, lens, dt):
    from lucid_kernels_b200 import paged_window_attention

    B = len(lens)
    kc, vc, table = pool_of(B, max(max(lens), 1), page, Hkv, dt, seed=7)
    for b, n in enumerate(lens):          # what no sequence owns, or lies behind one's end in its last page, holds anything
        if n % page:
            kc[table[b, n // page].long(), n % page:] = float("nan")
            vc[table[b, n // page].long(), n % page:] = float("inf")
    q = torch.randn(B, Hq, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dt)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = paged_window_attention(q, kc, vc, table, sl, window, sinks, check=True)
    ref, bound, _, _ = step_reference(q, kc, vc, table, lens, window, sinks, D ** -0.5)
    close(out, ref, bound, dt, "out")
    # strided queries: a slice of a projection
    wide = torch.randn(B, Hq + 4, D, device="cuda").to(dt)
    wide[:, 2:Hq + 2] = q
    assert torch.equal(paged_window_attention(wide[:, 2:Hq + 2], kc, vc, table, sl, window, sinks), out)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("page,Hq,Hkv,lens", [(16, 8, 4, [1, 0, 2, 17, 64, 500]), (64, 1, 1, [3000]), (128, 15, 1, [129, 128]), (1, 4, 2, [5, 1]),
                                              (32, 2, 2, [33] * 40)])
def test_paged_lucid_attention(page, Hq, Hkv, lens, dt):
    from lucid_kernels_b200 import paged_lucid_attention

    B, ks = len(lens), D ** -0.25
    kc, vc, table = pool_of(B, max(max(lens), 1), page, Hkv, dt, seed=8)
    kc.mul_(0.5)
    vc.mul_(0.1)
    for b, n in enumerate(lens):
        if n % page:
            kc[table[b, n // page].long(), n % page:] = float("nan")
            vc[table[b, n // page].long(), n % page:] = float("nan")
        if n:
            vc[table[b, (n - 1) // page].long(), (n - 1) % page] = float("nan")     # the new row's place is not read
    g = torch.Generator(device="cuda").manual_seed(2)
    q, v = torch.randn(B, Hq, D, device="cuda", generator=g).to(dt), torch.randn(B, Hkv, D, device="cuda", generator=g).to(dt)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref, bound, new, nb = step_reference(q, kc, vc, table, lens, None, 0, 0.1, v, ks)
    before = vc.clone()
    out = paged_lucid_attention(q, v, kc, vc, table, sl, k_scale=ks, scale=0.1, check=True)
    close(out, ref, bound, dt, "out")
    changed = torch.zeros(vc.shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        if n:
            at = int(table[b, (n - 1) // page]), (n - 1) % page
            close(vc[at], new[b], nb[b], dt, "v'")
            changed[at] = True
    assert torch.equal(vc[~changed].view(torch.int16), before[~changed].view(torch.int16))
    again = paged_lucid_attention(q, v, kc, vc, table, sl, k_scale=ks, scale=0.1, check=True)
    assert torch.equal(again, out)


@gpu
def test_cache_operators_captured_and_on_another_stream():
    from lucid_kernels_b200 import paged_append, paged_lucid_attention, paged_window_attention

    dt, B, Hq, Hkv, page = torch.bfloat16, 3, 4, 2, 32
    kc, vc, table = pool_of(B, 2000, page, Hkv, dt, seed=5)
    vc.mul_(1e-3)
    lens = torch.tensor([700, 31, 1999], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(B, h, D, device="cuda").to(dt) for h in (Hq, Hkv, Hkv))
    f = frequencies()

    def step(kc, vc):
        qr = paged_append(k, None, kc, vc, table, lens, q=q, inv_freq=f)
        a = paged_lucid_attention(qr, v, kc, vc, table, lens + 1, k_scale=D ** -0.25)
        return a, paged_window_attention(qr, kc, vc, table, lens + 1, 300, 4)

    k1, v1 = kc.clone(), vc.clone()
    want = step(k1, v1)
    side = torch.cuda.Stream()
    k2, v2 = kc.clone(), vc.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(k2, v2)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, other)) and torch.equal(k1, k2) and torch.equal(v1, v2)
    k3, v3 = kc.clone(), vc.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = step(k3, v3)
        graphs.append((g, r))
    for g, r in graphs * 2:
        k3.copy_(kc)
        v3.copy_(vc)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(r, want)) and torch.equal(v3, v1)
    lens.fill_(5)                                   # a replay reads the lengths of its own time
    k4, v4 = kc.clone(), vc.clone()
    want = step(k4, v4)
    k3.copy_(kc)
    v3.copy_(vc)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(graphs[0][1], want))


# ------------------------------------------------------------------------------------------------ together
@gpu
def test_prompt_and_steps_equal_one_long_run():
    """A LUCID layer and a window layer, prompt then tokens one by one through the cache, against the whole sequence at once:
    rotation, solve, V' and attention.  Reference: 64 bits from the 16-bit projections, with the cache's 16-bit keys."""
    from lucid_kernels_b200 import paged_append, paged_lucid_attention, paged_window_attention, window_attention
    from lucid_kernels_b200.cute import _forward_sub_fwd

    dt, P, extra, Hq, Hkv, page, W, S = torch.bfloat16, 256, 20, 4, 2, 16, 60, 3
    N, ks = P + extra, D ** -0.25
    g = torch.Generator(device="cuda").manual_seed(12)
    q, k, v = (torch.randn(N, h, D, device="cuda", generator=g).to(dt) for h in (Hq, Hkv, Hkv))
    k = (k * 0.7).to(dt)
    f = frequencies()
    out = {}
    for kind in ("window", "lucid"):
        kc, vc, table = pool_of(1, N, page, Hkv, dt, seed=3, fill=float("nan"))
        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, P], dtype=torch.int32, device="cuda")
        qr = paged_append(k[:P], v[:P], kc, vc, table, zero, cu_seqlens=cu, q=q[:P], inv_freq=f, check=True)
        pos = torch.arange(N, device="cuda")
        at = table[0].long()[pos // page], pos % page
        kr = kc[at][:P]
        if kind == "window":
            rows = [window_attention(qr[None], kr[None], v[None, :P], W, S)[0]]
        else:
            vp = _forward_sub_fwd(kr[None], v[None, :P], k_scale=ks)
            vc[at[0][:P], at[1][:P]] = vp[0]
            rows = [window_attention(qr[None], kr[None], vp, scale=ks * D ** -0.5)[0]]
        for n in range(P, N):
            have = torch.full((1,), n, dtype=torch.int32, device="cuda")
            qn = paged_append(k[n:n + 1], None if kind == "lucid" else v[n:n + 1], kc, vc, table, have, q=q[n:n + 1], inv_freq=f, check=True)
            if kind == "window":
                rows.append(paged_window_attention(qn, kc, vc, table, have + 1, W, S, check=True))
            else:
                rows.append(paged_lucid_attention(qn, v[n:n + 1], kc, vc, table, have + 1, k_scale=ks, scale=ks * D ** -0.5, check=True))
        out[kind] = torch.cat(rows).double(), kc[at].double(), vc[at].double()
    pos = torch.arange(N, device="cuda")
    qq = rotated(q, pos, f)
    for kind, (o, kk, vv) in out.items():
        scale = D ** -0.5 * (ks if kind == "lucid" else 1)
        for h in range(Hkv):
            V = v[:, h].double()
            if kind == "lucid":
                E = torch.exp(torch.tril(kk[:, h] @ kk[:, h].T * ks * ks)) * torch.tril(torch.ones(N, N, device="cuda", dtype=torch.float64))
                V = torch.linalg.solve_triangular(E, V, upper=False)
                assert float((vv[:, h] - V).norm() / V.norm()) < 0.01       # the solve's own tolerance
            for i in range(Hq // Hkv):
                x = h * (Hq // Hkv) + i
                ok = visible(N, N, None if kind == "lucid" else W, S, N, "cuda")
                ref = torch.softmax((qq[:, x] @ kk[:, h].T * scale).masked_fill(~ok, -math.inf), -1) @ V
                assert float((o[:, x] - ref).norm() / ref.norm()) < 0.01

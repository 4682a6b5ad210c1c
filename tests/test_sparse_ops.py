"""CPU: bindings and refusals of routing, the experts' products and the delta rule."""
import ctypes

import pytest
import torch

from llamatov_b200 import _lib, dense_ops as P


def _refused(name, text, *args):
    assert getattr(_lib.dense(), name)(*args) == 1
    assert text in _lib.last_error(), _lib.last_error()


one = ctypes.c_void_p(256)     # never dereferenced: validation fails first


def router(**kw):
    d = dict(n=64, top=6, score=0, groups=1, top_groups=1, renorm=1, scale=1.0)
    d.update(kw)
    return ctypes.byref(_lib.DnRouter(**d))


def choice(**kw):
    d = dict(ids=256, plan=None, T=3, top=2, n=8)
    d.update(kw)
    return ctypes.byref(_lib.DnChoice(**d))


def delta(**kw):
    d = dict(H=4, G=2, dp=16, dvp=24, q_scale=1.0, eps=1e-6, taps=4, conv=256, conv_b=256, dt_bias=256, A=256)
    d.update(kw)
    return ctypes.byref(_lib.DnDelta(**d))


def seqs(*items):
    q = _lib.DnSeqs(n=len(items))
    for i, (start, rows, S) in enumerate(items):
        q.start[i], q.rows[i], q.S[i] = start, rows, S
    return ctypes.byref(q)


@pytest.mark.parametrize("kw,ld,T,text", [
    (dict(), 63, 4, "ld=63"), (dict(n=1025), 2000, 4, "n=1025"), (dict(), 64, 0, "T=0"), (dict(score=2), 64, 4, "unknown score"),
    (dict(groups=7), 64, 4, "7 groups"), (dict(groups=64, top_groups=8), 64, 4, "at most 32 groups"), (dict(groups=4, top_groups=5), 64, 4, "5 of 4"),
    (dict(top=33), 64, 4, "top 33"), (dict(top=0), 64, 4, "top 0"), (dict(groups=8, top_groups=1, top=9), 64, 4, "top 9 of 8")])
def test_route_refusals(kw, ld, T, text):
    _refused("lt_dn_route", text, one, ld, one, one, T, router(**kw), None)
    _refused("lt_dn_route", "null", None, 64, one, one, 4, router(), None)


def test_experts_refusals():
    e = P.epilogue(_lib.DN_GLU, glu=(0, 0.0, 0.0))
    glu = lambda text, ldw=16, ldx=16, ldh=24, F=24, K=16, c=choice(), epi=e, W=one, ws=None: _refused(
        "lt_dn_experts_glu", text, W, ldw, one, ldx, one, ldh, 0, F, K, c, ctypes.byref(epi), ws, None)
    glu("null", W=None)
    glu("multiples of 8", K=12)
    glu("multiples of 8", ldw=8)
    glu("ldh=23", ldh=23)
    glu("aligned", W=ctypes.c_void_p(264))
    glu("workspace", c=choice(plan=256))
    glu("workspace", c=choice(plan=256), ws=ctypes.c_void_p(264))
    glu("null choice", c=choice(ids=None))
    glu("experts", c=choice(n=1025))
    glu("top", c=choice(top=33))
    glu("places", c=choice(T=1 << 28, top=8))
    glu("LT_DN_GLU", epi=P.epilogue())
    glu("LT_DN_GLU", epi=P.epilogue(_lib.DN_GLU, glu=(0, 0.0, 0.0), out_f32=True))
    s = lambda text, ldy=24, ldh=16, c=choice(), w=one: _refused("lt_dn_experts_sum", text, one, 16, one, ldh, one, ldy, 0, 24, 16, c, w, None, None, None)
    s("null", w=None)
    s("ldy=23", ldy=23)
    s("multiples of 8", ldh=12)
    s("without an order", c=choice(T=65536))
    s("workspace", c=choice(plan=256))
    _refused("lt_dn_experts_plan", "n=1025", one, 3, 2, 1025, one, None)
    _refused("lt_dn_experts_plan", "null", None, 3, 2, 8, one, None)
    L = _lib.dense()
    assert L.lt_dn_experts_plan_ints(5, 3, 8) == 24 and L.lt_dn_experts_glu_ws(5, 3, 16, 0) == 120 and L.lt_dn_experts_glu_ws(5, 3, 16, 1) == 0
    assert L.lt_dn_experts_sum_ws(5, 3, 9, 16, 1) == 136 and L.lt_dn_experts_sum_ws(5, 3, 9, 16, 0) == 256


def test_matrices_of_more_rows_than_an_int_counts_are_refused():
    """Tensor-map coordinates are ints: rows past 2^31 would be read as zeros."""
    e, F = P.epilogue(_lib.DN_GLU, glu=(0, 0.0, 0.0)), 1 << 20
    _refused("lt_dn_experts_glu", f"{1024 * 2 * F} rows", one, 8, one, 8, one, F, 0, F, 8, choice(n=1024, plan=256, T=400, top=4), ctypes.byref(e), one, None)
    _refused("lt_dn_experts_sum", f"{1024 * 2 * F} rows", one, 8, one, 8, one, 2 * F, 0, 2 * F, 8, choice(n=1024, plan=256, T=400, top=4), one, None, one, None)


def test_delta_refusals():
    rows = lambda text, d=delta(), q=seqs((0, 5, 256)), ld=96, ldh=4, ldo=96: _refused(
        "lt_dn_delta_rows", text, one, one, one, ld, one, ldh, one, ldh, one, ldo, 0, d, q, None)
    rows("multiple of the key heads", delta(H=3))
    rows("multiples of 8", delta(dp=12))
    rows("above 512", delta(dp=520))
    rows("eps", delta(eps=0.0))
    rows("number of sequences", q=ctypes.byref(_lib.DnSeqs(n=0)))
    rows("number of sequences", q=ctypes.byref(_lib.DnSeqs(n=9)))
    rows("state is null", q=seqs((0, 5, None)))
    rows("aligned", q=seqs((0, 5, 264)))
    rows("rows of a sequence", q=seqs((0, -1, 256)))
    rows("rows of a sequence", q=seqs((2 ** 31 - 2, 5, 256)))
    rows("one state", q=seqs((0, 5, 256), (5, 5, 256)))
    rows("share rows", q=seqs((0, 5, 256), (4, 5, 512)))
    rows("ldla=3", ldh=3)
    rows("ldo=95", ldo=95)
    rows("alignment", ld=100)
    rows("alignment", ldo=97)
    chunked = lambda text, d=delta(), q=seqs((0, 5, 256)), k=one, ld=96, ldo=96, ws=one: _refused(
        "lt_dn_delta_chunked", text, one, k, one, ld, one, 4, one, 4, one, ldo, d, q, ws, None)
    chunked("above 256", delta(dp=264))
    chunked("above 256", delta(dvp=520))
    chunked("alignment", k=ctypes.c_void_p(258))
    chunked("alignment", ld=100)
    chunked("alignment", ldo=97)
    chunked("null pointer", ws=None)
    chunked("one state", q=seqs((0, 5, 256), (5, 5, 256)))
    assert _lib.dense().lt_dn_delta_chunked_ws(delta(), seqs((0, 65, 256), (65, 0, 512))) == 2 * (4 * (1536 + 2 * 384 + 2 * 1024 + 68) + 2 * 512)
    step = lambda text, d=delta(), S=one: _refused("lt_dn_delta_step", text, one, one, one, one, S, one, 0, one, one, d, None)
    step("taps=0", delta(taps=0))
    step("null constants", delta(conv=None))
    step("aligned", S=ctypes.c_void_p(264))
    step("null pointer", S=None)


@pytest.mark.parametrize("lengths,H,d,dv", [
    ([4096] * 8, 32, 128, 128), ([20000] * 8, 32, 256, 512), ([9000], 64, 256, 512), ([5000, 0, 300, 64, 1], 4, 24, 40), ([70] * 11, 1, 8, 8),
    ([100000, 100], 16, 128, 128)])
def test_workspace_of_a_chunked_walk_is_bounded(monkeypatch, lengths, H, d, dv):
    """Whatever the number of sequences: a gigabyte, or one chunk of each; and every row is walked once, in order, in whole chunks."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    monkeypatch.setattr(P, "DELTA_CHUNKED_FROM", 1)
    rule = P.DeltaRule(H, H, d, dv, torch.bfloat16, 1.0, 1e-6)
    chunk = _lib.dense().lt_dn_delta_chunked_ws(rule._ref, seqs((0, 1, 256)))
    asked, walked = [], {}
    monkeypatch.setattr(torch, "empty", lambda n, **kw: asked.append(n) or torch.zeros(4))

    def call(name, *a):
        assert name == "lt_dn_delta_chunked"
        q = a[11]._obj
        assert asked[-1] == _lib.dense().lt_dn_delta_chunked_ws(a[10], a[11]) <= max(1 << 28, chunk * q.n)
        for j in range(q.n):
            if q.rows[j]:
                walked.setdefault(q.S[j], []).append((q.start[j], q.rows[j]))
    monkeypatch.setattr(_lib, "call", call)
    rule.rows(256, 256, 256, 3 * H * max(d, dv), 256, 256, H, 256, H * dv, [4096 * (i + 1) for i in range(len(lengths))], lengths)
    at = 0
    for i, n in enumerate(lengths):
        parts = walked.get(4096 * (i + 1), [])
        for start, rows in parts:
            assert start == at and (rows % 64 == 0 or (start, rows) == parts[-1])
            at += rows
        assert sum(rows for _, rows in parts) == n


def test_portions_have_one_workspace_at_a_time(monkeypatch):
    import weakref
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    monkeypatch.setattr(P, "DELTA_CHUNKED_FROM", 1)
    monkeypatch.setattr(P, "DELTA_PORTION", 64)
    rule = P.DeltaRule(2, 2, 16, 16, torch.bfloat16, 1.0, 1e-6)
    made, zeros = [], torch.zeros

    def empty(n, **kw):
        assert all(r() is None for r in made)
        t = zeros(4)
        made.append(weakref.ref(t))
        return t
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(_lib, "call", lambda *a: None)
    rule.rows(256, 256, 256, 96, 256, 256, 2, 256, 32, [4096 * (i + 1) for i in range(9)], [300] * 9)
    assert len(made) == 10


def test_no_rows_is_no_launch():
    n = _lib.launch_count()
    assert _lib.dense().lt_dn_delta_rows(one, one, one, 96, one, 4, one, 4, one, 96, 0, delta(), seqs((0, 0, 256), (7, 0, 512)), None) == 0
    assert _lib.launch_count() == n


def test_workspace_of_a_refused_call_is_none():
    size = _lib.dense().lt_dn_delta_chunked_ws
    assert size(delta(), seqs((0, 100, 256))) == 2 * size(delta(), seqs((0, 1, 256))) > 0
    assert size(None, seqs((0, 1, 256))) == 0 and size(delta(), None) == 0
    assert size(delta(), seqs((0, -70, 256))) == 0 and size(delta(G=3), seqs((0, 1, 256))) == 0


def test_objects_refuse():
    with pytest.raises(ValueError, match="score"):
        P.Router(8, 2, score="tanh")
    with pytest.raises(ValueError, match="top 9"):
        P.Router(8, 9)
    with pytest.raises(ValueError, match="groups"):
        P.Router(8, 2, groups=3)
    with pytest.raises(ValueError, match="bias"):
        P.Router(8, 2, bias=torch.zeros(7))
    with pytest.raises(ValueError, match="matrices"):
        P.Experts(torch.zeros(4, 4), gated=False)
    with pytest.raises(ValueError, match="matrices"):
        P.Experts(torch.zeros(2, 4, 8, dtype=torch.float16), gated=False)
    with pytest.raises(ValueError, match="gate and up"):
        P.Experts(torch.zeros(2, 5, 8), gated=True)
    with pytest.raises(ValueError, match="key heads"):
        P.DeltaRule(3, 2, 8, 8, torch.float32, 1.0, 1e-6)


def test_order_of_the_places_is_kept_for_another_stream(monkeypatch):
    """Products on another stream than plan's: the order's memory may not go back to plan's stream before they have read it."""
    now, kept = [7], []

    class Buf:
        data_ptr = staticmethod(lambda: 256)
        record_stream = staticmethod(lambda s: kept.append(s))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: f"stream {now[0]}")
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: now[0], raising=False)
    monkeypatch.setattr(torch.Tensor, "cuda", lambda t: t)
    monkeypatch.setattr(P, "_here", lambda t, what: t)
    monkeypatch.setattr(P, "GROUP_FROM", 1)
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: Buf())
    calls = []
    monkeypatch.setattr(_lib, "call", lambda name, *a: calls.append((name, a[-1])))
    up, down = P.Experts(torch.zeros(4, 8, 8), gated=True), P.Experts(torch.zeros(4, 8, 8), gated=False)
    places = up.plan(torch.zeros(3, 2, dtype=torch.int32), 3)
    up.hidden(256, 8, places, 256, 8)
    down.add_sum(256, 8, places, 256, 256, 8)
    assert kept == []
    now[0] = 9
    up.hidden(256, 8, places, 256, 8)
    assert kept == ["stream 9"]
    down.add_sum(256, 8, places, 256, 256, 8)
    assert kept == ["stream 9"] * 2
    assert calls == [("lt_dn_experts_plan", 7), ("lt_dn_experts_glu", 7), ("lt_dn_experts_sum", 7), ("lt_dn_experts_glu", 9), ("lt_dn_experts_sum", 9)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("K", [1, 9, 12, 63])
def test_columns_that_are_no_multiple_of_8_are_refused(monkeypatch, K, gated):
    """The products read whole units of 8 columns of a caller's rows, and a NaN there times a column of zeros is a NaN."""
    monkeypatch.setattr(torch.Tensor, "cuda", lambda t: t)
    with pytest.raises(ValueError, match=f"{K} columns"):
        P.Experts(torch.zeros(2, 6, K), gated=gated)
    assert P.Experts(torch.zeros(2, 6, 64), gated=gated).K == 64


def test_products_of_the_other_kind_of_matrices_are_refused(monkeypatch):
    """Gate and up rows are twice as many as the sums would count, so that every expert but the first would be another."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.Tensor, "cuda", lambda t: t)
    monkeypatch.setattr(_lib, "call", lambda name, *a: pytest.fail(f"{name} was called"))
    places = P.Places(torch.zeros(3, 2, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="gate and up rows"):
        P.Experts(torch.zeros(4, 8, 8), gated=True).add_sum(256, 8, places, 256, 256, 8)
    with pytest.raises(ValueError, match="gate and up rows"):
        P.Experts(torch.zeros(4, 8, 8), gated=False).hidden(256, 8, places, 256, 8)


@pytest.mark.parametrize("name,shape", [("conv", (4, 95)), ("conv", (3, 96)), ("conv", (96, 4)), ("conv_b", (95,)), ("dt_bias", (1,)), ("A", (2, 1))])
def test_constants_of_other_sizes_are_refused(monkeypatch, name, shape):
    """A token's step would read behind them."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(P, "_here", lambda t, what: t)
    sizes = {"conv": (4, 96), "conv_b": (96,), "dt_bias": (2,), "A": (2,)}
    make = lambda **kw: P.DeltaRule(2, 1, 24, 24, torch.float32, 1.0, 1e-6, taps=4, **{n: torch.zeros(kw.get(n, s)) for n, s in sizes.items()})
    assert make().desc.taps == 4
    with pytest.raises(ValueError, match=rf"^{name} "):
        make(**{name: shape})


def test_calls_that_do_not_fit_together_are_refused(monkeypatch):
    """Places of other experts, one state for two sequences, an object of another device (no device is reached)."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    monkeypatch.setattr(torch.Tensor, "cuda", lambda t: t)
    W = P.Experts(torch.zeros(4, 8, 8), gated=False)
    places = P.Places(torch.zeros(3, 2, dtype=torch.int32), 5)
    with pytest.raises(ValueError, match="places of 5 experts"):
        W.add_sum(1, 8, places, 1, 1, 8)
    with pytest.raises(ValueError, match="places of 5 experts"):
        P.Experts(torch.zeros(4, 8, 8), gated=True).hidden(1, 8, places, 1, 8)
    rule = P.DeltaRule(2, 2, 8, 8, torch.float32, 1.0, 1e-6)
    with pytest.raises(ValueError, match="one state"):
        rule.rows(1, 1, 1, 16, 1, 1, 2, 1, 16, [64, 128, 64], [1, 2, 3])
    with pytest.raises(ValueError, match="rows of sequences"):
        rule.rows(1, 1, 1, 16, 1, 1, 2, 1, 16, [64, 128], [1000, -1])
    with pytest.raises(ValueError, match="float16"):
        P.DeltaRule(2, 2, 8, 8, torch.float16, 1.0, 1e-6)
    with pytest.raises(ValueError, match="2 states"):
        rule.rows(1, 1, 1, 16, 1, 1, 2, 1, 16, [64, 128], [1, 2, 3])
    router = P.Router(4, 2, bias=torch.zeros(4))
    ids = torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="ids is on cpu"):
        W.plan(ids, 3)
    with pytest.raises(ValueError, match="contiguous int32"):
        W.plan(ids.long(), 3)
    with pytest.raises(ValueError, match="contiguous int32"):
        W.plan(ids, 2)
    for o in (W, rule, router):
        o.home = 1
    for call in (lambda: W.plan(ids, 3), lambda: W.add_sum(1, 8, P.Places(ids, 4), 1, 1, 8), lambda: router.rows(1, 4, 1, 1, 3),
                 lambda: rule.rows(1, 1, 1, 16, 1, 1, 2, 1, 16, [64], [1]), lambda: rule.step(1, 1, 1, 1, 1, 1, 1, 1)):
        with pytest.raises(ValueError, match="current device is cuda:0"):
            call()


def test_models_with_bad_sizes_are_refused(monkeypatch):
    """Packing refuses what does not fit together (no device is reached)."""
    from llamatov_b200 import mixers
    from tests import layered_util as U
    from tests import sparse_util as X

    class Pk:
        dtype, Ep, f32 = torch.float32, 80, 1

        def want(self, **kw):
            pass
    cfg = X.config(U)
    t = X.random_tensors(U, cfg)
    c = {"n_embd": cfg["width"], "norm_eps": 1e-5, "dtype": "float32"}
    get = lambda p, **change: (lambda n: change[n] if n in change else t[p + n])
    m = cfg["layers"][0]["mixer"]
    with pytest.raises(ValueError, match="key heads"):
        mixers.GatedDeltaMixer(Pk(), c, dict(m, key_heads=3), get("l0.mix."))
    with pytest.raises(ValueError, match="convolution"):
        mixers.GatedDeltaMixer(Pk(), c, dict(m, conv=3), get("l0.mix."))
    ff = cfg["layers"][0]["mlp"]
    with pytest.raises(ValueError, match="router"):
        mixers.gelu_experts(Pk(), c, dict(ff, experts=7), get("l0.mlp."))
    with pytest.raises(ValueError, match="down"):
        mixers.gelu_experts(Pk(), c, ff, get("l0.mlp.", down=t["l0.mlp.down"][:, :-1]))
    with pytest.raises(ValueError, match="top 9"):
        mixers.gelu_experts(Pk(), c, dict(ff, top=9), get("l0.mlp."))
    with pytest.raises(ValueError, match="groups"):
        mixers.clamped_experts(Pk(), c, dict(ff, groups=3, limit=1.0), get("l0.mlp."))


def test_oracle_of_the_delta_rule_is_the_chunked_equation():
    """The token-by-token restatement against the matrix form of a chunk, so that the tests' yardstick stands on two legs."""
    import numpy as np
    from oracle import sparse as O
    r = np.random.default_rng(0)
    T, H, G, d, dv = 23, 4, 2, 6, 5
    q, k, v = r.standard_normal((T, G, d)), r.standard_normal((T, G, d)), r.standard_normal((T, H, dv))
    la, beta, S0 = -r.random((T, H)), r.random((T, H)), r.standard_normal((H, dv, d))
    S = S0.copy()
    o = O.delta_rule(q, k, v, la, beta, S, 0.3, 1e-6)
    for h in range(H):
        kh = k[:, h // 2] / np.sqrt((k[:, h // 2] ** 2).sum(1, keepdims=True) + 1e-6)
        qh = 0.3 * q[:, h // 2] / np.sqrt((q[:, h // 2] ** 2).sum(1, keepdims=True) + 1e-6)
        c = np.cumsum(la[:, h])
        D = np.tril(np.exp(c[:, None] - c[None]))
        A = np.tril(beta[:, h, None] * D * (kh @ kh.T), -1)
        Uv = np.linalg.solve(np.eye(T) + A, beta[:, h, None] * (v[:, h] - np.exp(c)[:, None] * (kh @ S0[h].T)))
        assert np.allclose(o[:, h], np.exp(c)[:, None] * (qh @ S0[h].T) + (np.tril(qh @ kh.T) * D) @ Uv)
        assert np.allclose(S[h], np.exp(c[-1]) * S0[h] + (Uv * np.exp(c[-1] - c)[:, None]).T @ kh)

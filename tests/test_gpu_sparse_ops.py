"""GPU: routing, the experts' products and the delta rule, each alone against plain 64-bit arithmetic, at sizes and masks where it
can go wrong.

Tolerances.  fp32 sums of n products of unit variance are off by at most n 2^-24 of their absolute values and by about sqrt(n) 2^-24
as a rule; tests allow 8 sqrt(n) 2^-24 of the outputs' size, and half a step (2^-9 of the power of two below, so 2^-8 of the value at
most) for a result that is rounded to bf16."""
import ctypes

import numpy as np
import pytest
import torch

from llamatov_b200 import _lib, dense_ops as P
from oracle import layered as L
from tests.gpu_util import stream

pytestmark = pytest.mark.gpu
DT = {0: torch.bfloat16, 1: torch.float32}
E32 = 2.0 ** -24


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == set()


def _np(t):
    return t.detach().double().cpu().numpy()


def _randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _off(got, want, size=None):
    """Largest difference over the size (the largest) of the wanted values."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert np.isfinite(got).all()
    size = np.abs(want).max() if size is None else size
    return float(np.abs(got - want).max() / size if size else np.abs(got).max())


# --------------------------------------------------------------------------- routing

def route64(l, top, score, bias, groups, top_groups, renorm, scale):
    """Row by row, from the definition."""
    T, n = l.shape
    ids, w = np.zeros((T, top), np.int64), np.zeros((T, top))
    for t in range(T):
        x = np.where(np.isnan(l[t]), -np.inf, l[t])
        gone = x == -np.inf
        with np.errstate(invalid="ignore", over="ignore"):
            if score == "softmax":
                s = np.zeros(n) if gone.all() else np.exp(x - x.max())
                s = s / s.sum() if s.sum() > 0 else s
            else:
                s = 1 / (1 + np.exp(-x))
        s[gone] = 0
        c = s + (bias if bias is not None else 0)
        c[gone] = -np.inf
        size = n // groups
        best = [np.sort(c[g * size:(g + 1) * size])[::-1][:2].sum() for g in range(groups)]
        kept = sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups]
        order = sorted((e for g in kept for e in range(g * size, (g + 1) * size)), key=lambda e: (-c[e], e))[:top]
        ids[t], w[t] = order, s[order]
        if renorm:
            w[t] = w[t] / w[t].sum() if w[t].sum() > 0 else 0
    return ids, w * scale


def _route(l, n, top, ld=None, bias=None, **kw):
    T = l.shape[0]
    ids = torch.full((T + 1, top), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T + 1, top), -7.0, device="cuda")
    P.Router(n, top, bias=bias, **kw).rows(l.data_ptr(), l.shape[1], ids.data_ptr(), w.data_ptr(), T)
    assert (ids[T:] == -7).all() and (w[T:] == -7).all()
    return ids[:T].cpu().numpy(), _np(w[:T])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,n,top,groups,top_groups,biased", [
    (1, 1, 1, 1, 1, False), (1, 64, 6, 1, 1, False), (5, 33, 32, 1, 1, True), (257, 64, 8, 8, 3, True), (31, 96, 4, 32, 5, False),
    (64, 256, 8, 8, 4, True), (3, 300, 10, 4, 4, True), (9, 1024, 32, 16, 2, True), (7, 512, 1, 2, 1, False), (130, 12, 3, 12, 3, True)])
def test_route(score, T, n, top, groups, top_groups, biased):
    l = _randn((T, n + 3), T + n, scale=2.0)
    bias = _randn((n,), 5, scale=0.2) if biased else None
    ids, w = _route(l, n, top, bias=bias, score=score, groups=groups, top_groups=top_groups, scale=2.5)
    want, ww = route64(_np(l)[:, :n], top, score, None if bias is None else _np(bias), groups, top_groups, True, 2.5)
    assert np.array_equal(ids, want)
    assert np.allclose(w, ww, rtol=2 * E32, atol=0)        # one rounding of a 64-bit value
    ids2, w2 = _route(l, n, top, bias=bias, score=score, groups=groups, top_groups=top_groups, renorm=False)
    assert np.array_equal(ids2, want)
    assert np.allclose(w2, route64(_np(l)[:, :n], top, score, None if bias is None else _np(bias), groups, top_groups, False, 1.0)[1],
                       rtol=2 * E32, atol=0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,n,top,groups,top_groups", [(37, 1020, 10, 17, 5), (5, 1023, 32, 31, 31), (130, 1007, 7, 19, 1)])
def test_route_many_experts_a_lane(score, T, n, top, groups, top_groups):
    """Groups that are no power of two and have more than 32 experts, all of one lane; equal scores among them."""
    l = _randn((T, n), T, scale=2.0)
    l[::3] = torch.round(l[::3])
    l[1, :n // 2] = -float("inf")
    bias = _randn((n,), 6, scale=0.25).mul(8).round().div(8)
    ids, w = _route(l, n, top, bias=bias, score=score, groups=groups, top_groups=top_groups)
    want, ww = route64(_np(l), top, score, _np(bias), groups, top_groups, True, 1.0)
    assert np.array_equal(ids, want)
    assert np.allclose(w, ww, rtol=2 * E32, atol=1e-38)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_and_masks(score):
    n, inf = 16, float("inf")
    rows = [[0.0] * n, [1.0, 2.0] * 8, [-inf] * n, [-inf] * 15 + [3.0], [float("nan")] * 8 + [0.5] * 8, [5.0] + [-inf] * 14 + [float("nan")],
            [inf] + [0.0] * 15, [3.4e38] * n, [-3.4e38] * n, [-800.0] * 8 + [0.0] * 8, [88.0, -88.0] * 8]
    l = torch.tensor(rows).cuda()
    x = _np(torch.tensor(rows).clamp(max=3.402823466e38))
    for groups, top_groups, top in ((1, 1, 5), (4, 2, 6), (4, 4, 16), (16, 3, 3)):
        for bias in (None, -_randn((n,), 3).abs()):
            ids, w = _route(l, n, top, score=score, bias=bias, groups=groups, top_groups=top_groups)
            want, ww = route64(x, top, score, None if bias is None else _np(bias), groups, top_groups, True, 1.0)
            assert np.array_equal(ids, want), (groups, bias)
            assert np.allclose(w, ww, rtol=2 * E32, atol=1e-38)
    assert (w[2] == 0).all()


def test_route_decides_near_ties_in_64_bits():
    """Scores whose sums with the bias differ by far less than 2^-24."""
    n = 64
    l = torch.full((40, n), 0.25)
    l[torch.arange(40), torch.arange(40)] += 2.0 ** -24                # two steps up from 0.25
    ids, _ = _route(l.cuda(), n, 2, score="sigmoid", bias=torch.full((n,), 1000.0).cuda())
    assert np.array_equal(ids[:, 0], np.arange(40)) and np.array_equal(ids[:, 1], np.where(np.arange(40) == 0, 1, 0))


# --------------------------------------------------------------------------- experts

def _gelu(z):
    return L.gelu_tanh(z)


def _clamped(limit):
    return lambda g, u: np.minimum(g, limit) * L.sigmoid(1.702 * np.minimum(g, limit)) * (np.clip(u, -limit, limit) + 1)


GLU = {"gelu": ((0, 0.0, 0.0), lambda g, u: _gelu(g) * u), "clamped": ((1, 1.702, 1.2), _clamped(1.2))}


@pytest.fixture(params=["few", "group"])
def form(request, monkeypatch):
    """Both forms of the products, whatever the number of places."""
    monkeypatch.setattr(P, "GROUP_FROM", 1 if request.param == "group" else 10 ** 9)
    return request.param


def _ids(T, top, n, seed, how="spread"):
    g = torch.Generator().manual_seed(seed)
    if how == "one":                                   # everything to one expert (and its neighbours)
        return (torch.arange(top).repeat(T, 1) + n // 2).remainder(n).int()
    if how == "same":                                  # the same expert twice
        return torch.randint(0, n, (T, 1), generator=g).expand(T, top).contiguous().int()
    return torch.rand(T, n, generator=g).argsort(dim=1)[:, :top].contiguous().int()


SIZES = [  # T, top, n, K, F or M
    (1, 1, 1, 8, 1), (1, 2, 4, 24, 9), (1, 8, 64, 264, 136), (2, 3, 5, 40, 130), (17, 2, 3, 72, 33), (37, 4, 16, 896, 616), (64, 4, 8, 64, 128),
    (65, 1, 2, 128, 256), (200, 8, 16, 136, 264), (33, 32, 40, 16, 24), (300, 2, 70, 520, 136),
    (600, 1, 2, 200, 40), (515, 2, 2, 64, 300), (300, 2, 3, 136, 264), (290, 2, 3, 72, 520), (700, 1, 1, 64, 1030)]


def _check_glu(T, top, n, K, F, f32, how="spread", act="gelu", seed=1, ids=None):
    W, X = _randn((n, 2 * F, K), seed, DT[f32], 1.5 * K ** -0.5), _randn((T, K + 8), seed + 1, DT[f32])
    ids = _ids(T, top, n, seed + 2, how) if ids is None else ids
    dids = ids.cuda()
    op = P.Experts(W, gated=True, glu=GLU[act][0])
    H = torch.full((T * top + 2, F + 3), 7.0, dtype=DT[f32], device="cuda")
    op.hidden(X.data_ptr(), K + 8, op.plan(dids, T), H.data_ptr(), F + 3)
    x, w = _np(X)[:, :K], _np(W)
    got = _np(H)
    assert (got[T * top:] == 7).all() and (got[:, F:] == 7).all()
    for t in range(T):
        for j in range(top):
            e, row = int(ids[t, j]), got[t * top + j, :F]
            if not 0 <= e < n:
                assert (row == 7).all()
                continue
            v = w[e] @ x[t]
            want = GLU[act][1](v[:F], v[F:])
            # |d glu| <= |u| |d gelu| + |gelu| |du| with products of size about 1.5: sums of K products off by 8 sqrt(K) 2^-24
            tol = (8 * K ** 0.5 + 16) * E32 * (1 + np.abs(v[:F])) * (1 + np.abs(v[F:])) * 3
            assert (np.abs(row - want) <= tol + (0 if f32 else 2.0 ** -8 * np.abs(want))).all(), (t, j, np.abs(row - want).max())


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("T,top,n,K,F", SIZES)
def test_experts_glu(form, f32, T, top, n, K, F):
    _check_glu(T, top, n, K, F, f32)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("how", ["one", "same"])
def test_experts_glu_crowded(form, f32, how):
    _check_glu(150, 3, 9, 72, 136, f32, how, "clamped")
    _check_glu(3, 3, 9, 72, 136, f32, how, "clamped")


def _check_sum(T, top, n, K, M, f32, how="spread", ls=True, seed=11, ids=None):
    W, H = _randn((n, M, K), seed, DT[f32], K ** -0.5), _randn((T * top, K + 8), seed + 1, DT[f32])
    ids = _ids(T, top, n, seed + 2, how) if ids is None else ids
    w = torch.rand(T, top, generator=torch.Generator().manual_seed(seed)).cuda()
    s = _randn((M,), seed + 3) if ls else None
    Y0 = _randn((T + 1, M + 5), seed + 4)
    Y = Y0.clone()
    op = P.Experts(W, gated=False)
    op.add_sum(H.data_ptr(), K + 8, op.plan(ids.cuda(), T), w.data_ptr(), Y.data_ptr(), M + 5, ls=None if s is None else s.data_ptr())
    assert torch.equal(Y[T:], Y0[T:]) and torch.equal(Y[:, M:], Y0[:, M:])
    h, Wn, wn = _np(H)[:, :K].reshape(T, top, K), _np(W), _np(w)
    want, size = _np(Y0)[:T, :M].copy(), np.abs(_np(Y0)[:T, :M])
    for t in range(T):
        for j in range(top):
            e = int(ids[t, j])
            if 0 <= e < n:
                v = wn[t, j] * (Wn[e] @ h[t, j]) * (_np(s) if ls else 1)
                want[t] += v
                size[t] += wn[t, j] * (np.abs(Wn[e]) @ np.abs(h[t, j])) * (np.abs(_np(s)) if ls else 1)
    # a sum of K + top + 2 terms, each partial sum at most the sum of absolute values: n 2^-24 of it in the worst case
    assert (np.abs(_np(Y)[:T, :M] - want) <= (8 * K ** 0.5 + top + 2) * E32 * size).all()


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("T,top,n,K,M", SIZES)
def test_experts_sum(form, f32, T, top, n, K, M):
    _check_sum(T, top, n, K, M, f32)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("how", ["one", "same"])
def test_experts_sum_crowded(form, f32, how):
    _check_sum(150, 3, 9, 72, 136, f32, how, ls=False)
    _check_sum(3, 3, 9, 72, 136, f32, how, ls=False)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("T", [2, 90])
def test_experts_places_left_out(form, f32, T):
    """Ids below zero leave a place out; a token all of whose places are left out keeps its row."""
    ids = _ids(T, 4, 8, 3)
    ids[0] = -1
    ids[1, 2] = -5
    ids[T // 2, 0] = -1
    _check_glu(T, 4, 8, 72, 40, f32, ids=ids)
    _check_sum(T, 4, 8, 72, 40, f32, ids=ids)
    _check_glu(T, 4, 8, 72, 40, f32, ids=torch.full_like(ids, -1))
    _check_sum(T, 4, 8, 72, 40, f32, ids=torch.full_like(ids, -1))


@pytest.mark.parametrize("T", [2, 90])
def test_experts_ids_out_of_range_are_reported(form, T):
    ids = _ids(T, 4, 8, 3)
    ids[1, 1] = 8
    ids[T - 1, 3] = 2 ** 31 - 1
    _check_glu(T, 4, 8, 72, 40, 0, ids=ids)
    torch.cuda.synchronize()
    assert _lib.device_status() == {"bad_token"}
    _check_sum(T, 4, 8, 72, 40, 0, ids=ids)
    torch.cuda.synchronize()
    assert _lib.device_status() == {"bad_token"}


@pytest.mark.parametrize("T,top,n", [(1, 1, 1), (1, 8, 64), (100, 3, 7), (2048, 8, 256), (513, 2, 1024)])
def test_plan(T, top, n):
    ids = _ids(T, min(top, n), n, 7)
    ids.reshape(-1)[::11] = -1
    d = ids.cuda()
    plan = torch.full((_lib.dense().lt_dn_experts_plan_ints(T, ids.shape[1], n) + 1,), -9, dtype=torch.int32, device="cuda")
    _lib.call("lt_dn_experts_plan", d.data_ptr(), T, ids.shape[1], n, plan.data_ptr(), stream())
    flat, got = ids.reshape(-1).numpy(), plan.cpu().numpy()
    used = np.flatnonzero(flat >= 0)
    order = used[np.argsort(flat[used], kind="stable")]
    assert np.array_equal(got[:n + 1], np.searchsorted(np.sort(flat[used]), np.arange(n + 1)))
    assert np.array_equal(got[n + 1:n + 1 + len(order)], order)
    assert (got[n + 1 + len(order):] == -9).all()


# --------------------------------------------------------------------------- delta rule

def delta64(q, k, v, la, beta, S, q_scale, eps):
    """q, k [T, G, d], v [T, H, dv], S [H, dv, d] (a copy is advanced)."""
    T, H = v.shape[:2]
    per = H // q.shape[1]
    q, k = np.repeat(q, per, axis=1), np.repeat(k, per, axis=1)
    q = q_scale * q / np.sqrt((q ** 2).sum(-1, keepdims=True) + eps)
    k = k / np.sqrt((k ** 2).sum(-1, keepdims=True) + eps)
    S, o = S.copy(), np.zeros(v.shape)
    for t in range(T):
        S *= np.exp(la[t])[:, None, None]
        u = beta[t][:, None] * (v[t] - np.einsum("hvd,hd->hv", S, k[t]))
        S += u[:, :, None] * k[t][:, None, :]
        o[t] = np.einsum("hvd,hd->hv", S, q[t])
    return o, S


def _delta_case(lengths, H, G, d, dv, f32, seed=0, gap=0, strong=False, la=None, beta=None):
    """Rows [v | k | q | unused] of the sequences with `gap` rows between them."""
    g = torch.Generator().manual_seed(seed)
    C = H * dv + 2 * G * d
    R = sum(lengths) + gap * len(lengths)
    rows = torch.randn(R, C + 8, generator=g).to(DT[f32]).cuda()
    if la is None:
        la = -torch.rand(R, H, generator=g) * (30.0 if strong else 0.3)
    if beta is None:
        beta = torch.rand(R, H, generator=g)
    S = [torch.randn(H, dv, d, generator=g).cuda() for _ in lengths]
    return rows, la.float().cuda(), beta.float().cuda(), S


def _delta_run(rows, la, beta, S, lengths, H, G, d, dv, f32, gap=0, q_scale=0.25, eps=1e-6, call=None):
    """The rows through lt_dn_delta_rows, against 64 bits: largest error of o and of the states, over their size."""
    R, ld = rows.shape
    es = rows.element_size()
    o = torch.full((R, H * dv + 2), 7.0, device="cuda")
    op = P.DeltaRule(H, G, d, dv, DT[f32], q_scale, eps)
    v = rows.data_ptr()
    k = v + H * dv * es
    before = [s.clone() for s in S]
    if gap == 0:
        op.rows(k + G * d * es, k, v, ld, la.data_ptr(), beta.data_ptr(), H, o.data_ptr(), H * dv + 2, [s.data_ptr() for s in S], lengths)
    else:
        seqs = _lib.DnSeqs(n=len(lengths))
        at = 0
        for i, n in enumerate(lengths):
            at += gap
            seqs.start[i], seqs.rows[i], seqs.S[i] = at, n, S[i].data_ptr()
            at += n
        call(op, k + G * d * es, k, v, ld, la, beta, o, seqs)
    at, eo, eS = 0, 0.0, 0.0
    x, lan, ben, got = _np(rows), _np(la), _np(beta), _np(o)
    assert (got[:, H * dv:] == 7).all()
    for i, n in enumerate(lengths):
        assert (got[at:at + gap] == 7).all()
        at += gap
        r = x[at:at + n]
        if n:
            wo, wS = delta64(r[:, H * dv + G * d:H * dv + 2 * G * d].reshape(n, G, d), r[:, H * dv:H * dv + G * d].reshape(n, G, d),
                             r[:, :H * dv].reshape(n, H, dv), lan[at:at + n], ben[at:at + n], _np(before[i]), q_scale, eps)
            eo = max(eo, _off(got[at:at + n, :H * dv], wo.reshape(n, -1)))
            eS = max(eS, _off(_np(S[i]), wS))
        else:
            assert torch.equal(S[i], before[i])
        at += n
    return eo, eS


# A token's u k^T passes about 20 roundings (convolution, silu, norms, the product with the state, the correction), each 2^-24 of
# the value that is rounded, and so is off in proportion to its own size, not to the mean size of the state: errors are counted
# against the largest value.  They add up over tokens as random signs do, and what an error does to later corrections stays
# bounded (unit keys, beta at most 1): 16 sqrt(T) 2^-24, at least 64 2^-24 for few tokens (20 roundings, threefold).
def _delta_tol(n):
    return max(64, 16 * n ** 0.5) * E32


DELTA = [  # lengths, H, G, d, dv
    ([1], 1, 1, 8, 8), ([1], 3, 1, 24, 40), ([2, 1, 5], 4, 2, 16, 24), ([16], 2, 2, 64, 64), ([17, 0, 33], 4, 4, 128, 128), ([63, 64, 65], 6, 2, 40, 72),
    ([200], 2, 1, 136, 8), ([7] * 8, 2, 2, 8, 136), ([3] * 11, 1, 1, 32, 32), ([130, 1], 2, 2, 264, 16), ([5, 40], 1, 1, 512, 24), ([333], 3, 3, 72, 48)]


@pytest.fixture(params=["order", "order-f32", "chunks"])
def walk(request, monkeypatch):
    """Token order in both types, and chunks, whatever the number of rows: the value is f32."""
    monkeypatch.setattr(P, "DELTA_CHUNKED_FROM", 1 if request.param == "chunks" else 10 ** 9)
    return int(request.param == "order-f32")


@pytest.mark.parametrize("lengths,H,G,d,dv", DELTA)
def test_delta_rows(walk, lengths, H, G, d, dv):
    f32 = walk
    for strong in (False, True):
        rows, la, beta, S = _delta_case(lengths, H, G, d, dv, f32, seed=len(lengths) + d, strong=strong)
        eo, eS = _delta_run(rows, la, beta, S, lengths, H, G, d, dv, f32)
        assert eo <= _delta_tol(max(lengths)) and eS <= _delta_tol(max(lengths)), (eo, eS)


@pytest.mark.parametrize("lengths,H,G,d,dv", [
    ([130, 65], 2, 1, 256, 256), ([70], 1, 1, 192, 128), ([70, 64], 2, 1, 256, 512), ([129], 3, 3, 136, 72), ([200], 1, 1, 248, 504), ([65], 2, 2, 128, 512),
    ([140], 1, 1, 64, 200)])
def test_delta_chunks_of_large_heads(lengths, H, G, d, dv, monkeypatch):
    """Every variant of the chunked walk and of its outputs, full and with ragged tiles, and that it is the one that runs."""
    names, call = [], _lib.call
    monkeypatch.setattr(P, "DELTA_CHUNKED_FROM", 1)
    monkeypatch.setattr(_lib, "call", lambda name, *a: (names.append(name), call(name, *a)))
    for strong in (False, True):
        rows, la, beta, S = _delta_case(lengths, H, G, d, dv, 0, seed=d, strong=strong)
        eo, eS = _delta_run(rows, la, beta, S, lengths, H, G, d, dv, 0)
        assert eo <= _delta_tol(max(lengths)) and eS <= _delta_tol(max(lengths)), (eo, eS)
    assert names == ["lt_dn_delta_chunked"] * 2


@pytest.mark.parametrize("chunks,f32", [(0, 0), (0, 1), (1, 0)])
def test_delta_rows_between_other_rows(chunks, f32):
    lengths, H, G, d, dv = [5, 0, 70], 4, 2, 24, 40

    def call(op, q, k, v, ld, la, beta, o, seqs):
        args = (q, k, v, ld, la.data_ptr(), H, beta.data_ptr(), H, o.data_ptr(), H * dv + 2)
        if not chunks:
            _lib.call("lt_dn_delta_rows", *args, f32, op._ref, ctypes.byref(seqs), stream())
            return
        n = _lib.dense().lt_dn_delta_chunked_ws(op._ref, ctypes.byref(seqs))
        ws = torch.full((n + 4,), float("nan"), device="cuda")
        _lib.call("lt_dn_delta_chunked", *args, op._ref, ctypes.byref(seqs), ws.data_ptr(), stream())
        assert torch.isnan(ws[n:]).all()
    rows, la, beta, S = _delta_case(lengths, H, G, d, dv, f32, seed=4, gap=3)
    eo, eS = _delta_run(rows, la, beta, S, lengths, H, G, d, dv, f32, gap=3, call=call)
    assert eo <= _delta_tol(70) and eS <= _delta_tol(70)


@pytest.mark.parametrize("T", [3, 150])
def test_delta_extremes(walk, T):
    """Nothing written (beta 0), everything forgotten (la minus infinity), no decay, zero keys and queries, full corrections with
    keys that repeat, a growing state."""
    f32, H, G, d, dv = walk, 6, 6, 32, 24
    rows, la, beta, S = _delta_case([T], H, G, d, dv, f32, seed=9)
    la[:, 1:] = 0.0
    la[:, 0] = -float("inf")
    la[T // 2, 1] = -float("inf")
    la[:, 2] = -1e30
    la[:, 3] = 0.01
    beta[:, 1] = 0.0
    beta[:, 4] = 1.0
    k0 = H * dv
    rows[:, k0 + 4 * d:k0 + 5 * d] = rows[0, k0 + 4 * d:k0 + 5 * d]        # head 4: one key for all tokens
    rows[:, k0 + 5 * d:k0 + 6 * d] = 0.0                                   # head 5: no key
    rows[1, k0 + G * d:k0 + 2 * G * d] = 0.0                               # token 1: no query
    eo, eS = _delta_run(rows, la, beta, S, [T], H, G, d, dv, f32)
    assert eo <= _delta_tol(T) and eS <= _delta_tol(T), (eo, eS)


@pytest.mark.parametrize("what", ["v", "k", "q", "la", "beta"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_delta_rows_that_are_not_finite(walk, monkeypatch, what, value):
    """A number that is not finite reaches its head's outputs from its token on (in chunks: from its chunk on), and nothing else: the
    rows before, the other heads and the other sequences keep their bits."""
    f32, H, d, dv, lengths, at = walk, 2, 32, 24, [50, 200, 70], 50 + 135
    first = 50 + 128 if P.DELTA_CHUNKED_FROM == 1 else at
    out = []
    for bad in (False, True):
        rows, la, beta, S = _delta_case(lengths, H, H, d, dv, f32, seed=7)
        if bad:
            if what in ("la", "beta"):
                (la if what == "la" else beta)[at, 0] = value
            else:
                rows[at, {"v": 0, "k": H * dv, "q": H * dv + H * d}[what] + 3] = value
        o = torch.empty(sum(lengths), H * dv, device="cuda")
        v, es, ld = rows.data_ptr(), rows.element_size(), rows.shape[1]
        k = v + H * dv * es
        P.DeltaRule(H, H, d, dv, DT[f32], 0.25, 1e-6).rows(k + H * d * es, k, v, ld, la.data_ptr(), beta.data_ptr(), H, o.data_ptr(), H * dv,
                                                         [s.data_ptr() for s in S], lengths)
        out.append((o, S))
    (o, S), (p, Z) = out
    assert torch.equal(p[:first], o[:first]) and torch.equal(p[250:], o[250:]) and torch.equal(p[:, dv:], o[:, dv:])
    assert torch.equal(Z[0], S[0]) and torch.equal(Z[2], S[2]) and torch.equal(Z[1][1], S[1][1])
    reached = ~torch.isfinite(p[:, :dv])
    assert reached[at].any() and (what == "q" or reached[at:250].any(1).all())
    if what == "q":
        assert torch.equal(p[at + 1:250], o[at + 1:250]) and torch.equal(Z[1], S[1])


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("H,G,d,dv,taps", [(1, 1, 8, 8, 1), (4, 2, 16, 24, 4), (6, 3, 40, 72, 3), (2, 2, 128, 128, 4), (3, 1, 264, 16, 5), (2, 1, 512, 40, 2)])
def test_delta_steps(f32, H, G, d, dv, taps):
    """Tokens one by one from an empty ring, each with its convolution, against the whole sequence in 64 bits."""
    T, C = 2 * taps + 3, H * dv + 2 * G * d
    u = _randn((T, C), 1, DT[f32])
    conv, conv_b = _randn((taps, C), 2, scale=taps ** -0.5), _randn((C,), 3, scale=0.1)
    dt, beta, dt_bias, A = _randn((T, H), 4), torch.sigmoid(_randn((T, H), 5)), _randn((H,), 6), -torch.exp(_randn((H,), 7))
    op = P.DeltaRule(H, G, d, dv, DT[f32], d ** -0.5, 1e-6, taps=taps, conv=conv, conv_b=conv_b, dt_bias=dt_bias, A=A)
    S = torch.zeros(H, dv, d, device="cuda")
    ring = torch.full((taps, C), float("nan"), dtype=DT[f32], device="cuda")       # rows of positions that do not exist are not read
    ln, ticket = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    o = torch.empty(T, H * dv, device="cuda")
    for t in range(T):
        op.step(u[t].data_ptr(), dt[t].data_ptr(), beta[t].data_ptr(), ring.data_ptr(), S.data_ptr(), o[t].data_ptr(), ln.data_ptr(),
                ticket.data_ptr())
    assert ln.item() == T and ticket.item() == 0
    x = np.zeros((T, C))
    for t in range(T):
        for i in range(taps):
            if t - (taps - 1 - i) >= 0:
                x[t] += _np(conv)[i] * _np(u)[t - (taps - 1 - i)]
    x = L.silu(x + _np(conv_b))
    la = _np(A) * np.log1p(np.exp(_np(dt) + _np(dt_bias)))
    wo, wS = delta64(x[:, H * dv + G * d:].reshape(T, G, d), x[:, H * dv:H * dv + G * d].reshape(T, G, d), x[:, :H * dv].reshape(T, H, dv), la,
                     _np(beta), np.zeros((H, dv, d)), d ** -0.5, 1e-6)
    eo, eS = _off(_np(o), wo.reshape(T, -1)), _off(_np(S), wS)
    assert eo <= _delta_tol(T) and eS <= _delta_tol(T)


# --------------------------------------------------------------------------- as they are used together

@pytest.mark.parametrize("f32", [0, 1])
def test_places_left_out_are_not_read(form, f32):
    """NaN in rows, weights and outputs of places that are left out, and in the columns behind a row's last."""
    T, top, n, K, M = 70, 3, 5, 40, 24
    nan = float("nan")
    ids = _ids(T, top, n, 1)
    ids[::4] = -1
    ids[1::4, 1] = -1
    off = (ids < 0).cuda()
    X, H = _randn((T, K + 8), 2, DT[f32]), _randn((T * top, K + 8), 3, DT[f32])
    w = torch.rand(T, top, generator=torch.Generator().manual_seed(4)).cuda()
    Wg, Wd = _randn((n, 2 * M, K), 5, DT[f32], K ** -0.5), _randn((n, M, K), 6, DT[f32], K ** -0.5)
    gu, down = P.Experts(Wg, gated=True), P.Experts(Wd, gated=False)

    def run():
        places = gu.plan(ids.cuda(), T)
        h, y = torch.zeros(T * top, M, dtype=DT[f32], device="cuda"), torch.zeros(T, M, device="cuda")
        gu.hidden(X.data_ptr(), K + 8, places, h.data_ptr(), M)
        down.add_sum(H.data_ptr(), K + 8, places, w.data_ptr(), y.data_ptr(), M)
        return h, y
    want = run()
    X[:, K:], H[:, K:] = nan, nan
    X[off.all(1)] = nan
    H[off.reshape(-1)] = nan
    w[off] = nan
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("chunks,f32", [(0, 0), (0, 1), (1, 0)])
def test_delta_reads_no_rows_of_others(chunks, f32):
    lengths, H, G, d, dv = [5, 1, 70], 4, 2, 24, 40

    def call(op, q, k, v, ld, la, beta, o, seqs):
        args = (q, k, v, ld, la.data_ptr(), H, beta.data_ptr(), H, o.data_ptr(), H * dv + 2)
        if not chunks:
            _lib.call("lt_dn_delta_rows", *args, f32, op._ref, ctypes.byref(seqs), stream())
            return
        ws = torch.full((_lib.dense().lt_dn_delta_chunked_ws(op._ref, ctypes.byref(seqs)),), float("nan"), device="cuda")
        _lib.call("lt_dn_delta_chunked", *args, op._ref, ctypes.byref(seqs), ws.data_ptr(), stream())
    rows, la, beta, S = _delta_case(lengths, H, G, d, dv, f32, seed=4, gap=2)
    rows[:, -8:] = float("nan")
    for at in (0, 7, 10):
        for t in (rows, la, beta):
            t[at:at + 2] = float("nan")
    eo, eS = _delta_run(rows, la, beta, S, lengths, H, G, d, dv, f32, gap=2, call=call)
    assert eo <= _delta_tol(70) and eS <= _delta_tol(70)


class _Layer:
    """A router, experts and a delta rule on buffers of their own: one pass over them, as a layer makes it."""

    def __init__(self, T, f32, seed):
        n, top, E, F, H, d = 8, 2, 64, 40, 2, 32
        self.T, self.n, self.top, self.E, self.F, self.H, self.d = T, n, top, E, F, H, d
        dt = DT[f32]
        self.router = P.Router(n, top, score="sigmoid", bias=_randn((n,), seed, scale=0.1))
        self.gu = P.Experts(_randn((n, 2 * F, E), seed + 1, dt, E ** -0.5), gated=True)
        self.down = P.Experts(_randn((n, E, F), seed + 2, dt, F ** -0.5), gated=False)
        self.rule = P.DeltaRule(H, H, d, d, dt, d ** -0.5, 1e-6)
        self.logits, self.x = _randn((T, n), seed + 3), _randn((T, E), seed + 4, dt)
        self.row = _randn((T, 3 * H * d), seed + 5, dt)
        self.la, self.beta = -torch.rand(T, H, device="cuda"), torch.rand(T, H, device="cuda")
        self.S0, self.S = _randn((H, d, d), seed + 6), torch.empty(H, d, d, device="cuda")
        self.y, self.o = torch.empty(T, E, device="cuda"), torch.empty(T, H * d, device="cuda")
        self.h = torch.empty(T * top, F, dtype=dt, device="cuda")
        self.ids = torch.empty(T, top, dtype=torch.int32, device="cuda")
        self.w = torch.empty(T, top, device="cuda")

    def run(self):
        T, e, n = self.T, self.row.element_size(), self.H * self.d
        self.y.zero_()
        self.S.copy_(self.S0)
        self.router.rows(self.logits.data_ptr(), self.n, self.ids.data_ptr(), self.w.data_ptr(), T)
        places = self.gu.plan(self.ids, T)
        self.gu.hidden(self.x.data_ptr(), self.E, places, self.h.data_ptr(), self.F)
        self.down.add_sum(self.h.data_ptr(), self.F, places, self.w.data_ptr(), self.y.data_ptr(), self.E)
        r = self.row.data_ptr()
        self.rule.rows(r + 2 * n * e, r + n * e, r, 3 * n, self.la.data_ptr(), self.beta.data_ptr(), self.H, self.o.data_ptr(), n,
                       [self.S.data_ptr()], [T])

    def out(self):
        return [t.clone() for t in (self.ids, self.w, self.h, self.y, self.o, self.S)]


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("T", [1, 300])
def test_captured_passes_side_by_side(f32, T):
    """Two captured graphs replayed at once on two streams, with inputs changed after the capture, and eager passes on a stream of
    their own between them: every one gives what a pass alone gives, bit by bit."""
    a, b, c = _Layer(T, f32, 10), _Layer(T, f32, 20), _Layer(T, f32, 30)
    graphs = []
    for l in (a, b):
        l.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            l.run()
        graphs.append(g)
    for l, seed in ((a, 50), (b, 60)):
        l.logits.copy_(_randn((T, l.n), seed))
        l.x.copy_(_randn((T, l.E), seed + 1, DT[f32]))
        l.row.copy_(_randn((T, l.row.shape[1]), seed + 2, DT[f32]))
    want = []
    for l in (a, b, c):
        l.run()
        want.append(l.out())
        for t in (l.ids, l.w, l.h, l.y, l.o, l.S):
            t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            c.run()
    torch.cuda.synchronize()
    for l, ws in zip((a, b, c), want):
        for got, w in zip(l.out(), ws):
            assert torch.equal(got, w)


@pytest.mark.parametrize("f32", [0, 1])
def test_many_places(f32):
    """160000 places."""
    T, top, n, K, M = 20000, 8, 64, 40, 24
    ids = _ids(T, top, n, 1).cuda()
    X, W = _randn((T, K), 2, DT[f32]), _randn((n, 2 * M, K), 3, DT[f32], K ** -0.5)
    gu = P.Experts(W, gated=True)
    places = gu.plan(ids, T)
    h = torch.full((T * top, M), 7.0, dtype=DT[f32], device="cuda")
    gu.hidden(X.data_ptr(), K, places, h.data_ptr(), M)
    D, w = _randn((n, K, M), 4, DT[f32], M ** -0.5), torch.rand(T, top, device="cuda")
    y = torch.zeros(T, K, device="cuda")
    P.Experts(D, gated=False).add_sum(h.data_ptr(), M, places, w.data_ptr(), y.data_ptr(), K)
    want, size = torch.zeros(T, K, dtype=torch.float64, device="cuda"), torch.zeros(T, K, dtype=torch.float64, device="cuda")
    for j in range(top):
        e = ids[:, j].long()
        for t0 in range(0, T, 4000):
            s = slice(t0, t0 + 4000)
            v = torch.einsum("tmk,tk->tm", W[e[s]].double(), X[s].double())
            g, u = v[:, :M], v[:, M:]
            gu64 = 0.5 * g * (1 + torch.tanh((2 / np.pi) ** 0.5 * (g + 0.044715 * g ** 3))) * u
            hj = h.reshape(T, top, M)[s, j].double()
            tol = (8 * K ** 0.5 + 16) * E32 * (1 + g.abs()) * (1 + u.abs()) * 3 + (0 if f32 else 2.0 ** -8) * gu64.abs()     # as above
            assert ((hj - gu64).abs() <= tol).all()
            want[s] += w[s, j, None] * torch.einsum("tmk,tk->tm", D[e[s]].double(), hj)
            size[s] += w[s, j, None] * torch.einsum("tmk,tk->tm", D[e[s]].double().abs(), hj.abs())
    assert ((y - want).abs() <= (8 * M ** 0.5 + top + 2) * E32 * size).all()


@pytest.mark.parametrize("each", [15, 48, 200])
def test_grouped_products_in_several_rounds(each):
    """Three and more tiles a CTA, eleven blocks of k each (the last ragged), for 64, 128 and 256 places a tile: places of the ring and
    sets of accumulators are used again from one tile to the next.  Shares of the experts are unequal, some have none."""
    n, top, M, K = 34, 2, 4144, 648
    T = each * n // top
    g = torch.Generator().manual_seed(each)
    share = torch.rand(n - 2, generator=g) + 0.2
    ids = torch.multinomial(share, T * top, replacement=True, generator=g).reshape(T, top).int().cuda()
    W, X = _randn((n, M, K), 1, torch.bfloat16, 1.5 * K ** -0.5), _randn((T, K), 2, torch.bfloat16)
    H, w, Y0 = _randn((T * top, K), 3, torch.bfloat16), torch.rand(T, top, generator=g).cuda(), _randn((T, M), 4)
    gu, down, F = P.Experts(W, gated=True), P.Experts(W, gated=False), M // 2
    out = []
    for _ in range(2):
        places = gu.plan(ids, T)
        h, y = torch.full((T * top, F), 7.0, dtype=torch.bfloat16, device="cuda"), Y0.clone()
        gu.hidden(X.data_ptr(), K, places, h.data_ptr(), F)
        down.add_sum(H.data_ptr(), K, places, w.data_ptr(), y.data_ptr(), M)
        out.append((h, y))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    want, size = Y0.double(), Y0.double().abs()
    for e in range(n):
        at = (ids.reshape(-1) == e).nonzero()[:, 0]
        t, We = at // top, W[e].double()
        v = X[t].double() @ We.T
        a, b = v[:, :F], v[:, F:]
        glu = 0.5 * a * (1 + torch.tanh((2 / np.pi) ** 0.5 * (a + 0.044715 * a ** 3))) * b
        # of _check_glu; the tensor cores cut off at most 2^-23 of a sum at each of K / 16 steps, which 8 sqrt(K) 2^-24 covers up to K = 4096
        tol = (8 * K ** 0.5 + 16) * E32 * (1 + a.abs()) * (1 + b.abs()) * 3 + 2.0 ** -8 * glu.abs()
        assert ((h[at].double() - glu).abs() <= tol).all(), e
        a = w.reshape(-1)[at, None].double()
        want.index_add_(0, t, a * (H[at].double() @ We.T))
        size.index_add_(0, t, a * (H[at].double().abs() @ We.abs().T))
    assert ((y.double() - want).abs() <= (8 * K ** 0.5 + top + 2) * E32 * size).all()


def test_order_of_the_places_read_on_another_stream():
    """The products of a plan run on another stream, behind a delay, after the plan's object is gone and its stream allocates again."""
    T, top, n, K, F = 3000, 4, 16, 64, 40
    ids, X = _ids(T, top, n, 1).cuda(), _randn((T, K), 2, torch.bfloat16)
    gu = P.Experts(_randn((n, 2 * F, K), 3, torch.bfloat16, K ** -0.5), gated=True)
    h = torch.zeros(2, T * top, F, dtype=torch.bfloat16, device="cuda")
    gu.hidden(X.data_ptr(), K, gu.plan(ids, T), h[0].data_ptr(), F)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    places = gu.plan(ids, T)
    size = places.buf.numel()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)            # about 10 ms
        gu.hidden(X.data_ptr(), K, places, h[1].data_ptr(), F)
    del places
    junk = [torch.zeros(size, dtype=torch.int32, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(h[0], h[1]) and len(junk) == 8


def test_matrices_past_32_bits(form):
    """The last experts of matrices of 2.2e9 elements."""
    n, M, K, T = 131, 1024, 8192, 40
    W = torch.zeros(n, 2 * M, K, dtype=torch.bfloat16, device="cuda")
    W[-2:] = _randn((2, 2 * M, K), 1, torch.bfloat16, K ** -0.5)
    ids = (n - 2 + torch.arange(2 * T) % 2).reshape(T, 2).int().cuda()
    X, h = _randn((T, K), 2, torch.bfloat16), torch.empty(2 * T, M, dtype=torch.bfloat16, device="cuda")
    gu = P.Experts(W, gated=True, glu=GLU["clamped"][0])
    places = gu.plan(ids, T)
    gu.hidden(X.data_ptr(), K, places, h.data_ptr(), M)
    down = P.Experts(W, gated=False)
    y, w = torch.zeros(2 * T, 2 * M, device="cuda"), torch.ones(2 * T, 1, device="cuda")
    X2 = X.repeat_interleave(2, 0)
    places = down.plan(ids.reshape(-1, 1), 2 * T)
    down.add_sum(X2.data_ptr(), K, places, w.data_ptr(), y.data_ptr(), 2 * M)
    x = _np(X).repeat(2, 0).reshape(T, 2, K)
    for j in range(2):
        v = x[:, j] @ _np(W[n - 2 + j]).T
        size = np.abs(x[:, j]) @ np.abs(_np(W[n - 2 + j])).T
        assert (np.abs(_np(y).reshape(T, 2, -1)[:, j] - v) <= (8 * K ** 0.5 + 3) * E32 * size).all()
        want = GLU["clamped"][1](v[:, :M], v[:, M:])
        tol = (8 * K ** 0.5 + 16) * E32 * (1 + np.abs(v[:, :M])) * (1 + np.abs(v[:, M:])) * 3 + 2.0 ** -8 * np.abs(want)
        assert (np.abs(_np(h).reshape(T, 2, -1)[:, j] - want) <= tol).all()


def test_delta_long_sequences_in_portions(monkeypatch):
    """Sequences longer than a portion of the chunked walk give the bits of one portion."""
    lengths, H, G, d, dv = [300, 0, 65, 128, 1], 4, 2, 24, 40
    monkeypatch.setattr(P, "DELTA_CHUNKED_FROM", 1)
    out = []
    for portion in (4096, 128):
        monkeypatch.setattr(P, "DELTA_PORTION", portion)
        rows, la, beta, S = _delta_case(lengths, H, G, d, dv, 0, seed=6)
        eo, eS = _delta_run(rows, la, beta, S, lengths, H, G, d, dv, 0)
        assert eo <= _delta_tol(300) and eS <= _delta_tol(300)
        out.append(S)
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_delta_rows_far_apart(walk):
    """Rows 2^20 elements and more apart: offsets past 2^31."""
    f32, T, H, d = walk, 2100, 1, 8
    ld = 2 ** 20 + 32
    rows = torch.empty(T, ld, dtype=DT[f32], device="cuda")
    rows[:, :3 * d] = _randn((T, 3 * d), 1, DT[f32])
    o = torch.empty(T, ld, device="cuda")
    la, beta, S0 = -torch.rand(T, H, device="cuda") * 0.3, torch.rand(T, H, device="cuda"), _randn((H, d, d), 2)
    S = S0.clone()
    p, e = rows.data_ptr(), rows.element_size()
    P.DeltaRule(H, H, d, d, DT[f32], 0.25, 1e-6).rows(p + 2 * d * e, p + d * e, p, ld, la.data_ptr(), beta.data_ptr(), H, o.data_ptr(), ld,
                                                    [S.data_ptr()], [T])
    x = _np(rows[:, :3 * d])[:, None]
    wo, wS = delta64(x[..., 2 * d:], x[..., d:2 * d], x[..., :d], _np(la), _np(beta), _np(S0), 0.25, 1e-6)
    assert _off(_np(o[:, :d]), wo[:, 0]) <= _delta_tol(T) and _off(_np(S), wS) <= _delta_tol(T)

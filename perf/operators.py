"""Timed cases of the operators of sparse hybrid layers: the gated delta rule (a mixer's recurrence), routing to experts, and the
two products of the experts' feed-forward, through the calls that the mixers and feed-forwards of `layered` make.

Sizes are those of the mixer-layer models (widths 896, 2048 and 4096, heads of 64 and 128) with feed-forwards of many small experts.
Inputs come from the seed; recurrent states, rings and residual rows are updated in place, as in a reply.
"""
import math

import torch

own = False
F64 = torch.float64


def listed():
    return [
        # a reply's token: scores of 64 experts, the smallest call there is; launch latency
        dict(name="route-1", kind="route", tokens=1, experts=64, top=6, score="softmax", bias=False, groups=1, top_groups=1),
        # a long prompt's tokens, choice with a balancing bias inside the best groups
        dict(name="route-2048", kind="route", tokens=2048, experts=256, top=8, score="sigmoid", bias=True, groups=8, top_groups=4),
        # a reply's token through its experts' gate and up matrices: 67 MB of weights, memory bound
        dict(name="glu-1", kind="glu", dtype="bfloat16", tokens=1, experts=64, top=8, width=2048, ff=1024),
        # a prompt portion, every expert hit, tensor cores; the largest case
        dict(name="glu-2000", kind="glu", dtype="bfloat16", tokens=2000, experts=64, top=8, width=2048, ff=1024),
        # the fp32 option of the 896-wide model, a short question; odd sizes
        dict(name="glu-f32-37", kind="glu", dtype="float32", tokens=37, experts=16, top=4, width=896, ff=616),
        # the way back to the residual rows: one token, a short question with ragged shares, a prompt portion
        dict(name="sum-1", kind="sum", dtype="bfloat16", tokens=1, experts=64, top=8, width=2048, ff=1024),
        dict(name="sum-203", kind="sum", dtype="bfloat16", tokens=203, experts=32, top=4, width=4096, ff=1408),
        dict(name="sum-2000", kind="sum", dtype="bfloat16", tokens=2000, experts=64, top=8, width=2048, ff=1024),
        # a reply's token in a delta-rule layer: convolution, step sizes and recurrence
        dict(name="delta-step", kind="step", dtype="bfloat16", heads=32, key_heads=16, dim=128, vdim=128, taps=4),
        # prompts: one long portion, three questions of different lengths in one pass (heads of 64, keys shared by pairs)
        dict(name="delta-2048", kind="delta", dtype="bfloat16", lengths="2048", heads=16, key_heads=16, dim=128, vdim=128),
        dict(name="delta-ragged", kind="delta", dtype="bfloat16", lengths="701,64,333", heads=28, key_heads=14, dim=64, vdim=64),
        # the fp32 option, walked token by token
        dict(name="delta-f32", kind="delta", dtype="float32", lengths="300", heads=14, key_heads=14, dim=64, vdim=72),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "glu", "glu", "sum", "sum", "step", "delta", "delta", "delta"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        n = groups * _log(rng, max(2, 8 // groups), 512 // groups)
        top_groups = rng.randint(1, groups)
        return dict(kind=kind, tokens=_log(rng, 1, 2048), experts=n, top=min(rng.randint(1, 10), n // groups * top_groups),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, top_groups=top_groups)
    if kind in ("glu", "sum"):
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        n = _log(rng, 4, 128)
        width, ff = 8 * _log(rng, 16, 512), 8 * _log(rng, 8, 256)
        n = max(4, min(n, (1 << 27) // (width * ff)))
        top = rng.randint(1, min(8, n))
        most = min(2000 if dtype == "bfloat16" else 300, (1 << 35) // (top * width * ff))
        return dict(kind=kind, dtype=dtype, tokens=_log(rng, 1, max(2, most)), experts=n, top=top, width=width, ff=ff)
    G = rng.randint(1, 16)
    per = rng.choice([1, 2]) if G <= 16 else 1
    size = dict(heads=G * per, key_heads=G, dim=8 * rng.randint(2, 16), vdim=8 * rng.randint(2, 16))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if kind == "step":
        return dict(kind=kind, dtype=dtype, taps=rng.randint(2, 4), **size)
    n = rng.randint(1, 4)
    most = (2048 if dtype == "bfloat16" else 400) // n
    return dict(kind=kind, dtype=dtype, lengths=",".join(str(_log(rng, 1, most)) for _ in range(n)), **size)


# --------------------------------------------------------------------------- inputs

def _choice(g, T, n, top):
    """Experts of every token as a router that is not quite balanced gives them, and their weights."""
    s = torch.randn(T, n, generator=g, device="cuda") + 0.5 * torch.randn(n, generator=g, device="cuda")
    w, ids = torch.topk(torch.softmax(s, dim=1), top, dim=1)
    return ids.int().contiguous(), (w / w.sum(dim=1, keepdim=True)).contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = c["kind"]

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=dtype) * scale).contiguous()
    st = {"case": c}
    if kind == "route":
        st["logits"] = randn(c["tokens"], c["experts"], scale=1.5)
        st["bias"] = randn(c["experts"], scale=0.1) if c["bias"] else None
        if own:
            from llamatov_b200 import dense_ops
            st["op"] = dense_ops.Router(c["experts"], c["top"], score=c["score"], bias=st["bias"], groups=c["groups"],
                                        top_groups=c["top_groups"], renorm=True, scale=1.0)
        return st
    dt = getattr(torch, c["dtype"])
    if kind in ("glu", "sum"):
        T, n, top, E, F = c["tokens"], c["experts"], c["top"], c["width"], c["ff"]
        st["ids"], st["w"] = _choice(g, T, n, top)
        if kind == "glu":
            st["W"] = randn(n, 2 * F, E, dtype=dt, scale=E ** -0.5)          # gate rows, then up rows
            st["x"] = randn(T, E, dtype=dt)
        else:
            st["W"] = randn(n, E, F, dtype=dt, scale=F ** -0.5)
            st["h"] = randn(T, top, F, dtype=dt, scale=0.5)
            st["y"] = randn(T, E)                                             # the residual rows
            st["ls"] = 0.5 + 0.05 * randn(E)
        if own:
            from llamatov_b200 import dense_ops
            st["op"] = dense_ops.Experts(st["W"], gated=kind == "glu")
        return st
    H, G, d, dv = c["heads"], c["key_heads"], c["dim"], c["vdim"]
    st["q_scale"], st["eps"] = d ** -0.5, 1e-6
    C = H * dv + 2 * G * d
    if kind == "step":
        st["S"] = [randn(H, dv, d, scale=0.1)]
        st["row"] = randn(C, dtype=dt)                                        # values | keys | queries, ahead of the convolution
        st["ring"] = randn(c["taps"], C, dtype=dt)
        st["conv"], st["conv_b"] = randn(c["taps"], C, scale=c["taps"] ** -0.5), randn(C, scale=0.1)
        st["dt"], st["beta"] = randn(H), torch.sigmoid(randn(H))
        st["dt_bias"], st["A"] = randn(H, scale=0.5) - 2, -torch.exp(randn(H, scale=0.5))
        st["pos"] = 100
        if own:
            from llamatov_b200 import dense_ops
            st["op"] = dense_ops.DeltaRule(H, G, d, dv, dt, q_scale=st["q_scale"], eps=st["eps"], taps=c["taps"], conv=st["conv"],
                                           conv_b=st["conv_b"], dt_bias=st["dt_bias"], A=st["A"])
            st["len"] = torch.full((1,), st["pos"], dtype=torch.int32, device="cuda")
            st["ticket"] = torch.zeros(1, dtype=torch.int32, device="cuda")
            st["o"] = torch.empty(H, dv, device="cuda")
        return st
    lengths = [int(x) for x in c["lengths"].split(",")]
    T = sum(lengths)
    st["lengths"] = lengths
    st["S"] = [randn(H, dv, d, scale=0.1) for _ in lengths]
    x = randn(T, C)
    st["rows"] = (x * torch.sigmoid(x)).to(dt)                                # values | keys | queries, behind convolution and silu
    st["beta"] = torch.sigmoid(randn(T, H))
    rate = torch.exp(randn(H, scale=1.5) - 1)                                 # heads that forget slowly and ones that forget at once
    st["la"] = -(rate * torch.nn.functional.softplus(randn(T, H) - 2)).contiguous()
    if own:
        from llamatov_b200 import dense_ops
        st["op"] = dense_ops.DeltaRule(H, G, d, dv, dt, q_scale=st["q_scale"], eps=st["eps"])
    return st


# --------------------------------------------------------------------------- plain forms

def _route(st):
    """Choice values in 64 bits: what decides between two experts may differ in the last bits of 32."""
    c, l = st["case"], st["logits"].double()
    T, n = l.shape
    if c["score"] == "softmax":
        e = torch.exp(l - l.max(dim=1, keepdim=True).values)
        s = e / e.sum(dim=1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-l))
    choice = s if st["bias"] is None else s + st["bias"].double()
    if c["groups"] > 1:
        by = choice.reshape(T, c["groups"], -1)
        best = torch.sort(by, dim=2, descending=True, stable=True).values[:, :, :2].sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        out = torch.ones(T, c["groups"], dtype=torch.bool, device=l.device).scatter(1, kept, False)
        choice = by.masked_fill(out[:, :, None], -math.inf).reshape(T, n)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    w = s.gather(1, ids)
    return ids.int(), (w / w.sum(dim=1, keepdim=True)).float()


def _gelu(z):
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def _by_expert(ids, rows, n):
    """The places sorted by expert, each expert's padded to the longest share: (place [n, most], used [n, most])."""
    flat = ids.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    count = torch.bincount(flat, minlength=n)
    most = int(count.max())
    at = torch.arange(most, device=ids.device)
    used = at[None, :] < count[:, None]
    place = (torch.cumsum(count, 0) - count)[:, None] + at[None, :]
    return order[place.clamp(max=rows - 1)], used


def _products(W, x, ids, n, of_token):
    """x (a row per token, or per place) times the matrices of its experts: [places, rows of W], fp32."""
    P = ids.numel()
    if P <= n:                                   # few tokens: their experts' matrices
        xs = x[torch.arange(P, device=x.device) // ids.shape[1]] if of_token else x
        return torch.bmm(W[ids.reshape(-1).long()].float(), xs.float()[:, :, None])[:, :, 0]
    place, used = _by_expert(ids, P, n)
    xs = x.float()[place // ids.shape[1] if of_token else place]              # [n, most, K]
    out = torch.bmm(xs, W.float().transpose(1, 2))
    return torch.empty(P, W.shape[1], device=x.device).index_copy_(0, place[used], out[used])


def _glu(st):
    ids, W = st["ids"], st["W"]
    F = W.shape[1] // 2
    p = _products(W, st["x"], ids, W.shape[0], True)
    return (_gelu(p[:, :F]) * p[:, F:]).to(W.dtype).reshape(*ids.shape, F)


def _sum(st):
    ids, W = st["ids"], st["W"]
    p = _products(W, st["h"].reshape(ids.numel(), -1), ids, W.shape[0], False)
    st["y"] += st["ls"] * (st["w"][:, :, None] * p.reshape(*ids.shape, -1)).sum(dim=1)
    return st["y"]


def _unit(x, eps):
    return x / torch.sqrt((x * x).sum(dim=-1, keepdim=True) + eps)


def _inverse(A):
    """(I + A)^-1 of strictly lower triangular A [..., C, C], C a power of two: blocks of 1, 2, 4 .. rows at a time."""
    C = A.shape[-1]
    X = torch.eye(C, device=A.device).expand_as(A).clone()
    b = 1
    while b < C:
        at = torch.arange(0, C, 2 * b, device=A.device)
        i = at[:, None] + torch.arange(b, device=A.device)                    # rows of the first half of each pair
        lo = i + b
        first, second = X[..., i[:, :, None], i[:, None, :]], X[..., lo[:, :, None], lo[:, None, :]]
        X[..., lo[:, :, None], i[:, None, :]] = -(second @ A[..., lo[:, :, None], i[:, None, :]] @ first)
        b *= 2
    return X


def _split(rows, H, G, d, dv):
    v, k, q = rows.split([H * dv, G * d, G * d], dim=-1)
    per = H // G
    return (q.reshape(*q.shape[:-1], G, d).repeat_interleave(per, dim=-2), k.reshape(*k.shape[:-1], G, d).repeat_interleave(per, dim=-2),
            v.reshape(*v.shape[:-1], H, dv))


def _delta(st):
    """Chunks of up to 64 tokens of all sequences at once, in 32 bits."""
    c, lengths = st["case"], st["lengths"]
    H, G, d, dv = c["heads"], c["key_heads"], c["dim"], c["vdim"]
    B, longest = len(lengths), max(lengths)
    C = min(64, 1 << max(longest - 1, 0).bit_length())
    N = -(-longest // C)
    start = torch.tensor([sum(lengths[:i]) for i in range(B)], device="cuda")
    at = start[:, None] + torch.arange(N * C, device="cuda")
    used = torch.arange(N * C, device="cuda") < torch.tensor(lengths, device="cuda")[:, None]
    at = torch.where(used, at, 0)

    def chunks(x):                               # [B, H, N, C, ...]
        x = torch.where(used.reshape(B, N * C, *[1] * (x.dim() - 1)), x[at], 0)
        return x.reshape(B, N, C, *x.shape[2:]).movedim(3, 1)
    q, k, v = _split(st["rows"].float(), H, G, d, dv)
    q, k = st["q_scale"] * _unit(q, st["eps"]), _unit(k, st["eps"])
    q, k, v, beta, la = chunks(q), chunks(k), chunks(v), chunks(st["beta"]), chunks(st["la"])
    cum = torch.cumsum(la.double(), dim=-1)
    low = torch.ones(C, C, dtype=torch.bool, device="cuda").tril()
    decay = torch.where(low, torch.exp(torch.where(low, cum[..., :, None] - cum[..., None, :], 0.0)), 0.0).float()
    A = (beta[..., None] * (k @ k.transpose(-1, -2)) * decay).tril(-1)
    Tm = _inverse(A) * beta[..., None, :]
    P = (q @ k.transpose(-1, -2)) * decay
    grow, left = torch.exp(cum).float()[..., None], torch.exp(cum[..., -1:] - cum).float()[..., None]
    S = torch.stack(st["S"])                     # [B, H, dv, d]
    o = torch.empty(B, H, N, C, dv, device="cuda")
    for n in range(N):
        St = S.transpose(-1, -2)
        U = Tm[:, :, n] @ (v[:, :, n] - grow[:, :, n] * (k[:, :, n] @ St))
        o[:, :, n] = grow[:, :, n] * (q[:, :, n] @ St) + P[:, :, n] @ U
        S = grow[:, :, n, -1:] * S + U.transpose(-1, -2) @ (left[:, :, n] * k[:, :, n])
    for s, new in zip(st["S"], S):
        s.copy_(new)
    o = o.movedim(1, 3).reshape(B, N * C, H, dv)
    return torch.cat([o[b, :n] for b, n in enumerate(lengths)]), st["S"]


def _step(st):
    c, ring = st["case"], st["ring"]
    H, G, d, dv, taps = c["heads"], c["key_heads"], c["dim"], c["vdim"], c["taps"]
    ring[st["pos"] % taps] = st["row"]
    at = torch.tensor([(st["pos"] + 1 + i) % taps for i in range(taps)], device="cuda")      # oldest first
    x = (st["conv"] * ring[at].float()).sum(dim=0) + st["conv_b"]
    st["pos"] += 1
    q, k, v = _split(x * (1 / (1 + torch.exp(-x))), H, G, d, dv)
    q, k = st["q_scale"] * _unit(q, st["eps"]), _unit(k, st["eps"])
    z = st["dt"] + st["dt_bias"]
    a = torch.exp(st["A"] * (z.clamp(min=0) + torch.log1p(torch.exp(-z.abs()))))
    S = st["S"][0]
    S *= a[:, None, None]
    u = st["beta"][:, None] * (v - (S @ k[:, :, None])[:, :, 0])
    S += u[:, :, None] * k[:, None, :]
    return (S @ q[:, :, None])[:, :, 0], S, ring


# --------------------------------------------------------------------------- one pass

def run(st):
    c, kind = st["case"], st["case"]["kind"]
    if not own:
        return {"route": _route, "glu": _glu, "sum": _sum, "step": _step, "delta": _delta}[kind](st)
    op = st["op"]
    if kind == "route":
        T, top = c["tokens"], c["top"]
        ids, w = torch.empty(T, top, dtype=torch.int32, device="cuda"), torch.empty(T, top, device="cuda")
        op.rows(st["logits"].data_ptr(), c["experts"], ids.data_ptr(), w.data_ptr(), T)
        return ids, w
    if kind == "glu":
        T, top, F = c["tokens"], c["top"], c["ff"]
        h = torch.empty(T, top, F, dtype=st["x"].dtype, device="cuda")
        op.hidden(st["x"].data_ptr(), c["width"], op.plan(st["ids"], T), h.data_ptr(), F)
        return h
    if kind == "sum":
        op.add_sum(st["h"].data_ptr(), c["ff"], op.plan(st["ids"], c["tokens"]), st["w"].data_ptr(), st["y"].data_ptr(), c["width"],
                   ls=st["ls"].data_ptr())
        return st["y"]
    H, dv = c["heads"], c["vdim"]
    if kind == "step":
        op.step(st["row"].data_ptr(), st["dt"].data_ptr(), st["beta"].data_ptr(), st["ring"].data_ptr(), st["S"][0].data_ptr(),
                st["o"].data_ptr(), st["len"].data_ptr(), st["ticket"].data_ptr())
        return st["o"], st["S"][0], st["ring"]
    rows = st["rows"]
    T, C = rows.shape
    o = torch.empty(T, H, dv, device="cuda")
    v, es = rows.data_ptr(), rows.element_size()
    k = v + H * dv * es
    op.rows(k + c["key_heads"] * c["dim"] * es, k, v, C, st["la"].data_ptr(), st["beta"].data_ptr(), H, o.data_ptr(), H * dv,
            [s.data_ptr() for s in st["S"]], st["lengths"])
    return o, st["S"]


def work(case):
    """Each input read once, each output written once; of the matrices those that a balanced choice hits."""
    c = case
    if c["kind"] == "route":
        return {"bytes": 4 * c["tokens"] * c["experts"] + 8 * c["tokens"] * c["top"], "flops": 10 * c["tokens"] * c["experts"]}
    es = 2 if c["dtype"] == "bfloat16" else 4
    if c["kind"] in ("glu", "sum"):
        T, n, top, E, F = c["tokens"], c["experts"], c["top"], c["width"], c["ff"]
        hit = n * (1 - (1 - top / n) ** T)
        if c["kind"] == "glu":
            return {"bytes": hit * 2 * F * E * es + T * E * es + T * top * (F * es + 4), "flops": 4 * T * top * F * E}
        return {"bytes": hit * F * E * es + T * top * (F * es + 8) + 8 * T * E + 4 * E, "flops": 2 * T * top * F * E}
    H, G, d, dv = c["heads"], c["key_heads"], c["dim"], c["vdim"]
    C = H * dv + 2 * G * d
    if c["kind"] == "step":
        return {"bytes": 8 * H * d * dv + (c["taps"] + 1) * C * (es + 4) + 4 * H * dv, "flops": 7 * H * d * dv + 2 * c["taps"] * C}
    lengths = [int(x) for x in c["lengths"].split(",")]
    T = sum(lengths)
    return {"bytes": T * (C * es + 8 * H + 4 * H * dv) + 8 * H * d * dv * len(lengths), "flops": 7 * T * H * d * dv}


# --------------------------------------------------------------------------- 64 bits, from the definitions

def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["kind"] == "route":
        return _exact_route(st)
    if c["kind"] in ("glu", "sum"):
        return _exact_experts(st)
    H, G, d, dv = c["heads"], c["key_heads"], c["dim"], c["vdim"]
    per = H // G
    if c["kind"] == "step":
        pos, taps, ring = st["pos"], c["taps"], st["ring"].to(F64)
        ring[pos % taps] = st["row"].to(F64)
        x = st["conv_b"].to(F64)
        for i in range(taps):                     # tap i sees the input of taps - 1 - i positions ago
            x = x + st["conv"][i].to(F64) * ring[(pos - (taps - 1 - i)) % taps]
        x = x / (1 + torch.exp(-x))
        la = (st["A"].to(F64) * torch.log(1 + torch.exp(st["dt"].to(F64) + st["dt_bias"].to(F64))))[None]
        rows, beta, lengths, o_shape = x[None], st["beta"].to(F64)[None], [1], (H, dv)
    else:
        rows, beta, la, lengths, o_shape = st["rows"].to(F64), st["beta"].to(F64), st["la"].to(F64), st["lengths"], (-1, H, dv)
    v = rows[:, :H * dv].reshape(-1, H, dv)
    k = rows[:, H * dv:H * dv + G * d].reshape(-1, G, 1, d).expand(-1, G, per, d).reshape(-1, H, d)
    q = rows[:, H * dv + G * d:].reshape(-1, G, 1, d).expand(-1, G, per, d).reshape(-1, H, d)
    k = k * (k.square().sum(-1) + st["eps"]).rsqrt()[..., None]
    q = q * (q.square().sum(-1) + st["eps"]).rsqrt()[..., None] * st["q_scale"]
    o, states, t = torch.empty_like(v), [], 0
    decay = torch.exp(la)
    for S, n in zip(st["S"], lengths):
        S = S.to(F64)
        for t in range(t, t + n):
            S = S * decay[t, :, None, None]
            u = beta[t, :, None] * (v[t] - torch.einsum("hvd,hd->hv", S, k[t]))
            S = S + torch.einsum("hv,hd->hvd", u, k[t])
            o[t] = torch.einsum("hvd,hd->hv", S, q[t])
        t = t + 1
        states.append(S)
    o = o.reshape(o_shape)
    return (o, states[0], None) if c["kind"] == "step" else (o, states)


def _exact_route(st):
    c, l = st["case"], st["logits"].to(F64)
    s = torch.softmax(l, dim=1) if c["score"] == "softmax" else torch.sigmoid(l)
    choice = s.clone() if st["bias"] is None else s + st["bias"].to(F64)
    if c["groups"] > 1:
        size = c["experts"] // c["groups"]
        best = torch.stack([torch.topk(choice[:, g * size:(g + 1) * size], min(2, size), dim=1).values.sum(1) for g in range(c["groups"])], 1)
        order = torch.argsort(-best, dim=1, stable=True)
        for r in range(c["top_groups"], c["groups"]):
            drop = order[:, r:r + 1] * size + torch.arange(size, device="cuda")
            choice.scatter_(1, drop, -math.inf)
    w = []
    for _ in range(c["top"]):
        i = choice.argmax(dim=1, keepdim=True)
        w.append(s.gather(1, i))
        choice.scatter_(1, i, -math.inf)
    w = torch.cat(w, dim=1)
    return None, w / w.sum(dim=1, keepdim=True)


def _exact_experts(st):
    c, ids, W = st["case"], st["ids"], st["W"]
    glu = c["kind"] == "glu"
    out = torch.zeros(ids.numel(), W.shape[1], dtype=F64, device="cuda")
    for e in range(c["experts"]):
        at = (ids.reshape(-1) == e).nonzero()[:, 0]
        x = st["x"][at // c["top"]] if glu else st["h"].reshape(ids.numel(), -1)[at]
        out[at] = x.to(F64) @ W[e].to(F64).T
    if glu:
        gate, up = out[:, :c["ff"]], out[:, c["ff"]:]
        h = torch.nn.functional.gelu(gate, approximate="tanh") * up
        return h.reshape(c["tokens"], c["top"], c["ff"])
    y = (out.reshape(c["tokens"], c["top"], -1) * st["w"].to(F64)[:, :, None]).sum(dim=1)
    return st["y"].to(F64) + st["ls"].to(F64) * y

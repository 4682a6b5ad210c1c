"""Small random models with delta-rule mixers and feed-forwards of experts, for the tests, in both designs."""
import torch

from tests import layered_util as U
from tests import pakalix_util as K


def delta(heads=4, key_heads=2, dim=24, vdim=40, conv=4):
    return {"heads": heads, "key_heads": key_heads, "dim": dim, "vdim": vdim, "conv": conv}


def experts(n=8, top=2, ff=40, limit=0.9, **kw):
    return {"kind": "experts", "experts": n, "top": top, "ff": ff, "limit": limit, **kw}


BALANCED = dict(score="sigmoid", bias=True, groups=4, top_groups=2, scale=1.5)


def layers(design, all_experts=False):
    """A delta-rule layer with experts, one of the design's own with experts, a delta-rule layer with a dense feed-forward, one without."""
    top = (lambda n, t: n) if all_experts else (lambda n, t: t)
    own = U.layer("gla", U.gla()) if design is U else K.layer("mamba2", K.mamba2())
    out = [design.layer("gated_delta", delta()), own, design.layer("gated_delta", delta(3, 3, 16, 24, 3)), design.layer("gated_delta", delta(2, 1, 40, 8, 2), None)]
    out[0]["mlp"] = experts(8, top(8, 2), 40, shared_ff=24)
    extra = dict(BALANCED, groups=1, top_groups=1) if all_experts else BALANCED
    out[1]["mlp"] = experts(16, top(16, 3), 24, **extra)
    return out


def config(design, ly=None, **kw):
    if design is U:
        kw.setdefault("loop", {"start": 0, "stop": 2, "times": 2})
    return design.config(layers=layers(design) if ly is None else ly, **kw)


def random_tensors(design, cfg, seed=0):
    """The design's tensors, with those of the layers that it does not know in their place."""
    g = torch.Generator().manual_seed(seed + 1000)

    def lin(*shape, s=1.0):
        return (torch.randn(*shape, generator=g) * (s / shape[-1] ** 0.5)).bfloat16()

    def vec(n, mean=1.0, s=0.2):
        return (mean + s * torch.randn(n, generator=g)).bfloat16()
    known = "gla" if design is U else "mamba2"
    stand_in = U.gla() if design is U else K.mamba2()
    plain = dict(cfg, layers=[dict(ly, type=known if ly["type"] == "gated_delta" else ly["type"],
                                   mixer=stand_in if ly["type"] == "gated_delta" else ly["mixer"]) for ly in cfg["layers"]])
    t = design.random_tensors(plain, seed)
    E = cfg["width"]
    for i, ly in enumerate(cfg["layers"]):
        m, p = ly["mixer"], f"l{i}.mix."
        if ly["type"] == "gated_delta":
            for name in [n for n in t if n.startswith(p)]:
                del t[name]
            H, nv, nk = m["heads"], m["heads"] * m["vdim"], m["key_heads"] * m["dim"]
            t[p + "in"] = torch.cat([lin(2 * nv, E), lin(2 * nk, E), lin(H, E), lin(H, E, s=1.5)])
            t[p + "conv"], t[p + "conv.b"] = lin(nv + 2 * nk, m["conv"], s=1.5), vec(nv + 2 * nk, 0.0, 0.3)
            t[p + "dt_bias"], t[p + "A_log"], t[p + "norm"], t[p + "o"] = vec(H, -1.0, 1.0), vec(H, -1.0, 1.5), vec(m["vdim"]), lin(E, nv)
        ff = ly["mlp"]
        if ff is not None and ff["kind"] == "experts":
            p, n, F = f"l{i}.mlp.", ff["experts"], ff["ff"]
            t[p + "router"] = lin(n, E, s=2.0)
            if ff.get("bias"):
                t[p + "router.bias"] = vec(n, 0.0, 0.2)
            t[p + "gate"], t[p + "up"], t[p + "down"] = lin(n, F, E), lin(n, F, E), lin(n, E, F, s=2.0)
            if ff.get("shared_ff"):
                t[p + "shared.gate"], t[p + "shared.up"], t[p + "shared.down"] = lin(ff["shared_ff"], E), lin(ff["shared_ff"], E), lin(E, ff["shared_ff"])
    return t

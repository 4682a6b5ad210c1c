"""GPU: whole models with delta-rule mixers and feed-forwards of experts through the engine (prompt pass, token step, captured step,
sequences of a batch, generate), in both designs, against the plain restatements.

In bf16 a score may round to the other side of a close decision, and another expert is another output: there every expert of a layer
is chosen, so that what is compared is the arithmetic.  fp32 models choose."""
import json
import os

import numpy as np
import pytest
import torch

from llamatov_b200 import _lib, archs, dense_ops, dev_residency as dr, layered, llamatov_run as R, prefill as pf
from llamatov_b200.sequences import Sequences
from tests import layered_util as U
from tests import pakalix_util as K
from tests import sparse_util as X
from tests.test_gpu_layered import DTYPES, TOL, _portions, _tokens

pytestmark = pytest.mark.gpu
DESIGNS = {"Nugusun": U, "Pakalix": K}


@pytest.fixture(autouse=True)
def _clean():
    dr.reset_engine_state(); dr.apply_production_profile()
    yield
    assert _lib.device_status() == set()


def _model(name, dtype, seed=11, **kw):
    D = DESIGNS[name]
    cfg = X.config(D, X.layers(D, all_experts=dtype == "bfloat16"), **kw)
    t = X.random_tensors(D, cfg, seed)
    return D, cfg, t, U.product(cfg, t, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_models_whole_and_in_portions(name, dtype):
    D, cfg, t, (c, w) = _model(name, dtype)
    toks = _tokens(cfg, 300)
    want = D.oracle_logits(cfg, t, toks)
    S = Sequences(w, c, 320)
    for i, sizes in enumerate(([300], [1], [2], [97, 1], [5, 64, 1, 1, 2, 66, 3], [40, 41])):
        n = 60 if sizes[0] < 3 else 300
        got = _portions(S, i, toks[:n], sizes)
        assert U.rel_rms(got, want[:n]) < TOL[dtype], sizes
        S.end(i)


@pytest.mark.parametrize("form", ["few", "group"])
@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_layer_by_layer_against_the_oracle(name, form, monkeypatch):
    monkeypatch.setattr(dense_ops, "GROUP_FROM", 1 if form == "group" else 10 ** 9)
    from oracle import layered as L, pakalix as O
    for dtype in DTYPES:
        D, cfg, t, (c, w) = _model(name, dtype, 12)
        toks = _tokens(cfg, 70, 3)
        m = (L if D is U else O).Model(cfg, U.as_numpy(t)); m.run(toks)
        seen = []

        def tap(run, x):
            seen.append(run.slot)
            assert U.rel_rms(x.cpu().numpy(), m.taps[run.slot]) < TOL[dtype], run
        pf.prefill_resident(w, c, torch.tensor(toks), [None] * archs.of(c).n_slots(c), want_rows=[], tap=tap)
        assert seen == list(range(len(m.taps)))


@pytest.mark.parametrize("block", [layered.SequentialBlock, layered.ParallelBlock])
@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_both_blocks(monkeypatch, block, name):
    """Prompt pass and token steps agree (fp32) under both kinds of block."""
    monkeypatch.setattr(type(archs.by_name(name)), "block", block)
    D, cfg, t, (c, w) = _model(name, "float32", 13)
    for i in range(len(cfg["layers"])):
        for n in ("norm2", "ls1", "ls2"):
            w.setdefault(f"l{i}.{n}", torch.ones(cfg["width"]).bfloat16())
    c["residual_mult"] = 0.5
    S = Sequences(w, c, 100)
    toks = _tokens(cfg, 90, 4)
    a = S.step("a", toks, range(90)).numpy()
    assert np.isfinite(a).all() and U.rel_rms(_portions(S, "b", toks, [3, 1]), a) < 1e-4


@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_chunks_and_token_order_agree(name, monkeypatch):
    D, cfg, t, (c, w) = _model(name, "bfloat16", 14)
    toks = _tokens(cfg, 300)
    S = Sequences(w, c, 320)
    out = []
    for i, n in enumerate((1, 10 ** 9)):
        monkeypatch.setattr(dense_ops, "DELTA_CHUNKED_FROM", n)
        out.append(S.step(i, toks, range(300)).numpy())
    assert U.rel_rms(*out) < TOL["bfloat16"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_captured_step_equals_eager_step(name, dtype):
    D, cfg, t, (c, w) = _model(name, dtype, 15)
    toks = _tokens(cfg, 30)
    A = archs.of(c)
    A.ensure_buffers(w, c)
    kv = [None] * A.n_slots(c)
    eager = [dr.forward_pass_resident(w, c, torch.tensor([x]), torch.tensor([p]), kv).reshape(-1).numpy().copy() for p, x in enumerate(toks)]
    S = Sequences(w, c, 64)
    for p, x in enumerate(toks):
        for who in "ab":                 # two graphs of one model, replayed in turn
            assert np.array_equal(S.step(who, [x], [0]).numpy()[0], eager[p]), p
    assert S.live["a"].runner.captured


@pytest.mark.parametrize("form", ["few", "group"])
@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_bf16_models_that_choose(name, form, monkeypatch):
    """A prompt and tokens of bf16 models with 2 of 8 and 3 of 16 experts.  A choice may hang on a rounding of the scores, so the oracle is
    given the experts that the model chose; their weights are its own."""
    from llamatov_b200 import mixers
    from oracle import layered as L, pakalix as O, sparse
    monkeypatch.setattr(dense_ops, "GROUP_FROM", 1 if form == "group" else 10 ** 9)
    D = DESIGNS[name]
    cfg = X.config(D)
    t = X.random_tensors(D, cfg, 17)
    c, w = U.product(cfg, t, "bfloat16")
    chosen = []
    plan, step = dense_ops.Experts.plan, mixers.ExpertsFeedForward.step

    def seen_plan(self, ids, T):
        chosen.append(ids.clone())
        return plan(self, ids, T)

    def seen_step(self, pk, *a):
        step(self, pk, *a)
        chosen.append(pk.step.ids[:self.top].clone()[None])
    monkeypatch.setattr(dense_ops.Experts, "plan", seen_plan)
    monkeypatch.setattr(mixers.ExpertsFeedForward, "step", seen_step)
    route, own = sparse.route, []

    def given(l, m, bias):
        ids = next(fed)
        own.append(set(ids) == set(route(l, m, bias)[0]))
        s = sparse._sigmoid(l) if m.get("score") == "sigmoid" else np.exp(l - l.max()) / np.exp(l - l.max()).sum()
        return ids, s[ids] / s[ids].sum() * m.get("scale", 1.0)
    monkeypatch.setattr(sparse, "route", given)
    A = archs.of(c)
    A.ensure_buffers(w, c)
    toks, kv = _tokens(cfg, 100, 5), [None] * A.n_slots(c)
    m = (L if D is U else O).Model(cfg, U.as_numpy(t))
    for n, part in [(90, toks[:90])] + [(1, [x]) for x in toks[90:]]:
        chosen.clear()
        if n > 1:
            got = pf.prefill_resident(w, c, torch.tensor(part), kv, want_rows=list(range(n))).numpy().reshape(n, -1)
        else:
            got = dr.forward_pass_resident(w, c, torch.tensor(part), torch.tensor([m.pos]), kv).reshape(1, -1).numpy()
        fed = iter([row for ids in chosen for row in ids.tolist()])
        assert U.rel_rms(got, m.run(part)) < TOL["bfloat16"], n
        assert next(fed, None) is None
    assert np.mean(own) > 0.8                    # nearly all of them are the oracle's own


@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_sequences_in_one_prompt_pass(name):
    """More sequences than one launch of the delta rule takes, continued, then emptied and used again."""
    D, cfg, t, (c, w) = _model(name, "float32", 16)
    A = archs.of(c)
    q = [_tokens(cfg, 60, i) for i in range(11)]
    kvs = [[None] * A.n_slots(c) for _ in q]
    a = pf.prefill_resident(w, c, torch.tensor([x[:37] for x in q]), kvs, want_rows=list(range(37 * 11))).numpy().reshape(11, 37, -1)
    b = pf.prefill_resident(w, c, torch.tensor([x[37:] for x in q]), kvs, want_rows=list(range(23 * 11))).numpy().reshape(11, 23, -1)
    for i in (0, 7, 8, 10):
        assert U.rel_rms(np.concatenate([a[i], b[i]]), D.oracle_logits(cfg, t, q[i])) < TOL["float32"], i
    for kv in kvs[3]:
        kv.reset()
    again = pf.prefill_resident(w, c, torch.tensor([q[3][:37]]), [kvs[3]], want_rows=list(range(37))).numpy()
    assert U.rel_rms(again, a[3]) < 1e-5


@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_generate_from_a_folder(tmp_path, name):
    D, cfg, t, (c, w) = _model(name, "float32", 21)
    path = U.write_model(tmp_path / "m", cfg, t)
    prompt = _tokens(cfg, 20, 9)
    got = R.generate(path, prompt, 12, verbose=False, dtype="float32")
    lg = D.oracle_logits(cfg, t, got[:-1])
    s = np.sort(lg[19:], axis=1)
    assert (s[:, -1] - s[:, -2]).min() > 1e-3                # the tokens are decided
    assert got == prompt + lg[19:].argmax(axis=1).tolist()
    assert len(R.generate(path, prompt, 12, verbose=False)) == 32


def test_freed_state_is_empty():
    k = dr.DeviceDeltaState(2, 8, 8, 4, 48, torch.bfloat16)
    k.state.fill_(1.0); k.ring.fill_(1.0); k.length = 5
    k.reset()
    assert k.length == 0 and not k.state.any() and not k.ring.any()
    k.free()
    assert k.state is None and k.ring is None and k.ticket is None

"""CPU side of the token-policy operators: what the C entry points and the torch wrappers refuse (checked before anything touches a device), and the
64-bit reference against finite differences and against the distribution that verified drafts have to keep."""
import ctypes as C
import math
import types

import numpy as np
import pytest
import torch

import cleanba_amd.lib as L
from cleanba_amd import tokens as TK
from tests import token_ref as R


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(L.SO_PATH):
        L.build()
    return L.load()


P = 0x10000   # an aligned address that is never followed: each of these calls ends in a refusal


def message(rc, lib):
    assert rc == -1
    return lib.cbm_last_error().decode()


TOP = dict(ctx=None, logits=P, dtype=0, rows=4, vocab=100, stride=100, k=8, tau=1.0, idx=P, val=P, lse=P, ws=P, ws_bytes=1 << 30, stream=0)
DIS = dict(ctx=None, logits=P, dtype=1, rows=4, vocab=100, stride=100, tidx=P, tval=P, k=8, tlse=None, w=None, tau=1.0, loss=P, grad=P + (1 << 20), gstride=100, stream=0)
VER = dict(ctx=None, target=P, dtype=2, batch=4, drafts=3, vocab=100, tb=400, tp=100, draft=P, db=300, dp=100, tokens=P, n=None, ua=P, us=P, tau=1.0, out=P,
           acc=P, lp=None, ws=P, ws_bytes=1 << 30, stream=0)


@pytest.mark.parametrize("change, text", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 19) + 1), "vocab"), (dict(rows=-1), "rows"),
    (dict(rows=1 << 22), "2^22"), (dict(k=0), "k 0"), (dict(k=257), "k 257"), (dict(tau=0.0), "temperature"), (dict(tau=math.nan), "temperature"),
    (dict(tau=1e5), "temperature"), (dict(stride=99), "stride"), (dict(logits=None), "logits is null"), (dict(idx=None), "idx is null"),
    (dict(val=P + 2), "values is not aligned"), (dict(logits=P + 1), "logits is not aligned"), (dict(lse=None), "lse is null"),
    (dict(rows=1, vocab=131072, ws_bytes=16), "workspace holds 16"), (dict(rows=1, vocab=131072, ws=None), "workspace is null"), ({}, "null context"),
    (dict(rows=0), "null context")])
def test_top_logits_refuses(lib, change, text):
    assert text in message(lib.cbm_top_logits(*{**TOP, **change}.values()), lib)


@pytest.mark.parametrize("change, text", [
    (dict(dtype=7), "dtype"), (dict(vocab=-5), "vocab"), (dict(k=0), "k 0"), (dict(k=300), "k 300"), (dict(tau=-1.0), "temperature"), (dict(tau=1e-5), "temperature"),
    (dict(stride=50), "row stride"), (dict(gstride=50), "gradient stride"), (dict(tidx=None), "teacher_idx is null"), (dict(tval=None), "teacher_logits is null"),
    (dict(loss=None), "loss is null"), (dict(grad=P + 2), "overlaps"), (dict(grad=P, gstride=101), "overlaps"), (dict(grad=P + 1), "dlogits is not aligned"),
    ({}, "null context"), (dict(grad=P), "null context"), (dict(grad=None, gstride=0), "null context")])
def test_distill_refuses(lib, change, text):
    assert text in message(lib.cbm_distill_loss_grad(*{**DIS, **change}.values()), lib)


@pytest.mark.parametrize("change, text", [
    (dict(dtype=9), "dtype"), (dict(batch=-1), "rows"), (dict(drafts=-1), "drafts"), (dict(drafts=129), "drafts"), (dict(tau=-0.5), "temperature"), (dict(tau=math.inf), "temperature"),
    (dict(batch=1 << 20, drafts=100), "2^22 rows"), (dict(tp=-1), "negative stride"), (dict(db=-1), "negative stride"), (dict(target=None), "target_logits is null"),
    (dict(tokens=None), "draft_tokens is null"), (dict(ua=None), "u_accept is null"), (dict(us=None), "u_sample is null"), (dict(draft=P + 1), "draft_logits is not aligned"),
    (dict(out=None), "tokens is null"), (dict(acc=None), "accepted is null"), (dict(vocab=50000, tp=50000, tb=1 << 20, ws_bytes=0), "workspace holds 0"),
    (dict(vocab=50000, tp=50000, tb=1 << 20, ws=P + 4), "workspace is not aligned"), ({}, "null context"), (dict(tau=0.0, ua=None, us=None, draft=None), "null context")])
def test_verify_refuses(lib, change, text):
    assert text in message(lib.cbm_verify_drafts(*{**VER, **change}.values()), lib)


def test_workspace_queries(lib):
    assert lib.cbm_top_logits_workspace(1, 0, 1000, 4) == 0 and lib.cbm_top_logits_workspace(1, 100000, 1000, 4) == 0
    assert lib.cbm_top_logits_workspace(1, 1, 131072, 64) > 0
    assert "k 0" in message(lib.cbm_top_logits_workspace(1, 1, 1000, 0), lib) and "vocab" in message(lib.cbm_top_logits_workspace(1, 1, 0, 4), lib)
    assert lib.cbm_verify_drafts_workspace(1, 64, 8, 131072, 1, 1.0) >= lib.cbm_verify_drafts_workspace(1, 64, 8, 131072, 0, 1.0) > 0
    assert "drafts" in message(lib.cbm_verify_drafts_workspace(1, 64, 1000, 131072, 1, 1.0), lib)
    assert L.LEARNER_STREAM == C.c_void_p(-1).value


def test_wrappers_check_shapes_and_types():
    ctx = types.SimpleNamespace(cfg=types.SimpleNamespace(device=0))
    z = torch.zeros(3, 10)
    for bad, text in ((torch.zeros(3, 10, dtype=torch.float64), "float32"), (torch.tensor(1.0), "dimensions"), (torch.zeros(10, 3).t(), "dense"), (z, "context's device")):
        with pytest.raises(ValueError, match=text):
            TK.top_logits(ctx, bad, 2)
    with pytest.raises(ValueError, match="dimensions"):
        TK.verify_drafts(ctx, z, None, None, None)
    here = types.SimpleNamespace(cfg=types.SimpleNamespace(device=None))
    cpu = pytest.MonkeyPatch()
    cpu.setattr(TK, "_placed", lambda *a: None)   # shapes and types alone
    try:
        for kw, text in ((dict(teacher_idx=torch.zeros(3, 2, dtype=torch.int64)), "teacher_idx"), (dict(teacher_idx=torch.zeros(3, dtype=torch.int32)), "teacher_idx"),
                         (dict(teacher_logits=torch.zeros(3, 3)), "teacher_logits"), (dict(teacher_lse=torch.zeros(2)), "teacher_lse"),
                         (dict(row_weight=torch.zeros(3, dtype=torch.float64)), "row_weight")):
            with pytest.raises(ValueError, match=text):
                TK.distill_loss_grad(here, z, **{**dict(teacher_idx=torch.zeros(3, 2, dtype=torch.int32), teacher_logits=torch.zeros(3, 2)), **kw})
        t, ua, us = torch.zeros(2, 4, 10), torch.zeros(2, 3), torch.zeros(2)
        x = torch.zeros(2, 3, dtype=torch.int32)
        for args, kw, text in (((t, x.long(), ua, us), {}, "draft_tokens"), ((t, x, ua[:, :2], us), {}, "u_accept"), ((t, x, ua, None), {}, "u_sample"), ((t, x, None, us), {}, "u_accept"),
                               ((t, x, ua, us), dict(draft_logits=t), "draft_logits"), ((t, x, ua, us), dict(draft_logits=t[:, :3].half()), "draft_logits"),
                               ((t, x, ua, us), dict(n_draft=torch.zeros(2)), "n_draft"), ((t[:, :0], x, ua, us), {}, "one position")):
            with pytest.raises(ValueError, match=text):
                TK.verify_drafts(here, *args, **kw)
        with pytest.raises(ValueError, match="do not fold"):
            TK.top_logits(here, torch.zeros(3, 4, 10).transpose(0, 1), 2)
    finally:
        cpu.undo()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_reference_gradient_against_differences(tail, tau):
    """The formula's gradient is the loss's: central differences of step h leave h^2 / 6 times a third derivative (below 4 w / tau here) and 2^-52 / h."""
    rng = np.random.default_rng(1)
    V, w, h = 12, 1.7, 1e-4
    z = rng.normal(0, 2, V)
    z[7] = -math.inf
    idx, v = np.array([3, 0, -1, 3, 11]), rng.normal(0, 2, 5)   # an empty slot, one token twice
    lse = math.log(np.exp(v[[0, 1, 3, 4]] / tau).sum() + 2.0) if tail else None
    loss, g, _, _ = R.distill(z, idx, v, lse, w, tau)
    assert loss > 0 and math.isclose(g.sum(), 0.0, abs_tol=1e-13) and g[7] == 0.0
    for j in range(V):
        if j == 7:
            continue
        d = np.zeros(V)
        d[j] = h
        num = (R.distill(z + d, idx, v, lse, w, tau)[0] - R.distill(z - d, idx, v, lse, w, tau)[0]) / (2 * h)
        assert abs(num - g[j]) < h * h * w / tau + 1e-10


@pytest.mark.parametrize("looked_up", [False, True])
def test_reference_keeps_the_target_distribution(looked_up):
    """sum_x q(x) P(first token = t | x) = p(t): over a grid of G x G midpoints of the two random numbers each of the at most V + 1 borders moves a probability
    by at most 1 / G."""
    rng = np.random.default_rng(5)
    V, G, tau = 4, 24, 0.9
    target, draft = rng.normal(0, 1.5, (2, V)), rng.normal(0, 1.5, (1, V))
    p = R._dist(target[0], tau)
    q = R._dist(draft[0], tau) if not looked_up else np.eye(V)[2]
    got = np.zeros(V)
    for x in range(V):
        if q[x] == 0.0:
            continue
        for i in range(G):
            for j in range(G):
                out, _, _, _ = R.verify(target, None if looked_up else draft, [x], 1, [(i + 0.5) / G], (j + 0.5) / G, tau)
                got[out[0]] += q[x] / G / G
    assert np.abs(got - p).max() < (V + 1) / G / 2

"""GPU tests of the token-policy operators against the 64-bit reference (tests/token_ref.py).

Tolerances.  e = 2^-24 is half a step of fp32.  A row's sum of exponentials: an argument (z - m) c takes three roundings of relative e, which reach the sum
weighted by the probabilities, sum p |log2 p| <= log2 V; exp2 itself 2 e; a thread adds 16 terms and then one partial sum a chunk of 16 elements a thread, each
with a rescaling (3 e); the join across threads is fp64 (exp2 of the rescaling: 2 e).  So the sum is off by at most
    D(V) = e (16 + 3 ceil(V / (16 * 64)) + 3 log2 V + 8)   (64: the narrowest block; rows that a wider block takes are off by less)
relatively, and a log-sum-exp by that, absolutely, and by its own rounding e |lse|.  Probabilities s_j = exp2(..) / S: D + e (3 |log2 s_j| + 4)."""
import math

import numpy as np
import pytest
import torch

import cleanba_amd.lib as L
from cleanba_amd import tokens as TK
from tests import token_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E = R.EPS32


def D(V):
    return E * (16 + 3 * math.ceil(V / 1024) + 3 * math.log2(max(V, 2)) + 8)


@pytest.fixture(scope="module")
def ctx():
    cfg = L.default_config(L.ALGO_PPO)
    cfg.local_num_envs, cfg.num_actor_slots, cfg.num_steps, cfg.num_minibatches, cfg.update_epochs = 1, 1, 8, 1, 1
    c = L.Context(cfg)
    yield c
    c.close()


def cuda(a, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def logits(rng, shape, dtype, scale=2.5, masked=0.0):
    """(numpy float64 of what the type holds, tensor)"""
    z = rng.normal(0, scale, shape)
    if masked:
        z[rng.random(shape) < masked] = -math.inf
    t = torch.as_tensor(z, dtype=torch.float32).to(DT[dtype])
    return t.double().numpy(), t.cuda()


# ------------------------------------------------------------------------------------------ top_logits
def check_top(ctx, z, t, k, tau=1.0):
    idx, val, lse = (x.cpu().numpy() for x in TK.top_logits(ctx, t, k, temperature=tau))
    V = z.shape[-1]
    zr = z.reshape(-1, V)
    idx, val, lse = idx.reshape(-1, k), val.reshape(-1, k), lse.reshape(-1)
    for r in range(zr.shape[0]):
        ri, rv, rl = R.top(zr[r], k, tau)
        np.testing.assert_array_equal(idx[r], ri)
        np.testing.assert_array_equal(val[r], rv)
        if math.isfinite(rl):
            assert abs(lse[r] - rl) <= D(V) + E * abs(rl), (r, lse[r], rl)
        else:
            assert np.array_equal([lse[r]], [rl], equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, V, k", [(1, 1, 1), (5, 2, 3), (130, 18, 4), (7, 64, 16), (3, 65, 64), (4, 1000, 16), (2, 1024, 200), (3, 1025, 16), (3, 4096, 64), (2, 4097, 65),
                                        (1, 131072, 64), (3, 100003, 128), (2, 50021, 256), (1, 524288, 256), (600, 5000, 8), (1, 300, 256)])
def test_top_logits(ctx, dtype, rows, V, k):
    rng = np.random.default_rng(V * 7 + k)
    check_top(ctx, *logits(rng, (rows, V), dtype, masked=0.1 if rows % 2 else 0.0), k, tau=1.0 if k % 2 else 2.0)


@pytest.mark.parametrize("V, k", [(500, 16), (9000, 64), (70001, 256)])
def test_top_logits_orders_and_ties(ctx, V, k):
    """Orders that defeat a threshold from the first tokens, and rows of equal values: the lowest indices win."""
    up = np.arange(V, dtype=np.float64)
    rows = [up / V, -up / V, np.zeros(V), np.where(up % 2 == 0, 0.0, -0.0), np.floor(up / 97) % 3, np.where(up >= V - k, 5.0, 1.0), np.where(up % 256 == 3, 2.0, -1.0) + up * 0]
    z = np.stack(rows).astype(np.float32)
    check_top(ctx, z.astype(np.float64), cuda(z), k)
    h = torch.as_tensor(z).bfloat16()
    check_top(ctx, h.double().numpy(), h.cuda(), k)


def test_top_logits_special_values(ctx):
    V, k = 3000, 32
    rng = np.random.default_rng(0)
    z = rng.normal(0, 1, (8, V)).astype(np.float32)
    z[0] = -math.inf                       # nothing
    z[1, 5:] = -math.inf                   # fewer than k
    z[2, 17] = math.nan                    # never taken; lse NaN
    z[3, 40] = math.inf
    z[4] = -3e38                           # masks of the type's lowest values are values
    z[5] = np.where(np.arange(V) == 9, 3e38, -3e38)
    z[6] = math.nan
    z[7, ::2] = -math.inf
    idx, val, lse = (x.cpu().numpy() for x in TK.top_logits(ctx, cuda(z), k))
    for r in (0, 1, 3, 4, 5, 7):
        ri, rv, rl = R.top(z[r], k, 1.0)
        np.testing.assert_array_equal(idx[r], ri)
        np.testing.assert_array_equal(val[r], rv)
        assert lse[r] == rl or abs(lse[r] - rl) <= D(V) + E * abs(rl)
    assert 17 not in idx[2] and (idx[2] >= 0).all() and math.isnan(lse[2])
    assert (idx[6] == -1).all() and math.isnan(lse[6])


def test_top_logits_leading_axes_strides_and_addresses(ctx):
    """[T, E, V] as the rollouts are laid out, rows inside a wider buffer, every element alignment; what lies beside the rows is not read (NaN)."""
    rng = np.random.default_rng(3)
    z, t = logits(rng, (4, 3, 77), "bf16")
    check_top(ctx, z, t, 5)
    for dtype in ("f32", "f16", "bf16"):
        for off in range(9):
            buf = torch.full((6, 1100), math.nan, dtype=DT[dtype], device="cuda")
            z, t = logits(rng, (6, 1031), dtype)
            view = buf[:, off:off + 1031]
            view.copy_(t)
            check_top(ctx, z, view, 16)


def test_top_logits_row_of_a_large_buffer(ctx):
    """Row offsets beyond 2^31 elements and 2^32 bytes."""
    V = 131072
    t = torch.zeros(20000, V, dtype=torch.bfloat16, device="cuda")
    z, last = logits(np.random.default_rng(4), (2, V), "bf16")
    t[-2:] = last
    idx, val, lse = TK.top_logits(ctx, t, 8)
    i2, v2, l2 = TK.top_logits(ctx, last, 8)
    assert torch.equal(idx[-2:], i2) and torch.equal(val[-2:], v2) and (lse[-2:] - l2).abs().max() <= 2 * D(V) + 2 * E * l2.abs().max()
    assert torch.equal(idx[0].cpu(), torch.arange(8, dtype=torch.int32))
    del t
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------ distill_loss_grad
def check_distill(ctx, z, t, dtype, idx, v, tlse, w, tau, **kw):
    loss, grad = TK.distill_loss_grad(ctx, t, cuda(idx.astype(np.int32)), cuda(v.astype(np.float32)), None if tlse is None else cuda(tlse.astype(np.float32)),
                                      None if w is None else cuda(w.astype(np.float32)), temperature=tau, **kw)
    loss, grad = loss.cpu().numpy(), None if grad is None else grad.double().cpu().numpy()
    rows, V = z.shape
    d = D(V)
    for r in range(rows):
        wr = 1.0 if w is None else float(np.float32(w[r]))
        vr = v[r].astype(np.float32).astype(np.float64)
        rl, rg, s, share = R.distill(z[r], idx[r], vr, None if tlse is None else float(np.float32(tlse[r])), wr, tau)
        if math.isfinite(rl):
            # log S and log S_T: D each, weighted by at most sum t_k + t_T (<= 1 + what fp32 slots and lse leave)
            assert abs(loss[r] - rl) <= abs(wr) * tau * tau * 3.1 * d + E * abs(rl) + 1e-37, (r, loss[r], rl)
        else:
            assert np.array_equal([loss[r]], [rl], equal_nan=True), (r, loss[r], rl)
        if grad is None:
            continue
        # s_j and t_T s_j / s_T each with their relative error; the teacher's t_k in fp64; one rounding to fp32 (2 e: coefficient, product) and one to the type
        with np.errstate(divide="ignore"):
            bits = np.where(s > 0, -np.log2(np.maximum(s, 1e-300)), 0.0)
        rel = 2 * d + E * (3 * bits + 8)
        tol = abs(wr) * tau * (s * 1.01 + share) * rel + (R.HALF[dtype] + 4 * E) * np.abs(rg) * 1.01 + R.TINY[dtype]
        bad = ~(np.abs(grad[r] - rg) <= tol)
        assert not bad.any(), (r, int(bad.argmax()), grad[r][bad][:4], rg[bad][:4], tol[bad][:4])
    return loss, grad


def teacher(rng, z, k, tau, tail):
    """Top k of a teacher that the student resembles; its log-sum-exp when the tail counts."""
    t = z * 1.1 + rng.normal(0, 0.7, z.shape)
    t[~np.isfinite(t)] = -5.0
    idx = np.argsort(-t, axis=1, kind="stable")[:, :k]
    v = np.take_along_axis(t, idx, 1)
    return idx, v, np.array([R.lse64(r, tau) for r in t]) if tail else None


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, V, k", [(1, 1, 1), (3, 2, 1), (130, 18, 4), (7, 64, 64), (5, 513, 16), (3, 2051, 256), (4, 4096, 32), (3, 16385, 64), (3, 32768, 8), (2, 65543, 100),
                                        (2, 131072, 64), (2, 150001, 33), (1, 524288, 64)])
def test_distill(ctx, dtype, rows, V, k, tail):
    rng = np.random.default_rng(V + k)
    z, t = logits(rng, (rows, V), dtype)
    tau = 1.0 if k % 2 == 0 else 2.0
    idx, v, tlse = teacher(rng, z, k, tau, tail)
    w = None if rows == 1 else np.where(np.arange(rows) % 3 == 1, 0.0, 0.25 + np.arange(rows))
    check_distill(ctx, z, t, dtype, idx, v, tlse, w, tau)
    loss, none = check_distill(ctx, z, t, dtype, idx, v, tlse, w, tau, want_grad=False)
    assert none is None


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [40, 3001, 70000])
def test_distill_slots(ctx, V, tail):
    """Empty slots, indices outside the vocabulary, a token in several slots, a slot of logit -inf, rows without a teacher."""
    rng = np.random.default_rng(V)
    z, t = logits(rng, (6, V), "f32")
    idx = rng.integers(0, V, (6, 12))
    v = rng.normal(0, 2, (6, 12))
    idx[0, 3:] = -1
    idx[1, ::2] = V + 5
    idx[1, 1] = 2 ** 31 - 1
    idx[1, 3] = -2 ** 31
    idx[2, :] = 7
    idx[3, 4:8] = idx[3, 2]
    v[3, 9] = -math.inf
    idx[4, :] = -1
    v[5, :] = -math.inf
    lse = np.array([R.lse64(np.append(r, 1.5), 1.0) for r in v]) if tail else None
    loss, grad = check_distill(ctx, z, t, "f32", idx, v, lse, None, 1.0)
    if not tail:
        assert loss[4] == 0 and loss[5] == 0 and (grad[4:] == 0).all()


@pytest.mark.parametrize("tail", [False, True])
def test_distill_masked_students(ctx, tail):
    V, k = 5000, 16
    rng = np.random.default_rng(8)
    z = rng.normal(0, 2, (8, V)).astype(np.float32)
    idx, v, lse = teacher(rng, z.astype(np.float64), k, 1.0, tail)
    z[0] = -math.inf                                        # nothing: no loss
    z[1, rng.random(V) < 0.5] = -math.inf
    z[1, idx[1]] = 1.0
    z[2, idx[2, 3]] = -math.inf                             # the student masks what the teacher wants: +inf, the gradient is the formula's
    keep = np.zeros(V, bool)
    keep[idx[3]] = True
    z[3, ~keep] = -math.inf                                 # nothing outside the slots: the class of other tokens is left out
    z[4] = np.where(keep, 3e4, -3e38)                       # masks of the lowest values
    z[4, idx[4]] = 3e4
    z[5, idx[5]] = -200.0                                   # a student who gives the teacher's tokens nothing
    z[6, idx[6]] += 300.0                                   # and one who gives everything to them
    z[7, 1] = -math.inf
    loss, grad = check_distill(ctx, z.astype(np.float64), cuda(z), "f32", idx, v, lse, None, 1.0)
    assert loss[0] == 0 and (grad[0] == 0).all() and math.isinf(loss[2]) and np.isfinite(grad[2]).all()


def test_distill_poison_and_padding(ctx):
    """A NaN spoils its own row and no other; rows of weight 0 are not read; neighbours of the rows are neither read nor written."""
    V, k, rows = 2500, 8, 6
    rng = np.random.default_rng(9)
    z, t = logits(rng, (rows, V), "bf16")
    idx, v, _ = teacher(rng, z, k, 1.0, False)
    w = np.array([1.0, 0.0, 2.0, 0.0, 1.0, 1.0])
    t[1] = math.nan
    t[4, 100] = math.nan
    loss, grad = TK.distill_loss_grad(ctx, t, cuda(idx.astype(np.int32)), cuda(v.astype(np.float32)), row_weight=cuda(w.astype(np.float32)))
    assert loss[1] == 0 and loss[3] == 0 and (grad[1] == 0).all() and (grad[3] == 0).all()
    assert math.isnan(loss[4]) and grad[4].isnan().all() and grad[[0, 2, 5]].isfinite().all() and loss[[0, 2, 5]].isfinite().all()
    for dtype in ("f32", "bf16"):
        for off in (0, 1, 3, 8):
            z, t = logits(rng, (rows, V), dtype)
            buf = torch.full((rows, V + 20), math.nan, dtype=DT[dtype], device="cuda")
            view = buf[:, off:off + V]
            view.copy_(t)
            check_distill(ctx, z, view, dtype, idx, v, None, w, 1.0, in_place=True)
            beside = torch.ones(V + 20, dtype=torch.bool, device="cuda")
            beside[off:off + V] = False
            assert buf[:, beside].isnan().all()
            view.copy_(t)
            _, g = TK.distill_loss_grad(ctx, view, cuda(idx.astype(np.int32)), cuda(v.astype(np.float32)), row_weight=cuda(w.astype(np.float32)))   # (at these addresses: the order of a row's sum goes by its alignment)
            TK.distill_loss_grad(ctx, view, cuda(idx.astype(np.int32)), cuda(v.astype(np.float32)), row_weight=cuda(w.astype(np.float32)), in_place=True)
            assert torch.equal(g, view)


def test_distill_gradient_against_differences(ctx):
    """Central differences of the operator's own loss.  Step h = 2^-5: truncation h^2 w / tau, the two losses' roundings 2 (3.1 D + e |loss|) / 2 h."""
    V, k, tau, h = 300, 12, 1.5, 2.0 ** -5
    rng = np.random.default_rng(11)
    z, t = logits(rng, (1, V), "f32")
    for tail in (False, True):
        idx, v, tlse = teacher(rng, z, k, tau, tail)
        ti, tv, tl = cuda(idx.astype(np.int32)), cuda(v.astype(np.float32)), None if tlse is None else cuda(tlse.astype(np.float32))
        loss, g = TK.distill_loss_grad(ctx, t, ti, tv, tl, temperature=tau)
        step = torch.eye(V, device="cuda") * h
        both = [TK.distill_loss_grad(ctx, t + sign * step, ti.expand(V, k), tv.expand(V, k), None if tl is None else tl.expand(V), temperature=tau, want_grad=False)[0].double() for sign in (1, -1)]
        num = (both[0] - both[1]) / (2 * h)
        tol = h * h / tau + (tau * tau * 3.1 * D(V) + E * float(loss)) / h + E * 16 / h   # (t + step rounds: e |z| / h)
        assert (num - g[0].double()).abs().max() < tol < 0.01


# ------------------------------------------------------------------------------------------ verify_drafts
def drafts_case(rng, B, K, V, dtype, tau, looked_up, ragged, scale=3.0, noise=0.4, masked=0.0):
    base = rng.normal(0, scale, (B, K + 1, V))
    if masked:
        base[rng.random((B, K + 1, V)) < masked] = -math.inf
    def held(a):
        t = torch.as_tensor(a, dtype=torch.float32).to(DT[dtype])
        return t.double().numpy(), t.cuda()
    p, tp = held(base + rng.normal(0, noise, base.shape))
    q, tq = held(base[:, :K] + rng.normal(0, noise, (B, K, V)))
    x = np.zeros((B, K), np.int32)
    for b in range(B):
        for i in range(K):
            d = R._dist(q[b, i], tau if tau > 0 else 1.0)
            x[b, i] = rng.choice(V, p=d) if d is not None else 0
    n = rng.integers(0, K + 1, B).astype(np.int32) if ragged else None
    ua, us = rng.random((B, K), dtype=np.float32), rng.random(B, dtype=np.float32)
    return p, tp, None if looked_up else q, None if looked_up else tq, x, n, ua, us


def check_verify(ctx, p, tp, q, tq, x, n, ua, us, tau):
    B, K = x.shape
    V = p.shape[2]
    got = [t.cpu().numpy() for t in TK.verify_drafts(ctx, tp, cuda(x), cuda(ua), cuda(us), draft_logits=tq, n_draft=None if n is None else cuda(n), temperature=tau)]
    for b in range(B):
        tok, a, lp, margin = R.verify(p[b], None if q is None else q[b], x[b], K if n is None else n[b], ua[b], us[b], tau)
        # decisions nearer to their border than the sums' errors are not decided by the definition: none of these inputs has one
        assert margin > 8 * D(V), (b, margin)
        assert got[1][b] == a and got[0][b].tolist() == tok, (b, got[0][b], tok, got[1][b], a)
        assert np.all(np.abs(got[2][b] - np.array(lp)) <= D(V) + 2 * E * np.abs(lp)), (b, got[2][b], lp)
    return got


@pytest.mark.parametrize("looked_up, ragged", [(False, False), (False, True), (True, True)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, K, V", [(1, 1, 1), (3, 2, 2), (120, 7, 18), (5, 128, 33), (4, 3, 1000), (120, 7, 65), (9, 4, 64), (5, 30, 300), (70, 2, 2048), (2, 3, 129), (6, 0, 5000), (3, 5, 4096), (5, 4, 4097), (2, 6, 50021), (1, 4, 131072), (1, 1, 524288)])
def test_verify_drafts(ctx, dtype, B, K, V, looked_up, ragged):
    rng = np.random.default_rng(B * 1000 + V + K)
    tau = 1.0 if B % 2 else 0.8
    check_verify(ctx, *drafts_case(rng, B, K, V, dtype, tau, looked_up, ragged, masked=0.2 if V == 1000 else 0.0), tau)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, K, V", [(1, 0, 1), (7, 3, 18), (3, 5, 5001), (2, 2, 131072), (1, 1, 524288)])
def test_verify_greedy(ctx, dtype, B, K, V):
    rng = np.random.default_rng(V)
    p, tp, _, _, x, n, ua, us = drafts_case(rng, B, K, V, dtype, 0.0, True, False)
    for b in range(B):
        for i in range(K):
            if rng.random() < 0.8:
                x[b, i] = int(np.argmax(p[b, i]))
    got = TK.verify_drafts(ctx, tp, cuda(x) if K else None, None, None, temperature=0.0)
    for b in range(B):
        tok, a, lp, _ = R.verify(p[b], None, x[b], K, None, None, 0.0)
        assert got[0][b].tolist() == tok and int(got[1][b]) == a and (got[2][b] == 0).all()


@pytest.mark.parametrize("V", [30, 9000])
def test_verify_rows_without_distribution(ctx, V):
    """Masked, poisoned and impossible rows, tokens outside the vocabulary, lengths outside [0, drafts], at every place they can stand."""
    rng = np.random.default_rng(V)
    B, K = 12, 3
    p, _, q, _, x, _, ua, us = drafts_case(rng, B, K, V, "f32", 1.0, False, False)
    p, q = p.astype(np.float32), q.astype(np.float32)
    ua[:] *= 0.5
    n = np.full(B, K, np.int32)
    p[0, 0] = -math.inf                        # the first target row holds nothing
    p[1, 1, 3] = math.nan
    p[2, 3] = -math.inf                        # the row behind the last draft
    p[2, :3] = q[2]                            # (all accepted)
    q[3, 0] = -math.inf                        # a draft row that is no distribution: rejected, drawn from p
    q[4, 1, 2] = math.nan
    q[4, 0] = p[4, 0]
    p[5, 2, 1] = math.inf
    x[6, 0] = -1
    x[7, 1] = V
    q[7, 0] = p[7, 0]
    n[8], n[9] = -4, 100
    p[10, 0, :] = -math.inf
    p[10, 0, V - 1] = 0.0                      # one token alone
    q[11] = p[11, :3]                          # p == q: accepted whatever u
    q[11, 0, :] = -math.inf
    q[11, 0, 0] = 0.0
    p[11, 0, :] = -math.inf
    p[11, 0, 1:3] = 0.0
    x[11, 0] = 0                               # drafted with certainty, impossible in the target
    for qq, tq in ((q, cuda(q)), (None, None)):
        got = [t.cpu().numpy() for t in TK.verify_drafts(ctx, cuda(p), cuda(x), cuda(ua), cuda(us), draft_logits=tq, n_draft=cuda(n))]
        for b in range(B):
            tok, a, lp, margin = R.verify(p[b].astype(np.float64), None if qq is None else qq[b].astype(np.float64), x[b], n[b], ua[b], us[b], 1.0)
            assert margin > 8 * D(V)
            assert got[0][b].tolist() == tok and got[1][b] == a, (b, got[0][b], tok)
            assert np.all(np.abs(got[2][b] - np.array(lp)) <= D(V) + 2 * E * np.abs(lp))
    g = [t.cpu().numpy() for t in TK.verify_drafts(ctx, cuda(p), cuda(x), None, None, n_draft=cuda(n), temperature=0.0)]
    for b in range(B):
        tok, a, _, _ = R.verify(p[b].astype(np.float64), None, x[b], n[b], ua[b], us[b], 0.0)
        assert g[0][b].tolist() == tok and g[1][b] == a, (b, g[0][b], tok)


@pytest.mark.parametrize("looked_up, ragged", [(False, True), (False, False), (True, True)])
@pytest.mark.parametrize("dtype, B, K, V", [("bf16", 9, 8, 131072), ("f32", 500, 4, 4097), ("f16", 1, 33, 524288)])
def test_verify_large_calls(ctx, dtype, B, K, V, looked_up, ragged):
    """More than 2^24 logits: acceptance from fp32 sums, fp64 for the rows that tokens are drawn from."""
    if looked_up and V == 4097:
        B *= 2
    rng = np.random.default_rng(B + V)
    check_verify(ctx, *drafts_case(rng, B, K, V, dtype, 0.9, looked_up, ragged), 0.9)


@pytest.mark.parametrize("looked_up", [False, True])
def test_verify_a_batch_many_times(ctx, looked_up):
    """The same sequences, some of them without a distribution somewhere, once and 40 times over (a large call): the same tokens, log-probabilities within both errors."""
    rng = np.random.default_rng(3)
    B, K, V = 10, 3, 9000
    p, _, q, _, x, _, ua, us = drafts_case(rng, B, K, V, "f32", 1.0, False, False)
    n = rng.integers(0, K + 1, B).astype(np.int32)
    n[:6] = K
    p[0, 0] = -math.inf
    p[1, 1, 3] = math.nan
    p[2, 3, 7] = math.inf
    q[3, 0] = -math.inf
    q[4, 1, 2] = math.nan
    x[5, 0] = V
    args = [cuda(a.astype(np.float32) if a.dtype == np.float64 else a) for a in (p, x, ua, us)]
    tq, tn = None if looked_up else cuda(q.astype(np.float32)), cuda(n)
    one = TK.verify_drafts(ctx, *args, draft_logits=tq, n_draft=tn)
    R_ = 40 * (2 if looked_up else 1)
    many = TK.verify_drafts(ctx, *[a.repeat(R_, *[1] * (a.dim() - 1)) for a in args], draft_logits=None if tq is None else tq.repeat(R_, 1, 1), n_draft=tn.repeat(R_))
    for k in range(2):
        assert torch.equal(one[k].repeat(R_, *[1] * (one[k].dim() - 1)), many[k])
    assert (one[2].repeat(R_, 1) - many[2]).abs().max() <= 2 * D(V) + 4 * E * one[2].abs().max()


def test_verify_extreme_random_numbers(ctx):
    """u = 0, the largest float below 1 and 1 itself (outside the range: still a token that has weight)."""
    V = 9001
    z = np.full((4, 1, V), -math.inf, np.float32)
    z[:, 0, 100:8000:7] = 0.0
    us = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0, 0.5], np.float32)
    tok, _, lp = TK.verify_drafts(ctx, cuda(z), None, None, cuda(us))
    live = np.arange(100, 8000, 7)
    assert tok[:, 0].tolist() == [100, live[-1], live[-1], live[int(0.5 * live.size)]]
    assert np.allclose(lp.cpu().numpy(), -math.log(live.size), atol=D(V) + 1e-6)


@pytest.mark.parametrize("V, times", [(30, 1), (9000, 1), (30, 40000), (9000, 120)])
def test_verify_huge_logits(ctx, V, times):
    """Rows whose largest logit is a mask's lowest value, two such levels, the largest floats: equal ones share, all others have nothing.  Once, and as a large call."""
    rng = np.random.default_rng(V)
    low = -float(torch.finfo(torch.float32).max)
    B, K = 6, 2
    p = rng.normal(0, 3, (B, K + 1, V)).astype(np.float32)
    q = rng.normal(0, 3, (B, K, V)).astype(np.float32)
    q[:] = p[:, :K] + rng.normal(0, 0.3, q.shape)
    x = rng.integers(0, V, (B, K)).astype(np.int32)
    ua, us = rng.random((B, K), dtype=np.float32) * np.float32(0.5), rng.random(B, dtype=np.float32)
    p[0] = low                                # uniform
    q[0] = low
    p[1] = low                                # a level above the lowest: it alone
    p[1, :, 5:15] = -1e30
    x[1] = 5, 20
    q[1] = p[1, :K]
    p[2] = 1e38                               # the neighbour below the largest
    p[2, :, 3:7] = np.nextafter(np.float32(1e38), np.float32(np.inf))
    x[2] = 4, 2
    p[3] = np.where(rng.random((K + 1, V)) < 0.9, low, p[3]).astype(np.float32)   # an ordinary masked row
    q[3] = low                                # drafted from a uniform row
    x[3] = p[3, :K].argmax(1)
    p[4] = np.where(np.arange(V) % 2, np.float32(2.0**37), -np.float32(2.0**37))
    x[4] = 1, 2
    p[5] = 7e10 + 8192 * (np.arange(V) % 3)    # about 2^36: neighbouring floats
    x[5] = 2, 0
    for qq in (q, None):
        want = [R.verify(p[b].astype(np.float64), None if qq is None else qq[b].astype(np.float64), x[b], K, ua[b], us[b], 1.0) for b in range(B)]
        rep = [cuda(a).repeat(times, *[1] * (a.ndim - 1)) for a in (p, x, ua, us)]
        got = [t.view(times, B, *t.shape[1:]) for t in TK.verify_drafts(ctx, *rep, draft_logits=None if qq is None else cuda(qq).repeat(times, 1, 1))]
        for b in range(B):
            tok, a, lp, margin = want[b]
            assert margin > 8 * D(V)
            assert (got[1][:, b] == a).all() and (got[0][:, b].cpu() == torch.tensor(tok)).all(), (b, got[0][0, b], tok, got[1][0, b], a)
            assert (got[2][:, b].cpu().double() - torch.tensor(lp)).abs().max() <= D(V) + 2 * E * max(map(abs, lp)), (b, got[2][0, b], lp)


@pytest.mark.parametrize("u", [0.0, 1.0])
def test_verify_chunks_of_vanishing_weight(ctx, u):
    """Tokens of probability 2^-1010 before and behind the others are not drawn, not even by u = 0 or by the 1 that is out of range."""
    V = 3 * 2048
    z = np.full((1, 1, V), -700.0, np.float32)   # exp(-700) = 2^-1010
    z[0, 0, 2100:2110] = 0.0
    tok, acc, lp = TK.verify_drafts(ctx, cuda(z), None, None, cuda(np.array([u], np.float32)))
    assert tok.tolist() == [[2100 if u == 0.0 else 2109]] and acc.tolist() == [0]
    assert abs(float(lp) + math.log(10)) <= D(V) + 1e-6


def test_verify_strides_shared_rows_and_unread_rows(ctx):
    """Logits inside a wider buffer, a target row shared by the batch (stride 0), and rows behind a sequence's drafts: not read (NaN there changes nothing)."""
    rng = np.random.default_rng(6)
    B, K, V = 5, 4, 6001
    p, tp, q, tq, x, n, ua, us = drafts_case(rng, B, K, V, "bf16", 1.0, False, True)
    wide = torch.full((B, K + 1, V + 13), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, :, 3:3 + V] = tp
    dwide = torch.full((K, B, V + 1), math.nan, dtype=torch.bfloat16, device="cuda")
    dwide[:, :, 1:] = tq.transpose(0, 1)
    for b in range(B):
        wide[b, n[b] + 1:] = math.nan
        dwide[n[b]:, b] = math.nan
    check_verify(ctx, p, wide[:, :, 3:3 + V], q, dwide[:, :, 1:].transpose(0, 1), x, n, ua, us, 1.0)
    one = tp[:1].expand(B, K + 1, V)
    check_verify(ctx, np.repeat(p[:1], B, 0), one, q, tq, x, n, ua, us, 1.0)


def test_verified_drafts_keep_the_distribution(ctx):
    """sum_x q(x) P(first token = t | x) = p(t) over a G x G grid of the two random numbers: each of the at most V + 1 borders moves a probability by at most 1 / G."""
    rng = np.random.default_rng(12)
    V, G, tau = 5, 96, 0.7
    p, q = rng.normal(0, 1.5, (2, V)).astype(np.float32), rng.normal(0, 1.5, V).astype(np.float32)
    B = V * G * G
    mid = ((np.arange(G) + 0.5) / G).astype(np.float32)
    x = np.repeat(np.arange(V, dtype=np.int32), G * G)[:, None]
    ua = np.tile(np.repeat(mid, G), V)[:, None]
    us = np.tile(np.tile(mid, G), V)
    tok, _, _ = TK.verify_drafts(ctx, cuda(p).expand(B, 2, V), cuda(x), cuda(ua), cuda(us), draft_logits=cuda(q).expand(B, 1, V), temperature=tau)
    pd, qd = R._dist(p[0], tau), R._dist(q, tau)
    first = tok[:, 0].cpu().numpy()
    got = np.bincount(first, weights=qd[x[:, 0]] / G / G, minlength=V)
    assert np.abs(got - pd).max() < (V + 1) / G / 2


# ------------------------------------------------------------------------------------------ together, streams, graphs
def step(ctx, teacher_z, student_z, draft_z, u):
    """One distillation step and one serving step, as a program would make them."""
    idx, val, lse = TK.top_logits(ctx, teacher_z, 16)
    loss, grad = TK.distill_loss_grad(ctx, student_z, idx, val, teacher_lse=lse)
    drafted = torch.cat([TK.verify_drafts(ctx, draft_z[:, i:i + 1], None, None, u[:, i].contiguous())[0] for i in range(draft_z.shape[1])], 1)
    out, accepted, logp = TK.verify_drafts(ctx, teacher_z, drafted, u[:, 3:3 + draft_z.shape[1]].contiguous(), u[:, 7].contiguous(), draft_logits=draft_z)
    return idx, val, lse, loss, grad, drafted, out, accepted, logp


def step_inputs(seed, B=6, K=3, V=7001):
    g = torch.Generator("cuda").manual_seed(seed)
    teacher_z = torch.randn(B, K + 1, V, generator=g, device="cuda") * 2
    student_z = (teacher_z + torch.randn(B, K + 1, V, generator=g, device="cuda")).bfloat16()
    return teacher_z, student_z, teacher_z[:, :K] + 0.3 * torch.randn(B, K, V, generator=g, device="cuda"), torch.rand(B, 8, generator=g, device="cuda")


def test_a_run_of_them_together(ctx):
    teacher_z, student_z, draft_z, u = step_inputs(0)
    idx, val, lse, loss, grad, drafted, out, accepted, logp = (t.cpu().numpy() for t in (x.float() if x.dtype == torch.bfloat16 else x for x in step(ctx, teacher_z, student_z, draft_z, u)))
    B, P1, V = teacher_z.shape
    tz, sz, dz, un = teacher_z.double().cpu().numpy(), student_z.double().cpu().numpy(), draft_z.double().cpu().numpy(), u.cpu().numpy()
    for b in range(B):
        for i in range(P1):
            ri, rv, rl = R.top(tz[b, i], 16, 1.0)
            np.testing.assert_array_equal(idx[b, i], ri)
            dl, dg, s, share = R.distill(sz[b, i], ri, rv.astype(np.float64), float(lse[b, i]), 1.0, 1.0)
            assert abs(loss[b, i] - dl) <= 3.1 * D(V) + E * abs(dl)
            assert np.all(np.abs(grad[b, i] - dg) <= (s + share) * 1e-4 + 2.0 ** -8 * np.abs(dg) + 1e-30)
        for i in range(dz.shape[1]):
            tok, _, _, margin = R.verify(dz[b, i:i + 1], None, [], 0, [], un[b, i], 1.0)
            assert margin > 8 * D(V) and drafted[b, i] == tok[0]
        tok, a, _, margin = R.verify(tz[b], dz[b], drafted[b], dz.shape[1], un[b, 3:6], un[b, 7], 1.0)
        assert margin > 8 * D(V) and out[b].tolist() == tok and accepted[b] == a


def test_captured_and_replayed(ctx):
    """A graph of the whole step, replayed on new inputs with eager work between: every replay equals the eager run's bits."""
    ins = step_inputs(1)
    step(ctx, *ins)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(ctx, *ins)
    for seed in (2, 3, 4):
        new = step_inputs(seed)
        eager = [t.clone() for t in step(ctx, *new)]
        for a, b in zip(ins, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("looked_up", [False, True])
@pytest.mark.parametrize("B, K, V", [(120, 7, 18), (30, 3, 700), (4, 3, 9000), (64, 3, 50001), (6, 0, 5000)])
def test_verify_captured_and_replayed(ctx, B, K, V, looked_up):
    """Each form of the verification (one, two, three kernels) in a graph, replayed on new inputs with eager calls between."""
    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = 3 * torch.randn(B, K + 1, V, generator=g, device="cuda")
        d = t[:, :K] + 0.4 * torch.randn(B, K, V, generator=g, device="cuda")
        x = torch.randint(0, V, (B, K), generator=g, device="cuda", dtype=torch.int32)
        if K and seed % 2:
            x = d.argmax(-1).int()
        return t, x, torch.rand(B, K, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda"), d, torch.randint(0, K + 1, (B,), generator=g, device="cuda", dtype=torch.int32)

    def call(t, x, ua, us, d, n):
        return TK.verify_drafts(ctx, t, x, ua, us, draft_logits=None if looked_up or not K else d, n_draft=n)
    ins = inputs(1)
    call(*ins)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call(*ins)
    for seed in (2, 3, 4, 5):
        new = inputs(seed)
        eager = call(*new)
        for a, b in zip(ins, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


def test_two_streams_at_once(ctx):
    ins = [step_inputs(10 + i) for i in range(2)]
    want = [[t.clone() for t in step(ctx, *i)] for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(ctx, *ins[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for run in got[k]:
            for a, b in zip(run, want[k]):
                assert torch.equal(a, b)


def test_c_call_on_the_learner_stream_and_empty_calls(ctx):
    """The C entry point as a torch-free host calls it, and calls of no rows."""
    rng = np.random.default_rng(2)
    z = rng.normal(0, 2, (4, 50)).astype(np.float32)
    d = L.DevBuf(ctx, z)
    outs = [L.DevBuf(ctx, np.zeros((4, 3), np.int32)), L.DevBuf(ctx, np.zeros((4, 3), np.float32)), L.DevBuf(ctx, np.zeros(4, np.float32))]
    L._chk(ctx.lib.cbm_top_logits(ctx.h, d.ptr, L.F32, 4, 50, 50, 3, 1.0, outs[0].ptr, outs[1].ptr, outs[2].ptr, None, 0, L.LEARNER_STREAM))
    ctx.sync()
    for r in range(4):
        np.testing.assert_array_equal(outs[0].download()[r], R.top(z[r], 3, 1.0)[0])
    for b in [d] + outs:
        b.free()
    idx, val, lse = TK.top_logits(ctx, torch.zeros(0, 10, device="cuda"), 3)
    assert idx.shape == (0, 3) and lse.shape == (0,)
    loss, g = TK.distill_loss_grad(ctx, torch.zeros(2, 0, 10, device="cuda"), torch.zeros(2, 0, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, 0, 3, device="cuda"))
    assert loss.shape == (2, 0) and g.shape == (2, 0, 10)
    out, a, lp = TK.verify_drafts(ctx, torch.zeros(0, 3, 10, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, 2, device="cuda"), torch.zeros(0, device="cuda"))
    assert out.shape == (0, 3)
    with pytest.raises(L.CbmError, match="k 300"):
        TK.top_logits(ctx, torch.zeros(2, 400, device="cuda"), 300)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V, k", [(4000, 10), (40000, 33), (100000, 64), (70000, 100), (90000, 256)])
def test_top_logits_overflowing_rows(ctx, dtype, V, k):
    """Rows that keep beating the bar: rising in steps (many equal values each), the largest ones all in one thread's places, all equal but for a late few."""
    up = np.arange(V)
    z = np.stack([up // 50 / 64.0, up // 3000 * 1.0, np.where(up % 2048 < 8, 1.0 + up / V, 0.0), np.where(up % 8192 < 8, up // 8192, -1.0), np.where(up > V - 3, 2.0, 1.0), (up * 7919 % V) / V, up / V])
    t = torch.as_tensor(z, dtype=torch.float32).to(DT[dtype])
    check_top(ctx, t.double().numpy(), t.cuda(), k)

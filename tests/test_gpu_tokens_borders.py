"""GPU tests of the token-policy operators where two answers lie next to each other: equal rows, borders between tokens, huge and poisoned logits.

The 64-bit reference is tests/token_ref.py.  What a draw or an acceptance goes by is held to 64 bits: a probability's exponential is off by 1.33e-12 at most
(a series to the fourth power on [-1/64, 1/64] in powers of two, an argument of up to 1000 rounded once), its row's sum by the same, so that a probability and a
border between two tokens are off by at most 2.7e-12, and a log-probability by that and by its own rounding to fp32."""
import math

import numpy as np
import pytest
import torch

from cleanba_amd import tokens as TK
from tests import token_ref as R
from tests.test_gpu_tokens import D, DT, E, check_top, ctx, cuda, teacher  # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu
P64 = 2.7e-12   # a probability, relatively; a cumulative one


def repeated(arrays, times):
    return [torch.as_tensor(a).cuda().repeat(times, *[1] * (a.ndim - 1)) for a in arrays]


def verify_many(ctx, times, p, x, ua, us, q, n=None, tau=1.0):
    """The batch `times` over (a large call goes through other kernels), one copy's answers after all have been found the same."""
    tp, tx, tua, tus = repeated((p, x, ua, us), times)
    tq = None if q is None else repeated((q,), times)[0]
    tn = None if n is None else repeated((n,), times)[0]
    out = [t.view(times, len(x), *t.shape[1:]) for t in TK.verify_drafts(ctx, tp, tx, tua, tus, draft_logits=tq, n_draft=tn, temperature=tau)]
    for t in out:
        assert torch.equal(t, t[:1].expand_as(t))
    return [t[0].cpu().numpy() for t in out]


# ------------------------------------------------------------------------------------------ rejected with nothing left of p
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("V, times", [(30, 1), (9000, 1), (9000, 130)])   # one kernel, two, three
def test_verify_draws_from_p_where_the_draft_equals_it(ctx, V, times, dtype):
    """max(p - q, 0) is 0 everywhere where the rows are equal, or equal up to a constant: the token comes from p, not from what roundings leave of p - q.
    Logits are multiples of 2^-8 below 16 (12 bits and a sign: exact in fp16 up to 8), so that the shifted rows are shifted exactly."""
    rng = np.random.default_rng(V)
    B, K, tau = 24, 2, 0.9
    p = np.clip(np.round(rng.normal(0, 2, (B, K + 1, V)) * 64) / 64, -7, 7)
    q = p[:, :K].copy()
    x = rng.integers(0, V, (B, K)).astype(np.int32)
    ua, us = rng.random((B, K), dtype=np.float32) * np.float32(0.9), rng.random(B, dtype=np.float32)
    x[0:4, 0] = -1                             # outside the vocabulary: rejected
    x[4:8, 0] = V
    x[8:12, 0] = 7                             # masked in both rows: 0 < 0 is not
    p[8:12, 0, 7] = q[8:12, 0, 7] = -math.inf
    q[12:16] += np.array([1.0, -3.0, 0.25, 7.0])[:, None, None]   # equal up to a constant
    x[12:16, 0] = -1
    x[16:20, 1] = -1                           # the second draft (the first is accepted: u q < p)
    q[20:24, 0, 5] = -math.inf                 # but one token: it alone is left
    p[20:24, 0, 5] = -7.0
    x[20:24, 0] = -1
    p, q = (a.astype(np.float32 if dtype == "f32" else np.float16) for a in (p, q))
    tok, acc, lp = verify_many(ctx, times, p, x, ua, us, q, tau=tau)
    for b in range(B):
        want, a, logs, margin = R.verify(p[b].astype(np.float64), q[b].astype(np.float64), x[b], K, ua[b], us[b], tau)
        assert margin > 1e-5, (b, margin)      # (of the draw: a million times its distance from a border)
        assert tok[b].tolist() == want and acc[b] == a, (b, tok[b], want)
        assert np.all(np.abs(lp[b] - np.array(logs)) <= D(V) + 2 * E * np.abs(logs)), (b, lp[b], logs)


# ------------------------------------------------------------------------------------------ acceptances next to their border
@pytest.mark.parametrize("looked_up", [False, True])
@pytest.mark.parametrize("V, B, K", [(9001, 420, 3), (1000, 230, 40)])
def test_verify_accepts_by_64_bits_whatever_the_batch(ctx, V, B, K, looked_up):
    """u_accept on the floats next to p / q, on either side: a sum in fp32 would decide half of these wrongly.  Once in a large call, which sums in fp32 first, and
    a few sequences at a time."""
    rng = np.random.default_rng(17)
    tau = 0.8
    p = rng.normal(0, 2, (B, K + 1, V)).astype(np.float32)
    q = (p[:, :K] + rng.normal(0, 0.4, (B, K, V))).astype(np.float32)
    x = np.zeros((B, K), np.int32)
    ua = np.zeros((B, K), np.float32)
    us = rng.random(B, dtype=np.float32)
    for b in range(B):
        for i in range(K):
            pd, qd = R._dist(p[b, i], tau), np.ones(V) if looked_up else R._dist(q[b, i], tau)
            ratio = pd / qd
            ok = np.flatnonzero((ratio < 0.95) & (ratio > (1e-6 if looked_up else 0.2)))
            while True:
                x[b, i] = rng.choice(ok)
                border = ratio[x[b, i]]
                near = np.float32(border)
                below = near if float(near) < border else np.nextafter(near, np.float32(0))
                ua[b, i] = below if (b + i) % 2 else np.nextafter(below, np.float32(2))
                if 4 * P64 < abs(float(ua[b, i]) - border) / border:
                    break
            assert abs(float(ua[b, i]) - border) / border < 1.2e-7
    want = [R.verify(p[b], None if looked_up else q[b], x[b], K, ua[b], us[b], tau) for b in range(B)]
    assert len({a for _, a, _, _ in want}) > 1
    got = verify_many(ctx, 2 if looked_up and V == 9001 else 1, p, x, ua, us, None if looked_up else q, tau=tau)
    wrong = [b for b in range(B) if got[1][b] != want[b][1] or got[0][b].tolist() != want[b][0]]
    assert not wrong, (len(wrong), wrong[:8])
    few = [verify_many(ctx, 1, *(a[i:i + 7] for a in (p, x, ua, us)), None if looked_up else q[i:i + 7], tau=tau) for i in range(0, 70, 7)]
    for k in range(2):
        assert np.array_equal(np.concatenate([f[k] for f in few]), got[k][:70])


# ------------------------------------------------------------------------------------------ log-probabilities
@pytest.mark.parametrize("V, times", [(30, 1), (9000, 1), (9000, 500)])
def test_verify_log_probabilities_of_huge_logits(ctx, V, times):
    """Equal logits of 1e7 to 4.5e10: the token's exponent z log2(e) / tau and the row's are alike, their difference is exact."""
    z = np.float32([1e7, -3e7, 1.234567e9, 7.7777e9, -2.3456e10, 3.21e10, 4.1e10, 4.4321e10])
    p = np.repeat(z[:, None], V, 1)[:, None, :]
    B = len(z)
    live = 17
    p[:, 0, live:] = -math.inf
    _, _, lp = verify_many(ctx, times, p, np.zeros((B, 0), np.int32), np.zeros((B, 0), np.float32), np.full(B, 0.5, np.float32), None)
    assert np.abs(lp[:, 0] + math.log(live)).max() <= E * math.log(live) + 1e-10, lp[:, 0] + math.log(live)


# ------------------------------------------------------------------------------------------ draws next to their border
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V, B", [(300, 96), (50021, 48), (131072, 16)])
def test_verify_draws_next_to_a_border(ctx, V, B, dtype):
    """u_sample on the floats next to a cumulative probability, on either side: sums in fp32 would move many of these tokens.  Log-probabilities to fp32's
    own rounding."""
    rng = np.random.default_rng(V + 1)
    t = torch.as_tensor(rng.normal(0, 2, (B, 1, V)), dtype=torch.float32).to(DT[dtype])
    p = t.double().numpy()
    us, want, logs = np.zeros(B, np.float32), [], []
    for b in range(B):
        d = R._dist(p[b, 0], 1.0)
        c = np.cumsum(d) / d.sum()
        while True:
            j = int(rng.choice(np.flatnonzero((d[:-1] > 3e-7) & (d[1:] > 3e-7) & (c[:-1] < 0.999))))
            near = np.float32(c[j])
            below = near if float(near) < c[j] else np.nextafter(near, np.float32(0))
            u = below if b % 2 else np.nextafter(below, np.float32(2))
            if abs(float(u) - c[j]) > 1e-11:   # (the border itself is summed here to 1e-14)
                break
        us[b] = u
        want.append(j if b % 2 else j + 1)
        logs.append(math.log(d[want[-1]]))
    tok, _, lp = (x.cpu().numpy() for x in TK.verify_drafts(ctx, t.cuda(), None, None, cuda(us)))
    assert tok[:, 0].tolist() == want
    assert np.all(np.abs(lp[:, 0] - logs) <= 1.001 * E * np.abs(logs) + 1e-10)


# ------------------------------------------------------------------------------------------ NaN and infinities
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V, k", [(18, 4), (60, 64), (1000, 16), (3000, 200), (60000, 32)])   # a token a lane, one block a row (64 and 512 threads), split rows
def test_top_logits_poisoned_rows(ctx, V, k, dtype):
    """NaN is never taken and makes the log-sum-exp NaN, +inf is taken first and makes it +inf, at any place of a row; rows beside them do not notice."""
    rng = np.random.default_rng(V)
    z = rng.normal(0, 2, (12, V))
    z[1, 0] = z[2, V - 1] = z[3, V // 2] = z[4, ::2] = math.nan
    z[5, 1] = z[6, V - 1] = math.inf
    z[7] = math.nan
    z[8] = -math.inf
    z[9, 1:] = -math.inf
    z[10, :V - 1] = math.nan
    z[11, 3], z[11, 7] = math.inf, -math.inf
    t = torch.as_tensor(z, dtype=torch.float32).to(DT[dtype])
    check_top(ctx, t.double().numpy(), t.cuda(), k)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [40, 5001, 70001])
def test_distill_poisoned_rows(ctx, V, dtype, tail):
    """A NaN or +inf in a row, at a token of the teacher or at another, makes that row's loss and gradient NaN, and no other's."""
    rng = np.random.default_rng(V)
    z = rng.normal(0, 2, (8, V))
    idx, v, lse = teacher(rng, z, 8, 1.0, tail)
    other = [next(j for j in range(V) if j not in idx[r]) for r in range(8)]
    z[1, idx[1, 2]] = z[2, other[2]] = math.nan
    z[4, idx[4, 0]] = z[6, other[6]] = math.inf
    loss, grad = TK.distill_loss_grad(ctx, torch.as_tensor(z, dtype=torch.float32).to(DT[dtype]).cuda(), cuda(idx.astype(np.int32)), cuda(v.astype(np.float32)),
                                      None if lse is None else cuda(lse.astype(np.float32)))
    for r in range(8):
        if r in (1, 2, 4, 6):
            assert loss[r].isnan() and grad[r].isnan().all(), r
        else:
            assert loss[r].isfinite() and grad[r].isfinite().all(), r


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [18, 5001, 140001])
def test_distill_in_place_equals_out_of_place(ctx, V, dtype, tail):
    """The gradient over the logits themselves, rows of masks' lowest values (read a second time) and of weight 0 among them."""
    rng = np.random.default_rng(V)
    z = rng.normal(0, 2, (6, V))
    idx, v, lse = teacher(rng, z, 4, 1.0, tail)
    z[1] = np.where(rng.random(V) < 0.7, -3e38, z[1])
    z[2] = -3e38
    z[2, idx[2]] = -1e38
    z[3] = -3e38
    z[4, 1] = -math.inf
    w = np.array([1, 2, 0.5, 1, 1, 0])
    t = torch.as_tensor(z, dtype=torch.float32).to(DT[dtype]).cuda()
    args = [cuda(idx.astype(np.int32)), cuda(v.astype(np.float32)), None if lse is None else cuda(lse.astype(np.float32)), cuda(w.astype(np.float32))]
    loss, grad = TK.distill_loss_grad(ctx, t, *args)
    assert grad.isfinite().all()
    over, same = TK.distill_loss_grad(ctx, t, *args, in_place=True)
    assert same.data_ptr() == t.data_ptr() and torch.equal(over, loss) and torch.equal(same, grad)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("V, times", [(30, 1), (300, 1), (9000, 1), (9000, 130)])
def test_verify_poisoned_rows_of_16_bits(ctx, V, times, dtype):
    """NaN and +inf in target and draft rows, and rows of nothing: rejected, drawn from p or -1."""
    rng = np.random.default_rng(V)
    B, K = 10, 3
    base = rng.normal(0, 2, (B, K + 1, V))
    p = torch.as_tensor(base, dtype=torch.float32).to(DT[dtype])
    q = p[:, :K].clone()
    x = rng.integers(0, V, (B, K)).astype(np.int32)
    ua, us = rng.random((B, K), dtype=np.float32) * np.float32(0.5), rng.random(B, dtype=np.float32)
    p[0, 0, 0] = p[1, 1, V - 1] = p[2, 3, V // 2] = math.nan
    p[3, 0, 1] = p[4, 2, V - 1] = p[5, 3, 0] = math.inf
    q[6, 0, V - 1] = math.nan
    q[7, 1, 2] = math.inf
    q[8, 2] = -math.inf
    p[9, 1] = -math.inf
    tp, tq = p.cuda().repeat(times, 1, 1), q.cuda().repeat(times, 1, 1)
    tx, tua, tus = repeated((x, ua, us), times)
    for draft in (tq, None):
        tok, acc, _ = (t.view(times, B, *t.shape[1:]).cpu().numpy() for t in TK.verify_drafts(ctx, tp, tx, tua, tus, draft_logits=draft))
        for b in range(B):
            want, a, _, margin = R.verify(p[b].double().numpy(), None if draft is None else q[b].double().numpy(), x[b], K, ua[b], us[b], 1.0)
            assert margin > 1e-5
            assert (tok[:, b] == want).all() and (acc[:, b] == a).all(), (b, tok[0, b], want)


# ------------------------------------------------------------------------------------------ rows without a teacher
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [40, 5001, 140001])
def test_distill_rows_without_a_filled_slot(ctx, V, tail):
    """Loss and gradient are 0 whatever the row holds, a NaN or +inf among it."""
    rng = np.random.default_rng(V)
    z = rng.normal(0, 2, (5, V)).astype(np.float32)
    z[1, V // 2], z[2, 0] = math.nan, math.inf
    idx = np.full((5, 6), -1, np.int32)
    idx[3] = V
    idx[4, 2] = 3                              # a row that has one
    v = rng.normal(0, 1, (5, 6)).astype(np.float32)
    loss, grad = TK.distill_loss_grad(ctx, cuda(z), cuda(idx), cuda(v), cuda(np.float32([1, 1, -math.inf, 2, 3])) if tail else None)
    assert (loss[:4] == 0).all() and (grad[:4] == 0).all() and loss[4] > 0 and (grad[4] != 0).any()

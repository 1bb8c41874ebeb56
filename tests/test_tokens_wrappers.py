"""What the torch wrappers of the token-policy operators do around the C calls, without a GPU: the calls are recorded."""
import types

import pytest
import torch

from cleanba_amd import tokens as TK

HUGE = 2 ** 32 + 5   # 5 in the 32 bits that a C call takes


@pytest.fixture
def ctx(monkeypatch):
    """A context whose C calls do nothing but succeed, on tensors in host memory."""
    monkeypatch.setattr(TK, "_placed", lambda *a: None)
    monkeypatch.setattr(TK, "_raw_stream", lambda index: 0)
    calls = []

    def record(name):
        def call(*args):
            calls.append((name,) + args)
            return 0
        return call
    lib = types.SimpleNamespace(**{n: record(n) for n in ("cbm_top_logits", "cbm_distill_loss_grad", "cbm_verify_drafts")})
    return types.SimpleNamespace(cfg=types.SimpleNamespace(device=0), lib=lib, h=None, calls=calls)


def test_sizes_beyond_32_bits_are_refused(ctx):
    """They would be cut: of 2^32 + 5 tokens the first 5 would be looked at, of as many rows 5 answered."""
    one = torch.zeros(1, 1)
    rows, wide = one.expand(HUGE, 1), one.expand(1, HUGE)
    idx, val = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1)
    for call in (lambda: TK.top_logits(ctx, rows, 1), lambda: TK.top_logits(ctx, wide, 1), lambda: TK.top_logits(ctx, one, HUGE), lambda: TK.top_logits(ctx, one, -HUGE),
                 lambda: TK.distill_loss_grad(ctx, rows, idx, val), lambda: TK.distill_loss_grad(ctx, wide, idx, val),
                 lambda: TK.distill_loss_grad(ctx, one, idx.expand(1, HUGE), val.expand(1, HUGE)),
                 lambda: TK.verify_drafts(ctx, rows[:, None], None, None, torch.zeros(1)), lambda: TK.verify_drafts(ctx, wide[:, None], None, None, torch.zeros(1)),
                 lambda: TK.verify_drafts(ctx, one[None].expand(1, HUGE, 1), None, None, torch.zeros(1))):
        with pytest.raises(ValueError, match="more than any call takes"):
            call()
    assert not ctx.calls


def test_in_place_is_seen_by_autograd(ctx):
    """A backward that saved the logits must not take the gradient for them."""
    idx, val = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    w = torch.ones(3, 5, requires_grad=True)
    z = w.exp()                                # saves its result
    TK.distill_loss_grad(ctx, z, idx, val)
    z.sum().backward(retain_graph=True)        # out of place: nothing has changed
    _, grad = TK.distill_loss_grad(ctx, z, idx, val, in_place=True)
    assert grad is z
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()

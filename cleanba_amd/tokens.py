"""Operators of token policies on torch tensors: the teacher's top logits, distillation with its gradient, verification of drafted tokens.

The same C ABI as the rest of the host (include/cleanba_mi.h: cbm_top_logits, cbm_distill_loss_grad, cbm_verify_drafts, where the definitions stand); these
wrappers check shapes and types, allocate outputs and workspace with torch, and enqueue on torch's current stream of the tensors' device.  Nothing waits:
the results are ready in stream order, like those of any torch operator, and the calls can be captured into a torch.cuda.graph.  There is no autograd
node: as with the PPO and IMPALA losses the gradient is an output.

A training step of a student and a serving step of a draft:

    idx, values, lse = tokens.top_logits(ctx, teacher_logits, 64)
    loss, dlogits = tokens.distill_loss_grad(ctx, student_logits, idx, values, teacher_lse=lse, row_weight=weight)
    ...
    x, _, _ = tokens.verify_drafts(ctx, draft_logits[:, :1], None, None, u)          # no drafts: samples one token a sequence
    out, accepted, logprobs = tokens.verify_drafts(ctx, target_logits, drafted, u_accept, u_sample, draft_logits=draft_logits)
"""
import functools

import torch

from . import lib as L

_DTYPE = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}
# (new_empty of a tensor of the right type is quicker than empty by 0.3 us)
_empty, _i32, _f32, _u8 = torch.empty, torch.int32, torch.float32, torch.uint8
try:   # the handle alone: a Stream object costs 2 us, as much as the launch
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:   # a build of torch without it
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


# The calls below are made once a token: their checks read each attribute once, and what a plan needs of workspace is asked once a shape.
def _logits(dev, t, name, dims=None):
    """(CBM_ type, shape, strides) of a tensor of logits on device `dev`."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPE:
        raise ValueError(f"{name}: a float32, bfloat16 or float16 tensor is expected")
    shape, strides = t.shape, t.stride()
    if not shape or (dims is not None and len(shape) != dims):
        raise ValueError(f"{name}: {dims or 'one or more'} dimensions are expected, got {tuple(shape)}")
    if t.numel() > 0x7fffffff:
        _fits(shape[-1], f"{name}: tokens")
        _fits(shape[:-1].numel(), f"{name}: rows")
    if strides[-1] != 1 and shape[-1] > 1 and t.numel():
        raise ValueError(f"{name}: the vocabulary (the last axis) has to be dense, its stride is {strides[-1]}")
    _placed(dev, t, name)
    return _DTYPE[t.dtype], shape, strides


def _fits(n, name):
    if not -0x80000000 <= n <= 0x7fffffff:   # (the C calls take 32 bits, and ctypes cuts to them without a word)
        raise ValueError(f"{name}: {n} is more than any call takes")


def _placed(dev, t, name):
    if t.get_device() != dev:   # (-1: not on a GPU)
        raise ValueError(f"{name}: on {t.device}, the context's device is cuda:{dev}")


def _operand(dev, t, name, dtype, shape):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name}: a {str(dtype)[6:]} tensor of shape {tuple(shape)} is expected, got "
                         f"{(str(t.dtype)[6:], tuple(t.shape)) if isinstance(t, torch.Tensor) else type(t).__name__}")
    _placed(dev, t, name)
    return t if t.is_contiguous() else t.contiguous()


def _rows(t, shape, strides, name):
    """(rows, elements from row to row) of [..., vocab]; the leading axes have to fold into one."""
    dims = len(shape)
    if dims == 2:
        return shape[0], strides[0]
    if dims == 1:
        return 1, shape[0]
    try:
        t = t.view(-1, shape[-1]) if t.numel() else t.reshape(shape[:-1].numel(), shape[-1])
    except RuntimeError:
        raise ValueError(f"{name}: the leading axes of strides {strides} do not fold into rows of one stride") from None
    return t.shape[0], t.stride(0)


@functools.lru_cache(maxsize=4096)
def _top_workspace(dtype, rows, vocab, k):
    return _checked(L.load().cbm_top_logits_workspace(dtype, rows, vocab, k))


@functools.lru_cache(maxsize=4096)
def _verify_workspace(dtype, batch, drafts, vocab, with_draft, temperature):
    return _checked(L.load().cbm_verify_drafts_workspace(dtype, batch, drafts, vocab, with_draft, temperature))


def _checked(nbytes):
    if nbytes < 0:
        raise L.CbmError(L.load().cbm_last_error().decode())
    return nbytes


def _ptr(t):
    return None if t is None else t.data_ptr()


def top_logits(ctx, logits, k, temperature=1.0):
    """The k largest logits of each row of `logits` [..., vocab], falling, equal ones by rising index -> (idx int32 [..., k], values float32 [..., k],
    lse float32 [...] = log sum exp(logits / temperature)).  Slots beyond the logits above -inf hold -1 and -inf (cbm_top_logits)."""
    index, k = ctx.cfg.device, int(k)
    _fits(k, "k")
    dtype, shape, strides = _logits(index, logits, "logits")
    rows, stride = _rows(logits, shape, strides, "logits")
    vocab, lead, dev = shape[-1], shape[:-1], logits.device
    nbytes = _top_workspace(dtype, rows, vocab, k)
    ws = _empty((nbytes,), dtype=_u8, device=dev) if nbytes else None   # (held to the end of the call; behind it the allocator hands it out in stream order)
    idx = _empty(lead + (k,), dtype=_i32, device=dev)
    values = _empty(lead + (k,), dtype=_f32, device=dev)
    lse = values.new_empty(lead)
    if ctx.lib.cbm_top_logits(ctx.h, logits.data_ptr(), dtype, rows, vocab, stride, k, temperature, idx.data_ptr(), values.data_ptr(), lse.data_ptr(), _ptr(ws), nbytes,
                              _raw_stream(index)):
        L._chk(-1)
    return idx, values, lse


def distill_loss_grad(ctx, logits, teacher_idx, teacher_logits, teacher_lse=None, row_weight=None, temperature=1.0, want_grad=True, in_place=False):
    """Distillation of the student's `logits` [..., vocab] from a teacher's top logits (idx int32, float32 [..., k]) -> (loss float32 [...], dlogits or None).

    teacher_lse float32 [...] keeps the teacher's mass outside its slots as one more class; without it the teacher is a softmax over the slots.
    row_weight float32 [...] scales a row's loss and gradient; rows of weight 0 are not read.  in_place=True writes the gradient over the logits
    (their version counter rises).  Neither output has a graph: `logits.backward(dlogits)` takes a student further.  (cbm_distill_loss_grad)"""
    index = ctx.cfg.device
    dtype, shape, strides = _logits(index, logits, "logits")
    rows, stride = _rows(logits, shape, strides, "logits")
    vocab, lead = shape[-1], shape[:-1]
    if not isinstance(teacher_idx, torch.Tensor) or teacher_idx.dim() != len(shape):
        raise ValueError(f"teacher_idx: an int32 tensor of shape {tuple(lead) + ('k',)} is expected")
    k = teacher_idx.shape[-1]
    _fits(k, "teacher_idx: slots")
    slots = lead + (k,)
    teacher_idx = _operand(index, teacher_idx, "teacher_idx", _i32, slots)
    teacher_logits = _operand(index, teacher_logits, "teacher_logits", _f32, slots)
    if teacher_lse is not None:
        teacher_lse = _operand(index, teacher_lse, "teacher_lse", _f32, lead)
    if row_weight is not None:
        row_weight = _operand(index, row_weight, "row_weight", _f32, lead)
    loss = teacher_logits.new_empty(lead)
    grad, gstride = None, 0
    if want_grad:
        grad, gstride = (logits, stride) if in_place else (logits.new_empty(shape), vocab)
    if ctx.lib.cbm_distill_loss_grad(ctx.h, logits.data_ptr(), dtype, rows, vocab, stride, teacher_idx.data_ptr(), teacher_logits.data_ptr(), k,
                                     _ptr(teacher_lse), _ptr(row_weight), temperature, loss.data_ptr(), _ptr(grad), gstride, _raw_stream(index)):
        L._chk(-1)
    if grad is logits:
        torch.autograd.graph.increment_version(logits)   # as torch's own in-place operators: a backward that saved the logits notices
    return loss, grad


def verify_drafts(ctx, target_logits, draft_tokens, u_accept, u_sample, draft_logits=None, n_draft=None, temperature=1.0):
    """Verification of `draft_tokens` int32 [batch, drafts] against `target_logits` [batch, drafts + 1, vocab] -> (tokens int32 [batch, drafts + 1]: the
    accepted ones, one drawn token, then -1; accepted int32 [batch]; logprobs float32 [batch, drafts + 1] under the target, 0 behind the last).

    draft_logits [batch, drafts, vocab]: what the drafts were sampled from; None: they were looked up.  u_accept float32 [batch, drafts] and u_sample
    float32 [batch] are uniform numbers in [0, 1); n_draft int32 [batch] says how many drafts of a sequence count.  temperature 0 takes the largest
    logit and looks at neither.  draft_tokens and u_accept may be None where target_logits has one position: one token a sequence is sampled.
    (cbm_verify_drafts)"""
    index = ctx.cfg.device
    dtype, shape, tstride = _logits(index, target_logits, "target_logits", 3)
    batch, positions, vocab = shape
    drafts, dev, greedy = positions - 1, target_logits.device, temperature == 0
    if drafts < 0:
        raise ValueError("target_logits: one position at least is expected")
    two = (batch, drafts)
    if drafts or draft_tokens is not None:
        draft_tokens = _operand(index, draft_tokens, "draft_tokens", _i32, two)
    if u_accept is not None or (drafts and not greedy):
        u_accept = _operand(index, u_accept, "u_accept", _f32, two)
    if u_sample is not None or not greedy:
        u_sample = _operand(index, u_sample, "u_sample", _f32, (batch,))
    if n_draft is not None:
        n_draft = _operand(index, n_draft, "n_draft", _i32, (batch,))
    dstride = (0, 0)
    if draft_logits is not None:
        dtype2, shape2, dstride = _logits(index, draft_logits, "draft_logits", 3)
        if dtype2 != dtype or shape2 != (batch, drafts, vocab):
            raise ValueError(f"draft_logits: {str(target_logits.dtype)[6:]} {(batch, drafts, vocab)} is expected, got {str(draft_logits.dtype)[6:]} {tuple(shape2)}")
        if drafts == 0:
            draft_logits = None
    nbytes = _verify_workspace(dtype, batch, drafts, vocab, draft_logits is not None, temperature)
    ws = _empty((nbytes,), dtype=_u8, device=dev) if nbytes else None   # (held to the end of the call; behind it the allocator hands it out in stream order)
    tokens = _empty((batch, positions), dtype=_i32, device=dev)
    accepted = tokens.new_empty((batch,))
    logprobs = _empty((batch, positions), dtype=_f32, device=dev)
    if ctx.lib.cbm_verify_drafts(ctx.h, target_logits.data_ptr(), dtype, batch, drafts, vocab, tstride[0], tstride[1], _ptr(draft_logits), dstride[0], dstride[1],
                                 _ptr(draft_tokens), _ptr(n_draft), _ptr(u_accept), _ptr(u_sample), temperature, tokens.data_ptr(), accepted.data_ptr(),
                                 logprobs.data_ptr(), _ptr(ws), nbytes, _raw_stream(index)):
        L._chk(-1)
    return tokens, accepted, logprobs

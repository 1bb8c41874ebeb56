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
import torch

from . import lib as L

_DTYPE = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}
_empty, _i32, _f32 = torch.empty, torch.int32, torch.float32
try:   # the handle alone: a Stream object costs 2 us, as much as the launch
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:   # a build of torch without it
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


def _logits(ctx, t, name, dims=None):
    """CBM_ type of a tensor of logits."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPE:
        raise ValueError(f"{name}: a float32, bfloat16 or float16 tensor is expected")
    shape = t.shape
    if not shape or (dims is not None and len(shape) != dims):
        raise ValueError(f"{name}: {dims or 'one or more'} dimensions are expected, got {tuple(shape)}")
    if t.stride(-1) != 1 and shape[-1] > 1 and t.numel():
        raise ValueError(f"{name}: the vocabulary (the last axis) has to be dense, its stride is {t.stride(-1)}")
    _placed(ctx, t, name)
    return _DTYPE[t.dtype]


def _placed(ctx, t, name):
    if not t.is_cuda or t.get_device() != ctx.cfg.device:
        raise ValueError(f"{name}: on {t.device}, the context's device is cuda:{ctx.cfg.device}")


def _operand(ctx, t, name, dtype, shape):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name}: a {str(dtype)[6:]} tensor of shape {tuple(shape)} is expected, got "
                         f"{(str(t.dtype)[6:], tuple(t.shape)) if isinstance(t, torch.Tensor) else type(t).__name__}")
    _placed(ctx, t, name)
    return t if t.is_contiguous() else t.contiguous()


def _rows(t, name):
    """(rows, elements from row to row) of [..., vocab]; the leading axes have to fold into one."""
    dims = t.dim()
    if dims == 1:
        return 1, t.shape[0]
    if dims > 2:
        try:
            t = t.view(-1, t.shape[-1]) if t.numel() else t.reshape(t.shape[:-1].numel(), t.shape[-1])
        except RuntimeError:
            raise ValueError(f"{name}: the leading axes of strides {t.stride()} do not fold into rows of one stride") from None
    return t.shape[0], t.stride(0)


def _workspace(nbytes, device):
    if nbytes < 0:
        raise L.CbmError(L.load().cbm_last_error().decode())
    return _empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def top_logits(ctx, logits, k, temperature=1.0):
    """The k largest logits of each row of `logits` [..., vocab], falling, equal ones by rising index -> (idx int32 [..., k], values float32 [..., k],
    lse float32 [...] = log sum exp(logits / temperature)).  Slots beyond the logits above -inf hold -1 and -inf (cbm_top_logits)."""
    dtype = _logits(ctx, logits, "logits")
    rows, stride = _rows(logits, "logits")
    shape, dev, k = logits.shape, logits.device, int(k)
    vocab, lead = shape[-1], shape[:-1]
    ws = _workspace(ctx.lib.cbm_top_logits_workspace(dtype, rows, vocab, k), dev)
    idx = _empty(lead + (k,), dtype=_i32, device=dev)
    values = _empty(lead + (k,), dtype=_f32, device=dev)
    lse = _empty(lead, dtype=_f32, device=dev)
    L._chk(ctx.lib.cbm_top_logits(ctx.h, logits.data_ptr(), dtype, rows, vocab, stride, k, temperature, idx.data_ptr(), values.data_ptr(), lse.data_ptr(),
                                  _ptr(ws), 0 if ws is None else ws.numel(), _raw_stream(ctx.cfg.device)))
    return idx, values, lse


def distill_loss_grad(ctx, logits, teacher_idx, teacher_logits, teacher_lse=None, row_weight=None, temperature=1.0, want_grad=True, in_place=False):
    """Distillation of the student's `logits` [..., vocab] from a teacher's top logits (idx int32, float32 [..., k]) -> (loss float32 [...], dlogits or None).

    teacher_lse float32 [...] keeps the teacher's mass outside its slots as one more class; without it the teacher is a softmax over the slots.
    row_weight float32 [...] scales a row's loss and gradient; rows of weight 0 are not read.  in_place=True writes the gradient over the logits.
    (cbm_distill_loss_grad)"""
    dtype = _logits(ctx, logits, "logits")
    rows, stride = _rows(logits, "logits")
    shape, dev = logits.shape, logits.device
    vocab, lead = shape[-1], shape[:-1]
    if not isinstance(teacher_idx, torch.Tensor) or teacher_idx.dim() != logits.dim():
        raise ValueError(f"teacher_idx: an int32 tensor of shape {tuple(lead) + ('k',)} is expected")
    k = teacher_idx.shape[-1]
    teacher_idx = _operand(ctx, teacher_idx, "teacher_idx", torch.int32, lead + (k,))
    teacher_logits = _operand(ctx, teacher_logits, "teacher_logits", torch.float32, lead + (k,))
    if teacher_lse is not None:
        teacher_lse = _operand(ctx, teacher_lse, "teacher_lse", torch.float32, lead)
    if row_weight is not None:
        row_weight = _operand(ctx, row_weight, "row_weight", torch.float32, lead)
    loss = _empty(lead, dtype=_f32, device=dev)
    grad, gstride = None, 0
    if want_grad:
        grad = logits if in_place else torch.empty_like(logits, memory_format=torch.contiguous_format)
        gstride = stride if in_place else vocab
    L._chk(ctx.lib.cbm_distill_loss_grad(ctx.h, logits.data_ptr(), dtype, rows, vocab, stride, teacher_idx.data_ptr(), teacher_logits.data_ptr(), k,
                                         _ptr(teacher_lse), _ptr(row_weight), temperature, loss.data_ptr(), _ptr(grad), gstride,
                                         _raw_stream(ctx.cfg.device)))
    return loss, grad


def verify_drafts(ctx, target_logits, draft_tokens, u_accept, u_sample, draft_logits=None, n_draft=None, temperature=1.0):
    """Verification of `draft_tokens` int32 [batch, drafts] against `target_logits` [batch, drafts + 1, vocab] -> (tokens int32 [batch, drafts + 1]: the
    accepted ones, one drawn token, then -1; accepted int32 [batch]; logprobs float32 [batch, drafts + 1] under the target, 0 behind the last).

    draft_logits [batch, drafts, vocab]: what the drafts were sampled from; None: they were looked up.  u_accept float32 [batch, drafts] and u_sample
    float32 [batch] are uniform numbers in [0, 1); n_draft int32 [batch] says how many drafts of a sequence count.  temperature 0 takes the largest
    logit and looks at neither.  draft_tokens and u_accept may be None where target_logits has one position: one token a sequence is sampled.
    (cbm_verify_drafts)"""
    dtype = _logits(ctx, target_logits, "target_logits", 3)
    batch, positions, vocab = target_logits.shape
    drafts, dev = positions - 1, target_logits.device
    if drafts < 0:
        raise ValueError("target_logits: one position at least is expected")
    if drafts or draft_tokens is not None:
        draft_tokens = _operand(ctx, draft_tokens, "draft_tokens", torch.int32, (batch, drafts))
    if u_accept is not None or (drafts and temperature != 0):
        u_accept = _operand(ctx, u_accept, "u_accept", torch.float32, (batch, drafts))
    if u_sample is not None or temperature != 0:
        u_sample = _operand(ctx, u_sample, "u_sample", torch.float32, (batch,))
    if n_draft is not None:
        n_draft = _operand(ctx, n_draft, "n_draft", torch.int32, (batch,))
    dstride = (0, 0)
    if draft_logits is not None:
        if _logits(ctx, draft_logits, "draft_logits", 3) != dtype or tuple(draft_logits.shape) != (batch, drafts, vocab):
            raise ValueError(f"draft_logits: {str(target_logits.dtype)[6:]} {(batch, drafts, vocab)} is expected, got {str(draft_logits.dtype)[6:]} {tuple(draft_logits.shape)}")
        dstride = draft_logits.stride()
        if drafts == 0:
            draft_logits = None
    ws = _workspace(ctx.lib.cbm_verify_drafts_workspace(dtype, batch, drafts, vocab, draft_logits is not None, temperature), dev)
    tokens = _empty((batch, positions), dtype=_i32, device=dev)
    accepted = _empty(batch, dtype=_i32, device=dev)
    logprobs = _empty((batch, positions), dtype=_f32, device=dev)
    L._chk(ctx.lib.cbm_verify_drafts(ctx.h, target_logits.data_ptr(), dtype, batch, drafts, vocab, target_logits.stride(0), target_logits.stride(1),
                                     _ptr(draft_logits), dstride[0], dstride[1], _ptr(draft_tokens), _ptr(n_draft), _ptr(u_accept), _ptr(u_sample),
                                     temperature, tokens.data_ptr(), accepted.data_ptr(), logprobs.data_ptr(), _ptr(ws), 0 if ws is None else ws.numel(),
                                     _raw_stream(ctx.cfg.device)))
    return tokens, accepted, logprobs

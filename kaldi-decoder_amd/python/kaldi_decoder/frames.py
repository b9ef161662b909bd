"""Operators over a model's frame logits, on the GPU: the rows that the decoders read.

`token_scores`: the log-probability of a given token a row (a best path's, a transcript's), the
row's entropy, and its largest alternatives; differentiable, or with `token_scores_grad` by hand.
`distill_loss`: the divergence from a teacher's listed tokens -- what `token_scores(top=K)` of the
teacher's rows gives -- differentiable, or as loss and gradient in one call
(`distill_loss_and_grad`).

Rows are a CUDA tensor [N, V] or [B, T, V], float32, float16 or bfloat16, with unit stride over V
and any strides over the others (views of padded tensors are read in place); `lengths` [B] are the
valid rows of each utterance, as in `Batch.decode_tensor`: what lies behind is not read, scores 0
and gets gradient 0.  Sums are float32 whatever the rows' type.  Calls run on the current stream of
the tensors' device, allocate through torch's allocator and do not synchronise (but for `lengths`
that are not on the device yet): they can be captured into a graph.  A backward pass through
autograd that is to be captured needs its leaves to have no live graph from outside the capture, as
any of torch's; `token_scores_grad` and `distill_loss_and_grad` have no such condition.

(The reference leaves all of this to its callers; its DecodableCtc takes log-probabilities,
csrc/decodable-ctc.cc:28.)
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import cabi

MAX_TOP = 64      # alternatives a row
MAX_SLOTS = 256   # teacher's tokens a row
MAX_VOCAB = 1 << 24
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ID_BYTES = {torch.int32: 4, torch.int64: 8}


class TokenScores(NamedTuple):
    """`logp` (None without tokens) and `entropy` [...] float32; `top_logp` float32 and `top_ids`
    int32 [..., top] (None for top = 0), largest first, the lowest column first among equals, -inf /
    -1 where a row has fewer finite logits; `stats` [..., 2] float32, the row's maximum m and
    sum exp(x - m), which the gradient reads (log_softmax(x) = x - m - log of it)."""
    logp: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]
    stats: torch.Tensor


def _rows(logits, lengths, what="logits"):
    """(kd_frame_rows, tensors that it points into) of a tensor of rows."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES or not logits.is_cuda:
        raise ValueError(f"{what} must be a float32, float16 or bfloat16 CUDA tensor")
    shape = logits.shape
    stride = logits.stride()
    if len(shape) == 2:
        batch, (steps, vocab), bstride, rstride = 1, shape, 0, stride[0]
        if lengths is not None:
            raise ValueError(f"lengths need {what} [B, T, V]")
    elif len(shape) == 3:
        (batch, steps, vocab), bstride, rstride = shape, stride[0], stride[1]
        if lengths is not None:
            lengths = _lengths(lengths, batch, logits.device)
        elif bstride == steps * rstride:  # (one run of rows: no division by `steps` in the kernels)
            batch, steps = 1, batch * steps
    else:
        raise ValueError(f"{what} must be [N, V] or [B, T, V]")
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"{what}: V must be between 1 and 2^24")
    if stride[-1] != 1 and vocab != 1:
        raise ValueError(f"{what} need unit stride over the last (V) dimension")
    return cabi.FrameRows(logits.data_ptr(), batch, steps, vocab, bstride, rstride,
                          None if lengths is None else lengths.data_ptr(), _DTYPES[logits.dtype],
                          logits.device.index), lengths


def _lengths(lengths, batch, device):
    if not isinstance(lengths, torch.Tensor):
        lengths = torch.as_tensor(lengths)
    if lengths.shape != (batch,) or lengths.dtype not in _ID_BYTES:
        raise ValueError("lengths must be int32 or int64 [B]")
    return lengths.to(device=device, dtype=torch.int32).contiguous()


def _per_row(t, lead, device, dtypes, what):
    """A tensor of one value a row (shape `lead`), contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.device != device:
        raise ValueError(f"{what} must be a tensor of {' or '.join(str(d)[6:] for d in dtypes)} on {device}")
    if t.shape != lead:
        raise ValueError(f"{what} must have shape {list(lead)}, not {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _grad_out(out, logits):
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if not isinstance(out, torch.Tensor) or out.shape != logits.shape or out.dtype != logits.dtype \
            or out.device != logits.device:
        raise ValueError("out must have the logits' shape, dtype and device")
    if out.stride(-1) != 1 and out.shape[-1] != 1:
        raise ValueError("out needs unit stride over the last (V) dimension")
    return out


def _out_strides(out, rows):
    """`out`'s strides for the batch and steps of `rows` (or other rows, where those were joined)."""
    s = out.stride()
    if out.dim() == 2:
        return 0, s[0]
    if rows.batch == 1 and out.shape[0] != 1:  # joined
        if s[0] != out.shape[1] * s[1]:
            rows.batch, rows.steps = out.shape[0], out.shape[1]
            rows.batch_stride = rows.steps * rows.row_stride
            return s[0], s[1]
        return 0, s[1]
    return s[0], s[1]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _workspace(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _token_scores(logits, tokens, top, lengths):
    rows, keep = _rows(logits, lengths)
    lead, dev, L = logits.shape[:-1], logits.device, cabi.lib()
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be between 0 and {MAX_TOP}")
    f32 = torch.float32
    logp = top_logp = top_ids = None
    id_bytes = 0
    if tokens is not None:
        tokens = _per_row(tokens, lead, dev, _ID_BYTES, "tokens")
        id_bytes = _ID_BYTES[tokens.dtype]
        logp = torch.empty(lead, dtype=f32, device=dev)
    entropy = torch.empty(lead, dtype=f32, device=dev)
    stats = torch.empty((*lead, 2), dtype=f32, device=dev)
    if top:
        top_logp = torch.empty((*lead, top), dtype=f32, device=dev)
        top_ids = torch.empty((*lead, top), dtype=torch.int32, device=dev)
    ref = C.byref(rows)
    size = L.kd_token_scores_workspace(ref, top)
    ws = _workspace(size, dev)
    cabi._check(L.kd_token_scores(ref, _ptr(tokens), id_bytes, top, _ptr(logp), entropy.data_ptr(), stats.data_ptr(),
                                  _ptr(top_logp), _ptr(top_ids), _ptr(ws), size, _stream(dev)))
    return logp, entropy, top_logp, top_ids, stats


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, lengths):
        logp, entropy, top_logp, top_ids, stats = _token_scores(logits, tokens, top, lengths)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (top_logp, top_ids, stats) if t is not None])
        ctx.save_for_backward(logits, tokens, lengths, stats, entropy)
        return logp, entropy, top_logp, top_ids, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, *_):
        logits, tokens, lengths, stats, entropy = ctx.saved_tensors
        if g_logp is None and g_entropy is None:
            return None, None, None, None
        return _token_scores_grad(logits, tokens, lengths, stats, entropy, g_logp, g_entropy, None), None, None, None


def _token_scores_grad(logits, tokens, lengths, stats, entropy, g_logp, g_entropy, out):
    rows, keep = _rows(logits, lengths)
    lead, dev = logits.shape[:-1], logits.device
    f32 = (torch.float32,)
    id_bytes = 0
    if tokens is not None:
        tokens = _per_row(tokens, lead, dev, _ID_BYTES, "tokens")
        id_bytes = _ID_BYTES[tokens.dtype]
    stats = _per_row(stats, (*lead, 2), dev, f32, "stats")
    entropy = _per_row(entropy, lead, dev, f32, "entropy")
    if g_logp is not None:
        g_logp = _per_row(g_logp, lead, dev, f32, "grad_logp")
    if g_entropy is not None:
        g_entropy = _per_row(g_entropy, lead, dev, f32, "grad_entropy")
    out = _grad_out(out, logits)
    bs, rs = _out_strides(out, rows)
    cabi._check(cabi.lib().kd_token_scores_grad(C.byref(rows), _ptr(tokens), id_bytes, stats.data_ptr(),
                                                entropy.data_ptr(), _ptr(g_logp), _ptr(g_entropy), out.data_ptr(), bs,
                                                rs, _stream(dev)))
    return out


def token_scores(logits, tokens=None, top=0, lengths=None):
    """TokenScores of rows of logits: log softmax(row)[token] (`tokens` int32 or int64, shape
    logits.shape[:-1]; a token outside [0, V), such as -1 for padding, scores 0), the entropy of
    softmax(row), and the `top` <= 64 largest logits' columns and log-probabilities.

    A logit of -inf rules its column out (probability 0, never an alternative); a row of nothing else
    has logp -inf, entropy 0 and no alternatives.  NaN or +inf in a row: NaN.  `logp` and `entropy`
    are differentiable in the logits, the alternatives are not."""
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        if lengths is not None and logits.dim() == 3:
            lengths = _lengths(lengths, logits.shape[0], logits.device)
        return TokenScores(*_TokenScores.apply(logits, tokens, top, lengths))
    return TokenScores(*_token_scores(logits, tokens, top, lengths))


@torch.no_grad()
def token_scores_grad(logits, scores, tokens=None, lengths=None, grad_logp=None, grad_entropy=None, out=None):
    """The gradient of the logits for upstream gradients of scores.logp and scores.entropy (float32,
    shape logits.shape[:-1]; None: 0), where `scores` = token_scores(logits, tokens, ..., lengths).
    Written to `out` (the logits' shape and dtype, rows that do not overlap) or to a new tensor."""
    return _token_scores_grad(logits, tokens, lengths, scores.stats, scores.entropy, grad_logp, grad_entropy, out)


def _distill(logits, ids, teacher, weights, temperature, lengths, want_loss, stats, upstream, want_grad, out):
    rows, keep = _rows(logits, lengths)
    lead, dev, L = logits.shape[:-1], logits.device, cabi.lib()
    f32 = torch.float32
    if not isinstance(ids, torch.Tensor) or ids.dim() != logits.dim() or not 1 <= ids.shape[-1] <= MAX_SLOTS:
        raise ValueError(f"teacher_ids must be [..., K] with 1 <= K <= {MAX_SLOTS}, beside logits [..., V]")
    slots = ids.shape[-1]
    ids = _per_row(ids, (*lead, slots), dev, _ID_BYTES, "teacher_ids")
    teacher = _per_row(teacher, (*lead, slots), dev, _DTYPES, "teacher_logits")
    if weights is not None:
        weights = _per_row(weights, lead, dev, (f32,), "weights")
    if upstream is not None:
        upstream = _per_row(upstream, lead, dev, (f32,), "the loss's gradient")
    t = cabi.TeacherRows(ids.data_ptr(), teacher.data_ptr(), slots, _ID_BYTES[ids.dtype], _DTYPES[teacher.dtype])
    loss = torch.empty(lead, dtype=f32, device=dev) if want_loss else None
    bs = rs = 0
    if want_grad:
        out = _grad_out(out, logits)
        bs, rs = _out_strides(out, rows)
    ref = C.byref(rows)
    size = L.kd_distill_loss_workspace(ref) if want_loss else 0
    ws = _workspace(size, dev)
    cabi._check(L.kd_distill_loss(ref, C.byref(t), _ptr(weights), temperature, _ptr(loss), _ptr(stats), _ptr(upstream),
                                  _ptr(out), bs, rs, _ptr(ws), size, _stream(dev)))
    return loss, out


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, weights, temperature, lengths):
        stats = torch.empty((*logits.shape[:-1], 2), dtype=torch.float32, device=logits.device)
        loss, _ = _distill(logits, ids, teacher, weights, temperature, lengths, True, stats, None, False, None)
        ctx.save_for_backward(logits, ids, teacher, weights, lengths, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, ids, teacher, weights, lengths, stats = ctx.saved_tensors
        _, grad = _distill(logits, ids, teacher, weights, ctx.temperature, lengths, False, stats, g, True, None)
        return grad, None, None, None, None, None


def _constant(**tensors):
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and t.requires_grad:
            raise ValueError(f"{name} takes no gradient here: detach it")


def distill_loss(logits, teacher_ids, teacher_logits, weights=None, temperature=1.0, lengths=None):
    """Per row, weight * KL(q || p) over the tokens a teacher lists: q = softmax(teacher_logits /
    temperature) over the row's list, p = softmax(logits / temperature) over the vocabulary.

    `teacher_ids` (int32 or int64) and `teacher_logits` (float32, float16, bfloat16; log-probabilities
    serve as well) [..., K], K <= 256; an id outside [0, V), such as -1, marks an empty slot, one that
    is listed twice counts twice.  `weights` float32, shape logits.shape[:-1]: rows of weight 0, rows
    without a listed token and rows behind `lengths` are not read (loss 0, gradient 0).  The loss
    (float32, shape logits.shape[:-1]) is differentiable in the logits alone.  Where the weights are all that scales it
    (a mean: weights of 1 / rows), distill_loss_and_grad does the work of both passes in one."""
    _constant(teacher_logits=teacher_logits, weights=weights)
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        if lengths is not None and logits.dim() == 3:
            lengths = _lengths(lengths, logits.shape[0], logits.device)
        return _DistillLoss.apply(logits, teacher_ids, teacher_logits, weights, temperature, lengths)
    return _distill(logits, teacher_ids, teacher_logits, weights, temperature, lengths, True, None, None, False, None)[0]


@torch.no_grad()
def distill_loss_and_grad(logits, teacher_ids, teacher_logits, weights=None, temperature=1.0, lengths=None, out=None):
    """(loss, gradient of loss.sum() in the logits): distill_loss and its backward pass in one call,
    which reads rows of up to 32 KiB once.  The gradient goes to `out` (the logits' shape and dtype,
    rows that do not overlap) or to a new tensor."""
    return _distill(logits, teacher_ids, teacher_logits, weights, temperature, lengths, True, None, None, True, out)

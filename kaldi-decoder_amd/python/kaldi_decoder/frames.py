"""Operators over a model's frame logits, on the GPU: the rows that the decoders read.

`token_scores`: the log-probability of a given token a row (a best path's, a transcript's), the
row's entropy, and its largest alternatives; differentiable, or with `token_scores_grad` by hand.
`distill_loss`: the divergence from a teacher's listed tokens -- what `token_scores(top=K)` of the
teacher's rows gives -- differentiable, or as loss and gradient in one call
(`distill_loss_and_grad`).

Rows are a CUDA tensor [N, V] or [B, T, V], float32, float16 or bfloat16, with unit stride over V
and any strides over the others (views of padded tensors are read in place); `lengths` [B] are the
valid rows of each utterance, 0 to T as in `Batch.decode_tensor` (not checked here: they may be on
the GPU): what lies behind is not read, scores 0 and gets gradient 0.  Sums are float32 whatever the
rows' type.  Calls run on the current stream of the tensors' device, allocate through torch's
allocator and do not synchronise (but for `lengths` that are not on the device yet): they can be
captured into a graph.  A backward pass through autograd that is to be captured needs its leaves to
have no live graph from outside the capture, as any of torch's; `token_scores_grad` and
`distill_loss_and_grad` have no such condition.

What is differentiable is so once, backwards: a second derivative (create_graph) and forward mode (a
tensor that carries a tangent) raise an error.  `token_scores_grad` and `distill_loss_and_grad` are
outside autograd altogether.

(The reference leaves all of this to its callers; its DecodableCtc takes log-probabilities,
csrc/decodable-ctc.cc:28.)
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

try:
    from .lib import _frames
except ImportError as e:  # pragma: no cover
    raise ImportError("kaldi_decoder.frames: the native extension is not built. Run `make -C kaldi-decoder_amd` or "
                      f"`python __graft_entry__.py`; there is no CPU fallback. Original error: {e}") from e

MAX_TOP = 64      # alternatives a row
MAX_SLOTS = 256   # teacher's tokens a row
MAX_VOCAB = 1 << 24


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


def _tensors(logits, lengths):
    """lengths as a tensor (or None); `logits` is one."""
    if not isinstance(logits, torch.Tensor):
        raise ValueError("logits must be a float32, float16 or bfloat16 CUDA tensor")
    if lengths is None or isinstance(lengths, torch.Tensor):
        return lengths
    return torch.as_tensor(lengths)


def token_scores(logits, tokens=None, top=0, lengths=None):
    """TokenScores of rows of logits: log softmax(row)[token] (`tokens` int32 or int64, shape
    logits.shape[:-1]; a token outside [0, V), such as -1 for padding, scores 0), the entropy of
    softmax(row), and the `top` <= 64 largest logits' columns and log-probabilities.

    A logit of -inf rules its column out (probability 0, never an alternative); a row of nothing else
    has logp -inf, entropy 0 and no alternatives.  NaN or +inf in a row: NaN.  (A mask of a finite value
    instead leaves candidates: with fewer than `top` columns above it, the alternatives take 15 to 60 times
    as long.)  `logp` and `entropy` are differentiable in the logits, the alternatives are not."""
    lengths = _tensors(logits, lengths)
    return TokenScores._make(_frames.token_scores(logits, tokens, top, lengths))


def token_scores_grad(logits, scores, tokens=None, lengths=None, grad_logp=None, grad_entropy=None, out=None):
    """The gradient of the logits for upstream gradients of scores.logp and scores.entropy (float32,
    shape logits.shape[:-1]; None: 0), where `scores` = token_scores(logits, tokens, ..., lengths).
    Written to `out` (the logits' shape and dtype, rows that do not overlap, apart from everything that is
    read; `logits` itself will do) or to a new tensor."""
    return _frames.token_scores_grad(logits, tokens, _tensors(logits, lengths), scores.stats, scores.entropy, grad_logp,
                                     grad_entropy, out)


def distill_loss(logits, teacher_ids, teacher_logits, weights=None, temperature=1.0, lengths=None):
    """Per row, weight * KL(q || p) over the tokens a teacher lists: q = softmax(teacher_logits /
    temperature) over the row's list, p = softmax(logits / temperature) over the vocabulary;
    1e-6 <= temperature <= 1e6.

    `teacher_ids` (int32 or int64) and `teacher_logits` (float32, float16, bfloat16; log-probabilities
    serve as well) [..., K], K <= 256; an id outside [0, V), such as -1, or a logit of -inf marks an
    empty slot, a token that is listed twice counts twice.  `weights` float32, shape logits.shape[:-1]: rows
    of weight 0 and rows behind `lengths` are not read, rows without a listed token may hold anything (loss
    0, gradient 0).  The loss
    (float32, shape logits.shape[:-1]) is differentiable in the logits alone.  Where the weights are all
    that scales it (a mean: weights of 1 / rows), distill_loss_and_grad does the work of both passes in one."""
    return _frames.distill_loss(logits, teacher_ids, teacher_logits, weights, temperature, _tensors(logits, lengths))


def distill_loss_and_grad(logits, teacher_ids, teacher_logits, weights=None, temperature=1.0, lengths=None, out=None):
    """(loss, gradient of loss.sum() in the logits): distill_loss and its backward pass in one call,
    which reads rows of up to 64 KiB (many rows of up to 256 KiB) once.  The gradient goes to `out` (the
    logits' shape and dtype, rows that do not overlap, apart from everything that is read; `logits` itself will
    do) or to a new tensor."""
    return _frames.distill_loss_and_grad(logits, teacher_ids, teacher_logits, weights, temperature,
                                         _tensors(logits, lengths), out)

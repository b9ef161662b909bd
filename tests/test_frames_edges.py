"""kaldi_decoder.frames without a GPU: calls that are refused on the host, before anything is launched."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from kaldi_decoder import frames


def test_forward_mode_derivatives_are_refused():
    """A tangent would be dropped without a word: a derivative of 0."""
    x, ids, u = torch.randn(3, 5), torch.zeros(3, 2, dtype=torch.int32), torch.randn(3, 2)
    scores = frames.TokenScores(None, torch.zeros(3), None, None, torch.ones(3, 2))
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: frames.token_scores(dual), lambda: frames.distill_loss(dual, ids, u),
                     lambda: frames.distill_loss_and_grad(dual, ids, u),
                     lambda: frames.token_scores_grad(dual, scores)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="CUDA tensor"):  # (without its tangent, the next refusal)
            frames.token_scores(dual.detach())

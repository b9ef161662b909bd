"""kaldi_decoder.frames without a GPU: what is refused, by the Python layer and by the C entries, and
the oracle of the GPU tests against torch's autograd."""
import ctypes as C

import pytest
import torch

import frames_ref
from kaldi_decoder import cabi, frames


def _rows(**kw):
    r = cabi.FrameRows(4096, 1, 4, 10, 0, 10, None, 0, 0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _refused(rc, text):
    assert rc == -1 and text.encode() in cabi.lib().kd_last_error(), cabi.lib().kd_last_error()


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=3), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=2**24 + 1), "vocab"), (dict(batch=-1), "rows"),
    (dict(steps=2**31), "2^31"), (dict(batch=2**20, steps=2**20), "2^31"), (dict(row_stride=-1), "stride"),
    (dict(logits=None), "logits"), (dict(logits=4098), "aligned"), (dict(device=-1), "device"),
    (dict(steps=2**24, vocab=2**20), "too large"), (dict(steps=2**28, vocab=4), "too large"),
])
def test_rows_that_the_entries_refuse(bad, text):
    L, r = cabi.lib(), C.byref(_rows(**bad))
    one = 4096
    t = cabi.TeacherRows(one, one, 1, 4, 0)
    _refused(L.kd_token_scores(r, None, 0, 0, None, one, one, None, None, None, 0, None), text)
    _refused(L.kd_token_scores_grad(r, None, 0, one, one, None, None, one, 0, 10, None), text)
    _refused(L.kd_distill_loss(r, C.byref(t), None, 1.0, one, None, None, None, 0, 0, None, 0, None), text)
    assert L.kd_token_scores_workspace(r, 0) == 0 and L.kd_distill_loss_workspace(r, 1) == 0


def test_arguments_that_the_entries_refuse():
    L, r, one = cabi.lib(), C.byref(_rows()), 4096
    _refused(L.kd_token_scores(None, None, 0, 0, None, one, one, None, None, None, 0, None), "rows")
    _refused(L.kd_token_scores(r, None, 0, 65, None, one, one, one, one, None, 0, None), "top")
    _refused(L.kd_token_scores(r, None, 0, -1, None, one, one, one, one, None, 0, None), "top")
    _refused(L.kd_token_scores(r, one, 2, 0, one, one, one, None, None, None, 0, None), "token_bytes")
    _refused(L.kd_token_scores(r, one, 4, 0, None, one, one, None, None, None, 0, None), "output")
    _refused(L.kd_token_scores(r, None, 0, 2, None, one, one, None, one, None, 0, None), "output")
    _refused(L.kd_token_scores(r, None, 0, 0, None, None, one, None, None, None, 0, None), "output")
    _refused(L.kd_token_scores_grad(r, None, 0, None, one, None, one, one, 0, 10, None), "stats")
    _refused(L.kd_token_scores_grad(r, None, 0, one, None, None, one, one, 0, 10, None), "entropy")
    _refused(L.kd_token_scores_grad(r, None, 0, one, one, None, one, None, 0, 10, None), "grad")
    _refused(L.kd_token_scores_grad(r, None, 0, one, one, None, one, one, 0, 9, None), "overlap")
    _refused(L.kd_token_scores_grad(r, None, 0, one, one, None, one, 4098, 0, 10, None), "aligned")
    two = C.byref(_rows(batch=2, batch_stride=40))
    for strides in ((30, 10), (0, 10), (10, 10), (39, 10), (10, 19)):
        _refused(L.kd_token_scores_grad(two, None, 0, one, one, None, one, one, *strides, None), "overlap")
    long_ = C.byref(_rows(vocab=2**20, row_stride=2**20))
    need = L.kd_token_scores_workspace(long_, 8)
    assert need > 0 and L.kd_token_scores_workspace(r, 8) == 0
    _refused(L.kd_token_scores(long_, None, 0, 8, None, one, one, one, one, one, need - 1, None), "workspace")
    _refused(L.kd_token_scores(long_, None, 0, 8, None, one, one, one, one, None, need, None), "workspace")
    _refused(L.kd_token_scores(long_, None, 0, 8, None, one, one, one, one, one + 4, need, None), "workspace")

    def distill(rows=r, t=(one, one, 4, 4, 0), temperature=1.0, loss=one, stats=None, grad=None, ws=None, n=0):
        t = C.byref(cabi.TeacherRows(*t))
        return L.kd_distill_loss(rows, t, None, temperature, loss, stats, None, grad, 0, 10, ws, n, None)
    _refused(L.kd_distill_loss(r, None, None, 1.0, one, None, None, None, 0, 0, None, 0, None), "teacher")
    _refused(distill(t=(one, one, 0, 4, 0)), "between 1 and 256")
    _refused(distill(t=(one, one, 257, 4, 0)), "between 1 and 256")
    _refused(distill(t=(one, one, 4, 2, 0)), "id_bytes")
    _refused(distill(t=(one, one, 4, 4, 5)), "teacher's logits")
    _refused(distill(t=(None, one, 4, 4, 0)), "teacher's list")
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-39):
        _refused(distill(temperature=temperature), "temperature")
    _refused(distill(loss=None), "neither")
    _refused(distill(loss=None, grad=one), "stats")
    _refused(distill(rows=long_), "workspace")
    # no rows: nothing to do, and no GPU needed
    none = C.byref(_rows(steps=0, logits=None))
    assert L.kd_token_scores(none, None, 0, 3, None, None, None, None, None, None, 0, None) == 0
    assert L.kd_token_scores_grad(none, None, 0, None, None, None, None, None, 0, 0, None) == 0
    assert distill(rows=none) == 0


def test_only_cuda_tensors():
    x = torch.zeros(3, 5)
    for call in (lambda: frames.token_scores(x), lambda: frames.token_scores(x.requires_grad_()),
                 lambda: frames.distill_loss(x, torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 1)),
                 lambda: frames.token_scores(x.detach().double()), lambda: frames.token_scores([1.0])):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


def test_the_oracle_against_autograd():
    torch.manual_seed(0)
    x = (torch.randn(17, dtype=torch.float64) * 3).requires_grad_()
    lp = torch.log_softmax(x, -1)
    h = -(lp.exp() * lp).sum()
    (0.7 * lp[4] - 0.3 * h).backward()
    (logp, ent, _, alts), _ = frames_ref.row_scores(x.detach(), 4, 3)
    assert abs(logp - lp[4].item()) < 1e-12 and abs(ent - h.item()) < 1e-12
    assert [a for a, _ in alts] == torch.topk(lp, 3).indices.tolist()
    g, _ = frames_ref.row_scores_grad(x.detach(), 4, 0.7, -0.3)
    assert torch.allclose(g, x.grad, atol=1e-12)
    x.grad = None
    ids, u = [3, -1, 9, 3, 16], torch.randn(5, dtype=torch.float64)
    q = torch.softmax(u[[0, 2, 3, 4]] / 2, -1)
    lp = torch.log_softmax(x / 2, -1)[[3, 9, 3, 16]]
    loss = 1.5 * (q * (q.log() - lp)).sum()
    loss.backward()
    (ref, g), _ = frames_ref.row_distill(x.detach(), ids, u.tolist(), 1.5, 2.0)
    assert abs(ref - loss.item()) < 1e-12 and torch.allclose(g, x.grad, atol=1e-12)

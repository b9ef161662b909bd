"""kaldi_decoder.frames on the GPU at values, lengths and layouts that its documentation allows and that
only unusual batches have; against the definition in 64 bits (frames_ref.py) where there is a value."""

import pytest
import torch

import frames_ref

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")


@pytest.fixture(scope="module")
def frames():
    from kaldi_decoder import frames as f
    return f


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("slots", [2, 40, 200])
@pytest.mark.parametrize("v", [40, 500, 3000, 9000, 20000, 70000])
def test_small_weights_beside_ruled_out_tokens(frames, v, slots, dtype):
    """A listed token that the student has at -inf: the loss is infinite however small the teacher's
    probability times the weight is; at the type's lowest value it is what the formula says."""
    dt = DTYPES[dtype]
    rows = [(95.0, 1 / 32000), (88.0, 1e-9), (60.0, 1e-20), (60.0, -1e-20), (30.0, 0.5)]
    g = torch.Generator().manual_seed(v)
    x = torch.randn(2 * len(rows), v, generator=g).to(dt)
    ids = torch.full((len(x), slots), -1, dtype=torch.int32)
    ids[:, 0], ids[:, -1] = 1, 3
    u = torch.zeros(len(x), slots)
    w = torch.tensor([a[1] for a in rows] * 2)
    for r in range(len(x)):
        u[r, -1] = -rows[r % len(rows)][0]
        x[r, 3] = -INF if r < len(rows) else torch.finfo(dt).min
    for t in (1.0, 4.0):
        args = (ids.cuda(), (u * t).cuda(), w.cuda(), t)
        leaf = x.cuda().requires_grad_()
        later = frames.distill_loss(leaf, *args)
        later.sum().backward()
        both, grad = frames.distill_loss_and_grad(leaf.detach(), *args)
        assert torch.isfinite(grad).all() and torch.isfinite(leaf.grad).all()
        for r in range(len(x)):
            (ref, _), (tol, _) = frames_ref.row_distill(x[r], ids[r].tolist(), (u[r] * t).double().tolist(), w[r].item(), t)
            for got in (both, later.detach()):
                if r < len(rows):
                    assert got[r].item() == (INF if w[r] > 0 else -INF), (r, t, got[r].item())
                elif rows[r - len(rows)][0] <= 60:  # (further down q is below 2^-126 and has few bits)
                    # (the slots' terms are rounded once each: the bound's own u |ref|, twice)
                    assert abs(got[r].item() - ref) <= tol + 2 * frames_ref.U * abs(ref), (r, t, got[r].item(), ref)

"""kaldi_decoder.frames without a GPU: calls that are refused on the host, before anything is launched."""
import ctypes as C
import random

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd

from kaldi_decoder import cabi, frames


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


# ---- a gradient's place beside the logits' --------------------------------------------------------
# Host checks alone: long rows without the workspace that they need, so that a call which passes the checks of
# the gradient's place ends at the next one.

V = 40000  # (segments of a row: a workspace)


def _place(x, out, batch, steps, x_strides, out_strides, vocab=V, **reads):
    """"overlap", "across ..." or "" for a gradient at address `out` of logits at address `x`."""
    rows = cabi.FrameRows(x, batch, steps, vocab, *x_strides, reads.get("lengths"), 0, 0)
    far = 1 << 50
    teacher = cabi.TeacherRows(reads.get("ids", far), reads.get("logits", far), 3, 8, 2)
    assert cabi.lib().kd_distill_loss_workspace(C.byref(rows), 1) > 0
    rc = cabi.lib().kd_distill_loss(C.byref(rows), C.byref(teacher), reads.get("weights"), 1.0, reads.get("loss", far),
                                    reads.get("stats"), reads.get("upstream"), out, *out_strides, None, 0, None)
    text = cabi.lib().kd_last_error().decode()
    assert rc == -1
    return "" if "workspace" in text else text


def test_gradients_that_lie_across_the_logits():
    at, e = 1 << 40, 4
    one, two = (1, 6), (3, 6)
    wide = (0, V + 50)
    across = lambda *a, **k: "across" in _place(*a, **k)
    for off in (e, 40 * e, (V + 50) * e, -(V + 50) * e, (V + 49) * e, -e, 5 * (V + 50) * e, (5 * (V + 50) + V - 1) * e):
        assert across(at, at + off, *one, wide, wide), off  # padded rows, shifted by columns or whole rows
    for off in (6 * (V + 50) * e, -6 * (V + 50) * e, 5 * (V + 50) * e + V * e):
        assert not _place(at, at + off, *one, wide, wide), off
    assert not _place(at, at, *one, wide, wide)  # the logits themselves
    assert not _place(at, at, 1, 1, (7, 9), (5, 3))  # (strides that are never taken)
    assert not _place(at, at, 1, 6, (7, V), (5, V)) and not _place(at, at, 6, 1, (V, 7), (V, 5))
    assert across(at, at, *one, wide, (0, V + 51)) and across(at, at, *one, (0, 0), wide)
    assert across(at, at + 2 * e, *one, (0, 3), wide)
    # side by side in one tensor, by columns and by batch entries
    double = (0, 2 * V)
    for off in (V, -V, 11 * V):
        assert not _place(at, at + off * e, *one, double, double), off
    for off in (V - 1, 1 - V, V + 1, 2 * V, 9 * V - 1, 10 * V + 1):
        assert across(at, at + off * e, *one, double, double), off
    s3 = (14 * V, V)  # [3, 2, 7, V]: entry 0 or 1, steps of 6 of its 7
    for off in (7 * V, -7 * V, 6 * V, -6 * V, 8 * V, 21 * V, -21 * V, 34 * V, 52 * V):
        assert not _place(at, at + off * e, *two, s3, s3), off
    for off in (V, 5 * V, 9 * V, 14 * V, 28 * V, 28 * V + 5 * V, -28 * V, 13 * V, 6 * V - 1, -V):
        assert across(at, at + off * e, *two, s3, s3), off
    # [T, B, V] storage: the strides the other way round, and of both orders
    tb = (V + 8, 3 * (V + 8))
    assert not _place(at, at, *two, tb, tb) and across(at, at + (V + 8) * e, *two, tb, tb)
    assert across(at, at, *two, tb, (6 * (V + 8), V + 8))
    assert not _place(at, at + V * e, 3, 6, (2 * V, 6 * V), (2 * V, 6 * V))
    assert not _place(at, at + V * e, *two, (2 * V, 6 * V), (12 * V, 2 * V))
    # rows of other strides within each other's span, apart and not
    assert not _place(at, at + V * e, *one, double, (0, 4 * V)) and across(at, at + (V + 1) * e, *one, double, (0, 4 * V))
    assert not _place(at, at + V * e, *one, (0, 4 * V), double) and across(at, at + 4 * V * e, *one, (0, 4 * V), double)
    assert "overlap" in _place(at, 1 << 45, *one, wide, (0, V - 1))


def test_gradients_against_every_place():
    """The rules of strides against sets of elements, over small layouts."""
    rng, seen = random.Random(0), {True: 0, False: 0}
    k = V // 2  # elements that are in the same place or not: all sizes are multiples
    for _ in range(4000):
        batch, steps, width = rng.randint(1, 3), rng.randint(1, 3), rng.choice([2, 4])
        strides = [(rng.randint(0, 24), rng.randint(0, 24)) for _ in range(2)]
        if rng.random() < 0.5:
            strides[0] = strides[1]
        off = rng.randint(-40, 40)

        def cells(at, s):
            rows = [at + b * s[0] + t * s[1] for b in range(batch) for t in range(steps)]
            return [range(r, r + width) for r in rows]
        x, g = cells(0, strides[0]), cells(off, strides[1])
        inner = [i for r in g for i in r]
        got = _place(1 << 40, (1 << 40) + 4 * off * k, batch, steps, [s * k for s in strides[0]],
                     [s * k for s in strides[1]], width * k)
        if len(set(inner)) < len(inner):
            assert "overlap" in got
        elif "overlap" in got:  # (rows of one step between those of another: apart, but refused as before)
            assert batch > 1 and steps > 1
        else:
            want = bool(set(inner) & {i for r in x for i in r}) and [r.start for r in x] != [r.start for r in g]
            assert ("across" in got) == want, (batch, steps, width, strides, off, got)
            seen[want] += 1
    assert min(seen.values()) > 300, seen


def test_gradients_that_lie_across_other_inputs():
    at, g, s = 1 << 40, 1 << 41, (9 * V, V + 8)  # (rows of V columns and 8 more; 4 steps)
    row = (V + 8) * 4
    for name, size in (("lengths", 2 * 4), ("weights", 8 * 4), ("loss", 8 * 4), ("stats", 8 * 8), ("upstream", 8 * 4),
                       ("ids", 8 * 24), ("logits", 8 * 6)):
        for off in (0, -size + 2, row - 2, 3 * row + V * 4 - 4, 9 * V * 4 + 3 * row + V * 4 - 4, 9 * V * 4 - size + 4):
            assert "across" in _place(at, g, 2, 4, s, s, **{name: g + off}), (name, off)
        for off in (-size, 3 * row + V * 4, 9 * V * 4 - size, 9 * V * 4 + 3 * row + V * 4):
            assert not _place(at, g, 2, 4, s, s, **{name: g + off}), (name, off)
    rows = cabi.FrameRows(at, 2, 4, 10, 40, 10, None, 0, 0)
    for i in range(5):
        args = [1 << 50] * 5
        args[i] = g + 316
        rc = cabi.lib().kd_token_scores_grad(C.byref(rows), args[0], 4, *args[1:], g, 40, 10, None)
        assert rc == -1 and b"across" in cabi.lib().kd_last_error(), i


@pytest.mark.parametrize("vocab,most", [(4, 2 ** 28 - 16), (512, 2 ** 28 - 16), (2048, 2 ** 26 - 4), (8192, 2 ** 24 - 1)])
def test_the_largest_grid(vocab, most):
    """Rows of 16, 64 and 256 threads each: the last workgroup counts whole.  (Outputs that are missing end
    the calls that are not too large.)"""
    L, one = cabi.lib(), 4096
    teacher = C.byref(cabi.TeacherRows(one, one, 3, 4, 0))
    for rows, text in ((most, b""), (most + 1, b"too large")):
        r = C.byref(cabi.FrameRows(one, 1, rows, vocab, 0, vocab, None, 0, 0))
        for call, missing in (
                (lambda: L.kd_token_scores(r, None, 0, 0, None, None, None, None, None, None, 0, None), b"output"),
                (lambda: L.kd_token_scores_grad(r, None, 0, None, None, None, None, one, 0, vocab, None), b"stats"),
                (lambda: L.kd_distill_loss(r, teacher, None, 1.0, None, None, None, None, 0, 0, None, 0, None),
                 b"neither")):
            assert call() == -1 and (text or missing) in L.kd_last_error(), (rows, L.kd_last_error())


def test_best_path_through_columns_that_the_logits_do_not_have():
    class Decoded:  # (a batch of one utterance, decoded over wider rows)
        batch = 1

        def best_paths(self, use_final_probs):
            il = np.array([2, 0, 5, 1], np.int32)
            return [cabi.Path(True, il, il, il, np.zeros(4, np.float32), np.zeros(4, np.float32), (0.0, 0.0))]
    with pytest.raises(ValueError, match="column 4"):
        cabi.Batch.best_path_scores(Decoded(), torch.zeros(1, 3, 4))
    with pytest.raises(ValueError, match="3 frames"):
        cabi.Batch.best_path_scores(Decoded(), torch.zeros(1, 2, 9))
    with pytest.raises(ValueError, match="CUDA tensor"):  # (five columns are enough: the next refusal)
        cabi.Batch.best_path_scores(Decoded(), torch.zeros(1, 3, 5))


def test_a_gradient_over_the_transposed_logits():
    """As many steps as utterances: the same places, but each row's another row's."""
    at = 1 << 40
    for n in (2, 3):
        for a, b in (((n * V, V), (V, n * V)), ((V, n * V), (n * V, V)), ((V + 8, 5 * (V + 8)), (5 * (V + 8), V + 8))):
            assert "across the logits" in _place(at, at, n, n, a, b)
            assert not _place(at, at, n, n, a, a) and not _place(at, at, n, n, b, b)
    assert not _place(at, at, 1, 1, (V, 3 * V), (3 * V, V))
    assert not _place(at, at, 4, 1, (V, 9), (V, 7)) and not _place(at, at, 1, 4, (9, V), (7, V))

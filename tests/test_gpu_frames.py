"""kaldi_decoder.frames on the GPU against the definition in 64 bits (frames_ref.py: the bounds are
derived there), at the sizes, types, strides and masks where the kernels change their ways: a wave's
rows (8 KiB), a workgroup's (32 KiB), rows cut into segments; rows that a mask leaves empty."""
import math

import numpy as np
import pytest
import torch

import frames_ref
from frames_ref import half_step

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")


@pytest.fixture(scope="module")
def frames():
    from kaldi_decoder import frames as f
    return f


def _logits(n, v, dtype, seed, pad=0):
    """Rows of many kinds: plain, peaked, equal, partly and wholly masked."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, v, generator=g) * 3
    lowest = torch.finfo(dtype).min
    for r in range(n):
        kind = r % 8
        if kind == 1:
            x[r, torch.randint(v, (1,), generator=g)] += 20
        elif kind == 2:
            x[r] = 0.5                                    # all equal: ties everywhere
        elif kind == 3:
            x[r, torch.rand(v, generator=g) < 0.6] = -INF
        elif kind == 4:
            x[r, torch.rand(v, generator=g) < 0.6] = lowest
        elif kind == 5:
            x[r] = -INF                                   # empty
            if r >= 8:
                x[r, torch.randint(v, (3,), generator=g)] = 1.0  # all but empty
        elif kind == 6:
            x[r] = lowest if r < 8 else torch.randint(-2, 3, (v,), generator=g).float() * 0.0  # -0 and 0
            if r >= 8:
                x[r, torch.rand(v, generator=g) < 0.5] *= -1
        elif kind == 7:
            x[r] = torch.randint(0, 4, (v,), generator=g).float() + 100  # few values, far from 0
    x = x.to(dtype)
    wide = torch.full((n, v + pad), 7.0, dtype=dtype, device="cuda")
    wide[:, :v] = x.cuda()
    return x, wide[:, :v]


def _close(got, want, tol):
    # (float32 ends at (2 - 2^-23) 2^127: what is further out by half a step or more rounds to infinity --
    # 1.05 times float32's lowest value as a log-probability, weighted by 1.05 or more, is such a loss)
    if abs(want) >= (2 - 2.0 ** -24) * 2.0 ** 127:
        want = math.copysign(INF, want)
    if math.isnan(want) or math.isinf(want):
        return (math.isnan(want) and math.isnan(got)) or got == want
    return abs(got - want) <= tol


def _check_scores(sc, x, tokens, top, valid=None):
    ref = {k: (None if t is None else t.detach().cpu().reshape(x.shape[0], -1)) for k, t in sc._asdict().items()}
    for r in range(x.shape[0]):
        tok = int(tokens[r]) if tokens is not None else -1
        if valid is not None and not valid[r]:
            assert ref["entropy"][r, 0] == 0 and ref["stats"][r].tolist() == [0, 0]
            assert tokens is None or ref["logp"][r, 0] == 0
            assert not top or (ref["top_ids"][r].eq(-1).all() and ref["top_logp"][r].eq(-INF).all())
            continue
        (logp, ent, (m, s), alts), (tol_l, tol_h, tol_s, tol_a) = frames_ref.row_scores(x[r], tok, top)
        assert _close(ref["entropy"][r, 0].item(), ent, tol_h), (r, ref["entropy"][r, 0].item(), ent, tol_h)
        assert ref["stats"][r, 0].item() == m or math.isnan(s), (r, m)
        assert _close(ref["stats"][r, 1].item(), s, tol_s), (r, ref["stats"][r, 1].item(), s, tol_s)
        if tokens is not None:
            assert _close(ref["logp"][r, 0].item(), logp, tol_l), (r, ref["logp"][r, 0].item(), logp, tol_l)
        if top:
            assert ref["top_ids"][r].tolist() == [a for a, _ in alts], (r, ref["top_ids"][r].tolist(), alts)
            for k in range(top):
                assert _close(ref["top_logp"][r, k].item(), alts[k][1], tol_a[k]), (r, k)


SIZES = [1, 2, 3, 4, 5, 7, 8, 9, 63, 64, 65, 255, 500, 501, 513, 2047, 2048, 2049, 4095, 4096, 4097, 8192, 8193, 16384,
         16385, 20001, 65537]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("v", SIZES)
def test_token_scores(frames, dtype, v):
    top = [1, 8, 16, 17, 64, 5, 0][SIZES.index(v) % 7]
    n = 18 if v < 5000 else 9
    x, dev = _logits(n, v, DTYPES[dtype], v, pad=[0, 1, 3, 8][v % 4])
    g = torch.Generator().manual_seed(v)
    tokens = torch.randint(0, v, (n,), generator=g, dtype=torch.int64 if v % 2 else torch.int32)
    tokens[n // 2] = -1
    tokens[n // 2 + 1] = v
    _check_scores(frames.token_scores(dev, tokens.cuda(), top=top), x, tokens, top)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("top", [1, 2, 15, 16, 17, 33, 63, 64])
@pytest.mark.parametrize("v", [40, 500, 3000, 9000, 40000])
def test_alternatives(frames, dtype, top, v):
    x, dev = _logits(16, v, DTYPES[dtype], top, pad=top % 2)
    _check_scores(frames.token_scores(dev, top=top), x, None, top)


def test_alternatives_in_one_lane_or_segment(frames):
    """All the large values where one lane, one chunk, one segment holds them; sorted rows."""
    for v in (400, 2000, 9000, 70000):
        x = torch.stack([torch.arange(v).float() / 64, -torch.arange(v).float() / 64, torch.zeros(v), torch.zeros(v),
                         (torch.arange(v) // 97).float()])
        x[2, v // 2: v // 2 + 64] = torch.arange(64).float()
        x[3, ::256] = 1 + (torch.arange(v)[::256] % 5).float()
        _check_scores(frames.token_scores(x.cuda(), top=64), x, None, 64)


def test_nan_and_inf(frames):
    for v in (100, 9000, 30000):
        x = torch.randn(4, v)
        x[0, v // 3], x[1, v // 2], x[2, 5], x[2, 9] = float("nan"), INF, INF, -INF
        tokens = torch.tensor([0, 1, 5, 3], dtype=torch.int32)
        sc = frames.token_scores(x.cuda(), tokens.cuda(), top=4)
        for r in range(3):
            assert torch.isnan(sc.logp[r]) and torch.isnan(sc.entropy[r])
            assert sc.top_ids[r].eq(-1).all() and torch.isnan(sc.top_logp[r]).all()
        _check_scores(frames.TokenScores(*(t[3:] for t in sc)), x[3:], tokens[3:], 4)
        g = frames.token_scores_grad(x.cuda(), sc, tokens.cuda(), None, torch.ones(4).cuda())
        assert torch.isnan(g[:3]).all() and torch.isfinite(g[3]).all()
        ids = torch.tensor([[0, 1]] * 4, dtype=torch.int32).cuda()
        t = torch.randn(4, 2)
        loss, g = frames.distill_loss_and_grad(x.cuda(), ids, t.cuda())
        assert torch.isnan(loss[:3]).all() and torch.isfinite(loss[3]) and torch.isnan(g[:3]).all()
        x = torch.randn(3, v)
        t = torch.tensor([[float("nan"), 0.0], [INF, 0.0], [-INF, 1.0]])
        loss, g = frames.distill_loss_and_grad(x.cuda(), ids[:3], t.cuda())
        assert torch.isnan(loss[:2]).all() and torch.isnan(g[:2, :2]).all() and torch.isfinite(g[:, 2:]).all()
        (ref, gr), (tol, tol_g) = frames_ref.row_distill(x[2], [0, 1], t[2].tolist(), 1.0, 1.0)
        assert abs(loss[2].item() - ref) <= tol and ((g[2].cpu().double() - gr).abs() <= tol_g + 2**-24 * gr.abs()).all()


def _padded(b, t, v, dtype, seed, order):
    """[B, T, V] over storage in another order, with lengths 0 .. T."""
    x, _ = _logits(b * t, v, dtype, seed)
    x = x.reshape(b, t, v)
    if order == "tbv":
        dev = x.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    elif order == "wide":
        dev = torch.empty(b + 1, t + 2, v + 5, dtype=dtype, device="cuda").fill_(float("nan"))[1:, 1:-1, 3:-2]
        dev.copy_(x)
    else:
        dev = x.cuda()
    lengths = torch.arange(b) * t // max(1, b - 1)
    return x, dev, lengths


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("order", ["plain", "tbv", "wide"])
@pytest.mark.parametrize("v", [33, 500, 5001, 33001])
def test_padded_batches(frames, dtype, order, v):
    b, t = 4, 5
    x, dev, lengths = _padded(b, t, v, DTYPES[dtype], v, order)
    tokens = (torch.arange(b * t) * 7 % v).reshape(b, t).to(torch.int32)
    valid = (torch.arange(t) < lengths[:, None]).reshape(-1).tolist()
    flat = x.reshape(b * t, v)
    for given in (None, lengths.cuda(), lengths.to(torch.int32).tolist(), lengths.numpy()):
        sc = frames.token_scores(dev, tokens.cuda(), top=6, lengths=given)
        assert sc.top_ids.shape == (b, t, 6) and sc.stats.shape == (b, t, 2) and sc.logp.shape == (b, t)
        _check_scores(sc, flat, tokens.reshape(-1), 6, None if given is None else valid)
    # the gradients of rows behind the lengths are zeros; those of the others as if alone
    up = torch.randn(b, t).cuda()
    g = frames.token_scores_grad(dev, sc, tokens.cuda(), lengths.cuda(), up, up)
    one = frames.token_scores_grad(dev.reshape(b * t, v), frames.token_scores(dev.reshape(b * t, v), tokens.reshape(-1).cuda()),
                                   tokens.reshape(-1).cuda(), None, up.reshape(-1), up.reshape(-1)).reshape(b, t, v)
    keep = torch.tensor(valid).reshape(b, t, 1).cuda()
    assert torch.equal(g, torch.where(keep, one, torch.zeros_like(one)))
    ids = (torch.arange(b * t * 3).reshape(b, t, 3) * 5 % v).to(torch.int32).cuda()
    u = torch.randn(b, t, 3).cuda()
    loss, g = frames.distill_loss_and_grad(dev, ids, u, None, 2.0, lengths)
    loss1, one = frames.distill_loss_and_grad(dev.reshape(b * t, v), ids.reshape(-1, 3), u.reshape(-1, 3), None, 2.0)
    keep2 = keep.squeeze(-1)
    assert torch.equal(loss, torch.where(keep2, loss1.reshape(b, t), torch.zeros_like(loss)))
    assert torch.equal(g, torch.where(keep, one.reshape(b, t, v), torch.zeros_like(g)))


def test_strides_of_the_gradient(frames):
    """`out` in any layout whose rows do not overlap; what lies between its rows is left alone."""
    for v in (50, 6000, 20000):
        x = torch.randn(3, 4, v).cuda()
        tokens = torch.randint(0, v, (3, 4)).cuda()
        sc = frames.token_scores(x, tokens)
        up = torch.randn(3, 4).cuda()
        ids, u = torch.randint(0, v, (3, 4, 5)).cuda(), torch.randn(3, 4, 5).cuda()
        want = frames.token_scores_grad(x, sc, tokens, None, up, up)
        _, want2 = frames.distill_loss_and_grad(x, ids, u)
        for make in (lambda: torch.full((4, 3, v), 9.0).cuda().transpose(0, 1),
                     lambda: torch.full((4, 6, v + 3), 9.0).cuda()[:3, 1:5, 2:-1],
                     lambda: torch.full((3, 9, v), 9.0).cuda()[:, :8:2]):
            out = make()
            got = frames.token_scores_grad(x, sc, tokens, None, up, up, out=out)
            assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
            base = out._base
            out.fill_(9.0)
            assert base.eq(9.0).all()  # (nothing around it was written)
            frames.distill_loss_and_grad(x, ids, u, out=out)
            assert torch.equal(out, want2)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("v", [1, 2, 7, 64, 500, 501, 2049, 4097, 8193, 16385, 40001])
def test_token_scores_gradient(frames, dtype, v):
    dt = DTYPES[dtype]
    x, dev = _logits(16, v, dt, v + 1, pad=v % 3)
    g = torch.Generator().manual_seed(v)
    tokens = torch.randint(0, v, (16,), generator=g)
    tokens[9] = -1
    up, uh = torch.randn(16, generator=g), torch.randn(16, generator=g)
    leaf = dev.detach().requires_grad_()
    sc = frames.token_scores(leaf, tokens.cuda())
    got = []
    for outs, ups in (((sc.logp, sc.entropy), (up.cuda(), uh.cuda())), ((sc.logp,), (up.cuda(),)),
                      ((sc.entropy,), (uh.cuda(),))):
        got.append(torch.autograd.grad(outs, (leaf,), ups, retain_graph=True)[0].cpu())
    hand = frames.token_scores_grad(dev, sc, tokens.cuda(), None, up.cuda(), uh.cuda()).cpu()
    assert torch.equal(hand, got[0])
    for which, (a, b) in enumerate(((1, 1), (1, 0), (0, 1))):
        for r in range(16):
            ref, tol = frames_ref.row_scores_grad(x[r], int(tokens[r]), a * up[r].item(), b * uh[r].item())
            tol = tol + half_step(dt) * (ref.abs() + tol) + (2.0 ** -25 if dt == torch.float16 else 0)
            off = (got[which][r].double() - ref).abs()
            assert (off <= tol).all(), (which, r, off.max(), (off - tol).argmax())


@pytest.mark.parametrize("tdtype", list(DTYPES))
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("v,k,t", [(1, 1, 1.0), (5, 3, 2.0), (64, 64, 1.0), (500, 8, 2.0), (501, 65, 0.5), (2049, 13, 4.0),
                                   (4097, 200, 1.0), (9000, 256, 2.0), (20001, 64, 1.0), (66000, 100, 3.0)])
def test_distillation(frames, dtype, tdtype, v, k, t):
    dt = DTYPES[dtype]
    n = 18
    x, dev = _logits(n, v, dt, v + k, pad=v % 3)
    g = torch.Generator().manual_seed(v + k)
    ids = torch.stack([torch.randperm(max(v, k), generator=g)[:k] % v for _ in range(n)])
    ids = ids.to(torch.int64 if k % 2 else torch.int32)
    u = (torch.randn(n, k, generator=g) * 2 - 3).to(DTYPES[tdtype])
    if k > 2:
        ids[1, 1] = ids[1, 0]               # listed twice
        ids[2, :2] = torch.tensor([-1, v])  # empty slots
        u[9, 1] = -INF
        ids[10] = ids[10, 0]                # one token in every slot
    if k > 1:
        ids[3, 1:] = -1
    ids[8] = -7                             # no slot filled
    w = torch.rand(n, generator=g) + 0.5
    w[11] = 0
    w[12] = -1.0
    args = (ids.cuda(), u.cuda(), w.cuda(), t)
    loss, grad = frames.distill_loss_and_grad(dev, *args)
    alone = frames.distill_loss(dev, *args)
    leaf = dev.detach().requires_grad_()
    up = torch.randn(n, generator=g)
    later = frames.distill_loss(leaf, *args)
    grad2, = torch.autograd.grad((later,), (leaf,), (up.cuda(),))
    assert torch.equal(alone.nan_to_num(-5), later.detach().nan_to_num(-5))
    loss, alone, grad, grad2 = loss.cpu(), alone.cpu(), grad.cpu(), grad2.cpu()
    for r in range(n):
        for got, scale in ((grad, 1.0), (grad2, up[r].item())):
            (ref, gr), (tol, tol_g) = frames_ref.row_distill(x[r], ids[r].tolist(), u[r].double().tolist(), w[r].item(), t,
                                                             scale)
            # (the loss alone may deal a row out in another way than loss and gradient: each by its own bound)
            for one in (loss, alone):
                assert _close(one[r].item(), ref, tol + frames_ref.U * abs(ref) if abs(ref) < INF else 0), (r, one[r].item(), ref, tol)
            tol_g = tol_g + half_step(dt) * (gr.abs() + tol_g) + (2.0 ** -25 if dt == torch.float16 else 0)
            off = (got[r].double() - gr).abs()
            assert (off <= tol_g).all(), (r, off.max(), (off - tol_g).argmax())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("v", [64, 500, 5000, 9000, 16385, 70000])
def test_gradient_over_the_logits(frames, dtype, v):
    """`out` = the logits: the slots' logits are read before any lane writes."""
    x = (torch.randn(40, v) * 3).to(DTYPES[dtype]).cuda()
    ids = torch.stack([torch.randperm(v)[:64] for _ in range(40)]).cuda()
    u, tokens, up = torch.randn(40, 64).cuda(), ids[:, 0].contiguous(), torch.randn(40).cuda()
    loss, want = frames.distill_loss_and_grad(x, ids, u)
    mine = x.clone()
    loss2, got = frames.distill_loss_and_grad(mine, ids, u, out=mine)
    assert got.data_ptr() == mine.data_ptr() and torch.equal(mine, want) and torch.equal(loss, loss2)
    sc = frames.token_scores(x, tokens)
    want = frames.token_scores_grad(x, sc, tokens, None, up, up)
    mine = x.clone()
    frames.token_scores_grad(mine, sc, tokens, None, up, up, out=mine)
    assert torch.equal(mine, want)


@pytest.mark.parametrize("dtype,n,v", [("f32", 40, 20001), ("bf16", 33, 65536), ("f16", 32, 40003), ("f32", 130, 40001),
                                       ("bf16", 128, 131072), ("f16", 129, 70001)])
def test_distillation_of_many_long_rows(frames, dtype, n, v):
    """Enough rows for a workgroup of 1024 to take each whole (80 to 256 KiB): by the oracle, and next to
    the same rows a few at a time, which are cut into segments."""
    dt = DTYPES[dtype]
    x, dev = _logits(n, v, dt, v, pad=v % 2)
    g = torch.Generator().manual_seed(n)
    ids = torch.stack([torch.randperm(v, generator=g)[:40] for _ in range(n)])
    ids[1, 1], ids[3, 2], ids[9] = ids[1, 0], -1, -1
    u, w = torch.randn(n, 40, generator=g) * 2, torch.rand(n, generator=g) + 0.5
    w[10] = 0
    loss, grad = frames.distill_loss_and_grad(dev, ids.cuda(), u.cuda(), w.cuda(), 2.0)
    mine = dev.clone()
    loss2, grad2 = frames.distill_loss_and_grad(mine, ids.cuda(), u.cuda(), w.cuda(), 2.0, out=mine)
    assert torch.equal(loss, loss2) and torch.equal(grad, grad2) and grad2.data_ptr() == mine.data_ptr()
    few, few_grad = frames.distill_loss_and_grad(dev[:20], ids[:20].cuda(), u[:20].cuda(), w[:20].cuda(), 2.0)
    for r in list(range(20)) + [n - 1]:
        (ref, gr), (tol, tol_g) = frames_ref.row_distill(x[r], ids[r].tolist(), u[r].double().tolist(), w[r].item(), 2.0)
        tol_g = tol_g + half_step(dt) * (gr.abs() + tol_g) + (2.0 ** -25 if dt == torch.float16 else 0)
        for one, one_grad in ((loss, grad),) + (((few, few_grad),) if r < 20 else ()):
            assert _close(one[r].item(), ref, tol + frames_ref.U * abs(ref) if abs(ref) < INF else 0), (r, one[r].item(), ref)
            assert ((one_grad[r].cpu().double() - gr).abs() <= tol_g).all(), r


def test_many_rows_and_the_longest(frames):
    """Three million rows of four; one row of 2^24 columns, with ties at the last places."""
    x = torch.randn(3000000, 4).cuda()
    tokens = torch.randint(0, 4, (3000000,)).cuda()
    sc = frames.token_scores(x, tokens, top=2)
    lp = torch.log_softmax(x.double(), -1)
    # (four terms, |d| < 12: u (4 + 3 * 12 + 2 + 4 * 12) bounds logp, rounded up)
    tol = 100 * frames_ref.U
    assert (sc.logp - lp.gather(-1, tokens[:, None]).squeeze(-1)).abs().max() <= tol
    assert (sc.entropy + (lp.exp() * lp).sum(-1)).abs().max() <= 4 * tol
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(sc.top_ids.long(), order)
    assert (sc.top_logp - lp.gather(-1, order)).abs().max() <= tol
    v = 1 << 24
    for dt in (torch.float32, torch.bfloat16):
        x = torch.randn(1, v).to(dt)
        x[0, -1] = 9.0
        tokens = torch.tensor([v - 1])
        _check_scores(frames.token_scores(x.cuda(), tokens.cuda(), top=64), x, tokens, 64)
        ids, u = torch.tensor([[v - 1, 0, 5, v // 2]]), torch.randn(1, 4)
        loss, g = frames.distill_loss_and_grad(x.cuda(), ids.cuda(), u.cuda())
        (ref, gr), (tol, tol_g) = frames_ref.row_distill(x[0], ids[0].tolist(), u[0].double().tolist(), 1.0, 1.0)
        assert abs(loss.item() - ref) <= tol + frames_ref.U * abs(ref)
        assert ((g[0].cpu().double() - gr).abs() <= tol_g + half_step(dt) * (gr.abs() + tol_g)).all()


@pytest.mark.parametrize("v", [30, 700, 5000, 20000, 50000])
def test_autograd_of_padded_batches(frames, v):
    """Graphs over [B, T, V] with lengths from the host, without tokens, with alternatives; rows that are
    not read (behind the lengths, of weight 0) may hold anything."""
    lengths = [4, 0, 2]
    x = torch.randn(3, 4, v).cuda()
    x[0, 3] = x[2, 2:] = x[1] = float("nan")
    lengths[0] = 3
    tokens = torch.randint(0, v, (3, 4)).cuda()
    leaf = x.clone().requires_grad_()
    up = torch.randn(3, 4).cuda()
    sc = frames.token_scores(leaf, None, top=3, lengths=lengths)
    assert sc.logp is None and sc.entropy.requires_grad and not sc.top_logp.requires_grad and not sc.stats.requires_grad
    got, = torch.autograd.grad(sc.entropy, leaf, up)
    want = frames.token_scores_grad(x, frames.token_scores(x, lengths=lengths), None, torch.tensor(lengths), None, up)
    assert torch.equal(got, want) and got.isfinite().all() and got[1].eq(0).all() and got[0, :3].ne(0).any()
    sc = frames.token_scores(leaf, tokens, top=3, lengths=lengths)
    assert sc.logp[1].eq(0).all() and sc.logp.isfinite().all()
    got, = torch.autograd.grad((sc.logp * up).sum() + sc.entropy.sum(), leaf)
    want = frames.token_scores_grad(x, sc, tokens, lengths, up, torch.ones(3, 4).cuda())
    assert torch.equal(got, want)
    ids, u, w = torch.randint(0, v, (3, 4, 9)).cuda(), torch.randn(3, 4, 9).cuda(), torch.rand(3, 4).cuda()
    loss = frames.distill_loss(leaf, ids, u, w, 1.5, lengths)
    got, = torch.autograd.grad((loss * up).sum(), leaf)
    loss2, one = frames.distill_loss_and_grad(x, ids, u, w, 1.5, lengths)
    # (upstream gradients are multiplied in before the one rounding)
    assert (got - one * up[..., None]).abs().max() <= 1e-6 and loss.isfinite().all() and loss2.isfinite().all()
    skip = torch.where(torch.isnan(x).any(-1), 0.0, w.double()).float()
    loss3, three = frames.distill_loss_and_grad(x, ids, u, skip, 1.5)
    assert torch.equal(loss3, loss2) and torch.equal(three, one)


def test_a_gradient_may_not_lie_across_the_logits(frames):
    base = torch.randn(5 * 40 + 3).cuda()
    x, out = base[:200].view(5, 40), base[3:].view(5, 40)
    ids, u = torch.zeros(5, 1, dtype=torch.int32).cuda(), torch.zeros(5, 1).cuda()
    with pytest.raises(RuntimeError, match="memory location"):
        frames.distill_loss_and_grad(x, ids, u, out=out)
    wide = torch.randn(5, 80).cuda()  # (side by side in one storage: apart)
    _, want = frames.distill_loss_and_grad(wide[:, :40].clone(), ids, u)
    _, got = frames.distill_loss_and_grad(wide[:, :40], ids, u, out=wide[:, 40:])
    assert torch.equal(got, want)


def test_written_in_place_is_noticed(frames):
    """A graph that saved the logits refuses to go backward once a gradient was written over them."""
    x = torch.randn(3, 50).cuda()
    leaf = x.clone().requires_grad_()
    y = leaf * 1.0
    ids, u = torch.zeros(3, 1, dtype=torch.int32).cuda(), torch.zeros(3, 1).cuda()
    loss = frames.distill_loss(y, ids, u)
    frames.distill_loss_and_grad(y.detach(), ids, u, out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


def test_gradients_against_differences(frames):
    """Directional derivatives by central differences of the forward kernels.  Along v, |v| <= 1/2, the
    third derivative of logp is a third cumulant of v: at most 1; the entropy's a joint cumulant of
    x, v, v, v: at most 8 times the rows' range R; the loss's as logp's.  With step h the difference is
    off by h^2 / 6 of that and by the values' error / h."""
    h = 2.0 ** -4
    for v in (37, 700, 10000, 40000):
        g = torch.Generator().manual_seed(v)
        x = (torch.rand(5, v, generator=g) * 4).cuda()
        d = (torch.rand(5, v, generator=g) - 0.5).cuda()
        tokens = torch.randint(0, v, (5,), generator=g).cuda()
        leaf = x.clone().requires_grad_()
        sc = frames.token_scores(leaf, tokens)
        gl, = torch.autograd.grad(sc.logp.sum(), leaf, retain_graph=True)
        gh, = torch.autograd.grad(sc.entropy.sum(), leaf)
        a, b = frames.token_scores(x + h * d, tokens), frames.token_scores(x - h * d, tokens)
        noise = 2 * frames_ref.U * 200 * 4 / h
        assert (((a.logp - b.logp) / (2 * h) - (gl * d).sum(-1)).abs() <= h * h / 6 + noise).all()
        assert (((a.entropy - b.entropy) / (2 * h) - (gh * d).sum(-1)).abs() <= h * h / 6 * 8 * 4 + noise).all()
        ids, u = torch.randint(0, v, (5, 6), generator=g).cuda(), torch.randn(5, 6, generator=g).cuda()
        _, gd = frames.distill_loss_and_grad(x, ids, u)
        a, b = frames.distill_loss(x + h * d, ids, u), frames.distill_loss(x - h * d, ids, u)
        assert (((a - b) / (2 * h) - (gd * d).sum(-1)).abs() <= h * h / 6 + noise).all()


def test_broadcast_inputs(frames):
    """Expanded logits (stride 0) and upstream gradients that are broadcast, as .sum() makes them."""
    x = torch.randn(1, 600).cuda().requires_grad_()
    tokens = torch.arange(4).cuda()
    sc = frames.token_scores(x.expand(4, 600), tokens)
    (sc.logp.sum() + 0.5 * sc.entropy.mean()).backward()
    ref = x.detach().double().requires_grad_()
    lp = torch.log_softmax(ref, -1)
    (lp[0, :4].sum() - 0.5 * (lp.exp() * lp).sum()).backward()
    assert (x.grad.double() - ref.grad).abs().max() <= 4 * 200 * frames_ref.U
    with pytest.raises(RuntimeError):  # once differentiable
        leaf = torch.randn(2, 30).cuda().requires_grad_()
        g, = torch.autograd.grad(frames.token_scores(leaf, tokens[:2]).logp.sum(), leaf, create_graph=True)
        g.sum().backward()


def test_refusals(frames):
    x = torch.randn(2, 3, 20).cuda()
    tok = torch.zeros(2, 3, dtype=torch.int32).cuda()
    ids, u = torch.zeros(2, 3, 4, dtype=torch.int32).cuda(), torch.zeros(2, 3, 4).cuda()
    for call in (lambda: frames.token_scores(x, tok[:1]), lambda: frames.token_scores(x, tok.float()),
                 lambda: frames.token_scores(x, tok.cpu()), lambda: frames.token_scores(x, top=65),
                 lambda: frames.token_scores(x, top=-1), lambda: frames.token_scores(x[0, 0]),
                 lambda: frames.token_scores(x[..., ::2]), lambda: frames.token_scores(x[..., :0]),
                 lambda: frames.token_scores(x, lengths=[1]), lambda: frames.token_scores(x, lengths=[0.5, 1.5]),
                 lambda: frames.token_scores(x[0], lengths=[1, 2, 3]),
                 lambda: frames.distill_loss(x, ids[..., 0], u), lambda: frames.distill_loss(x, ids, u[..., :3]),
                 lambda: frames.distill_loss(x, ids, u.double()), lambda: frames.distill_loss(x, ids.float(), u),
                 lambda: frames.distill_loss(x, ids, u, tok), lambda: frames.distill_loss(x, ids, u.clone().requires_grad_()),
                 lambda: frames.distill_loss_and_grad(x, ids, u, out=x[..., :19]),
                 lambda: frames.distill_loss_and_grad(x, ids, u, out=x.half())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: frames.distill_loss(x, ids, u, None, 0.0),
                 lambda: frames.distill_loss_and_grad(x, ids, u, out=x[:1].expand(2, 3, 20))):
        with pytest.raises(RuntimeError, match="bad argument"):
            call()
    sc = frames.token_scores(x[:, :0], tok[:, :0], top=3)  # no rows
    assert sc.logp.shape == (2, 0) and sc.top_ids.shape == (2, 0, 3)
    loss, g = frames.distill_loss_and_grad(x[:0], ids[:0], u[:0])
    assert loss.shape == (0, 3) and g.shape == (0, 3, 20)


def test_side_stream_and_two_at_once(frames):
    """Calls on two streams at once, each with its own workspace."""
    xs = [torch.randn(40, 70000).cuda() for _ in range(2)]
    tokens = torch.arange(40).cuda()
    want = [frames.token_scores(x, tokens, top=9) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(frames.token_scores(xs[i], tokens, top=9))
    torch.cuda.synchronize()
    for i in range(2):
        for sc in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(sc, want[i]))


@pytest.mark.parametrize("v", [500, 9000, 70000])
def test_captured_and_replayed(frames, v):
    """Two graphs over the same inputs, replayed in turn with eager work between; new inputs in place."""
    n = 12
    x, tokens = torch.randn(n, v).cuda(), torch.randint(0, v, (n,)).cuda()
    ids, u = torch.randint(0, v, (n, 7)).cuda(), torch.randn(n, 7).cuda()
    up = torch.randn(n).cuda()

    def step():
        sc = frames.token_scores(x, tokens, top=5)
        g = frames.token_scores_grad(x, sc, tokens, None, up, up)
        loss, dx = frames.distill_loss_and_grad(x, ids, u, None, 2.0)
        return [*sc, g, loss, dx]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step())
        graphs.append(gr)
    for i in range(4):
        x.copy_(torch.randn(n, v))
        for gr in graphs:
            gr.replay()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_far_offsets(frames):
    """Rows that lie past 2^31 elements and bytes of their tensor."""
    n, v = 70000, 33000
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    rows = [0, 1, 32537, 65100, 65101, n - 1]
    x.fill_(-1.0)
    small = torch.randn(len(rows), v).to(torch.bfloat16)
    x[rows] = small.cuda()
    tokens = torch.full((n,), 17, dtype=torch.int32, device="cuda")
    sc = frames.token_scores(x, tokens, top=3)
    at = torch.tensor(rows).cuda()
    _check_scores(frames.TokenScores(*(t[at] for t in sc)), small, tokens[:len(rows)].cpu(), 3)
    # one row with a huge stride, and one call over the far half alone
    far = torch.as_strided(x, (2, v), ((n - 1) * v, 1))
    _check_scores(frames.token_scores(far, tokens[:2], top=3), small[[0, -1]], tokens[:2].cpu(), 3)
    ids = torch.arange(4, dtype=torch.int32, device="cuda").expand(2, 4).contiguous()
    u = torch.randn(2, 4).cuda()
    loss, g = frames.distill_loss_and_grad(far, ids, u, out=far.clone())
    loss2, g2 = frames.distill_loss_and_grad(small[[0, -1]].cuda(), ids, u)
    assert torch.equal(loss, loss2) and torch.equal(g, g2)
    frames.distill_loss_and_grad(far, ids, u, out=far)  # (in place)
    assert torch.equal(far, g2)


def test_teacher_student_and_decode(frames):
    """The operators as they are used together: a teacher's alternatives, the student's loss and a step
    down its gradient, a decode of the student's rows, and the scores of the best paths it returned."""
    from kaldi_decoder import cabi, synth
    V, T, B = 40, 30, 4
    g = synth.hlg_graph(V=V, n_words=200, n_hist=200, avg_succ=8, seed=4)
    teacher = torch.stack([torch.from_numpy(synth.make_logprobs(T, V, i, peak=6.0, lexicon=g["lexicon"])) for i in range(B)])
    lengths = torch.tensor([30, 17, 1, 30], dtype=torch.int32)
    alts = frames.token_scores(teacher.cuda(), top=16, lengths=lengths)
    torch.manual_seed(1)
    student = (torch.randn(B, T, V) * 0.5).cuda().requires_grad_()
    w = torch.full((B, T), 1.0 / int(lengths.sum())).cuda()
    loss = frames.distill_loss(student, alts.top_ids, alts.top_logp, w, 1.0, lengths)
    loss.sum().backward()
    loss2, grad = frames.distill_loss_and_grad(student.detach(), alts.top_ids, alts.top_logp, w, 1.0, lengths)
    assert torch.equal(loss, loss2) and torch.equal(grad, student.grad)
    for b in range(B):
        for t in (0, 16, 29):
            if t >= lengths[b]:
                assert loss[b, t] == 0 and grad[b, t].eq(0).all()
                continue
            (ref, gr), (tol, tg) = frames_ref.row_distill(student[b, t].detach().cpu(), alts.top_ids[b, t].tolist(),
                                                          alts.top_logp[b, t].double().tolist(), w[0, 0].item(), 1.0)
            assert abs(loss[b, t].item() - ref) <= tol + frames_ref.U * abs(ref)
            assert ((grad[b, t].cpu().double() - gr).abs() <= tg + frames_ref.U * gr.abs()).all()
    # the student that has the teacher's rows: decode, and score what came back
    rows = teacher.cuda()
    bt = cabi.Batch(cabi.Graph(g), max_batch=B, beam=10.0)
    bt.decode_tensor(rows, lengths)
    paths, tokens, sc = bt.best_path_scores(rows, lengths, top=3)
    assert tokens.shape == (B, T)
    for b in range(B):
        n = int(lengths[b])
        assert paths[b].ok and tokens[b, :n].cpu().tolist() == (paths[b].isyms - 1).tolist()
        assert tokens[b, n:].eq(-1).all() and sc.logp[b, n:].eq(0).all()
        # make_logprobs' rows are normalised: log p is the log-probability that the search added up
        lp = rows[b, torch.arange(n), tokens[b, :n].long()]
        assert (sc.logp[b, :n] - lp).abs().max() < 1e-5
        assert abs(-sc.logp[b, :n].double().sum().item() - paths[b].total_cost[1]) < 1e-3
    with pytest.raises(ValueError):
        bt.best_path_scores(rows[:2])
    with pytest.raises(ValueError):
        bt.best_path_scores(rows[:, :10])
    assert np.isfinite(sc.entropy.cpu().numpy()).all()

"""kaldi_decoder.frames on the GPU at values, lengths and layouts that its documentation allows and that
only unusual batches have; against the definition in 64 bits (frames_ref.py) where there is a value."""
import ctypes as C

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


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("v", [40, 500, 1000, 3000, 9000, 20000, 40000, 100000])
def test_no_probability_above_one(frames, v, dtype):
    """Rows that one token has almost to itself, at many heights: its own term makes the sum at least 1,
    so no log-probability is above 0, and no entropy or divergence below."""
    n = 200
    x = torch.full((n, v), -INF)
    x[1::2] = -1.0
    x[:, 2] = torch.linspace(-130, 130, n)
    x = x.to(DTYPES[dtype]).cuda()
    tokens = torch.full((n,), 2, dtype=torch.int32).cuda()
    for top in (0, 3, 40):
        sc = frames.token_scores(x, tokens, top=top)
        assert (sc.stats[:, 1] >= 1).all() and (sc.entropy >= 0).all() and (sc.logp <= 0).all()
        assert not top or (sc.top_logp <= 0).all()
    for t in (1.0, 0.7, 3.0):
        loss, _ = frames.distill_loss_and_grad(x, tokens[:, None], torch.zeros(n, 1).cuda(), None, t)
        alone = frames.distill_loss(x, tokens[:, None], torch.zeros(n, 1).cuda(), None, t)
        assert (loss >= 0).all() and (alone >= 0).all()
    # rows without a finite value, and rows with NaN, are what they were
    x[0], x[1, 0] = -INF, float("nan")
    sc = frames.token_scores(x, tokens)
    assert sc.stats[0].tolist() == [-INF, 0] and sc.entropy[0] == 0 and torch.isnan(sc.stats[1, 1])


def test_factors_of_the_gradient(frames):
    """weight * upstream / temperature, where the product of two of them leaves float32's range and that
    of all three does not."""
    for v in (40, 3000, 20000, 70000):
        x = torch.randn(4, v, generator=torch.Generator().manual_seed(v))
        ids, u = torch.tensor([[1, 3]] * 4), torch.zeros(4, 2)
        w = torch.tensor([1e35, 1e-36, 1.0, 1e-30])
        up = torch.tensor([1e-36, 1e30, 0.5, 1e30])
        for t in (1e-4, 1e4):
            leaf = (x * t).cuda().requires_grad_()
            loss = frames.distill_loss(leaf, ids.cuda(), (u * t).cuda(), w.cuda(), t)
            got, = torch.autograd.grad(loss, leaf, up.cuda())
            for r in range(4):
                _, gr = frames_ref.row_distill(leaf[r].detach().cpu(), ids[r].tolist(), (u[r] * t).double().tolist(),
                                               w[r].double().item(), t, up[r].double().item())[0]
                tol = frames_ref.row_distill(leaf[r].detach().cpu(), ids[r].tolist(), (u[r] * t).double().tolist(),
                                             w[r].double().item(), t, up[r].double().item())[1][1]
                assert ((got[r].cpu().double() - gr).abs() <= tol + 2 * frames_ref.U * gr.abs()).all(), (v, r, t)


def test_forward_mode_derivatives_are_refused(frames):
    import torch.autograd.forward_ad as fwd
    x, ids, u = torch.randn(3, 40).cuda(), torch.zeros(3, 2, dtype=torch.int32).cuda(), torch.randn(3, 2).cuda()
    sc = frames.token_scores(x, ids[:, 0])
    up = torch.ones(3).cuda()
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: frames.token_scores(dual(x)), lambda: frames.token_scores(dual(x).requires_grad_()),
                     lambda: frames.distill_loss(dual(x), ids, u), lambda: frames.distill_loss(x, ids, dual(u)),
                     lambda: frames.distill_loss(x, ids, u, dual(up)),
                     lambda: frames.distill_loss_and_grad(dual(x), ids, u),
                     lambda: frames.token_scores_grad(x, sc, ids[:, 0], None, dual(up))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(frames.token_scores(dual(x).detach()).entropy, sc.entropy)


def test_a_gradient_within_padded_tensors(frames):
    """`out` in the storage of the logits or of another input: refused where an element would be in the
    place of another that is read, right where it is not."""
    for v in (40, 3000, 20000, 70000):
        wide = torch.randn(2, 5, 2 * v + 3).cuda()
        ids, u = torch.randint(0, v, (2, 4, 3)).cuda(), torch.randn(2, 4, 3).cuda()
        x = wide[:, :4, :v]
        tokens, up = ids[..., 0].contiguous(), torch.randn(2, 4).cuda()
        sc = frames.token_scores(x, tokens)
        before = wide.clone()
        version = wide._version
        for out in (wide[:, :4, 1:v + 1], wide[:, :4, v - 1:2 * v - 1], wide[:, 1:, :v], wide[:, 1:, v // 2:v // 2 + v],
                    wide.flatten()[5:5 + 8 * v].view(2, 4, v)):
            for call in (lambda: frames.distill_loss_and_grad(x, ids, u, out=out),
                         lambda: frames.token_scores_grad(x, sc, tokens, None, up, up, out=out),
                         lambda: frames.distill_loss_and_grad(x[0], ids[0], u[0], out=out[0])):
                with pytest.raises(RuntimeError, match="across the logits"):
                    call()
        assert torch.equal(wide, before) and wide._version == version
        loss, want = frames.distill_loss_and_grad(x.clone(), ids, u)
        for out in (wide[:, :4, v:2 * v], wide[:, :4, v + 3:], wide[:, :4, :v]):  # (the last: the logits themselves)
            loss2, got = frames.distill_loss_and_grad(x, ids, u, out=out)
            assert torch.equal(got, want) and got.data_ptr() == out.data_ptr() and torch.equal(loss, loss2)
            assert wide._version > version
            assert torch.equal(wide[:, 4], before[:, 4])
    # other inputs
    u = torch.randn(3, 4, 8).cuda()
    x, ids = torch.randn(3, 4, 8).cuda(), torch.arange(8).expand(3, 4, 8).cuda()
    with pytest.raises(RuntimeError, match="across the teacher's logits"):
        frames.distill_loss_and_grad(x, ids, u, out=u)
    sc = frames.token_scores(x, ids[..., 0])
    up = x.new_zeros(13)
    with pytest.raises(RuntimeError, match="across grad_logp"):
        frames.token_scores_grad(x[..., :1], sc, ids[..., 0], None, up[1:].view(3, 4), None, out=up[:12].view(3, 4, 1))


def test_rows_of_weight_zero_are_not_read(frames):
    """Long rows, cut into segments: those of weight 0 leave no partial results in the workspace."""
    from kaldi_decoder import cabi
    n, v = 16, 70000
    x = torch.randn(n, v).cuda()
    ids, u = torch.zeros(n, 1, dtype=torch.int32).cuda(), torch.zeros(n, 1).cuda()
    w = (torch.arange(n) % 2).float().cuda()
    loss = torch.empty(n).cuda()
    rows = cabi.FrameRows(x.data_ptr(), 1, n, v, 0, v, None, 0, 0)
    teacher = cabi.TeacherRows(ids.data_ptr(), u.data_ptr(), 1, 4, 0)
    bytes_ = cabi.lib().kd_distill_loss_workspace(C.byref(rows), 0)
    ws = torch.full((bytes_,), 0x5a, dtype=torch.uint8).cuda()
    assert cabi.lib().kd_distill_loss(C.byref(rows), C.byref(teacher), w.data_ptr(), 1.0, loss.data_ptr(), None, None,
                                      None, 0, 0, ws.data_ptr(), bytes_, torch.cuda.current_stream().cuda_stream) == 0
    want = frames.distill_loss(x, ids, u)
    assert torch.equal(loss, torch.where(w > 0, want, torch.zeros_like(want)))
    part = ws[:bytes_ - 256].view(n, -1)  # (16 bytes a segment, all rows' first; then 8 bytes a row)
    assert part[0::2].eq(0x5a).all() and part[1::2].ne(0x5a).any(-1).all()


def test_scores_of_utterances_without_a_path(frames):
    """An utterance whose search died scores -inf, not the 0 of a certain one; columns that the logits do
    not have are an error."""
    from kaldi_decoder import cabi, synth
    # 0 -1-> 1 -2-> 2 (final), and no way on: a third frame leaves no token
    g = synth.graph_from_arcs(3, 0, [(0, 1, 1, 1, 0.0), (1, 2, 2, 2, 0.0)], {2: 0.0})
    x = torch.log_softmax(torch.randn(3, 4, 5, generator=torch.Generator().manual_seed(0)), -1).cuda()
    for lengths in ([2, 3, 4], torch.tensor([2, 3, 4]).cuda(), torch.tensor([2, 3, 4], dtype=torch.int32)):
        bt = cabi.Batch(cabi.Graph(g), max_batch=3, beam=100.0)
        bt.decode_tensor(x, lengths)
        paths, tokens, sc = bt.best_path_scores(x, lengths, top=2)
        assert [p.ok for p in paths] == [True, False, False]
        assert tokens[0].tolist() == [0, 1, -1, -1] and tokens[1:].eq(-1).all()
        assert torch.isfinite(sc.logp[0]).all() and sc.logp[0, 2:].eq(0).all()
        assert sc.logp[1].tolist() == [-INF, -INF, -INF, 0.0] and sc.logp[2].eq(-INF).all()
        assert sc.entropy[1, :3].gt(0).all()
    leaf = x.clone().requires_grad_()
    sc = bt.best_path_scores(leaf)[2]
    assert sc.logp[1:].eq(-INF).all()
    sc.logp[0].sum().backward()
    assert leaf.grad[1:].eq(0).all() and leaf.grad[0].ne(0).any()
    with pytest.raises(ValueError, match="column"):
        bt.best_path_scores(x[..., :1])


def test_inference_tensors(frames):
    """`out` made in inference mode is written there and, outside of it, refused before anything is."""
    x, ids, u = torch.randn(3, 40).cuda(), torch.arange(2).expand(3, 2).cuda(), torch.randn(3, 2).cuda()
    loss, want = frames.distill_loss_and_grad(x, ids, u)
    with torch.inference_mode():
        out = torch.zeros(3, 40).cuda()
        loss2, got = frames.distill_loss_and_grad(x, ids, u, out=out)
        assert torch.equal(got, want) and torch.equal(loss, loss2) and torch.equal(out, want)
        sc = frames.token_scores(x, ids[:, 0], top=3)
        out.zero_()
    assert torch.equal(sc.logp, frames.token_scores(x, ids[:, 0]).logp)
    with pytest.raises(RuntimeError, match="inference"):
        frames.distill_loss_and_grad(x, ids, u, out=out)
    with pytest.raises(RuntimeError, match="inference"):
        frames.token_scores_grad(x, sc, ids[:, 0], None, loss, None, out=out)
    torch.cuda.synchronize()
    assert out.eq(0).all()


@pytest.mark.parametrize("v", [55, 500, 2000, 5003, 20001, 70000])
def test_precision_of_peaked_rows(frames, v):
    """Rows that one token has nearly to itself, where log p, the entropy and the gradient at the token are what is
    left of 1: as near to 64 bits as sums of f32 in pairs are.  With s = 1 + r, r the others' share, s is off by
    half a step of its own (2^-24, it is below 2) and, of the additions that 1 takes part in -- N levels of the sum
    --, by half a step each: the mean over rows of independent errors of N + 1 roundings, each at most 2^-24 and
    even from -2^-24 to 2^-24, is at most sqrt((N + 1) / 3) 2^-24, and log p is off by that (and by steps of its
    own, far smaller).  The levels: 2 or 3 within 16 bytes, at most 8 16-byte pieces, 6 over a wave's lanes, 3 over
    waves, 1 over segments."""
    n = 512
    g = torch.Generator().manual_seed(v)
    x = torch.randn(n, v, generator=g)
    tokens = torch.randint(0, v, (n,), generator=g)
    x.scatter_(1, tokens[:, None], 11 + torch.log(torch.tensor(v / 500.0)) + 4 * torch.rand(n, 1, generator=g))
    sc = frames.token_scores(x.cuda(), tokens.cuda())
    lp = torch.log_softmax(x.double(), -1).gather(1, tokens[:, None]).squeeze(1)
    assert lp.min() > -0.5  # (the rows are what they are meant to be)
    off = (sc.logp.cpu().double() - lp).abs().mean().item()
    assert off <= ((3 + 8 + 6 + 3 + 1 + 1) / 3) ** 0.5 * 2 ** -24, off * 2 ** 24


def test_a_gradient_over_the_transposed_logits(frames):
    """As many steps as utterances: `out` = the logits' transpose is the same memory in another order."""
    x = torch.randn(4, 4, 300).cuda()
    ids, u = torch.zeros(4, 4, 2, dtype=torch.int32).cuda(), torch.randn(4, 4, 2).cuda()
    before = x.clone()
    with pytest.raises(RuntimeError, match="across the logits"):
        frames.distill_loss_and_grad(x, ids, u, out=x.transpose(0, 1))
    with pytest.raises(RuntimeError, match="across the logits"):
        frames.token_scores_grad(x.transpose(0, 1), frames.token_scores(x), None, None, None, u[..., 0].contiguous(), out=x)
    assert torch.equal(x, before)
    _, want = frames.distill_loss_and_grad(before, ids, u)
    t = x.transpose(0, 1)
    _, got = frames.distill_loss_and_grad(t, ids.transpose(0, 1), u.transpose(0, 1), out=t)
    assert torch.equal(x, want)

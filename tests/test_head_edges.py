"""linear_softmax_loss and linear_softmax_grad where results go wrong first:
rows that are nearly certain, scores of any size, few rows over many tiles of
classes, a strong z-loss in float16, NaN in whole tiles, the ends of the
allowed sizes."""
import math

import pytest

torch = pytest.importorskip("torch")

from bsscl_gbm import linear_softmax_grad, linear_softmax_loss, tensor_ops  # noqa: E402
from head_model import E, Head, half_step  # noqa: E402
from test_softmax_head import DTYPES, make  # noqa: E402


def picked(rows, vocab, tops, gap, dtype=torch.float32):
    """hidden, weight and labels whose scores are exact: the weight's first 64
    rows pick a column of hidden each and the others are 0, so that class
    v < 64 scores hidden[:, v] and every other class 0."""
    w = torch.zeros(vocab, 64, dtype=dtype)
    w[:64] = torch.eye(64, dtype=dtype)
    top = torch.tensor(tops, dtype=torch.float64)[torch.arange(rows) % len(tops)]
    y = torch.arange(rows) * 7 % 64
    g = torch.Generator().manual_seed(rows)
    h = top[:, None] - gap * (1 + torch.rand(rows, 64, generator=g, dtype=torch.float64))
    h[torch.arange(rows), y] = top
    return h.to(dtype).cuda(), w.cuda(), y.cuda()


# -- rows that are nearly certain, scores of any size -----------------------
TOPS = [t + k / 16 for k in range(16) for t in (10, 13, 23, 27, 46, 57, 90, 120)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [32, 384])
def test_nearly_certain_rows(rows):
    """No loss below 0 and no p above 1 where the other classes lie 12 to 24
    below the label (or 10 to 127, those at 0), and losses as fine as float32
    sums near 1 allow.

    The scores are exact.  A tile's sum and those of all tiles take at most 64
    additions to a value in [1, 2), each off by 2^-24, logf and expm1f 4 of
    2^-24 of less than 1: 72 e.  The other classes' p are exponentials of at
    most 24, whose difference and product with log2 e are rounded once each and
    whose constant is off by half as much: 60 e, and 36 e for the exponential,
    the sum and the factors."""
    print(f"[case] head nearly certain {rows}", flush=True)
    h, w, y = picked(rows, 640, TOPS, 12.0)
    z = torch.cat([h.double(), torch.zeros(rows, 576, dtype=torch.float64, device="cuda")], 1)
    at = torch.arange(rows, device="cuda")
    rest = z - z[at, y][:, None]
    rest[at, y] = -math.inf
    loss = torch.log1p(rest.exp().sum(1))
    got = linear_softmax_grad(h, w, y, reduction="sum")
    for r in (linear_softmax_loss(h, w, y, reduction="sum"), got):
        assert float(r.row_loss.min()) >= 0
        assert float((r.row_loss.double() - loss).abs().max()) <= 72 * E
    ds = torch.exp(rest - loss[:, None])[:, :64]
    ds[at, y] = torch.expm1(-loss)
    assert float(got.d_hidden[at, y].max()) <= 0
    off = (got.d_hidden.double() - ds).abs()
    tol = 96 * E * ds.abs() + 1e-44
    tol[at, y] = 72 * E
    assert bool((off <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 40])
@pytest.mark.parametrize("top", [-3e4, 1e6, -3e9, 1e10, 1e30])
def test_scores_of_any_size(top, rows):
    """Only differences to the maximum are exponentials, whatever it is: 63
    classes lie far below the label, which is certain if its score is above 0
    and (with 576 classes at 0) has no mass otherwise."""
    print(f"[case] head scores {top} {rows}", flush=True)
    for dtype in [torch.float32, torch.bfloat16] + ([torch.float16] if abs(top) < 6e4 else []):
        h, w, y = picked(rows, 640, [top], abs(top) / 4, dtype)
        at = torch.arange(rows, device="cuda")
        top_y = h.double()[at, y]
        want = torch.zeros(rows, dtype=torch.float64, device="cuda") if top > 0 else \
            math.log(576) - top_y
        got = linear_softmax_grad(h, w, y, reduction="sum")
        for r in (linear_softmax_loss(h, w, y, reduction="sum"), got):
            assert float((r.row_loss.double() - want).abs().max()) <= 4 * E * float(want.max())
            lse = top_y if top > 0 else torch.full_like(top_y, math.log(576))
            assert float((r.lse.double() - lse).abs().max()) <= 4 * E * float(lse.abs().max())
        ds = torch.zeros_like(got.d_hidden)
        if top < 0:
            ds[at, y] = -1
        assert torch.equal(got.d_hidden, ds)


# -- NaN in whole tiles ------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,classes", [(1, 9000, 8192), (9, 8500, 128), (3, 40000, 20000),
                                                (40, 33500, 128), (300, 70000, 256)])
def test_nan_in_whole_tiles_of_classes(rows, vocab, classes):
    """Classes whose weights are all NaN make every row's loss NaN, also where
    they fill whole tiles in front of sound ones."""
    print(f"[case] head NaN tiles {rows} x {vocab}, {classes}", flush=True)
    for dtype in (torch.bfloat16, torch.float32):
        h, w, y = make(rows, 64, vocab, dtype, seed=rows)
        y[:] = vocab - 1
        w[:classes] = float("nan")
        for r in (linear_softmax_loss(h, w, y), linear_softmax_grad(h, w, y)):
            assert bool(torch.isnan(r.loss))
            assert bool(torch.isnan(r.row_loss).all()) and bool(torch.isnan(r.lse).all())


# -- a strong z-loss in float16 ----------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("factor", [20.0, 63.0, 81.0, 200.0, 600.0])
@pytest.mark.parametrize("rows,vocab", [(48, 700), (700, 33000)])
def test_strong_z_loss_in_float16(factor, rows, vocab):
    """1 + 2 zeta lse far above 1, with most of the mass on another class than
    the label.  The operand's scale then falls by as much (to the next power of
    two, and log(vocab) may be in the bound of lse twice over): its half step
    2^-35 grows by at most 4 factor / 32."""
    print(f"[case] head z-loss {factor} {rows} x {vocab}", flush=True)
    h, w, y = make(rows, 72, vocab, torch.float16, seed=3, spread=1.0, left_out=0.1)
    h = (h.float() + 40.0 * w[(y + 1) % vocab].float()).half()
    lse = torch.logsumexp(h.double() @ w.double().T, 1)[y >= 0]
    zeta = (factor - 1) / (2 * float(lse.median()))
    u = torch.linspace(0.25, 1.0, rows).cuda()
    m = Head(h, w, y, row_weight=u, z_loss=zeta, reduction="sum")
    more = float(u.max()) * 2.0 ** -35 * 4 * max(1.0, factor * float(lse.max() / lse.median()) / 32)
    m.tol_d_hidden += more * m.w.abs().sum(0)
    m.tol_d_weight += more * m.h.abs().sum(0)
    m.check(linear_softmax_grad(h, w, y, row_weight=u, z_loss=zeta, reduction="sum"))


@pytest.mark.gpu
@pytest.mark.parametrize("zeta", [0.5, 30.0])
def test_strong_z_loss_below_zero_in_float16(zeta):
    """lse far below 0: 1 + 2 zeta lse far below -1.  (Head takes the factor's
    sign into the exponentials' share of a tolerance: twice the share's size
    gives it back.)"""
    print(f"[case] head z-loss {zeta}, lse below 0", flush=True)
    h, w, y = make(300, 64, 200, torch.float16, seed=4, spread=1.0)
    h[:, 0], w[:, 0] = -8.0, 8.0  # every score 64 lower
    m = Head(h, w, y, z_loss=zeta)
    assert float(m.lse.max()) < -40
    f = (1 + 2 * zeta * m.lse).abs()[:, None]
    err = 66 * E * (m.h.abs() @ m.w.abs().T).amax(1, keepdim=True)
    e_exp = 3 * err + 664 * E + 4 * E * m.lse.abs()[:, None]
    p = torch.exp(m.h @ m.w.T - m.lse[:, None])
    back = 2 * f * e_exp / 300 * (p + torch.zeros_like(p).scatter_(1, y[:, None], 1.0))
    more = 2.0 ** -35 * 4 * float(f.max()) / 32 / 300
    m.tol_d_hidden += more * m.w.abs().sum(0) + back @ m.w.abs()
    m.tol_d_weight += more * m.h.abs().sum(0) + back.T @ m.h.abs()
    m.check(linear_softmax_grad(h, w, y, z_loss=zeta))


@pytest.mark.gpu
def test_strong_z_loss_in_several_pieces_in_float16():
    """Each piece has an operand scale of its own; lse rises from piece to
    piece, and the sums over pieces are of the same unit."""
    rows, vocab = 600, 1_100_003
    print(f"[case] head z-loss pieces {rows} x 8 x {vocab}", flush=True)
    h, w, y = make(rows, 8, vocab, torch.float16, seed=4)
    h = (h.float() * torch.linspace(0.2, 6.0, rows).cuda()[:, None]).half()
    kw = dict(z_loss=4.0, reduction="sum", grad_scale=1 / 16)
    m = Head(h, w, y, **kw)
    f = float((1 + 8 * m.lse).abs().max())
    assert f > 100
    more = 2.0 ** -35 * 4 * f / 32 / 16
    m.tol_d_hidden += more * m.w.abs().sum(0)
    m.tol_d_weight += more * m.h.abs().sum(0)
    m.check(linear_softmax_grad(h, w, y, **kw))
    del m
    torch.cuda.empty_cache()


# -- autograd ---------------------------------------------------------------------
def _needs_grad(h, w, u):
    return [(h.clone().requires_grad_(), w, u), (h, w.clone().requires_grad_(), u),
            (h, w, u.clone().requires_grad_())]


def check_no_backward(h, w, y, u):
    want = linear_softmax_loss(h, w, y, row_weight=u)
    for h2, w2, u2 in _needs_grad(h, w, u):
        got = linear_softmax_loss(h2, w2, y, row_weight=u2)
        leaf = torch.ones((), device=h.device, requires_grad=True)
        for a, b in zip(got, want):
            assert a.requires_grad and torch.equal(a, b) and float(a.detach().sum()) == float(b.sum())
            with pytest.raises(RuntimeError, match="linear_softmax_grad"):
                (a.sum() + leaf).backward()
        with torch.no_grad():
            assert not linear_softmax_loss(h2, w2, y, row_weight=u2).loss.requires_grad
    assert not any(t.requires_grad for t in want)
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(h, torch.ones_like(h))
        with pytest.raises(RuntimeError, match="forward mode"):
            linear_softmax_loss(dual, w, y)
        assert not linear_softmax_loss(h, w, y).loss.requires_grad


def test_a_missing_backward_is_said(monkeypatch):
    """The same outputs, by a stand-in for the kernels' call."""
    h, w, y = make(6, 8, 20, torch.float32, device="cpu")

    def head(hidden, weight, labels, row_weight, *options):
        row = (hidden.detach() @ weight.detach().T).logsumexp(1)
        return [row.sum(), row, row.clone()]

    monkeypatch.setattr(tensor_ops, "_head", head)
    check_no_backward(h, w, y, torch.ones(6))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 50])
def test_a_missing_backward_is_said_on_the_gpu(rows):
    h, w, y = make(rows, 64, 300, torch.float32)
    check_no_backward(h, w, y, torch.ones(rows).cuda())
    got = linear_softmax_grad(h.requires_grad_(), w.requires_grad_(), y)
    assert not any(t.requires_grad for t in got)
    h.backward(got.d_hidden)
    assert torch.equal(h.grad, got.d_hidden)

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
def test_strong_z_loss_in_replayed_graphs():
    """The range of a call's scores is its own: inputs that shrink from replay
    to replay have the gradients of eager calls."""
    print("[case] head z-loss graph", flush=True)
    h, w, y = make(300, 64, 700, torch.float16, seed=9, spread=4.0)
    start = h.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = linear_softmax_grad(h, w, y, z_loss=20.0, grad_scale=1 / 16)
    for k in (4.0, 1.0, 0.25, 2.0):
        h.copy_(start * k)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, linear_softmax_grad(h, w, y, z_loss=20.0, grad_scale=1 / 16)):
            assert bool(torch.isfinite(b).all()) and torch.equal(a, b)


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


# -- few rows over many tiles -------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("vocab", [8193, 33000, 140001])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33])
def test_few_rows_over_many_tiles(rows, vocab, dtype):
    """Every division of a row's tiles among waves, several tiles a lane."""
    print(f"[case] head few rows {rows} x {vocab} {dtype}", flush=True)
    h, w, y = make(rows, 64, vocab, DTYPES[dtype], seed=rows)
    u = torch.linspace(-0.5, 2.0, rows).cuda() if rows > 1 else None
    if rows > 2:
        y[1] = (-100, vocab, 1 << 40)[rows % 3]
        h[1] = float("nan")
    for kw in (dict(), dict(reduction="sum", z_loss=0.01, softcap=6.0)):
        Head(h, w, y, row_weight=u, **kw).check(linear_softmax_loss(h, w, y, row_weight=u, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 8, 32])
def test_few_rows_that_weigh_nothing(rows):
    h, w, y = make(rows, 64, 9000, torch.bfloat16, seed=rows)
    u = torch.tensor([1.5, -1.5] * (rows // 2)).cuda()
    got = linear_softmax_loss(h, w, y, row_weight=u)
    assert float(got.loss) == 0 and float(got.row_loss.min()) > 0
    y[:] = -1
    for reduction in ("mean", "sum"):
        got = linear_softmax_loss(h, w, y, row_weight=u, reduction=reduction)
        assert all(not t.any() for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows", [1, 20, 64])
def test_few_rows_all_left_out(rows, dtype):
    """No row counts: zeros, whatever the rows hold."""
    print(f"[case] head few rows left out {rows} {dtype}", flush=True)
    h, w, y = make(rows, 64, 9000, DTYPES[dtype], seed=rows)
    h[:], y[:] = float("nan"), -100
    for r in (linear_softmax_grad(h, w, y), linear_softmax_grad(h, w, y, reduction="sum"),
              linear_softmax_loss(h, w, y)):
        assert all(not t.any() for t in r)


# -- the ends of the sizes ------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,width,vocab", [(40, 65536, 300), (7, 65536, 129), (33, 40001, 70)])
def test_wide_rows(rows, width, vocab, dtype):
    """64 columns spread over wide rows of zeros, in small numbers whose scores
    are exact: the losses have the narrow rows' bits, the gradients lie within
    two tolerances of theirs (the sums' order differs) and are 0 elsewhere."""
    print(f"[case] head wide {rows} x {width} x {vocab} {dtype}", flush=True)
    t = DTYPES[dtype]
    g = torch.Generator().manual_seed(width + rows)
    at = torch.cat([torch.randperm(width - 66, generator=g)[:61] + 65,
                    torch.tensor([0, 64, width - 1])]).cuda()
    h = (torch.randint(-3, 4, (rows, 64), generator=g) / 4).to(t).cuda()
    w = (torch.randint(-3, 4, (vocab, 64), generator=g) / 4).to(t).cuda()
    y = torch.randint(-5, vocab, (rows,), generator=g).cuda()
    h_wide, w_wide = (torch.zeros(len(x), width, dtype=t, device="cuda") for x in (h, w))
    h_wide[:, at], w_wide[:, at] = h, w
    m = Head(h, w, y)
    want, got = linear_softmax_grad(h, w, y), linear_softmax_grad(h_wide, w_wide, y)
    m.check(want)
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a, b)
    for a, b, tol in ((got.d_hidden, want.d_hidden, m.tol_d_hidden),
                      (got.d_weight, want.d_weight, m.tol_d_weight)):
        assert bool(((a[:, at].double() - b.double()).abs() <= 2 * tol).all())
        a[:, at] = 0
        assert not a.any()
    few, narrow = linear_softmax_loss(h_wide, w_wide, y), linear_softmax_loss(h, w, y)
    m.check(narrow)
    m.check(few)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_more_rows_than_a_piece_holds(dtype):
    """2^20 rows and more are scored in two pieces, with a small vocabulary."""
    rows = (1 << 20) + 777
    print(f"[case] head {rows} rows {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(6)
    h = torch.randn(rows, 8, generator=g, device="cuda").to(DTYPES[dtype])
    w = torch.randn(50, 8, generator=g, device="cuda").to(DTYPES[dtype])
    y = torch.randint(-10, 50, (rows,), generator=g, device="cuda")
    y[: rows // 50] = -1
    m = Head(h, w, y)
    m.check(linear_softmax_loss(h, w, y))
    m.check(linear_softmax_grad(h, w, y))
    y[:] = torch.randint(0, 50, (rows,), generator=g, device="cuda")
    m = Head(h, w, y)
    m.check(linear_softmax_loss(h, w, y))
    m.check(linear_softmax_grad(h, w, y))


@pytest.mark.gpu
def test_loss_in_several_pieces_of_a_large_vocabulary():
    """40,000 rows x 1.1 million classes take two pieces for their statistics;
    rows scored by themselves (one piece) have the same values."""
    print("[case] head loss pieces 40000 x 8 x 1100003", flush=True)
    h, w, y = make(40000, 8, 1_100_003, torch.bfloat16, seed=5, left_out=0.1)
    got = linear_softmax_loss(h, w, y, reduction="sum")
    for a in (0, 20000, 35000, 39700):
        Head_part = Head(h[a:a + 300], w, y[a:a + 300], reduction="sum")
        part = linear_softmax_loss(h[a:a + 300], w, y[a:a + 300], reduction="sum")
        Head_part.check(part)
        assert bool(((got.row_loss[a:a + 300] - part.row_loss).abs()
                     <= 2 * Head_part.tol_row_loss).all())
        assert bool(((got.lse[a:a + 300] - part.lse).abs() <= 2 * Head_part.tol_lse).all())
        del Head_part
    total = float(got.row_loss.double().sum())
    assert abs(float(got.loss) - total) <= 4 * E * total
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_of_the_weight_megabytes_apart(dtype):
    """Rows too far apart for the tiles' 32-bit offsets."""
    print(f"[case] head rows of the weight apart {dtype}", flush=True)
    h, w, y = make(50, 64, 9, DTYPES[dtype], seed=6)
    want = linear_softmax_grad(h, w, y)
    stride = (1 << 31) // 256 // w.element_size() + 8
    far = torch.empty(9 * stride, dtype=w.dtype, device="cuda").as_strided((9, 64), (stride, 1))
    far.copy_(w)
    for a, b in zip(linear_softmax_grad(h, far, y), want):
        assert torch.equal(a, b)
    got = linear_softmax_loss(h[:3], far, y[:3])
    assert torch.equal(got.row_loss, linear_softmax_grad(h[:3], w, y[:3]).row_loss)


# -- long sums ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,width,vocab", [(8, 65536, 140), (33, 16384, 300), (100, 8192, 260)])
def test_long_sums_of_one_sign(rows, width, vocab, dtype):
    """Sums of equal terms, whose roundings lean to one side: at most 256 terms
    are added to one sum before it is added to the next, so that a score is off
    by (256 + width / 128) e of its size, where one chain would take width / 4
    steps (width / 32 in 16 bits); lse and losses as scores, and 640 e of lse."""
    print(f"[case] head long sums {rows} x {width} x {vocab} {dtype}", flush=True)
    t = DTYPES[dtype]
    c = torch.linspace(1.0, 1.9, vocab).to(t).cuda()
    w = (c * 20 / width).to(t)[:, None].expand(vocab, width).contiguous()
    h = torch.full((rows, width), 1 / 3).to(t).cuda()
    y = torch.arange(rows).cuda() * 7 % vocab
    z = h[0, 0].double() * width * w[:, 0].double()
    lse = torch.logsumexp(z, 0)
    off = (256 + width / 128) * E * float(z.max())
    for got in (linear_softmax_loss(h, w, y), linear_softmax_grad(h, w, y)):
        assert float((got.lse.double() - lse).abs().max()) <= off + 640 * E * float(lse)
        assert float((got.row_loss.double() - (lse - z[y])).abs().max()) \
            <= 2 * off + 640 * E * float(lse)


# -- the label's value ----------------------------------------------------------
def label_share(got, exact, along, own):
    """Root mean square over rows of the relative error that all of a row's
    columns share along `along`: what the label's value is off by, since the
    other errors differ from column to column."""
    err = got.double() - exact
    return float((((err * along).sum(1) / (along * along).sum(1) / own) ** 2).mean().sqrt())


@pytest.mark.parametrize("rest,ok", [(1.0, True), (0.0, False), (-1.0, False)])
def test_label_share_sees_the_label_s_rounding(rest, ok):
    """A label's value rounded to bfloat16 (8 bits), with its rest added,
    forgotten or subtracted."""
    g = torch.Generator().manual_seed(2)
    along = torch.randn(100, 1024, generator=g, dtype=torch.float64)
    own = -(0.3 + 0.7 * torch.rand(100, generator=g, dtype=torch.float64))
    held = own.bfloat16().double()
    got = ((held + rest * (own - held))[:, None] * along).bfloat16()
    share = label_share(got, own[:, None] * along, along, own)
    assert (share <= 0.1 * half_step(torch.bfloat16)) == ok


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_label_s_value_is_not_rounded(dtype):
    """Surprising labels (p < 1e-3) of unequal weights: d_hidden has the
    label's value from float32; d_weight, with equal weights, has p - 1 to p or
    to the half step below 1.  What rounds the outputs (half a step, independent
    from column to column) leaves sqrt(3 / 1024) of 0.58 half steps in the share,
    rounding p the same times p; the label's own rounding would be about 0.4."""
    print(f"[case] head label's value {dtype}", flush=True)
    t = DTYPES[dtype]
    rows, width, vocab = 200, 1024, 5000
    g = torch.Generator().manual_seed(14)
    w = (torch.randn(vocab, width, generator=g) / 16).to(t).cuda()
    h = torch.randn(rows, width, generator=g).to(t).cuda()
    y = torch.randperm(vocab, generator=g)[:rows].cuda()
    u = (0.3 + 0.7 * torch.rand(rows, generator=g)).cuda()
    for weight in (u, None):
        m = Head(h, w, y, row_weight=weight, reduction="sum")
        p = torch.exp(-m.row_loss)
        some = p < 1e-3
        assert int(some.sum()) > 100
        got = linear_softmax_grad(h, w, y, row_weight=weight, reduction="sum")
        own = (p - 1) * (1 if weight is None else weight.double())
        share = label_share(got.d_hidden[some], m.d_hidden[some], m.w[y[some]], own[some])
        assert share <= 0.1 * half_step(t)
        if weight is None:
            share = label_share(got.d_weight[y[some]], m.d_weight[y[some]], m.h[some], own[some])
            kept = torch.clamp(p[some], max=half_step(t) / 2).square().mean().sqrt()
            assert share <= 0.1 * half_step(t) + float(kept)


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 20, 32, 33, 64])
def test_label_s_value_is_not_rounded_in_d_weight_of_few_rows(rows, dtype):
    """Labels of any probability and unequal weights, rows left out among them.
    The outputs' rounding leaves sqrt(3 / 4096) of 0.58 half steps in the share;
    the label's own would be about 0.4 (of one row, anything below 1)."""
    print(f"[case] head label's value in d_weight {rows} {dtype}", flush=True)
    t = DTYPES[dtype]
    width, vocab = 4096, 3001
    g = torch.Generator().manual_seed(rows)
    w = torch.randn(vocab, width, generator=g) / 32
    y = torch.randperm(vocab, generator=g)[:rows]
    h = torch.randn(rows, width, generator=g) + w[y] * (1 + 2 * torch.rand(rows, 1, generator=g))
    h, w, y = h.to(t).cuda(), w.to(t).cuda(), y.cuda()
    if rows > 5:
        y[3:rows:7] = -1
    u = (0.3 + 0.7 * torch.rand(rows, generator=g)).cuda()
    m = Head(h, w, y, row_weight=u)
    own = (torch.exp(-m.row_loss) - 1) * u.double() / u.double()[y >= 0].sum()
    got = linear_softmax_grad(h, w, y, row_weight=u)
    m.check(got)
    k = y >= 0
    assert label_share(got.d_weight[y[k]], m.d_weight[y[k]], m.h[k], own[k]) <= 0.1 * half_step(t)
    assert label_share(got.d_hidden[k], m.d_hidden[k], m.w[y[k]], own[k]) <= 0.1 * half_step(t)

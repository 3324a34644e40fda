"""linear_softmax_loss and linear_softmax_grad against their formulas in
float64 (head_model.py), and their refusals."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import bsscl_gbm  # noqa: E402
from bsscl_gbm import _native, linear_softmax_grad, linear_softmax_loss  # noqa: E402
from head_model import Head  # noqa: E402

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(rows, width, vocab, dtype, seed=0, spread=2.0, left_out=0.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(vocab, width, generator=g) * (spread / width ** 0.5)).to(dtype)
    h = torch.randn(rows, width, generator=g)
    y = torch.randint(0, vocab, (rows,), generator=g)
    h = (h + torch.rand(rows, 1, generator=g) * 3 * w[y].float()).to(dtype)
    if left_out:
        y[torch.rand(rows, generator=g) < left_out] = -100
    return h.to(device), w.to(device), y.to(device)


# ---------------------------------------------------------------------------
# On the CPU: the model itself, and calls that are refused
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("softcap,z_loss,reduction", [(0.0, 0.0, "mean"), (3.0, 0.02, "mean"),
                                                      (0.0, 0.1, "sum")])
def test_model_gradient_is_the_difference_quotient(softcap, z_loss, reduction):
    h, w, y = make(7, 5, 11, torch.float32, seed=3, left_out=0.3, device="cpu")
    h, w = h.double(), w.double()
    u = torch.linspace(0.5, 2.0, 7).float()
    kw = dict(row_weight=u, reduction=reduction, softcap=softcap, z_loss=z_loss)

    def loss(a, b):
        m = Head.__new__(Head)
        Head.__init__(m, a, b, y, **kw)
        return float(m.loss)

    m = Head(h, w, y, **kw)
    step = 1e-5  # truncation ~ step^2, cancellation ~ 1e-16 / step: both near 1e-10
    for x, grad, other in ((h, m.d_hidden, 0), (w, m.d_weight, 1)):
        for i in range(0, x.numel(), 3):
            d = torch.zeros_like(x).reshape(-1)
            d[i] = step
            d = d.reshape(x.shape)
            up = loss(h + d, w) if other == 0 else loss(h, w + d)
            down = loss(h - d, w) if other == 0 else loss(h, w - d)
            assert abs((up - down) / (2 * step) - float(grad.reshape(-1)[i])) < 1e-7


def test_refuses_tensors_that_do_not_fit():
    h, w, y = make(4, 8, 16, torch.float32, device="cpu")
    for args, kw, what in [
            ((h, w, y), {}, "GPU"),
            ((h.numpy(), w, y), {}, "torch tensors"),
            ((h, w.bfloat16(), y), {}, "must both be"),
            ((h.double(), w.double(), y), {}, "must both be"),
            ((h[:, :7], w, y), {}, "do not fit"),
            ((h, w[0], y), {}, "do not fit"),
            ((h, w, y[:3]), {}, "labels"),
            ((h, w, y.float()), {}, "int64 or int32"),
            ((h, w, y), dict(reduction="none"), "reduction"),
            ((h, w, y), dict(row_weight=torch.ones(3)), "row_weight"),
            ((h, w, y), dict(row_weight=torch.ones(4).double()), "row_weight"),
            ((h, w, y), dict(softcap=-1.0), "softcap"),
            ((h[:0], w, y[:0]), dict(softcap=float("inf")), "softcap"),
            ((h, w, y), dict(softcap=1e-9), "softcap"),
            ((h, w, y), dict(z_loss=float("nan")), "z_loss")]:
        for fn in (linear_softmax_loss, linear_softmax_grad):
            with pytest.raises(ValueError, match=what):
                fn(*args, **kw)


def test_refuses_a_grad_scale_that_is_not_finite():
    h, w, y = make(4, 8, 16, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="grad_scale"):
        linear_softmax_grad(h, w, y, grad_scale=float("inf"))


def test_c_entries_refuse_bad_sizes():
    L = _native.lib()
    size = ctypes.c_int64()

    def ws(dtype, rows, width, vocab):
        return L.bsscl_head_workspace(dtype, rows, width, vocab, None, width, 1,
                                      ctypes.byref(size))

    assert ws(0, 5, 8, 9) == _native.BSSCL_OK and size.value > 0
    for bad in [(3, 5, 8, 9), (-1, 5, 8, 9), (0, 0, 8, 9), (0, 5, 0, 9), (0, 5, 8, 0),
                (0, 8000001, 8, 9), (0, 5, 65537, 9), (0, 5, 8, 4000001)]:
        assert ws(*bad) == _native.BSSCL_EINVAL
        assert L.bsscl_last_error()
    fake = ctypes.c_void_p(4096)  # never read: every call below is refused on the host

    def loss(ws_bytes=1 << 40, h=fake, hs=8, ws_ptr=fake, red=1, cap=0.0, zl=0.0):
        return L.bsscl_head_loss(0, None, 0, h, hs, fake, 8, fake, None, 5, 8, 9, red, cap, zl,
                                 fake, fake, fake, ws_ptr, ws_bytes)

    for kw in [dict(ws_bytes=16), dict(h=None), dict(hs=7), dict(ws_ptr=ctypes.c_void_p(4100)),
               dict(red=2), dict(cap=-1.0), dict(cap=1e-9), dict(cap=float("inf")), dict(cap=float("nan")), dict(zl=-0.1),
               dict(zl=float("inf"))]:
        assert loss(**kw) == _native.BSSCL_EINVAL, kw


# ---------------------------------------------------------------------------
# On the GPU
# ---------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 64, 2), (2, 7, 3), (5, 33, 70), (16, 64, 64), (17, 128, 255),
         (64, 256, 256), (65, 130, 257), (255, 96, 1000), (257, 200, 513), (300, 72, 4099),
         (129, 1001, 777)]


def _both(h, w, y, grad_scale=1.0, **kw):
    m = Head(h, w, y, grad_scale=grad_scale, **kw)
    m.check(linear_softmax_loss(h, w, y, **kw))
    got = linear_softmax_grad(h, w, y, grad_scale=grad_scale, **kw)
    m.check(got)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,width,vocab", SIZES)
def test_sizes(rows, width, vocab, dtype):
    print(f"[case] head {rows} x {width} x {vocab} {dtype}", flush=True)
    h, w, y = make(rows, width, vocab, DTYPES[dtype], seed=rows + width)
    _both(h, w, y, grad_scale=256.0 if dtype == "fp16" else 1.0)


# Enough tiles for the largest shape, at edges of it in every axis.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,width,vocab,kw", [
    (513, 264, 40001, {}), (300, 1001, 33000, {}), (2100, 256, 12800, dict(left_out=0.4)),
    (700, 328, 20011, dict(softcap=20.0, z_loss=1e-3, left_out=0.2)),
    (129, 520, 70000, dict(left_out=0.1))])
def test_large_tiles(rows, width, vocab, kw, dtype):
    print(f"[case] head {rows} x {width} x {vocab} {kw} {dtype}", flush=True)
    kw = dict(kw)
    h, w, y = make(rows, width, vocab, DTYPES[dtype], seed=rows, left_out=kw.pop("left_out", 0.0))
    u = torch.rand(rows, generator=torch.Generator().manual_seed(1)).cuda()
    _both(h, w, y, row_weight=u, grad_scale=512.0 if dtype == "fp16" else 1.0, **kw)
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("kw", [dict(softcap=4.0), dict(z_loss=0.01), dict(reduction="sum"),
                                dict(softcap=30.0, z_loss=1e-4, reduction="sum")],
                         ids=["cap", "z", "sum", "all"])
def test_options(kw, dtype):
    print(f"[case] head options {kw} {dtype}", flush=True)
    h, w, y = make(100, 72, 600, DTYPES[dtype], seed=5, spread=5.0, left_out=0.3)
    u = torch.linspace(-0.5, 2.0, 100, device="cuda")
    u[7] = 0.0
    _both(h, w, y, row_weight=u, grad_scale=64.0, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_rows_left_out(dtype):
    """Rows without a label change nothing, whatever they hold; all of them
    left out gives zeros."""
    h, w, y = make(700, 64, 300, DTYPES[dtype], seed=9)
    masks = {"all": torch.ones(700, dtype=torch.bool), "none but one": torch.arange(700) != 350,
             "first": torch.arange(700) < 256, "last": torch.arange(700) >= 256,
             "every other": torch.arange(700) % 2 == 0}
    for name, mask in masks.items():
        print(f"[case] head rows left out: {name} {dtype}", flush=True)
        mask = mask.cuda()
        for label in (-100, -1, 300, 1 << 40):
            y2, h2 = y.clone(), h.clone()
            y2[mask] = label
            h2[mask] = float("nan")
            got = _both(h2, w, y2)
            h2[mask] = float("inf")
            again = linear_softmax_grad(h2, w, y2)
            for a, b in zip(got, again):
                assert torch.equal(a, b)
        if name == "all":
            assert all(float(t.float().abs().sum()) == 0 for t in got)


@pytest.mark.gpu
def test_weights_that_sum_to_zero_give_zeros():
    h, w, y = make(8, 16, 40, torch.float32)
    u = torch.tensor([1.0, -1.0] * 4, device="cuda")
    got = linear_softmax_grad(h, w, y, row_weight=u)
    assert float(got.loss) == 0 and not got.d_hidden.any() and not got.d_weight.any()
    assert float(got.row_loss.min()) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_layouts(dtype):
    """Strided, offset and batched inputs give the bits of contiguous ones."""
    h, w, y = make(96, 64, 500, DTYPES[dtype], seed=11)
    want = linear_softmax_grad(h, w, y)

    def wide(x, before, after):
        big = torch.full((x.shape[0], x.shape[1] + before + after), float("nan"), dtype=x.dtype,
                         device="cuda")
        big[:, before:before + x.shape[1]] = x
        return big[:, before:before + x.shape[1]]

    strided_labels = torch.stack([y, y + 1], 1)[:, 0]
    for name, args in {
            "aligned gap": (wide(h, 0, 16), wide(w, 0, 16), y),
            "odd offset": (wide(h, 1, 2), wide(w, 3, 2), y),
            "transposed": (h.t().contiguous().t(), w.t().contiguous().t(), y),
            "labels": (h, w, strided_labels), "int32": (h, w, y.int()),
            "negated views": (torch._neg_view(-h), torch._neg_view(-w), y),
            "batched": (h.reshape(4, 24, 64), w, y.reshape(4, 24)),
            "batch slice": (torch.cat([h.reshape(4, 24, 64)] * 2, 1)[:, :24], w,
                            y.reshape(4, 24))}.items():
        print(f"[case] head layout {name} {dtype}", flush=True)
        got = linear_softmax_grad(*args)
        assert got.d_hidden.shape == args[0].shape and got.lse.shape == args[2].shape
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(b.shape), b), name


@pytest.mark.gpu
def test_no_rows():
    h, w, y = make(4, 16, 20, torch.float32)
    got = linear_softmax_grad(h[:0], w, y[:0])
    assert float(got.loss) == 0 and got.row_loss.numel() == 0 and not got.d_weight.any()
    assert float(linear_softmax_loss(h[:0], w, y[:0]).loss) == 0


@pytest.mark.gpu
def test_large_scores():
    """Scores of thousands: only differences to the maximum are exponentials."""
    h, w, y = make(70, 64, 300, torch.float32, seed=2, spread=600.0)
    _both(h, w, y)
    h, w, y = make(70, 64, 300, torch.bfloat16, seed=2, spread=600.0)
    _both(h, w, y)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [9, 200])
def test_caps_far_above_the_scores_change_nothing(rows):
    """c tanh(s / c) = s - s^3 / (3 c^2) + ...: 4e-6 at c = 10,000 for scores of
    11; rounding adds 2 steps of 2^-24 of tanh's relative error and as much for
    the quotient and the product, 4e-6 together."""
    h, w, y = make(rows, 64, 700, torch.float32, seed=12, spread=2.0)
    assert float((h @ w.T).abs().max()) < 20
    plain = linear_softmax_loss(h, w, y, reduction="sum")
    most = float((h @ w.T).abs().max())
    capped = linear_softmax_loss(h, w, y, reduction="sum", softcap=1e4)
    tol = most ** 3 / 3e8 * 1.1 + 12 * 2.0 ** -24 * most
    assert float((plain.lse - capped.lse).abs().max()) <= tol
    assert float((plain.row_loss - capped.row_loss).abs().max()) <= 2 * tol


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-3, 64.0, 65.0, 1000.0])
def test_caps(cap):
    h, w, y = make(150, 72, 900, torch.float32, seed=13, spread=5.0, left_out=0.2)
    _both(h, w, y, softcap=cap)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_in_several_pieces(dtype):
    """A vocabulary whose exponentials take several pieces of the rows, with
    rows left out, so that pieces are shorter than the host's."""
    vocab = 1_100_003 if dtype == "bf16" else 600_011
    for left in (0.0, 0.5):
        print(f"[case] head pieces {vocab} {dtype} left out {left}", flush=True)
        h, w, y = make(600, 8, vocab, DTYPES[dtype], seed=4, left_out=left)
        got = linear_softmax_grad(h, w, y)
        Head(h, w, y).check(got)
        del got
        torch.cuda.empty_cache()


@pytest.mark.gpu
def test_wide_rows_in_several_pieces():
    """As above with both products in one launch."""
    print("[case] head pieces 2700 x 264 x 262147", flush=True)
    h, w, y = make(2700, 264, 262147, torch.bfloat16, seed=4, left_out=0.1)
    got = linear_softmax_grad(h, w, y)
    Head(h, w, y).check(got)
    del got
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows", [5, 300])
def test_nan_stays_where_it_belongs(rows, dtype):
    """A NaN in a counting row: its own loss and d_hidden, and all of d_weight;
    the other rows are what they are without it."""
    print(f"[case] head NaN {rows} {dtype}", flush=True)
    h, w, y = make(rows, 64, 500, DTYPES[dtype], seed=17)
    want = linear_softmax_grad(h, w, y, reduction="sum")
    few = linear_softmax_loss(h, w, y, reduction="sum")
    h[2, 5] = float("nan")
    others = torch.arange(rows, device="cuda") != 2
    got = linear_softmax_grad(h, w, y, reduction="sum")
    for g, x in ((got, want), (linear_softmax_loss(h, w, y, reduction="sum"), few)):
        assert bool(torch.isnan(g.loss)) and bool(torch.isnan(g.row_loss[2]))
        assert bool(torch.isnan(g.lse[2]))
        assert torch.equal(g.row_loss[others], x.row_loss[others])
        assert torch.equal(g.lse[others], x.lse[others])
    assert bool(torch.isnan(got.d_hidden[2]).all()) and bool(torch.isnan(got.d_weight).all())
    assert torch.equal(got.d_hidden[others], want.d_hidden[others])


@pytest.mark.gpu
def test_one_token_without_a_batch():
    h, w, y = make(1, 64, 300, torch.bfloat16, seed=1)
    want = linear_softmax_grad(h, w, y)
    got = linear_softmax_grad(h[0], w, y[0])
    assert got.row_loss.shape == () and got.d_hidden.shape == (64,)
    assert torch.equal(got.d_hidden, want.d_hidden[0]) and torch.equal(got.loss, want.loss)
    score = linear_softmax_loss(h[0], w, y[0])
    assert abs(float(score.row_loss) - float(want.row_loss)) <= 1e-5 * abs(float(want.row_loss))


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls that overlap have workspaces of their own."""
    cases = [make(400, 128, 3000, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [linear_softmax_grad(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(linear_softmax_grad(*cases[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            for a, b in zip(g, want[k]):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_gradient_is_the_difference_quotient():
    """Central differences of the kernel's loss along random directions.  The
    loss's rounding (2^-24 of about 8, over a step of 2^-5) and the third
    derivative (at most step^2 / 6 of a few cubes of |W| |d| < 4) stay below
    1e-4 + 2e-2 |gradient|; the sum of a wrong sign or factor would not."""
    h, w, y = make(50, 40, 333, torch.float32, seed=8, left_out=0.2)
    kw = dict(softcap=8.0, z_loss=0.01, reduction="mean")
    got = linear_softmax_grad(h, w, y, **kw)
    g = torch.Generator().manual_seed(1)
    step = 2.0 ** -5
    for x, grad, at in ((h, got.d_hidden, 0), (w, got.d_weight, 1)):
        for _ in range(4):
            d = torch.randn(x.shape, generator=g).cuda()
            d = d / d.norm()
            args = [h, w]
            args[at] = x + step * d
            up = linear_softmax_loss(*args, y, **kw).loss
            args[at] = x - step * d
            down = linear_softmax_loss(*args, y, **kw).loss
            quotient = float(up.double() - down.double()) / (2 * step)
            want = float((grad.double() * d.double()).sum())
            assert abs(quotient - want) < 1e-4 + 2e-2 * abs(want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 300])
def test_streams_and_graphs(rows):
    """Another stream than the default one, and two captured graphs replayed
    in turn on inputs that change in place, against eager calls."""
    print(f"[case] head graphs {rows} rows", flush=True)
    h, w, y = make(rows, 64, 700, torch.bfloat16, seed=21)
    h2, w2, y2 = make(rows, 64, 700, torch.bfloat16, seed=22)
    want = linear_softmax_grad(h, w, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_softmax_grad(h, w, y)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs = []
    for args in ((h, w, y), (h2, w2, y2)):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = linear_softmax_grad(*args), linear_softmax_loss(*args)
        graphs.append((g, args, out))
    for k in range(4):
        for g, args, out in graphs:
            args[0].copy_(make(rows, 64, 700, torch.bfloat16, seed=30 + k)[0])
            args[2].copy_(make(rows, 64, 700, torch.bfloat16, seed=40 + k, left_out=0.2)[2])
            g.replay()
        torch.cuda.synchronize()
        for g, args, out in graphs:
            for a, b in zip(out[0], linear_softmax_grad(*args)):
                assert torch.equal(a, b)
            for a, b in zip(out[1], linear_softmax_loss(*args)):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_c_entry_leaves_gaps_alone(dtype):
    """Row strides above the width: what lies between rows stays as it was."""
    print(f"[case] head strides {dtype}", flush=True)
    h, w, y = make(70, 72, 333, DTYPES[dtype], seed=6, left_out=0.1)
    want = linear_softmax_grad(h, w, y)
    L = _native.lib()
    code = {"bf16": 0, "fp16": 1, "fp32": 2}[dtype]
    for pad in (8, 5):
        dh = torch.full((70, 72 + pad), 7.0, dtype=h.dtype, device="cuda")
        dw = torch.full((333, 72 + pad), 7.0, dtype=h.dtype, device="cuda")
        out = torch.full((1 + 70 + 70 + 3,), 7.0, device="cuda")
        size = ctypes.c_int64()
        _native.check(L.bsscl_head_workspace(code, 70, 72, 333, w.data_ptr(), 72, 1,
                                             ctypes.byref(size)))
        ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        _native.check(L.bsscl_head_grad(
            0, None, code, h.data_ptr(), 72, w.data_ptr(), 72, y.data_ptr(), None, 70, 72, 333, 1,
            0.0, 0.0, 1.0, out.data_ptr(), out[1:].data_ptr(), out[71:].data_ptr(), dh.data_ptr(),
            72 + pad, dw.data_ptr(), 72 + pad, ws.data_ptr(), ws.numel()))
        torch.cuda.synchronize()
        assert torch.equal(dh[:, :72], want.d_hidden) and torch.equal(dw[:, :72], want.d_weight)
        assert bool((dh[:, 72:] == 7).all()) and bool((dw[:, 72:] == 7).all())
        assert bool((out[141:] == 7).all()) and torch.equal(out[71:141], want.lse)


def test_exported():
    for name in ("linear_softmax_loss", "linear_softmax_grad", "grad_norm", "clip_grads"):
        assert name in bsscl_gbm.__all__ and callable(getattr(bsscl_gbm, name))

"""grad_norm and clip_grads against float64, their refusals, and the step
that they make together with linear_softmax_grad."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

from bsscl_gbm import _native, clip_grads, grad_norm, linear_softmax_grad  # noqa: E402
from head_model import E, Head, half_step  # noqa: E402

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(sizes, seed=0, scale=1.0, dtypes=DTYPES):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(dtypes[i % len(dtypes)]).cuda()
            for i, n in enumerate(sizes)]


def norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def check(ts, out, norm, max_norm, inv_scale):
    """Squares and their sum are float64: norm is rounded once (and read back
    as float32), the factor once, a product twice (float32, then its dtype)."""
    want = abs(inv_scale) * norm64(ts)
    assert abs(float(norm) - want) <= 2 * E * want
    f = inv_scale * (max_norm / want if want > max_norm else 1.0)
    for t, o in zip(ts, out):
        exact = t.double() * f
        tiny = torch.finfo(t.dtype).smallest_normal * torch.finfo(t.dtype).eps
        tol = (half_step(t.dtype) + 4 * E) * exact.abs() + tiny
        assert bool(((o.double() - exact).abs() <= tol).all())


# -- on the CPU ---------------------------------------------------------------
def test_refuses_lists_on_the_cpu():
    x = torch.zeros(4)
    for bad, what in [([], "empty"), ([x], "GPU"), ([x.numpy()], "torch tensors"),
                      ([x.double()], "must be bfloat16")]:
        with pytest.raises(ValueError, match=what):
            grad_norm(bad)
        with pytest.raises(ValueError, match=what):
            clip_grads(bad, 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grads([x], bad)


def test_c_entries_refuse():
    """Every call is refused on the host before an address is used."""
    L = _native.lib()
    n = 3
    lengths = (ctypes.c_int64 * n)(100, 0, 50)
    codes = (ctypes.c_int32 * n)(0, 1, 2)
    at = [0x10000, 0, 0x20000]
    ptrs = (ctypes.c_void_p * n)(*at)
    size = ctypes.c_int64()
    assert L.bsscl_grad_norm_workspace(n, lengths, ctypes.byref(size)) == 0 and size.value > 0
    assert L.bsscl_grad_norm_workspace(1, (ctypes.c_int64 * 1)(-1), ctypes.byref(size)) == 1
    assert L.bsscl_grad_norm_workspace(-1, None, ctypes.byref(size)) == 1
    norm, ws = ctypes.c_void_p(0x30000), ctypes.c_void_p(0x40000)

    def clip(out=at, ts=ptrs, codes=codes, max_norm=1.0, inv=1.0, norm=norm, ws=ws, size=1 << 20):
        outs = (ctypes.c_void_p * n)(*out)
        return L.bsscl_clip_grads(0, None, n, ts, outs, lengths, codes, inv, max_norm, norm, ws,
                                  size)

    for kw in [dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(inv=float("inf")),
               dict(norm=None), dict(ws=None), dict(ws=ctypes.c_void_p(0x40008)), dict(size=100),
               dict(codes=(ctypes.c_int32 * n)(0, 1, 5)), dict(out=[0, 0, 0x20000]),
               dict(ts=(ctypes.c_void_p * n)(0x10001, 0, 0x20000)),
               dict(out=[0x10002, 0, 0x20000]),       # an out over its own tensor, shifted
               dict(out=[0x20000 - 2, 0, 0x20000]),   # over the other out
               dict(out=[0x50000, 0, 0x50000 + 198]),  # outs over each other
               dict(out=[0x50000, 0, 0x10000])]:      # over another tensor
        assert clip(**kw) == _native.BSSCL_EINVAL, kw
        assert L.bsscl_last_error()


# -- on the GPU ---------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [0], [0, 3, 0], [7, 16384, 16385, 1, 40000],
                                   [5] * 300, [1000003, 13], list(range(1, 260))],
                         ids=["one", "nothing", "empty", "edges", "many", "large", "ragged"])
@pytest.mark.parametrize("inv_scale", [1.0, -1.0 / 128])
def test_norm_and_clip(sizes, inv_scale):
    print(f"[case] clip {len(sizes)} tensors, {sum(sizes)} values, {inv_scale}", flush=True)
    ts = make(sizes, seed=len(sizes))
    full = abs(inv_scale) * norm64(ts)
    assert abs(float(grad_norm(ts, inv_scale=inv_scale)) - full) <= 2 * E * full
    for max_norm in (0.3 * full, 2 * full, 0.0):
        out = [torch.full_like(t, 9.0) for t in ts]
        norm = clip_grads(ts, max_norm, inv_scale=inv_scale, out=out)
        check(ts, out, norm, max_norm, inv_scale)
        same = [t.clone() for t in ts]
        norm2 = clip_grads(same, max_norm, inv_scale=inv_scale)
        assert torch.equal(norm, norm2)
        for a, b in zip(same, out):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_and_orders():
    """Views that begin at odd elements, transposed tensors, and neighbours in
    one buffer that must stay as they are."""
    buf = torch.randn(100001, generator=torch.Generator().manual_seed(1)).cuda()
    for dtype in DTYPES:
        print(f"[case] clip offsets {dtype}", flush=True)
        for a, b, c, d in ((1, 20000, 20001, 100000), (3, 17, 18, 99999), (8, 40008, 40016, 80016)):
            x = buf.to(dtype)
            keep = x.clone()
            ts = [x[a:b], x[c:d]]
            want = [t.clone() for t in ts]
            norm = clip_grads(ts, 1.0)
            check(want, ts, norm, 1.0, 1.0)
            rest = torch.ones(len(x), dtype=torch.bool, device="cuda")
            rest[a:b] = False
            rest[c:d] = False
            assert torch.equal(x[rest], keep[rest])
    t = torch.randn(30, 40, 5).cuda().permute(2, 0, 1)
    o = torch.empty_like(t)
    norm = clip_grads([t], 0.5, out=[o])
    check([t], [o], norm, 0.5, 1.0)
    # Tensors and outs of different alignments to 16 bytes.
    x, y = buf.half(), torch.zeros(100001, dtype=torch.float16, device="cuda")
    norm = clip_grads([x[1:90000]], 0.5, out=[y[2:90001]])
    check([x[1:90000]], [y[2:90001]], norm, 0.5, 1.0)
    assert not y[:2].any() and not y[90001:].any()


@pytest.mark.gpu
def test_values_beyond_float32_squares():
    big = torch.full((1000,), 3e38, device="cuda")
    small = torch.full((1000,), 1e-30, device="cuda")
    assert float(grad_norm([small])) == pytest.approx(1e-30 * math.sqrt(1000), rel=1e-6)
    assert math.isinf(float(grad_norm([big])))  # beyond float32: nothing is clipped
    ts = [big.clone()]
    clip_grads(ts, 1.0)
    assert torch.equal(ts[0], big)
    for max_norm in (1.0, 1e-4):  # factors below float32's normal range
        ts = [big[:1] / 2]
        clip_grads(ts, max_norm)
        assert float(ts[0]) == pytest.approx(max_norm, rel=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_norms_that_are_not_finite_clip_nothing(bad):
    for dtype in DTYPES:
        ts = make([5000, 33], seed=3, dtypes=[dtype])
        ts[1][7] = bad
        keep = [t.clone() for t in ts]
        norm = clip_grads(ts, 1.0)
        assert not math.isfinite(float(norm))
        for a, b in zip(ts, keep):
            assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


@pytest.mark.gpu
def test_refuses_overlaps_and_gaps():
    x = torch.ones(100, device="cuda")
    for ts in ([x, x], [x, x[50:]], [x[:60], x[40:]]):
        with pytest.raises(ValueError, match="overlap"):
            clip_grads(ts, 1.0)
        assert bool((x == 1).all())
        assert float(grad_norm(ts)) == pytest.approx(norm64(ts))  # reading twice is fine
    for t in (x[::2], x.expand(3, 100)):
        with pytest.raises(ValueError, match="dense"):
            clip_grads([t], 1.0)
    for out in ([x.half()], [x[:50]], [x, x], [torch.ones(10, 10, device="cuda")]):
        with pytest.raises(ValueError, match="out must match"):
            clip_grads([torch.ones(100, device="cuda")], 1.0, out=out)


@pytest.mark.gpu
def test_streams_and_graphs():
    print("[case] clip graphs", flush=True)
    sizes = [40000, 5, 17777] * 60
    lists = [make(sizes, seed=1), make(sizes, seed=2)]
    graphs = []
    for ts in lists:
        out = [torch.empty_like(t) for t in ts]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norm = clip_grads(ts, 1.0, inv_scale=0.5, out=out)
        graphs.append((g, ts, out, norm))
    side = torch.cuda.Stream()
    for k in range(3):
        for g, ts, out, norm in graphs:
            for t in ts:
                t.mul_(1.5)
            g.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        for g, ts, out, norm in graphs:
            with torch.cuda.stream(side):
                other = [torch.empty_like(t) for t in ts]
                again = clip_grads(ts, 1.0, inv_scale=0.5, out=other)
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(again, norm)
            for a, b in zip(other, out):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_training_step_with_the_head(dtype):
    """Loss and gradient, norm, clipping and the update, three steps, each
    against float64 from the same inputs."""
    print(f"[case] step {dtype}", flush=True)
    g = torch.Generator().manual_seed(5)
    h = torch.randn(90, 48, generator=g).to(dtype).cuda()
    w = (torch.randn(400, 48, generator=g) * 0.3).to(dtype).cuda()
    y = torch.randint(-1, 400, (90,), generator=g).cuda()
    scale, max_norm = 256.0, 0.05
    for _ in range(3):
        got = linear_softmax_grad(h, w, y, grad_scale=scale)
        Head(h, w, y, grad_scale=scale).check(got)
        grads = [got.d_hidden, got.d_weight]
        before = [t.clone() for t in grads]
        norm = clip_grads(grads, max_norm, inv_scale=1.0 / scale)
        check(before, grads, norm, max_norm, 1.0 / scale)
        assert norm64(grads) <= max_norm * (1 + 2 * half_step(dtype))
        w = (w.float() - 2.0 * grads[1].float()).to(dtype)


@pytest.mark.gpu
def test_factors_next_to_the_smallest_normal_float32():
    """Factors that are 1 but for a power of two scale all the same."""
    x = torch.linspace(1.0, 2.0, 1000, device="cuda")
    for inv_scale in (2.0 ** -126, math.nextafter(2.0 ** -126, 0.0), 2.0 ** -127):
        t, o = x.clone(), torch.empty_like(x)
        clip_grads([t], 1.0, inv_scale=inv_scale)
        clip_grads([x], 1.0, inv_scale=inv_scale, out=[o])
        assert torch.equal(t, o)
        exact = x.double() * inv_scale
        assert bool(((t.double() - exact).abs() <= 2.0 ** -149).all())


def test_refuses_an_inv_scale_beyond_float32():
    """A factor that float32 holds as infinite would turn zeros into NaN."""
    L = _native.lib()
    norm, ws = ctypes.c_void_p(0x30000), ctypes.c_void_p(0x40000)
    at = (ctypes.c_void_p * 1)(0x10000)
    length, code = (ctypes.c_int64 * 1)(100), (ctypes.c_int32 * 1)(2)
    for inv in (1e39, -1e39, 3.5e38):
        assert L.bsscl_clip_grads(0, None, 1, at, at, length, code, inv, 1.0, norm, ws,
                                  1 << 20) == _native.BSSCL_EINVAL
        assert L.bsscl_grad_norm(0, None, 1, at, length, code, inv, norm, ws,
                                 1 << 20) == _native.BSSCL_EINVAL
        assert b"inv_scale" in L.bsscl_last_error()


@pytest.mark.gpu
def test_refuses_to_write_tensors_that_require_gradients():
    """model.parameters() in the place of their gradients, for one."""
    x = torch.ones(100, device="cuda")
    p = torch.nn.Parameter(x.clone())
    for args, kw in ((([p], 1.0), {}), (([x, p], 1.0), {}), (([p * 2], 1.0), {}),
                     (([x], 1.0), dict(out=[p]))):
        with pytest.raises(ValueError, match="require gradients"):
            clip_grads(*args, **kw)
        assert bool((p == 1).all()) and bool((x == 1).all())
    assert float(grad_norm([p])) == 10.0  # reading is fine
    clip_grads([p], 1.0, out=[x])
    assert float(x[0]) == pytest.approx(0.1)
    with torch.no_grad():
        clip_grads([p], 1.0)
    assert float(p.detach()[0]) == pytest.approx(0.1)


@pytest.mark.gpu
def test_tensors_saved_for_backward_are_known_to_be_written():
    for into_out in (False, True):
        x, o = torch.ones(100, device="cuda"), torch.zeros(100, device="cuda")
        w = torch.ones(100, device="cuda", requires_grad=True)
        written = o if into_out else x
        loss = (w * written).sum()  # saves it
        before = (x._version, o._version)
        clip_grads([x], 1.0, out=[o] if into_out else None)
        assert written._version == before[into_out] + 1
        assert (o, x)[into_out]._version == before[not into_out]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        t = torch.ones(100, device="cuda")
        clip_grads([t], 1.0)
    assert float(t[0]) == pytest.approx(0.1)
    clip_grads([t], 0.5)  # an inference tensor counts no versions
    assert float(t[0]) == pytest.approx(0.05)


@pytest.mark.gpu
def test_out_of_the_same_memory_order():
    """Strides of axes of size 1 say nothing; others, shapes and negated views
    have to match."""
    x = torch.randn(1, 64, generator=torch.Generator().manual_seed(3)).cuda()
    t = torch.as_strided(x, (1, 64), (7, 1))
    o = torch.empty(1, 64, device="cuda")
    check([t], [o], clip_grads([t], 0.5, out=[o]), 0.5, 1.0)
    a, b = torch.ones(8, 16, device="cuda"), torch.ones(16, 8, device="cuda")
    for ts, out in (([a], [b]), ([a], [b.t()]), ([b.t()], [a]), ([a, b], [a.clone(), b.t()]),
                    ([a], [torch._neg_view(a.clone())]), ([a], [a.clone(), b])):
        with pytest.raises(ValueError, match="out must match"):
            clip_grads(ts, 1.0, out=out)
    clip_grads([b.t()], 1.0, out=[torch.empty_like(b).t()])

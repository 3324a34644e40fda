"""linear_softmax_loss and linear_softmax_grad where results go wrong first:
rows that are nearly certain, scores of any size, few rows over many tiles of
classes, a strong z-loss in float16, NaN in whole tiles, the ends of the
allowed sizes."""
import math

import pytest

torch = pytest.importorskip("torch")

from bsscl_gbm import linear_softmax_grad, linear_softmax_loss  # noqa: E402
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

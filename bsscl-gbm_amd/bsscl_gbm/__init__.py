"""bsscl-gbm on MI355X: the reference's binary histogram-GBM estimator
(src/bsscl_gbm/__init__.py:5-9 exports HybridHistGBMNumbaV1_0_1) backed by
hand-written HIP kernels for gfx950, and operators on device tensors: the
softmax head over a large vocabulary, the norm and clipping of gradients."""

from .estimator import HybridHistGBMNumbaV1_0_1
from .tensor_ops import clip_grads, grad_norm, linear_softmax_grad, linear_softmax_loss

__version__ = "1.0.1"
__all__ = ["HybridHistGBMNumbaV1_0_1", "linear_softmax_loss", "linear_softmax_grad", "grad_norm",
           "clip_grads"]

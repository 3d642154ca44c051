"""Symbolic tensor of the graph IR (counterpart of the reference's tensor.py:4-25).

A Tensor carries shape / dtype / layout and, once the runtime has planned
memory, a Storage.  Arithmetic sugar builds Op nodes; nothing is computed until
the runtime executes the graph.  dtype is a numpy dtype or utils.BF16.
"""
from __future__ import annotations

from math import prod

from .utils import contiguous_strides


class Tensor:
    __slots__ = ("shape", "dtype", "grad_dtype", "device", "strides", "offset", "is_contiguous",
                 "requires_grad", "grad", "op", "init_val", "storage", "name", "dirty_rows")

    def __init__(self, shape, dtype, strides=None, offset=0, is_contiguous=True, requires_grad=True,
                 init_val=None, device=None, name="", grad_dtype=None):
        self.shape = tuple(shape)
        self.dtype = dtype
        self.grad_dtype = dtype if grad_dtype is None else grad_dtype
        self.device = device
        self.strides = tuple(strides) if strides is not None else contiguous_strides(self.shape)
        self.offset = offset
        self.is_contiguous = is_contiguous
        self.requires_grad = requires_grad
        self.grad = None
        self.op = None          # the OpNode that produces this tensor, None for leaves
        self.init_val = init_val
        self.storage = None
        self.name = name
        # for the gradient of an embedding table: the id lists (storages) whose rows are all
        # that is not zero in it, [] when it is all zero, None when that is not known
        self.dirty_rows = None

    # -- autograd entry (tensor.py:27-30) ---------------------------------------
    def backward(self, grad_scale=1.0, accumulate_parameter_grads=False):
        from .runtime import Runtime
        Runtime.get_default().backward(self, grad_scale=grad_scale,
                                       accumulate_parameter_grads=accumulate_parameter_grads)

    @property
    def ndim(self):
        return len(self.shape)

    @property
    def numel(self):
        return prod(self.shape)

    def __repr__(self):
        label = f"{self.name}: " if self.name else ""
        grad = ", requires_grad" if self.requires_grad else ""
        return f"Tensor({label}shape={self.shape} dtype={self.dtype} device={self.device}{grad})"

    # -- op sugar: the reference's names (tensor.py:45-47, 93-105) ---------------
    def __add__(self, other):
        from .op import AddOp
        return AddOp()(self, other)

    def __mul__(self, other):
        from .op import MulOp
        return MulOp()(self, other)

    def exp(self):
        from .op import ExpOp
        return ExpOp()(self)

    def log(self):
        from .op import LogOp
        return LogOp()(self)

    def rsqrt(self):
        from .op import RsqrtOp
        return RsqrtOp()(self)

    def softmax(self, dim):
        from .op import SoftmaxOp
        return SoftmaxOp(dim)(self)

    # views and layout changes (tensor.py:57-75)
    def view(self, *shape):
        from .op import ViewOp
        return ViewOp(shape)(self)

    def reshape(self, *shape):
        from .op import ReshapeOp
        return ReshapeOp(shape)(self)

    def transpose(self, dim0, dim1):
        from .op import TransposeOp
        return TransposeOp(dim0, dim1)(self)

    def permute(self, *dims):
        from .op import PermuteOp
        return PermuteOp(dims)(self)

    def contiguous(self):
        from .op import ContiguousOp
        return ContiguousOp()(self)

    def gather(self, weight):
        from .op import GatherOp
        return GatherOp()(self, weight)

    def layer_norm(self, gamma, beta, eps=1e-5):
        from .op import LayerNormOp
        return LayerNormOp(eps=eps)(self, gamma, beta)

    def gelu(self):
        from .op import GELUOp
        return GELUOp()(self)

    def cross_entropy(self, labels, dim=-1):
        from .op import CrossEntropyLossOp
        return CrossEntropyLossOp(dim)(self, labels)

    # -- what logits say about given tokens, and learning from another model's top logits ----
    def token_logprobs(self, tokens, top=0, entropy=False, scale=1.0):
        """TokenLogprobs(logp, entropy, top_ids, top_logp) of softmax(scale * self) over the last axis"""
        from .op import TokenLogprobsOp
        return TokenLogprobsOp(top=top, entropy=entropy, scale=scale)(self, tokens)

    def distill_topk(self, teacher_ids, teacher_values, tail=False, scale=1.0, teacher_scale=1.0):
        """KL divergence of softmax(scale * self) from a teacher's top classes, per row"""
        from .op import TopKDistillOp
        return TopKDistillOp(tail=tail, scale=scale, teacher_scale=teacher_scale)(self, teacher_ids, teacher_values)

    # -- ops the reference only has inside its fused kernels ----------------------
    def rms_norm(self, gamma=None, eps=1e-6):
        from .op import RMSNormOp
        return RMSNormOp(eps=eps)(self, gamma) if gamma is not None else RMSNormOp(eps=eps)(self)

    def add_layer_norm(self, residual, gamma, beta, eps=1e-5):
        """returns (h, y): h = self + residual, y = LayerNorm(h)"""
        from .op import AddLayerNormOp
        return AddLayerNormOp(eps=eps)(self, residual, gamma, beta)

    def add_rms_norm(self, residual, gamma=None, eps=1e-6):
        """returns (h, y): h = self + residual, y = RMSNorm(h)"""
        from .op import AddRMSNormOp
        return AddRMSNormOp(eps=eps)(self, residual, gamma) if gamma is not None \
            else AddRMSNormOp(eps=eps)(self, residual)

    def bias_gelu(self, bias):
        """GELU(self + bias), bias the trailing [C]"""
        from .op import BiasGELUOp
        return BiasGELUOp()(self, bias)

    def relu2(self):
        from .op import ReLUSquaredOp
        return ReLUSquaredOp()(self)

    def swiglu(self):
        from .op import SwiGLUOp
        return SwiGLUOp()(self)

    def embedding_sum(self, wte, wpe):
        from .op import EmbeddingSumOp
        return EmbeddingSumOp()(self, wte, wpe)

"""Node-wise MLP operators on rows of fp32 / bf16 / fp16: layer norm, dropout from the counter hash of the fused epilogues, the
16-bit Linear with its epilogue, and log probabilities of labels with entropy and top alternatives.

They stand beside the fp32 operators of ``ops`` (act_norm, the fused dropouts, linear, node_head): the pieces of a residual block
``x + dropout(linear_act(linear_act(layer_norm(x), W1, b1, "gelu"), W2, b2))`` over node embeddings, and of its answers.  Every
operator takes ``[..., width]`` tensors on a ROCm device (rows of any pitch and alignment; other strides are copied), runs on the
current stream of that device, keeps its sums and statistics in fp32, is differentiable once in every floating input (a second backward
pass raises RuntimeError, a forward-mode tangent NotImplementedError), allocates through torch (so it may be captured into a graph) and
gives the same bits on every call.  No CPU / torch fallback.

The checks, autograd nodes and calls of the C entries are in csrc/ops_mlp.cpp: small calls are bound by the host.
"""
from typing import NamedTuple, Optional, Union

import torch

from . import _lib
from .ops import ACT_CODE, new_dropout_seed

#: activations of linear_act: those of the layers and the two that need a density or a sigmoid
LINEAR_ACT_CODE = {**ACT_CODE, "gelu": 5, "silu": 6}
MAX_NORM_WIDTH, MAX_TOPK = 16384, 64

_native = None


def _host():
    global _native
    if _native is None:
        _native = _lib.load_ops_mlp()
    return _native


def layer_norm(x: torch.Tensor, scale: Optional[torch.Tensor] = None, offset: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * scale + offset`` over the last dimension (biased variance, at most 16384 wide), in x's type.
    ``scale`` / ``offset`` ``[width]``: fp32 or x's type, both of one type; None is 1 / 0.  A row with an infinity or NaN is NaN."""
    return (_native or _host()).layer_norm(x, scale, offset, eps)


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor, None] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + mask * x / (1 - p)`` for ``0 <= p < 1``, in x's type (one rounding).  The mask is the rule of the fused epilogues
    (``ops.dropout_keep_mask(rows, width, p, seed)``, rows counted over the leading dimensions) and is never stored: the backward pass
    forms it again.  ``seed``: an int; an int64 tensor of one element on x's device, read when the kernel runs (a replayed graph takes
    the value it holds then; do not change it between a forward pass and its backward pass); None draws ``ops.new_dropout_seed()`` (a
    graph captured with an int or None keeps that seed: every replay has the same mask).
    A dropped element is 0 even where x is infinite or NaN."""
    if seed is None:
        seed = new_dropout_seed()
    if isinstance(seed, torch.Tensor):
        return (_native or _host()).dropout(x, p, 0, seed, residual)
    seed = int(seed)
    if not 0 <= seed < 1 << 64:
        raise ValueError("dropout: the seed is an unsigned 64-bit number")
    return (_native or _host()).dropout(x, p, seed, None, residual)


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "I",
               residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in bf16 or fp16: x ``[..., K]``, weight ``[N, K]`` and residual ``[..., N]`` of one type,
    bias ``[N]`` in that type or fp32; products and the epilogue in fp32, one rounding at the end.  ``act``: a key of
    ``LINEAR_ACT_CODE``.  fp32 operands go through ``ops.linear`` / ``ops.linear_act_norm``.

    A NaN pre-activation stays NaN through every activation but relu, where it is 0 and passes no gradient (the rule of the layers' own
    relu).

    For the backward pass one bit of every pre-activation is kept (relu, leakyrelu) or its fp16 value (the others), and
    ``dz = dy act'(z)`` is rounded to the operands' type (the matrix cores take 16-bit operands) before dx, dW and db are formed of it:
    gradients through elu, tanh, gelu and silu are good to about two half steps of the operands' type instead of one.  An identity keeps
    and rounds nothing."""
    code = LINEAR_ACT_CODE.get(act)
    if code is None:
        raise NotImplementedError(f"linear_act: activation {act!r} is not provided ({sorted(LINEAR_ACT_CODE)})")
    return (_native or _host()).linear_act(x, weight, bias, code, residual)


class LabelLogprobs(NamedTuple):
    """``logprob`` / ``entropy`` ``[...]`` and ``top_logprob`` / ``top_index`` ``[..., topk]`` (fp32 and int64)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor
    top_index: torch.Tensor


def label_logprobs(logits: torch.Tensor, label: torch.Tensor, topk: int = 0) -> LabelLogprobs:
    """Log-softmax of ``logits`` ``[..., C]`` (fp32 / bf16 / fp16) at ``label`` ``[...]`` (int32 / int64), the entropy of the softmax and
    the ``topk`` (at most 64) largest log probabilities with their indices, largest first, ties to the lowest index; all scores in fp32,
    differentiable in the logits, without an ``[..., C]`` intermediate.

    A negative label stands for none: its log probability is 0 and passes no gradient; a label >= C gives NaN.  A logit of -inf has
    probability 0; a row without a finite logit answers -inf, entropy 0 and gradient 0; +inf or NaN makes its row NaN.  At most 67108856
    rows, 16777215 of more than 1024 logits (a workgroup each)."""
    return LabelLogprobs(*(_native or _host()).label_logprobs(logits, label, topk))

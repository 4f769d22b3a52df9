"""Node-wise MLP operators on rows of fp32 / bf16 / fp16: layer norm, dropout from the counter hash of the fused epilogues, the
16-bit Linear with its epilogue, and log probabilities of labels with entropy and top alternatives.

They stand beside the fp32 operators of ``ops`` (act_norm, the fused dropouts, linear, node_head): the pieces of a residual block
``x + dropout(linear_act(linear_act(layer_norm(x), W1, b1, "gelu"), W2, b2))`` over node embeddings, and of its answers.  Every
operator takes ``[..., width]`` tensors on a ROCm device (rows of any pitch and alignment; other strides are copied), runs on the
current stream of that device, keeps its sums and statistics in fp32, is differentiable once in every floating input, allocates through
torch (so it may be captured into a graph) and gives the same bits on every call.  No CPU / torch fallback.
"""
from typing import NamedTuple, Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check
from .ops import ACT_CODE, _need_cuda, _stream, new_dropout_seed

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}           # SL_F32, SL_BF16, SL_F16
#: activations of linear_act: those of the layers and the two that need a density or a sigmoid
LINEAR_ACT_CODE = {**ACT_CODE, "gelu": 5, "silu": 6}
MAX_NORM_WIDTH, MAX_TOPK = 16384, 64


def _one_device(*ts):
    """All operands on one ROCm device."""
    _need_cuda(*ts)
    dev = None
    for t in ts:
        if t is not None:
            if dev is not None and t.device != dev:
                raise ValueError(f"operands on {dev} and {t.device}")
            dev = t.device
    return dev


def _float_rows(name, t):
    if t.dtype not in _DT:
        raise TypeError(f"{name}: {t.dtype} (float32, bfloat16 or float16)")
    if t.dim() < 1:
        raise ValueError(f"{name}: a tensor of rows is needed")
    return _DT[t.dtype]


def _rows(t: Optional[torch.Tensor]):
    """``t`` as [rows, width] with unit stride along the row and a pitch of at least the width (copied if it has neither)."""
    if t is None:
        return None
    if t.dim() != 2:
        t = t.reshape(t.shape[:-1].numel(), t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
        if t.shape[0] <= 1 or t.stride(0) < t.shape[1]:        # (size-1 dimensions may keep any stride)
            t = t.as_strided(t.shape, (max(1, t.shape[1]), 1))
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _ld(t):
    return 0 if t is None else t.stride(0)


class _on:
    """The device guard of a launch: the kernels of a device are launched with it current."""
    __slots__ = ("d", "back")

    def __init__(self, device):
        self.d = device.index

    def __enter__(self):
        self.back = torch._C._cuda_getDevice()
        if self.back != self.d:
            torch._C._cuda_setDevice(self.d)

    def __exit__(self, *a):
        if self.back != self.d:
            torch._C._cuda_setDevice(self.back)


def _needs_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ---------------------------------------------------------------- layer norm

def _ln_fwd(x, scale, offset, eps, want_stats):
    x2 = _rows(x)
    n, F = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(n, 2, dtype=torch.float32, device=x.device) if want_stats else None
    w = scale if scale is not None else offset
    if n:
        with _on(x.device):
            check(_lib.load().sl_layer_norm_fwd(_DT[x.dtype], 0 if w is None else _DT[w.dtype], x2.data_ptr(), x2.stride(0), _ptr(scale), _ptr(offset),
                                                n, F, eps, y.data_ptr(), F, _ptr(stats), _stream(x)))
    return y, stats, x2


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, offset, eps):
        y, stats, _ = _ln_fwd(x, scale, offset, eps, True)
        ctx.save_for_backward(x, scale, offset, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, scale, offset, stats = ctx.saved_tensors
        x2, dy2 = _rows(x), _rows(dy)
        n, F = x2.shape
        need = ctx.needs_input_grad
        lib = _lib.load()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        ds = torch.empty_like(scale) if scale is not None and need[1] else None
        do = torch.empty_like(offset) if offset is not None and need[2] else None
        part = None
        if ds is not None or do is not None:
            part = torch.empty(max(1, int(lib.sl_layer_norm_partial_floats(n, F))), dtype=torch.float32, device=x.device)
        w = scale if scale is not None else offset
        with _on(x.device):
            check(lib.sl_layer_norm_bwd(_DT[x.dtype], 0 if w is None else _DT[w.dtype], x2.data_ptr(), x2.stride(0), dy2.data_ptr(), dy2.stride(0),
                                        _ptr(scale), _ptr(stats), n, F, _ptr(dx), F, _ptr(ds), _ptr(do), _ptr(part), _stream(x)))
        return dx, ds, do, None


def layer_norm(x: torch.Tensor, scale: Optional[torch.Tensor] = None, offset: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * scale + offset`` over the last dimension (biased variance, at most 16384 wide), in x's type.
    ``scale`` / ``offset`` ``[width]``: fp32 or x's type, both of one type; None is 1 / 0.  A row with an infinity or NaN is NaN."""
    _float_rows("layer_norm", x)
    F = x.shape[-1]
    if not 1 <= F <= MAX_NORM_WIDTH:
        raise ValueError(f"layer_norm: rows of {F} elements (1 to {MAX_NORM_WIDTH})")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps {eps}")
    kinds = {t.dtype for t in (scale, offset) if t is not None}
    if len(kinds) > 1 or not kinds <= {torch.float32, x.dtype}:
        raise TypeError(f"layer_norm: scale / offset of type {kinds} for rows of {x.dtype}")
    for t in (scale, offset):
        if t is not None and tuple(t.shape) != (F,):
            raise ValueError(f"layer_norm: scale / offset of shape {tuple(t.shape)} for rows of {F}")
    _one_device(x, scale, offset)
    if _needs_grad(x, scale, offset):
        scale, offset = (None if t is None else t.contiguous() for t in (scale, offset))
        return _LayerNorm.apply(x, scale, offset, float(eps))
    return _ln_fwd(x, None if scale is None else scale.contiguous(), None if offset is None else offset.contiguous(), float(eps), False)[0]


# ---------------------------------------------------------------- dropout

def _drop(x, p, seed, residual):
    x2, r2 = _rows(x), _rows(residual)
    n, F = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    host, dev = (0, seed.data_ptr()) if isinstance(seed, torch.Tensor) else (seed, None)
    if n and F:
        with _on(x.device):
            check(_lib.load().sl_dropout(_DT[x.dtype], x2.data_ptr(), x2.stride(0), _ptr(r2), _ld(r2), n, F, p, host, dev, y.data_ptr(), F, _stream(x)))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, seed, p):
        ctx.p = p
        ctx.seed = None if isinstance(seed, torch.Tensor) else seed
        ctx.save_for_backward(seed if ctx.seed is None else None)
        return _drop(x, p, seed, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        seed = ctx.saved_tensors[0] if ctx.seed is None else ctx.seed
        dx = _drop(dy, ctx.p, seed, None) if ctx.needs_input_grad[0] else None
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor, None] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + mask * x / (1 - p)`` for ``0 <= p < 1``, in x's type (one rounding).  The mask is the rule of the fused epilogues
    (``ops.dropout_keep_mask(rows, width, p, seed)``, rows counted over the leading dimensions) and is never stored: the backward pass
    forms it again.  ``seed``: an int; an int64 tensor of one element on x's device, read when the kernel runs (a replayed graph takes
    the value it holds then; do not change it between a forward pass and its backward pass); None draws ``ops.new_dropout_seed()``.
    A dropped element is 0 even where x is infinite or NaN."""
    _float_rows("dropout", x)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout: probability {p} (0 <= p < 1)")
    if not float(p) < 1.0 - 2.0 ** -25:
        raise ValueError(f"dropout: probability {p} rounds to 1 in fp32")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"dropout: residual {residual.dtype} {tuple(residual.shape)} for x {x.dtype} {tuple(x.shape)}")
    if seed is None:
        seed = new_dropout_seed()
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError("dropout: a seed tensor is one int64")
        _one_device(x, residual, seed)
    else:
        seed = int(seed)
        if not 0 <= seed < 1 << 64:
            raise ValueError("dropout: the seed is an unsigned 64-bit number")
        _one_device(x, residual)
    if _needs_grad(x, residual):
        return _Dropout.apply(x, residual, seed, float(p))
    return _drop(x, float(p), seed, residual)


# ---------------------------------------------------------------- the 16-bit Linear

def _lin_fwd(x, W, b, residual, act, keep):
    x2, r2, W = _rows(x), _rows(residual), _rows(W)
    M, K = x2.shape
    N = W.shape[0]
    y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device)
    lib = _lib.load()
    kept = torch.empty(max(16, int(lib.sl_linear16_kept_bytes(act, M, N))), dtype=torch.uint8, device=x.device) if keep else None
    if M:
        with _on(x.device):
            check(lib.sl_linear16_fwd(_DT[x.dtype], x2.data_ptr(), x2.stride(0), W.data_ptr(), W.stride(0), _ptr(b),
                                      int(b is not None and b.dtype == torch.float32), _ptr(r2), _ld(r2), M, N, K, act,
                                      y.data_ptr(), N, _ptr(kept), _stream(x)))
    return y, kept


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W, b, residual, act):
        y, kept = _lin_fwd(x, W, b, residual, act, act != 0)
        ctx.act = act
        ctx.bias = None if b is None else b.dtype
        ctx.save_for_backward(x, W, kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, W, kept = ctx.saved_tensors
        x2, w2, dy2 = _rows(x), _rows(W), _rows(dy)
        M, K = x2.shape
        N = w2.shape[0]
        need = ctx.needs_input_grad
        dres = dy if need[3] else None
        if not any(need[:3]):
            return None, None, None, dres, None
        lib = _lib.load()
        dev = x.device
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
        db = torch.empty(N, dtype=ctx.bias, device=dev) if ctx.bias is not None and need[2] else None
        dW = torch.empty(N, K, dtype=x.dtype, device=dev) if need[1] or db is not None else None
        ws = torch.empty(max(16, int(lib.sl_linear16_bwd_scratch_bytes(ctx.act, M, N, K))), dtype=torch.uint8, device=dev)
        with _on(dev):
            check(lib.sl_linear16_bwd(_DT[x.dtype], x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0), dy2.data_ptr(), dy2.stride(0),
                                      _ptr(kept), M, N, K, ctx.act, _ptr(dx), K, _ptr(dW), K, _ptr(db), int(ctx.bias == torch.float32),
                                      ws.data_ptr(), _stream(x)))
        return dx, (dW if need[1] else None), db, dres, None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "I",
               residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in bf16 or fp16: x ``[..., K]``, weight ``[N, K]`` and residual ``[..., N]`` of one type,
    bias ``[N]`` in that type or fp32; products and the epilogue in fp32, one rounding at the end.  ``act``: a key of
    ``LINEAR_ACT_CODE``.  fp32 operands go through ``ops.linear`` / ``ops.linear_act_norm``.

    For the backward pass one bit of every pre-activation is kept (relu, leakyrelu) or its fp16 value (the others), and
    ``dz = dy act'(z)`` is rounded to the operands' type (the matrix cores take 16-bit operands); an identity keeps and rounds nothing."""
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"linear_act: {x.dtype} (bfloat16 or float16; fp32 products are ops.linear / ops.linear_act_norm)")
    _float_rows("linear_act", x)
    if act not in LINEAR_ACT_CODE:
        raise NotImplementedError(f"linear_act: activation {act!r} is not provided ({sorted(LINEAR_ACT_CODE)})")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.dtype != x.dtype or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"linear_act: weight {weight.dtype} {tuple(weight.shape)} for x {x.dtype} {tuple(x.shape)}")
    N = weight.shape[0]
    if bias is not None and (tuple(bias.shape) != (N,) or bias.dtype not in (torch.float32, x.dtype)):
        raise ValueError(f"linear_act: bias {bias.dtype} {tuple(bias.shape)} for {N} outputs of {x.dtype}")
    if residual is not None and (residual.shape != x.shape[:-1] + (N,) or residual.dtype != x.dtype):
        raise ValueError(f"linear_act: residual {residual.dtype} {tuple(residual.shape)} for an output of {x.dtype} {tuple(x.shape[:-1]) + (N,)}")
    _one_device(x, weight, bias, residual)
    bias = None if bias is None else bias.contiguous()
    if _needs_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, LINEAR_ACT_CODE[act])
    return _lin_fwd(x, weight, bias, residual, LINEAR_ACT_CODE[act], False)[0]


# ---------------------------------------------------------------- log probabilities of labels

class LabelLogprobs(NamedTuple):
    """``logprob`` / ``entropy`` ``[...]`` and ``top_logprob`` / ``top_index`` ``[..., topk]`` (fp32 and int64)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor
    top_index: torch.Tensor


def _lp_fwd(x, label, k):
    x2 = _rows(x)
    n, C = x2.shape
    lead, dev = x.shape[:-1], x.device
    lib = _lib.load()
    stat = torch.empty((4,) + lead, dtype=torch.float32, device=dev)        # logprob, entropy, (maximum, log2-sum) pairs
    top = torch.empty(lead + (k,), dtype=torch.float32, device=dev)
    idx = torch.empty(lead + (k,), dtype=torch.int64, device=dev)
    if n:
        need = int(lib.sl_label_logprobs_scratch_bytes(_DT[x.dtype], n, C, k))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        s = stat.data_ptr()
        with _on(dev):
            check(lib.sl_label_logprobs_fwd(_DT[x.dtype], x2.data_ptr(), x2.stride(0), label.data_ptr(), int(label.dtype == torch.int64), n, C, k,
                                            s, s + 4 * n, s + 8 * n, top.data_ptr(), idx.data_ptr(), _ptr(ws), _stream(x)))
    return stat[0], stat[1], top, idx, stat[2:]


class _LabelLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, label, k):
        lp, ent, top, idx, rowstat = _lp_fwd(x, label, k)
        ctx.k = k
        ctx.save_for_backward(x, label, ent, idx, rowstat)
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)
        return lp, ent, top, idx

    @staticmethod
    @once_differentiable
    def backward(ctx, dlp, dent, dtop, _didx):
        if dlp is None and dent is None and dtop is None:
            return None, None, None
        x, label, ent, idx, rowstat = ctx.saved_tensors
        x2 = _rows(x)
        n, C = x2.shape
        g = [None if t is None or t.numel() == 0 else t.contiguous() for t in (dlp, dent, dtop)]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if n:
            with _on(x.device):
                check(_lib.load().sl_label_logprobs_bwd(_DT[x.dtype], x2.data_ptr(), x2.stride(0), label.data_ptr(), int(label.dtype == torch.int64),
                                                        n, C, ctx.k, rowstat.data_ptr(), ent.data_ptr(), _ptr(idx), _ptr(g[0]), _ptr(g[1]), _ptr(g[2]),
                                                        dx.data_ptr(), C, _stream(x)))
        return dx, None, None


def label_logprobs(logits: torch.Tensor, label: torch.Tensor, topk: int = 0) -> LabelLogprobs:
    """Log-softmax of ``logits`` ``[..., C]`` (fp32 / bf16 / fp16) at ``label`` ``[...]`` (int32 / int64), the entropy of the softmax and
    the ``topk`` (at most 64) largest log probabilities with their indices, largest first, ties to the lowest index; all scores in fp32,
    differentiable in the logits, without an ``[..., C]`` intermediate.

    A negative label stands for none: its log probability is 0 and passes no gradient; a label >= C gives NaN.  A logit of -inf has
    probability 0; a row without a finite logit answers -inf, entropy 0 and gradient 0; +inf or NaN makes its row NaN."""
    _float_rows("label_logprobs", logits)
    C = logits.shape[-1]
    if label.dtype not in (torch.int32, torch.int64) or label.shape != logits.shape[:-1]:
        raise ValueError(f"label_logprobs: label {label.dtype} {tuple(label.shape)} for logits {tuple(logits.shape)}")
    if C < 1 or not 0 <= int(topk) <= min(C, MAX_TOPK):
        raise ValueError(f"label_logprobs: topk {topk} of {C} classes (at most {MAX_TOPK})")
    _one_device(logits, label)
    label = label.contiguous()
    if _needs_grad(logits):
        return LabelLogprobs(*_LabelLogprobs.apply(logits, label, int(topk)))
    return LabelLogprobs(*_lp_fwd(logits, label, int(topk))[:4])

"""CPU: what the node-wise MLP operators (shadow_gnn_amd/ops_mlp.py, sl_layer_norm_* / sl_dropout / sl_linear16_* /
sl_label_logprobs_*) refuse, at the Python entries and at the C entries -- before anything reaches a GPU."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from shadow_gnn_amd import _lib, ops_mlp

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: ops_mlp.layer_norm(_t(4, 8, dtype=torch.float64)), TypeError),
    (lambda: ops_mlp.layer_norm(_t(4, 8, dtype=torch.int32)), TypeError),
    (lambda: ops_mlp.layer_norm(_t(4, 0)), ValueError),
    (lambda: ops_mlp.layer_norm(_t(1, 16385)), ValueError),
    (lambda: ops_mlp.layer_norm(_t(4, 8), eps=-1.0), ValueError),
    (lambda: ops_mlp.layer_norm(_t(4, 8), eps=float("nan")), ValueError),
    (lambda: ops_mlp.layer_norm(_t(4, 8), _t(8, dtype=F16)), TypeError),
    (lambda: ops_mlp.layer_norm(_t(4, 8), _t(8, dtype=F32), _t(8)), TypeError),
    (lambda: ops_mlp.layer_norm(_t(4, 8, dtype=F32), _t(8)), TypeError),
    (lambda: ops_mlp.layer_norm(_t(4, 8), _t(7)), ValueError),
    (lambda: ops_mlp.layer_norm(_t(4, 8), None, _t(8, 1)), ValueError),
    (lambda: ops_mlp.layer_norm(_t(4, 8)), RuntimeError),                      # a CPU tensor: there is no fallback
    (lambda: ops_mlp.dropout(_t(4, 8), 1.0, 1), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), -0.1, 1), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), float("nan"), 1), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), 1.0 - 2.0 ** -40, 1), ValueError),      # 1 in fp32
    (lambda: ops_mlp.dropout(_t(4, 8), 0.5, -1), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), 0.5, 1 << 64), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), 0.5, torch.zeros(2, dtype=torch.int64)), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), 0.5, torch.zeros(1, dtype=torch.int32)), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), 0.5, 1, residual=_t(4, 7)), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), 0.5, 1, residual=_t(1, 8)), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), 0.5, 1, residual=_t(4, 8, dtype=F32)), ValueError),
    (lambda: ops_mlp.dropout(_t(4, 8), 0.5, 1), RuntimeError),
    (lambda: ops_mlp.linear_act(_t(4, 8, dtype=F32), _t(5, 8, dtype=F32)), TypeError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(5, 8), act="prelu"), NotImplementedError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(5, 7)), ValueError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(5, 8, dtype=F16)), ValueError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(0, 8)), ValueError),
    (lambda: ops_mlp.linear_act(_t(4, 0), _t(5, 0)), ValueError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(5, 8), _t(4)), ValueError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(5, 8), _t(5, dtype=F16)), ValueError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(5, 8), residual=_t(4, 8)), ValueError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(5, 8), residual=_t(4, 5, dtype=F32)), ValueError),
    (lambda: ops_mlp.linear_act(_t(4, 8), _t(5, 8)), RuntimeError),
    (lambda: ops_mlp.label_logprobs(_t(4, 8), torch.zeros(4)), ValueError),
    (lambda: ops_mlp.label_logprobs(_t(4, 8), torch.zeros(3, dtype=torch.int64)), ValueError),
    (lambda: ops_mlp.label_logprobs(_t(4, 8), torch.zeros(4, dtype=torch.int64), topk=9), ValueError),
    (lambda: ops_mlp.label_logprobs(_t(4, 100), torch.zeros(4, dtype=torch.int64), topk=65), ValueError),
    (lambda: ops_mlp.label_logprobs(_t(4, 8), torch.zeros(4, dtype=torch.int64), topk=-1), ValueError),
    (lambda: ops_mlp.label_logprobs(_t(4, 0), torch.zeros(4, dtype=torch.int64)), ValueError),
    (lambda: ops_mlp.label_logprobs(_t(4, 8, dtype=torch.int64), torch.zeros(4, dtype=torch.int64)), TypeError),
    (lambda: ops_mlp.label_logprobs(_t(4, 8), torch.zeros(4, dtype=torch.int64)), RuntimeError),
])
def test_python_entries_refuse(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call,shape", [
    (lambda t: ops_mlp.layer_norm(t), (4, 8)),
    (lambda t: ops_mlp.layer_norm(_t(4, 8, dtype=F32), t), (8,)),
    (lambda t: ops_mlp.layer_norm(_t(4, 8, dtype=F32), _t(8, dtype=F32), t), (8,)),
    (lambda t: ops_mlp.dropout(t, 0.5, 1), (4, 8)),
    (lambda t: ops_mlp.dropout(_t(4, 8, dtype=F32), 0.5, 1, residual=t), (4, 8)),
    (lambda t: ops_mlp.linear_act(t.to(BF16), _t(5, 8)), (4, 8)),
    (lambda t: ops_mlp.linear_act(_t(4, 8), t.to(BF16)), (5, 8)),
    (lambda t: ops_mlp.linear_act(_t(4, 8), _t(5, 8), t), (5,)),
    (lambda t: ops_mlp.linear_act(_t(4, 8), _t(5, 8), residual=t.to(BF16)), (4, 5)),
    (lambda t: ops_mlp.label_logprobs(t, torch.zeros(4, dtype=torch.int64)), (4, 8)),
])
def test_forward_mode_tangents_are_refused(call, shape, grad):
    """A tangent of any floating input, also where nothing requires a gradient: an error, not an output without one."""
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = forward_ad.make_dual(torch.zeros(*shape), torch.ones(*shape))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)


_BUF = (C.c_char * 4096)()
P = (C.addressof(_BUF) + 255) // 256 * 256          # a host address: the calls below return before any kernel could see it


@pytest.mark.parametrize("name,args", [
    ("sl_layer_norm_fwd", (3, 0, P, 8, None, None, 1, 8, 1e-5, P, 8, None, None)),            # type
    ("sl_layer_norm_fwd", (1, 2, P, 8, P, None, 1, 8, 1e-5, P, 8, None, None)),               # weight type
    ("sl_layer_norm_fwd", (1, 0, P, 8, None, None, 1, 0, 1e-5, P, 8, None, None)),            # width
    ("sl_layer_norm_fwd", (1, 0, P, 16385, None, None, 1, 16385, 1e-5, P, 16385, None, None)),
    ("sl_layer_norm_fwd", (1, 0, P, 7, None, None, 1, 8, 1e-5, P, 8, None, None)),            # pitch
    ("sl_layer_norm_fwd", (1, 0, P, 8, None, None, 1, 8, -1.0, P, 8, None, None)),            # eps
    ("sl_layer_norm_fwd", (1, 0, None, 8, None, None, 1, 8, 1e-5, P, 8, None, None)),         # null
    ("sl_layer_norm_bwd", (1, 0, P, 8, P, 8, None, None, 1, 8, P, 8, None, None, None, None)),   # no statistics
    ("sl_layer_norm_bwd", (1, 0, P, 8, P, 8, None, P, 5000, 8, P, 8, P, None, None, None)),      # weight gradient without scratch
    ("sl_layer_norm_bwd", (1, 0, P, 8, P, 8, None, P, 1, 8, P, 4, None, None, None, None)),      # pitch
    ("sl_dropout", (4, P, 8, None, 0, 1, 8, 0.5, 1, None, P, 8, None)),
    ("sl_dropout", (1, P, 8, None, 0, 1, 8, 1.0, 1, None, P, 8, None)),
    ("sl_dropout", (1, P, 8, None, 0, 1, 8, float("nan"), 1, None, P, 8, None)),
    ("sl_dropout", (1, P, 4, None, 0, 1, 8, 0.5, 1, None, P, 8, None)),
    ("sl_dropout", (1, P, 8, P, 4, 1, 8, 0.5, 1, None, P, 8, None)),
    ("sl_dropout", (1, P, 8, None, 0, 1, 8, 0.5, 1, None, None, 8, None)),
    ("sl_linear16_fwd", (0, P, 8, P, 8, None, 0, None, 0, 1, 8, 8, 0, P, 8, None, None)),     # fp32
    ("sl_linear16_fwd", (1, P, 8, P, 8, None, 0, None, 0, 1, 8, 8, 7, P, 8, None, None)),     # activation
    ("sl_linear16_fwd", (1, P, 8, P, 8, None, 0, None, 0, 1, 0, 8, 0, P, 8, None, None)),     # N = 0
    ("sl_linear16_fwd", (1, P, 4, P, 8, None, 0, None, 0, 1, 8, 8, 0, P, 8, None, None)),     # pitch
    ("sl_linear16_fwd", (1, P, 8, P, 8, None, 0, P, 4, 1, 8, 8, 0, P, 8, None, None)),        # residual pitch
    ("sl_linear16_fwd", (1, P, 8, P, 8, None, 0, None, 0, 1, 8, 8, 1, P, 8, P + 8, None)),       # alignment of what is kept
    ("sl_linear16_bwd", (1, P, 8, P, 8, P, 8, None, 1, 8, 8, 1, P, 8, None, 0, None, 0, P, None)),    # an activation without what it kept
    ("sl_linear16_bwd", (1, P, 8, P, 8, P, 8, None, 1, 8, 8, 0, P, 8, None, 0, P, 0, P, None)),       # db without dW
    ("sl_linear16_bwd", (1, P, 8, P, 8, P, 8, None, 1, 8, 8, 0, P, 8, None, 0, None, 0, None, None)),  # no scratch
    ("sl_label_logprobs_fwd", (5, P, 8, P, 1, 1, 8, 0, P, P, P, None, None, None, None)),
    ("sl_label_logprobs_fwd", (1, P, 8, P, 1, 1, 8, 9, P, P, P, P, P, None, None)),              # k > C
    ("sl_label_logprobs_fwd", (1, P, 100, P, 1, 1, 100, 65, P, P, P, P, P, None, None)),         # k > 64
    ("sl_label_logprobs_fwd", (1, P, 4, P, 1, 1, 8, 0, P, P, P, None, None, None, None)),        # pitch
    ("sl_label_logprobs_fwd", (1, P, 8, P, 1, 1, 8, 2, P, P, P, None, None, None, None)),        # no place for the alternatives
    ("sl_label_logprobs_fwd", (1, P, 131072, P, 1, 1, 131072, 0, P, P, P, None, None, None, None)),   # a split row without scratch
    ("sl_label_logprobs_bwd", (1, P, 8, P, 1, 1, 8, 0, P, P, None, None, None, None, None, 8, None)),  # no dx
    ("sl_label_logprobs_bwd", (1, P, 8, P, 1, 1, 8, 2, P, P, None, None, None, P, P, 8, None)),        # dtop without indices
    ("sl_dropout", (1, P, 1 << 32, None, 0, 1, (1 << 31) + 8, 0.5, 1, None, P, 1 << 32, None)),        # columns are counted in 32 bits
    ("sl_linear16_fwd", (1, P, 4, P, 4, None, 0, None, 0, (1 << 31) - 1, 1, 4, 0, P, 1, None, None)),   # a launch of 2^32 threads and more
    ("sl_linear16_fwd", (1, P, 8, P, 8, None, 0, None, 0, (1 << 31) - 1, 1 << 24, 8, 0, P, 1 << 24, None, None)),
    ("sl_linear16_bwd", (1, P, 8, P, 8, P, 1 << 22, None, (1 << 31) - 1, 72, 8, 0, P, 8, None, 0, None, 0, P, None)),
    ("sl_linear16_bwd", (1, P, 1 << 24, P, 1 << 24, P, 1 << 24, None, 1, 1 << 24, 1 << 24, 0, P, 1 << 24, None, 0, None, 0, P, None)),
    ("sl_label_logprobs_fwd", (1, P, 2000, P, 1, 1 << 25, 2000, 0, P, P, P, None, None, None, None)),
])
def test_c_entries_refuse(name, args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == _lib.SG_ERR_INVALID
    assert lib.sg_last_error()


def test_sizes_of_scratch():
    lib = _lib.load()
    assert lib.sl_layer_norm_partial_floats(0, 64) == 0
    assert lib.sl_layer_norm_partial_floats(1, 64) == 0                      # one workgroup writes the gradient itself
    assert lib.sl_layer_norm_partial_floats(100000, 64) >= 128
    assert lib.sl_layer_norm_partial_floats(1 << 20, 20000) == 0
    assert lib.sl_label_logprobs_scratch_bytes(0, 1000, 47, 5) == 0          # rows in registers
    assert lib.sl_label_logprobs_scratch_bytes(1, 1, 131072, 10) > 0         # one row: split
    assert lib.sl_linear16_bwd_scratch_bytes(1, 0, 8, 8) > 0
    assert lib.sl_linear16_kept_bytes(0, 10, 64) == 0 and lib.sl_linear16_kept_bytes(1, 10, 129) == 320 and lib.sl_linear16_kept_bytes(5, 10, 129) == 10 * 136 * 2
    # the largest weight of the documented range (2^34 tiles): a size, not a division by their number in 32 bits
    assert lib.sl_linear16_bwd_scratch_bytes(0, 1000, 1 << 24, 1 << 24) > 1 << 48


def test_scratch_of_a_backward_call():
    """The scratch holds what a call goes through memory with: dz where a kernel reads it, the transposed weight where it is read, partial
    products where rows are cut into slices; the size by the shape alone covers every alignment, pitch and set of gradients."""
    lib = _lib.load()

    def size(act, M, N, K, x=P, ldx=None, ldw=None, dy=P, lddy=None, dx=1, dw=1):
        return lib.sl_linear16_bwd_scratch_bytes_for(act, x, ldx or K, ldw or K, dy, lddy or N, M, N, K, dx, dw)

    M, dz, part = 289127, 289127 * 256 * 2, 251 * 256 * 256 * 4               # (slices of 18 stages of 64 rows: 251)
    assert size(0, M, 256, 256) < part + (1 << 20)                              # an identity reads dy as it is
    assert size(1, M, 256, 256) < part + (1 << 20)                              # relu: both products mask dy themselves
    assert dz + part < size(5, M, 256, 256) < dz + part + (1 << 20)             # gelu: dx forms dz, dW reads it
    assert dz + part < size(1, M, 256, 256, dy=P + 2) < dz + part + (1 << 20)   # rows of dy that are not whole words
    assert size(5, M, 256, 256, dw=0) == 0                                      # dx alone: no dz in memory
    assert size(1, 256, 256, 256) == 0                                          # few rows: nothing
    assert size(0, 32768, 4096, 1024, dw=0) == 4096 * 1024 * 2                  # a wide dx: the transposed weight
    assert size(2, 32768, 4096, 1024) == 4096 * (1024 + 32768) * 2 + 4096 * 4
    for act in (0, 1, 5):
        for M in (0, 1, 300, 513, 5000, 20011, 98304):
            for N in (1, 40, 47, 64, 72, 256, 1000, 1001):
                for K in (1, 8, 100, 256, 1024, 1001):
                    most = lib.sl_linear16_bwd_scratch_bytes(act, M, N, K)
                    for x, dy, ldw, dx, dw in ((P, P, K, 1, 1), (P + 2, P, K, 1, 1), (P, P + 2, K, 1, 1), (P + 2, P + 2, 1 << 22, 1, 1), (P, P, K, 1, 0), (P, P + 2, K, 0, 1)):
                        assert size(act, M, N, K, x=x, dy=dy, ldw=ldw, dx=dx, dw=dw) <= most

"""Node-wise MLP operators (shadow_gnn_amd/ops_mlp.py) against plain implementations in 64 bits.

Tolerances are counted, not chosen: an output in t bits is off by at most half a step (eps / 2 of the value) plus what its fp32
computation may lose, u = 2^-24 per operation on the magnitudes that enter it; each test states its count."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _assert_within(got, want, tol, what):
    """|got - want| <= half a step of got's type + tol, element by element; NaN and infinities agree.  What is rounded is the value v
    with |v - want| <= tol, so the half step is one of |v| <= |want| + tol: |got - want| <= tol + eps / 2 (|want| + tol)."""
    got64, want = got.detach().double(), want.detach().double()
    assert got64.shape == want.shape, what
    same = (got64 == want) | (got64.isnan() & want.isnan())
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps      # (a subnormal result: half its step)
    bad = ~same & ~((got64 - want).abs() <= _half(got.dtype) * (want.abs() + tol) * (1 + 1e-6) + tiny + tol)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        t = tol.expand(want.shape)[tuple(at)].item() if isinstance(tol, torch.Tensor) else tol
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {got64[tuple(at)].item()!r} for {want[tuple(at)].item()!r} "
                             f"(tolerance {t:.3g} + half a step)")


def _pitched(t, pitch, shift=0):
    """The values of t as a view of rows `pitch` apart, `shift` elements into its storage."""
    n, F = t.shape
    buf = torch.full((shift + max(1, n) * pitch,), 7.0, dtype=t.dtype, device=t.device)
    v = buf[shift:].as_strided((n, F), (pitch, 1))
    v.copy_(t)
    return v


# ---------------------------------------------------------------- layer norm

def _ln_ref(x, s, o, eps, dy):
    x64 = x.double()
    d = x64 - x64.mean(-1, keepdim=True)
    r = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = d * r
    sc = torch.ones_like(x64[0]) if s is None else s.double()
    y = n * sc + (0 if o is None else o.double())
    g = dy.double() * sc
    dx = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    return y, dx, (dy.double() * n).sum(0), dy.double().sum(0), n, r, g


def _ln_check(x, s, o, eps, dy):
    from shadow_gnn_amd import ops_mlp
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, s, o)]
    y = ops_mlp.layer_norm(*leaves, eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    grads = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    ry, rdx, rds, rdo, n, r, g = _ln_ref(x, s, o, eps, dy)
    ax = x.double().abs().amax(-1, keepdim=True)
    # mean and deviations: at most 16 + 10 roundings per sum of a row, on values up to max|x|; n = d r inherits them times r
    dn = 64 * U * r * ax
    sc = 1.0 if s is None else s.double().abs()
    _assert_within(y, ry, dn * sc + 8 * U * (n.abs() * sc + (0 if o is None else o.double().abs())), "y")
    ag, an = g.abs().amax(-1, keepdim=True), n.abs().amax(-1, keepdim=True)
    _assert_within(next(grads), rdx, r * ag * (64 * U * (1 + an) ** 2 + 4 * dn * (1 + an)), "dx")
    # a column's sum: each lane adds a 1/1024 .. 1/4096 share of the rows in turn, then at most 4 + 4 + 32 + 32 partial sums
    adds = 96 + x.shape[0] / 256
    if s is not None:
        _assert_within(next(grads), rds, adds * U * (dy.double() * n).abs().sum(0) + (dy.double().abs() * (dn + 4 * U * n.abs())).sum(0), "dscale")
    if o is not None:
        _assert_within(next(grads), rdo, adds * U * dy.double().abs().sum(0), "doffset")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,F", [(1, 1), (1, 256), (3, 7), (33, 40), (1024, 256), (5000, 256), (257, 128), (100, 129), (77, 512), (64, 602), (33, 800),
                                 (19, 1024), (9, 1025), (7, 4096), (5, 5001), (3, 16384), (2, 16383), (70000, 16)])
def test_layer_norm(dtype, n, F):
    g = _gen(n * 7 + F)
    x = (torch.randn(n, F, device=DEV, generator=g) * 1.5 + torch.randn(n, 1, device=DEV, generator=g)).to(dtype)
    w = dtype if (n + F) % 2 else F32
    _ln_check(x, _randn(g, F, dtype=w) * 0.2 + 1, _randn(g, F, dtype=w), 1e-5, _randn(g, n, F, dtype=dtype))


@pytest.mark.parametrize("which", ["none", "scale", "offset"])
def test_layer_norm_without_weights(which):
    g = _gen(5)
    x, dy = _randn(g, 65, 96, dtype=BF16), _randn(g, 65, 96, dtype=BF16)
    _ln_check(x, _randn(g, 96) if which == "scale" else None, _randn(g, 96) if which == "offset" else None, 1e-9, dy)


def test_layer_norm_strides_and_leading_dimensions():
    from shadow_gnn_amd import ops_mlp
    g = _gen(6)
    base = _randn(g, 50, 64, dtype=F16)
    s, o, dy = _randn(g, 64), _randn(g, 64), _randn(g, 50, 64, dtype=F16)
    want = ops_mlp.layer_norm(base, s, o)
    for v in (_pitched(base, 72), _pitched(base, 65), _pitched(base, 64, 3), _pitched(base, 71, 1), base.t().contiguous().t()):
        assert torch.equal(v, base)
        # (the element-wise path adds a row's values in another order than the word path)
        _assert_within(ops_mlp.layer_norm(v, s, o), want.double(), 2 * _half(F16) * want.double().abs() + 1e-5, "strided")
        _ln_check(v, s, o, 1e-5, _pitched(dy, 70))
    assert torch.equal(ops_mlp.layer_norm(base.view(5, 10, 64), s, o).view(50, 64), want)
    assert torch.equal(ops_mlp.layer_norm(base[7], s, o), want[7])
    x = base.clone().requires_grad_(True)
    ops_mlp.layer_norm(x, s, o).sum().backward()                   # an expanded gradient
    _assert_within(x.grad, _ln_ref(base, s, o, 1e-5, torch.ones_like(base))[1], 1e-4, "sum().backward()")


def test_layer_norm_empty_and_special_rows():
    from shadow_gnn_amd import ops_mlp
    s = torch.ones(32, device=DEV, requires_grad=True)
    o = torch.zeros(32, device=DEV, requires_grad=True)
    x = torch.empty(0, 32, dtype=BF16, device=DEV, requires_grad=True)
    y = ops_mlp.layer_norm(x, s, o)
    gx, gs, go = torch.autograd.grad(y, (x, s, o), torch.empty_like(y))
    assert y.shape == (0, 32) and gx.shape == (0, 32) and not gs.any() and not go.any()
    g = _gen(8)
    x = _randn(g, 6, 32)
    x[1] = 3.25                                                     # no spread: the offset alone
    x[2, 5] = float("inf")
    x[3, 0] = float("nan")
    x[4] *= 1e18                                                    # (squares reach 1e36: inside fp32)
    y = ops_mlp.layer_norm(x, s, o + 2.0)
    assert torch.equal(y[1], torch.full((32,), 2.0, device=DEV))
    assert y[2].isnan().all() and y[3].isnan().all()
    keep = [0, 4, 5]
    _assert_within(y[keep], _ln_ref(x[keep], s, o + 2.0, 1e-5, x[keep])[0], 1e-5, "neighbours of special rows")


def test_layer_norm_backward_is_reproducible_and_matches_differences():
    from shadow_gnn_amd import ops_mlp
    g = _gen(9)
    x, s, o, dy = _randn(g, 20000, 256, dtype=BF16), _randn(g, 256), _randn(g, 256), _randn(g, 20000, 256, dtype=BF16)
    leaves = [t.requires_grad_(True) for t in (x, s, o)]
    first = torch.autograd.grad(ops_mlp.layer_norm(*leaves), leaves, dy)
    for _ in range(3):
        again = torch.autograd.grad(ops_mlp.layer_norm(*leaves), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    # central differences of the definition in 64 bits along a direction (step 1e-4: its own error is 1e-8 of the third derivative)
    x, s, o, dy = _randn(g, 7, 96), _randn(g, 96), _randn(g, 96), _randn(g, 7, 96)
    leaves = [t.requires_grad_(True) for t in (x, s, o)]
    grads = torch.autograd.grad(ops_mlp.layer_norm(*leaves), leaves, dy)
    dirs = [_randn(g, *t.shape).double() for t in leaves]
    f = lambda h: (_ln_ref(*[(t.detach().double() + h * d) for t, d in zip(leaves, dirs)], 1e-5, dy)[0] * dy.double()).sum()  # noqa: E731
    want = (f(1e-4) - f(-1e-4)) / 2e-4
    got = sum((a.double() * d).sum() for a, d in zip(grads, dirs))
    size = sum((a.double() * d).abs().sum() for a, d in zip(grads, dirs))
    assert abs(got - want) <= 256 * U * size + 1e-6 * size


# ---------------------------------------------------------------- dropout

def _drop_check(x, p, seed, residual, dy):
    from shadow_gnn_amd import ops, ops_mlp
    leaves = [x.detach().requires_grad_(True)] + ([] if residual is None else [residual.detach().requires_grad_(True)])
    y = ops_mlp.dropout(leaves[0], p, seed, residual=None if residual is None else leaves[1])
    grads = torch.autograd.grad(y, leaves, dy)
    host = int(seed)
    keep = ops.dropout_keep_mask(x.shape[0], x.shape[1], p, host, DEV) if p > 0 else torch.ones(x.shape, dtype=torch.bool, device=DEV)
    scale = 1.0 / (1.0 - p)
    kept = torch.where(keep, x.double() * scale, torch.zeros((), dtype=torch.float64, device=DEV))
    # 1 / (1 - p) of the fp32 p: off by (p + 2) u / (1 - p) of itself at most; one product, one sum
    rel = (4 + 4 * scale) * U
    if residual is None:
        assert not y[~keep].any(), "a dropped element is zero"
        want = kept
        tol = rel * kept.abs()
    else:
        assert torch.equal(y[~keep], residual[~keep])
        want = kept + residual.double()
        tol = rel * kept.abs() + U * want.abs()
        assert torch.equal(grads[1], dy)
    _assert_within(y, want, tol, "y")
    kd = torch.where(keep, dy.double() * scale, torch.zeros((), dtype=torch.float64, device=DEV))
    _assert_within(grads[0], kd, rel * kd.abs(), "dx")
    return y


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,F", [(1, 1), (1, 2), (5, 7), (64, 40), (1000, 256), (333, 602), (129, 801), (3, 5000), (2000, 47), (1, 100001), (4097, 8)])
def test_dropout(dtype, n, F):
    g = _gen(n + F)
    x, r, dy = (_randn(g, n, F, dtype=dtype) for _ in range(3))
    _drop_check(x, 0.35, 0x1234567890ABCDEF >> 2, r, dy)
    _drop_check(x, 0.1, 17, None, dy)


@pytest.mark.parametrize("p", [0.0, 1e-6, 0.5, 0.999, 0.99999])
def test_dropout_probabilities(p):
    g = _gen(3)
    x, r, dy = (_randn(g, 300, 64, dtype=F32) for _ in range(3))
    y = _drop_check(x, p, 99, r, dy)
    if p == 0.0:
        assert torch.equal(y, x + r)


def test_dropout_strides_special_values_and_seeds():
    from shadow_gnn_amd import ops, ops_mlp
    g = _gen(4)
    x, r, dy = (_randn(g, 90, 64, dtype=BF16) for _ in range(3))
    want = ops_mlp.dropout(x, 0.4, 7, residual=r)
    for xv, rv in ((_pitched(x, 72), r), (x, _pitched(r, 65)), (_pitched(x, 64, 1), _pitched(r, 64, 3)), (x.t().contiguous().t(), r), (_pitched(x, 67, 5), _pitched(r, 80))):
        assert torch.equal(ops_mlp.dropout(xv, 0.4, 7, residual=rv), want)
    assert torch.equal(ops_mlp.dropout(x.view(9, 10, 64), 0.4, 7, residual=r.view(9, 10, 64)).view(90, 64), want)
    assert ops_mlp.dropout(x[:0], 0.4, 7).shape == (0, 64)
    # a dropped infinity or NaN is a zero
    keep = ops.dropout_keep_mask(90, 64, 0.4, 7, DEV)
    bad = torch.where(keep, x, torch.full_like(x, float("nan")))
    bad[0] = torch.where(keep[0], x[0], torch.full_like(x[0], float("inf")))
    assert torch.equal(ops_mlp.dropout(bad, 0.4, 7, residual=r), want)
    # a seed on the device, at its largest too; both forms give one mask
    for seed in (7, 0, (1 << 62) - 1, (1 << 63) - 1):
        t = torch.tensor([seed], dtype=torch.int64, device=DEV)
        _drop_check(x, 0.4, t, r, dy)
        assert torch.equal(ops_mlp.dropout(x, 0.4, t, residual=r), ops_mlp.dropout(x, 0.4, seed, residual=r))
    torch.manual_seed(5)
    a = ops_mlp.dropout(x, 0.4)
    b = ops_mlp.dropout(x, 0.4)
    torch.manual_seed(5)
    assert torch.equal(a, ops_mlp.dropout(x, 0.4)) and not torch.equal(a, b)
    # changing a seed tensor between the passes is an error, not another mask
    t = torch.tensor([3], dtype=torch.int64, device=DEV)
    xg = x.clone().requires_grad_(True)
    y = ops_mlp.dropout(xg, 0.4, t)
    t.add_(1)
    with pytest.raises(RuntimeError):
        y.backward(dy)


def test_dropout_same_mask_as_the_fused_epilogues():
    from shadow_gnn_amd import ops, ops_mlp
    g = _gen(12)
    x = _randn(g, 200, 64)
    idx = torch.arange(200, device=DEV, dtype=torch.int32)
    fused, seed = ops.LazyRows(x, idx).gather_dropped(0.3)
    assert torch.equal(ops_mlp.dropout(x, 0.3, seed) != 0, fused[:, :64] != 0)


# ---------------------------------------------------------------- the 16-bit Linear

def _act64(name, z):
    nn = torch.nn.functional
    return {"I": lambda t: t, "relu": nn.relu, "elu": nn.elu, "tanh": torch.tanh, "leakyrelu": lambda t: nn.leaky_relu(t, 0.2), "gelu": nn.gelu,
            "silu": nn.silu}[name](z)


def _lin_check(x, W, b, act, res, dy):
    from shadow_gnn_amd import ops_mlp
    dt = x.dtype
    src = [x, W, b, res]
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in src]
    y = ops_mlp.linear_act(leaves[0], leaves[1], leaves[2], act=act, residual=leaves[3])
    assert y.dtype == dt and y.shape == x.shape[:-1] + (W.shape[0],)
    grads = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    with torch.no_grad():                       # (without gradients the pre-activation is not kept: the same result)
        assert torch.equal(y, ops_mlp.linear_act(x, W, b, act=act, residual=res))
    x64, W64 = x.double(), W.double()
    K = W.shape[1]
    z = x64 @ W64.t() + (0 if b is None else b.double())
    mag = x64.abs() @ W64.abs().t() + (0 if b is None else b.double().abs())
    ez = (K + 4) * U * mag                      # K products added in fp32, in any order
    zr = z.clone().requires_grad_(True)
    h = _act64(act, zr)
    slope, = torch.autograd.grad(h.sum(), zr)
    h = h.detach()
    want = h + (0 if res is None else res.double())
    # slopes are at most 1.13; the activations' own forms are good to 2^-20 of max(1, |z|)
    approx = 0.0 if act in ("I", "relu", "leakyrelu") else 2.0 ** -20 * z.abs().clamp(min=1.0)
    _assert_within(y, want, 1.13 * ez + approx + 2 * U * (h.abs() + want.abs()), "y")
    # dz: z kept to half an fp16 step, slopes change by at most 1 per unit of z (relu and leakyrelu: they jump where z may have either sign)
    kept = ez + 2.0 ** -11 * z.abs() + 2.0 ** -25
    dy64 = dy.double()
    dz = dy64 * slope
    edz = torch.zeros_like(z)
    if act in ("relu", "leakyrelu"):
        edz = dy64.abs() * (z.abs() <= ez) + (_half(dt) * dz.abs() if act == "leakyrelu" else 0)
    elif act != "I":
        edz = dy64.abs() * (kept + 2.0 ** -19) + _half(dt) * (dz.abs() + dy64.abs() * kept)
    if act != "I":
        edz = edz + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps + 2 * U * dz.abs()
    adz = dz.abs() + edz
    N, M = W.shape[0], x.shape[0]
    _assert_within(next(grads), dz @ W64, edz @ W64.abs() + (N + 4) * U * (adz @ W64.abs()), "dx")
    _assert_within(next(grads), dz.t() @ x64, edz.t() @ x64.abs() + (M + 4) * U * (adz.t() @ x64.abs()), "dW")
    if b is not None:
        _assert_within(next(grads), dz.sum(0), edz.sum(0) + (M + 4) * U * adz.sum(0), "db")
    if res is not None:
        assert torch.equal(next(grads), dy)


_SIZES = [(1, 1, 1), (1, 64, 8), (3, 5, 7), (17, 31, 33), (128, 128, 64), (129, 257, 65), (256, 256, 256), (1000, 47, 500), (300, 172, 602), (2049, 96, 100),
          (63, 1000, 513), (4096, 8, 24), (130, 384, 1000), (5, 2000, 72), (9000, 5, 600), (9000, 600, 5), (8300, 9, 15)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,N,K", _SIZES)
def test_linear_act(dtype, M, N, K):
    g = _gen(M + N + K)
    x, W, res, dy = _randn(g, M, K, dtype=dtype), _randn(g, N, K, dtype=dtype, scale=K ** -0.5), _randn(g, M, N, dtype=dtype), _randn(g, M, N, dtype=dtype)
    b = _randn(g, N, dtype=F32 if N % 2 else dtype)
    _lin_check(x, W, b, "gelu", res, dy)
    _lin_check(x, W, None, "I", None, dy)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["I", "relu", "leakyrelu", "gelu"])
@pytest.mark.parametrize("M,N,K", [(16384, 256, 256), (20001, 256, 128), (16400, 128, 256), (33333, 64, 96), (16447, 40, 128), (17000, 200, 256), (16385, 248, 136), (16384, 8, 8)])
def test_linear_act_tall_and_narrow(dtype, act, M, N, K):
    """The form with the weight in registers, its gradients with dy masked (or dz formed) in the tile."""
    g = _gen(M + N + K)
    x, W = _randn(g, M, K, dtype=dtype), _randn(g, N, K, dtype=dtype, scale=K ** -0.5)
    _lin_check(x, W, _randn(g, N), act, _randn(g, M, N, dtype=dtype), _randn(g, M, N, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["I", "relu", "leakyrelu", "silu"])
@pytest.mark.parametrize("M,N,K", [(98304, 256, 256), (98311, 136, 128), (98335, 96, 200), (100003, 250, 144), (98321, 47, 160)])
def test_linear_act_all_of_the_weight_gradient_at_once(dtype, act, M, N, K):
    """Rows enough for one workgroup to hold all of dW; operands pitched, and dy in rows of whole words and not."""
    g = _gen(M + N + K)
    x, W, dy = _randn(g, M, K, dtype=dtype), _randn(g, N, K, dtype=dtype, scale=K ** -0.5), _randn(g, M, N, dtype=dtype)
    _lin_check(_pitched(x, K + 8), W, _randn(g, N), act, None, _pitched(dy, N // 8 * 8 + 16))
    _lin_check(x, W, None, act, None, dy)


@pytest.mark.parametrize("act", ["I", "relu", "tanh"])
def test_linear_act_tall_and_narrow_in_parts(act):
    """Single gradients, pitched operands and rows that are no whole words: the forms mix."""
    from shadow_gnn_amd import ops_mlp
    g = _gen(71)
    M, N, K = 16500, 96, 104
    x, W, b, dy = _randn(g, M, K, dtype=BF16), _randn(g, N, K, dtype=BF16, scale=0.1), _randn(g, N), _randn(g, M, N, dtype=BF16)
    full = [t.clone().requires_grad_(True) for t in (x, W, b)]
    full = torch.autograd.grad(ops_mlp.linear_act(*full, act=act), full, dy)
    for i in range(3):
        ins = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, W, b))]
        got, = torch.autograd.grad(ops_mlp.linear_act(*ins, act=act), (ins[i],), dy)
        assert torch.equal(got, full[i]), i
    for xv, dv in ((_pitched(x, 112), _pitched(dy, 104)), (_pitched(x, 105), dy), (x, _pitched(dy, 97)), (_pitched(x, 104, 1), _pitched(dy, 96, 3))):
        _lin_check(xv, W, b, act, None, dv)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["I", "relu", "elu", "tanh", "leakyrelu", "gelu", "silu"])
def test_linear_act_activations(dtype, act):
    g = _gen(31)
    x, W = _randn(g, 333, 80, dtype=dtype, scale=2.0), _randn(g, 72, 80, dtype=dtype, scale=0.2)
    _lin_check(x, W, _randn(g, 72, dtype=dtype), act, _randn(g, 333, 72, dtype=dtype), _randn(g, 333, 72, dtype=dtype))
    # pre-activations far out and next to zero
    x = x * torch.logspace(-7, 1.5, 333, device=DEV)[:, None].to(dtype)
    _lin_check(x, W, None, act, None, _randn(g, 333, 72, dtype=dtype))


def test_linear_act_strides_and_shapes():
    from shadow_gnn_amd import ops_mlp
    g = _gen(32)
    x, W, b, res, dy = _randn(g, 150, 96, dtype=BF16), _randn(g, 40, 96, dtype=BF16, scale=0.1), _randn(g, 40), _randn(g, 150, 40, dtype=BF16), _randn(g, 150, 40, dtype=BF16)
    want = ops_mlp.linear_act(x, W, b, act="relu", residual=res)
    for xv, wv, rv in ((_pitched(x, 104), W, res), (_pitched(x, 97), W, _pitched(res, 41)), (x, _pitched(W, 99, 1), res), (_pitched(x, 96, 1), _pitched(W, 96, 3), _pitched(res, 40, 1)),
                       (x.t().contiguous().t(), W.t().contiguous().t(), res.t().contiguous().t())):
        assert torch.equal(ops_mlp.linear_act(xv, wv, b, act="relu", residual=rv), want)       # (one order of products on both loaders)
        _lin_check(xv, wv, b, "relu", rv, _pitched(dy, 43))
    assert torch.equal(ops_mlp.linear_act(x.view(3, 50, 96), W, b, act="relu", residual=res.view(3, 50, 40)).view(150, 40), want)
    assert torch.equal(ops_mlp.linear_act(x[9], W, b, act="relu", residual=res[9]), want[9])
    W1 = W.clone().requires_grad_(True)
    ops_mlp.linear_act(x, W1).sum().backward()                    # an expanded gradient
    _assert_within(W1.grad, torch.ones(150, 40, device=DEV).double().t() @ x.double(), 200 * U * x.double().abs().sum(0).expand(40, 96), "expanded dy")


@pytest.mark.parametrize("act", ["I", "gelu"])
def test_linear_act_empty_and_partial_gradients(act):
    from shadow_gnn_amd import ops_mlp
    g = _gen(33)
    W, b = _randn(g, 40, 96, dtype=BF16).requires_grad_(True), _randn(g, 40).requires_grad_(True)
    x = torch.empty(0, 96, dtype=BF16, device=DEV, requires_grad=True)
    y = ops_mlp.linear_act(x, W, b, act=act)
    gx, gw, gb = torch.autograd.grad(y, (x, W, b), torch.empty_like(y))
    assert gx.shape == (0, 96) and not gw.any() and not gb.any()
    x, dy = _randn(g, 200, 96, dtype=BF16).requires_grad_(True), _randn(g, 200, 40, dtype=BF16)
    res = _randn(g, 200, 40, dtype=BF16).requires_grad_(True)
    full = torch.autograd.grad(ops_mlp.linear_act(x, W, b, act=act, residual=res), (x, W, b, res), dy)
    for i in range(4):                                            # each input alone
        ins = [t if j == i else t.detach() for j, t in enumerate((x, W, b, res))]
        got, = torch.autograd.grad(ops_mlp.linear_act(ins[0], ins[1], ins[2], act=act, residual=ins[3]), (ins[i],), dy)
        assert torch.equal(got, full[i])


def test_linear_act_special_values_stay_in_their_rows():
    from shadow_gnn_amd import ops_mlp
    g = _gen(34)
    x, W = _randn(g, 140, 100, dtype=F16), _randn(g, 70, 100, dtype=F16, scale=0.1)
    for act in ("I", "relu", "gelu", "silu", "tanh", "elu"):
        want = ops_mlp.linear_act(x, W, act=act)
        bad = x.clone()
        bad[3, 99] = float("nan")
        bad[139, 0] = float("inf")
        got = ops_mlp.linear_act(bad, W, act=act)
        rows = [i for i in range(140) if i not in (3, 139)]
        assert torch.equal(got[rows], want[rows])
        assert got[3].isnan().all() or act == "relu"
    # the slopes at pre-activations past fp16's range: z = +-1e6 saturates what is kept for the backward pass
    xb = torch.ones(2, 8, dtype=BF16, device=DEV, requires_grad=True)
    Wb = (torch.tensor([[1.0], [-1.0]], device=DEV) * torch.full((2, 8), 125000.0, device=DEV)).to(BF16)
    for act, hi, lo in (("relu", 1, 0), ("elu", 1, 0), ("tanh", 0, 0), ("leakyrelu", 1, 0.2), ("gelu", 1, 0), ("silu", 1, 0)):
        gx, = torch.autograd.grad(ops_mlp.linear_act(xb, Wb, act=act), xb, torch.ones(2, 2, dtype=BF16, device=DEV))
        want = hi * Wb[0].double() + torch.tensor(lo, dtype=BF16).double().item() * Wb[1].double()
        _assert_within(gx, want.expand(2, 8), 0.0, act)


@pytest.mark.parametrize("M,N,K", [(40, 24, 40), (9000, 24, 40), (9000, 600, 40)])
def test_linear_act_nan_pre_activations(M, N, K):
    """A NaN stays NaN through every activation but relu, whose rule makes it 0 and passes no gradient."""
    from shadow_gnn_amd import ops_mlp
    g = _gen(36)
    x, W = _randn(g, M, K, dtype=BF16), _randn(g, N, K, dtype=BF16, scale=0.1)
    x[M // 2, 3] = float("nan")
    for act in ("I", "relu", "elu", "tanh", "leakyrelu", "gelu", "silu"):
        leaf = x.clone().requires_grad_(True)
        y = ops_mlp.linear_act(leaf, W, act=act)
        assert y.isnan().any(1).nonzero().tolist() == ([] if act == "relu" else [[M // 2]]), act
        assert y[M // 2].isnan().all() if act != "relu" else not y[M // 2].any(), act
        dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
        if act == "relu":
            assert not dx[M // 2].any() and not dx.isnan().any()


def test_linear_act_reproducible_and_differences():
    from shadow_gnn_amd import ops_mlp
    g = _gen(35)
    leaves = [_randn(g, 30000, 100, dtype=BF16).requires_grad_(True), _randn(g, 72, 100, dtype=BF16, scale=0.1).requires_grad_(True), _randn(g, 72).requires_grad_(True)]
    dy = _randn(g, 30000, 72, dtype=BF16)
    first = torch.autograd.grad(ops_mlp.linear_act(*leaves, act="silu"), leaves, dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(ops_mlp.linear_act(*leaves, act="silu"), leaves, dy)))
    for act in ("tanh", "gelu", "silu", "elu"):
        leaves = [_randn(g, 40, 24, dtype=F16).requires_grad_(True), _randn(g, 16, 24, dtype=F16, scale=0.3).requires_grad_(True), _randn(g, 16).requires_grad_(True)]
        dy = _randn(g, 40, 16, dtype=F16)
        grads = torch.autograd.grad(ops_mlp.linear_act(*leaves, act=act), leaves, dy)
        dirs = [_randn(g, *t.shape).double() for t in leaves]

        def f(h):
            a, w, c = [t.detach().double() + h * d for t, d in zip(leaves, dirs)]
            return (_act64(act, a @ w.t() + c) * dy.double()).sum()

        want = (f(1e-4) - f(-1e-4)) / 2e-4
        size = sum((a.double() * d).abs().sum() for a, d in zip(grads, dirs))
        got = sum((a.double() * d).sum() for a, d in zip(grads, dirs))
        assert abs(got - want) <= 4 * _half(F16) * size


# ---------------------------------------------------------------- log probabilities of labels

def _lp_check(x, label, k, seed=0, grads=True):
    from shadow_gnn_amd import ops_mlp
    n, C = x.shape
    leaf = x.detach().requires_grad_(grads)
    out = ops_mlp.label_logprobs(leaf, label, topk=k)
    x64 = x.double()
    m = x64.amax(1, keepdim=True)
    lse = m + (x64 - m).exp().sum(1, keepdim=True).log()
    lp = x64 - lse
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    H = -plp.sum(1)
    has = (label >= 0)
    at = label.clamp(min=0).long()[:, None]
    fin = torch.where(x64.isinf(), torch.zeros_like(x64), x64).abs().amax(1)
    # the sum's relative error: its longest chain of additions (a lane's share, then the joins) and 2 u |x log2 e| of every exponent's
    # argument (the row's maximum bounds it); the logarithm and the label's difference add a few roundings of the log-sum's size
    S = U * (64 + C / 64 + 8 * fin)
    e_lp = (S + 4 * U * (fin + lse[:, 0].abs()))
    _assert_within(out.logprob, torch.where(has, lp.gather(1, at)[:, 0], torch.zeros_like(H)), e_lp + 4 * U * lp.gather(1, at)[:, 0].abs().nan_to_num(posinf=0), "logprob")
    d = torch.where(p > 0, lp, torch.zeros_like(lp))
    e_H = (S + 8 * U) * (2 + (p * d.abs()).sum(1)) + 8 * U * (p * d * d).sum(1)
    _assert_within(out.entropy, H, e_H, "entropy")
    order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(out.top_index, order)
    top64 = lp.gather(1, order)
    _assert_within(out.top_logprob, top64, e_lp[:, None] + 4 * U * top64.abs().nan_to_num(posinf=0), "top")
    if not grads:
        return
    g = _gen(seed)
    a, h, t = _randn(g, n), _randn(g, n, scale=0.3), _randn(g, n, k)
    outs, gs = [out.logprob, out.entropy] + ([out.top_logprob] if k else []), [a, h] + ([t] if k else [])
    dx, = torch.autograd.grad(outs, leaf, gs, retain_graph=True)
    a64 = torch.where(has, a.double(), torch.zeros_like(H))
    total = a64 + t.double().sum(1)
    lpH = torch.where(p > 0, lp + H[:, None], torch.zeros_like(p))
    want = -p * total[:, None] - h.double()[:, None] * p * lpH
    want.scatter_add_(1, at, a64[:, None])
    if k:
        want.scatter_add_(1, order, t.double())
    size = p * (a64.abs() + t.double().abs().sum(1))[:, None] + p * h.double().abs()[:, None] * (lpH.abs() + 1)
    tol = size * (e_lp + 16 * U)[:, None] * 2 + p * (h.double().abs() * e_H)[:, None] + (16 + 2 * k) * U * size
    extra = torch.zeros_like(want).scatter_add_(1, at, a64.abs()[:, None])
    if k:
        extra.scatter_add_(1, order, t.double().abs())
    _assert_within(dx, want, tol + 4 * U * extra, "dlogits")
    # each gradient alone: the others are absent, not zeros
    only, = torch.autograd.grad(out.entropy, leaf, h, retain_graph=True)
    _assert_within(only, -h.double()[:, None] * p * lpH, tol, "entropy's gradient")
    if k:
        only, = torch.autograd.grad(out.top_logprob, leaf, t)
        w = -p * t.double().sum(1)[:, None]
        w.scatter_add_(1, order, t.double())
        _assert_within(only, w, tol + 4 * U * extra, "the alternatives' gradient")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,C,k", [(1, 1, 1), (1, 2, 2), (5, 3, 0), (300, 40, 5), (1024, 47, 5), (333, 64, 64), (100, 65, 3), (257, 172, 10), (64, 256, 0), (50, 257, 20), (33, 1000, 7),
                                   (19, 1024, 64), (9, 1025, 5), (700, 2000, 3), (5, 5001, 64), (3, 40000, 10), (1, 131072, 10), (2, 200001, 20)])
def test_label_logprobs(dtype, n, C, k):
    g = _gen(n + C + k)
    x = _randn(g, n, C, dtype=dtype, scale=3.0)
    label = torch.randint(0, C, (n,), device=DEV, generator=g)
    label[n // 2] = -1
    _lp_check(x, label.int() if C % 2 else label, k, seed=C)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("C", [47, 172, 1000, 3000, 66000])
def test_label_logprobs_masks_ties_and_special_rows(dtype, C):
    from shadow_gnn_amd import ops_mlp
    g = _gen(C)
    k = 20
    x = _randn(g, 12, C, dtype=dtype, scale=2.0)
    label = torch.randint(0, C, (12,), device=DEV, generator=g)
    x[1] = 0                                               # every value equal: the lowest indices
    x[2] = torch.finfo(dtype).min                          # the type's lowest value everywhere: a uniform row, not an empty one
    x[3, C // 3:] = float("-inf")                          # a masked end
    x[4, ::2] = float("-inf")
    x[5] = torch.finfo(dtype).min
    x[5, C - 1] = 3.0                                      # a mask by the lowest value
    x[6, :] = (x[6] * 2).round() / 2                       # many ties
    x[7] = torch.where(torch.arange(C, device=DEV) % 2 == 0, torch.zeros((), device=DEV, dtype=dtype), -torch.zeros((), device=DEV, dtype=dtype))   # +0 and -0 tie
    x[8] = torch.linspace(-30, 30, C, device=DEV).to(dtype)                # ascending: the best arrive last
    x[9] = torch.linspace(30, -30, C, device=DEV).to(dtype)
    x[10] = float("-inf")
    x[10, C // 2] = -5.0                                   # one value left
    label[3], label[4], label[10] = 0, 1, C // 2
    ok = [i for i in range(12) if i not in (4, 5, 2)]
    _lp_check(x[ok], label[ok], k)
    _lp_check(x[[4, 5, 2]], label[[4, 5, 2]], k, grads=False)
    # no finite logit; an infinity; a NaN
    y = _randn(g, 4, C, dtype=dtype).requires_grad_(True)
    z = y.detach().clone()
    z[0] = float("-inf")
    z[1, C // 2] = float("inf")
    z[2, C - 1] = float("nan")
    z.requires_grad_(True)
    out = ops_mlp.label_logprobs(z, label[:4], topk=3)
    assert out.logprob[0] == float("-inf") and out.entropy[0] == 0 and (out.top_logprob[0] == float("-inf")).all()
    assert out.top_index[0].tolist() == [0, 1, 2]
    assert out.logprob[1:3].isnan().all() and out.entropy[1:3].isnan().all() and out.top_logprob[1:3].isnan().all()
    assert out.top_index[1, 0] == C // 2 and out.top_index[2, 0] == C - 1
    dz, = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], z, [torch.ones(4, device=DEV), torch.ones(4, device=DEV), torch.ones(4, 3, device=DEV)])
    assert not dz[0].any() and dz[1].isnan().all() and dz[2].isnan().all() and dz[3].isfinite().all()
    want = ops_mlp.label_logprobs(y, label[:4], topk=3)
    assert torch.equal(out.logprob[3], want.logprob[3]) and torch.equal(out.top_index[3], want.top_index[3])
    # labels: none, the last class, past the end
    lab = torch.tensor([-1, C - 1, C, -100], device=DEV)
    out = ops_mlp.label_logprobs(y, lab)
    dy, = torch.autograd.grad(out.logprob, y, torch.ones(4, device=DEV))
    assert out.logprob[0] == 0 and out.logprob[3] == 0 and out.logprob[1].isfinite() and out.logprob[2].isnan()
    assert not dy[0].any() and not dy[3].any() and dy[1].isfinite().all() and dy[2].isnan().all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("C", [47, 172, 3000])
def test_label_logprobs_rows_without_a_finite_logit_have_gradient_zero(dtype, C):
    """... whatever comes back for their scores: a square of -inf has an infinite gradient, its mean over nothing a NaN."""
    from shadow_gnn_amd import ops_mlp
    g = _gen(46)
    x = _randn(g, 5, C, dtype=dtype)
    x[1:4] = float("-inf")
    x.requires_grad_(True)
    out = ops_mlp.label_logprobs(x, torch.tensor([1, 2, -1, C - 1, 0], device=DEV), topk=2)
    dx, = torch.autograd.grad(out.logprob.square().sum() + out.top_logprob.square().sum(), x, retain_graph=True)
    assert not dx[1:4].any() and dx[[0, 4]].isfinite().all() and dx[[0, 4]].any(1).all()
    for bad in (float("nan"), float("inf"), -float("inf")):
        a, h, t = torch.full((5,), bad, device=DEV), torch.full((5,), bad, device=DEV), torch.full((5, 2), bad, device=DEV)
        dx, = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, [a, h, t], retain_graph=True)
        assert not dx[1:4].any() and dx[[0, 4]].isnan().any(1).all()


def test_label_logprobs_strides_and_shapes():
    from shadow_gnn_amd import ops_mlp
    g = _gen(44)
    for C in (47, 172, 5000):
        x = _randn(g, 60, C, dtype=F16, scale=2.0)
        label = torch.randint(0, C, (60,), device=DEV, generator=g)
        for v in (_pitched(x, C + 8), _pitched(x, C + 1), _pitched(x, C, 1), _pitched(x, C + 5, 3), x.t().contiguous().t()):
            _lp_check(v, label, 5)
        want = ops_mlp.label_logprobs(x, label, topk=5)
        got = ops_mlp.label_logprobs(x.view(3, 20, C), label.view(3, 20), topk=5)
        assert got.logprob.shape == (3, 20) and got.top_index.shape == (3, 20, 5)
        assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
        wide = torch.stack([label, label], 1)[:, 0]                # a strided label
        assert torch.equal(ops_mlp.label_logprobs(x, wide).logprob, want.logprob)
        one = ops_mlp.label_logprobs(x[4], label[4], topk=5)
        assert one.logprob.shape == () and torch.equal(one.top_index, want.top_index[4])
    empty = ops_mlp.label_logprobs(torch.empty(0, 9, device=DEV, requires_grad=True), torch.empty(0, dtype=torch.int64, device=DEV), topk=2)
    assert empty.logprob.shape == (0,) and empty.top_index.shape == (0, 2)
    e = torch.empty(0, 9, device=DEV, requires_grad=True)
    gx, = torch.autograd.grad(ops_mlp.label_logprobs(e, torch.empty(0, dtype=torch.int64, device=DEV)).logprob.sum(), e)
    assert gx.shape == (0, 9)


def test_label_logprobs_gradient_matches_differences():
    from shadow_gnn_amd import ops_mlp
    g = _gen(45)
    for C in (30, 1500):
        x = _randn(g, 6, C, scale=2.0).requires_grad_(True)
        label = torch.randint(0, C, (6,), device=DEV, generator=g)
        a, h, t, d = _randn(g, 6), _randn(g, 6), _randn(g, 6, 4), _randn(g, 6, C).double()
        out = ops_mlp.label_logprobs(x, label, topk=4)
        dx, = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, [a, h, t])

        def f(s):
            lp = torch.log_softmax(x.detach().double() + s * d, 1)
            return (lp.gather(1, label[:, None])[:, 0] * a).sum() - ((lp.exp() * lp).sum(1) * h).sum() + (lp.gather(1, out.top_index) * t).sum()

        want = (f(1e-4) - f(-1e-4)) / 2e-4
        assert abs((dx.double() * d).sum() - want) <= 1e-5 * (dx.double() * d).abs().sum()


# ---------------------------------------------------------------- bounds, devices, streams, graphs

def test_rows_behind_the_last_stay_as_they_were():
    """Outputs written through the C entries into pitched buffers: nothing but the rows' own elements changes."""
    from shadow_gnn_amd import _lib
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    g = _gen(51)
    for F in (40, 47, 256, 300):
        n, pitch = 37, F + 9
        x, W, r = _randn(g, n, F, dtype=BF16), _randn(g, F, F, dtype=BF16), _randn(g, n, F, dtype=BF16)
        stat = torch.full((4, n + 5), 5.0, device=DEV)
        lab = torch.zeros(n, dtype=torch.int64, device=DEV)
        ws = torch.empty(1 << 24, dtype=torch.uint8, device=DEV)
        kept = torch.zeros(n * 1024, dtype=torch.uint8, device=DEV)
        for off in (0, 1):
            calls = {
                "ln": lambda y: lib.sl_layer_norm_fwd(1, 0, x.data_ptr(), F, None, None, n, F, 1e-5, y, pitch, None, st),
                "ln_bwd": lambda y: lib.sl_layer_norm_bwd(1, 0, x.data_ptr(), F, r.data_ptr(), F, None, stat.data_ptr(), n, F, y, pitch, None, None, None, st),
                "drop": lambda y: lib.sl_dropout(1, x.data_ptr(), F, r.data_ptr(), F, n, F, 0.5, 3, None, y, pitch, st),
                "lin": lambda y: lib.sl_linear16_fwd(1, x.data_ptr(), F, W.data_ptr(), F, None, 0, r.data_ptr(), F, n, F, F, 1, y, pitch, kept.data_ptr(), st),
                "lin_dx": lambda y: lib.sl_linear16_bwd(1, x.data_ptr(), F, W.data_ptr(), F, r.data_ptr(), F, kept.data_ptr(), n, F, F, 1, y, pitch, None, 0, None, 0, ws.data_ptr(), st),
                "lin_dw": lambda y: lib.sl_linear16_bwd(1, x[:, :37].contiguous().data_ptr() if F > 37 else 0, 37, W.data_ptr(), F, r.data_ptr(), F, None, n, 37, 37, 0, None, 0, y, pitch, None, 0, ws.data_ptr(), st),
                "lp_bwd": lambda y: lib.sl_label_logprobs_bwd(1, x.data_ptr(), F, lab.data_ptr(), 1, n, F, 0, stat[0].data_ptr(), stat[1].data_ptr(), None, stat[2].data_ptr(), None, None, y, pitch, st),
            }
            for name, call in calls.items():
                buf = torch.full(((n + 3) * pitch + 8,), 77.0, dtype=BF16, device=DEV)
                width = 37 if name == "lin_dw" else F
                assert call(buf.data_ptr() + 2 * off) == 0, name
                torch.cuda.synchronize()
                rows = buf[off:off + (n + 3) * pitch].view(n + 3, pitch)
                assert (rows[:n, width:] == 77).all() and (rows[n:] == 77).all() and (buf[:off] == 77).all() and (buf[off + (n + 3) * pitch:] == 77).all(), (name, F, off)
                assert not (rows[:n, :width] == 77).all(), name


@pytest.mark.parametrize("M,N,K,act", [
    (98309, 256, 256, 1), (98309, 136, 72, 5), (98309, 72, 136, 0), (98309, 47, 256, 0),       # dz^T x of all of dW at once
    (16411, 256, 256, 1), (16411, 128, 72, 5), (16387, 72, 136, 4), (16393, 40, 16, 0),      # tall, narrow: whole words
    (1111, 1100, 264, 2), (1111, 1100, 263, 1),                                             # 128 x 128 tiles, words and any rows
    (4100, 4200, 520, 6),                                                                   # 256 x 256 tiles
    (530, 300, 100, 1), (512, 300, 101, 5),                                                 # rows on both sides of the few-row gradient
])
def test_linear16_writes_its_own_elements_only(M, N, K, act):
    """Outputs in pitched buffers, what is kept and the scratch in buffers of the stated sizes: all that lies behind stays as it was."""
    from shadow_gnn_amd import _lib
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    g = _gen(57)
    x, W, r = _randn(g, M, K, dtype=BF16), _randn(g, N, K, dtype=BF16, scale=K ** -0.5), _randn(g, M, N, dtype=BF16)
    kb, sb = lib.sl_linear16_kept_bytes(act, M, N), lib.sl_linear16_bwd_scratch_bytes(act, M, N, K)
    kept = torch.full((kb + 4096,), 0x5A, dtype=torch.uint8, device=DEV)
    ws = torch.full((sb + 4096,), 0x5A, dtype=torch.uint8, device=DEV)

    def rows(n, width):
        return torch.full((n + 3, width + 16), 77.0, dtype=BF16, device=DEV)

    y, dx, dw, db = rows(M, N), rows(M, K), rows(N, K), torch.full((N + 64,), 77.0, device=DEV)
    assert lib.sl_linear16_fwd(1, x.data_ptr(), K, W.data_ptr(), K, None, 0, r.data_ptr(), N, M, N, K, act, y.data_ptr(), N + 16, kept.data_ptr() if act else None, st) == 0
    assert lib.sl_linear16_bwd(1, x.data_ptr(), K, W.data_ptr(), K, r.data_ptr(), N, kept.data_ptr() if act else None, M, N, K, act, dx.data_ptr(), K + 16,
                               dw.data_ptr(), K + 16, db.data_ptr(), 1, ws.data_ptr(), st) == 0
    torch.cuda.synchronize()
    assert (kept[kb:] == 0x5A).all() and (ws[sb:] == 0x5A).all() and (db[N:] == 77).all()
    for t, n, width in ((y, M, N), (dx, M, K), (dw, N, K)):
        assert (t[:, width:] == 77).all() and (t[n:] == 77).all() and (t[:n, :width] != 77).any(1).all()


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("wants", ["both", "dx", "dW"])
@pytest.mark.parametrize("M,N,K,act", [(98309, 256, 256, 1), (98309, 136, 72, 5), (98309, 72, 136, 0), (98309, 47, 256, 0), (16411, 128, 72, 4), (16393, 40, 16, 0), (1111, 1100, 264, 2),
                                       (1111, 1100, 264, 0), (530, 300, 100, 1), (512, 304, 104, 5), (9000, 40, 1024, 0), (9000, 72, 1024, 0)])
def test_linear16_backward_stays_in_the_scratch_of_its_call(M, N, K, act, wants, shift):
    """sl_linear16_bwd with exactly the scratch stated for its operands: what lies behind stays as it was, the gradients are those of a
    call with the shape's largest scratch."""
    from shadow_gnn_amd import _lib
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    g = _gen(65)
    x, W, dy = _randn(g, M, K, dtype=BF16), _randn(g, N, K, dtype=BF16, scale=K ** -0.5), _randn(g, M * N + 8, dtype=BF16)[shift:][:M * N].view(M, N)
    y, kept = torch.empty_like(dy), torch.empty(lib.sl_linear16_kept_bytes(act, M, N) + 16, dtype=torch.uint8, device=DEV)
    assert lib.sl_linear16_fwd(1, x.data_ptr(), K, W.data_ptr(), K, None, 0, None, 0, M, N, K, act, y.data_ptr(), N, kept.data_ptr() if act else None, st) == 0
    most = lib.sl_linear16_bwd_scratch_bytes(act, M, N, K)
    exact = lib.sl_linear16_bwd_scratch_bytes_for(act, x.data_ptr(), K, K, dy.data_ptr(), N, M, N, K, wants != "dW", wants != "dx")
    assert exact <= most
    got = []
    for size in (exact, most):
        ws = torch.full((size + 4096,), 0x5A, dtype=torch.uint8, device=DEV)
        dx, dw, db = torch.zeros(M, K, dtype=BF16, device=DEV), torch.zeros(N, K, dtype=BF16, device=DEV), torch.zeros(N, device=DEV)
        assert lib.sl_linear16_bwd(1, x.data_ptr(), K, W.data_ptr(), K, dy.data_ptr(), N, kept.data_ptr() if act else None, M, N, K, act,
                                   dx.data_ptr() if wants != "dW" else None, K, dw.data_ptr() if wants != "dx" else None, K,
                                   db.data_ptr() if wants != "dx" else None, 1, ws.data_ptr(), st) == 0
        torch.cuda.synchronize()
        assert (ws[size:] == 0x5A).all()
        got.append((dx, dw, db))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert got[0][0].any() == (wants != "dW") and got[0][1].any() == (wants != "dx")


def test_gradients_are_differentiable_once():
    """create_graph gives the same gradients; a second backward pass through them is an error, not zeros."""
    from shadow_gnn_amd import ops_mlp
    g = _gen(58)
    x, W, s = _randn(g, 64, 64, dtype=BF16).requires_grad_(True), _randn(g, 64, 64, dtype=BF16, scale=0.1).requires_grad_(True), _randn(g, 64).requires_grad_(True)
    label = torch.randint(0, 64, (64,), device=DEV, generator=g)
    dy = _randn(g, 64, 64, dtype=BF16).requires_grad_(True)
    for f in (lambda: ops_mlp.layer_norm(x, s, s), lambda: ops_mlp.dropout(x, 0.5, 3), lambda: ops_mlp.linear_act(x, W, act="gelu")):
        plain = torch.autograd.grad(f(), x, dy.detach())[0]
        twice = torch.autograd.grad(f(), x, dy, create_graph=True)[0]
        assert torch.equal(plain, twice.detach())
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(twice.float().sum(), dy)
    first = torch.autograd.grad(ops_mlp.label_logprobs(x, label).entropy.sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiable once"):
        first.float().sum().backward()


@pytest.mark.parametrize("act", ["relu", "elu", "tanh", "leakyrelu", "gelu", "silu"])
@pytest.mark.parametrize("which", ["weight", "bias"])
def test_gradients_of_a_first_layer_are_differentiable_once(act, which):
    """Raw features and a constant dy: dW and db still depend on the weight and the bias, through act'(z)."""
    from shadow_gnn_amd import ops_mlp
    g = _gen(61)
    x, W, b = _randn(g, 64, 48, dtype=BF16), _randn(g, 40, 48, dtype=BF16, scale=0.1), _randn(g, 40)
    leaf = (W if which == "weight" else b).requires_grad_(True)
    y = ops_mlp.linear_act(x, W, b, act=act)
    plain, = torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
    first, = torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)
    assert torch.equal(first.detach(), plain)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (y.float().sum() + first.float().square().sum()).backward()
    # an identity's gradients of constants are constants: the penalty adds nothing, here as in torch
    y = ops_mlp.linear_act(x, W, b)
    first, = torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)
    got, = torch.autograd.grad(y.float().sum() + first.float().square().sum(), leaf)
    assert torch.equal(got, first)


def test_a_bias_may_change_before_the_backward_pass():
    from shadow_gnn_amd import ops_mlp
    g = _gen(62)
    x, W, b, dy = _randn(g, 64, 48, dtype=BF16), _randn(g, 40, 48, dtype=BF16, scale=0.1), _randn(g, 40).requires_grad_(True), _randn(g, 64, 40, dtype=BF16)
    want, = torch.autograd.grad(ops_mlp.linear_act(x, W, b, act="gelu"), b, dy)
    y = ops_mlp.linear_act(x, W, b, act="gelu")
    with torch.no_grad():
        b.add_(1)
    assert torch.equal(torch.autograd.grad(y, b, dy)[0], want)


def test_forward_mode_tangents_are_refused():
    """A tangent of an input or of the gradient that a backward pass starts from: an error, not zeros."""
    from shadow_gnn_amd import ops_mlp
    g = _gen(63)
    x, W, s, label = _randn(g, 64, 64, dtype=BF16), _randn(g, 64, 64, dtype=BF16, scale=0.1), _randn(g, 64), torch.zeros(64, dtype=torch.int64, device=DEV)
    for f in (lambda t: ops_mlp.layer_norm(t, s, s), lambda t: ops_mlp.dropout(t, 0.5, 3), lambda t: ops_mlp.linear_act(t, W, s, act="gelu"),
              lambda t: ops_mlp.label_logprobs(t, label, topk=2).entropy):
        for leaf in (x, x.clone().requires_grad_(True)):
            with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                f(forward_ad.make_dual(leaf, torch.ones_like(x)))
        y = f(leaf)
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)
        assert torch.autograd.grad(y, leaf, torch.ones_like(y))[0].shape == x.shape


def test_one_tensor_in_several_places():
    """Scale and offset, x and residual, x and weight may be one tensor: its gradient is the sum of both places'."""
    from shadow_gnn_amd import ops_mlp
    g = _gen(59)
    x, s, dy = _randn(g, 128, 128, dtype=BF16), _randn(g, 128), _randn(g, 128, 128, dtype=BF16)

    def both(f, t):
        one = t.clone().requires_grad_(True)
        a, b = t.clone().requires_grad_(True), t.clone().requires_grad_(True)
        y, z = f(one, one), f(a, b)
        assert torch.equal(y, z)
        got, want = torch.autograd.grad(y, one, dy)[0], torch.autograd.grad(z, [a, b], dy)
        assert torch.equal(got, want[0] + want[1])

    both(lambda a, b: ops_mlp.layer_norm(x, a, b), s)
    both(lambda a, b: ops_mlp.dropout(a, 0.3, 4, residual=b), x)
    both(lambda a, b: ops_mlp.linear_act(a, x, act="relu", residual=b), x)
    both(lambda a, b: ops_mlp.linear_act(a, b, act="silu"), x)


def test_tensors_changed_before_the_backward_pass_are_noticed():
    from shadow_gnn_amd import ops_mlp
    g = _gen(60)
    W, label = _randn(g, 64, 64, dtype=BF16).requires_grad_(True), torch.zeros(64, dtype=torch.int64, device=DEV)
    seed = torch.tensor([5], device=DEV)
    x = _randn(g, 64, 64, dtype=BF16)

    def changed(f, t, leaf):
        y = f()
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.sum(), leaf)

    changed(lambda: ops_mlp.linear_act(x, W), x, W)
    changed(lambda: ops_mlp.dropout(W, 0.5, seed), seed, W)
    changed(lambda: ops_mlp.label_logprobs(W, label).logprob, label, W)


def test_offsets_past_32_bits():
    """Rows 2^30 + 8 elements apart: the third begins past 2^31 elements."""
    from shadow_gnn_amd import ops, ops_mlp
    g = _gen(52)
    pitch = (1 << 30) + 8
    buf = torch.empty(2 * pitch + 1024, dtype=BF16, device=DEV)
    x = buf.as_strided((3, 256), (pitch, 1))
    base = _randn(g, 3, 256, dtype=BF16)
    x.copy_(base)
    assert torch.equal(ops_mlp.layer_norm(x), ops_mlp.layer_norm(base))
    assert torch.equal(ops_mlp.dropout(x, 0.5, 9, residual=x), ops_mlp.dropout(base, 0.5, 9, residual=base))
    W, label = _randn(g, 64, 256, dtype=BF16), torch.tensor([1, 2, 3], device=DEV)
    assert torch.equal(ops_mlp.linear_act(x, W, act="relu"), ops_mlp.linear_act(base, W, act="relu"))
    for a, b in zip(ops_mlp.label_logprobs(x, label, topk=3), ops_mlp.label_logprobs(base, label, topk=3)):
        assert torch.equal(a, b)
    # a contiguous array of more than 2^31 elements: the last rows' masks and values
    n, F = (1 << 31) // 254 + 3, 254
    flat = buf[:n * F].view(n, F) if n * F <= buf.numel() else torch.empty(n, F, dtype=BF16, device=DEV)
    flat[-2:] = base[:2, :F]
    y = ops_mlp.dropout(flat, 0.5, 11)
    keep = ops.dropout_keep_mask(n, 1, 0.5, 11, DEV)              # (column 0 of every row)
    del keep
    row = torch.tensor([n - 2, n - 1], device=DEV)
    M32 = 0xFFFFFFFF
    rowh = (ops._mix32((row & M32) ^ 11) + (row >> 32)) & M32
    c = torch.arange(F, device=DEV)
    h = ops._mix32((rowh[:, None] + ops._mul32(c >> 1, 0x9E3779B1)[None, :]) & M32)
    kept = torch.where((c & 1) == 1, h >> 16, h & 0xFFFF) >= 32768
    assert torch.equal(y[-2:], torch.where(kept, base[:2, :F] * 2, torch.zeros((), dtype=BF16, device=DEV)))


def test_negating_views():
    """The imaginary part of a conjugate negates on reading; rows of one element and vectors of one are taken without a copy."""
    from shadow_gnn_amd import ops_mlp
    g = _gen(64)

    def view(*shape):
        t = torch.complex(_randn(g, *shape), _randn(g, *shape)).conj().imag
        assert t.is_neg()
        return t

    def same(f, *views):
        def run(ts):
            ts = [t.detach().requires_grad_(True) for t in ts]
            y = f(*ts)
            return (y,) + torch.autograd.grad(y, ts, y.detach())
        for a, b in zip(run(views), run([t.resolve_neg() for t in views])):
            assert torch.equal(a, b)

    label = torch.zeros(9, dtype=torch.int64, device=DEV)
    same(lambda x, s, o: ops_mlp.layer_norm(x, s, o), view(9, 1), view(1), view(1))
    same(lambda x, r: ops_mlp.dropout(x, 0.25, 3, residual=r), view(9, 1), view(9, 1))
    same(lambda b: ops_mlp.linear_act(torch.ones(9, 8, dtype=BF16, device=DEV), torch.ones(1, 8, dtype=BF16, device=DEV), b, act="gelu").float(), view(1))
    same(lambda x: ops_mlp.label_logprobs(x, label).logprob, view(9, 1))
    same(lambda x: ops_mlp.label_logprobs(x, label).entropy, view(9, 5))
    x = _randn(g, 9, 1).requires_grad_(True)
    dy = view(9, 1)
    assert torch.equal(*[torch.autograd.grad(ops_mlp.dropout(x, 0.0, 1), x, t)[0] for t in (dy, dy.resolve_neg())])
    x = _randn(g, 5).requires_grad_(True)
    dy = view(5)[2]
    out = ops_mlp.label_logprobs(x, torch.tensor(3, device=DEV)).logprob
    assert torch.equal(*[torch.autograd.grad(out, x, t, retain_graph=True)[0] for t in (dy, dy.resolve_neg())])


def test_other_streams():
    from shadow_gnn_amd import ops_mlp
    g = _gen(53)
    x, W, label = _randn(g, 3000, 256, dtype=BF16), _randn(g, 256, 256, dtype=BF16, scale=0.1), torch.randint(0, 256, (3000,), device=DEV, generator=g)

    def block():
        h = ops_mlp.linear_act(ops_mlp.layer_norm(x), W, act="gelu", residual=x)
        return ops_mlp.label_logprobs(ops_mlp.dropout(h, 0.2, 5), label, topk=4)

    want = block()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:                                              # two calls at once, each on its own stream
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(block())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def _residual_block(x, p, label, seed):
    """Pre-norm residual MLP and its answers, as a program would write it."""
    from shadow_gnn_amd import ops_mlp
    h = ops_mlp.layer_norm(x, p["s"], p["o"])
    h = ops_mlp.linear_act(h, p["W1"], p["b1"], act="gelu")
    h = ops_mlp.linear_act(h, p["W2"], p["b2"])
    x = ops_mlp.dropout(h, 0.25, seed, residual=x)
    return ops_mlp.label_logprobs(ops_mlp.linear_act(x, p["W3"], p["b3"]), label, topk=3)


def _block_params(g, F, C, dtype):
    p = {"s": _randn(g, F) * 0.1 + 1, "o": _randn(g, F, scale=0.1), "W1": _randn(g, 2 * F, F, dtype=dtype, scale=F ** -0.5), "b1": _randn(g, 2 * F, scale=0.1),
         "W2": _randn(g, F, 2 * F, dtype=dtype, scale=(2 * F) ** -0.5), "b2": _randn(g, F, scale=0.1), "W3": _randn(g, C, F, dtype=dtype, scale=F ** -0.5), "b3": _randn(g, C, scale=0.1)}
    return {k: v.requires_grad_(True) for k, v in p.items()}


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_residual_block_and_its_gradients(dtype):
    from shadow_gnn_amd import ops
    g = _gen(54)
    n, F, C = 777, 104, 47
    x, label, p = _randn(g, n, F, dtype=dtype).requires_grad_(True), torch.randint(0, C, (n,), device=DEV, generator=g), None
    p = _block_params(g, F, C, dtype)
    out = _residual_block(x, p, label, 21)
    w = _randn(g, n)
    loss = -(out.logprob * w).sum() - 0.1 * out.entropy.sum()
    names = list(p)
    grads = torch.autograd.grad(loss, [x] + [p[k] for k in names])
    x64 = x.detach().double().requires_grad_(True)
    q = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    var, mean = torch.var_mean(x64, 1, correction=0, keepdim=True)
    h = (x64 - mean) / torch.sqrt(var + 1e-5) * q["s"] + q["o"]
    h = torch.nn.functional.gelu(h @ q["W1"].t() + q["b1"]) @ q["W2"].t() + q["b2"]
    h = x64 + h * ops.dropout_keep_mask(n, F, 0.25, 21, DEV) / 0.75
    lp = torch.log_softmax(h @ q["W3"].t() + q["b3"], 1)
    loss64 = -(lp.gather(1, label[:, None])[:, 0] * w).sum() + 0.1 * (lp.exp() * lp).sum()
    want = torch.autograd.grad(loss64, [x64] + [q[k] for k in names])
    # six tensors are rounded to 16 bits on the way forward and six on the way back: at most 12 half steps of a value's size, which add
    # like independent errors over a row (2-norms are compared, factor 2 for the slopes' curvature)
    for name, a, b in zip(["x"] + names, grads, want):
        assert (a.double() - b).norm() <= 24 * _half(dtype) * b.norm(), name
    assert (out.logprob.double() - lp.gather(1, label[:, None])[:, 0]).norm() <= 12 * _half(dtype) * (h @ q["W3"].t()).norm()


def test_captured_and_replayed():
    """Forward and backward in one graph, the seed on the device: every replay equals the eager result for that seed, with eager work
    and synchronisations between replays; two graphs of the same operators share nothing."""
    g = _gen(55)
    n, F, C = 1500, 96, 3000                                        # (3000 classes: the streamed form, split over workgroups)
    label = torch.randint(0, C, (n,), device=DEV, generator=g)
    p = {k: v.detach() for k, v in _block_params(g, F, C, BF16).items()}
    x0 = _randn(g, n, F, dtype=BF16)

    def passes(x, q, seed):
        out = _residual_block(x, q, label, seed)
        grads = torch.autograd.grad([out.logprob, out.entropy], [x] + list(q.values()), [torch.ones_like(out.logprob), torch.ones_like(out.entropy)])
        return list(out) + list(grads)

    def fresh():
        return x0.clone().requires_grad_(True), {k: v.clone().requires_grad_(True) for k, v in p.items()}

    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        x, q = fresh()
        seed = torch.tensor([1], dtype=torch.int64, device=DEV)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            passes(x, q, seed)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs = passes(x, q, seed)
        graphs.append((gr, x, seed, outs))
    for step in range(4):
        for which, (gr, x, seed, outs) in enumerate(graphs):
            s = 100 * step + which
            seed.fill_(s)
            x.data.copy_(x0 * (1 + step))
            gr.replay()
            torch.cuda.synchronize()
            xe, qe = fresh()
            xe.data.mul_(1 + step)
            want = passes(xe, qe, s)
            for i, (a, b) in enumerate(zip(outs, want)):
                assert torch.equal(a, b), (step, which, i)


def test_kernel_timer_sees_the_operators():
    from shadow_gnn_amd import ops
    g = _gen(56)
    x, label = _randn(g, 100, 64, dtype=BF16), torch.zeros(100, dtype=torch.int64, device=DEV)
    p = _block_params(g, 64, 40, BF16)
    with ops.KernelTimer() as t:
        _residual_block(x, p, label, 1)
        torch.cuda.synchronize()
        names = set(t.summary())
    assert {"layer_norm_fwd_F64", "dropout_F64", "label_logprobs_fwd_C40"} <= names and any(n.startswith("linear16_fwd") for n in names)

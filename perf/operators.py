"""Cases of the node-wise MLP operators (shadow_gnn_amd/ops_mlp.py): layer norm, counter-based dropout, the 16-bit matrix product
with its epilogue, and log probabilities of labels with entropy and top alternatives.

Sizes: 289127 rows of 256 are the sampled nodes of one 1024-root batch of the benchmark's products workload at its hidden width,
1024 / 256 rows the roots of a batch, 500 / 602 / 800 feature and hidden widths of the training configurations, 47 / 172 the
classes of products / papers100M; the wide products and the long label axis are generic."""
import math

import numpy as np
import torch

own = False

_DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_ACTS = ("I", "relu", "elu", "tanh", "leakyrelu", "gelu", "silu")


def listed():
    return [
        # layer norm of the root embeddings of one batch when answering: one short launch
        {"name": "ln_roots_f32", "op": "layer_norm", "rows": 1024, "width": 256, "dtype": "float32", "train": False},
        # ... of every sampled node of a training batch, forward and backward
        {"name": "ln_nodes_bf16_train", "op": "layer_norm", "rows": 289127, "width": 256, "dtype": "bfloat16", "train": True},
        # ... at the widest hidden size of the training configurations
        {"name": "ln_wide_f16_train", "op": "layer_norm", "rows": 16385, "width": 800, "dtype": "float16", "train": True},
        # dropout added to the residual stream of a training batch, forward and backward
        {"name": "drop_nodes_bf16_train", "op": "dropout", "rows": 289127, "width": 256, "dtype": "bfloat16", "p": 0.35, "residual": True, "train": True},
        # input dropout of raw fp32 features whose width is no multiple of four
        {"name": "drop_feat602_f32", "op": "dropout", "rows": 50021, "width": 602, "dtype": "float32", "p": 0.1, "residual": False, "train": False},
        # one residual MLP product over the roots of a batch when answering
        {"name": "lin_roots_bf16", "op": "linear_act", "rows": 256, "k": 256, "n": 256, "dtype": "bfloat16", "act": "relu", "bias": True, "residual": True, "train": False},
        # the same over every sampled node, forward and all gradients
        {"name": "lin_nodes_bf16_train", "op": "linear_act", "rows": 289127, "k": 256, "n": 256, "dtype": "bfloat16", "act": "relu", "bias": True, "residual": True, "train": True},
        # a wide expansion, bound by the matrix cores
        {"name": "lin_expand_f16", "op": "linear_act", "rows": 32768, "k": 1024, "n": 4096, "dtype": "float16", "act": "gelu", "bias": True, "residual": False, "train": False},
        # a classifier over 47 classes on 500 raw features (rows not 16-byte aligned), forward and all gradients
        {"name": "lin_classes_bf16_train", "op": "linear_act", "rows": 20011, "k": 500, "n": 47, "dtype": "bfloat16", "act": "I", "bias": True, "residual": False, "train": True},
        # one row over a long axis: a single answer
        {"name": "lp_one_f16", "op": "label_logprobs", "rows": 1, "classes": 131072, "dtype": "float16", "topk": 10, "train": False},
        # predictions of a whole training batch over the papers100M classes, with their gradients
        {"name": "lp_nodes_f32_train", "op": "label_logprobs", "rows": 289127, "classes": 172, "dtype": "float32", "topk": 5, "train": True},
        # a long label axis in training
        {"name": "lp_long_bf16_train", "op": "label_logprobs", "rows": 2048, "classes": 131072, "dtype": "bfloat16", "topk": 0, "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Half of the widths are multiples of eight (rows of whole 16-byte words), the others any."""
    w = _log_int(rng, lo, hi)
    return max(8, w // 8 * 8) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(("layer_norm", "dropout", "linear_act", "label_logprobs"))
    dtype = rng.choice(("bfloat16", "float16") if op == "linear_act" else ("float32", "bfloat16", "float16"))
    train = rng.random() < 0.6
    if op in ("layer_norm", "dropout"):
        width = _width(rng, 16, 1024)
        c = {"op": op, "rows": _log_int(rng, 1, min(300000, 70_000_000 // width)), "width": width, "dtype": dtype, "train": train}
        if op == "dropout":
            c["p"] = rng.choice((0.1, 0.25, 0.35, 0.5, 0.9))
            c["residual"] = rng.random() < 0.5
        return c
    if op == "linear_act":
        k, n = _width(rng, 16, 2048), _width(rng, 16, 2048)
        most = min(300000, 70_000_000 // max(k, n), int(4.5e10 // (k * n)))
        return {"op": op, "rows": _log_int(rng, 1, most), "k": k, "n": n, "dtype": dtype, "act": rng.choice(_ACTS),
                "bias": rng.random() < 0.8, "residual": rng.random() < 0.5, "train": train}
    classes = _log_int(rng, 2, 200000)
    return {"op": op, "rows": _log_int(rng, 1, min(300000, 50_000_000 // classes)), "classes": classes, "dtype": dtype,
            "topk": min(classes, rng.choice((0, 1, 5, 10, 20))), "train": train}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, train = _DT[case["dtype"]], case["train"]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    def leaf(t):
        return t.requires_grad_(True) if train else t

    s = {"case": case, "seed": int(seed) * 0x9E3779B97F4A7C15 % (1 << 62)}
    m = case["rows"]
    if case["op"] == "layer_norm":
        f = case["width"]
        # activations of a residual stream: every row has a level and a spread of its own
        x = torch.randn(m, f, device="cuda", generator=g) * (0.5 + torch.rand(m, 1, device="cuda", generator=g)) + randn(m, 1, dtype=torch.float32)
        s["x"] = leaf(x.to(dt))
        s["scale"] = leaf(1.0 + 0.1 * randn(f, dtype=torch.float32))
        s["offset"] = leaf(0.1 * randn(f, dtype=torch.float32))
        if train:
            s["dy"] = randn(m, f)
    elif case["op"] == "dropout":
        f = case["width"]
        s["x"] = leaf(randn(m, f))
        s["residual"] = leaf(randn(m, f)) if case["residual"] else None
        if train:
            s["dy"] = randn(m, f)
    elif case["op"] == "linear_act":
        k, n = case["k"], case["n"]
        s["x"] = leaf(randn(m, k))
        s["weight"] = leaf(randn(n, k, scale=k ** -0.5))
        s["bias"] = leaf(randn(n, scale=0.1)) if case["bias"] else None
        s["residual"] = leaf(randn(m, n)) if case["residual"] else None
        if train:
            s["dy"] = randn(m, n)
    else:
        c = case["classes"]
        s["logits"] = leaf(randn(m, c, scale=2.5))
        label = torch.randint(0, c, (m,), device="cuda", generator=g)
        # one row in sixteen has no label
        s["label"] = torch.where(torch.rand(m, device="cuda", generator=g) < 1.0 / 16, torch.full_like(label, -1), label)
        if train:
            s["dlp"] = randn(m, dtype=torch.float32)
            s["dent"] = 0.1 * randn(m, dtype=torch.float32)
    return s


# ---------------------------------------------------------------- plain forms

def _act(name, z):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "elu":
        return torch.where(z > 0, z, torch.expm1(z))
    if name == "tanh":
        return torch.tanh(z)
    if name == "leakyrelu":
        return torch.where(z > 0, z, 0.2 * z)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "elu":
        return torch.where(z > 0, torch.ones_like(z), torch.exp(z))
    if name == "tanh":
        return 1.0 - torch.tanh(z) ** 2
    if name == "leakyrelu":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, 0.2))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _mix(h):
    """The 32-bit finaliser of the mask rule on int64 tensors of 32-bit values (products kept below 2^63 in two halves)."""
    h = h ^ (h >> 16)
    h = (((h & 0xFFFF) * 0x85EBCA6B) + ((((h >> 16) * 0xCA6B) & 0xFFFF) << 16)) & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = (((h & 0xFFFF) * 0xC2B2AE35) + ((((h >> 16) * 0xAE35) & 0xFFFF) << 16)) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _kept(rows, width, p, seed, device):
    """The documented mask rule: row hash, one finaliser per pair of columns, a 16-bit field per element."""
    r = torch.arange(rows, device=device)
    row = (_mix((r & 0xFFFFFFFF) ^ (seed & 0xFFFFFFFF)) + (r >> 32) + (seed >> 32)) & 0xFFFFFFFF
    pair = torch.arange((width + 1) // 2, device=device)
    step = ((pair & 0xFFFF) * 0x9E3779B1 + ((((pair >> 16) * 0x79B1) & 0xFFFF) << 16)) & 0xFFFFFFFF
    h = _mix((row[:, None] + step[None, :]) & 0xFFFFFFFF)
    field = torch.stack((h & 0xFFFF, h >> 16), dim=2).reshape(rows, -1)[:, :width]
    return field >= int(min(max(float(np.float32(p)) * 65536.0, 1.0), 65535.0))


def _plain_layer_norm(s):
    x, w, b = s["x"].float(), s["scale"].float(), s["offset"].float()
    d = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + 1e-5)
    n = d * r
    y = (n * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * n).sum(0), dy.sum(0)


def _plain_dropout(s):
    x, c = s["x"], s["case"]
    keep = _kept(c["rows"], c["width"], c["p"], s["seed"], x.device) if c["p"] > 0 else None
    scale = 1.0 / (1.0 - c["p"])

    def masked(t):
        return torch.where(keep, t.float() * scale, torch.zeros((), device=t.device)) if keep is not None else t.float()

    y = masked(x)
    if c["residual"]:
        y = y + s["residual"].float()
    if not c["train"]:
        return y.to(x.dtype)
    return (y.to(x.dtype), masked(s["dy"]).to(x.dtype)) + ((s["dy"],) if c["residual"] else ())


def _plain_linear_act(s):
    c, x, w = s["case"], s["x"].float(), s["weight"].float()
    dt = s["x"].dtype
    z = x @ w.t()
    if c["bias"]:
        z = z + s["bias"].float()
    y = _act(c["act"], z)
    if c["residual"]:
        y = y + s["residual"].float()
    y = y.to(dt)
    if not c["train"]:
        return y
    dz = s["dy"].float()
    if c["act"] != "I":
        dz = dz * _act_slope(c["act"], z)
    out = (y, (dz @ w).to(dt), (dz.t() @ x).to(dt))
    if c["bias"]:
        out += (dz.sum(0).to(dt),)
    return out + ((s["dy"],) if c["residual"] else ())


def _order_key(x):
    """int64 keys that order the values of a row and, among equal values, put the lowest index first (all keys distinct)."""
    bits = x.float().contiguous().view(torch.int32).to(torch.int64)
    bits = torch.where(bits == -(1 << 31), torch.zeros_like(bits), bits)                # -0 and +0 are equal
    value = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return value * (1 << 24) - torch.arange(x.shape[1], device=x.device)


def _plain_label_logprobs(s):
    c, x = s["case"], s["logits"].float()
    label = s["label"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lp = (x - m) - torch.log(total)
    p = e / total
    ent = -(p * lp).sum(1)
    has = label >= 0
    at = label.clamp(min=0)[:, None]
    chosen = torch.where(has, lp.gather(1, at)[:, 0], torch.zeros_like(ent))
    idx = torch.topk(_order_key(s["logits"]), c["topk"], dim=1).indices if c["topk"] else torch.empty(c["rows"], 0, dtype=torch.int64, device=x.device)
    out = (chosen, ent, lp.gather(1, idx), idx)
    if not c["train"]:
        return out
    dlp = torch.where(has, s["dlp"], torch.zeros_like(ent))[:, None]
    d = -p * dlp - s["dent"][:, None] * p * (lp + ent[:, None])
    d.scatter_add_(1, at, dlp)
    return out + (d.to(s["logits"].dtype),)


_PLAIN = {"layer_norm": _plain_layer_norm, "dropout": _plain_dropout, "linear_act": _plain_linear_act, "label_logprobs": _plain_label_logprobs}


# ---------------------------------------------------------------- the framework's operators

def _own(s):
    from shadow_gnn_amd import ops_mlp
    c = s["case"]
    if c["op"] == "layer_norm":
        y, leaves = ops_mlp.layer_norm(s["x"], s["scale"], s["offset"], eps=1e-5), (s["x"], s["scale"], s["offset"])
    elif c["op"] == "dropout":
        y = ops_mlp.dropout(s["x"], c["p"], s["seed"], residual=s["residual"])
        leaves = (s["x"], s["residual"])
    elif c["op"] == "linear_act":
        y = ops_mlp.linear_act(s["x"], s["weight"], s["bias"], act=c["act"], residual=s["residual"])
        leaves = (s["x"], s["weight"], s["bias"], s["residual"])
    else:
        out = ops_mlp.label_logprobs(s["logits"], s["label"], topk=c["topk"])
        out = (out.logprob, out.entropy, out.top_logprob, out.top_index)
        if not c["train"]:
            return out
        return out + torch.autograd.grad((out[0], out[1]), (s["logits"],), (s["dlp"], s["dent"]))
    if not c["train"]:
        return y
    return (y,) + torch.autograd.grad(y, [t for t in leaves if t is not None], s["dy"])


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    m, train = case["rows"], case["train"]
    if case["op"] == "layer_norm":
        f = case["width"]
        if not train:
            return {"bytes": 2 * m * f * e + 8 * f, "flops": 8 * m * f}
        return {"bytes": 4 * m * f * e + 16 * f, "flops": 20 * m * f}
    if case["op"] == "dropout":
        f = case["width"]
        streams = 2 + case["residual"] + (2 if train else 0)
        return {"bytes": streams * m * f * e, "flops": 10 * m * f}
    if case["op"] == "linear_act":
        k, n = case["k"], case["n"]
        elems = m * k + n * k + m * n * (1 + case["residual"]) + (n if case["bias"] else 0)
        if train:
            elems += m * n + m * k + n * k + (n if case["bias"] else 0)
        return {"bytes": elems * e, "flops": 2 * m * k * n * (3 if train else 1)}
    c, t = case["classes"], case["topk"]
    by = m * c * e + m * (8 + 8 + 12 * t)
    return {"bytes": by + (m * c * e + 8 * m if train else 0), "flops": (12 if train else 6) * m * c}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def _keep_by_rule(rows, width, p, seed):
    """The mask rule in numpy's wrapping 32-bit arithmetic."""
    def mix(h):
        h ^= h >> np.uint32(16)
        h *= np.uint32(0x85EBCA6B)
        h ^= h >> np.uint32(13)
        h *= np.uint32(0xC2B2AE35)
        h ^= h >> np.uint32(16)
        return h
    row = mix(np.arange(rows, dtype=np.uint32) ^ np.uint32(seed & 0xFFFFFFFF)) + np.uint32(seed >> 32)
    step = np.arange((width + 1) // 2, dtype=np.uint32) * np.uint32(0x9E3779B1)
    h = mix(row[:, None] + step[None, :])
    field = np.empty((rows, 2 * step.size), np.uint16)
    field[:, 0::2] = h & np.uint32(0xFFFF)
    field[:, 1::2] = h >> np.uint32(16)
    return field[:, :width] >= int(min(max(float(np.float32(p)) * 65536.0, 1.0), 65535.0))


def _ref_act(name, z):
    nn = torch.nn.functional
    return {"I": lambda: z, "relu": lambda: nn.relu(z), "elu": lambda: nn.elu(z), "tanh": lambda: torch.tanh(z),
            "leakyrelu": lambda: nn.leaky_relu(z, 0.2), "gelu": lambda: nn.gelu(z), "silu": lambda: nn.silu(z)}[name]()


def exact(case, seed):
    s = prepare(case, seed)
    train = case["train"]

    def wide(name):
        t = s[name]
        return None if t is None else t.detach().double().requires_grad_(train)

    if case["op"] == "layer_norm":
        leaves = [wide("x"), wide("scale"), wide("offset")]
        var, mean = torch.var_mean(leaves[0], 1, correction=0, keepdim=True)
        y = (leaves[0] - mean) / torch.sqrt(var + 1e-5) * leaves[1] + leaves[2]
    elif case["op"] == "dropout":
        leaves = [wide("x"), wide("residual")]
        y = leaves[0]
        if case["p"] > 0:
            keep = torch.from_numpy(_keep_by_rule(case["rows"], case["width"], case["p"], s["seed"])).cuda()
            y = y * keep / (1.0 - case["p"])
        if leaves[1] is not None:
            y = y + leaves[1]
    elif case["op"] == "linear_act":
        leaves = [wide("x"), wide("weight"), wide("bias"), wide("residual")]
        y = leaves[0].matmul(leaves[1].t())
        if leaves[2] is not None:
            y = y + leaves[2]
        y = _ref_act(case["act"], y)
        if leaves[3] is not None:
            y = y + leaves[3]
    else:
        x = wide("logits")
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        ent = -(lp.exp() * lp).sum(1)
        has, rows = s["label"] >= 0, torch.arange(case["rows"], device="cuda")
        chosen = torch.where(has, lp[rows, s["label"].clamp(min=0)], torch.zeros_like(ent))
        top = torch.topk(lp.detach(), case["topk"], dim=1).values if case["topk"] else lp.detach()[:, :0]
        out = (chosen.detach(), ent.detach(), top, None)
        if not train:
            return out
        return out + torch.autograd.grad((chosen, ent), (x,), (s["dlp"].double(), s["dent"].double()))
    if not train:
        return y.detach()
    return (y.detach(),) + torch.autograd.grad(y, [t for t in leaves if t is not None], s["dy"].double())

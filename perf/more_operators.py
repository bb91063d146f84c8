"""Measured cases of the node-wise operators around the feed-forward block: normalised rows, dense layers, dense layers of
many experts.

* ``norm``: total = x + residual, in the tensors' type; y = weight * total / sqrt(mean(total^2) + eps). Its backward takes
  gradients of both outputs and gives those of x, residual (one and the same) and weight. With ``eight`` y comes in e4m3
  with a float32 scale for each row, s = max(|y|, 2^-100) / 448, as round(y / s).
* ``dense``: y = residual + act_scale act(scale x W^T + bias), each part optional; the backward gives all gradients. With
  ``eight`` x and W are e4m3 with a scale for each of their rows, forward only, y in 16 bits.
* ``grouped``: y[r] = act_scale act(scale x[r] W[e]^T + bias[e]) for the rows offsets[e] <= r < offsets[e + 1] of expert e;
  rows in none give zeros. The backward gives all gradients, zero for an expert without rows.

``run`` computes them in plain torch operations, or with ``own`` through ``flashcart_amd.nn.functional``. ``exact``
states them again in float64.
"""

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
# 1 / sqrt(E[act(z)^2]) of a standard normal z, as the rescaled activations of the framework's layers
ACT_SCALE = {"silu": 1.6765324703310907, "sigmoid": 1.8462285453386054, "gelu": 1.0, "none": 1.0}


def listed():
    return [
        # one token of a running sequence: latency
        dict(name="norm_one_f16", op="norm", n=1, width=4096, dtype="float16", residual=True, eight=False, train=False),
        # the invariant channels of the 25,000 atoms of a cell in training
        dict(name="norm_atoms_f32", op="norm", n=25000, width=128, dtype="float32", residual=True, eight=False, train=True),
        # activations of a large training batch
        dict(name="norm_train_bf16", op="norm", n=16384, width=4096, dtype="bfloat16", residual=True, eight=False, train=True),
        # what an 8-bit product reads, rows of a prompt
        dict(name="norm_eight_bf16", op="norm", n=8192, width=5120, dtype="bfloat16", residual=True, eight=True, train=False),
        # one row through a wide layer: the weight is read once
        dict(name="dense_one_bf16", op="dense", n=1, width=4096, out=10240, dtype="bfloat16", act="silu", bias=True,
             residual=False, eight=False, train=False),
        # a residual layer on the invariant channels of 25,000 atoms, forward and all gradients
        dict(name="dense_atoms_f32", op="dense", n=25000, width=128, out=128, dtype="float32", act="silu", bias=True,
             residual=True, eight=False, train=True),
        # sizes that divide by nothing, forward and all gradients
        dict(name="dense_ragged_f16", op="dense", n=1537, width=519, out=1031, dtype="float16", act="gelu", bias=True,
             residual=True, eight=False, train=True),
        # the largest: a training step of a wide layer
        dict(name="dense_train_bf16", op="dense", n=16384, width=2048, out=5632, dtype="bfloat16", act="silu", bias=True,
             residual=False, eight=False, train=True),
        # a prompt through a layer in 8 bits, added to the residual
        dict(name="dense_eight_bf16", op="dense", n=8192, width=4096, out=5120, dtype="bfloat16", act="none", bias=True,
             residual=True, eight=True, train=False),
        # a few tokens, each at a few of many experts: the weights of those that have rows are read once
        dict(name="grouped_rows64_bf16", op="grouped", n=64, experts=64, width=2048, out=1024, dtype="bfloat16", act="silu",
             bias=False, skew=False, spare=0, train=False),
        # a layer with weights of its own for each of four elements, 25,000 atoms sorted by element
        dict(name="grouped_atoms_f32", op="grouped", n=25000, experts=4, width=128, out=128, dtype="float32", act="silu",
             bias=True, skew=False, spare=0, train=True),
        # a training step of 32 experts, some with several times the rows of others, the batch padded at its end
        dict(name="grouped_train_bf16", op="grouped", n=16384, experts=32, width=2048, out=2816, dtype="bfloat16",
             act="silu", bias=False, skew=True, spare=100, train=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "dense", "dense", "grouped"])
    dtype = rng.choice(sorted(DTYPES))
    train = rng.random() < 0.6
    if op == "norm":
        eight = not train and rng.random() < 0.5
        width = _log(rng, 4, 12000)
        return dict(op=op, n=_log(rng, 1, max(1, (1 << 25) // width)), width=width, dtype=dtype,
                    residual=rng.random() < 0.7, eight=eight, train=train)
    act = rng.choice(sorted(ACT_SCALE))
    slow = 4 if dtype == "float32" else 1
    if op == "dense":
        eight = not train and dtype != "float32" and rng.random() < 0.5
        width, out = _log(rng, 16, 8192), _log(rng, 16, 8192)
        most = 16384 * 2048 * 5632 // (width * out * slow)
        n = _log(rng, 1, max(1, min(32768, most, (1 << 27) // max(width, out))))
        if rng.random() < 0.5:  # widths as most programs choose them
            width, out = -(-width // 64) * 64, -(-out // 64) * 64
            n = max(1, n * 3 // 4) if n > 64 else n
        return dict(op=op, n=n, width=width, out=out, dtype=dtype, act=act, bias=rng.random() < 0.6,
                    residual=rng.random() < 0.5, eight=eight, train=train)
    experts = _log(rng, 2, 128)
    width, out = _log(rng, 16, 4096), _log(rng, 16, 4096)
    if rng.random() < 0.5:
        width, out = -(-width // 64) * 64, -(-out // 64) * 64
    experts = max(2, min(experts, (1 << 27) // (width * out)))
    most = 16384 * 2048 * 2816 // (width * out * slow)
    n = _log(rng, 1, max(1, min(32768, most, (1 << 26) // max(width, out))))
    return dict(op=op, n=n, experts=experts, width=width, out=out, dtype=dtype, act=act, bias=rng.random() < 0.5,
                skew=rng.random() < 0.5, spare=rng.choice([0, 0, 1, 37]), train=train)


def _bytes(case):
    return 4 if case["dtype"] == "float32" else 2


def _to_eight(y):
    """(n, width) float32 as e4m3 and a scale for each row."""
    scale = y.abs().amax(dim=1, keepdim=True).clamp(min=2.0 ** -100) / 448
    return (y / scale).clamp(-448, 448).to(torch.float8_e4m3fn), scale[:, 0]


def prepare(case, seed):
    dtype, n, width, train = DTYPES[case["dtype"]], case["n"], case["width"], case["train"]
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape, dtype=dtype, scale=1.0):
        return (torch.randn(*shape, device=DEVICE, generator=gen) * scale).to(dtype)

    state = dict(op=case["op"], train=train)
    if case["op"] == "norm":
        state.update(x=normal(n, width).requires_grad_(train), eight=case["eight"],
                     residual=normal(n, width).requires_grad_(train) if case["residual"] else None,
                     weight=(1 + normal(width, dtype=torch.float32, scale=0.1)).to(dtype).requires_grad_(train))
        if train:
            state["grad"] = normal(n, width)
            if case["residual"]:
                state["grad_total"] = normal(n, width)
        return state
    out, act = case["out"], case["act"]
    state.update(act=None if act == "none" else act, act_scale=ACT_SCALE[act], scale=width ** -0.5)
    if case["op"] == "dense":
        state.update(eight=case["eight"], bias=normal(out).requires_grad_(train) if case["bias"] else None,
                     residual=normal(n, out).requires_grad_(train) if case["residual"] else None)
        if case["eight"]:
            state["x"], state["x_scale"] = _to_eight(normal(n, width, dtype=torch.float32))
            state["weight"], state["weight_scale"] = _to_eight(normal(out, width, dtype=torch.float32))
            state["dtype"] = dtype
        else:
            state.update(x=normal(n, width).requires_grad_(train), weight=normal(out, width).requires_grad_(train))
        if train:
            state["grad"] = normal(n, out)
        return state
    experts, rows = case["experts"], n + case["spare"]
    share = torch.arange(1, experts + 1, device=DEVICE, dtype=torch.float32) ** (-0.5 if case["skew"] else 0.0)
    share = share[torch.randperm(experts, device=DEVICE, generator=gen)]
    count = torch.bincount(torch.multinomial(share, n, replacement=True, generator=gen), minlength=experts)
    offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
    state.update(x=normal(rows, width).requires_grad_(train), weight=normal(experts, out, width).requires_grad_(train),
                 bias=normal(experts, out).requires_grad_(train) if case["bias"] else None, offsets=offsets,
                 most=int(count.max()))
    if train:
        state["grad"] = normal(rows, out)
    return state


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["op"]](state)


def _own(s):
    from flashcart_amd.nn import functional as F

    if s["op"] == "norm":
        if s["eight"]:
            return F.rms_norm_add_quantized(s["x"], s["residual"], s["weight"], EPS)
        y, total = F.rms_norm_add(s["x"], s["residual"], s["weight"], EPS)
        if not s["train"]:
            return y, total
        if s["residual"] is None:
            return (y.detach(), total.detach(), *torch.autograd.grad(y, (s["x"], s["weight"]), s["grad"]))
        return (y.detach(), total.detach(), *torch.autograd.grad((y, total), (s["x"], s["residual"], s["weight"]),
                                                                 (s["grad"], s["grad_total"])))
    if s["op"] == "dense":
        if s["eight"]:
            return (F.quantized_dense(s["x"], s["x_scale"], s["weight"], s["weight_scale"], s["bias"], s["act"],
                                      s["act_scale"], s["scale"], s["residual"], s["dtype"]),)
        y = F.dense(s["x"], s["weight"], s["bias"], s["act"], s["act_scale"], s["scale"], s["residual"])
        wanted = [t for t in (s["x"], s["weight"], s["bias"], s["residual"]) if t is not None]
    else:
        y = F.grouped_dense(s["x"], s["weight"], s["offsets"], s["bias"], s["act"], s["act_scale"], s["scale"])
        wanted = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
    if not s["train"]:
        return (y,)
    return (y.detach(), *torch.autograd.grad(y, wanted, s["grad"]))


@torch.no_grad()
def _plain_norm(s):
    dtype = s["x"].dtype
    total = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(dtype)
    t, w = total.float(), s["weight"].float()
    inv = 1 / torch.sqrt((t * t).mean(dim=1, keepdim=True) + EPS)
    xhat = t * inv
    y = xhat * w
    if s["eight"]:
        return (*_to_eight(y), total)
    if not s["train"]:
        return y.to(dtype), total.detach()
    g = s["grad"].float()
    gw = g * w
    dx = inv * (gw - xhat * (gw * xhat).mean(dim=1, keepdim=True))
    dw = (g * xhat).sum(dim=0).to(dtype)
    if s["residual"] is None:
        return y.to(dtype), total.detach(), dx.to(dtype), dw
    dx = (dx + s["grad_total"].float()).to(dtype)
    return y.to(dtype), total, dx, dx, dw


def _act(z, name):
    """act(z) and its derivative."""
    if name is None:
        return z, torch.ones_like(z)
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    sig = 1 / (1 + torch.exp(-z))
    if name == "sigmoid":
        return sig, sig * (1 - sig)
    return z * sig, sig * (1 + z * (1 - sig))


@torch.no_grad()
def _plain_dense(s):
    x, w = s["x"].float(), s["weight"].float()
    z = (x @ w.t()) * s["scale"]
    if s["eight"]:
        z = z * s["x_scale"][:, None] * s["weight_scale"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    a, d = _act(z, s["act"])
    y = a * s["act_scale"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not s["train"]:
        return (y.to(s["dtype"] if s["eight"] else s["x"].dtype),)
    dtype = s["x"].dtype
    dz = s["grad"].float() * d * s["act_scale"]
    grads = [((dz @ w) * s["scale"]).to(dtype), ((dz.t() @ x) * s["scale"]).to(dtype)]
    if s["bias"] is not None:
        grads.append(dz.sum(dim=0).to(dtype))
    if s["residual"] is not None:
        grads.append(s["grad"])
    return (y.to(dtype), *grads)


@torch.no_grad()
def _plain_grouped(s):
    """Each expert's rows in a block of as many rows as the largest expert has, one batched product."""
    dtype, offsets, n = s["x"].dtype, s["offsets"], s["x"].shape[0]
    w = s["weight"].float()
    at = offsets[:-1, None] + torch.arange(s["most"], device=offsets.device)
    used = (at < offsets[1:, None])[..., None]
    at = at.clamp(max=n - 1)
    rows = torch.arange(n, device=offsets.device)
    inside = (rows < offsets[-1])[:, None]
    expert = (torch.searchsorted(offsets, rows, right=True) - 1).clamp(max=w.shape[0] - 1)
    place = (rows - offsets[expert]).clamp(max=s["most"] - 1)

    def blocks(t):
        return torch.where(used, t.float()[at], 0.0)

    def lines(t):
        return torch.where(inside, t[expert, place], 0.0).to(dtype)

    x = blocks(s["x"])
    z = torch.bmm(x, w.transpose(1, 2).contiguous()) * s["scale"]
    if s["bias"] is not None:
        z = z + s["bias"].float()[:, None]
    a, d = _act(z, s["act"])
    y = lines(a * s["act_scale"])
    if not s["train"]:
        return (y,)
    dz = blocks(s["grad"]) * d * s["act_scale"]
    grads = [lines(torch.bmm(dz, w) * s["scale"]), (torch.bmm(dz.transpose(1, 2).contiguous(), x) * s["scale"]).to(dtype)]
    if s["bias"] is not None:
        grads.append(dz.sum(dim=1).to(dtype))
    return (y, *grads)


_PLAIN = {"norm": _plain_norm, "dense": _plain_dense, "grouped": _plain_grouped}


def work(case):
    n, width, size, train = case["n"], case["width"], _bytes(case), case["train"]
    if case["op"] == "norm":
        streams = 2 + 2 * case["residual"] - case["eight"] * (1 - 1 / size)
        if train:  # both gradients and the rows that the first pass wrote, the gradient of x
            streams += 3 + case["residual"]
        return dict(bytes=int(streams * n * width * size) + (1 + train) * width * size, flops=n * width * (12 if train else 5))
    out = case["out"]
    if case["op"] == "dense":
        read = 1 if case["eight"] else size
        total = (n * width + width * out) * read + n * out * size * (1 + case["residual"]) + out * size * case["bias"]
        if train:
            total += (n * width + width * out + n * out) * size + out * size * case["bias"]
        return dict(bytes=total, flops=(6 if train else 2) * n * width * out)
    experts = case["experts"]
    used = experts if case["skew"] else int(math.ceil(experts * (1 - (1 - 1 / experts) ** n)))  # expected, of even shares
    total = (n * (width + out) + min(used, n) * width * out) * size
    if train:
        total += (n * (width + out) + experts * width * out) * size
    return dict(bytes=total, flops=(6 if train else 2) * n * width * out)


def exact(case, seed):
    s = prepare(case, seed)
    dtype = DTYPES[case["dtype"]]
    f = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "gelu": torch.nn.functional.gelu, None: torch.clone}
    if case["op"] == "norm":
        total = s["x"].detach().double()
        if s["residual"] is not None:  # as it is stored: y is the norm of that
            total = (total + s["residual"].detach().double()).to(dtype).double()
        total.requires_grad_(s["train"])
        weight = s["weight"].detach().double().requires_grad_(s["train"])
        y = weight * torch.rsqrt(total.pow(2).mean(-1, True) + EPS) * total
        if case["eight"]:
            scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1).clamp_min(2.0 ** -100) / 448
            return torch.div(y, scale[:, None]).float().to(torch.float8_e4m3fn).double(), scale, total
        if not s["train"]:
            return y, total
        dx, dw = torch.autograd.grad(y, (total, weight), s["grad"].double())
        if s["residual"] is None:
            return y.detach(), total.detach(), dx, dw
        dx = dx + s["grad_total"].double()
        return y.detach(), total.detach(), dx, dx, dw
    leaves = {k: s[k].detach().double() for k in ("x", "weight", "bias", "residual") if s.get(k) is not None}
    if case.get("eight"):
        leaves["x"] = leaves["x"] * s["x_scale"].double()[:, None]
        leaves["weight"] = leaves["weight"] * s["weight_scale"].double()[:, None]
    for t in leaves.values():
        t.requires_grad_(s["train"])

    def layer(x, weight, bias):
        return s["act_scale"] * f[s["act"]](torch.nn.functional.linear(x * s["scale"], weight, bias))

    if case["op"] == "dense":
        y = layer(leaves["x"], leaves["weight"], leaves.get("bias"))
        if "residual" in leaves:
            y = leaves["residual"] + y
    else:
        ends = s["offsets"].tolist()
        parts = [layer(leaves["x"][a:b], leaves["weight"][e], leaves["bias"][e] if "bias" in leaves else None)
                 for e, (a, b) in enumerate(zip(ends, ends[1:]))]
        y = torch.cat(parts + [leaves["x"].new_zeros(case["spare"], case["out"])])
    if not s["train"]:
        return (y,)
    return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), s["grad"].double()))

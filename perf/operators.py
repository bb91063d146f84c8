"""Measured cases of the node-wise operators: element/token embedding, gated feed-forward block, residual dropout.

* ``embedding``: rows of a table by index, times a scale; the table's gradient sums the rows of each index.
* ``feed_forward``: y = s_out (c act(g) u) W_out^T with [g | u] = s_in x W_in^T, W_in (2 hidden, width) the gate's
  rows above the other projection's; its backward gives the gradients of x and of both weights.
* ``dropout``: residual + keep x / (1 - p); keep[e] compares word e % 4 of the Philox4x32-10 block whose counter is
  (e // 4, offset) and whose key is the seed with floor(p 2^32). Its backward applies the same mask again.

``run`` computes them in plain torch operations, or with ``own`` through ``flashcart_amd.nn.functional``. ``exact``
states them again in float64.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
# 1 / sqrt(E[act(z)^2]) of a standard normal z, as the rescaled activations of the framework's layers
ACT_SCALE = {"silu": 1.6765324703310907, "sigmoid": 1.8462285453386054, "gelu": 1.0}


def listed():
    return [
        # element features of both ends of every edge of a 25,000-atom cell with four species (16 features, as the
        # element-dependent interaction has them), forward and gradient: very long runs of few rows
        dict(name="embed_edges_f32", op="embedding", n=1083777, rows=4, width=16, dtype="float32", ids="uniform",
             pad=False, train=True),
        # element embedding of the atoms of that cell, 128 channels, a table of all elements, forward and gradient
        dict(name="embed_atoms_f32", op="embedding", n=25000, rows=119, width=128, dtype="float32", ids="zipf", pad=False,
             train=True),
        # a training batch of tokens: few rows of a large table are common and most are rare, index 0 pads
        dict(name="embed_tokens_bf16", op="embedding", n=16384, rows=32000, width=1024, dtype="bfloat16", ids="zipf",
             pad=True, train=True),
        # one token of a running sequence: latency
        dict(name="embed_one_f16", op="embedding", n=1, rows=32000, width=4096, dtype="float16", ids="zipf", pad=False,
             train=False),
        # one row through a wide block: both weights are read once
        dict(name="ffn_one_bf16", op="feed_forward", n=1, width=4096, hidden=10240, dtype="bfloat16", act="silu",
             train=False),
        # a few dozen rows at once
        dict(name="ffn_rows48_f16", op="feed_forward", n=48, width=2048, hidden=5504, dtype="float16", act="gelu",
             train=False),
        # the invariant channels of 25,000 atoms, forward and all gradients
        dict(name="ffn_atoms_f32", op="feed_forward", n=25000, width=128, hidden=512, dtype="float32", act="silu",
             train=True),
        # sizes that divide by nothing, forward and all gradients
        dict(name="ffn_ragged_f16", op="feed_forward", n=1537, width=519, hidden=1031, dtype="float16", act="sigmoid",
             train=True),
        # the largest: a training step of a wide block
        dict(name="ffn_train_bf16", op="feed_forward", n=16384, width=2048, hidden=5632, dtype="bfloat16", act="silu",
             train=True),
        # the smallest dropout, odd sizes, no residual
        dict(name="dropout_small_f16", op="dropout", n=7, width=129, dtype="float16", p=0.1, residual=False, train=True),
        # the invariant channels of 25,000 atoms in training
        dict(name="dropout_atoms_f32", op="dropout", n=25000, width=128, dtype="float32", p=0.2, residual=True, train=True),
        # activations of a large training batch
        dict(name="dropout_train_bf16", op="dropout", n=16384, width=4096, dtype="bfloat16", p=0.1, residual=True,
             train=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embedding", "feed_forward", "feed_forward", "dropout"])
    dtype = rng.choice(sorted(DTYPES))
    train = rng.random() < 0.7
    if op == "embedding":
        width = _log(rng, 8, 4096)
        n = _log(rng, 1, min(1 << 20, (1 << 26) // width))
        rows = _log(rng, 2, min(1 << 17, (1 << 27) // width))
        return dict(op=op, n=n, rows=rows, width=width, dtype=dtype, ids=rng.choice(["uniform", "zipf"]),
                    pad=rng.random() < 0.5, train=train)
    if op == "feed_forward":
        width, hidden = _log(rng, 16, 4096), _log(rng, 16, 10240)
        most = 6 * 16384 * 2048 * 5632 // (6 * width * hidden * (4 if dtype == "float32" else 1))
        n = _log(rng, 1, max(1, min(32768, most, (1 << 28) // max(width, hidden))))
        if rng.random() < 0.5:  # widths as most programs choose them
            width, hidden = -(-width // 64) * 64, -(-hidden // 64) * 64
            n = max(1, n * 3 // 4) if n > 64 else n
        return dict(op=op, n=n, width=width, hidden=hidden, dtype=dtype, act=rng.choice(sorted(ACT_SCALE)), train=train)
    width = _log(rng, 1, 8192)
    n = _log(rng, 1, max(1, (1 << 25) // width))
    return dict(op=op, n=n, width=width, dtype=dtype, p=rng.choice([0.0, 0.1, 0.25, 0.5, 0.9]), residual=rng.random() < 0.6,
                train=train)


def _bytes(case):
    return 4 if case["dtype"] == "float32" else 2


def prepare(case, seed):
    dtype = DTYPES[case["dtype"]]
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=DEVICE, generator=gen) * scale).to(dtype)

    n, width, train = case["n"], case["width"], case["train"]
    if case["op"] == "embedding":
        u = torch.rand(n, device=DEVICE, generator=gen, dtype=torch.float64)
        rows = case["rows"]
        ids = (u * rows if case["ids"] == "uniform" else torch.exp(u * math.log(rows + 1)) - 1).long().clamp_(0, rows - 1)
        state = dict(ids=ids, table=normal(rows, width).requires_grad_(train), scale=math.sqrt(width),
                     padding_idx=0 if case["pad"] else None)
        if train:
            state["grad"] = normal(n, width)
    elif case["op"] == "feed_forward":
        hidden = case["hidden"]
        state = dict(x=normal(n, width).requires_grad_(train), w_in=normal(2 * hidden, width).requires_grad_(train),
                     w_out=normal(width, hidden).requires_grad_(train), act=case["act"],
                     act_scale=ACT_SCALE[case["act"]], scale_in=width ** -0.5, scale_out=hidden ** -0.5)
        if train:
            state["grad"] = normal(n, width)
    else:
        state = dict(x=normal(n, width).requires_grad_(train), p=case["p"],
                     residual=normal(n, width).requires_grad_(train) if case["residual"] else None,
                     rng=torch.tensor([int(seed) * 0x9E3779B97F4A7C15 % (1 << 63), int(seed) % 1000], device=DEVICE))
        if train:
            state["grad"] = normal(n, width)
    state["op"], state["train"] = case["op"], train
    return state


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["op"]](state)


def _own(s):
    from flashcart_amd.nn import functional as F

    if s["op"] == "embedding":
        out = F.embedding(s["ids"], s["table"], s["scale"], s["padding_idx"])
        wanted = (s["table"],)
    elif s["op"] == "feed_forward":
        out = F.gated_feed_forward(s["x"], s["w_in"], s["w_out"], s["act"], s["act_scale"], s["scale_in"], s["scale_out"])
        wanted = (s["x"], s["w_in"], s["w_out"])
    else:
        out = F.dropout_add(s["x"], s["residual"], s["p"], s["rng"])
        wanted = (s["x"],) if s["residual"] is None else (s["x"], s["residual"])
    if not s["train"]:
        return (out,)
    return (out.detach(), *torch.autograd.grad(out, wanted, s["grad"]))


@torch.no_grad()
def _plain_embedding(s):
    table, ids = s["table"], s["ids"]
    out = (table[ids].float() * s["scale"]).to(table.dtype)
    if not s["train"]:
        return (out,)
    # sorted by index, each row's sum is a difference of running sums (64 bits: runs of 10^5 terms)
    ids, order = torch.sort(ids, stable=True)
    upto = torch.cumsum(s["grad"][order].double().t().contiguous(), dim=1)
    rows = torch.arange(table.shape[0], device=ids.device)
    upto = torch.cat([upto.new_zeros(upto.shape[0], 1), upto], dim=1)
    total = (upto[:, torch.searchsorted(ids, rows, right=True)] - upto[:, torch.searchsorted(ids, rows)]).t().contiguous()
    total *= s["scale"]
    if s["padding_idx"] is not None:
        total[s["padding_idx"]] = 0
    return out, total.to(table.dtype)


def _act(g, name):
    """act(g) and its derivative."""
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    sig = 1 / (1 + torch.exp(-g))
    if name == "sigmoid":
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


@torch.no_grad()
def _plain_feed_forward(s):
    dtype, hidden = s["x"].dtype, s["w_out"].shape[1]
    x, w_in, w_out = s["x"].float(), s["w_in"].float(), s["w_out"].float()
    pre = (x @ w_in.t()) * s["scale_in"]
    gate, up = pre[:, :hidden], pre[:, hidden:]
    a, d = _act(gate, s["act"])
    h = s["act_scale"] * a * up
    y = (h @ w_out.t()) * s["scale_out"]
    if not s["train"]:
        return (y.to(dtype),)
    grad = s["grad"].float()
    dh = (grad @ w_out) * (s["scale_out"] * s["act_scale"])
    dpre = torch.cat([dh * up * d, dh * a], dim=1)
    return (y.to(dtype), ((dpre @ w_in) * s["scale_in"]).to(dtype), ((dpre.t() @ x) * s["scale_in"]).to(dtype),
            ((grad.t() @ h) * s["scale_out"]).to(dtype))


_LOW = 0xFFFFFFFF


def _words(n, rng):
    """Words 0 .. n - 1 of the generator as int64 numbers below 2^32 (products wrap at 64 bits, which keeps both halves)."""
    block = torch.arange(-(-n // 4), device=rng.device)
    k0, k1 = rng[0] & _LOW, (rng[0] >> 32) & _LOW
    c0, c1 = block & _LOW, block >> 32
    c2, c3 = (rng[1] & _LOW).expand_as(block), ((rng[1] >> 32) & _LOW).expand_as(block)
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:n]


@torch.no_grad()
def _plain_dropout(s):
    x, p = s["x"], s["p"]
    keep = (_words(x.numel(), s["rng"]) >= int(p * 2 ** 32)).view(x.shape)
    factor = 1 / (1 - p)
    out = torch.where(keep, x.float() * factor, 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    out = out.to(x.dtype)
    if not s["train"]:
        return (out,)
    gx = torch.where(keep, s["grad"].float() * factor, 0.0).to(x.dtype)
    return (out, gx) if s["residual"] is None else (out, gx, s["grad"])


_PLAIN = {"embedding": _plain_embedding, "feed_forward": _plain_feed_forward, "dropout": _plain_dropout}


def work(case):
    n, width, size, train = case["n"], case["width"], _bytes(case), case["train"]
    if case["op"] == "embedding":
        touched = min(n, case["rows"])
        total = n * 8 + (touched + n) * width * size
        if train:
            total += (n + case["rows"]) * width * size
        return dict(bytes=total, flops=n * width * (2 if train else 1))
    if case["op"] == "feed_forward":
        hidden = case["hidden"]
        weights = 3 * width * hidden
        if not train:
            return dict(bytes=(weights + 2 * n * width) * size, flops=2 * n * weights)
        return dict(bytes=(2 * weights + 4 * n * width) * size, flops=6 * n * weights)
    streams = 2 + case["residual"] + (2 * train) + (train and case["residual"])
    return dict(bytes=streams * n * width * size, flops=2 * n * width)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        table = s["table"].detach().double()
        out = torch.index_select(table, 0, s["ids"]) * s["scale"]
        if not s["train"]:
            return (out,)
        g = torch.zeros_like(table).index_add_(0, s["ids"], s["grad"].double()) * s["scale"]
        if s["padding_idx"] is not None:
            g[s["padding_idx"]] = 0
        return out, g
    if case["op"] == "feed_forward":
        leaves = [s[k].detach().double().requires_grad_(s["train"]) for k in ("x", "w_in", "w_out")]
        x, w_in, w_out = leaves
        gate, up = torch.chunk(torch.nn.functional.linear(x, w_in) * s["scale_in"], 2, dim=-1)
        f = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "gelu": torch.nn.functional.gelu}[s["act"]]
        y = torch.nn.functional.linear(s["act_scale"] * f(gate) * up, w_out) * s["scale_out"]
        if not s["train"]:
            return (y,)
        return (y.detach(), *torch.autograd.grad(y, leaves, s["grad"].double()))
    x = s["x"].detach().double()
    threshold = math.floor(s["p"] * 4294967296.0)
    keep = (_words_by_halves(x.numel(), [int(v) for v in s["rng"].tolist()]) >= threshold).view(x.shape)
    factor = 1.0 / (1.0 - s["p"])
    out = torch.where(keep, x * factor, torch.zeros_like(x))
    if s["residual"] is not None:
        out = out + s["residual"].detach().double()
    if not s["train"]:
        return (out,)
    gx = s["grad"].double() * keep * factor
    return (out, gx) if s["residual"] is None else (out, gx, s["grad"].double())


def _words_by_halves(n, rng):
    """The generator again: 32-bit products from 16-bit halves, nothing wraps."""
    m, seed, offset = 2 ** 32, rng[0] % 2 ** 64, rng[1] % 2 ** 64
    block = torch.arange((n + 3) // 4, device=DEVICE)
    words = [block % m, block // m, torch.full_like(block, offset % m), torch.full_like(block, offset // m)]
    key = [seed % m, seed // m]

    def product(a, b):
        low, high = a * (b % 65536), a * (b // 65536)
        mid = low // 65536 + high
        return mid // 65536, (mid % 65536) * 65536 + low % 65536

    for r in range(10):
        if r:
            key = [(key[0] + 0x9E3779B9) % m, (key[1] + 0xBB67AE85) % m]
        h0, l0 = product(words[0], 0xD2511F53)
        h1, l1 = product(words[2], 0xCD9E8D57)
        words = [h1 ^ words[1] ^ key[0], l1, h0 ^ words[3] ^ key[1], l0]
    return torch.stack(words, dim=1).flatten()[:n]

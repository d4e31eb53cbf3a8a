"""The gated fully connected unit and the dropout without a stored mask: cases
that stand for their use, their plain forms and their values in 64 bits.

    gated unit   H = keep * act(X Wg + bg) * (X Wu + bu) / (1 - p)
    dropout      y = keep * x / (1 - p)

`keep` comes from the framework's counter-based generator: element i takes word
i % 4 of Philox4x32-10 at counter (i // 4, offset), key (seed), and stays where
that word, as a 32-bit float times 2^-32, is not below p.
"""

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


# ------------------------------------------------------------------ cases
def _gated(name, m, k, n, dtype, act, bias, train, p):
    return {"name": name, "op": "gated", "m": m, "k": k, "n": n,
            "dtype": dtype, "act": act, "bias": bias, "train": train, "p": p}


def _dropout(name, rows, cols, dtype, p):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols,
            "dtype": dtype, "p": p}


def listed():
    return [
        # one image through a gated fc7 of VGG-F: latency of a single answer
        _gated("gated-eval-1", 1, 4096, 4096, "bf16", "silu", True, False, 0.0),
        # a dozen images through a gated fc6: the small evaluation batch
        _gated("gated-eval-12", 12, 9216, 4096, "bf16", "gelu", True, False,
               0.0),
        # evaluation in fp16 at the width of many rows
        _gated("gated-eval-2048", 2048, 2048, 8192, "fp16", "sigmoid", False,
               False, 0.0),
        # VGG-16's fc6 trained with a small batch: weights dominate
        _gated("gated-train-64", 64, 25088, 4096, "bf16", "relu", True, True,
               0.5),
        # VGG-F's fc6 at the framework's training batch, with its dropout
        _gated("gated-train-256", 256, 9216, 4096, "bf16", "silu", True, True,
               0.5),
        # odd sizes in every direction, as a pruned head has them
        _gated("gated-train-odd", 1003, 1001, 2747, "fp16", "gelu_tanh", True,
               True, 0.1),
        # the unit over very many rows: the matrix cores are the bound
        _gated("gated-train-8192", 8192, 4096, 8192, "bf16", "silu", False,
               True, 0.0),
        # between fc6 and fc7 at the training batch: launches are the bound
        _dropout("dropout-fc", 256, 4096, "bf16", 0.5),
        # a length that no vector width divides
        _dropout("dropout-odd", 1, 1000003, "fp32", 0.1),
        # the first convolution's activations of a whole batch
        _dropout("dropout-map", 256 * 54 * 54, 64, "bf16", 0.2),
        # a long pass over memory
        _dropout("dropout-long", 65537, 4096, "fp16", 0.3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.35:
        cols = _log_int(rng, 1, 8192)
        rows = max(1, _log_int(rng, 1 << 10, 1 << 28) // cols)
        return _dropout("", rows, cols, rng.choice(("bf16", "fp16", "fp32")),
                        rng.choice((0.1, 0.2, 0.25, 0.3, 0.5, 0.9)))
    train = rng.random() < 0.6
    m = _log_int(rng, 1, 8192)
    k, n = _log_int(rng, 64, 25088), _log_int(rng, 64, 8192)
    if rng.random() < 0.6:          # most widths are multiples of a vector
        k, n = max(64, k // 32 * 32), max(64, n // 32 * 32)
    while m * k * n > 8192 * 4096 * 8192:
        m = max(1, m // 2)
    return _gated("", m, k, n, rng.choice(("bf16", "bf16", "fp16")),
                  rng.choice(ACTS), rng.random() < 0.5, train,
                  rng.choice((0.0, 0.1, 0.5)) if train else 0.0)


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        t = torch.randn(*shape, generator=gen, device=DEVICE)
        return t.mul_(scale).to(dtype)

    state = {"case": case, "seed": 1234 + seed, "offset": 1 + seed % 1000}
    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        state["x"] = normal(*shape).requires_grad_()
        state["dy"] = normal(*shape)
        return state
    m, k, n = case["m"], case["k"], case["n"]
    grad = case["train"]
    leaves = [normal(m, k), normal(k, n, scale=math.sqrt(2.0 / k)),
              normal(k, n, scale=math.sqrt(2.0 / k))]
    if case["bias"]:
        leaves += [normal(n, scale=0.1), normal(n, scale=0.1)]
    state["leaves"] = [t.requires_grad_(grad) for t in leaves]
    if grad:
        state["dh"] = normal(m, n, scale=0.1)
    return state


# ------------------------------------------------------------- plain form
_LOW = 0xFFFFFFFF


def _keep(shape, p, seed, offset, device):
    """Which elements stay: Philox4x32-10 with whole numbers of 64 bits."""
    total = math.prod(shape)
    keep = torch.empty(total, dtype=torch.bool, device=device)
    step = 1 << 26                        # bounds the memory of the rounds
    for begin in range(0, total, step):
        end = min(total, begin + step)
        c = torch.arange(begin // 4, (end + 3) // 4, device=device)
        c0, c1 = c & _LOW, c >> 32
        c2 = torch.full_like(c, offset & _LOW)
        c3 = torch.full_like(c, 0x243F6A88)
        k0, k1 = seed & _LOW, 0xBB67AE85
        for _ in range(10):
            a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
            c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, \
                ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
            k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
        words = torch.stack((c0, c1, c2, c3), 1).reshape(-1)
        unit = words.to(torch.float32) * 2.0 ** -32
        keep[begin:end] = (unit >= p)[:end - begin]
    return keep.view(shape)


def _act(name, g):
    """The activation and its derivative, elementwise."""
    if name == "relu":
        one = (g > 0).to(g.dtype)
        return g * one, one
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(
            2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (
            1 + 3 * 0.044715 * g * g)
    s = 1 / (1 + torch.exp(-g))
    if name == "sigmoid":
        return s, s * (1 - s)
    return g * s, s * (1 + g * (1 - s))


def _plain_dropout(state):
    case, x, dy = state["case"], state["x"].detach(), state["dy"]
    keep = _keep(x.shape, case["p"], state["seed"], state["offset"], x.device)
    scale = 1 / (1 - case["p"])
    return tuple(torch.where(keep, t.float() * scale, 0.0).to(t.dtype)
                 for t in (x, dy))


def _plain_gated(state):
    case = state["case"]
    leaves = [t.detach().float() for t in state["leaves"]]
    x, wg, wu = leaves[:3]
    dtype = state["leaves"][0].dtype
    g, u = x @ wg, x @ wu
    if case["bias"]:
        g, u = g + leaves[3], u + leaves[4]
    a, da = _act(case["act"], g)
    h = a * u
    factor = None
    if case["p"] > 0:
        keep = _keep(h.shape, case["p"], state["seed"], state["offset"],
                     h.device)
        factor = keep.float() / (1 - case["p"])
        h = h * factor
    out = [h]
    if case["train"]:
        dh = state["dh"].float()
        if factor is not None:
            dh = dh * factor
        dg, du = dh * u * da, dh * a
        out += [dg @ wg.t() + du @ wu.t(), x.t() @ dg, x.t() @ du]
        if case["bias"]:
            out += [dg.sum(0), du.sum(0)]
    return tuple(t.to(dtype) for t in out)


# ---------------------------------------------------------------- the pass
def run(state):
    case = state["case"]
    if not own:
        return (_plain_dropout if case["op"] == "dropout"
                else _plain_gated)(state)
    from distributed_vgg_f_amd import ops
    if case["op"] == "dropout":
        y = ops.dropout(state["x"], case["p"], state["seed"], state["offset"])
        dx, = torch.autograd.grad(y, state["x"], state["dy"])
        return y.detach(), dx
    x, wg, wu, *bias = state["leaves"]
    bg, bu = bias if bias else (None, None)
    h = ops.gated_linear(x, wg, wu, bg, bu, act=case["act"], p=case["p"],
                         seed=state["seed"], offset=state["offset"])
    if not case["train"]:
        return (h,)
    return (h.detach(),) + torch.autograd.grad(h, state["leaves"], state["dh"])


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * n * size, "flops": 2 * n}
    m, k, n = case["m"], case["k"], case["n"]
    bias = 2 * n if case["bias"] else 0
    elems, flops = m * k + 2 * k * n + m * n + bias, 4 * m * n * k
    if case["train"]:
        elems, flops = 2 * elems, 3 * flops
    return {"bytes": elems * size, "flops": flops}


# -------------------------------------------------------- values in 64 bits
def _mul_wide(a, const):
    """High and low words of a 32-bit product, from limbs of 16 bits."""
    al, ah = a % 65536, a // 65536
    bl, bh = const % 65536, const // 65536
    low = al * bl
    mid = al * bh + low // 65536
    mid2 = ah * bl + mid % 65536
    return ah * bh + mid // 65536 + mid2 // 65536, \
        (mid2 % 65536) * 65536 + low % 65536


def _stays(index, p, seed, offset):
    """Truth values for flat indices, by the generator's definition."""
    block, word = index // 4, index % 4
    state = [block % 2 ** 32, block // 2 ** 32,
             torch.full_like(block, offset % 2 ** 32),
             torch.full_like(block, 0x243F6A88)]
    key = [seed % 2 ** 32, 0xBB67AE85]
    for _ in range(10):
        h0, l0 = _mul_wide(state[0], 0xD2511F53)
        h1, l1 = _mul_wide(state[2], 0xCD9E8D57)
        state = [h1.bitwise_xor(state[1]).bitwise_xor(key[0]), l1,
                 h0.bitwise_xor(state[3]).bitwise_xor(key[1]), l0]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32,
               (key[1] + 0xBB67AE85) % 2 ** 32]
    value = torch.stack(state).gather(0, word.unsqueeze(0)).squeeze(0)
    return value.to(torch.float32) / 2.0 ** 32 >= p


def _factor(shape, p, seed, offset):
    total = math.prod(shape)
    out = torch.zeros(total, dtype=torch.float64, device=DEVICE)
    for begin in range(0, total, 1 << 24):
        index = torch.arange(begin, min(total, begin + (1 << 24)),
                             device=DEVICE)
        out[index] = _stays(index, p, seed, offset).double() / (1 - p)
    return out.view(shape)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "dropout":
        shape = tuple(state["x"].shape)
        factor = _factor(shape, case["p"], state["seed"], state["offset"])
        return tuple(t.detach().double() * factor
                     for t in (state["x"], state["dy"]))
    x, wg, wu, *bias = [t.detach().double() for t in state["leaves"]]
    g, u = x.mm(wg), x.mm(wu)
    if bias:
        g += bias[0]
        u += bias[1]
    name = case["act"]
    g.requires_grad_(case["train"])
    if name == "silu":
        a = g * torch.sigmoid(g)
    elif name == "sigmoid":
        a = torch.sigmoid(g)
    elif name == "relu":
        a = torch.relu(g)
    elif name == "gelu":
        a = g * torch.special.ndtr(g)
    else:
        a = g * torch.sigmoid(2 * math.sqrt(2 / math.pi)
                              * (g + 0.044715 * g ** 3))
    factor = 1.0
    if case["p"] > 0:
        factor = _factor(tuple(g.shape), case["p"], state["seed"],
                         state["offset"])
    h = a.detach() * u * factor
    if not case["train"]:
        return (h,)
    dh = state["dh"].double() * factor
    du = dh * a.detach()
    dg, = torch.autograd.grad(a, g, dh * u)
    out = (h, dg.mm(wg.t()) + du.mm(wu.t()), x.t().mm(dg), x.t().mm(du))
    if bias:
        out += (dg.sum(0), du.sum(0))
    return out

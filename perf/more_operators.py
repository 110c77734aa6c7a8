"""Cases of the framework's operators of a training step over a frozen base in
microscaled 4 bits: packing, the block-scaled product with its input gradient,
and the AdamW step over many tensors with gradient clipping, its states in 32
or in 8 bits.

``run`` computes a case in its plain form (elementary torch operations in 32
bits, rounded once) or, where ``own`` is true, through the package's public
entry points; ``exact`` gives the same outputs from the definitions in 64
bits.
"""
import math
import os
import sys

import torch

#: set from outside: True makes ``run`` call the framework's operators
own = False

MX = 32                     # values of a row that share one scale of the 4-bit form
SB = 256                    # values of a tensor that share the scales of its 8-bit states
M_TOP = 448.0               # largest value of the first moment's codes (e4m3)
R_TOP = 507904.0            # largest value of the codes of the second moment's root: 31 * 2^14
FLUSH = 2.0 ** -100         # blocks whose largest magnitude is below this are stored as zeros
BETAS, EPS, DECAY, LR, MAX_NORM, STEPS = (0.9, 0.999), 1e-8, 0.01, 2e-4, 0.3, 100
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------- cases

def listed():
    """The sizes of the 7B projections that the benchmark and the tests use
    (4096, 11008, rank 16 and 64), and odd ones."""
    return [
        # the adapter of one projection, as a first experiment trains it
        dict(name="adam_one", op="adam", kind="adapters", layers=1, d=1093, f=1093, rank=8, bits=32, clip=False,
             master=False, dtype="f32"),
        # all adapters of a 7B model, 448 small tensors, clipped
        dict(name="adam_adapters", op="adam", kind="adapters", layers=32, d=4096, f=11008, rank=16, bits=32, clip=True,
             master=False, dtype="f32"),
        # the same in 16 bits with 8-bit states
        dict(name="adam8_adapters", op="adam", kind="adapters", layers=32, d=4096, f=11008, rank=64, bits=8, clip=True,
             master=False, dtype="bf16"),
        # one decoder block trained whole, its weights in bf16 with what their rounding leaves kept beside them
        dict(name="adam8_block", op="adam", kind="weights", layers=1, d=4096, f=11008, rank=0, bits=8, clip=False,
             master=True, dtype="bf16"),
        # one token's hidden state on its way into a projection
        dict(name="pack_1", op="pack", rows=1, k=4096, dtype="bf16"),
        # a checkpoint's projection
        dict(name="pack_11008", op="pack", rows=11008, k=4096, dtype="bf16"),
        # one chat request decoding through the query projection
        dict(name="linear_1", op="linear", mode="apply", rows=1, k=4096, n=4096, bias=False, dtype="bf16"),
        # a full decode batch through the up projection
        dict(name="linear_64", op="linear", mode="apply", rows=64, k=4096, n=11008, bias=False, dtype="bf16"),
        # prompts of a few requests of uneven length through the down projection
        dict(name="linear_2047", op="linear", mode="apply", rows=2047, k=11008, n=4096, bias=True, dtype="f16"),
        # a training batch through the up projection
        dict(name="train_8192", op="linear", mode="train", rows=8192, k=4096, n=11008, bias=False, dtype="bf16"),
        # odd sizes
        dict(name="train_1111", op="linear", mode="train", rows=1111, k=1093, n=1089, bias=True, dtype="f16"),
        # two operands that are packed already
        dict(name="product_4096", op="product", rows=4096, k=4096, n=4096, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adam", "adam", "adam", "pack", "linear", "linear", "linear", "product"])
    wide = [1024, 1088, 2048, 4096, 8192, 11008]
    size = lambda: rng.choice(wide) if rng.random() < 0.5 else _log(rng, 65, 11008)  # noqa: E731
    if op == "adam":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32", "f32"])
        c = dict(op=op, kind=rng.choice(["adapters", "adapters", "weights"]), bits=rng.choice([8, 8, 32]),
                 clip=rng.random() < 0.5, master=dtype == "bf16" and rng.random() < 0.5, dtype=dtype)
        if c["kind"] == "adapters":
            return dict(c, layers=_log(rng, 1, 32), d=_log(rng, 65, 4096), f=_log(rng, 65, 11008),
                        rank=rng.choice([8, 16, 16, 32, 64]))
        return dict(c, layers=1, d=_log(rng, 65, 4096), f=_log(rng, 65, 8192), rank=0)
    if op == "pack":
        return dict(op=op, rows=_log(rng, 1, 8192), k=size(), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if op == "product":
        return dict(op=op, rows=_log(rng, 1, 8192), k=size(), n=size(), dtype=rng.choice(["bf16", "f16"]))
    return dict(op=op, mode=rng.choice(["apply", "apply", "train"]), rows=_log(rng, 1, 8192), k=size(), n=size(),
                bias=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "f16"]))


def _shapes(c):
    """The trained tensors: A and B of the seven projections of each layer, or
    the projections and norms themselves."""
    d, f, r = c["d"], c["f"], c["rank"]
    pairs = [(d, d)] * 4 + [(d, f)] * 2 + [(f, d)]
    if c["kind"] == "weights":
        return (pairs + [(d,), (d,)]) * c["layers"]
    return [s for k, n in pairs for s in ((k, r), (n, r))] * c["layers"]


def _places(c):
    """(first, values, shape) of each tensor in one buffer: every tensor begins
    at a whole block of SB values."""
    found, at = [], 0
    for s in _shapes(c):
        n = math.prod(s)
        found.append((at, n, s))
        at += -(-n // SB) * SB
    return found, at


def work(c):
    e = _SIZE[c["dtype"]]
    if c["op"] == "adam":
        n = sum(math.prod(s) for s in _shapes(c))
        # gradients read, parameters read and written, both moments read and written
        moved = n * (3 * e + (16 if c["bits"] == 32 else 4)) + (n // SB * 16 if c["bits"] == 8 else 0)
        # the clipped norm needs every gradient before the first update
        return {"bytes": moved + (n * e if c["clip"] else 0) + (n * 4 if c["master"] else 0), "flops": 16 * n}
    m, k = c["rows"], c["k"]
    if c["op"] == "pack":
        # packed, and its values read back
        return {"bytes": m * k * 2 * e + 2 * (m * k // 2 + m * -(-k // MX)), "flops": 6 * m * k}
    n = c["n"]
    four = lambda rows: rows * (k // 2 + -(-k // MX))  # noqa: E731
    if c["op"] == "product":
        return {"bytes": four(m) + four(n) + m * n * e, "flops": 2 * m * n * k}
    moved = m * k * e + four(n) + m * n * e + (n * e if c["bias"] else 0)
    if c["mode"] == "apply":
        return {"bytes": moved, "flops": 2 * m * n * k}
    return {"bytes": moved + m * n * e + four(n) + m * k * e, "flops": 4 * m * n * k}


# ------------------------------------------------------------------ inputs

def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


def _draws(c, seed):
    """The inputs of a case, from the seed alone."""
    dev, dt = _device(), _DT[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    if c["op"] == "adam":
        places, total = _places(c)
        keep = torch.zeros(total, dtype=torch.bool, device=dev)
        for at, n, _ in places:
            keep[at:at + n] = True
        # gradients of some rows are much larger than the others'; the moments are of such gradients before
        size = torch.exp(1.5 * normal(total // SB, 1)).expand(-1, SB).reshape(-1) * 1e-4
        grad = normal(total).mul_(size)
        m = normal(total).mul_(size).mul_(0.3).add_(grad, alpha=0.2)
        v = size.square().mul_(torch.exp(0.7 * normal(total)))
        p = normal(total).mul_(0.02)
        for t in (grad, m, v, p):
            t.mul_(keep)
        return dict(p=p.to(dt), grad=grad.to(dt), m=m, v=v)
    m, k = c["rows"], c["k"]
    # a few features of the activations are much larger than the rest
    x = normal(m, k)
    x[:, :: max(1, k // 7)] *= 6.0
    s = dict(x=x.to(dt))
    if c["op"] == "pack":
        return s
    s["w"] = normal(c["n"], k).mul_(0.02).to(dt)
    if c["op"] == "linear":
        s["bias"] = normal(c["n"]).mul_(0.1).to(dt) if c["bias"] else None
        if c["mode"] == "train":
            s["dy"] = normal(m, c["n"]).mul_(0.1).to(dt)
    return s


def prepare(case, seed):
    s = _draws(case, seed)
    s["case"] = case
    if case["op"] == "adam":
        s["step"] = STEPS
        if case["bits"] == 8:
            s["m"], s["v"] = _kept_m(s["m"]), _kept_r(s["v"].sqrt()).square()
    elif case["op"] != "pack":
        # a frozen weight is packed once, when the model is loaded
        s["w4"] = _kept4(s["w"].float())
        if case["op"] == "product":
            s["x4"] = _kept4(s["x"].float())
    if own:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocm-qlora_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        if case["op"] == "adam":
            from rocm_qlora.optim import AdamW
            params = []
            for at, n, shape in _places(case)[0]:
                params.append(torch.nn.Parameter(s["p"][at:at + n].view(shape)))
                params[-1].grad = s["grad"][at:at + n].view(shape)
            s["adam"] = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                              remainder=case["master"], max_grad_norm=MAX_NORM if case["clip"] else None)
            s["adam"].set_moments(s["m"], s["v"], STEPS)
        elif case["op"] != "pack":
            from rocm_qlora.mx4 import pack_mx4
            s["packed_w"] = pack_mx4(s["w"])
            if case["op"] == "product":
                s["packed_x"] = pack_mx4(s["x"])
            elif case["mode"] == "train":
                s["x"].requires_grad_()
    elif case["op"] == "adam" and case["master"]:
        s["master"] = s["p"].float()
    return s


# --------------------------------------------------------------------- run

def run(s):
    c = s["case"]
    if c["op"] == "adam":
        return _own_adam(s) if own else _plain_adam(s)
    if c["op"] == "pack":
        return _own_pack(s) if own else _plain_pack(s)
    if c["op"] == "product":
        return _own_product(s) if own else _plain_product(s)
    return _own_linear(s) if own else _plain_linear(s)


def _own_adam(s):
    adam = s["adam"]
    adam.step()
    m, v = adam.moments()
    return [s["p"], m, v, adam.grad_norm]


def _own_pack(s):
    from rocm_qlora.mx4 import pack_mx4, unpack_mx4
    return [unpack_mx4(pack_mx4(s["x"]))]


def _own_product(s):
    from rocm_qlora.mx4 import mx4_matmul
    return [mx4_matmul(s["packed_x"], s["packed_w"], dtype=_DT[s["case"]["dtype"]])]


def _own_linear(s):
    from rocm_qlora.mx4 import mx4_linear
    y = mx4_linear(s["x"], s["packed_w"], s["bias"])
    if s["case"]["mode"] == "apply":
        return [y]
    return [y, *torch.autograd.grad(y, s["x"], s["dy"])]


def _kept4(x):
    """The values that the 4-bit codes of x [rows, K] stand for (32 bits): blocks
    of MX values of a row share the scale 2^e, e = floor(log2 max|x|) - 2; a
    code is the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6}, ties to even."""
    m, k = x.shape
    blocks = torch.nn.functional.pad(x, (0, -k % MX)).view(m, -1, MX)
    e = torch.frexp(blocks.abs().amax(-1, keepdim=True)).exponent.sub_(3).clamp_(min=-127)
    y = torch.ldexp(blocks, -e)
    a = y.abs().clamp_(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    y = torch.copysign(torch.round(a / step) * step, y)
    return torch.ldexp(y, e).view(m, -1)[:, :k].contiguous()


def _kept_m(x):
    """The values that the 8-bit codes of first moments stand for: blocks of SB
    values, code = e4m3(x * (448 / max|x|)), scale = max|x| / 448."""
    blocks = x.view(-1, SB)
    top = blocks.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, M_TOP)
    codes = torch.where(top < FLUSH, 0.0, blocks * most.div(top.clamp(min=FLUSH))).to(torch.float8_e4m3fn).float()
    return (codes * torch.where(top < FLUSH, 0.0, top.div(most))).view(-1)


def _kept_r(r):
    """The values that the 8-bit codes of second moments' roots stand for: a
    code of 4 exponent and 4 mantissa bits holds the whole numbers up to 31,
    then 16 steps to each power of two, up to R_TOP; what is not zero does not
    become zero."""
    blocks = r.view(-1, SB)
    top = blocks.amax(-1, keepdim=True)
    most = torch.full_like(top, R_TOP)
    t = torch.where(top < FLUSH, 0.0, blocks * most.div(top.clamp(min=FLUSH)))
    step = torch.ldexp(torch.ones_like(t), torch.frexp(t).exponent.sub_(5).clamp_(min=0))
    code = torch.where((blocks > 0.0) & (top >= FLUSH), (torch.round(t / step) * step).clamp(min=1.0), 0.0)
    return (code * torch.where(top < FLUSH, 0.0, top.div(most))).view(-1)


def _plain_adam(s):
    c, dt = s["case"], s["p"].dtype
    s["step"] += 1
    b1, b2 = BETAS
    g = s["grad"].float()
    norm = g.double().square().sum().sqrt().float() if c["clip"] else None
    if c["clip"]:
        g = g * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
    m = s["m"] * b1 + g * (1.0 - b1)
    v = s["v"] * b2 + g * g * (1.0 - b2)
    p = s["master"] if c["master"] else s["p"].float()
    p = p * (1.0 - LR * DECAY)
    root = v.sqrt()
    p = p - (LR / (1.0 - b1 ** s["step"])) * m / (root / math.sqrt(1.0 - b2 ** s["step"]) + EPS)
    if c["bits"] == 8:
        m, v = _kept_m(m), _kept_r(root).square()
    if c["master"]:
        s["master"] = p
    s["p"], s["m"], s["v"] = p.to(dt), m, v
    return [s["p"], m, v, norm]


def _plain_pack(s):
    return [_kept4(s["x"].float()).to(s["x"].dtype)]


def _plain_product(s):
    return [(s["x4"] @ s["w4"].t()).to(s["x"].dtype)]


def _plain_linear(s):
    x, dt = s["x"].float(), s["x"].dtype
    y = _kept4(x) @ s["w4"].t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["mode"] == "apply":
        return [y.to(dt)]
    return [y.to(dt), (s["dy"].float() @ s["w4"]).to(dt)]


# ------------------------------------------------------------------- exact

def _kept4_64(x):
    """_kept4 by its definition, in 64 bits: the nearest level of the eight."""
    m, k = x.shape
    out = torch.zeros(m, k, dtype=torch.float64, device=x.device)
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    between = (levels[1:] + levels[:-1]) / 2
    # a tie goes to the level with the even number: up out of the odd levels, and not out of the even ones
    odd = torch.arange(7, device=x.device) % 2 == 1
    for at in range(0, k, MX):
        part = x[:, at:at + MX].double()
        top = part.abs().max(1).values.clamp(min=2.0 ** -125)
        # floor(log2(top)) is the exponent that a 64-bit float holds; the scale's own bits are made of it
        scale = (((top.view(torch.int64) >> 52) - 2) << 52).view(torch.float64)[:, None]
        a = part.abs() / scale
        code = sum(((a > b) | ((a == b) & o)).long() for b, o in zip(between, odd))
        out[:, at:at + MX] = levels[code] * scale * torch.sign(part)
    return out


def exact(case, seed):
    c, s = case, _draws(case, seed)
    f8 = torch.float64
    if c["op"] == "adam":
        if c["bits"] == 8:  # the states in hand are those of the codes
            s["m"], s["v"] = _kept_m(s["m"]), _kept_r(s["v"].sqrt()).square()
        t, (b1, b2) = STEPS + 1, BETAS
        g = s["grad"].to(f8)
        norm = torch.linalg.vector_norm(g) if c["clip"] else None
        if c["clip"]:
            g *= min(1.0, MAX_NORM / (float(norm) + 1e-6))
        m = torch.lerp(g, s["m"].to(f8), b1)
        v = torch.lerp(g.square_(), s["v"].to(f8), b2)
        p = s["p"].to(f8) * (1.0 - LR * DECAY)
        p -= LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt_() + EPS)
        # the 8-bit states are codes of rounded moments: they have no value of their own in 64 bits
        return [p, m, v, norm] if c["bits"] == 32 else [p, None, None, norm]
    x = _kept4_64(s["x"])
    if c["op"] == "pack":
        return [x]
    w = _kept4_64(s["w"])
    y = x @ w.t()
    if c["op"] == "product":
        return [y]
    if s["bias"] is not None:
        y += s["bias"].to(f8)
    return [y, s["dy"].to(f8) @ w] if c["mode"] == "train" else [y]

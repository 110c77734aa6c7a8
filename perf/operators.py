"""Cases of the framework's training and serving operators: adapters of many
requests beside a shared projection, activations kept in 8 bits for the
backward pass, and the paired preference loss, each with its gradient.

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

BETA = 0.1
BLOCK = 128                 # values of a row that share one 8-bit scale
FLUSH = 2.0 ** -100         # blocks whose largest magnitude is below this are stored as zeros
IGNORE = -100               # label of a position that does not count
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------- cases

def listed():
    """The sizes of the 7B projections and vocabulary that the benchmark and
    the tests use (4096, 11008, 32000, rank 16 and 64), and odd ones."""
    return [
        # one chat request decoding through the query projection
        dict(name="decode_1", op="adapters", mode="apply", rows=1, k=4096, n=4096, rank=16, count=8, skew=1,
             dtype="bf16"),
        # a full decode batch, 32 customers' adapters, through the up projection
        dict(name="decode_64", op="adapters", mode="apply", rows=64, k=4096, n=11008, rank=16, count=32, skew=1,
             dtype="bf16"),
        # prompts of a few requests of uneven length through the down projection
        dict(name="prompts_2047", op="adapters", mode="apply", rows=2047, k=11008, n=4096, rank=64, count=5, skew=3,
             dtype="f16"),
        # a training batch of two adapters (policy and a rival) over one base
        dict(name="train_8192", op="adapters", mode="train", rows=8192, k=4096, n=4096, rank=16, count=2, skew=1,
             dtype="bf16"),
        # the gated MLP of a short batch
        dict(name="swiglu_61", op="checkpoint", mode="swiglu", rows=61, k=11008, dtype="bf16"),
        # the gated MLP of a training batch
        dict(name="swiglu_8192", op="checkpoint", mode="swiglu", rows=8192, k=11008, dtype="bf16"),
        # one adapted layer of a training batch, its input kept in 8 bits
        dict(name="layer8_8192", op="checkpoint", mode="layer", rows=8192, k=4096, n=11008, rank=16, count=1, skew=1,
             dtype="bf16"),
        # the same with odd sizes, two adapters and the larger rank
        dict(name="layer8_1111", op="checkpoint", mode="layer", rows=1111, k=1093, n=1088, rank=64, count=2, skew=2,
             dtype="f16"),
        # one pair of short answers
        dict(name="pair_64", op="preference", pairs=1, length=64, prompt=17, vocab=32000, smooth=0.0, form="sigmoid",
             dtype="bf16"),
        # a usual micro-batch: prompts do not count
        dict(name="pairs_1024", op="preference", pairs=2, length=1024, prompt=300, vocab=32000, smooth=0.1,
             form="sigmoid", dtype="bf16"),
        # a large batch
        dict(name="pairs_2048", op="preference", pairs=4, length=2048, prompt=200, vocab=32000, smooth=0.0,
             form="sigmoid", dtype="bf16"),
        # a large vocabulary of odd size, 32-bit logits, answers averaged over their length
        dict(name="pairs_vocab", op="preference", pairs=2, length=301, prompt=40, vocab=131073, smooth=0.0, form="ipo",
             dtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adapters", "adapters", "checkpoint", "checkpoint", "preference", "preference"])
    wide = [1024, 1088, 2048, 4096, 8192, 11008]
    size = lambda: rng.choice(wide) if rng.random() < 0.6 else _log(rng, 65, 11008)  # noqa: E731
    if op == "adapters":
        mode = rng.choice(["apply", "apply", "train"])
        rank = rng.choice([8, 16, 16, 32, 64, 128])
        return dict(op=op, mode=mode, rows=_log(rng, 1, 8192), k=size(), n=size(), rank=rank,
                    count=min(_log(rng, 1, 64), 2048 // rank), skew=rng.randint(1, 4), dtype=rng.choice(["bf16", "f16"]))
    if op == "checkpoint":
        if rng.random() < 0.5:
            dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
            return dict(op=op, mode="swiglu", rows=_log(rng, 1, 4096 if dtype == "f32" else 8192), k=size(), dtype=dtype)
        return dict(op=op, mode="layer", rows=_log(rng, 1, 8192), k=size(), n=size(), rank=rng.choice([8, 16, 32, 64]),
                    count=rng.randint(1, 4), skew=rng.randint(1, 4), dtype=rng.choice(["bf16", "f16"]))
    pairs, vocab = rng.randint(1, 4), rng.choice([32000, 32001, _log(rng, 1000, 131073), _log(rng, 1000, 131073)])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    most = min(2048, int(1.0e9 / (2 * pairs * vocab * _SIZE[dtype])))
    length = _log(rng, 2, max(3, most))
    return dict(op=op, pairs=pairs, length=length, prompt=rng.randint(0, length // 2), vocab=vocab,
                smooth=rng.choice([0.0, 0.1]), form=rng.choice(["sigmoid", "sigmoid", "ipo"]), dtype=dtype)


def _answers(c):
    """(first, last) label position of each sequence that counts: the prompt
    before and the padding after do not.  Lengths differ between sequences."""
    found = []
    for b in range(2 * c["pairs"]):
        first = min(c["length"], max(1, c["prompt"]))
        room = c["length"] - first
        found.append((first, c["length"] - (room * ((3 * b) % 7)) // 14))
    return found


def work(c):
    e = _SIZE[c["dtype"]]
    if c["op"] == "preference":
        counted = sum(last - first for first, last in _answers(c))
        every = 2 * c["pairs"] * c["length"]
        # the logits that count read once, the gradient written once, labels read
        return {"bytes": (counted + every) * c["vocab"] * e + 8 * every, "flops": 9 * counted * c["vocab"]}
    if c["mode"] == "swiglu":
        m, k = c["rows"], c["k"]
        blocks = m * -(-k // BLOCK)
        # forward: gate and up read, the product and the packed copies written (a 16-bit product's too, for the
        # projection after it); backward: the product's gradient and two packed copies read, two gradients written
        copies = 2 if c["dtype"] == "f32" else 3
        return {"bytes": m * k * (3 * e + copies) + 4 * copies * blocks + m * k * (3 * e + 2) + 8 * blocks,
                "flops": 40 * m * k}
    m, k, n, r, used = c["rows"], c["k"], c["n"], c["rank"], min(c["rows"], c["count"])
    weights = used * r * (k + n) * e
    moved = {"bytes": m * (k + 2 * n) * e + weights + 4 * m, "flops": 2 * m * r * (k + n)}
    if c["mode"] == "apply":
        return moved
    moved["flops"] += 4 * m * r * (k + n)
    if c["mode"] == "train":
        # backward: dy and x read, dx and the adapters' gradients written
        moved["bytes"] += m * (n + 2 * k) * e + weights + c["count"] * r * (k + n) * e
    else:
        # forward also writes x's packed copy; backward reads it in x's place
        moved["bytes"] += m * k + 4 * m * -(-k // BLOCK)
        moved["bytes"] += m * n * e + m * k * (1 + e) + 4 * m * -(-k // BLOCK) + weights + c["count"] * r * (k + n) * e
    return moved


# ------------------------------------------------------------------ inputs

def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


def _draws(c, seed):
    """The inputs of a case, from the seed alone."""
    dev, dt = _device(), _DT[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    if c["op"] == "preference":
        b, length, v = 2 * c["pairs"], c["length"], c["vocab"]
        labels = torch.randint(0, v, (b, length), generator=g, device=dev)
        logits = torch.empty(b, length, v, dtype=dt, device=dev)
        ref = torch.zeros(b, length, device=dev)
        for i, (first, last) in enumerate(_answers(c)):
            x = normal(length, v).mul_(2.0)
            # a trained model gives the next token a good score most of the time
            lift = 9.0 + 4.0 * normal(length - 1, 1)
            x[:-1].scatter_add_(1, labels[i, 1:, None], lift)
            logits[i] = x
            labels[i, :first] = IGNORE
            labels[i, last:] = IGNORE
            if last > first:
                y = logits[i, first - 1:last - 1].float()
                at = y.gather(1, labels[i, first:last, None])[:, 0] - y.logsumexp(-1)
                # the reference model is near the policy, which has moved toward the chosen answers
                moved = (4.0 + 4.0 * torch.rand(1, generator=g, device=dev)) * (1 if i < c["pairs"] else -1)
                ref[i, first:last] = at - moved / (last - first) + 0.05 * normal(last - first)
        return dict(logits=logits, labels=labels, ref=ref)
    m, k = c["rows"], c["k"]
    if c["mode"] == "swiglu":
        # the two halves of one projection's output; a few features are larger than the rest
        both = normal(m, 2 * k)
        both[:, :: max(1, k // 5)] *= 2.5
        both = both.to(dt)
        return dict(gate=both[:, :k], up=both[:, k:], dh=normal(m, k).mul_(0.1).to(dt))
    n, r, a = c["n"], c["rank"], c["count"]
    x = normal(m, k)
    x[:, :: max(1, k // 7)] *= 6.0
    # requests share adapters unevenly, and about one row in nine has none
    ids = (torch.rand(m, generator=g, device=dev) ** c["skew"] * a).long().clamp_(max=a - 1)
    if a > 1:
        ids = torch.where(torch.rand(m, generator=g, device=dev) < 0.11, torch.full_like(ids, -1), ids)
    if m > 64:  # tokens of a request come together; a decode step has one of each request
        ids = ids.sort(stable=True).values
    s = dict(x=x.to(dt), ids=ids, base=normal(m, n).to(dt),
             A=(normal(a, k, r) / math.sqrt(k)).to(dt), B=normal(a, n, r).mul_(0.3).to(dt),
             scaling=0.5 + torch.rand(a, generator=g, device=dev))
    if c["mode"] != "apply":
        s["dy"] = normal(m, n).mul_(0.1).to(dt)
    return s


def prepare(case, seed):
    s = _draws(case, seed)
    s["case"] = case
    if own:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocm-qlora_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        if case["op"] == "preference":
            s["logits"].requires_grad_()
        elif case["mode"] == "swiglu":
            s["gate"].requires_grad_(), s["up"].requires_grad_()
        else:
            from rocm_qlora.lora import AdapterPlan
            # which rows use which adapter: known once a batch, used by every layer
            s["plan"] = AdapterPlan(s["ids"], case["count"])
            if case["mode"] != "apply":
                for name in ("x", "A", "B"):
                    s[name].requires_grad_()
    return s


# --------------------------------------------------------------------- run

def run(s):
    c = s["case"]
    if c["op"] == "preference":
        return _own_preference(s) if own else _plain_preference(s)
    if c["mode"] == "swiglu":
        return _own_swiglu(s) if own else _plain_swiglu(s)
    return _own_adapters(s) if own else _plain_adapters(s)


def _own_adapters(s):
    from rocm_qlora.activation8 import pack_activation
    from rocm_qlora.lora import adapters_add
    c = s["case"]
    if c["mode"] == "apply":
        return [adapters_add(s["base"], s["x"], s["A"], s["B"], s["scaling"], s["plan"])]
    packed = pack_activation(s["x"]) if c["mode"] == "layer" else None
    y = adapters_add(s["base"], s["x"], s["A"], s["B"], s["scaling"], s["plan"], packed_x=packed)
    return [y, *torch.autograd.grad(y, (s["x"], s["A"], s["B"]), s["dy"])]


def _own_swiglu(s):
    from rocm_qlora.activation8 import swiglu8, unpack_activation
    if s["case"]["dtype"] == "f32":
        h, kept = swiglu8(s["gate"], s["up"]), None
    else:
        h, packed = swiglu8(s["gate"], s["up"], pack_output=True)
        kept = unpack_activation(packed)
    dgate, dup = torch.autograd.grad(h, (s["gate"], s["up"]), s["dh"])
    return [h, kept, dgate, dup]


def _own_preference(s):
    from rocm_qlora.preference import preference_loss
    c = s["case"]
    out = preference_loss(s["logits"], s["labels"], s["ref"], beta=BETA, label_smoothing=c["smooth"], form=c["form"])
    dlogits, = torch.autograd.grad(out.loss, s["logits"])
    return [out.loss, out.logps, out.chosen_rewards, out.rejected_rewards, dlogits]


def _kept8(x):
    """The values that 8-bit codes of x stand for (32 bits): blocks of BLOCK
    values of a row, code = round(x * (127 / max|x|)), scale = max|x| / 127."""
    m, k = x.shape
    pad = -k % BLOCK
    blocks = torch.nn.functional.pad(x, (0, pad)).view(m, -1, BLOCK)
    top = blocks.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, 127.0)
    codes = torch.where(top < FLUSH, 0.0, torch.round(blocks * most.div(top.clamp(min=FLUSH))))
    scale = torch.where(top < FLUSH, 0.0, top.div(most))
    return (codes * scale).view(m, -1)[:, :k]


def _plain_adapters(s):
    """All adapters' products, of which each row keeps its own's."""
    c, dt = s["case"], s["x"].dtype
    a, r = c["count"], c["rank"]
    x = s["x"].float()
    A = s["A"].float().transpose(0, 1).reshape(c["k"], a * r)
    B = s["B"].float().transpose(0, 1).reshape(c["n"], a * r)
    mine = (s["ids"][:, None] == torch.arange(a, device=x.device)) * s["scaling"]
    mine = mine[:, :, None].expand(-1, -1, r).reshape(-1, a * r)
    t = (x @ A) * mine
    y = (s["base"].float() + t @ B.t()).to(dt)
    if c["mode"] == "apply":
        return [y]
    dy = s["dy"].float()
    gt = (dy @ B) * mine
    kept = _kept8(x) if c["mode"] == "layer" else x
    dx = (gt @ A.t()).to(dt)
    dA = (kept.t() @ gt).view(c["k"], a, r).transpose(0, 1).to(dt)
    dB = (dy.t() @ t).view(c["n"], a, r).transpose(0, 1).to(dt)
    return [y, dx, dA, dB]


def _plain_swiglu(s):
    g, u, dh, dt = s["gate"].float(), s["up"].float(), s["dh"].float(), s["gate"].dtype
    h = (g / (1.0 + torch.exp(-g)) * u).to(dt)
    kept = _kept8(h.float()).to(dt) if dt != torch.float32 else None
    g, u = _kept8(g), _kept8(u)
    p = 1.0 / (1.0 + torch.exp(-g))
    return [h, kept, (dh * u * p * (1.0 + g * (1.0 - p))).to(dt), (dh * g * p).to(dt)]


def _plain_preference(s):
    c, logits, labels = s["case"], s["logits"], s["labels"]
    p = c["pairs"]
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    # position l is scored on the token after it
    target = torch.nn.functional.pad(labels[:, 1:], (0, 1), value=IGNORE)
    counts = target != IGNORE
    at = target.clamp(min=0)[:, :, None]
    logp = (x.gather(-1, at) - top - torch.log(total))[:, :, 0]
    logps = torch.where(counts, logp, 0.0).sum(-1)
    length = counts.sum(-1).clamp(min=1)
    ref = torch.nn.functional.pad(s["ref"][:, 1:], (0, 1))
    ratio = torch.where(counts, logp - ref, 0.0).sum(-1)
    rewards = BETA * ratio
    if c["form"] == "ipo":
        d = ratio / length
        off = d[:p] - d[p:] - 1.0 / (2.0 * BETA)
        loss = (off * off).mean()
        slope = 2.0 * off / p
        each = torch.cat([slope, -slope]) / length
    else:
        z = rewards[:p] - rewards[p:]
        w = c["smooth"]
        soft = torch.log1p(torch.exp(-z.abs()))
        loss = ((1.0 - w) * (soft + (-z).clamp(min=0)) + w * (soft + z.clamp(min=0))).mean()
        slope = BETA * (1.0 / (1.0 + torch.exp(-z)) - (1.0 - w)) / p
        each = torch.cat([slope, -slope])
    each = torch.where(counts, each[:, None], 0.0)[:, :, None]
    d = e.mul_(-each / total).scatter_add_(-1, at, each)
    return [loss, logps, rewards[:p], rewards[p:], d.to(logits.dtype)]


# ------------------------------------------------------------------- exact

def _kept8_64(x):
    """_kept8 by its definition: codes and scales as the format holds them
    (32-bit scale and reciprocal, the product rounded to the nearest whole)."""
    m, k = x.shape
    out = torch.zeros(m, k, dtype=torch.float64, device=x.device)
    for at in range(0, k, BLOCK):
        part = x[:, at:at + BLOCK].double()
        top = part.abs().max(1).values
        live = top >= FLUSH
        by = torch.where(live, torch.full_like(top, 127.0) / top, 0.0).float().double()
        code = (part * by[:, None]).float().double().round()
        out[:, at:at + BLOCK] = code * torch.where(live, top / torch.full_like(top, 127.0), 0.0).float().double()[:, None]
    return out


def exact(case, seed):
    c, s = case, _draws(case, seed)
    f8 = torch.float64
    if c["op"] == "preference":
        p, ans = c["pairs"], _answers(c)
        logits = s["logits"]
        sums, keep = [], []
        for i, (first, last) in enumerate(ans):
            y = logits[i, first - 1:last - 1].to(f8) if last > first else logits[i, :0].to(f8)
            lp = torch.log_softmax(y, -1)
            sums.append(lp.gather(1, s["labels"][i, first:last, None]).sum())
            keep.append(lp.exp_())
        ref = torch.stack([s["ref"][i, first:last].to(f8).sum() for i, (first, last) in enumerate(ans)])
        logps = torch.stack(sums)
        d = torch.zeros(logits.shape, dtype=f8, device=logits.device)
        loss, slopes = 0.0, [None] * (2 * p)
        for j in range(p):
            n1, n2 = (max(1, ans[i][1] - ans[i][0]) for i in (j, p + j))
            if c["form"] == "ipo":
                off = (logps[j] - ref[j]) / n1 - (logps[p + j] - ref[p + j]) / n2 - 0.5 / BETA
                loss = loss + off ** 2 / p
                slopes[j], slopes[p + j] = 2 * off / (p * n1), -2 * off / (p * n2)
            else:
                z = BETA * (logps[j] - ref[j] - logps[p + j] + ref[p + j])
                w = c["smooth"]
                loss = loss - ((1 - w) * torch.nn.functional.logsigmoid(z) + w * torch.nn.functional.logsigmoid(-z)) / p
                slope = BETA * (w * torch.sigmoid(z) - (1 - w) * torch.sigmoid(-z)) / p
                slopes[j], slopes[p + j] = slope, -slope
        for i, (first, last) in enumerate(ans):
            if last > first:
                q = keep[i].neg_()
                q.scatter_add_(1, s["labels"][i, first:last, None], torch.ones_like(q[:, :1]))
                d[i, first - 1:last - 1] = q * slopes[i]
        rewards = BETA * (logps - ref)
        return [loss, logps, rewards[:p], rewards[p:], d]
    if c["mode"] == "swiglu":
        g, u, dh = s["gate"].to(f8), s["up"].to(f8), s["dh"].to(f8)
        h = torch.nn.functional.silu(g) * u
        g, u = _kept8_64(s["gate"]), _kept8_64(s["up"])
        q = torch.sigmoid(g)
        # the packed copy is of the rounded product: it has no value of its own in 64 bits
        return [h, None, dh * u * (q + g * q * (1 - q)), dh * g * q]
    y = s["base"].to(f8)
    x = s["x"].to(f8)
    full = c["mode"] != "apply"
    kept = _kept8_64(s["x"]) if c["mode"] == "layer" else x
    dx, dA, dB = torch.zeros_like(x), torch.zeros_like(s["A"], dtype=f8), torch.zeros_like(s["B"], dtype=f8)
    for a in range(c["count"]):
        at = (s["ids"] == a).nonzero()[:, 0]
        if not len(at):
            continue
        A, B, w = s["A"][a].to(f8), s["B"][a].to(f8), s["scaling"][a].to(f8)
        t = w * (x[at] @ A)
        y[at] += t @ B.t()
        if full:
            dy = s["dy"][at].to(f8)
            gt = w * (dy @ B)
            dx[at] = gt @ A.t()
            dA[a] = kept[at].t() @ gt
            dB[a] = dy.t() @ t
    return [y, dx, dA, dB] if full else [y]

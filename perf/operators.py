"""Cases of the operators over large item vocabularies: table lookups with their gradient, losses on whole rows of logits, and
scores from an 8-bit item table.  `run` computes a case in plain torch, or with `own` set by the library's operators."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BETA, SMOOTHING, TEMPERATURE = 0.1, 0.05, 2.0


def _lib():
    import recbole_gnn_amd
    return recbole_gnn_amd


def listed():
    return [
        # one answering step of 32 users: a few rows of a 16-bit item table (Gowalla's item count); latency counts
        {"name": "embed-step", "op": "embed", "dtype": "bf16", "train": False, "n": 32, "rows": 40982, "d": 64},
        # the ids of one training batch (users, positives, negatives of 2 048 triples) against a Gowalla-sized table
        {"name": "embed-batch", "op": "embed", "dtype": "f32", "train": True, "n": 6144, "rows": 40982, "d": 64},
        # a long packed batch of item sequences with wide rows
        {"name": "embed-long", "op": "embed", "dtype": "bf16", "train": True, "n": 65536, "rows": 131072, "d": 1024},
        # a small student on an ml-100k-sized catalogue
        {"name": "distill-small", "op": "distill", "dtype": "f32", "train": True, "n": 64, "vocab": 1683, "k": 10},
        # one training step: 2 048 users' logits over Gowalla's items against a teacher's 32 best
        {"name": "distill-step", "op": "distill", "dtype": "bf16", "train": True, "n": 2048, "vocab": 40982, "k": 32},
        # validation of a student over Amazon-Book's items: the loss alone
        {"name": "distill-eval", "op": "distill", "dtype": "f32", "train": False, "n": 4096, "vocab": 91600, "k": 20},
        # four pairs of short sessions on an ml-100k-sized catalogue
        {"name": "prefer-small", "op": "prefer", "dtype": "f32", "pairs": 4, "tokens": 40, "vocab": 1683},
        # 32 pairs of sessions over Gowalla's items
        {"name": "prefer-step", "op": "prefer", "dtype": "bf16", "pairs": 32, "tokens": 4096, "vocab": 40982},
        # two pairs of long sequences over a large vocabulary
        {"name": "prefer-long", "op": "prefer", "dtype": "f16", "pairs": 2, "tokens": 6001, "vocab": 131072},
        # one user's scores of Gowalla's items: the table is read once
        {"name": "int8-user", "op": "int8", "dtype": "f32", "out": "f32", "b": 1, "n": 40982, "k": 128},
        # full-sort scores of an evaluation batch at the engine's usual width
        {"name": "int8-batch", "op": "int8", "dtype": "f32", "out": "f32", "b": 4096, "n": 40982, "k": 64},
        # a wide head: 4 096 tokens against 16 384 channels
        {"name": "int8-wide", "op": "int8", "dtype": "bf16", "out": "bf16", "b": 4096, "n": 16384, "k": 8192},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "distill", "prefer", "int8"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "embed":
        rows, d = _log(rng, 2, 131072), _log(rng, 1, 1024)
        return {"op": op, "dtype": dtype, "train": rng.random() < 0.75, "n": _log(rng, 1, 65536), "rows": rows, "d": d}
    if op == "distill":
        vocab = _log(rng, 2, 131072)
        n = _log(rng, 1, min(4096, max(1, 180_000_000 // vocab)))
        return {"op": op, "dtype": dtype, "train": rng.random() < 0.75, "n": n, "vocab": vocab, "k": rng.randint(1, min(64, vocab))}
    if op == "prefer":
        vocab = _log(rng, 2, 131072)
        return {"op": op, "dtype": dtype, "pairs": _log(rng, 1, 64), "tokens": _log(rng, 1, min(8192, max(1, 360_000_000 // vocab))),
                "vocab": vocab}
    b, k = _log(rng, 1, 4096), _log(rng, 1, 8192)
    return {"op": op, "dtype": dtype, "out": rng.choice(["f32", "bf16"]), "b": b, "n": _log(rng, 1, min(131072, 160_000_000 // b)), "k": k}


def _ids(n, rows, g, dev):
    """Item ids as they come: a few items take most of the occurrences; row 0 is the padding item, and some places hold no id."""
    u = torch.rand(n, generator=g, device=dev, dtype=torch.float64)
    ids = (rows * u * u * u).long().clamp_(0, rows - 1)
    ids = (ids * 7919) % rows
    ids[torch.rand(n, generator=g, device=dev) < 0.02] = -1
    return ids


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).mul_(scale).to(dt)

    op, s = case["op"], dict(case)
    if op == "embed":
        s["table"] = normal(case["rows"], case["d"], scale=0.1)
        s["ids"] = _ids(case["n"], case["rows"], g, dev)
        s["scale"] = math.sqrt(case["d"])
        if case["train"]:
            s["grad"] = normal(case["n"], case["d"])
    elif op == "distill":
        n, v, k = case["n"], case["vocab"], case["k"]
        s["logits"] = normal(n, v, scale=2.0)
        s["idx"] = torch.randint(v, (n, k), generator=g, device=dev)
        s["val"] = torch.randn(n, k, generator=g, device=dev).mul_(2.0).add_(4.0).sort(dim=1, descending=True).values
        # lists that ended early, as a top-k of few candidates leaves them
        left = torch.randint(1, 4 * k + 1, (n, 1), generator=g, device=dev)
        none = torch.arange(k, device=dev)[None, :] >= left
        s["idx"][none], s["val"][none] = -1, -math.inf
        s["weight"] = torch.full((n,), 1.0 / n, device=dev)
    elif op == "prefer":
        m, v, p = case["tokens"], case["vocab"], case["pairs"]
        r = random.Random(seed)
        cuts = sorted(r.randint(0, m) for _ in range(2 * p - 1))
        s["offsets"] = torch.tensor([0] + cuts + [m], device=dev)
        s["logits"] = normal(m, v, scale=2.0)
        s["targets"] = torch.randint(v, (m,), generator=g, device=dev)
        s["targets"][torch.rand(m, generator=g, device=dev) < 0.25] = -1  # the prompts' tokens
        seqs = (s["offsets"][1:] - s["offsets"][:-1]).double()
        s["ref"] = (-(math.log(v) + 2.0) * 0.75 * seqs + 3.0 * torch.randn(2 * p, generator=g, device=dev).double()).float()
    else:
        b, n, k = case["b"], case["n"], case["k"]
        s["u"] = normal(b, k)
        items = torch.randn(n, k, generator=g, device=dev)
        ld = (k + 63) // 64 * 64
        scale = (items.abs().amax(dim=1).double() / 127.0).float()
        codes = torch.zeros(n, ld, dtype=torch.int8, device=dev)
        codes[:, :k] = (items / scale[:, None]).round_().clamp_(-127, 127).to(torch.int8)
        s["codes"], s["scales"] = codes[:, :k], scale
    return s


def run(s):
    op = s["op"]
    if op == "embed":
        return _embed_own(s) if own else _embed(s)
    if op == "distill":
        return _distill_own(s) if own else _distill(s)
    if op == "prefer":
        return _prefer_own(s) if own else _prefer(s)
    return _int8_own(s) if own else _int8(s)


def _embed_own(s):
    rbg = _lib()
    out = rbg.embedding(s["table"], s["ids"], scale=s["scale"], padding_idx=0)
    if not s["train"]:
        return {"out": out}
    return {"out": out, "grad": rbg.embedding_grad(s["grad"], s["ids"], s["rows"], scale=s["scale"], padding_idx=0)}


def _embed(s):
    ids, table = s["ids"], s["table"]
    there = (ids >= 0)[:, None]
    out = {"out": (table[ids.clamp(min=0)].float() * s["scale"] * there).to(table.dtype)}
    if s["train"]:
        g = s["grad"].float() * s["scale"] * (there & (ids != 0)[:, None])
        out["grad"] = torch.zeros(s["rows"], s["d"], device=g.device).index_add_(0, ids.clamp(min=0), g).to(table.dtype)
    return out


def _distill_own(s):
    rbg = _lib()
    if not s["train"]:
        return {"loss": rbg.distill_topk(s["logits"], s["idx"], s["val"], temperature=TEMPERATURE)}
    loss, grad = rbg.distill_topk_grad(s["logits"], s["idx"], s["val"], temperature=TEMPERATURE, row_weight=s["weight"])
    return {"loss": loss, "grad": grad}


def _distill(s):
    t = TEMPERATURE
    z = s["logits"].float() / t
    z -= z.amax(dim=1, keepdim=True)
    there = s["idx"] >= 0
    idx = s["idx"].clamp(min=0)
    e = z.exp()
    total = e.sum(dim=1, keepdim=True)
    logq = z.gather(1, idx) - total.log()
    v = torch.where(there, s["val"] / t, -math.inf)
    logp = v - v.amax(dim=1, keepdim=True)
    logp = logp - logp.exp().sum(dim=1, keepdim=True).log()
    p = logp.exp()
    loss = t * t * torch.where(there, p * (logp - logq), 0.0).sum(dim=1)
    if not s["train"]:
        return {"loss": loss}
    q = e.div_(total)
    q.scatter_add_(1, idx, -p)
    return {"loss": loss, "grad": q.mul_(t * s["weight"][:, None]).to(s["logits"].dtype)}


def _prefer_own(s):
    loss, margin, grad = _lib().preference_grad(s["logits"], s["targets"], s["offsets"], s["ref"], beta=BETA, label_smoothing=SMOOTHING)
    return {"loss": loss, "margin": margin, "grad": grad}


def _prefer(s):
    y, offsets = s["targets"], s["offsets"]
    m, seqs = y.shape[0], offsets.shape[0] - 1
    z = s["logits"].float()
    e = z - z.amax(dim=1, keepdim=True)
    at = torch.arange(m, device=y.device)
    there, yc = y >= 0, y.clamp(min=0)
    zt = e[at, yc]
    e.exp_()
    total = e.sum(dim=1)
    logp = torch.where(there, zt - total.log(), 0.0)
    seq = torch.bucketize(at, offsets[1:], right=True)
    sums = torch.zeros(seqs, dtype=torch.float64, device=y.device).index_add_(0, seq, logp.double()) - s["ref"].double()
    h = BETA * (sums[0::2] - sums[1::2])
    loss = (1.0 - SMOOTHING) * torch.log1p(torch.exp(-h.abs())) + SMOOTHING * torch.log1p(torch.exp(-h.abs()))
    loss = loss + (1.0 - SMOOTHING) * (-h).clamp(min=0) + SMOOTHING * h.clamp(min=0)
    dh = SMOOTHING / (1.0 + torch.exp(-h)) - (1.0 - SMOOTHING) / (1.0 + torch.exp(h))
    coef = torch.stack([BETA * dh, -BETA * dh], dim=1).reshape(-1)[seq].float() * there
    e.mul_((-coef / total)[:, None])
    e[at, yc] += coef
    return {"loss": loss.float(), "margin": h.float(), "grad": e.to(s["logits"].dtype)}


def _int8_own(s):
    return _lib().score_int8(s["u"], s["codes"], s["scales"], out_dtype=DTYPES[s["out"]])


def _int8(s):
    u = s["u"].float()
    su = (u.abs().amax(dim=1).double() / 127.0).float()
    q = (u.double() / su.double()[:, None]).float().round_().clamp_(-127, 127)
    out = q @ s["codes"].float().t()
    return out.mul_(su[:, None]).mul_(s["scales"][None, :]).to(DTYPES[s["out"]])


def work(case):
    op, size = case["op"], SIZE[case["dtype"]]
    if op == "embed":
        n, d = case["n"], case["d"]
        moved = 8 * n + size * d * (min(n, case["rows"]) + n)
        if case["train"]:
            moved += size * d * (n + case["rows"])
        return {"bytes": moved, "flops": n * d * (2 if case["train"] else 1)}
    if op == "distill":
        cells = case["n"] * case["vocab"]
        return {"bytes": cells * size * (2 if case["train"] else 1) + 12 * case["n"] * case["k"], "flops": cells * (6 if case["train"] else 4)}
    if op == "prefer":
        cells = case["tokens"] * case["vocab"]
        return {"bytes": 2 * cells * size + 8 * case["tokens"], "flops": 6 * cells}
    b, n, k = case["b"], case["n"], case["k"]
    return {"bytes": b * k * size + n * k + 4 * n + b * n * SIZE[case["out"]], "flops": 2 * b * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _embed64, "distill": _distill64, "prefer": _prefer64, "int8": _int864}[case["op"]](s)


def _embed64(s):
    ids, v = s["ids"], s["rows"]
    padded = torch.cat([s["table"].double(), s["table"].new_zeros(1, s["d"]).double()])
    out = {"out": padded[torch.where(ids < 0, v, ids)] * s["scale"]}
    if s["train"]:
        total = torch.zeros(v + 1, s["d"], dtype=torch.float64, device=ids.device)
        total.index_add_(0, torch.where(ids <= 0, v, ids), s["grad"].double())
        out["grad"] = total[:v] * s["scale"]
    return out


def _distill64(s):
    t, w = TEMPERATURE, s["weight"].double()
    losses, grads = [], []
    for lo in range(0, s["n"], 256):
        z = s["logits"][lo:lo + 256].double() / t
        idx, val = s["idx"][lo:lo + 256], s["val"][lo:lo + 256].double()
        there = idx >= 0
        p = torch.softmax(torch.where(there, val / t, -math.inf), dim=1)
        logq = torch.log_softmax(z, dim=1)
        at = torch.where(there, idx, 0)
        terms = torch.xlogy(p, p) - p * logq.gather(1, at)
        losses.append(t * t * torch.where(there, terms, 0.0).sum(dim=1))
        if s["train"]:
            grad = logq.exp()
            grad.scatter_add_(1, at, -p)
            grads.append((grad * (t * w[lo:lo + 256, None])).float() if s["dtype"] != "f32" else grad * (t * w[lo:lo + 256, None]))
    out = {"loss": torch.cat(losses)}
    if s["train"]:
        out["grad"] = torch.cat(grads)
    return out


def _prefer64(s):
    y, offsets, m = s["targets"], s["offsets"].tolist(), s["tokens"]
    logp = torch.zeros(m, dtype=torch.float64, device=y.device)
    for lo in range(0, m, 256):
        z = torch.log_softmax(s["logits"][lo:lo + 256].double(), dim=1)
        yy = y[lo:lo + 256]
        logp[lo:lo + 256] = torch.where(yy >= 0, z.gather(1, yy.clamp(min=0)[:, None])[:, 0], 0.0)
    sums = torch.stack([logp[a:b].sum() for a, b in zip(offsets[:-1], offsets[1:])]) - s["ref"].double()
    h = (BETA * (sums[0::2] - sums[1::2])).requires_grad_()
    with torch.enable_grad():
        loss = -(1.0 - SMOOTHING) * torch.nn.functional.logsigmoid(h) - SMOOTHING * torch.nn.functional.logsigmoid(-h)
        (dh,) = torch.autograd.grad(loss.sum(), h)
    coef = torch.zeros(m, dtype=torch.float64, device=y.device)
    for i, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        coef[a:b] = (BETA if i % 2 == 0 else -BETA) * dh[i // 2]
    coef = torch.where(y >= 0, coef, 0.0)
    grads = []
    for lo in range(0, m, 256):
        grad = torch.softmax(s["logits"][lo:lo + 256].double(), dim=1).neg_()
        grad[torch.arange(grad.shape[0], device=y.device), y[lo:lo + 256].clamp(min=0)] += 1.0
        grad *= coef[lo:lo + 256, None]
        grads.append(grad if s["dtype"] == "f32" else grad.float())
    return {"loss": loss.detach(), "margin": h.detach(), "grad": torch.cat(grads)}


def _int864(s):
    # the codes are defined in 32 bits (a scale of one 127th, a quotient, its nearest whole number); the products are exact in 64
    u = s["u"].double()
    su = (u.abs().amax(dim=1) / 127.0).float().double()
    q = torch.clamp(torch.round((u / su[:, None]).float().double()), -127.0, 127.0)
    return torch.matmul(q, s["codes"].double().t().contiguous()) * (su[:, None] * s["scales"].double()[None, :])

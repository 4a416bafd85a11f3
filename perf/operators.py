"""The vocabulary operators as work to be measured: embedding rows and their gradient, softmax cross entropy over a large
vocabulary with its gradients, distillation from a teacher's top logits with its gradients.

`own = False`: plain torch operations in 32 bits, rounded once at the end.  `own = True`: the calls a user makes of
`gossipnet_amd.vocab`.  `exact` is the definition in 64 bits."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST_FLOPS = 6 * 4096 * 131072 * 4096        # the largest listed case
MOST_FLOPS_F32 = 6 * 1500 * 32001 * 1024     # fp32 stands for smaller heads


def listed():
    return [
        # one step of answering: a handful of token rows fetched from a large table
        {"name": "embed_single_tokens", "op": "embed_forward", "M": 7, "V": 128000, "D": 4096, "dtype": "bf16", "scaled": False, "padding": 0.0},
        # a training batch's rows, weighted per token
        {"name": "embed_batch", "op": "embed_forward", "M": 16384, "V": 50257, "D": 1024, "dtype": "bf16", "scaled": True, "padding": 0.05},
        # detections' class rows scaled by their scores (2000 detections, 80 classes and background, 128 features): table and score gradients
        {"name": "embed_grad_classes", "op": "embed_backward", "M": 2000, "V": 81, "D": 128, "dtype": "f32", "scaled": True, "padding": 0.0},
        # the gradient of a large table from a long batch with padding
        {"name": "embed_grad_batch", "op": "embed_backward", "M": 32768, "V": 128000, "D": 2048, "dtype": "bf16", "scaled": False, "padding": 0.1},
        # detections classified from the network's 128 features, a training step
        {"name": "xent_classes", "op": "xent", "train": True, "M": 2000, "V": 81, "D": 128, "dtype": "f32", "padding": 0.1},
        # the score of one token: the weights are read once
        {"name": "xent_single_token", "op": "xent", "train": False, "M": 1, "V": 128000, "D": 4096, "dtype": "bf16", "padding": 0.0},
        # a small training batch with an odd vocabulary, padded rows
        {"name": "xent_ragged", "op": "xent", "train": True, "M": 1111, "V": 50257, "D": 1024, "dtype": "bf16", "padding": 0.25},
        # fp32 weights and features, odd sizes
        {"name": "xent_f32", "op": "xent", "train": True, "M": 777, "V": 32001, "D": 768, "dtype": "f32", "padding": 0.05},
        # a full training step's head
        {"name": "xent_large", "op": "xent", "train": True, "M": 4096, "V": 131072, "D": 4096, "dtype": "bf16", "padding": 0.0},
        # a few rows against a teacher's eight best
        {"name": "distill_few_rows", "op": "distill", "train": True, "M": 48, "K": 8, "V": 32000, "D": 2048, "dtype": "f16", "tau": 2.0, "padding": 0.1},
        # how far a student is from its teacher, without gradients
        {"name": "distill_score", "op": "distill", "train": False, "M": 515, "K": 32, "V": 65537, "D": 1536, "dtype": "bf16", "tau": 1.0, "padding": 0.1},
        # a training step of distillation
        {"name": "distill_large", "op": "distill", "train": True, "M": 2048, "K": 64, "V": 100352, "D": 2048, "dtype": "bf16", "tau": 1.5, "padding": 0.1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    d = _log(rng, 64, 4096)
    kind = rng.random()
    return max(64, d // 64 * 64) if kind < 0.6 else max(64, d // 8 * 8) if kind < 0.85 else d


def draw(rng):
    op = rng.choice(["embed_forward", "embed_backward", "xent", "xent", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    V, D = _log(rng, 81, 131072), _width(rng)
    padding = rng.choice([0.0, 0.05, 0.3])
    if op.startswith("embed"):
        return {"op": op, "M": _log(rng, 1, 32768), "V": V, "D": D, "dtype": dtype, "scaled": rng.random() < 0.5, "padding": padding}
    case = {"op": op, "train": rng.random() < 0.7, "M": _log(rng, 1, 4096), "V": V, "D": D, "dtype": dtype, "padding": padding}
    if op == "distill":
        case["K"] = min(_log(rng, 1, 128), V)
        case["tau"] = rng.choice([1.0, 1.5, 2.0, 4.0])
    most = MOST_FLOPS_F32 if dtype == "f32" else MOST_FLOPS
    while 6 * case["M"] * V * D > most:
        case["M"] = max(1, case["M"] // 2 + 1)
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _zipf(n, V, g):
    """Token ids as text has them: frequency about 1 / rank, spread over the table."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    rank = torch.exp(u * math.log(V)).long().clamp_(1, V) - 1
    return (rank * 7919 + 13) % V


def _drop(n, share, g):
    """Exactly round(n * share) positions, at random."""
    return torch.randperm(n, device="cuda", generator=g)[:int(round(n * share))]


def prepare(case, seed):
    g = _generator(seed)
    M, V, D, t = case["M"], case["V"], case["D"], DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"].startswith("embed"):
        s["ids"] = _zipf(M, V, g)
        s["ids"][_drop(M, case["padding"], g)] = -1
        s["table"] = torch.randn(V, D, device="cuda", generator=g).to(t)
        s["token_scale"] = torch.rand(M, device="cuda", generator=g) if case["scaled"] else None
        s["scale"] = float(D) ** 0.5
        if case["op"] == "embed_backward":
            s["dy"] = (torch.randn(M, D, device="cuda", generator=g) / M).to(t)
        return s
    s["w"] = torch.randn(V, D, device="cuda", generator=g).mul_(1.5 * D ** -0.5).to(t)
    x = torch.randn(M, D, device="cuda", generator=g)
    if case["op"] == "xent":
        labels = _zipf(M, V, g)
        x += 4.0 * s["w"][labels].float()            # the row leans towards its label, as a trained one does
        labels[_drop(M, case["padding"], g)] = -100
        s["labels"] = labels
    else:
        K = case["K"]
        first = _zipf(M, V, g)
        step = 2 * torch.randint(1, max(2, V // (2 * K)), (M, 1), device="cuda", generator=g) - 1
        ids = (first[:, None] + step * torch.arange(K, device="cuda")) % V
        x += 4.0 * s["w"][first].float()
        top = torch.randn(M, K, device="cuda", generator=g).mul_(2.0).add_(8.0).sort(dim=1, descending=True)[0]
        # a teacher that kept fewer than K of some rows, and none of others
        have = torch.randint(K // 2 + 1, K + 1, (M, 1), device="cuda", generator=g)
        ids[torch.arange(K, device="cuda") >= have] = -1
        ids[_drop(M, case["padding"], g)] = -1
        s["top_ids"], s["top_logits"] = ids.int(), top
    s["x"] = x.to(t)
    s["dloss"] = torch.full((M,), 1.0 / M, device="cuda")
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _own(s):
    from gossipnet_amd import vocab
    op = s["op"]
    if op == "embed_forward":
        return vocab.embed_forward(s["ids"], s["table"], s["scale"], s["token_scale"])
    if op == "embed_backward":
        dtable, dscale = vocab.embed_backward(s["ids"], s["dy"], s["table"], s["scale"], s["token_scale"], need_dscale=s["scaled"])
        return (dtable, dscale) if s["scaled"] else (dtable,)
    if op == "xent":
        loss, lse, hit = vocab.xent_forward(s["x"], s["w"], s["labels"])
        if not s["train"]:
            return loss, lse, hit
        return (loss, lse, hit) + vocab.xent_backward(s["x"], s["w"], s["labels"], lse, hit, s["dloss"])
    loss, lse, hit = vocab.distill_forward(s["x"], s["w"], s["top_ids"], s["top_logits"], s["tau"])
    if not s["train"]:
        return loss, lse, hit
    return (loss, lse, hit) + vocab.distill_backward(s["x"], s["w"], s["top_ids"], s["top_logits"], lse, hit, s["dloss"], s["tau"])


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _plain(s):
    op = s["op"]
    if op == "embed_forward":
        keep = s["ids"] >= 0
        y = s["table"][s["ids"].clamp_min(0)].float() * s["scale"]
        if s["token_scale"] is not None:
            y = y * s["token_scale"][:, None]
        return (y * keep[:, None]).to(s["table"].dtype)
    if op == "embed_backward":
        keep = s["ids"] >= 0
        ids = s["ids"].clamp_min(0)
        dy = s["dy"].float() * s["scale"] * keep[:, None]
        weighted = dy * s["token_scale"][:, None] if s["scaled"] else dy
        dtable = torch.zeros(s["V"], s["D"], device="cuda").index_add_(0, ids, weighted).to(s["dy"].dtype)
        return (dtable, (dy * s["table"][ids].float()).sum(1)) if s["scaled"] else (dtable,)
    x, w = s["x"].float(), s["w"].float()
    if op == "xent":
        tau, ids = 1.0, s["labels"][:, None]
        keep = ids >= 0
        q = keep.float()
        entropy = torch.zeros(s["M"], device="cuda")
    else:
        tau, ids = s["tau"], s["top_ids"].long()
        keep = ids >= 0
        t = torch.where(keep, s["top_logits"] / tau, torch.full_like(s["top_logits"], -1e30))
        e = torch.exp(t - t.amax(1, keepdim=True)) * keep
        total = e.sum(1, keepdim=True).clamp_min(1e-30)
        q = e / total
        entropy = (q * torch.where(keep, t - t.amax(1, keepdim=True) - total.log(), torch.zeros_like(t))).sum(1)
    some = keep.any(1)
    z = x @ w.t()
    hit = torch.gather(z, 1, ids.clamp_min(0)) * keep / tau
    if tau != 1.0:
        z = z / tau
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = (top + total.log())[:, 0] * some
    loss = (entropy + lse - (q * hit).sum(1)) * some
    if op == "xent":
        hit = hit[:, 0]
    if not s["train"]:
        return loss, lse, hit
    p = e / total
    p.scatter_add_(1, ids.clamp_min(0), -q)
    p *= (s["dloss"] * some / tau)[:, None]
    return loss, lse, hit, (p @ w).to(s["x"].dtype), (p.t() @ x).to(s["w"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    M, V, D, size = case["M"], case["V"], case["D"], 4 if case["dtype"] == "f32" else 2
    kept = M - int(round(M * case["padding"]))
    if case["op"] == "embed_forward":
        return {"bytes": 8 * M + kept * D * size + M * D * size + (4 * M if case["scaled"] else 0), "flops": kept * D}
    if case["op"] == "embed_backward":
        more = 8 * M + min(kept, V) * D * size if case["scaled"] else 0
        return {"bytes": 8 * M + kept * D * size + V * D * size + more, "flops": 2 * kept * D}
    K = case.get("K", 1)
    rows = (kept * D + V * D) * size + 8 * M + 4 * M * K + (8 * M if case["op"] == "xent" else 8 * M * K)
    flops = 2 * kept * V * D
    if case["train"]:
        return {"bytes": rows + (M * D + V * D) * size + 4 * M, "flops": 3 * flops}
    return {"bytes": rows, "flops": flops}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    M, V, D, op = case["M"], case["V"], case["D"], case["op"]
    if op.startswith("embed"):
        valid = torch.nonzero(s["ids"] >= 0)[:, 0]
        ids = s["ids"][valid]
        factor = torch.full((valid.numel(), 1), s["scale"], dtype=torch.float64, device="cuda")
        each = s["token_scale"][valid].double()[:, None] if case["scaled"] else 1.0
        if op == "embed_forward":
            y = torch.zeros(M, D, dtype=torch.float64, device="cuda")
            y[valid] = s["table"].double()[ids] * factor * each
            return y
        dy = s["dy"].double()[valid] * factor
        dtable = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_put_((ids,), dy * each, accumulate=True)
        if not case["scaled"]:
            return (dtable,)
        dscale = torch.zeros(M, dtype=torch.float64, device="cuda")
        dscale[valid] = torch.einsum("md,md->m", dy, s["table"].double()[ids])
        return dtable, dscale
    w = s["w"].double()
    tau = case.get("tau", 1.0)
    K = case.get("K", 1)
    loss, lse = (torch.zeros(M, dtype=torch.float64, device="cuda") for _ in range(2))
    hit = torch.zeros(M, K, dtype=torch.float64, device="cuda")
    dx = torch.zeros(M, D, dtype=torch.float64, device="cuda")
    dw = torch.zeros(V, D, dtype=torch.float64, device="cuda") if case["train"] else None
    for a in range(0, M, 1024):
        rows = slice(a, min(M, a + 1024))
        x = s["x"][rows].double()
        logp = x.mm(w.t()).div_(tau)
        l = torch.logsumexp(logp, 1)
        if op == "xent":
            ids = s["labels"][rows].reshape(-1, 1)
            target = torch.zeros_like(ids, dtype=torch.float64)
        else:
            ids = s["top_ids"][rows].long()
            target = s["top_logits"][rows].double() / tau
        valid = ids >= 0
        logq = torch.log_softmax(target.masked_fill(~valid, -math.inf), 1)
        some = valid.any(1)
        q = torch.where(valid, logq.exp(), torch.zeros_like(logq))
        h = torch.where(valid, logp.gather(1, ids.clamp_min(0)), torch.zeros_like(q))
        terms = torch.where(valid, q * (logq - h + l[:, None]), torch.zeros_like(q))
        loss[rows], lse[rows], hit[rows] = terms.sum(1), torch.where(some, l, torch.zeros_like(l)), h
        if case["train"]:
            dz = torch.exp(logp - l[:, None])
            flat = torch.arange(dz.shape[0], device="cuda")[:, None].expand_as(ids)
            dz.index_put_((flat[valid], ids[valid]), -q[valid], accumulate=True)
            dz *= torch.where(some, s["dloss"][rows].double() / tau, torch.zeros_like(l))[:, None]
            dx[rows] = dz.mm(w)
            dw.addmm_(dz.t(), x)
    if op == "xent":
        hit = hit[:, 0]
    return (loss, lse, hit, dx, dw) if case["train"] else (loss, lse, hit)

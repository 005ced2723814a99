"""The language-model operators beside the search, as they are measured.

embed_bags      token ids -> the vectors that IvfUsqIndex searches: per bag of tokens the scaled,
                weighted sum (or mean) of rows of an embedding table; its gradient by sorted tokens.
token_logprobs  log probability of a given token per row of logits, the distribution's entropy and
                its top alternatives; its gradient; and the same for the mixture of the model's
                distribution with the tokens of the neighbours that a search returned.

Each case is a dict; run() is one call (a training case: the call and its gradients).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------- cases
def _bags(name, rows, dim, bags, tokens, dtype, out, mean=False, weighted=False, lookup=False,
          train=False):
    return {"name": name, "op": "embed_bags", "rows": rows, "dim": dim, "bags": bags,
            "tokens": tokens, "dtype": dtype, "out": out, "mean": mean, "weighted": weighted,
            "lookup": lookup, "train": train}


def _probs(name, n, vocab, dtype, top, temperature=1.0, masked=0.0, k=0, train=False):
    return {"name": name, "op": "token_logprobs", "n": n, "vocab": vocab, "dtype": dtype,
            "top": top, "temperature": temperature, "masked": masked, "k": k, "train": train}


def listed():
    return [
        # one query typed by a user, embedded and searched: latency
        _bags("embed_one_query", 32000, 768, 1, 12, "f32", "f32", mean=True),
        # a search batch of 10,000 queries from a 16-bit table, f32 vectors for the index
        _bags("embed_query_batch", 128000, 768, 10000, 150001, "bf16", "f32", mean=True,
              weighted=True),
        # a few long documents before they are added to an index
        _bags("embed_documents", 50257, 128, 37, 300007, "f16", "f32", mean=True),
        # a training step of the query encoder: bags and the gradients of table and weights
        _bags("train_query_batch", 32000, 768, 10000, 150001, "f32", "f32", mean=True,
              weighted=True, train=True),
        # a small fine-tuning step at an odd width
        _bags("train_small", 10007, 100, 257, 3001, "bf16", "f32", weighted=True, train=True),
        # a language model's input embedding, one row per token, and its gradient
        _bags("train_lookup", 50257, 768, 16384, 16384, "bf16", "bf16", lookup=True, train=True),
        # one generated token: its log probability and five alternatives
        _probs("score_one_token", 1, 128000, "bf16", 5),
        # a decoding batch under a grammar: most of the vocabulary masked, some requests finished
        _probs("score_masked_batch", 64, 32000, "f32", 20, temperature=0.7, masked=0.9),
        # scoring prompts at an odd vocabulary: rows that start at odd elements
        _probs("score_prompts", 4099, 50257, "bf16", 5),
        # a training step on log probabilities with an entropy term
        _probs("train_tokens", 4096, 128000, "bf16", 0, train=True),
        # nearest-neighbour language modelling, a decoding batch with the index's top 10
        _probs("neighbours_decode", 16, 32000, "f32", 5, k=10),
        # the same over prompts with the index's top 100
        _probs("neighbours_prompts", 2048, 50257, "f16", 10, k=100),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["bags", "bags", "lookup", "probs", "probs", "neighbours"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    train = rng.random() < 0.5
    if kind in ("bags", "lookup"):
        dim = _log_int(rng, 32, 1024)
        rows = _log_int(rng, 1000, 128000)
        tokens = _log_int(rng, 1, 150000)
        bags = tokens if kind == "lookup" else _log_int(rng, 1, min(10000, max(tokens, 2)))
        c = _bags("", rows, dim, bags, tokens, dtype,
                  dtype if kind == "lookup" else "f32",
                  mean=kind == "bags" and rng.random() < 0.5,
                  weighted=kind == "bags" and rng.random() < 0.5,
                  lookup=kind == "lookup", train=train)
    else:
        vocab = _log_int(rng, 100, 128000)
        n = _log_int(rng, 1, min(8192, (1 << 27) // vocab))
        k = rng.choice([1, 10, 100]) if kind == "neighbours" else 0
        c = _probs("", n, vocab, dtype, rng.choice([0, 1, 5, 20]),
                   temperature=rng.choice([1.0, 1.0, 0.7, 1.3]),
                   masked=rng.choice([0.0, 0.0, 0.5]), k=k, train=train and not k)
    del c["name"]
    return c


# ---------------------------------------------------------------------------- inputs
def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(shape, g):
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32)


def _zipf(n, rows, g):
    """n token ids whose frequency falls as 1 / rank, the low ids most frequent."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return ((rows + 1.0) ** u).long().sub_(1).clamp_(0, rows - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "embed_bags":
        rows, dim, bags, n = case["rows"], case["dim"], case["bags"], case["tokens"]
        s["table"] = (_randn((rows, dim), g) * dim ** -0.5).to(DTYPES[case["dtype"]])
        s["tokens"] = _zipf(n, rows, g)
        s["offsets"] = s["weights"] = None
        if not case["lookup"]:
            cuts = torch.randint(0, n + 1, (bags - 1,), generator=g, device="cuda").sort().values
            ends = torch.tensor([0, n], device="cuda")
            s["offsets"] = torch.cat([ends[:1], cuts, ends[1:]])
        if case["weighted"]:
            s["weights"] = _rand(n, g) * 0.9 + 0.1
        s["scale"] = dim ** 0.5 if case["lookup"] else 1.0
        if case["train"]:
            s["grad"] = _randn((bags, dim), g).to(DTYPES[case["out"]])
        return s
    n, vocab, dt = case["n"], case["vocab"], DTYPES[case["dtype"]]
    # logits of a trained model: a broad bell and a few likely tokens
    logits = _randn((n, vocab), g).mul_(2.0)
    likely = torch.randint(0, vocab, (n, 8), generator=g, device="cuda")
    logits.scatter_add_(1, likely, _rand((n, 8), g) * 10.0)
    s["tokens"] = torch.where(_rand(n, g) < 0.8, likely[:, 0],
                              torch.randint(0, vocab, (n,), generator=g, device="cuda"))
    if case["masked"]:
        logits.masked_fill_(_rand((n, vocab), g) < case["masked"], -math.inf)
        logits[16::17] = -math.inf  # finished requests
    s["logits"] = logits.to(dt)
    if case["k"]:
        # as the index returns them: ascending distances (-inner product), (-1, +inf) padding
        k, total = case["k"], 1000000
        s["ids"] = torch.randint(0, total, (n, k), generator=g, device="cuda")
        s["distances"] = _randn((n, k), g).sub_(12.0).sort(1).values
        short = torch.randint(0, 2 * k, (n, 1), generator=g, device="cuda")
        pad = torch.arange(k, device="cuda")[None, :] > short
        s["ids"].masked_fill_(pad, -1)
        s["distances"].masked_fill_(pad, math.inf)
        s["values"] = _zipf(total, vocab, g)
    if case["train"]:
        s["g_logprobs"] = _randn(n, g).div_(n)
        s["g_entropy"] = _randn(n, g).mul_(0.01 / n)
    return s


# ---------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "embed_bags":
        if own:
            return _own_bags(state, case)
        return _plain_bags(state, case)
    if own:
        return _own_probs(state, case)
    return _plain_probs(state, case)


def _own_bags(s, case):
    from hanns_b200 import embed_bags
    leaves = [s["table"]] + ([] if s["weights"] is None else [s["weights"]])
    if case["train"]:
        leaves = [t.detach().requires_grad_() for t in leaves]
    out = embed_bags(leaves[0], s["tokens"], s["offsets"], *leaves[1:], scale=s["scale"],
                     mean=case["mean"], out_dtype=DTYPES[case["out"]])
    if not case["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, leaves, s["grad"]))


def _own_probs(s, case):
    from hanns_b200 import Neighbours, token_logprobs
    near, logits = None, s["logits"]
    if case["train"]:
        logits = logits.detach().requires_grad_()
    if case["k"]:
        near = Neighbours(s["ids"], s["distances"], s["values"], weight=0.25, temperature=2.0)
    r = token_logprobs(logits, s["tokens"], top=case["top"], temperature=case["temperature"],
                       neighbours=near)
    if not case["train"]:
        return r.logprobs, r.entropy, r.top_tokens, r.top_logprobs
    grad, = torch.autograd.grad([r.logprobs, r.entropy], [logits],
                                [s["g_logprobs"], s["g_entropy"]])
    return r.logprobs.detach(), r.entropy.detach(), r.top_tokens, r.top_logprobs.detach(), grad


def _sums(rows, to, found):
    """Sums of found's rows by the row they go to; 64 bits, for a bag or a token of any length."""
    out = torch.zeros(rows, found.shape[1], device=found.device, dtype=torch.float64)
    return out.index_add_(0, to, found.double())


def _plain_bags(s, case):
    table, tokens, n = s["table"], s["tokens"], case["tokens"]
    coef = torch.full((n,), s["scale"], device=table.device)
    if s["weights"] is not None:
        coef = coef * s["weights"]
    bag = None
    inv = None
    if s["offsets"] is not None:
        lengths = s["offsets"][1:] - s["offsets"][:-1]
        bag = torch.repeat_interleave(torch.arange(case["bags"], device=table.device), lengths,
                                      output_size=n)
        if case["mean"]:
            inv = (1.0 / lengths.clamp(min=1).float())[bag]
            coef = coef * inv
    found = table[tokens].float()
    out = found * coef[:, None]
    if bag is not None:
        out = _sums(case["bags"], bag, out)
    out = out.to(DTYPES[case["out"]])
    if not case["train"]:
        return out
    g = s["grad"].float()
    g = g if bag is None else g[bag]
    d_table = _sums(case["rows"], tokens, g * coef[:, None]).to(table.dtype)
    if s["weights"] is None:
        return out, d_table
    d_weights = (found * g).sum(1) * s["scale"]
    return out, d_table, d_weights if inv is None else d_weights * inv


def _top(x, top):
    """The top columns of each row of x (f32), ties to the lowest index; -1 where there is none."""
    if not top:
        return torch.zeros(x.shape[0], 0, dtype=torch.long, device=x.device)
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    cols = torch.arange(x.shape[1], device=x.device)
    best = torch.topk((key << 32) | (0xFFFFFFFF - cols), top, dim=1).values
    idx = 0xFFFFFFFF - (best & 0xFFFFFFFF)
    return torch.where(x.gather(1, idx) > -math.inf, idx, -1)


def _plain_probs(s, case):
    if case["k"]:
        return _plain_neighbours(s, case)
    inv_t = 1.0 / case["temperature"]
    x = s["logits"].float()
    top_m = x.amax(1, keepdim=True)
    live = top_m > -math.inf
    y = (x - top_m.where(live, torch.zeros_like(top_m))) * inv_t
    e = torch.exp(y)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    ey = (e * y).nan_to_num_(nan=0.0)  # exp(-inf) * -inf
    entropy = (log_z - ey.sum(1, keepdim=True) / z).where(live, torch.zeros_like(z))
    del ey
    log_p = (y - log_z).where(live, torch.full_like(z, -math.inf))
    logprobs = log_p.gather(1, s["tokens"][:, None])[:, 0]
    ids = _top(x, case["top"])
    top_logprobs = log_p.gather(1, ids.clamp(min=0)).masked_fill(ids < 0, -math.inf)
    if not case["train"]:
        return logprobs, entropy[:, 0], ids, top_logprobs
    p = e.div_(z).where(live, torch.zeros_like(e))
    gl, gh = s["g_logprobs"][:, None], s["g_entropy"][:, None]
    grad = (gh * (log_p + entropy) + gl) * p
    grad = grad.nan_to_num_(nan=0.0).neg_()
    grad.scatter_add_(1, s["tokens"][:, None], gl.where(live, torch.zeros_like(gl)))
    grad = (grad * inv_t).to(s["logits"].dtype)
    return logprobs, entropy[:, 0], ids, top_logprobs, grad


def _plain_neighbours(s, case):
    """64 bits: the top alternatives are ordered by values of two sources."""
    lam, inv_t = 0.25, 1.0 / case["temperature"]
    x = s["logits"].double()
    near = s["values"][s["ids"].clamp(min=0)]
    ok = (s["ids"] >= 0) & (x.gather(1, near) > -math.inf)  # a masked token stays masked
    d = s["distances"].double().masked_fill(~ok, math.inf)
    w = torch.exp((d.amin(1, keepdim=True) - d) / 2.0).where(ok, torch.zeros_like(d))
    some = ok.any(1, keepdim=True)
    w = w / w.sum(1, keepdim=True).where(some, torch.ones_like(w[:, :1]))
    lam = torch.full_like(w[:, :1], lam).where(some, torch.zeros_like(w[:, :1]))
    top_m = x.amax(1, keepdim=True)
    live = top_m > -math.inf
    e = torch.exp((x - top_m.where(live, torch.zeros_like(top_m))) * inv_t)
    z = e.sum(1, keepdim=True)
    p = e / z.where(live, torch.ones_like(z)) * (1.0 - lam)
    p.scatter_add_(1, near, w * lam)
    log_p = torch.log(p)
    entropy = -(p * log_p).nan_to_num_(nan=0.0).sum(1)
    logprobs = log_p.gather(1, s["tokens"][:, None])[:, 0]
    best = torch.sort(p, dim=1, descending=True, stable=True)
    most, idx = best.values[:, :case["top"]], best.indices[:, :case["top"]]
    idx = idx.where(most > 0, torch.full_like(idx, -1))
    return logprobs.float(), entropy.float(), idx, torch.log(most).float()


# ---------------------------------------------------------------------------- what a pass needs
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "embed_bags":
        rows, dim, n, bags = case["rows"], case["dim"], case["tokens"], case["bags"]
        edges = np.log(np.arange(1, rows + 2)) / math.log(rows + 1.0)
        touched = float(np.sum(1.0 - np.exp(n * np.log1p(-np.minimum(np.diff(edges), 1 - 1e-12)))))
        b = touched * dim * size[case["dtype"]] + n * 8 + bags * dim * size[case["out"]]
        b += 0 if case["lookup"] else (bags + 1) * 8
        b += 4 * n if case["weighted"] else 0
        f = 2.0 * n * dim
        if case["train"]:
            b += bags * dim * size[case["out"]] + rows * dim * size[case["dtype"]]
            f += 2.0 * n * dim
            if case["weighted"]:
                b += 4 * n
                f += 2.0 * n * dim
        return {"bytes": b, "flops": f}
    n, vocab, k = case["n"], case["vocab"], case["k"]
    b = n * vocab * size[case["dtype"]] + n * (8 + 4 + 4) + n * case["top"] * 12
    b += n * k * (8 + 4 + 8)
    f = 6.0 * n * vocab
    if case["train"]:
        b += n * vocab * size[case["dtype"]] + n * 8
        f += 7.0 * n * vocab
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "embed_bags":
            return _exact_bags(s, case)
        return _exact_probs(s, case)


def _segments(rows, start, stop):
    """Sums of rows[start[i]:stop[i]], from one running sum in 64 bits."""
    run = torch.zeros(rows.shape[0] + 1, rows.shape[1], dtype=torch.float64, device=rows.device)
    torch.cumsum(rows, 0, out=run[1:])
    return run[stop] - run[start]


def _exact_bags(s, case):
    if case["tokens"] * case["dim"] > 1 << 28:
        return None
    dev, n = s["table"].device, case["tokens"]
    off = torch.arange(n + 1, device=dev) if s["offsets"] is None else s["offsets"]
    pos = torch.arange(n, device=dev)
    bag = torch.searchsorted(off, pos, right=True) - 1
    size = (off[1:] - off[:-1]).double()
    coef = torch.full((n,), float(s["scale"]), dtype=torch.float64, device=dev)
    if case["mean"]:
        coef = coef / size[bag]
    weight = torch.ones_like(coef) if s["weights"] is None else s["weights"].detach().double()
    found = s["table"].detach().double()[s["tokens"]]
    out = _segments(found * (coef * weight)[:, None], off[:-1], off[1:])
    if not case["train"]:
        return out
    g = s["grad"].double()[bag]
    order = torch.argsort(s["tokens"], stable=True)
    sorted_tokens = s["tokens"][order]
    ids = torch.arange(case["rows"], device=dev)
    d_table = _segments((g * (coef * weight)[:, None])[order],
                        torch.searchsorted(sorted_tokens, ids),
                        torch.searchsorted(sorted_tokens, ids, right=True))
    if s["weights"] is None:
        return out, d_table
    return out, d_table, torch.einsum("td,td->t", found, g) * coef


def _exact_probs(s, case):
    n, top = case["n"], case["top"]
    x = s["logits"].detach().double() / case["temperature"]
    empty = torch.isneginf(x).all(1)
    log_p = x - torch.logsumexp(x, 1, keepdim=True).masked_fill(empty[:, None], 0.0)
    if case["k"]:
        token = s["values"][s["ids"].clamp(min=0)]
        banned = torch.isneginf(x.gather(1, token)) | (s["ids"] < 0)
        d = (s["distances"].double() / -2.0).masked_fill(banned, -math.inf)
        some = ~banned.all(1)
        knn = torch.softmax(d, 1).nan_to_num(0.0)
        p = torch.zeros_like(x)
        p.scatter_add_(1, token, 0.25 * knn)
        p += torch.exp(log_p) * torch.where(some, 0.75, 1.0).double()[:, None]
        log_p = torch.log(p).masked_fill(empty[:, None], -math.inf)
    p = torch.exp(log_p)
    entropy = torch.special.entr(p).sum(1)
    logprobs = log_p[torch.arange(n, device=x.device), s["tokens"]]
    most = torch.topk(log_p, top, dim=1).values
    if not case["train"]:
        return logprobs, entropy, None, most
    gl, gh = s["g_logprobs"].double()[:, None], s["g_entropy"].double()[:, None]
    grad = -p * gl + gh * (torch.special.entr(p) - p * entropy[:, None])
    keep = torch.where(empty, 0.0, gl[:, 0])
    grad[torch.arange(n, device=x.device), s["tokens"]] += keep
    return logprobs, entropy, None, most, grad / case["temperature"]

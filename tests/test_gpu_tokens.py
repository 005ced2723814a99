"""embed_bags and token_logprobs against their formulas in 64 bits.

Tolerances count roundings.  u = 2^-24 is f32's half step; a result in a 16-bit type has one
rounding of finfo.eps / 2 (and half its smallest step) on top.  A sum of n f32 products has at
most (n + 4) u of the sum of their magnitudes.  For the softmax sums: a thread adds at most
`seq` terms, each with a power of two to 2^-22 = 4 u and an exponent of three roundings, a
rescaling when its maximum grows (at most once a term, 4 u more), and a tree of fewer than 32
additions: (8 seq + 64) u of the sum, plus 4 u per unit of the exponent that counts.
"""
import math

import numpy as np
import pytest
import torch

from hanns_b200 import Neighbours, embed_bags, token_logprobs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(v, dt):
    if dt == F32:
        return U * v.abs()
    tiny = 2.0 ** -25 if dt == F16 else 0.0
    return torch.finfo(dt).eps / 2 * v.abs() + tiny


def close(got, want, tol, what):
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    # f32 holds magnitudes below 2^128 - 2^103 (its largest value is 2^128 - 2^104 and the half
    # step above it 2^103): what is larger rounds to infinity, e.g. 2 * -3.4e38
    want = torch.where(want.abs() >= 2.0 ** 128 - 2.0 ** 103, want.sign() * math.inf, want)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:5], want[bad][:5],
                           torch.as_tensor(tol).expand_as(want)[bad][:5])


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ embed_bags
def bag_formula(table, tokens, offsets, weights, scale, mean):
    """(values, magnitudes, longest bag) in 64 bits."""
    e, n = table.double().cpu(), tokens.numel()
    tokens = tokens.cpu().long()
    off = torch.arange(n + 1) if offsets is None else offsets.cpu().long()
    w = torch.ones(n, dtype=torch.float64) if weights is None else weights.double().cpu()
    out = torch.zeros(off.numel() - 1, e.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    longest = 1
    coef = torch.zeros(n, dtype=torch.float64)  # factor of each position, 0 where it does not count
    bag = torch.full((n,), -1)
    for i in range(off.numel() - 1):
        lo, hi = int(off[i]), int(off[i + 1])
        t = tokens[lo:hi]
        ok = (t >= 0) & (t < e.shape[0])
        c = scale / (max(int(ok.sum()), 1) if mean else 1)
        terms = e[t[ok]] * w[lo:hi][ok][:, None] * c
        out[i], mag[i] = terms.sum(0), terms.abs().sum(0)
        longest = max(longest, hi - lo)
        bag[lo:hi] = torch.where(ok, i, -1)
        coef[lo:hi] = torch.where(ok, c, 0.0)
    return out, mag, longest, bag, coef, w


def bag_grads(table, tokens, bag, coef, w, g):
    e, g, tokens = table.double().cpu(), g.double().cpu(), tokens.cpu().long()
    ok = bag >= 0
    dt = torch.zeros(e.shape, dtype=torch.float64)
    mag = torch.zeros_like(dt)
    terms = g[bag[ok]] * (coef * w)[ok][:, None]
    dt.index_add_(0, tokens[ok], terms)
    mag.index_add_(0, tokens[ok], terms.abs())
    dw, dwm = torch.zeros_like(coef), torch.zeros_like(coef)
    prod = e[tokens[ok]] * g[bag[ok]]
    dw[ok], dwm[ok] = prod.sum(1) * coef[ok], prod.abs().sum(1) * coef[ok].abs()
    often = int(torch.bincount(tokens[ok], minlength=1).max()) if ok.any() else 1
    return dt, mag, dw, dwm, often


def check_bags(table, tokens, offsets, weights, scale=1.0, mean=False, out_dtype=None, seed=0, grad=None):
    out_dtype = out_dtype or table.dtype
    leaf = table.detach().requires_grad_()
    wleaf = None if weights is None else weights.detach().requires_grad_()
    got = embed_bags(leaf, tokens, offsets, wleaf, scale=scale, mean=mean, out_dtype=out_dtype)
    want, mag, longest, bag, coef, w = bag_formula(table, tokens, offsets, weights, scale, mean)
    assert got.dtype == out_dtype
    flat = got.detach().reshape(want.shape)
    close(flat, want, (longest + 6) * U * mag + half_step(want, out_dtype), "out")
    plain = embed_bags(table, tokens, offsets, weights, scale=scale, mean=mean, out_dtype=out_dtype)
    assert torch.equal(plain, got.detach())
    if grad is None:
        grad = torch.randn(flat.shape, generator=gen(seed + 1)).to(out_dtype).cuda()
    leaves = [leaf] + ([] if weights is None else [wleaf])
    grads = torch.autograd.grad(got, leaves, grad.reshape(got.shape), retain_graph=True)
    dt, dmag, dw, dwm, often = bag_grads(table, tokens, bag, coef, w, grad)
    assert grads[0].dtype == table.dtype
    close(grads[0], dt, (often + 6) * U * dmag + half_step(dt, table.dtype), "d_table")
    if weights is not None:
        close(grads[1], dw, (table.shape[1] + 6) * U * dwm, "d_weights")
    again = torch.autograd.grad(got, leaves, grad.reshape(got.shape))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    return got, grads


def offsets_of(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.long).cuda()


def random_bags(seed, rows, lengths, bad=0.1):
    n = int(sum(lengths))
    t = torch.randint(0, rows, (n,), generator=gen(seed))
    drop = torch.rand(n, generator=gen(seed + 1)) < bad
    t[drop] = torch.tensor([-1, rows, 2 ** 40, -2 ** 40])[torch.randint(0, 4, (int(drop.sum()),), generator=gen(seed + 2))]
    return t.cuda(), offsets_of(lengths)


@pytest.mark.parametrize("dtype, out", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("dim", [1, 7, 32, 100, 128, 264, 768, 1030])
def test_bags_of_every_kind(dtype, out, dim):
    rows, lengths = 61, [3, 0, 1, 0, 0, 40, 7, 33, 2, 0]
    table = torch.randn(rows, dim, generator=gen(dim)).to(dtype).cuda()
    tokens, offsets = random_bags(dim, rows, lengths)
    weights = (torch.rand(tokens.numel(), generator=gen(5)) + 0.1).cuda()
    for mean in (False, True):
        for w in (None, weights):
            check_bags(table, tokens, offsets, w, scale=1.7, mean=mean, out_dtype=out, seed=dim)


@pytest.mark.parametrize("lengths", [[5000], [0, 64, 65, 63, 0, 129, 128, 1], [300, 0, 0, 700, 1, 2, 500, 64],
                                     [1] * 70 + [64] + [1] * 63 + [200]])
@pytest.mark.parametrize("dim, dtype", [(20, F32), (768, F32), (128, BF16), (33, F16)])
def test_long_bags_and_tokens(lengths, dim, dtype):
    """Bags and runs of one token on both sides of the length at which they are cut, and one
    token that takes most positions."""
    for rows in (3, 1, 500):
        table = torch.randn(rows, dim, generator=gen(1)).to(dtype).cuda()
        tokens, offsets = random_bags(7, rows, lengths, bad=0.05)
        weights = torch.randn(tokens.numel(), generator=gen(5)).cuda()
        check_bags(table, tokens, offsets, weights, mean=True, out_dtype=F32)
        check_bags(table, tokens, offsets, None, mean=False)


def test_many_tokens_are_cut_in_longer_pieces():
    """More than 64 * 4,096 positions."""
    n, rows = 300_000, 5
    table = torch.randn(rows, 8, generator=gen(1)).cuda()
    tokens = torch.randint(0, rows, (n,), generator=gen(2)).cuda()
    check_bags(table, tokens, torch.tensor([0, 1, n - 5, n]).cuda(), torch.rand(n, generator=gen(3)).cuda(), mean=True)


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 511, 512, 70_000, 300_000])
def test_sort_at_every_key_width(rows):
    n = 5000
    table = torch.randn(rows, 4, generator=gen(rows)).cuda()
    tokens = torch.randint(0, rows, (n,), generator=gen(1))
    tokens[::7], tokens[3::11] = rows - 1, 0
    check_bags(table, tokens.cuda(), offsets_of([n // 2, 0, n - n // 2]), torch.rand(n, generator=gen(2)).cuda())


@pytest.mark.parametrize("rows", [31, 33, 9472, 9473, 18_945, 40_001, 160_007, 310_003])
def test_rows_without_a_token_are_cleared(rows):
    """At every number of rows a warp clears, with tokens in the first, the last and some rows."""
    table = torch.randn(rows, 5, generator=gen(rows)).cuda()
    tokens = torch.tensor([0, rows - 1, rows // 2, rows // 2, min(31, rows - 1), rows - 2]).cuda()
    torch.full((rows, 5), math.nan, device="cuda")  # what the allocator may hand to the gradient
    check_bags(table, tokens, None, None)
    check_bags(table, tokens[:0], None, None)


def test_lookup_shapes_and_types():
    table = torch.randn(50, 24, generator=gen(0)).to(BF16).cuda()
    for shape in ((), (1,), (7,), (3, 5), (2, 0, 4)):
        tokens = torch.randint(-1, 51, shape, generator=gen(1)).cuda()
        got = embed_bags(table, tokens, scale=24 ** 0.5)
        assert got.shape == shape + (24,)
        if tokens.numel():
            check_bags(table, tokens.reshape(-1), None, None, scale=24 ** 0.5)
    t32 = torch.tensor([3, -1, 49], dtype=torch.int32).cuda()
    assert torch.equal(embed_bags(table, t32), embed_bags(table, t32.long()))
    off = torch.tensor([0, 2, 3], dtype=torch.int32).cuda()
    assert torch.equal(embed_bags(table, t32, off), embed_bags(table, t32.long(), off.long()))


def test_nothing_to_do():
    table = torch.randn(5, 8).cuda().requires_grad_()
    none = torch.zeros(0, dtype=torch.long).cuda()
    out = embed_bags(table, none, torch.zeros(4, dtype=torch.long).cuda(), mean=True)
    assert out.shape == (3, 8) and not out.any()
    assert not torch.autograd.grad(out.sum(), table)[0].any()
    out = embed_bags(table, none, torch.zeros(1, dtype=torch.long).cuda())
    assert out.shape == (0, 8)
    assert not torch.autograd.grad(out.sum(), table)[0].any()
    assert embed_bags(table, none).shape == (0, 8)
    w = torch.ones(4).cuda().requires_grad_()
    out = embed_bags(table, torch.full((4,), -1).cuda(), torch.tensor([0, 4]).cuda(), w, mean=True)
    assert not out.any()
    assert not any(g.any() for g in torch.autograd.grad(out.sum(), [table, w]))


def test_positions_outside_every_bag():
    table = torch.randn(9, 16, generator=gen(0)).cuda()
    tokens = torch.randint(0, 9, (12,), generator=gen(1)).cuda()
    w = torch.rand(12, generator=gen(2)).cuda()
    check_bags(table, tokens, torch.tensor([3, 5, 5, 9]).cuda(), w, mean=True)


@pytest.mark.parametrize("n, empty", [(37, 33_000), (3000, 32_000), (3000, 36_000), (5000, 7000), (5000, 9500)])
@pytest.mark.parametrize("place", ["front", "middle", "end"])
def test_many_empty_bags(n, empty, place):
    """On both sides of the number from which positions search for their bags; tokens in front of
    the first bag and behind the last."""
    cuts = np.arange(2, n - 1, 7)
    at = {"front": cuts[0], "middle": cuts[len(cuts) // 2] + 1, "end": cuts[-1]}[place]
    offsets = torch.from_numpy(np.sort(np.concatenate([cuts, np.full(empty, at)]))).cuda()
    tokens, _ = random_bags(n, 50, [n])
    table = torch.randn(50, 2, generator=gen(1)).cuda()
    check_bags(table, tokens, offsets, torch.rand(n, generator=gen(2)).cuda(), mean=True)


def test_padding_rows_are_not_read():
    """A NaN row that no counted token names does not spread."""
    table = torch.randn(4, 64).cuda()
    table[0] = math.nan
    out = embed_bags(table, torch.tensor([1, -1, 2, 3, 7]).cuda(), torch.tensor([0, 3, 5]).cuda())
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("start, width", [(0, 64), (1, 63), (2, 48), (4, 100), (3, 7)])
def test_strided_tables_and_gradients(dtype, start, width):
    """Rows that start at odd elements, tables that are slices, gradients that are slices or
    broadcast."""
    wide = torch.randn(40, 131, generator=gen(3)).to(dtype).cuda()
    tokens, offsets = random_bags(3, 20, [4, 0, 9, 100])
    table = wide[::2, start:start + width]
    check_bags(table, tokens, offsets, None, out_dtype=F32)
    g = torch.randn(4, 131, generator=gen(4)).cuda()[:, start:start + width]
    check_bags(table, tokens, offsets, None, out_dtype=F32, grad=g)
    check_bags(table, tokens, offsets, None, out_dtype=F32, grad=g[:1].expand(4, width))
    check_bags(table, tokens, offsets, None, out_dtype=F32, grad=torch.ones(1, 1).cuda().expand(4, width))


def test_bag_gradient_against_differences():
    """The operator is linear in the table and in the weights: a difference is the gradient's
    inner product.  Small integers, so that every sum is exact."""
    r = gen(9)
    table = torch.randint(-4, 5, (30, 12), generator=r).float().cuda()
    step = torch.randint(-3, 4, (30, 12), generator=r).float().cuda()
    tokens, offsets = random_bags(4, 30, [5, 70, 0, 13])
    w = torch.randint(1, 4, (tokens.numel(),), generator=r).float().cuda()
    dw = torch.randint(-2, 3, (tokens.numel(),), generator=r).float().cuda()
    g = torch.randint(-3, 4, (4, 12), generator=r).float().cuda()
    leaf, wl = table.clone().requires_grad_(), w.clone().requires_grad_()
    gt, gw = torch.autograd.grad(embed_bags(leaf, tokens, offsets, wl), [leaf, wl], g)
    base = embed_bags(table, tokens, offsets, w)
    assert ((embed_bags(table + step, tokens, offsets, w) - base) * g).sum() == (gt * step).sum()
    assert ((embed_bags(table, tokens, offsets, w + dw) - base) * g).sum() == (gw * dw).sum()


def test_table_behind_two_billion_elements():
    rows, dim = 3_000_000, 768
    table = torch.zeros(rows, dim, dtype=F16, device="cuda")
    table[-3:] = torch.arange(3, device="cuda")[:, None] + 1
    tokens = torch.tensor([rows - 1, rows - 3, rows, 0, rows - 2]).cuda()
    leaf = table.requires_grad_()
    out = embed_bags(leaf, tokens, torch.tensor([0, 2, 5]).cuda(), out_dtype=F32)
    assert (out[0] == 4).all() and (out[1] == 2).all()
    g, = torch.autograd.grad(out, leaf, torch.tensor([[1.0], [2.0]]).cuda().expand(2, dim))
    assert (g[-1] == 1).all() and (g[-3] == 1).all() and (g[-2] == 2).all() and (g[0] == 2).all()
    assert g.sum(dtype=torch.float64) == 6 * dim


def test_bags_refuse_bad_arguments():
    t, i = torch.zeros(4, 8).cuda(), torch.zeros(3, dtype=torch.long).cuda()
    off = torch.tensor([0, 3]).cuda()
    for bad in (lambda: embed_bags(t, i.cpu()), lambda: embed_bags(t, i.float()),
                lambda: embed_bags(t[0], i), lambda: embed_bags(t, i, off.cpu()),
                lambda: embed_bags(t, i.reshape(1, 3), off), lambda: embed_bags(t, i, off, torch.ones(2).cuda()),
                lambda: embed_bags(t, i, off, torch.ones(3).cuda().half()), lambda: embed_bags(t, i, off[:0]),
                lambda: embed_bags(t.half(), i, out_dtype=BF16), lambda: embed_bags(t, i, scale=math.inf),
                lambda: embed_bags(t[:, :0], i)):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ token_logprobs
def prob_formula(x, temperature, token):
    """Log probabilities, entropy, the given tokens' log probabilities in 64 bits; NaN for undefined
    rows, -inf and 0 for empty ones."""
    x = x.double().cpu() / temperature
    m = x.amax(1, keepdim=True)
    undefined = x.isnan().any(1) | (x == math.inf).any(1)
    empty = (x == -math.inf).all(1)
    plain = ~(undefined | empty)
    log_p = torch.full_like(x, -math.inf)
    log_p[undefined] = math.nan
    y = x[plain] - m[plain]
    log_p[plain] = y - y.exp().sum(1, keepdim=True).log()
    p = log_p.exp()
    h = -(torch.where(p > 0, p * log_p, 0.0)).sum(1)
    h[undefined] = math.nan
    token = token.cpu().long()
    inside = (token >= 0) & (token < x.shape[1])
    lp = log_p.gather(1, token.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    lp[~inside & ~undefined] = 0.0
    return log_p, h, lp, inside, plain


def top_formula(x, top):
    """By logit, ties to the lower token, no masked ones; -1 elsewhere."""
    x = x.double().cpu()
    ids = torch.full((x.shape[0], top), -1)
    for r in range(x.shape[0]):
        if x[r].isnan().any() or (x[r] == math.inf).any():
            continue
        order = sorted(range(x.shape[1]), key=lambda v: (-float(x[r, v]), v))[:top] if x.shape[1] < 300 \
            else torch.sort(x[r], descending=True, stable=True).indices[:top].tolist()
        order = [v for v in order if x[r, v] > -math.inf]
        ids[r, :len(order)] = torch.tensor(order, dtype=torch.long)
    return ids


def seq_of(vocab):
    return 40 + vocab / 256


def prob_tol(x, log_p, vocab, temperature):
    """(of the softmax sum, of log probabilities, of the entropy)."""
    s = (8 * seq_of(vocab) + 64) * U
    y = (x.double().cpu() / temperature)
    log_s = -(log_p.amax(1, keepdim=True)).nan_to_num(0.0, 0.0, 0.0)
    span = torch.where(log_p.isfinite(), -log_p, 0.0)
    tol_lp = s + 4 * U * (span + 2 * log_s + 1)
    reach = (log_s + 1)[:, 0]  # sum of p |y| is at most log s
    return s, tol_lp, 2 * s * (1 + reach) + 8 * U * (reach + 1)


def check_probs(x, tokens, top=0, temperature=1.0, seed=0, train=True):
    """x [n, vocab] on the GPU (any strides)."""
    n, vocab = x.shape
    leaf = x.detach().requires_grad_(train)
    got = token_logprobs(leaf, tokens, top=top, temperature=temperature)
    log_p, h, lp, inside, plain = prob_formula(x, temperature, tokens)
    s, tol, tol_h = prob_tol(x, log_p, vocab, temperature)
    token = tokens.cpu().long().clamp(0, vocab - 1)
    close(got.logprobs.detach(), lp, tol.gather(1, token[:, None])[:, 0], "logprobs")
    close(got.entropy.detach(), h, tol_h, "entropy")
    ids = top_formula(x, top)
    assert torch.equal(got.top_tokens.cpu(), ids)
    want = log_p.gather(1, ids.clamp(min=0)).masked_fill((ids < 0) & ~log_p[:, :1].isnan(), -math.inf)
    close(got.top_logprobs.detach(), want, tol.gather(1, ids.clamp(min=0)), "top_logprobs")
    plain_call = token_logprobs(x.detach(), tokens, top=top, temperature=temperature)
    for a, b in zip(plain_call, got):
        assert torch.equal(a.nan_to_num(7.0), b.detach().nan_to_num(7.0))
    if not train:
        return
    r = gen(seed + 1)
    gl, gh = torch.randn(n, generator=r), torch.randn(n, generator=r)
    gt = torch.randn(n, top, generator=r)
    outs, gs = [got.logprobs, got.entropy], [gl.cuda(), gh.cuda()]
    if top:
        outs.append(got.top_logprobs)
        gs.append(gt.cuda())
    d, = torch.autograd.grad(outs, leaf, gs)
    assert d.dtype == x.dtype
    gl, gh, gt = gl.double() * inside, gh.double()[:, None], gt.double() * (ids >= 0)
    total = (gl + gt.sum(1))[:, None]
    p = log_p.exp()
    inner = torch.where(p > 0, gh * (log_p.nan_to_num(0.0, 0.0, 0.0) + h[:, None]), 0.0)
    own = torch.zeros_like(p).scatter_add_(1, token[:, None], gl[:, None]).scatter_add_(1, ids.clamp(min=0), gt)
    want = (own - p * (total + inner)) / temperature
    want[~plain & ~h.isnan()] = 0.0
    want[h.isnan()] = math.nan
    size = p * (total.abs() + gh.abs() * (torch.where(log_p.isfinite(), -log_p, 0.0) + h[:, None] + 1))
    tol_d = ((s + 16 * U) * size * 2 + 4 * U * torch.where(log_p.isfinite(), -log_p, 0.0) * size
             + p * gh.abs() * (tol_h[:, None] + tol) + 4 * U * (own.abs() + size)) / temperature
    close(d, want, tol_d.nan_to_num(0.0) + half_step(want.nan_to_num(0.0), x.dtype) + 2.0 ** -120, "d_logits")


def some_logits(seed, n, vocab, dtype, scale=3.0):
    return (torch.randn(n, vocab, generator=gen(seed)) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 5, 8, 31, 33, 100, 257, 1000, 4099, 32771])
def test_probs_of_every_width(dtype, vocab):
    for n, top, temperature in ((1, 0, 1.0), (3, 1, 0.7), (19, 5, 1.3), (2, 32, 1.0)):
        x = some_logits(vocab + n, n, vocab, dtype)
        tokens = torch.randint(-1, vocab + 1, (n,), generator=gen(n)).cuda()
        check_probs(x, tokens, top, temperature)


@pytest.mark.parametrize("dtype, n, vocab", [(F32, 1, 128_003), (BF16, 1, 128_000), (BF16, 5, 50_257),
                                             (F16, 40, 70_001), (F32, 330, 20_000), (BF16, 600, 9_001)])
def test_few_and_many_rows(dtype, n, vocab):
    """One row on a cluster of blocks to a block per row."""
    x = some_logits(n, n, vocab, dtype)
    x[:, 17] = x[:, 19000 % vocab] = 14.0  # a tie at the top, in different blocks
    check_probs(x, torch.randint(0, vocab, (n,), generator=gen(1)).cuda(), 20)


@pytest.mark.parametrize("n, vocab, dtype", [(1, 128_000, BF16), (3, 40_000, F32), (111, 17_000, F16),
                                             (222, 9_000, F32), (223, 20_000, BF16), (445, 9_000, BF16)])
@pytest.mark.parametrize("top", [0, 1, 16, 17, 32])
def test_shared_rows_with_any_alternatives(n, vocab, dtype, top):
    """Rows shared by two, four and eight blocks and by none, on both sides of each rule."""
    x = some_logits(n + top, n, vocab, dtype)
    x[:, 3] = x[:, vocab - 2] = 14.0
    check_probs(x, torch.randint(0, vocab, (n,), generator=gen(1)).cuda(), top)


def special_rows(vocab, dtype):
    low = torch.finfo(dtype).min
    x = torch.randn(16, vocab, generator=gen(2)) * 2
    x[0] = -math.inf                              # empty
    x[1] = -math.inf; x[1, vocab // 2] = 3.0      # one token left
    x[2] = low                                    # masked with the type's lowest value
    x[3, : vocab - 1] = low
    x[4, 1] = math.nan
    x[5, vocab - 1] = math.inf
    x[6] = 0.0                                    # ties alone
    x[7] = torch.arange(vocab) * 1e-3             # climbing
    x[8] = -torch.arange(vocab) * 1e-3            # falling
    x[9, ::2] = -math.inf
    x[10] = 0.0; x[10, 1::2] = -0.0               # one logit, two signs
    x[11, : vocab // 3] = -math.inf
    x[12] = torch.finfo(dtype).max
    x[13, : vocab - 2] = -math.inf                # fewer than the alternatives asked for
    x[14] = low; x[14, 0] = torch.finfo(dtype).max
    x[15] = math.nan
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [3, 64, 1500, 40_000])
def test_masks_ties_and_undefined_rows(dtype, vocab):
    x = special_rows(vocab, dtype)
    for token in (0, vocab - 1, vocab // 2, -1):
        check_probs(x, torch.full((16,), token).cuda(), 7)
    check_probs(x, torch.full((16,), 1).cuda(), 32, temperature=2.0)
    check_probs(x, torch.full((16,), 1).cuda(), 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_climbing_rows_overflow_the_candidates(dtype):
    """Every element is above the threshold of the elements before it."""
    x = torch.linspace(-20, 20, 100_000).repeat(3, 1)
    x[1] = x[1].flip(0)
    x[2] = torch.randint(0, 3, (100_000,), generator=gen(0)).float()  # thousands of ties at the top
    x = x.to(dtype).cuda()
    for n in (1, 3):
        check_probs(x[:n], torch.full((n,), 99_000).cuda(), 32, train=False)
    check_probs(x.repeat(120, 1)[:340], torch.full((340,), 5).cuda(), 5, train=False)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("start, width", [(0, 200), (1, 200), (3, 1021), (5, 64), (8, 1000)])
def test_strided_logits(dtype, start, width):
    wide = some_logits(1, 14, 1031, dtype)
    tokens = torch.randint(0, width, (7,), generator=gen(1)).cuda()
    check_probs(wide[::2, start:start + width], tokens, 4)
    check_probs(wide[:1, start:start + width].expand(7, width), tokens, 4)
    check_probs(wide.t()[start:start + 14, :9].t().contiguous().t()[:9, :], torch.zeros(9, dtype=torch.long).cuda(), 2)


def test_prob_shapes_and_broadcast_gradients():
    x = some_logits(3, 12, 50, F32).reshape(3, 4, 50).requires_grad_()
    tokens = torch.randint(0, 50, (3, 4), generator=gen(0)).cuda()
    r = token_logprobs(x, tokens, top=2)
    assert r.logprobs.shape == r.entropy.shape == (3, 4) and r.top_tokens.shape == r.top_logprobs.shape == (3, 4, 2)
    d, = torch.autograd.grad(r.logprobs.sum(), x)
    want = torch.nn.functional.one_hot(tokens, 50) - torch.softmax(x.detach().double(), -1)
    close(d, want.cpu(), (8 * seq_of(50) + 96) * U * torch.ones(1), "d")
    one = token_logprobs(x[0, 0], tokens[0, 0])
    assert one.logprobs.shape == () and one.logprobs == r.logprobs[0, 0]
    none = token_logprobs(x[:0], tokens[:0], top=3)
    assert none.logprobs.shape == (0, 4) and none.top_tokens.shape == (0, 4, 3)
    assert torch.autograd.grad(token_logprobs(x[:0], tokens[:0]).logprobs.sum(), x)[0].abs().sum() == 0
    assert torch.equal(token_logprobs(x, tokens.int()).logprobs, r.logprobs)


def test_prob_gradient_against_differences():
    """Central differences of the outputs computed in 64 bits at the same f32 logits: the f32
    gradient is within its own roundings of them (the differences' error is about 1e-9)."""
    n, vocab, t = 4, 37, 0.8
    x = some_logits(5, n, vocab, F32)
    tokens = torch.randint(0, vocab, (n,), generator=gen(0)).cuda()
    gl, gh = torch.randn(n, generator=gen(1)), torch.randn(n, generator=gen(2))
    leaf = x.clone().requires_grad_()
    r = token_logprobs(leaf, tokens, temperature=t)
    d, = torch.autograd.grad([r.logprobs, r.entropy], leaf, [gl.cuda(), gh.cuda()])

    def value(z):
        lp = torch.log_softmax(z / t, 1)
        return (gl.double() * lp.gather(1, tokens.cpu()[:, None])[:, 0] - gh.double() * (lp.exp() * lp).sum(1))

    z, eps = x.double().cpu(), 1e-5
    want = torch.zeros(n, vocab, dtype=torch.float64)
    for v in range(vocab):
        e = torch.zeros(n, vocab, dtype=torch.float64)
        e[:, v] = eps
        want[:, v] = (value(z + e) - value(z - e)) / (2 * eps)
    close(d, want, 1e-8 + (8 * seq_of(vocab) + 128) * U * 8 * torch.ones(1), "differences")


def test_logits_behind_two_billion_elements():
    n, vocab = 17_000, 131_072
    x = torch.zeros(n, vocab, dtype=BF16, device="cuda")
    x[-1, -5] = 9.0
    tokens = torch.full((n,), vocab - 5, device="cuda")
    leaf = x.requires_grad_()
    r = token_logprobs(leaf, tokens, top=1)
    z = math.exp(9.0) + vocab - 1
    assert abs(float(r.logprobs[-1].detach()) - (9 - math.log(z))) < 1e-5
    assert int(r.top_tokens[-1, 0]) == vocab - 5 and int(r.top_tokens[-2, 0]) == 0
    g = torch.zeros(n, device="cuda")
    g[-1] = 1.0
    d, = torch.autograd.grad(r.logprobs, leaf, g)
    assert abs(float(d[-1, -5]) - (1 - math.exp(9.0) / z)) < 2 ** -8
    assert not d[:-1].any()


def test_probs_refuse_bad_arguments():
    x, t = torch.zeros(3, 9).cuda(), torch.zeros(3, dtype=torch.long).cuda()
    near = Neighbours(t[:, None], torch.zeros(3, 1).cuda(), t)
    for bad in (lambda: token_logprobs(x, t.cpu()), lambda: token_logprobs(x, t[:2]), lambda: token_logprobs(x, t.float()),
                lambda: token_logprobs(x, t, top=33), lambda: token_logprobs(x, t, top=-1),
                lambda: token_logprobs(x, t, temperature=0.0), lambda: token_logprobs(x, t, temperature=math.nan),
                lambda: token_logprobs(x[:, :0], t), lambda: token_logprobs(x.double(), t),
                lambda: token_logprobs(x.clone().requires_grad_(), t, neighbours=near),
                lambda: token_logprobs(x, t, neighbours=Neighbours(t, torch.zeros(3).cuda(), t)),
                lambda: token_logprobs(x, t, neighbours=Neighbours(t[:, None], torch.zeros(3, 2).cuda(), t)),
                lambda: token_logprobs(x, t, neighbours=Neighbours(t[:, None], torch.zeros(3, 1).cuda(), t.cpu())),
                lambda: token_logprobs(x, t, neighbours=Neighbours(t[:, None], torch.zeros(3, 1).cuda(), t, weight=1.1)),
                lambda: token_logprobs(x, t, neighbours=Neighbours(t[:, None], torch.zeros(3, 1).cuda(), t, temperature=0))):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ neighbours
def near_formula(x, tokens, ids, dist, values, weight, tau, temperature, top):
    log_q, h, lp, inside, plain = prob_formula(x, temperature, tokens)
    n, vocab = log_q.shape
    xd, tokens = x.double().cpu(), tokens.cpu()
    want_ids = top_formula(x, top)
    want_top = log_q.gather(1, want_ids.clamp(min=0)).masked_fill((want_ids < 0) & plain[:, None], -math.inf)
    log_p = log_q.clone()
    for r in range(n):
        if not plain[r]:
            continue
        w = torch.zeros(vocab, dtype=torch.float64)
        found = [(int(values[i]), float(d)) for i, d in zip(ids[r].tolist(), dist[r].tolist())
                 if 0 <= i < len(values) and math.isfinite(d)]
        found = [(v, d) for v, d in found if 0 <= v < vocab and xd[r, v] > -math.inf]
        if not found or weight == 0.0:
            continue
        best = min(d for _, d in found)
        for v, d in found:
            w[v] += math.exp((best - d) / tau)
        wt = float(np.float32(weight))
        p = (1.0 - wt) * log_q[r].exp() + wt * w / w.sum()
        # a token of no neighbour has ln p = ln(1 - weight) + ln q, also where q itself is below
        # what 64 bits hold (ln q < -745)
        log_keep = math.log(1.0 - wt) if wt < 1.0 else -math.inf
        log_p[r] = torch.where(w > 0, p.log(), log_keep + log_q[r])
        h[r] = -torch.where(p > 0, p * p.log(), 0.0).sum()
        lp[r] = log_p[r, tokens[r].clamp(0, vocab - 1)] if inside[r] else 0.0
        order = torch.sort(log_p[r], descending=True, stable=True).indices[:top]
        order = order[log_p[r, order] > -math.inf]
        want_ids[r], want_top[r] = -1, -math.inf
        want_ids[r, :len(order)], want_top[r, :len(order)] = order, log_p[r, order]
    return log_p, lp, h, want_ids, want_top


def check_near(x, tokens, ids, dist, values, weight=0.25, tau=1.5, temperature=1.0, top=5):
    near = Neighbours(ids, dist, values, weight, tau)
    got = token_logprobs(x, tokens, top=top, temperature=temperature, neighbours=near)
    log_p, lp, h, want_ids, want_top = near_formula(x, tokens, ids.cpu(), dist.cpu(), values.cpu(), weight, tau,
                                                    temperature, top)
    log_q = prob_formula(x, temperature, tokens)[0]
    s, tol, tol_h = prob_tol(x, log_q, x.shape[1], temperature)
    flat = (s + 2 ** -20) * 2
    close(got.logprobs, lp, flat + 4 * U * lp.abs().nan_to_num(0, 0, 0), "logprobs")
    # the neighbours' terms move the entropy by the change of ln s and of q
    close(got.entropy, h, tol_h * 3 + flat, "entropy")
    assert torch.equal(got.top_tokens.cpu(), want_ids)
    close(got.top_logprobs, want_top, flat + 4 * U * want_top.abs().nan_to_num(0, 0, 0), "top_logprobs")


def found(seed, n, k, total, short=True):
    g = gen(seed)
    ids = torch.randint(0, total, (n, k), generator=g)
    dist = (torch.randn(n, k, generator=g) - 12).sort(1).values
    if short:
        pad = torch.arange(k)[None] > torch.randint(0, 2 * k, (n, 1), generator=g)
        ids[pad], dist[pad] = -1, math.inf
    return ids.cuda(), dist.cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("k, vocab, total", [(1, 7, 5), (10, 1000, 500), (33, 33, 40), (100, 5003, 3000), (1024, 2000, 9000)])
def test_neighbours_mixture(dtype, k, vocab, total):
    n = 9
    x = some_logits(k, n, vocab, dtype)
    ids, dist = found(k, n, k, total)
    values = torch.randint(-1, vocab + 1, (total,), generator=gen(k)).cuda()
    tokens = torch.randint(-1, vocab, (n,), generator=gen(k)).cuda()
    tokens[1] = max(int(values[ids[1, 0].clamp(min=0)]), 0) if int(values[ids[1, 0].clamp(min=0)]) < vocab else 0
    for weight, top, temperature in ((0.25, 5, 1.0), (0.9, 32, 0.7), (1.0, 3, 1.0), (0.0, 4, 1.0), (0.5, 0, 1.0)):
        check_near(x, tokens, ids, dist, values, weight, 1.5, temperature, top)


def test_neighbours_that_do_not_count():
    vocab, total = 300, 50
    x = special_rows(vocab, F32)
    n = x.shape[0]
    ids, dist = found(3, n, 12, total, short=False)
    values = torch.randint(0, vocab, (total,), generator=gen(1)).cuda()
    ids[:, 0], ids[:, 1] = total, -2 ** 40
    dist[:, 2], dist[:, 3], dist[:, 4] = math.nan, math.inf, -math.inf
    check_near(x, torch.full((n,), 2).cuda(), ids, dist, values, 0.4)
    check_near(x, torch.full((n,), 2).cuda(), torch.full_like(ids, -1), dist, values, 0.4)
    check_near(x, torch.full((n,), 2).cuda(), ids, dist, torch.full_like(values, vocab), 0.4)
    # one token for all of them, and far apart in distance
    check_near(x, torch.full((n,), 2).cuda(), ids, dist * 40, torch.full_like(values, 2), 0.4)
    x = some_logits(0, 4, 64, F32)
    empty = torch.zeros(4, 0).cuda()
    a = token_logprobs(x, torch.zeros(4, dtype=torch.long).cuda(), top=3, neighbours=Neighbours(empty.long(), empty, values))
    b = token_logprobs(x, torch.zeros(4, dtype=torch.long).cuda(), top=3)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    c = token_logprobs(x, torch.zeros(4, dtype=torch.long).cuda(), top=3,
                       neighbours=Neighbours(ids[:4], dist[:4], values[:0]))
    assert all(torch.equal(p, q) for p, q in zip(c, b))


def test_equal_probabilities_go_to_the_lower_token():
    x = torch.zeros(2, 40).cuda()
    ids = torch.tensor([[3, 1, 2, 0], [0, 1, 2, 3]]).cuda()
    values = torch.tensor([30, 20, 25, 39]).cuda()
    check_near(x, torch.tensor([20, 0]).cuda(), ids, torch.full((2, 4), -5.0).cuda(), values, 0.5, top=8)


# ------------------------------------------------------------------ streams, graphs, together
def test_other_streams():
    table = torch.randn(500, 96, generator=gen(0)).cuda()
    tokens, offsets = random_bags(1, 500, [200, 3, 0, 90])
    x = some_logits(1, 5, 3000, BF16)
    t = torch.randint(0, 3000, (5,), generator=gen(1)).cuda()
    want = embed_bags(table, tokens, offsets, mean=True), *token_logprobs(x, t, top=4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append((embed_bags(table, tokens, offsets, mean=True), *token_logprobs(x, t, top=4)))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_captured_calls_replay_on_new_inputs():
    """Two graphs, of a training step each, captured beside each other and replayed in turn."""
    table = torch.randn(300, 64, generator=gen(0)).cuda()
    tokens, offsets = random_bags(1, 300, [100, 0, 30, 200])
    weights = torch.rand(330, generator=gen(2)).cuda()
    x = some_logits(2, 6, 5000, BF16)
    t = torch.randint(0, 5000, (6,), generator=gen(3)).cuda()
    g = torch.randn(4, 64, generator=gen(4)).cuda()
    gl = torch.randn(6, generator=gen(5)).cuda()
    ids, dist = found(1, 6, 20, 100)
    values = torch.randint(0, 5000, (100,), generator=gen(6)).cuda()

    def step():
        leaf, w, z = table.detach().requires_grad_(), weights.detach().requires_grad_(), x.detach().requires_grad_()
        out = embed_bags(leaf, tokens, offsets, w, mean=True)
        r = token_logprobs(z, t, top=5)
        near = token_logprobs(x, t, top=5, neighbours=Neighbours(ids, dist, values))
        return (out.detach(), *torch.autograd.grad(out, [leaf, w], g), r.logprobs.detach(), r.entropy.detach(),
                r.top_tokens, *torch.autograd.grad([r.logprobs, r.entropy], z, [gl, gl]), *near)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(3):
        tokens.copy_(random_bags(seed + 10, 300, [100, 0, 30, 200])[0])
        x.copy_(some_logits(seed, 6, 5000, BF16))
        ids.copy_(found(seed, 6, 20, 100)[0].clamp(min=0))
        dist.copy_(found(seed, 6, 20, 100, short=False)[1])
        want = [o.clone() for o in step()]
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def capture(step):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


def test_captures_of_every_launch_rule():
    """One row on a cluster, a warp a row, a block a row; the sort in one block and in several; a
    lookup; bags with pieces."""
    cases = []
    for n, vocab, top in ((1, 128_000, 3), (9, 700, 3), (9, 1900, 0), (700, 9_000, 0), (700, 9_000, 4)):
        x = some_logits(n, n, vocab, BF16)
        t = torch.randint(0, vocab, (n,), generator=gen(1)).cuda()
        g = torch.randn(n, generator=gen(2)).cuda()

        def probs(x=x, t=t, g=g, top=top):
            z = x.detach().requires_grad_()
            r = token_logprobs(z, t, top=top)
            return r.logprobs.detach(), r.entropy.detach(), r.top_tokens, *torch.autograd.grad(r.logprobs, z, g)

        cases.append((probs, lambda x=x: x.neg_()))
    for n, bags in ((4096, 3), (9001, 40), (5000, 0)):
        table = torch.randn(800, 48, generator=gen(n)).cuda()
        tokens = torch.randint(-1, 800, (n,), generator=gen(3)).cuda()
        offsets = offsets_of([n // bags] * bags + [n % bags]) if bags else None
        out_rows = n if offsets is None else offsets.numel() - 1
        g = torch.randn(out_rows, 48, generator=gen(4)).cuda()

        def bag(table=table, tokens=tokens, offsets=offsets, g=g):
            leaf = table.detach().requires_grad_()
            out = embed_bags(leaf, tokens, offsets, mean=offsets is not None)
            return out.detach(), *torch.autograd.grad(out, leaf, g)

        cases.append((bag, lambda tokens=tokens: tokens.copy_(tokens.flip(0))))
    for step, change in cases:
        graph, out = capture(step)
        for _ in range(2):
            change()
            want = [o.clone() for o in step()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_calls_from_several_threads():
    import threading
    table = torch.randn(3000, 200, generator=gen(0)).to(BF16).cuda()
    tokens, offsets = random_bags(1, 3000, [300, 2, 0, 9000, 40])
    x = some_logits(1, 40, 30_011, F32)
    t = torch.randint(0, 30_011, (40,), generator=gen(1)).cuda()

    def work():
        leaf, z = table.detach().requires_grad_(), x.detach().requires_grad_()
        out = embed_bags(leaf, tokens, offsets, mean=True, out_dtype=F32)
        r = token_logprobs(z, t, top=6)
        return (out.detach(), *torch.autograd.grad(out, leaf, torch.ones_like(out)), r.logprobs.detach(), r.top_tokens,
                *torch.autograd.grad(r.entropy, z, torch.ones_like(r.entropy)))

    want = work()
    torch.cuda.synchronize()
    wrong = []

    def many():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(15):
                got = work()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(1)

    threads = [threading.Thread(target=many) for _ in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


def test_second_derivatives_are_refused():
    table = torch.randn(5, 8).cuda().requires_grad_()
    out = embed_bags(table, torch.tensor([1, 2]).cuda())
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(out.sum(), table, create_graph=True)
    x = torch.randn(2, 9).cuda().requires_grad_()
    r = token_logprobs(x, torch.tensor([1, 2]).cuda())
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(r.logprobs.sum(), x, create_graph=True)


def test_broadcast_inputs_get_the_sum_of_their_gradients():
    """One row for the whole table, one weight for all positions, one row of logits for all tokens."""
    tokens, offsets = random_bags(1, 6, [40, 3, 0, 70], bad=0.0)
    row = torch.randint(-3, 4, (1, 16), generator=gen(0)).float().cuda().requires_grad_()
    one = torch.full((1,), 2.0).cuda().requires_grad_()
    g = torch.randint(-2, 3, (4, 16), generator=gen(1)).float().cuda()
    d_row, d_one = torch.autograd.grad(embed_bags(row.expand(6, 16), tokens, offsets, one.expand(113)), [row, one], g)
    lengths = (offsets[1:] - offsets[:-1]).float()
    assert torch.equal(d_row[0], (g * lengths[:, None]).sum(0) * 2.0)
    assert d_one[0] == (g * lengths[:, None] * row.detach()).sum()
    x = some_logits(3, 1, 300, F32).requires_grad_()
    t = torch.randint(0, 300, (50,), generator=gen(2)).cuda()
    d, = torch.autograd.grad(token_logprobs(x.expand(50, 300), t).logprobs.sum(), x)
    want = torch.bincount(t, minlength=300).double() - 50 * torch.softmax(x.detach().double(), 1)
    # fifty gradients, each within its own roundings, and their sum
    close(d, want.cpu(), 50 * ((8 * seq_of(300) + 96) * U + 50 * U) * torch.ones(1), "d")


@pytest.fixture(scope="module")
def small_index():
    from hanns_b200 import METRIC_IP, IvfUsqConfig, IvfUsqIndex
    rng = np.random.default_rng(5)
    idx = IvfUsqIndex(IvfUsqConfig(64, 16, 8, metric_type=METRIC_IP))
    base = rng.normal(size=(3000, 64)).astype(np.float32)
    idx.train(base)
    idx.add(base)
    return idx


@pytest.mark.parametrize("stream", [False, True])
def test_tokens_to_search_to_next_token(small_index, stream):
    """Token ids in, embedded, searched, and the neighbours' tokens mixed into the model's."""
    from hanns_b200 import SearchRequest
    vocab, n = 700, 33
    table = torch.randn(vocab, 64, generator=gen(0)).to(BF16).cuda()
    tokens, offsets = random_bags(1, vocab, np.random.default_rng(0).integers(1, 20, n).tolist())
    req = SearchRequest(top_k=10, nprobe=8)
    q = embed_bags(table, tokens, offsets, mean=True, out_dtype=F32)
    res = small_index.search(q.cpu().numpy(), req)
    with torch.cuda.stream(torch.cuda.Stream() if stream else torch.cuda.current_stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        ids, dist = small_index.search_tokens(table, tokens, offsets, req)
        x = q @ table.float().t()
        given = torch.randint(0, vocab, (n,), generator=gen(3)).cuda()
        values = torch.randint(0, vocab, (3000,), generator=gen(4)).cuda()
        got = small_index.token_logprobs(q, x, given, values, req, weight=0.3, knn_temperature=2.0, top=6)
        torch.cuda.current_stream().synchronize()
    assert np.array_equal(ids.cpu().numpy().reshape(-1), res.ids)
    assert np.array_equal(dist.cpu().numpy().reshape(-1).view(np.uint32), res.distances.view(np.uint32))
    want = token_logprobs(x, given, top=6, neighbours=Neighbours(ids, dist, values, 0.3, 2.0))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_near(x, given, ids, dist, values, 0.3, 2.0, 1.0, 6)


def test_more_probes_than_lists_and_no_rows(small_index):
    from hanns_b200 import SearchRequest
    table = torch.randn(50, 64, generator=gen(0)).cuda()
    tokens, offsets = random_bags(1, 50, [3, 4])
    a = small_index.search_tokens(table, tokens, offsets, SearchRequest(top_k=4, nprobe=16))
    b = small_index.search_tokens(table, tokens, offsets, SearchRequest(top_k=4, nprobe=1000))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    none = torch.zeros(0, dtype=torch.long).cuda()
    ids, dist = small_index.search_tokens(table, none, none.new_zeros(1), SearchRequest(top_k=4))
    assert ids.shape == dist.shape == (0, 4)
    r = small_index.token_logprobs(torch.zeros(0, 64).cuda(), torch.zeros(0, 9).cuda(), none, tokens, SearchRequest(top_k=4), top=2)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 2)


def test_index_methods_refuse(small_index):
    from hanns_b200 import SearchRequest
    req = SearchRequest(top_k=3)
    t = torch.zeros(3, dtype=torch.long).cuda()
    off = torch.tensor([0, 3]).cuda()
    for bad in (lambda: small_index.search_tokens(torch.zeros(5, 63).cuda(), t, off, req),
                lambda: small_index.search_tokens(torch.zeros(5, 64), t, off, req),
                lambda: small_index.search_tokens(np.zeros((5, 64), np.float32), t, off, req),
                lambda: small_index.search_tokens(torch.zeros(5, 64).cuda(), t, None, req),
                lambda: small_index.token_logprobs(torch.zeros(3, 63).cuda(), torch.zeros(3, 9).cuda(), t, t, req),
                lambda: small_index.token_logprobs(torch.zeros(2, 64).cuda(), torch.zeros(3, 9).cuda(), t, t, req)):
        with pytest.raises(ValueError):
            bad()


def test_training_step_of_a_token_encoder():
    """Both operators in one loss: bags against a tied table; gradients against autograd in 64 bits."""
    vocab, dim = 400, 32
    table = (torch.randn(vocab, dim, generator=gen(0)) * 0.3).cuda()
    tokens, offsets = random_bags(2, vocab, [5, 9, 1, 30, 2], bad=0.0)
    given = torch.randint(0, vocab, (5,), generator=gen(1)).cuda()
    leaf = table.clone().requires_grad_()
    bags = embed_bags(leaf, tokens, offsets, mean=True)
    r = token_logprobs(bags.double().matmul(leaf.double().t()).float(), given)
    loss = -r.logprobs.sum() - 0.1 * r.entropy.sum()
    got, = torch.autograd.grad(loss, leaf)
    ref = table.double().cpu().requires_grad_()
    b64 = torch.stack([ref[tokens.cpu()[int(a):int(b)]].mean(0) for a, b in zip(offsets[:-1], offsets[1:])])
    lp = torch.log_softmax(b64 @ ref.t(), 1)
    (-lp.gather(1, given.cpu()[:, None]).sum() + 0.1 * (lp.exp() * lp).sum()).backward()
    # f32 logits and gradients: a few hundred roundings of values near 1
    close(got, ref.grad, 512 * U * (1 + ref.grad.abs()), "d_table")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [300, 9001])
@pytest.mark.parametrize("temperature, g_entropy", [(0.01, 65536.0), (1.0, 2.0 ** 30), (1e-5, 1.0)])
def test_masked_logits_have_no_gradient_however_large_the_entropys(dtype, vocab, temperature, g_entropy):
    """A scaled loss's gradient of the entropy times a masked element's exponent is out of f32's range."""
    x = some_logits(vocab, 3, vocab, dtype, scale=0.01)
    x[:, 1::2] = -math.inf
    x = x.requires_grad_()
    r = token_logprobs(x, torch.tensor([0, 2, 4]).cuda(), temperature=temperature)
    d, = torch.autograd.grad(r.entropy, x, torch.full((3,), g_entropy).cuda())
    assert (d[:, 1::2] == 0).all()
    if dtype != F16:  # (out of its range otherwise)
        log_p, h, _, _, _ = prob_formula(x.detach(), temperature, torch.zeros(3))
        p = log_p.exp()
        inner = torch.where(p > 0, log_p.nan_to_num(0.0, 0.0, 0.0) + h[:, None], 0.0)
        want = -p * g_entropy * inner / temperature
        s, tol, tol_h = prob_tol(x.detach(), log_p, vocab, temperature)
        size = p * g_entropy * (torch.where(log_p.isfinite(), -log_p, 0.0) + h[:, None] + 1)
        tol_d = ((2 * s + 16 * U) * size + 4 * U * torch.where(log_p.isfinite(), -log_p, 0.0) * size
                 + p * g_entropy * (tol_h[:, None] + tol.nan_to_num(0.0)) + 4 * U * size) / temperature
        # a p below f32's smallest normal value 2^-126 is 0 on the GPU: its term is at most
        # 2^-126 (126 ln 2 + H + 1) g / T, and H is at most ln 9001 < 10
        lost = 2.0 ** -126 * 100 * g_entropy / temperature
        close(d, want, tol_d.nan_to_num(0.0) + half_step(want, dtype) + lost, "d_logits")


# ------------------------------------------------------------------ logits of any size
def large_rows(vocab, dtype):
    """Masks of -1e9 to -1e30, rows of nothing else, and rows whose largest logit is as far from 0."""
    g = gen(vocab)
    x = torch.randn(12, vocab, generator=g) * 3
    for r, low in enumerate((-1e9, -1e10, -1e12, -1e20, -1e30)):
        x[r, : vocab - vocab // 4] = low
    x[5] = -1e10
    x[6] = -1e30
    x[7] = -1e20 * (1 + torch.rand(vocab, generator=g))
    x[8] = 1e10
    x[8, ::3] -= 4096.0
    x[9] = 3e12 * torch.rand(vocab, generator=g)
    x[10, ::2] = 1e30
    x[11, ::2] = -3e10
    top = torch.finfo(dtype).max
    return x.clamp(-top, top).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [300, 3000, 70_001])
@pytest.mark.parametrize("temperature", [1e-9, 1e-6, 1.0, 1e8])
def test_logits_far_from_zero(dtype, vocab, temperature):
    x = large_rows(vocab, dtype)
    tokens = torch.randint(0, vocab, (12,), generator=gen(1)).cuda()
    tokens[::2] = vocab - 1
    # f16 gradients of 1 / temperature are out of range
    check_probs(x, tokens, 5, temperature, train=dtype != F16 or temperature >= 1.0)
    check_probs(x.repeat(60, 1), tokens.repeat(60), 0, temperature, train=False)


# ------------------------------------------------------------------ derivatives there are not
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(grad):
    from torch.autograd import forward_ad as fw
    table, w = torch.randn(6, 8).cuda().requires_grad_(grad), torch.rand(3).cuda().requires_grad_(grad)
    tokens, offsets = torch.tensor([1, 2, 0]).cuda(), torch.tensor([0, 2, 3]).cuda()
    x = torch.randn(3, 9).cuda().requires_grad_(grad)
    near = Neighbours(tokens[:, None], torch.zeros(3, 1).cuda(), tokens)
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))

        for call in (lambda: embed_bags(dual(table), tokens), lambda: embed_bags(dual(table), tokens, offsets),
                     lambda: embed_bags(table, tokens, offsets, dual(w)), lambda: token_logprobs(dual(x), tokens, top=2),
                     lambda: token_logprobs(dual(x.detach()), tokens, neighbours=near),
                     lambda: token_logprobs(x.detach(), tokens, neighbours=Neighbours(
                         tokens[:, None], dual(torch.zeros(3, 1).cuda()), tokens))):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        # inputs without a tangent are not refused
        assert embed_bags(table, tokens, offsets, w).shape == (2, 8)
        assert token_logprobs(x, tokens).logprobs.shape == (3,)


def test_backward_frees_what_the_forward_call_kept():
    """All of it is saved as tensors: hooks see it, and it goes with a pass that keeps no graph."""
    x = torch.randn(70_000, 8).cuda().requires_grad_()
    tokens = torch.zeros(70_000, dtype=torch.long).cuda()
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(tuple(t.shape)) or t, lambda t: t):
        r = token_logprobs(x, tokens)
    assert (70_000, 4) in seen
    held = torch.cuda.memory_allocated()
    loss = r.logprobs.sum()
    d, = torch.autograd.grad(loss, x)
    del d, loss
    assert torch.cuda.memory_allocated() <= held - 70_000 * 16


def test_a_table_updated_before_the_backward_pass():
    """The table's gradient does not read the table; the weights' does, and torch refuses it then."""
    table, w = torch.randn(9, 8).cuda().requires_grad_(), torch.rand(5).cuda().requires_grad_()
    tokens, offsets = torch.tensor([1, 8, 1, -1, 3]).cuda(), torch.tensor([0, 3, 5]).cuda()
    g = torch.randn(2, 8).cuda()
    want = torch.autograd.grad(embed_bags(table, tokens, offsets, w.detach(), mean=True), table, g)
    out = embed_bags(table, tokens, offsets, w.detach(), mean=True)
    both = embed_bags(table, tokens, offsets, w)
    with torch.no_grad():
        table.mul_(3.0)
    assert torch.equal(torch.autograd.grad(out, table, g)[0], want[0])
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(both, [table, w], g)


def test_distances_with_gradients_are_refused():
    x, t = torch.randn(3, 9).cuda(), torch.tensor([1, 2, 0]).cuda()
    dist = torch.rand(3, 1).cuda().requires_grad_()
    near = Neighbours(t[:, None], dist, t)
    with pytest.raises(ValueError, match="distances"):
        token_logprobs(x, t, neighbours=near)
    with torch.no_grad():
        got = token_logprobs(x, t, neighbours=near)
    want = token_logprobs(x, t, neighbours=Neighbours(t[:, None], dist.detach(), t))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_memory_of_a_gradient_of_the_table_alone():
    """Weights without a gradient: the same table gradient, with no more memory than without weights."""
    n, dim = 200_000, 256
    table = torch.randn(1000, dim, generator=gen(0)).cuda().requires_grad_()
    tokens = torch.randint(0, 1000, (n,), generator=gen(1)).cuda()
    offsets, w = offsets_of([n // 4] * 4), torch.rand(n, generator=gen(2)).cuda()
    g = torch.randn(4, dim, generator=gen(3)).cuda()
    peak, grads = {}, {}
    for name, weights, leaves in (("none", None, [table]), ("alone", w, [table]),
                                  ("both", w.clone().requires_grad_(), None)):
        out = embed_bags(table, tokens, offsets, weights)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads[name] = torch.autograd.grad(out, leaves or [table, weights], g)[0]
        peak[name] = torch.cuda.max_memory_allocated() - before
    assert torch.equal(grads["alone"], grads["both"])
    assert peak["alone"] == peak["none"] and peak["both"] >= peak["alone"] + 4 * n * dim // 32


def test_as_many_bags_as_there_may_be():
    """2^31 - 2 of them, three tokens in the last three: indexes of offsets reach 2^31 - 2."""
    n = 2 ** 31 - 2
    offsets = torch.zeros(n + 1, dtype=torch.long, device="cuda")
    offsets[-3:] = torch.tensor([1, 2, 3]).cuda()
    table = torch.tensor([[1.0], [2.0], [4.0], [8.0]]).to(BF16).cuda().requires_grad_()
    tokens = torch.tensor([3, 1, 3]).cuda()
    out = embed_bags(table, tokens, offsets)
    assert out.shape == (n, 1) and out[-3:, 0].tolist() == [8.0, 2.0, 8.0]
    assert not out.detach()[:-3].any()
    g, = torch.autograd.grad(out, table, torch.full((1, 1), 3.0).to(BF16).cuda().expand(n, 1))
    assert g[:, 0].tolist() == [0.0, 3.0, 0.0, 6.0]


# ------------------------------------------------------------------ inputs at their edges
def test_weights_alone_have_a_gradient():
    """A frozen table: the weights' gradient is the one that comes with the table's."""
    for dtype, rows, n, dim in ((F32, 50, 300, 33), (BF16, 3000, 9001, 128)):
        table = torch.randn(rows, dim, generator=gen(0)).to(dtype).cuda()
        tokens, offsets = random_bags(1, rows, [n // 3, 0, n // 3, 5])
        w = torch.rand(tokens.numel(), generator=gen(2)).cuda().requires_grad_()
        g = torch.randn(4, dim, generator=gen(3)).cuda()
        alone, = torch.autograd.grad(embed_bags(table, tokens, offsets, w, mean=True, out_dtype=F32), w, g)
        _, (_, both) = check_bags(table, tokens, offsets, w.detach(), mean=True, out_dtype=F32, grad=g)
        assert torch.equal(alone, both)


def test_weights_outside_every_bag_do_not_count():
    table = torch.randn(9, 16, generator=gen(0)).cuda()
    tokens = torch.randint(0, 9, (5000,), generator=gen(1)).cuda()
    w = torch.rand(5000, generator=gen(2))
    w[:7], w[4000:] = math.nan, math.inf
    offsets = torch.tensor([7, 20, 20, 4000]).cuda()
    inside = w.clone()
    inside[:7] = inside[4000:] = 0.0
    w, inside = w.cuda().requires_grad_(), inside.cuda().requires_grad_()
    leaf, g = table.clone().requires_grad_(), torch.randn(3, 16, generator=gen(3)).cuda()
    got, want = embed_bags(leaf, tokens, offsets, w, mean=True), embed_bags(leaf, tokens, offsets, inside, mean=True)
    assert torch.equal(got, want) and torch.isfinite(got).all()
    for a, b in zip(torch.autograd.grad(got, [leaf, w], g), torch.autograd.grad(want, [leaf, inside], g)):
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("n", [300, 9001])
def test_offsets_outside_the_tokens(n):
    """Ascending ones past both ends are the ends; of others the results are not specified, but
    nothing else is touched."""
    table = torch.randn(40, 24, generator=gen(0)).cuda().requires_grad_()
    tokens = torch.randint(0, 40, (n,), generator=gen(1)).cuda()
    offsets = torch.tensor([-2 ** 62, -5, 3, n // 2, n // 2, n + 9, 2 ** 62]).cuda()
    g = torch.randn(6, 24, generator=gen(2)).cuda()
    want = embed_bags(table, tokens, offsets.clamp(0, n), mean=True)
    got = embed_bags(table, tokens, offsets, mean=True)
    assert torch.equal(got, want)
    d_want, = torch.autograd.grad(want, table, g)
    assert torch.equal(torch.autograd.grad(got, table, g)[0], d_want)
    for seed in range(3):
        wild = torch.randint(-n, 2 * n, (7,), generator=gen(seed)).cuda()
        wild[seed] = (-2 ** 63, 2 ** 63 - 1, 0)[seed]
        torch.autograd.grad(embed_bags(table, tokens, wild, mean=True), table, g)
    assert torch.equal(embed_bags(table, tokens, offsets, mean=True), want)


def test_values_and_ids_of_32_bits():
    x = some_logits(0, 9, 500, F32)
    tokens = torch.randint(0, 500, (9,), generator=gen(1)).cuda()
    ids, dist = found(2, 9, 20, 60)
    values = torch.randint(-1, 501, (60,), generator=gen(3)).cuda()
    want = token_logprobs(x, tokens, top=4, neighbours=Neighbours(ids, dist, values))
    got = token_logprobs(x, tokens.int(), top=4, neighbours=Neighbours(ids.int(), dist, values.int()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_index_methods_refuse_what_is_no_matrix_or_no_tensor(small_index):
    from hanns_b200 import SearchRequest
    req, t = SearchRequest(top_k=3), torch.zeros(3, dtype=torch.long).cuda()
    for bad in (lambda: small_index.search_tokens(torch.zeros(()).cuda(), t, torch.tensor([0, 3]).cuda(), req),
                lambda: small_index.search_tokens(torch.zeros(64).cuda(), t, torch.tensor([0, 3]).cuda(), req),
                lambda: small_index.token_logprobs(torch.zeros(()).cuda(), torch.zeros(9).cuda(), t[0], t, req),
                lambda: small_index.token_logprobs(torch.zeros(3, 64).cuda(), torch.zeros(3, 9).cuda(), [0, 1, 2], t, req)):
        with pytest.raises(ValueError):
            bad()

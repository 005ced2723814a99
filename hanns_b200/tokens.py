"""Language-model operators beside the search, on torch CUDA tensors.

embed_bags      token ids -> vectors to search with (or to add), from an embedding table
token_logprobs  log probabilities of given tokens from logits, their entropy and the most likely
                alternatives; with `neighbours` those of the mixture with what a search found

Both go through the C ABI (hanns_gpu_embed_bags_*, hanns_gpu_token_logprobs_*,
hanns_gpu_neighbour_logprobs_device), run on the current stream of the tensors' device,
take their scratch from torch's allocator and are differentiable once, in reverse mode.  Bad
arguments raise ValueError, GPU failures and derivatives that there are not RuntimeError.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib as L

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _check(rc: int, what: str):
    if rc != 0:
        msg = L.last_error()
        if rc == 2:
            raise ValueError(f"{what}: {msg}")
        raise RuntimeError(f"{what} failed ({rc}): {msg}")


def _need(ok, what: str):
    if not ok:
        raise ValueError(what)


# (messages are put together only when they are raised: these run on every call)
def _cuda(t, name):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device, not {t.device}")


def _on(t, device, name):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, not {t.device}")


def _ids(t, device, name):
    _on(t, device, name)
    if t.dtype != torch.int64:
        if t.dtype != torch.int32:
            raise ValueError(f"{name} must be int64 or int32, not {t.dtype}")
        t = t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """t with its last dimension dense, or a copy (rows may be any distance apart)."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _run(dev, work, *args):
    """work(stream, *args) with dev current, on dev's current stream."""
    index = dev.index
    if torch.cuda.current_device() == index:
        return work(torch._C._cuda_getCurrentRawStream(index), *args)
    with torch.cuda.device(dev):
        return work(torch._C._cuda_getCurrentRawStream(index), *args)


def _workspace(nbytes, device, b):
    if nbytes < 0:
        raise ValueError(f"embed_bags: {L.last_error()}")
    if not nbytes:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    b.workspace, b.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _once(what):
    """Gradients are enabled in a backward pass only where it is to be differentiated itself."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} can be differentiated once only")


def _no_tangent(what, *tensors):
    """Inputs of a forward-mode derivative need not require gradients: their results would come
    without a tangent, which stands for zero."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


# ---------------------------------------------------------------------------- embed_bags
def _bags(shape, dtype, table, tokens, offsets, weights, scale, mean, out_dtype, inv_counts):
    n = tokens.shape[0]
    return L.EmbedBags(_DTYPES[dtype], _DTYPES[out_dtype], shape[1], int(mean), shape[0],
                       0 if table is None else table.stride(0), n,
                       n if offsets is None else offsets.shape[0] - 1, scale, 0, _ptr(table),
                       tokens.data_ptr(), _ptr(offsets), _ptr(weights), None, 0, _ptr(inv_counts), None, 0)


def _embed_bags(table, tokens, offsets, weights, scale, mean, out_dtype, keep):
    """The vectors, and with `keep` what a mean's gradient needs (1 / c_i)."""
    dev = table.device
    n_bags = tokens.shape[0] if offsets is None else offsets.shape[0] - 1
    inv = torch.empty(n_bags, dtype=torch.float32, device=dev) if mean and keep else None
    out = torch.empty((n_bags, table.shape[1]), dtype=out_dtype, device=dev)
    b = _bags(table.shape, table.dtype, table, tokens, offsets, weights, scale, mean, out_dtype, inv)
    b.out, b.out_ld = out.data_ptr(), table.shape[1]
    _run(dev, _embed_bags_call, b, dev)
    return out, inv


def _embed_bags_call(stream, b, dev):
    lib, ref = L.lib(), C.byref(b)
    ws = _workspace(lib.hanns_gpu_embed_bags_workspace_bytes(ref), dev, b)  # noqa: F841 (kept until enqueued)
    _check(lib.hanns_gpu_embed_bags_device(ref, stream), "embed_bags")


class _EmbedBags(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, offsets, weights, scale, mean, out_dtype):
        out, inv = _embed_bags(table, tokens, offsets, weights, scale, mean, out_dtype, True)
        # only the weights' gradient reads the table, which may be updated in place otherwise
        ctx.save_for_backward(table if ctx.needs_input_grad[3] else None, tokens, offsets, weights, inv)
        ctx.args = table.shape, table.dtype, scale, mean, out_dtype
        return out

    @staticmethod
    def backward(ctx, grad):
        _once("embed_bags")
        d_table, d_weights = _embed_bags_grad(grad, *ctx.saved_tensors, *ctx.args,
                                              ctx.needs_input_grad[0], ctx.needs_input_grad[3])
        return d_table, None, None, d_weights, None, None, None


def _embed_bags_grad(grad, table, tokens, offsets, weights, inv, shape, dtype, scale, mean, out_dtype,
                     want_table, want_weights):
    dev = tokens.device
    grad = _rows(grad)
    # the weights' gradient is a by-product of the table's
    d_table = torch.empty(shape, dtype=dtype, device=dev)
    d_weights = torch.empty(tokens.shape[0], dtype=torch.float32, device=dev) if want_weights else None
    b = _bags(shape, dtype, table, tokens, offsets, weights, scale, mean, out_dtype, inv)
    _run(dev, _embed_bags_grad_call, b, grad, d_table, d_weights)
    return d_table if want_table else None, d_weights


def _embed_bags_grad_call(stream, b, grad, d_table, d_weights):
    lib, ref = L.lib(), C.byref(b)
    ws = _workspace(lib.hanns_gpu_embed_bags_grad_workspace_bytes(ref), d_table.device, b)  # noqa: F841 (kept until enqueued)
    _check(lib.hanns_gpu_embed_bags_grad_device(ref, grad.data_ptr(), grad.stride(0), d_table.data_ptr(),
                                                d_table.shape[1], _ptr(d_weights), stream), "embed_bags")


def embed_bags(table, tokens, offsets=None, weights=None, *, scale: float = 1.0, mean: bool = False,
               out_dtype=None):
    """Bags of token ids to vectors:

        out[i] = scale / c_i * sum over bag i's tokens t_j of weights[j] * table[t_j]

    table      [rows, dim], float32, float16 or bfloat16; rows may be strided
    tokens     int64 or int32 ids.  With `offsets` one-dimensional: bag i is
               tokens[offsets[i]:offsets[i + 1]].  Without, any shape: every token is a bag
               (a lookup), and the result has the shape tokens.shape + (dim,)
    offsets    ascending int64 or int32 [bags + 1], or None
    weights    float32 [len(tokens)] factors, or None
    mean       divide by c_i, the bag's counted tokens (else c_i = 1)
    out_dtype  the table's type (default) or float32, which IvfUsqIndex searches

    A token outside [0, rows) is not counted (-1 pads, as in search results); an empty bag
    gives zeros; positions outside every bag do not count.  Sums are f32, rounded once.
    Differentiable in table (a dense gradient) and weights; the gradients add a token's terms in
    the order of its positions and do not change from run to run.
    """
    _cuda(table, "table")
    _need(table.dim() == 2 and table.shape[0] > 0 and table.shape[1] > 0, "table must be [rows, dim]")
    dev = table.device
    out_dtype = out_dtype or table.dtype
    _need(out_dtype is torch.float32 or out_dtype is table.dtype, "out_dtype must be the table's type or float32")
    tokens = _ids(tokens, dev, "tokens")
    shape = tokens.shape
    if offsets is None:
        if tokens.dim() != 1:
            tokens = tokens.reshape(-1)
    else:
        _need(tokens.dim() == 1, "tokens must be one-dimensional when offsets are given")
        offsets = _ids(offsets, dev, "offsets")
        _need(offsets.dim() == 1 and offsets.numel() > 0, "offsets must be [bags + 1]")
    if weights is not None:
        _on(weights, dev, "weights")
        _need(weights.dtype == torch.float32, "weights must be float32")
        _need(weights.numel() == tokens.numel(), "weights must have one value per token")
        if weights.dim() != 1 or not weights.is_contiguous():
            weights = weights.reshape(-1).contiguous()
    if forward_ad._current_level >= 0:
        _no_tangent("embed_bags", table, weights)
    scale = float(scale)
    _need(scale == scale and abs(scale) != float("inf"), "scale must be finite")
    args = _rows(table), tokens, offsets, weights, scale, bool(mean), out_dtype
    if (table.requires_grad or weights is not None and weights.requires_grad) and torch.is_grad_enabled():
        out = _EmbedBags.apply(*args)
    else:
        out, _ = _embed_bags(*args, False)
    return out.reshape(*shape, table.shape[1]) if offsets is None and len(shape) != 1 else out


# ---------------------------------------------------------------------------- token_logprobs
class TokenLogprobs(NamedTuple):
    """logprobs and entropy have the tokens' shape, the alternatives one more dimension."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_tokens: torch.Tensor
    top_logprobs: torch.Tensor


@dataclass
class Neighbours:
    """What a search found for each row, and what it says about the next token.

    ids, distances  [..., k] as the search returns them (smaller is nearer, -1 / +inf pads)
    values          [stored ids] int64 or int32: the token that goes with each id
    weight          share of the neighbours in the mixture, in [0, 1]
    temperature     of softmax(-distance / temperature) over the neighbours
    """
    ids: torch.Tensor
    distances: torch.Tensor
    values: torch.Tensor
    weight: float = 0.25
    temperature: float = 1.0


def _probs(logits, tokens, top, temperature, out):
    n, vocab = logits.shape
    return L.TokenLogprobs(_DTYPES[logits.dtype], top, n, vocab, logits.stride(0), temperature, 0,
                           logits.data_ptr(), tokens.data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
                           out[2].data_ptr(), out[3].data_ptr(), _ptr(out[4]))


def _token_logprobs(logits, tokens, top, temperature, near, keep):
    """logprobs, entropy, top tokens, top logprobs and, with `keep`, the rows' statistics."""
    dev, n = logits.device, logits.shape[0]
    f32 = torch.float32
    out = (torch.empty(n, dtype=f32, device=dev), torch.empty(n, dtype=f32, device=dev),
           torch.empty((n, top), dtype=torch.int64, device=dev), torch.empty((n, top), dtype=f32, device=dev),
           torch.empty((n, 4), dtype=f32, device=dev) if keep or near is not None else None)
    _run(dev, _token_logprobs_call, _probs(logits, tokens, top, temperature, out), near)
    return out


def _token_logprobs_call(stream, t, near):
    lib, ref = L.lib(), C.byref(t)
    rc = lib.hanns_gpu_token_logprobs_device(ref, stream)
    if rc == 0 and near is not None:
        ids, distances, values, weight, knn_temperature = near
        rc = lib.hanns_gpu_neighbour_logprobs_device(
            ref, ids.data_ptr(), distances.data_ptr(), ids.shape[-1], values.data_ptr(), values.numel(),
            weight, knn_temperature, stream)
    _check(rc, "token_logprobs")


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, temperature):
        lp, h, tt, tl, stats = _token_logprobs(logits, tokens, top, temperature, None, True)
        ctx.mark_non_differentiable(tt)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, tt, stats)
        ctx.args = top, temperature
        return lp, h, tt, tl

    @staticmethod
    def backward(ctx, g_logprobs, g_entropy, _, g_top):
        _once("token_logprobs")
        logits, tokens, tt, stats = ctx.saved_tensors
        top, temperature = ctx.args
        if g_logprobs is not None:
            g_logprobs = g_logprobs.contiguous()
        if g_entropy is not None:
            g_entropy = g_entropy.contiguous()
        if g_top is not None:
            g_top = g_top.contiguous()
        d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        n, vocab = logits.shape
        # the forward call's outputs are not read: any non-null pointer stands for them
        ptr = logits.data_ptr()
        t = L.TokenLogprobs(_DTYPES[logits.dtype], top, n, vocab, logits.stride(0), temperature, 0, ptr,
                            tokens.data_ptr(), ptr, ptr, tt.data_ptr(), ptr, stats.data_ptr())
        _run(logits.device, _token_logprobs_grad_call, t, g_logprobs, g_entropy, g_top, d)
        return d, None, None, None


def _token_logprobs_grad_call(stream, t, g_logprobs, g_entropy, g_top, d):
    _check(L.lib().hanns_gpu_token_logprobs_grad_device(
        C.byref(t), _ptr(g_logprobs), _ptr(g_entropy), _ptr(g_top), d.data_ptr(), d.shape[1], stream),
        "token_logprobs")


def token_logprobs(logits, tokens, *, top: int = 0, temperature: float = 1.0,
                   neighbours: Neighbours | None = None) -> TokenLogprobs:
    """Log probabilities of given tokens under softmax(logits / temperature), the entropy of
    that distribution, and its `top` most likely tokens.

    logits  [..., vocab] float32, float16 or bfloat16; rows may be strided
    tokens  [...] int64 or int32; a token outside [0, vocab) (-1 pads) gives 0 and no gradient
    top     0 to 32 alternatives, larger logit first and ties to the lower token; (-1, -inf)
            where fewer logits are unmasked

    -inf masks a token.  A row of -inf alone gives log probability -inf, entropy 0 and no
    alternatives (and a zero gradient); a row with NaN or +inf gives NaN.  Differentiable in
    logits, through logprobs, entropy and top_logprobs.

    With `neighbours` the distribution is (1 - weight) * model + weight * neighbours (nearest-
    neighbour language modelling): a neighbour counts when its id is in [0, len(values)), its
    distance is finite and its token is in the vocabulary and not masked; a row without such a
    neighbour keeps the model's distribution.  Scoring only: not differentiable.
    """
    _cuda(logits, "logits")
    _need(logits.dim() >= 1 and logits.shape[-1] > 0, "logits must be [..., vocab]")
    dev, vocab = logits.device, logits.shape[-1]
    tokens = _ids(tokens, dev, "tokens")
    _need(tokens.shape == logits.shape[:-1], "tokens must have the shape of logits without its last dimension")
    top, temperature = int(top), float(temperature)
    _need(0 <= top <= 32, "top must be in [0, 32]")
    near = None
    if neighbours is not None:
        _need(not (logits.requires_grad and torch.is_grad_enabled()),
              "token_logprobs with neighbours is not differentiable: detach the logits")
        ids = _ids(neighbours.ids, dev, "neighbours.ids")
        _on(neighbours.distances, dev, "neighbours.distances")
        _need(neighbours.distances.dtype == torch.float32, "neighbours.distances must be float32")
        _need(not (neighbours.distances.requires_grad and torch.is_grad_enabled()),
              "token_logprobs with neighbours is not differentiable: detach the distances")
        _need(ids.dim() >= 1 and ids.shape[:-1] == tokens.shape and ids.shape == neighbours.distances.shape,
              "neighbours.ids and .distances must be tokens.shape + (k,)")
        values = _ids(neighbours.values, dev, "neighbours.values")
        _need(values.dim() == 1, "neighbours.values must be one-dimensional")
        near = (ids, neighbours.distances.contiguous(), values, float(neighbours.weight),
                float(neighbours.temperature))
    if forward_ad._current_level >= 0:
        _no_tangent("token_logprobs", logits, near and near[1])
    plain = logits.dim() == 2
    args = _rows(logits), tokens, top, temperature
    if not plain:
        args = args[0].reshape(-1, vocab), tokens.reshape(-1), top, temperature
    if logits.requires_grad and torch.is_grad_enabled():
        out = _TokenLogprobs.apply(*args)
    else:
        out = _token_logprobs(*args, near, False)
    if plain:
        return TokenLogprobs(*out[:4])
    s = tokens.shape
    return TokenLogprobs(out[0].reshape(s), out[1].reshape(s), out[2].reshape(*s, top), out[3].reshape(*s, top))

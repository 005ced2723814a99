"""Refusals of the token operators that need no GPU: argument checks of the Python entry points
and of the C ABI, which returns before it touches the device."""
import ctypes as C

import pytest
import torch

from hanns_b200 import Neighbours, _lib as L, embed_bags, token_logprobs


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        embed_bags(torch.zeros(4, 8), torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(4, 8), torch.zeros(4, dtype=torch.long))
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        embed_bags(torch.zeros(4, 8, dtype=torch.float64), torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="tensor"):
        token_logprobs([[0.0]], torch.zeros(1, dtype=torch.long))


def bags(**kw):
    b = L.EmbedBags(dtype=0, out_dtype=0, dim=8, mean=0, rows=10, ld=8, n_tokens=6, n_bags=2, scale=1.0,
                    table=256, tokens=256, offsets=256, out=256, out_ld=8)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


@pytest.mark.parametrize("kw, what", [
    (dict(dtype=7), "element type"), (dict(out_dtype=-1), "element type"),
    (dict(dtype=1, out_dtype=2), "f32 or of the table's type"), (dict(dim=0), "dim"),
    (dict(rows=0), "rows"), (dict(rows=1 << 31), "rows"), (dict(n_tokens=-1), "n_tokens"),
    (dict(n_tokens=1 << 31), "n_tokens"), (dict(n_bags=-1), "n_bags"),
    (dict(offsets=None), "own bag"), (dict(table=None), "null"), (dict(tokens=None), "null"),
    (dict(out=None), "null"), (dict(n_tokens=100000), "workspace"),
    (dict(n_tokens=100000, workspace=256, workspace_bytes=8), "too small"),
    (dict(n_tokens=100000, workspace=264, workspace_bytes=1 << 40), "aligned")])
def test_embed_bags_refuses(kw, what):
    b = bags(**kw)
    assert L.lib().hanns_gpu_embed_bags_device(C.byref(b), None) == 2
    assert what in L.last_error()


def test_embed_bags_grad_refuses():
    lib = L.lib()
    assert lib.hanns_gpu_embed_bags_device(None, None) == 2
    assert lib.hanns_gpu_embed_bags_workspace_bytes(C.byref(bags(dim=-1))) == -1
    assert lib.hanns_gpu_embed_bags_grad_workspace_bytes(C.byref(bags(dim=-1))) == -1
    assert lib.hanns_gpu_embed_bags_workspace_bytes(C.byref(bags())) == 0
    assert lib.hanns_gpu_embed_bags_grad_workspace_bytes(C.byref(bags())) > 0
    b = bags()
    assert lib.hanns_gpu_embed_bags_grad_device(C.byref(b), None, 8, 256, 8, None, None) == 2
    assert "null gradient" in L.last_error()
    assert lib.hanns_gpu_embed_bags_grad_device(C.byref(b), 256, 8, 256, 8, None, None) == 2
    assert "workspace" in L.last_error()
    b = bags(mean=1)
    assert lib.hanns_gpu_embed_bags_grad_device(C.byref(b), 256, 8, 256, 8, None, None) == 2
    assert "inv_counts" in L.last_error()
    b = bags(table=None)
    assert lib.hanns_gpu_embed_bags_grad_device(C.byref(b), 256, 8, None, 0, 256, None) == 2
    assert "table" in L.last_error()


def probs(**kw):
    t = L.TokenLogprobs(dtype=0, top=2, n=3, vocab=10, ld=10, temperature=1.0, logits=256, tokens=256,
                        logprobs=256, entropy=256, top_tokens=256, top_logprobs=256, stats=256)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("kw, what", [
    (dict(dtype=3), "element type"), (dict(n=-1), "n must"), (dict(vocab=0), "vocab"),
    (dict(vocab=1 << 31), "vocab"), (dict(top=33), "top"), (dict(top=-1), "top"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(logprobs=None), "null"),
    (dict(top_tokens=None), "alternatives"), (dict(logits=258), "misaligned"), (dict(stats=260), "stats")])
def test_token_logprobs_refuses(kw, what):
    t = probs(**kw)
    assert L.lib().hanns_gpu_token_logprobs_device(C.byref(t), None) == 2
    assert what in L.last_error()


def test_token_logprobs_grad_and_neighbours_refuse():
    lib = L.lib()
    t = probs(stats=None)
    assert lib.hanns_gpu_token_logprobs_grad_device(C.byref(t), 256, None, None, 256, 10, None) == 2
    assert "stats" in L.last_error()
    t = probs()
    assert lib.hanns_gpu_token_logprobs_grad_device(C.byref(t), 256, None, None, None, 10, None) == 2
    assert lib.hanns_gpu_token_logprobs_grad_device(C.byref(t), 256, None, None, 258, 10, None) == 2
    assert "misaligned" in L.last_error()
    for k, weight, temp, what in [(-1, 0.5, 1.0, "k must"), (1025, 0.5, 1.0, "k must"), (4, -0.1, 1.0, "weight"),
                                  (4, 1.5, 1.0, "weight"), (4, float("nan"), 1.0, "weight"),
                                  (4, 0.5, 0.0, "temperature")]:
        assert lib.hanns_gpu_neighbour_logprobs_device(C.byref(t), 256, 256, k, 256, 9, weight, temp, None) == 2
        assert what in L.last_error()
    assert lib.hanns_gpu_neighbour_logprobs_device(C.byref(t), None, 256, 4, 256, 9, 0.5, 1.0, None) == 2
    t = probs(stats=None)
    assert lib.hanns_gpu_neighbour_logprobs_device(C.byref(t), 256, 256, 4, 256, 9, 0.5, 1.0, None) == 2
    assert "stats" in L.last_error()


def test_names_are_exported():
    import hanns_b200
    for n in ("embed_bags", "token_logprobs", "Neighbours", "TokenLogprobs"):
        assert n in hanns_b200.__all__ and hasattr(hanns_b200, n)
    with pytest.raises(AttributeError):
        hanns_b200.no_such_name
    assert Neighbours(None, None, None).weight == 0.25


class FakeStream:
    def __init__(self, handle):
        self.cuda_stream, self.waited = handle, []

    def wait_stream(self, other):
        self.waited.append(other)


@pytest.mark.parametrize("fails", [False, True])
def test_the_current_stream_waits_for_a_search_that_failed(monkeypatch, fails):
    """Streams and the search are stand-ins: a search may fail after parts of it were enqueued."""
    from hanns_b200 import IvfUsqConfig, IvfUsqIndex
    cur, own = FakeStream(0), FakeStream(7)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *size, device, **kw: empty(*size, **kw))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev: cur)
    monkeypatch.setattr(torch.cuda, "Stream", lambda dev: own)
    idx = IvfUsqIndex.__new__(IvfUsqIndex)
    idx.config, idx.device, idx._h = IvfUsqConfig(4, 1, 8), 0, None

    def search_device(*args, stream):
        assert stream == 7 and own.waited == [cur] and not cur.waited
        if fails:
            raise RuntimeError("out of memory")

    monkeypatch.setattr(idx, "search_device", search_device, raising=False)
    if fails:
        with pytest.raises(RuntimeError, match="out of memory"):
            idx._search_tensors(torch.zeros(2, 4), 3, 1)
    else:
        idx._search_tensors(torch.zeros(2, 4), 3, 1)
    assert cur.waited == [own]


def test_the_tables_gradient_alone_needs_no_room_for_inner_products():
    lib = L.lib()
    n, dim = 100_000, 768
    kw = dict(n_tokens=n, n_bags=10, dim=dim, ld=dim, out_ld=dim)
    plain = lib.hanns_gpu_embed_bags_grad_workspace_bytes(C.byref(bags(**kw)))
    alone = lib.hanns_gpu_embed_bags_grad_workspace_bytes(C.byref(bags(weights=256, table=None, **kw)))
    both = lib.hanns_gpu_embed_bags_grad_workspace_bytes(C.byref(bags(weights=256, **kw)))
    assert alone == plain
    assert both - alone >= n * 4 * dim // 32
    # and asks for no more
    b = bags(weights=256, table=None, workspace=256, workspace_bytes=alone - 1, **kw)
    assert lib.hanns_gpu_embed_bags_grad_device(C.byref(b), 256, dim, 256, dim, None, None) == 2
    assert "too small" in L.last_error()


@pytest.mark.parametrize("kw, what", [
    (dict(table=258), "misaligned"), (dict(table=257, dtype=2), "misaligned"), (dict(tokens=260), "misaligned"),
    (dict(offsets=260), "misaligned"), (dict(weights=258), "misaligned"), (dict(inv_counts=257, mean=1), "misaligned"),
    (dict(out=258), "misaligned"), (dict(out=258, dtype=2), "misaligned"), (dict(ld=-8), "backwards"),
    (dict(out_ld=7), "overlap"), (dict(out_ld=0), "overlap"), (dict(out_ld=-8), "overlap")])
def test_embed_bags_refuses_what_its_kernels_cannot_address(kw, what):
    b = bags(**{"n_tokens": 100_000, "workspace": 256, "workspace_bytes": 8, **kw})  # (refused anyway: too small)
    assert L.lib().hanns_gpu_embed_bags_device(C.byref(b), None) == 2
    assert what in L.last_error()


def test_embed_bags_grad_refuses_what_its_kernels_cannot_address():
    lib = L.lib()
    for args, kw, what in [((258, 8, 256, 8, None), {}, "misaligned"), ((256, 8, 258, 8, None), {}, "misaligned"),
                           ((256, 8, 256, 8, 258), dict(weights=256), "misaligned"),
                           ((256, -8, 256, 8, None), {}, "backwards"), ((256, 8, 256, 7, None), {}, "overlap"),
                           ((256, 8, 256, 8, 256), dict(weights=256, ld=-8), "backwards")]:
        b = bags(**kw)  # (no workspace: refused anyway)
        assert lib.hanns_gpu_embed_bags_grad_device(C.byref(b), *args, None) == 2
        assert what in L.last_error()


@pytest.mark.parametrize("kw, what", [
    (dict(tokens=260), "misaligned"), (dict(logprobs=258), "misaligned"), (dict(entropy=257), "misaligned"),
    (dict(top_tokens=260), "misaligned"), (dict(top_logprobs=258), "misaligned"), (dict(ld=-10), "backwards")])
def test_token_logprobs_refuses_what_its_kernels_cannot_address(kw, what):
    lib = L.lib()
    for call in (lambda t: lib.hanns_gpu_token_logprobs_device(C.byref(t), None),
                 lambda t: lib.hanns_gpu_neighbour_logprobs_device(C.byref(t), 256, 256, 4, 256, 9, 0.0, 1.0, None)):
        assert call(probs(**kw)) == 2
        assert what in L.last_error()


def test_token_logprobs_grad_and_neighbours_refuse_what_their_kernels_cannot_address():
    lib = L.lib()
    for args, what in [((258, None, None, 256, 10), "misaligned"), ((None, 257, None, 256, 10), "misaligned"),
                       ((None, None, 258, 256, 10), "misaligned"), ((256, None, None, 256, 9), "overlap"),
                       ((256, None, None, 256, -10), "overlap")]:
        t = probs()
        assert lib.hanns_gpu_token_logprobs_grad_device(C.byref(t), *args, None) == 2
        assert what in L.last_error()
    for ids, dist, values in ((260, 256, 256), (256, 258, 256), (256, 256, 260)):
        t = probs()
        assert lib.hanns_gpu_neighbour_logprobs_device(C.byref(t), ids, dist, 4, values, 9, 0.5, 1.0, None) == 2
        assert "misaligned" in L.last_error()

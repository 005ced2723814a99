"""Calls on one index handle, on any streams and threads, work in the order in which they were made:
the handle's buffers are one call's after the other's."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DIM, VOCAB = 64, 500


def make_index(n=20_000):
    from hanns_b200 import METRIC_IP, IvfUsqConfig, IvfUsqIndex
    rng = np.random.default_rng(5)
    idx = IvfUsqIndex(IvfUsqConfig(DIM, 64, 8, metric_type=METRIC_IP))
    base = rng.normal(size=(n, DIM)).astype(np.float32)
    idx.train(base, kmeans_iters=5)
    idx.add(base)
    return idx


@pytest.fixture(scope="module")
def index():
    return make_index()


def request():
    from hanns_b200 import SearchRequest
    return SearchRequest(top_k=20, nprobe=32)


def batch(seed, bags):
    """table, tokens, offsets of `bags` bags of four tokens."""
    import torch
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(VOCAB, DIM, generator=g).cuda()
    tokens = torch.randint(0, VOCAB, (4 * bags,), generator=g).cuda()
    return table, tokens, torch.arange(0, 4 * bags + 1, 4).cuda()


def alone(index, args):
    import torch
    torch.cuda.synchronize()
    got = index.search_tokens(*args, request())
    torch.cuda.synchronize()
    return got


def same(a, b):
    import torch
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_host_search_right_behind_search_tokens(index):
    import torch
    first = batch(1, 30_000)
    host = np.random.default_rng(2).normal(size=(5000, DIM)).astype(np.float32)
    want, want_host = alone(index, first), index.search(host, request())
    for stream in (None, torch.cuda.Stream()):
        for _ in range(3):
            with torch.cuda.stream(stream):
                got = index.search_tokens(*first, request())
                res = index.search(host, request())
            torch.cuda.synchronize()
            assert same(got, want)
            assert np.array_equal(res.ids, want_host.ids)
            assert np.array_equal(res.distances.view(np.uint32), want_host.distances.view(np.uint32))


def test_search_tokens_on_several_streams(index):
    import torch
    batches = [batch(s, n) for s, n in ((1, 30_000), (2, 9000), (3, 17))]
    want = [alone(index, b) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    for _ in range(4):
        got = []
        for s, b in zip(streams, batches):
            with torch.cuda.stream(s):
                got.append(index.search_tokens(*b, request()))
        got.append(index.search_tokens(*batches[1], request()))  # and on the default one
        torch.cuda.synchronize()
        assert all(same(g, w) for g, w in zip(got, want + [want[1]]))


def test_search_tokens_from_several_threads(index):
    import torch
    batches = [batch(s, 4000 + 1000 * s) for s in range(3)]
    want = [alone(index, b) for b in batches]
    wrong = []

    def many(i):
        with torch.cuda.stream(torch.cuda.Stream() if i else torch.cuda.default_stream()):
            for _ in range(8):
                got = index.search_tokens(*batches[i], request())
                torch.cuda.current_stream().synchronize()
                if not same(got, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=many, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_rows_added_behind_a_search_in_flight():
    import torch
    idx = make_index(8000)
    first = batch(1, 30_000)
    more = np.random.default_rng(3).normal(size=(6000, DIM)).astype(np.float32)
    before = alone(idx, first)
    with torch.cuda.stream(torch.cuda.Stream()):
        got = idx.search_tokens(*first, request())
        idx.add(more)
    torch.cuda.synchronize()
    assert same(got, before)
    fresh = make_index(8000)
    fresh.add(more)
    assert same(alone(idx, first), alone(fresh, first))


def test_prepared_search_and_rerank_behind_a_search_in_flight(index):
    """The device entry points beside search, on another stream."""
    import ctypes as C

    import torch
    from hanns_b200 import _lib as L
    lib, first, n = L.lib(), batch(1, 30_000), 700
    q = torch.randn(n, DIM, generator=torch.Generator().manual_seed(4)).cuda()
    rows = torch.randint(0, 20_000, (n, 9), generator=torch.Generator().manual_seed(5)).cuda()
    parts = np.zeros(5, np.int64)
    assert lib.hanns_gpu_ivf_usq_query_state_bytes(index._h, 32, parts.ctypes.data_as(L.i64p)) == 0
    want = alone(index, first)
    results = []
    for behind in (False, True):
        out = torch.zeros(n, 9, device="cuda")
        state = [torch.zeros(n * int(b), dtype=torch.uint8, device="cuda") for b in parts[:4]]
        torch.cuda.synchronize()
        if behind:
            got = index.search_tokens(*first, request())
        s = torch.cuda.Stream()
        assert lib.hanns_gpu_ivf_usq_rerank_rows_device(index._h, q.data_ptr(), n, rows.data_ptr(), 9, out.data_ptr(),
                                                        s.cuda_stream) == 0
        assert lib.hanns_gpu_ivf_usq_prepare_device(index._h, q.data_ptr(), n, 32, *[t.data_ptr() for t in state],
                                                    None, C.c_void_p(s.cuda_stream)) == 0
        torch.cuda.synchronize()
        results.append([out, *state])
    assert same(got, want)
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("own_stream", [False, True])
def test_an_index_freed_behind_a_search_in_flight(own_stream):
    import torch
    first = batch(1, 30_000)
    want = alone(make_index(8000), first)
    idx = make_index(8000)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if own_stream else None):
        got = idx.search_tokens(*first, request())
        idx.close()
    make_index(1000)  # takes what the index gave back
    torch.cuda.synchronize()
    assert same(got, want)


def test_searches_are_not_captured(index):
    import torch
    args = batch(1, 100)
    want = alone(index, args)
    queries, logits, t = torch.randn(4, DIM).cuda(), torch.zeros(4, 9).cuda(), torch.zeros(4, dtype=torch.long).cuda()
    for call in (lambda: index.search_tokens(*args, request()),
                 lambda: index.token_logprobs(queries, logits, t, t, request())):
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    torch.cuda.synchronize()
    assert same(index.search_tokens(*args, request()), want)

"""The workspace of the paged 4-bit cache's calls (include/holo_b200.h,
holo_kv4.work): the library's own, that of a Kv4Cache, and what else may run
beside or between the calls that use it."""
import ctypes as C
import threading
import time

import pytest
import torch

import holo_b200 as hb
from test_kv4_gpu import filled, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv4(dev):
    from holo_b200 import kv4
    return kv4


class Bare:
    """Calls of the C ABI on a cache without a workspace: the library's own is taken."""

    def __init__(self, kv4, cache):
        self.cache, self.lib = cache, hb.load()
        self.desc = kv4.Kv4Desc.from_buffer_copy(cache.desc)
        self.desc.work = None
        self.at = C.addressof(self.desc)

    def _stream(self):
        self.desc.stream = torch.cuda.current_stream().cuda_stream or 1   # 1: cudaStreamLegacy

    def attention(self, layer, q, out):
        self._stream()
        return self.lib.cuda_kv4_attention(self.at, layer, out.data_ptr(), q.data_ptr(), hb.DT_F32, 0, 0, q.shape[1], 0.0,
                                           None, q.shape[0])

    def extend(self, counts, start):
        self._stream()
        return self.lib.cuda_kv4_extend(self.at, None, counts.data_ptr(), start.data_ptr(), counts.numel())


def queries(n, heads, hd, seed):
    return torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(seed)).cuda()


def test_caches_of_different_shapes_share_the_librarys_workspace(kv4):
    """Caches of 672 counters and of a few, call after call on one stream: an extend and a split attention of small ones between the
    split attentions of the large one.  Each result is the one with a workspace of the cache's own."""
    big, _ = filled(kv4, [700 + 11 * i for i in range(40)], 8, 64, 16, 1, spare=0)
    small, _ = filled(kv4, [9000, 20], 1, 64, 16, 2)
    qb, qs = queries(40, 8, 64, 3), queries(2, 4, 64, 4)
    want_big, want_small = big.attention(0, qb), small.attention(0, qs)
    big_bare, small_bare = Bare(kv4, big), Bare(kv4, small)
    for rc in (small_bare.attention(0, qs, torch.empty_like(qs)), big_bare.attention(0, qb, torch.empty_like(qb))):
        assert rc == hb.HOLO_OK   # whatever the buffer has to grow by is there
    grown = kv4.Kv4Cache(1, 1, 64, 16, n_pages=1200, max_seqs=2, max_pages=1200)   # its extend lists 1000 pages in the plan
    grown_bare, counts, start = Bare(kv4, grown), ints(16000, 0), ints(0, 0)
    for i in range(3):
        out_s, out_b = torch.full_like(qs, 7.0), torch.full_like(qb, 7.0)
        assert small_bare.attention(0, qs, out_s) == hb.HOLO_OK
        assert grown_bare.extend(counts, start) == hb.HOLO_OK
        assert big_bare.attention(0, qb, out_b) == hb.HOLO_OK
        grown.release(ints(0))
        big.check()
        assert torch.equal(out_s, want_small), i
        assert torch.equal(out_b, want_big), i


def test_a_call_that_needs_more_workspace_inside_a_capture(kv4):
    """The library's own workspace is made, or grows, while the call's stream is being captured: the capture goes on, and its
    replays are right."""
    cache, _ = filled(kv4, [900, 30], 64, 64, 16, 6)
    wide = kv4.Kv4Cache(1, 64, 64, 16, pool=cache.pool, tables=torch.cat([cache.tables] * 1500).contiguous(),
                        lens=torch.cat([cache.lens] * 1500).contiguous(), refs=cache.refs)   # 768,000 counters
    q = queries(2, 64, 64, 7)
    want, bare, out = cache.attention(0, q), Bare(kv4, wide), torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rc = bare.attention(0, q, out)
    assert rc == hb.HOLO_OK
    for _ in range(3):
        out.fill_(7)
        graph.replay()
        wide.check()
        assert torch.equal(out, want)


def test_a_captured_call_outlives_the_growth_of_the_workspace(kv4):
    """A graph holds the library's own workspace as it was when it was captured; a later call that needs more leaves that alone."""
    cache, _ = filled(kv4, [3000, 30], 1, 64, 16, 8)
    q = queries(2, 4, 64, 9)
    want, bare, out = cache.attention(0, q), Bare(kv4, cache), torch.zeros_like(q)
    bare.attention(0, q, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bare.attention(0, q, out)
    many = kv4.Kv4Cache(1, 256, 64, 16, n_pages=40, max_seqs=4000, max_pages=40)   # 2,048,000 counters
    assert Bare(kv4, many).attention(0, queries(4000, 256, 64, 1), torch.empty(4000, 256, 64, device="cuda")) == hb.HOLO_OK
    taken = [torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda") for _ in range(40)]
    for _ in range(3):
        out.fill_(7)
        graph.replay()
        cache.check()
        assert torch.equal(out, want)
    assert all(bool((t == -1).all()) for t in taken)


def test_clearing_the_status_leaves_calls_under_way_alone(kv4):
    """cuda_clear_status while split attentions with the library's own workspace run on another stream."""
    cache, _ = filled(kv4, [60000, 7000], 1, 64, 64, 10)
    q = queries(2, 8, 64, 11)
    want, bare, side = cache.attention(0, q), Bare(kv4, cache), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty(8, *q.shape, device="cuda")
        for _ in range(400):
            out.fill_(7)
            for o in out:
                assert bare.attention(0, q, o) == hb.HOLO_OK
            bare.lib.cuda_clear_status()
            side.synchronize()
            assert all(torch.equal(o, want) for o in out)


def test_one_cache_on_several_streams(kv4):
    """Split attentions of one cache that run beside each other, each stream's with queries of its own, and a captured one among
    them: none takes another's counts or partial results."""
    cache, _ = filled(kv4, [60000, 7000], 1, 64, 64, 12)
    qs = [queries(2, 8, 64, 20 + i) for i in range(4)]
    want = [cache.attention(0, q) for q in qs]
    cache.check()
    outs = [torch.empty(30, *q.shape, device="cuda").fill_(7) for q in qs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for o in outs[3]:
            cache.attention(0, qs[3], o)
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(5):
        for o in outs:
            o.fill_(7)
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[3]):
            graph.replay()
        for i in range(30):
            for s, q, o in zip(streams[:3], qs, outs):
                with torch.cuda.stream(s):
                    cache.attention(0, q, o[i])
        torch.cuda.synchronize()
        cache.check()
        for o, w in zip(outs, want):
            assert all(torch.equal(x, w) for x in o)


def test_threads_with_streams_of_their_own(kv4):
    """A call takes the stream that is current in its thread, whatever another thread enters meanwhile."""
    cache, _ = filled(kv4, [100], 1, 64, 64, 12)
    meet, seen = threading.Barrier(2), {}

    def call(stream):
        def entered(at):   # in the library, without the interpreter's lock
            meet.wait(timeout=20)
            time.sleep(0.05)
            seen[stream.cuda_stream] = kv4.Kv4Desc.from_address(at).stream
            return hb.HOLO_OK
        with torch.cuda.stream(stream):
            cache._call("test", entered)

    streams = [torch.cuda.Stream() for _ in range(2)]
    threads = [threading.Thread(target=call, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == {s.cuda_stream: s.cuda_stream for s in streams}

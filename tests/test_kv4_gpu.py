"""The paged 4-bit cache (include/holo_b200.h, cuda_kv4_*): rows written and
read back, attention over it, and its page operations, against plain 64-bit
forms on the host (serving_reference.py)."""
import numpy as np
import pytest
import torch

import holo_b200 as hb
import serving_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def kv4(dev):
    from holo_b200 import kv4
    return kv4


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cu_of(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def filled(kv4, lens, n_kv, hd, page, seed, dtype=torch.float32, layers=1, spare=3, spread=1.0):
    """A cache with rows of normal values in pages of a shuffled order, and the values that it holds (64-bit, a sequence each)."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    cache = kv4.Kv4Cache(layers, n_kv, hd, page, sum(used) + spare, len(lens) + 2, max(used + [1]) + 1)
    order = torch.randperm(sum(used) + spare, generator=g).int()
    at = 0
    for i, n in enumerate(used):
        cache.tables[i, :n] = order[at:at + n].cuda()
        cache.refs[order[at:at + n].long().cuda()] = 1
        cache.lens[i] = lens[i]
        at += n
    total = sum(lens)
    held = []
    for layer in range(layers):
        k, v = (torch.randn(total, n_kv, hd, generator=g).mul(spread).to(dtype).cuda() for _ in range(2))
        cache.append(layer, k, v, cu_of(lens), torch.zeros(len(lens), dtype=torch.int32, device="cuda"))
        held.append([ref.values(*ref.quantise(x.float().cpu().numpy())) for x in (k, v)])
    cache.check()
    return cache, held


# ---- rows in and out ----

@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,lens", [(16, [1, 0, 33]), (48, [47, 100]), (64, [65, 3, 128])])
def test_append_places_codes_and_read_returns_them(kv4, hd, dtype, page, lens):
    """The pool's bytes are those of the format's description, and the rows read back are its values, exactly (their rounding to
    the rows' type included)."""
    n_kv, rng = 3, np.random.default_rng(hd + page)
    used = [-(-n // page) for n in lens]
    pages = rng.permutation(sum(used) + 2)
    cache = kv4.Kv4Cache(2, n_kv, hd, page, sum(used) + 2, len(lens), max(used) + 1)
    host, at = np.zeros(tuple(cache.pool.shape), np.uint8), 0
    rows = [torch.tensor(rng.standard_normal((sum(lens), n_kv, hd)), dtype=DTYPES[dtype]) for _ in range(2)]
    for x in rows:
        x[0, 0, :32] = 0.0                         # a group of zeros: scale 0
        x[-1, 1, 3], x[-1, 1, 9] = 4.0, -4.0       # equal magnitudes: the first gives the scale
        x[-1, 2, 40] *= 1000
    got = [ref.quantise(x.float().numpy()) for x in rows]
    for i, n in enumerate(used):
        mine = pages[at:at + n]
        cache.tables[i, :n] = torch.tensor(mine, dtype=torch.int32)
        at += n
        first = sum(lens[:i])
        for p in range(lens[i]):
            for h in range(n_kv):
                for side in (0, 1):
                    c, d = got[side]
                    ref.place(host, 1, mine[p // page], h, p % page, hd, side, c[first + p, h], d[first + p, h])
    start = torch.zeros(len(lens), dtype=torch.int32, device="cuda")
    k, v = (x.cuda() for x in rows)
    cache.append(1, k, v, cu_of(lens), start)
    assert np.array_equal(cache.pool.cpu().numpy(), host)
    kb, vb = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    cache.read(1, cu_of(lens), start, kb, vb)
    cache.check()
    for x, (c, d) in ((kb, got[0]), (vb, got[1])):
        assert torch.equal(x.cpu(), torch.tensor(ref.values(c, d)).to(DTYPES[dtype]))


def test_append_strided_unaligned_rows_in_the_middle(kv4):
    """Rows inside a wider matrix, one element off any wide alignment, appended at positions that start inside a block, to
    sequences out of order; a sequence with start -1 is left out."""
    n_kv, hd, page = 2, 64, 32
    cache = kv4.Kv4Cache(1, n_kv, hd, page, 8, 4, 3)
    cache.tables[3, :2] = ints(5, 2)
    cache.tables[1, :1] = ints(7)
    wide = torch.randn(12, 1 + 3 * n_kv * hd, device="cuda")
    k = wide[:, 1:1 + n_kv * hd].unflatten(1, (n_kv, hd))
    v = wide[:, 1 + n_kv * hd:1 + 2 * n_kv * hd].unflatten(1, (n_kv, hd))
    cu, start, seqs = ints(0, 7, 9, 12), ints(29, -1, 3), ints(3, 0, 1)
    cache.append(0, k, v, cu, start, seqs)
    kb, vb = torch.empty(12, n_kv, hd, device="cuda"), torch.empty(12, n_kv, hd, device="cuda")
    cache.read(0, cu, start, kb, vb, seqs)
    cache.check()
    for x, y in ((k, kb), (v, vb)):
        want = ref.values(*ref.quantise(x.cpu().numpy()))
        want[7:9] = 0.0
        assert np.array_equal(y.cpu().numpy(), want.astype(np.float32))
    pool = cache.pool.cpu().numpy()
    codes, scales = ref.quantise(v.cpu().numpy())
    assert np.array_equal(ref.fetch(pool, 0, 2, 1, 3, hd, 1), ref.values(codes, scales)[6, 1])   # position 35 of sequence 3
    touched = {(5, b) for b in (1,)} | {(2, 0), (7, 0)}
    for p in range(8):
        for b in range(2):
            assert pool[0, p, :, b].any() == ((p, b) in touched), (p, b)


def test_groups_with_nan_or_infinity_read_back_as_nan(kv4):
    cache = kv4.Kv4Cache(1, 1, 64, 16, 2, 1, 1)
    cache.tables[0, 0] = 1
    k = torch.randn(2, 1, 64, device="cuda")
    v = k.clone()
    k[0, 0, 5], v[1, 0, 60] = float("nan"), float("inf")
    cache.append(0, k, v, ints(0, 2), ints(0))
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    cache.read(0, ints(0, 2), ints(0), kb, vb)
    cache.check()
    assert kb[0, 0, :32].isnan().all() and not kb[0, 0, 32:].isnan().any() and not kb[1].isnan().any()
    assert vb[1, 0, 32:].isnan().all() and not vb[1, 0, :32].isnan().any() and not vb[0].isnan().any()


# ---- attention ----

def check_attention(kv4, lens, heads, n_kv, hd, page, dtype, seed, layers=1, scale=0.0, spread=1.0, qmul=1.0):
    cache, held = filled(kv4, lens, n_kv, hd, page, seed, layers=layers, spread=spread)
    layer = layers - 1
    q = (torch.randn(len(lens), heads, hd, generator=torch.Generator().manual_seed(seed + 1)) * qmul).to(DTYPES[dtype]).cuda()
    out = torch.full_like(q, 7.0)
    cache.attention(layer, q, out, scale=scale)
    again = cache.attention(layer, q, scale=scale)
    cache.check()
    assert torch.equal(out, again)   # nothing of a call is left for the next, and no order depends on timing
    y, qs, first = out.double().cpu().numpy(), q.double().cpu().numpy(), 0
    for i, n in enumerate(lens):
        for h in range(heads):
            k, v = (x[first:first + n, h // (heads // n_kv)] for x in held[layer])
            want, _ = ref.attend(qs[i, h:h + 1], k, v, scale or hd ** -0.5)
            tol = ref.bound(qs[i, h], k, v, scale or hd ** -0.5, dtype)
            assert np.abs(y[i, h] - want[0]).max() <= tol, (i, h, n)
        first += n


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd", [(4, 2, 64), (8, 1, 128), (7, 1, 128), (3, 3, 256), (32, 2, 128), (12, 1, 256)])
def test_attention_matches_formula(kv4, dtype, heads, n_kv, hd):
    check_attention(kv4, [1, 0, 16, 17, 31, 33, 64, 200], heads, n_kv, hd, 32, dtype, heads + hd)


@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_attention_page_sizes_and_layers(kv4, page):
    check_attention(kv4, [page - 1, page, page + 1, 5 * page + 7, 0], 8, 2, 128, page, "f16", page, layers=2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_long_and_ragged(kv4, dtype):
    """One long sequence split over many CTAs beside short ones."""
    check_attention(kv4, [9000, 1, 3, 500], 4, 1, 128, 64, dtype, 5)


@pytest.mark.parametrize("spread,qmul", [(1e-3, 1.0), (300.0, 0.01), (1.0, 1e4), (30.0, 30.0)])
def test_attention_scale_of_values(kv4, spread, qmul):
    """Small and large keys, values and queries: no step's range is left (sharp softmax weights at the large ones)."""
    check_attention(kv4, [700], 2, 2, 64, 64, "f32", 8, spread=spread, qmul=qmul)


def test_attention_reads_only_its_own_positions(kv4):
    """What lies past a sequence's end in its last page, and in pages that it does not hold, changes nothing: there are NaN scales there."""
    lens, hd, page = [37, 64, 0], 128, 64
    cache, _ = filled(kv4, lens, 2, hd, page, 3)
    q = torch.randn(3, 8, hd, device="cuda")
    want = cache.attention(0, q).clone()
    k = torch.randn(page - 37, 2, hd, device="cuda").fill_(float("nan"))
    cache.append(0, k, k, ints(0, page - 37), ints(37), ints(0))
    unheld = (cache.refs == 0).nonzero().view(-1)
    cache.pool[0, unheld] = 255
    got = cache.attention(0, q)
    cache.check()
    assert torch.equal(got, want) and not got[2].any()


def test_attention_nan_in_a_held_position_shows(kv4):
    cache, _ = filled(kv4, [40, 40], 1, 64, 64, 3)
    k = torch.zeros(1, 1, 64, device="cuda").fill_(float("nan"))
    cache.append(0, k, torch.zeros_like(k), ints(0, 1), ints(39), ints(0))
    out = cache.attention(0, torch.randn(2, 4, 64, device="cuda"))
    cache.check()
    assert out[0].isnan().all() and not out[1].isnan().any()


def test_attention_strides_lists_and_streams(kv4):
    """Queries inside a wider matrix, a list of sequences out of order, and a stream of one's own."""
    cache, held = filled(kv4, [20, 300, 5], 2, 64, 32, 11)
    wide = torch.randn(2, 3, 8, 64, device="cuda")
    q = wide[:, 1]
    want = cache.attention(0, torch.stack([wide[0, 1], wide[1, 1], wide[0, 1]])[[1, 0, 0]].contiguous())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.zeros(2, 2, 8, 64, device="cuda")
        cache.attention(0, q, out[:, 1], seqs=ints(1, 0))
    side.synchronize()
    cache.check()
    assert torch.equal(out[0, 1], want[1]) and torch.equal(out[1, 1], want[0]) and not out[:, 0].any()


def test_attention_offsets_past_32_bits(kv4):
    """Blocks that lie more than 4 GiB into a layer: the same pages at the start and at the end give the same result."""
    n_kv, hd, page = 8, 128, 64
    pages = (5 << 30) // (n_kv * page // 16 * 18 * hd)
    cache = kv4.Kv4Cache(1, n_kv, hd, page, pages, 2, 4)
    cache.tables[0], cache.tables[1] = ints(0, 1, 2, 3), ints(pages - 1, pages - 2, pages - 3, pages - 4)
    cache.lens[:] = 250
    x = torch.randn(2, 250, n_kv, hd, device="cuda")
    for i in range(2):
        cache.append(0, x[0], x[1], ints(0, 250), ints(0), ints(i))
    q = torch.randn(1, 8, hd, device="cuda").expand(2, 8, hd).contiguous()
    out = cache.attention(0, q)
    cache.check()
    assert torch.equal(out[0], out[1]) and out.abs().max() > 0


def test_attention_in_a_captured_graph(kv4):
    cache, _ = filled(kv4, [100, 3], 2, 128, 64, 2)
    q = torch.randn(2, 4, 128, device="cuda")
    want = cache.attention(0, q).clone()
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention(0, q, out)
    graph.replay()
    cache.check()
    assert torch.equal(out, want)


# ---- pages ----

class Model:
    """The page operations on the host, from their description."""

    def __init__(self, cache):
        self.page, self.tables, self.lens, self.refs = (cache.desc.page_tokens, cache.tables.cpu().numpy().copy(),
                                                        cache.lens.cpu().numpy().copy(), cache.refs.cpu().numpy().copy())
        self.pool = cache.pool.cpu().numpy().copy()

    def same(self, cache):
        cache.check()
        for name in ("tables", "lens", "refs", "pool"):
            assert np.array_equal(getattr(cache, name).cpu().numpy(), getattr(self, name)), name

    def extend(self, counts, seqs):
        start, out = [], False
        free = list(np.flatnonzero(self.refs == 0))
        taken = 0
        for s, c in zip(seqs, counts):
            need = -(-(self.lens[s] + c) // self.page) - -(-self.lens[s] // self.page)
            if self.lens[s] + c > self.page * self.tables.shape[1]:
                start.append(-1)
                continue
            taken += need
            if need and taken > len(free):
                start.append(-1)
                continue
            mine = free[taken - need:taken]
            first = -(-self.lens[s] // self.page)
            self.tables[s, first:first + need] = mine
            self.refs[mine] = 1
            start.append(self.lens[s])
            self.lens[s] += c
        return start

    def fork(self, parents, children):
        free = list(np.flatnonzero(self.refs == 0))
        taken = 0
        before = self.lens.copy()
        for p, k in zip(parents, children):
            full, part = divmod(before[p], self.page)
            if part:
                taken += 1
                if taken > len(free):
                    continue
                new = free[taken - 1]
                self.pool[:, new] = self.pool[:, self.tables[p, full]]
                self.refs[new] = 1
            self.tables[k] = -1
            self.tables[k, :full] = self.tables[p, :full]
            for e in self.tables[p, :full]:
                self.refs[e] += 1
            if part:
                self.tables[k, full] = new
            self.lens[k] = before[p]

    def release(self, seqs):
        for s in seqs:
            for e in self.tables[s, :-(-self.lens[s] // self.page)]:
                self.refs[e] -= 1
            self.tables[s], self.lens[s] = -1, 0

    def compact(self):
        live = int((self.refs > 0).sum())
        src = [p for p in range(live, len(self.refs)) if self.refs[p]]
        dst = [p for p in range(live) if not self.refs[p]]
        for s, d in zip(src, dst):
            self.pool[:, d] = self.pool[:, s]
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.tables[self.tables == s] = d


@pytest.mark.parametrize("page,layers,n_pages,seed", [(16, 1, 40, 0), (32, 3, 9, 1), (64, 2, 5000, 2), (48, 1, 9000, 3)])
def test_page_operations_match_description(kv4, page, layers, n_pages, seed):
    """Random runs of extend, fork, release and compact, against the host's; pools larger than one step of the plan among them."""
    rng = np.random.default_rng(seed)
    cache = kv4.Kv4Cache(layers, 1, 64, page, n_pages, 24, 12)
    cache.pool.random_(0, 256)
    model = Model(cache)
    for step in range(12):
        seqs = rng.permutation(24)[:rng.integers(1, 9)]
        counts = rng.integers(0, 3 * page, len(seqs))
        start = cache.extend(ints(*counts), ints(*seqs))
        want = model.extend(counts, seqs)
        assert start.tolist() == want
        cache.lib.cuda_clear_status()   # a full pool is part of the run
        if step % 2:
            held, empty = np.flatnonzero(model.lens), np.flatnonzero(model.lens == 0)
            n = min(3, len(held), len(empty))
            if n:
                parents, children = rng.choice(held, n), empty[:n]
                cache.fork(ints(*parents), ints(*children))
                model.fork(parents, children)
                cache.lib.cuda_clear_status()
        gone = rng.permutation(24)[:4]
        cache.release(ints(*gone))
        model.release(gone)
        model.same(cache)
        if step % 3 == 2:
            cache.compact()
            model.compact()
            model.same(cache)
            live = int((model.refs > 0).sum())
            assert (model.refs[live:] == 0).all()


def test_compact_moves_pages_of_the_whole_pool(kv4):
    """Every second page held: half of them move, in every layer, and the attention's result stays."""
    cache = kv4.Kv4Cache(3, 2, 64, 16, 600, 5, 100)
    held = torch.arange(1, 600, 2)
    cache.tables[:3] = held[:300].view(3, 100).int().cuda()
    cache.lens[:3] = 1600 - 5
    cache.refs[held.cuda()] = 1
    rows = torch.randn(2, 3 * 1595, 2, 64, device="cuda")
    for layer in range(3):
        cache.append(layer, rows[0] + layer, rows[1], ints(0, 1595, 3190, 4785), ints(0, 0, 0))
    model = Model(cache)
    q = torch.randn(3, 6, 64, device="cuda")
    before = [cache.attention(layer, q).clone() for layer in range(3)]
    cache.compact()
    model.compact()
    model.same(cache)
    for layer in range(3):
        assert torch.equal(cache.attention(layer, q), before[layer])


def test_copy_pages_in_every_layer(kv4):
    cache = kv4.Kv4Cache(4, 2, 128, 32, 20, 1, 1)
    cache.pool.random_(0, 256)
    want = cache.pool.clone()
    src, dst = ints(3, 19, 3), ints(0, 7, 12)
    want[:, dst.long()] = want[:, src.long()]
    cache.copy_pages(src, dst)
    cache.check()
    assert torch.equal(cache.pool, want)


# ---- refusals ----

def test_refusals(kv4):
    from holo_b200.kv4 import Kv4Cache
    with pytest.raises(ValueError):
        Kv4Cache(1, 1, 96, 16, 2, 1, 1)
    with pytest.raises(ValueError):
        Kv4Cache(1, 1, 64, 24, 2, 1, 1)
    cache = Kv4Cache(1, 2, 64, 16, 4, 2, 2)
    q = torch.zeros(2, 4, 64, device="cuda")
    with pytest.raises(ValueError):
        cache.attention(0, torch.zeros(2, 4, 128, device="cuda"))
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        cache.attention(1, q)                                       # no such layer
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        cache.attention(0, torch.zeros(2, 3, 64, device="cuda"))    # 3 heads over 2
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_UNSUPPORTED)):
        cache.attention(0, torch.zeros(2, 34, 64, device="cuda"))   # 17 heads a KV head
    with pytest.raises(TypeError):
        cache.attention(0, q.double())
    with pytest.raises(ValueError):
        cache.attention(0, q.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError):
        cache.attention(0, q.cpu())
    k = torch.zeros(3, 2, 64, device="cuda")
    with pytest.raises(TypeError):
        cache.append(0, k, k.half(), ints(0, 3), ints(0))
    with pytest.raises(ValueError):
        cache.append(0, k.expand(3, 2, 64)[:1].expand(3, 2, 64), k, ints(0, 3), ints(0))
    with pytest.raises(TypeError):
        cache.release(torch.tensor([0], device="cuda"))
    bare = Kv4Cache(1, 2, 64, 16, pool=cache.pool, tables=cache.tables, lens=cache.lens)
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        bare.compact()                                              # no refs
    cache.check()


def test_kernels_report_what_they_leave_out(kv4):
    """No free page, and numbers out of range: recorded, and nothing outside is touched."""
    cache = kv4.Kv4Cache(1, 1, 64, 16, 2, 3, 4)
    start = cache.extend(ints(16, 40), ints(0, 1))
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_NOMEM)):
        cache.check()
    assert start.tolist() == [0, -1] and cache.lens.tolist() == [16, 0, 0] and cache.refs.tolist() == [1, 0]
    before = cache.pool.clone()
    cache.tables[2, 0] = 99
    k = torch.ones(1, 1, 64, device="cuda")
    for seqs, row in ((ints(7), ints(0)), (ints(2), ints(0)), (ints(0), ints(1000))):
        cache.append(0, k, k, ints(0, 1), row, seqs)
        with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
            cache.check()
    cache.copy_pages(ints(0), ints(5))
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        cache.check()
    cache.release(ints(-1))
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        cache.check()
    assert torch.equal(cache.pool, before)


def test_vectors_of_another_device_are_refused(kv4):
    cache = kv4.Kv4Cache(1, 1, 64, 16, 4, 2, 2)
    host, here = torch.ones(1, dtype=torch.int32), ints(1)
    x = torch.zeros(1, 1, 64, device="cuda")
    for call in (lambda: cache.extend(host), lambda: cache.extend(here, start=host), lambda: cache.append(0, x, x, cu_of([1]), host),
                 lambda: cache.append(0, x, x, cu_of([1]).cpu(), here), lambda: cache.append(0, x.cpu(), x, cu_of([1]), here),
                 lambda: cache.attention(0, x.cpu()), lambda: cache.attention(0, x, out=x.cpu())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cache.extend(here, host), lambda: cache.fork(host, here), lambda: cache.release(host),
                 lambda: cache.copy_pages(here, host)):
        with pytest.raises(TypeError):
            call()
    cache.check()
    assert cache.lens.tolist() == [0, 0]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_rows_at_odd_addresses(kv4, dtype, hd):
    """Rows that no wide load or store takes give the same bits."""
    cache, _ = filled(kv4, [70, 1, 0, 600], 2, hd, 32, 21)
    q = torch.randn(4, 6, hd, generator=torch.Generator().manual_seed(2)).to(DTYPES[dtype]).cuda()
    want = cache.attention(0, q)
    wide_q, wide_o = (torch.zeros(4, 6 * hd + 3, dtype=q.dtype, device="cuda") for _ in range(2))
    wide_q[:, 1:-2] = q.flatten(1)
    cache.attention(0, wide_q[:, 1:-2].unflatten(1, (6, hd)), wide_o[:, 1:-2].unflatten(1, (6, hd)))
    cache.check()
    assert torch.equal(wide_o[:, 1:-2].unflatten(1, (6, hd)), want)
    assert not wide_o[:, 0].any() and not wide_o[:, -2:].any()


def test_attention_of_many_sequences(kv4):
    """More sequences than a CTA has threads, several a CTA, empty ones among them: each as it comes out alone (none is long
    enough to be cut)."""
    lens = np.random.default_rng(4).integers(0, 512, 300)
    lens[[0, 7, 150, 298, 299]] = 0, 512, 1, 0, 64
    cache, held = filled(kv4, lens.tolist(), 2, 64, 64, 31)
    q = torch.randn(300, 6, 64, generator=torch.Generator().manual_seed(9)).cuda()
    got = cache.attention(0, q).clone()
    for i in (0, 7, 8, 127, 128, 150, 255, 256, 298, 299):
        alone = cache.attention(0, q[i:i + 1], seqs=ints(i))
        assert torch.equal(alone[0], got[i]), i
    turned = torch.arange(299, -1, -1, dtype=torch.int32, device="cuda")
    assert torch.equal(cache.attention(0, q.flip(0), seqs=turned).flip(0), got)
    cache.check()
    assert torch.equal(got.flatten(1).any(1).cpu(), torch.tensor(lens > 0))


@pytest.mark.parametrize("lens,heads,n_kv,hd", [([33], 4, 2, 64), ([2047, 100], 4, 4, 128), ([20000], 8, 1, 128), ([900], 12, 1, 256)])
def test_attention_of_fp32_rows_keeps_fp32(kv4, lens, heads, n_kv, hd):
    """The norm of the error against 64 bits.  q and the weights are held to 2^-22, and so is a block's sum in the tensor core (16
    positions, cut to 24 bits at up to four times the result); scores of size s, here up to about 5, are off by s 2^-22, and a
    weight by as much; fp32's own roundings are half of each.  Each enters once a position, independently: no more than the sum
    of their sizes relative to the result, (1 + 1 + 1 + 5 / 2) 2^-22 = 1.3e-6.  (fp16 weights would leave 1e-4.)"""
    cache, held = filled(kv4, lens, n_kv, hd, 64, 41)
    q = torch.randn(len(lens), heads, hd, generator=torch.Generator().manual_seed(43)).cuda()
    y, qs, first = cache.attention(0, q).double().cpu().numpy(), q.double().cpu().numpy(), 0
    cache.check()
    for i, n in enumerate(lens):
        want = np.stack([ref.attend(qs[i, h:h + 1], *(x[first:first + n, h * n_kv // heads] for x in held[0]), hd ** -0.5)[0][0]
                         for h in range(heads)])
        assert np.linalg.norm(y[i] - want) <= 1.3e-6 * np.linalg.norm(want), i
        first += n


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_zero_queries_and_a_small_scale(kv4, dtype):
    """Scores of 0, whatever the scale: the mean of the values, also where a unit's last positions are masked."""
    cache, held = filled(kv4, [37, 1], 2, 64, 64, 51)
    q = torch.zeros(2, 4, 64, dtype=DTYPES[dtype], device="cuda")
    for scale in (0.0, 1e-10, 1e-30):
        y = cache.attention(0, q, scale=scale).double().cpu().numpy()
        for i, (a, n) in enumerate(((0, 37), (37, 1))):
            v = held[0][1][a:a + n]
            tol = ref.bound(np.zeros((1, 64)), held[0][0][a:a + n, 0], v, 1.0, dtype)
            assert np.abs(y[i] - v.mean(0).repeat(2, 0)).max() <= tol
    cache.check()


@pytest.mark.parametrize("dtype,hd", [("f32", 64), ("f16", 128), ("bf16", 256)])
def test_attention_of_many_short_sequences(kv4, dtype, hd):
    """All of one unit of work or empty: several items a CTA, a warp each, as an item comes out that a CTA has to itself, and as the
    formula has it."""
    lens = np.random.default_rng(6).integers(0, 65, 300)
    lens[[0, 7, 150, 298, 299]] = 0, 64, 1, 0, 64
    cache, held = filled(kv4, lens.tolist(), 4, hd, 16, 61)
    q = torch.randn(300, 12, hd, generator=torch.Generator().manual_seed(8)).to(DTYPES[dtype]).cuda()
    got = cache.attention(0, q).clone()
    ends = np.cumsum(lens)
    for i in (0, 7, 8, 127, 128, 150, 255, 256, 298, 299):
        assert torch.equal(cache.attention(0, q[i:i + 1], seqs=ints(i))[0], got[i]), i
        k, v = (x[ends[i] - lens[i]:ends[i]] for x in held[0])
        for h in range(12):
            qh = q[i, h:h + 1].double().cpu().numpy()
            want, _ = ref.attend(qh, k[:, h // 3], v[:, h // 3], hd ** -0.5)
            tol = ref.bound(qh, k[:, h // 3], v[:, h // 3], hd ** -0.5, dtype)
            assert np.abs(got[i, h].double().cpu().numpy() - want[0]).max() <= tol, (i, h)
    cache.check()
    assert torch.equal(got.flatten(1).any(1).cpu(), torch.tensor(lens > 0))


# ---- entries of a table that name no page ----

@pytest.mark.parametrize("entry", [-1, 10 ** 6, -2 ** 31])
@pytest.mark.parametrize("lens,heads,n_kv,hd,dtype", [
    ([40, 64, 3, 0], 4, 2, 64, "f32"),               # an item each
    ([30] * 500, 4, 2, 64, "f16"),                   # a warp takes several items
    ([900, 5000, 200, 7], 16, 1, 128, "bf16"),       # split over CTAs
    ([300, 1200, 40], 3, 3, 256, "f32")])
def test_attention_over_an_entry_that_names_no_page(kv4, lens, heads, n_kv, hd, dtype, entry):
    """The sequence is left out: zeros, and not the values of another page.  The others are as they were, and so is the next call."""
    cache, _ = filled(kv4, lens, n_kv, hd, 32, 71)
    q = torch.randn(len(lens), heads, hd, generator=torch.Generator().manual_seed(72)).to(DTYPES[dtype]).cuda()
    want = cache.attention(0, q).clone()
    held = cache.tables[1].clone()
    for col in {0, (lens[1] - 1) // 32}:
        cache.tables[1, col] = entry
        out = cache.attention(0, q, torch.full_like(q, 7.0))
        with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
            cache.check()
        assert not out[1].any()
        rest = torch.arange(len(lens)) != 1
        assert torch.equal(out[rest], want[rest])
        cache.tables[1] = held
    cache.tables[1, -1] = entry                      # past the sequence's pages: nobody's concern
    assert torch.equal(cache.attention(0, q), want)
    cache.check()


def test_attention_over_missing_pages_among_short_and_long_sequences(kv4):
    """Runs of one-unit items, of which only one warp has anything, before long ones whose first loads are under way meanwhile:
    every second long sequence lacks its last page, and no other one comes out otherwise for it."""
    lens = ([20] * 40 + [450]) * 16
    cache, _ = filled(kv4, lens, 2, 64, 32, 73)
    q = torch.randn(len(lens), 4, 64, generator=torch.Generator().manual_seed(74)).cuda()
    want = cache.attention(0, q).clone()
    gone = torch.arange(40, len(lens), 82)
    cache.tables[gone.cuda(), 449 // 32] = -1
    out = cache.attention(0, q)
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        cache.check()
    want[gone.cuda()] = 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("layers", [2, 600])   # one launch; a plan and a grid
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_fork_of_a_parent_that_lacks_a_page(kv4, layers, entry):
    """Its child stays empty and no page is taken for it; the other children are forked."""
    cache, _ = filled(kv4, [100, 70, 33, 0, 0, 0], 1, 64, 32, 81, layers=1)
    cache = kv4.Kv4Cache(layers, 1, 64, 32, pool=cache.pool.expand(layers, -1, -1, -1, -1).contiguous(), tables=cache.tables,
                         lens=cache.lens, refs=cache.refs)
    for col in (0, 2):                            # a whole page of the second parent, its last one
        held = cache.tables[1].clone()
        cache.tables[1, col] = entry
        model = Model(cache)
        cache.fork(ints(0, 1, 2), ints(3, 4, 5))
        with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
            cache.check()
        model.fork([0, 2], [3, 5])
        model.same(cache)
        cache.tables[1] = held
        cache.release(ints(3, 4, 5))


def test_extend_and_fork_of_more_sequences_than_a_step_of_the_plan(kv4):
    """2500 sequences: the sums over the list go on from step to step, up to the last free page."""
    rng = np.random.default_rng(7)
    counts = rng.integers(0, 70, 2500)
    need = int((-(-counts // 16)).sum())
    cache = kv4.Kv4Cache(1, 1, 64, 16, need + 900, 5000, 6)
    cache.pool.random_(0, 256)
    model = Model(cache)
    seqs = rng.permutation(5000)[:2500]
    start = cache.extend(ints(*counts), ints(*seqs))
    assert start.tolist() == model.extend(counts, seqs)
    model.same(cache)
    empty = np.flatnonzero(model.lens == 0)
    parents = rng.choice(np.flatnonzero(model.lens), 2400)   # (no parent is a child)
    cache.fork(ints(*parents), ints(*empty[:2400]))
    model.fork(parents, empty[:2400])
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_NOMEM)):   # more last pages than are free
        cache.check()
    model.same(cache)
    more = rng.integers(0, 30, 3000)
    cache.release(ints(*range(0, 2000)))
    model.release(range(0, 2000))
    assert cache.extend(ints(*more), ints(*range(1000, 4000))).tolist() == model.extend(more, range(1000, 4000))
    cache.lib.cuda_clear_status()
    model.same(cache)


@pytest.mark.parametrize("length", [-1, -2 ** 31, 3 * 16 + 1, 2 ** 31 - 1])
def test_lengths_that_the_tables_cannot_hold(kv4, length):
    """A length that is negative or past the table's columns is recorded and followed nowhere: the sequence is left as it is, and the
    others in the call are served."""
    cache = kv4.Kv4Cache(2, 1, 64, 16, 40, 6, 3)
    cache.extend(ints(20, 20, 20))
    cache.check()
    cache.lens[1] = length
    before = [x.clone() for x in (cache.tables, cache.refs, cache.lens, cache.pool)]
    start = cache.extend(ints(1, 1), ints(1, 2))
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        cache.check()
    assert start.tolist() == [-1, 20]
    before[2][2] = 21
    model = Model(cache)
    cache.fork(ints(1, 0), ints(3, 4))
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        cache.check()
    model.fork([0], [4])
    model.same(cache)
    cache.release(ints(1, 4))
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        cache.check()
    model.release([4])
    model.same(cache)
    for x, y in zip((cache.tables, cache.refs, cache.lens), before):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("side", [0, 1])
def test_values_too_large_for_their_scale(kv4, dtype, side):
    """A group whose largest value is past 8 times fp16's largest has no scale: it reads back as NaN, and a sequence that holds it
    attends to NaN, whichever way its products would round.  The largest that has one (524,159 rounds to 8 * 65,504) is a value."""
    cache, held = filled(kv4, [50, 40, 30], 1, 64, 32, 91)
    g = torch.Generator().manual_seed(92)          # small components among large ones: sums that are not exact
    q = (torch.randn(3, 16, 64, generator=g) * 10 ** (-4 * torch.rand(3, 16, 64, generator=g))).to(DTYPES[dtype]).cuda()
    want = cache.attention(0, q).clone()
    x = [torch.randn(1, 1, 64, generator=torch.Generator().manual_seed(93 + s)).cuda() for s in range(2)]
    back = [torch.empty_like(y) for y in x]
    for value, fits in ((524159.0, True), (524160.0, False), (-6e5, False), (3e38, False)):
        x[side][0, 0, 40] = value
        cache.append(0, *x, ints(0, 1), ints(49), ints(0))
        cache.read(0, ints(0, 1), ints(49), *back, ints(0))
        got = cache.attention(0, q)
        cache.check()
        assert back[side][0, 0, 32:].isnan().all() != fits and back[side][0, 0, 32:].isfinite().all() == fits
        assert back[side][0, 0, :32].isfinite().all() and back[1 - side].isfinite().all()
        assert torch.equal(got[1:], want[1:])
        if not fits:
            assert got[0].isnan().all() if side == 0 else (got[0, :, 32:].isnan().all() and got[0, :, :32].isfinite().all())


def test_a_cache_over_tensors_that_do_not_make_one(kv4):
    """A pool without its tables or lengths, and tensors of other shapes and types, are refused by name."""
    pool = torch.zeros(1, 4, 2, 1, 18 * 64, dtype=torch.uint8, device="cuda")
    tables, lens = torch.full((3, 2), -1, dtype=torch.int32, device="cuda"), ints(0, 0, 0)
    good = dict(pool=pool, tables=tables, lens=lens, refs=ints(0, 0, 0, 0))
    kv4.Kv4Cache(1, 2, 64, 16, **good)
    for change in (dict(tables=None), dict(lens=None), dict(tables=tables[0]), dict(tables=tables.long()), dict(tables=tables.t()),
                   dict(lens=lens[:2]), dict(lens=lens.float()), dict(refs=ints(0, 0)), dict(pool=pool.view(-1)),
                   dict(pool=pool.view(torch.int8)), dict(tables=[[0, 1]]), dict(pool=None), dict(pool=None, tables=None)):
        with pytest.raises(TypeError, match="Kv4Cache"):
            kv4.Kv4Cache(1, 2, 64, 16, **(good | change))
    for change in (dict(tables=tables.cpu()), dict(lens=lens.cpu()), dict(refs=good["refs"].cpu())):
        with pytest.raises(ValueError, match="Kv4Cache"):
            kv4.Kv4Cache(1, 2, 64, 16, **(good | change))

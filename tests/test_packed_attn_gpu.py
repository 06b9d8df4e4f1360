"""Attention over packed prompts (include/holo_b200.h, cuda_attention_packed)
against the formula in 64 bits (serving_reference.py)."""
import numpy as np
import pytest
import torch

import holo_b200 as hb
import serving_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def packed(dev):
    from holo_b200.attention import attention_packed
    return attention_packed


def cu_of(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def rows(lens, heads, n_kv, hd, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(sum(lens), h, hd, generator=g) * m).to(DTYPES[dtype]).cuda()
            for h, m in ((heads, spread), (n_kv, spread), (n_kv, 1.0))]


def check(packed, lens, heads, n_kv, hd, dtype, seed, scale=0.0, spread=1.0, some=None):
    q, k, v = rows(lens, heads, n_kv, hd, dtype, seed, spread)
    out, lse = torch.full_like(q, 9.0), torch.full((heads, sum(lens)), 9.0, device="cuda")
    packed(q, k, v, cu_of(lens), out, lse, scale)
    assert torch.equal(packed(q, k, v, cu_of(lens), scale=scale), out)
    torch.cuda.synchronize()
    y, qs, ks, vs = (x.double().cpu().numpy() for x in (out, q, k, v))
    sc, ls = scale or hd ** -0.5, lse.double().cpu().numpy()
    for h in some or range(heads):
        a = 0
        for n in lens:
            kh, vh, qh = ks[a:a + n, h * n_kv // heads], vs[a:a + n, h * n_kv // heads], qs[a:a + n, h]
            if n:
                want, sums = ref.attend(qh, kh, vh, sc, causal=True)
                assert np.abs(y[a:a + n, h] - want).max() <= ref.bound(qh, kh, vh, sc, dtype), (h, n)
                # scores off by s, the sum of n exps by (n + 8) 2^-23
                s = hd * 2.0 ** -22 * np.abs(qh).max() * np.abs(kh).max() * sc
                assert np.abs(ls[h, a:a + n] - sums).max() <= 2 * s + (n + 8) * 2.0 ** -23 + 2.0 ** -22 * np.abs(sums).max()
            a += n


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd", [(4, 2, 64), (3, 1, 128), (2, 2, 256), (8, 1, 128)])
def test_matches_formula(packed, dtype, heads, n_kv, hd):
    """Lengths about the tiles' edges, empty sequences first, between and last."""
    check(packed, [0, 1, 127, 128, 0, 129, 3, 255, 256, 257, 0], heads, n_kv, hd, dtype, heads + hd)


@pytest.mark.parametrize("hd", [64, 128])
def test_long_sequence(packed, hd):
    check(packed, [1500, 77], 2, 1, hd, "bf16", 4)


def test_many_short_sequences(packed):
    lens = list(np.random.default_rng(0).integers(0, 20, 300))
    check(packed, lens, 4, 1, 64, "f16", 5, some=[0, 3])


@pytest.mark.parametrize("spread,scale", [(1.0, 0.5), (6.0, 0.0), (1e-3, 0.0)])
def test_scales(packed, spread, scale):
    """Sharp softmax weights, flat ones, and a scale of one's own."""
    check(packed, [300, 40], 2, 1, 128, "f16", 6, scale=scale, spread=spread)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_in_masked_places_change_nothing(packed, hd, bad):
    """A sequence whose keys and values are not finite leaves its neighbours alone, and a token that is not finite leaves the
    earlier ones of its own sequence alone; those after it show it."""
    lens = [70, 90, 130]
    q, k, v = rows(lens, 4, 2, hd, "f16", 7)
    cu = cu_of(lens)
    want = packed(q, k, v, cu).clone()
    k[75:160], v[75:160] = bad, bad        # from token 5 of the second sequence on
    got = packed(q, k, v, cu)
    assert torch.equal(got[:75], want[:75]) and torch.equal(got[160:], want[160:])
    assert got[75:160].isnan().all()


@pytest.mark.parametrize("n", [390, 520, 650, 1300])
def test_values_in_masked_places_of_a_long_sequence(packed, n):
    """The same at the end of a sequence of several key tiles, whichever place in the load ring its last tile has; and repeated
    calls over memory that other values have been in agree."""
    q, k, v = rows([n, 200], 2, 1, 128, "bf16", n)
    cu = cu_of([n, 200])
    want = packed(q, k, v, cu).clone()
    k2, v2 = k.clone(), v.clone()
    v2[n:], k2[n:] = float("nan"), float("nan")
    v2[n - 20:n], k2[n - 20:n] = float("inf"), float("nan")
    for _ in range(3):
        got = packed(q, k2, v2, cu)
        assert torch.equal(got[:n - 20], want[:n - 20]) and got[n - 20:].isnan().all()
        assert torch.equal(packed(q, k, v, cu), want)


@pytest.mark.parametrize("lens", [[64, 65, 1, 192], [1500, 77]])
def test_wide_heads(packed, lens):
    """Head size 256: its key tiles of 64, their edges, and many of them."""
    check(packed, lens, 4, 2, 256, "bf16", 11, spread=2.0)


@pytest.mark.parametrize("n", [60, 130, 321, 700])
def test_values_in_masked_places_of_wide_heads(packed, n):
    q, k, v = rows([n, 200], 2, 1, 256, "f16", n)
    cu = cu_of([n, 200])
    want = packed(q, k, v, cu).clone()
    k2, v2 = k.clone(), v.clone()
    v2[n:], k2[n:] = float("nan"), float("nan")
    v2[n - 20:n], k2[n - 20:n] = float("inf"), float("nan")
    for _ in range(3):
        got = packed(q, k2, v2, cu)
        assert torch.equal(got[:n - 20], want[:n - 20]) and got[n - 20:].isnan().all()
        assert torch.equal(packed(q, k, v, cu), want)


def test_strides(packed):
    """q, k and v as columns of one matrix of rows, heads before rows, and an odd offset that no wide load takes."""
    lens, heads, n_kv, hd = [130, 30], 4, 2, 64
    total = sum(lens)
    q, k, v = rows(lens, heads, n_kv, hd, "f16", 8)
    want = packed(q, k, v, cu_of(lens))
    both = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    cut = [x.unflatten(1, (-1, hd)) for x in both.split([heads * hd, n_kv * hd, n_kv * hd], 1)]
    assert torch.equal(packed(*cut, cu_of(lens)), want)
    turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    out = torch.empty(heads, total, hd, dtype=q.dtype, device="cuda").transpose(0, 1)
    assert torch.equal(packed(*turned, cu_of(lens), out=out), want)
    odd = torch.zeros(total, 1 + both.shape[1], dtype=both.dtype, device="cuda")
    odd[:, 1:] = both
    cut = [x.unflatten(1, (-1, hd)) for x in odd[:, 1:].split([heads * hd, n_kv * hd, n_kv * hd], 1)]
    got = packed(*cut, cu_of(lens))
    tol = ref.bound(*(x.double().cpu().numpy().reshape(-1, hd) for x in (q, k, v)), hd ** -0.5, "f16")
    assert (got.double() - want.double()).abs().max() <= 2 * tol


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [128, 256])
def test_rows_at_odd_addresses(packed, dtype, hd):
    """Rows that no wide load takes, each of q, k and v and out, and their log-sum-exp: within both kernels' bounds of each other."""
    lens, heads, n_kv = [66, 0, 1, 130], 4, 2
    q, k, v = rows(lens, heads, n_kv, hd, dtype, 12)
    cu, total = cu_of(lens), sum(lens)
    lse = [torch.zeros(heads, total, device="cuda") for _ in range(2)]
    want = packed(q, k, v, cu, lse=lse[0])

    def odd(x):
        wide = torch.zeros(total, x.shape[1] * hd + 3, dtype=x.dtype, device="cuda")
        wide[:, 1:-2] = x.flatten(1)
        return wide[:, 1:-2].unflatten(1, (-1, hd))

    tol = 2 * ref.bound(*(x.double().cpu().numpy().reshape(-1, hd) for x in (q, k, v)), hd ** -0.5, dtype)
    for case in ((odd(q), k, v, None), (q, odd(k), odd(v), None), (q, k, v, odd(torch.zeros_like(q)))):
        got = packed(*case[:3], cu, out=case[3], lse=lse[1])
        assert (got.double() - want.double()).abs().max() <= tol
        assert (lse[0] - lse[1]).abs().max() <= 1e-4   # scores of up to about 6, sums of hd products rounded at random: 6 sqrt(hd) 2^-22 on both sides, and twice that


def test_rows_outside_the_sequences_keep_their_memory(packed):
    """cu_seqlens that does not reach the last rows: no more than those rows' results may change."""
    q, k, v = rows([200], 2, 1, 64, "f16", 9)
    want = packed(q, k, v, cu_of([200]))
    out = torch.zeros_like(q)
    packed(q, k, v, cu_of([150]), out=out)
    assert torch.equal(out[:150], want[:150])


def test_streams_and_graphs(packed):
    q, k, v = rows([300, 20], 2, 1, 128, "bf16", 10)
    cu = cu_of([300, 20])
    want = packed(q, k, v, cu).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = packed(q, k, v, cu)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed(q, k, v, cu, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_refusals(packed):
    q, k, v = rows([10], 4, 2, 64, "f16", 1)
    cu = cu_of([10])
    with pytest.raises(TypeError):
        packed(q.float(), k.float(), v, cu)
    with pytest.raises(TypeError):
        packed(q, k, v.bfloat16(), cu)
    with pytest.raises(TypeError):
        packed(q, k, v, cu.long())
    with pytest.raises(ValueError):
        packed(q, k[:9], v[:9], cu)
    with pytest.raises(ValueError):
        packed(q, k, v.transpose(1, 2).contiguous().transpose(1, 2), cu)
    with pytest.raises(ValueError):
        packed(q, k[:1].expand_as(k), v, cu)
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_UNSUPPORTED)):
        packed(q.float(), k.float(), v.float(), cu)
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_UNSUPPORTED)):
        packed(q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), cu)
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        packed(q[:, :3], k, v, cu)
    with pytest.raises(RuntimeError, match=str(hb.HOLO_E_ARG)):
        packed(q, k, v, cu, scale=-1.0)
    assert packed(q[:0], k[:0], v[:0], cu_of([0])).shape == (0, 4, 64)


def microseconds(call):
    for _ in range(2):
        call()
    times = []
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return min(times)


@pytest.mark.parametrize("n,heads,n_kv,hd,dtype", [
    (4096, 2, 1, 128, "f16"), (3000, 2, 2, 64, "bf16"), (2100, 1, 1, 256, "f16"), (40000, 2, 1, 128, "bf16")])
def test_values_that_rows_see(packed, n, heads, n_kv, hd, dtype):
    """Values of v that are not finite, in an early token, in a later one and in the last tiles: the rows before them are what they
    would be without, those from them on have them in the one dim that they are in, and no call is a multiple slower than the
    walk over V that looks for them and a second pass cost (a few times the call without)."""
    q, k, v = rows([n, 100], heads, n_kv, hd, dtype, 13)
    cu = cu_of([n, 100])
    places = [(5, 3, float("nan")), (17, 10, float("inf")), (n // 2, 10, -float("inf")), (n - 300, 33, -float("inf")),
              (n - 3, 40, float("inf")), (n - 1, 63, float("nan"))]
    clean, bad = v.clone(), v.clone()
    for i, d, x in places:
        clean[i, 0, d], bad[i, 0, d] = 0, x
    want, lse = packed(q, k, clean, cu, lse=(a := torch.empty(heads, n + 100, device="cuda"))), a
    lse2 = torch.empty_like(lse)
    got = packed(q, k, bad, cu, lse=lse2)
    assert hb.load().cuda_last_status() == hb.HOLO_OK
    add = torch.zeros(n + 100, hd, device="cuda")
    for i, d, x in places:
        add[i:n, d] += x
    want = want.float()
    want[:, :heads // n_kv] += add[:, None]
    g, finite = got.float(), want.isfinite()
    assert torch.equal(g.isnan(), want.isnan()) and torch.equal(g[want.isinf()], want[want.isinf()])
    tol = 2 * ref.bound(*(x.double().cpu().numpy().reshape(-1, hd) for x in (q, k, clean)), hd ** -0.5, dtype)
    assert (g - want)[finite].abs().max() <= tol
    assert (lse - lse2).abs().max() <= 1e-4
    assert microseconds(lambda: packed(q, k, bad, cu)) <= 20 * microseconds(lambda: packed(q, k, clean, cu))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_large_bfloat16_values_do_not_overflow(packed, hd):
    """Values near the type's largest: their weighted sums before the division pass fp32's range, the rows do not.  Scores that
    rise along the keys, so that the weights before the division are large."""
    lens, heads = [700, 3], 2
    q, k, v = rows(lens, heads, 1, hd, "bf16", 14)
    q.fill_(1)
    k[:] = (torch.arange(703, device="cuda")[:, None, None] / 703 * 6 * hd ** -0.5).to(k.dtype)
    v = (v.float() * 2.0 ** 120).bfloat16()
    got = packed(q, k, v, cu_of(lens))
    small = packed(q, k, (v.float() * 2.0 ** -100).bfloat16(), cu_of(lens))
    assert hb.load().cuda_last_status() == hb.HOLO_OK and got.isfinite().all()
    assert torch.equal((got.float() * 2.0 ** -100).bfloat16(), small)
    v[600, 0, 1] = float("nan")
    bad = packed(q, k, v, cu_of(lens))
    assert bad[600:700, :, 1].isnan().all() and bad[:600].isfinite().all() and bad[700:].isfinite().all()
    got[600:700, :, 1] = bad[600:700, :, 1] = 0
    assert torch.equal(got, bad)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rows_outside_the_sequences_are_not_written(packed, hd):
    """A cu_seqlens that ends before the rows do, at every place in a tile: out and lse past it keep what they hold, of rows that
    TMA takes and of rows at odd addresses."""
    q, k, v = rows([300], 2, 1, hd, "f16", 15)
    want, odd = packed(q, k, v, cu_of([300])), torch.zeros(300, 2 * hd + 1, dtype=q.dtype, device="cuda")
    odd[:, 1:] = q.flatten(1)
    tol = 2 * ref.bound(*(x.double().cpu().numpy().reshape(-1, hd) for x in (q, k, v)), hd ** -0.5, "f16")
    for end in (1, 127, 128, 150, 257, 299):
        for rows_q in (q, odd[:, 1:].unflatten(1, (2, hd))):
            out, lse = torch.full_like(q, 9.0), torch.full((2, 300), 9.0, device="cuda")
            packed(rows_q, k, v, cu_of([end]), out=out, lse=lse)
            assert (out[end:] == 9).all() and (lse[:, end:] == 9).all()
            assert (out[:end] - want[:end]).abs().max() <= tol


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_small_weights_beside_a_large_one(packed, hd, dtype):
    """A first key whose weight is 2^25.2 times each other's, and 100,000 others that together have 0.25 % of it: they are not
    lost.  The result is theirs alone (the first value is 0): a weight's rounding, 2^-9 at most (bf16) and 2^-11 at most for those
    of fp16 that keep its 11 bits, the sum of 100,000 such terms, 100,000 2^-24 = 0.6 % at most, and the result's own rounding:
    within 1.5 % of it."""
    n = 100000
    q, k, v = torch.ones(n, 1, hd), torch.zeros(n, 1, hd), torch.ones(n, 1, hd)
    k[0], v[0] = 17.5 * hd ** -0.5, 0.0
    q, k, v = (x.to(DTYPES[dtype]).cuda() for x in (q, k, v))
    got = packed(q, k, v, cu_of([n]))[:, 0].double()
    ratio = torch.exp(-(k[0].double().sum() * hd ** -0.5))     # of another weight to the first one's
    others = torch.arange(n, device="cuda").double() * ratio
    want = (others / (1 + others))[:, None]
    assert ((got - want).abs()[1000:] <= 0.015 * want[1000:]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_of_keys_with_the_smallest_weights(packed, hd, dtype):
    """An infinite value of a key whose score lies 200 below those after it, and above those before it: a weight is positive in
    the formula, so the rows from it on are infinite there.  Of rows that TMA takes and of rows at odd addresses."""
    n, heads = 300, 2
    q, k, v = rows([n], heads, 1, hd, dtype, 16)
    q.fill_(1)
    k.zero_()
    k[:50] = -400 * hd ** -0.5
    k[50:200] = -200 * hd ** -0.5
    v[60, 0, 3], v[10, 0, 5], v[199, 0, 7], v[250, 0, 9] = float("inf"), -float("inf"), float("nan"), float("inf")
    odd = torch.zeros(n, heads * hd + 1, dtype=q.dtype, device="cuda")
    odd[:, 1:] = q.flatten(1)
    for rows_q in (q, odd[:, 1:].unflatten(1, (heads, hd))):
        lse = torch.empty(heads, n, device="cuda")
        y = packed(rows_q, k, v, cu_of([n]), lse=lse)
        assert (y[60:, :, 3] == float("inf")).all() and y[:60, :, 3].isfinite().all()
        assert (y[10:, :, 5] == -float("inf")).all() and y[:10, :, 5].isfinite().all()
        assert y[199:, :, 7].isnan().all() and y[:199, :, 7].isfinite().all()
        assert (y[250:, :, 9] == float("inf")).all() and y[:250, :, 9].isfinite().all()
        rest = [d for d in range(hd) if d not in (3, 5, 7, 9)]
        assert y[..., rest].isfinite().all() and lse.isfinite().all()

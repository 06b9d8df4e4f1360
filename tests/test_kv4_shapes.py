"""Sizes of the paged 4-bit cache (include/holo_b200.h, cuda_kv4_pool_bytes and
cuda_kv4_work_bytes): host arithmetic, no device."""
import ctypes as C

import pytest

import holo_b200 as hb
import serving_reference as ref
from holo_b200.kv4 import Kv4Desc


def sizes(**change):
    shape = dict(n_layers=2, n_kv_heads=4, head_dim=128, page_tokens=64, n_pages=10, max_seqs=3, max_pages=5)
    d = Kv4Desc(**(shape | change))
    lib = hb.load()
    return lib.cuda_kv4_pool_bytes(C.addressof(d)), lib.cuda_kv4_work_bytes(C.addressof(d))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 48, 256])
def test_pool(hd, page):
    pool, work = sizes(head_dim=hd, page_tokens=page)
    assert pool == 2 * 10 * 4 * page * (hd // 32) * 36   # 18 bytes a group of 32, keys and values
    assert work > 0


def test_a_pool_past_32_bits():
    assert sizes(n_layers=80, n_pages=1 << 20, n_kv_heads=8)[0] == 80 * (1 << 20) * 8 * 4 * 18 * 128


@pytest.mark.parametrize("change", [
    dict(head_dim=96), dict(head_dim=0), dict(page_tokens=24), dict(page_tokens=0), dict(page_tokens=272), dict(n_layers=0),
    dict(n_kv_heads=0), dict(n_pages=0), dict(n_pages=-1), dict(n_pages=(1 << 20) + 1), dict(max_seqs=0), dict(max_seqs=(1 << 16) + 1),
    dict(max_pages=0)])
def test_shapes_that_are_refused(change):
    assert sizes(**change) == (0, 0)
    assert hb.load().cuda_last_status() == hb.HOLO_OK


def test_the_layout_names_every_code_once():
    """The reference layout of the tests covers a block's 16 hd code bytes, two codes each, and its scales once."""
    for hd in (64, 128, 256):
        codes = {ref.half_at(hd, side, p, d) for side in (0, 1) for p in range(16) for d in range(hd)}
        assert len(codes) == 32 * hd and {o for o, _ in codes} == set(range(16 * hd))
        scales = {ref.scale_at(hd, side, p, d) for side in (0, 1) for p in range(16) for d in range(0, hd, 32)}
        assert scales == set(range(16 * hd, 18 * hd, 2))

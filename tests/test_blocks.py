"""The 8-bit block cache without a GPU: arguments that are refused, host arithmetic, the oracle's rounding."""
import ctypes
import math

import pytest
import torch

import blocks_oracle as orc


def _view(pkg, **kw):
    f = dict(k=4096, v=4096, ks=4096, vs=4096, table=4096, ends=4096, status=0, n_pages=4, Hkv=2, page_size=16, dh=128, B=2, max_blocks=2,
             store=0)
    f.update(kw)
    return ctypes.byref(pkg._lib.Blocks(*f.values()))


def test_struct_layout(pkg):
    lib = pkg._lib.load()
    assert lib.sphkv_struct_size(5) == ctypes.sizeof(pkg._lib.Blocks) == 7 * 8 + 7 * 4 + 4


@pytest.mark.parametrize("kw,rc", [(dict(k=0), -1), (dict(ends=0), -1), (dict(table=0), -1), (dict(ks=0), -1), (dict(dh=96), -1),
                                   (dict(page_size=48), -1), (dict(B=0), -1), (dict(Hkv=0), -1), (dict(store=2), -2), (dict(k=4104), -3),
                                   (dict(n_pages=2 ** 27), -5), (dict(max_blocks=2 ** 27), -5), (dict(B=2 ** 21), -5)])
def test_bad_caches_are_refused(pkg, kw, rc):
    lib, view = pkg._lib.load(), _view(pkg, **kw)
    assert lib.sphkv_blocks_append(view, 4096, 4096, 0, 256, 128, 256, 128, None, 2, None) == rc
    assert lib.sphkv_blocks_read(view, 4096, 4096, 0, None, 2, None) == rc
    assert lib.sphkv_blocks_decode(view, 4096, 1, 512, 128, None, 4096, 1, None, 4096, 1 << 30, 4, 0.1, None) == rc
    assert lib.sphkv_blocks_attend(view, 4096, 1, 512, 128, None, 2, None, 4096, 1, 4096, 1 << 30, 4, 0.1, None) == rc
    assert lib.sphkv_last_error()


def test_bad_arguments_are_refused(pkg):
    lib, view = pkg._lib.load(), _view(pkg)
    st = (256, 128, 256, 128)
    assert lib.sphkv_blocks_append(None, 4096, 4096, 0, *st, None, 2, None) == -1
    assert lib.sphkv_blocks_append(view, None, 4096, 0, *st, None, 2, None) == -1
    assert lib.sphkv_blocks_append(view, 4096, 4096, 3, *st, None, 2, None) == -2
    assert lib.sphkv_blocks_append(view, 4096, 4096, 0, *st, None, 3, None) == -1   # 3 rows, two sequences
    assert lib.sphkv_blocks_append(view, 4097, 4096, 1, *st, None, 2, None) == -3
    assert lib.sphkv_blocks_append(view, 4096, 4096, 0, *st, None, 2 ** 30, None) == -5
    assert lib.sphkv_blocks_append(view, None, None, 0, *st, None, 0, None) == 0    # no rows: nothing to do
    assert lib.sphkv_blocks_read(view, 4104, 4096, 0, None, 2, None) == -3
    assert lib.sphkv_blocks_read(view, 4096, None, 0, None, 2, None) == -1
    dec = lambda q=4096, qt=1, out=4096, ot=1, scratch=4096, nb=1 << 30, hq=4: lib.sphkv_blocks_decode(  # noqa: E731
        view, q, qt, 512, 128, None, out, ot, None, scratch, nb, hq, 0.1, None)
    assert dec(q=None) == -1 and dec(out=None) == -1 and dec(qt=5) == -2 and dec(ot=-1) == -2 and dec(hq=5) == -1 and dec(hq=18) == -5
    assert dec(q=4097) == -3 and dec(out=4097) == -3
    att = lambda qt=1, out=4096, hq=4: lib.sphkv_blocks_attend(view, 4096, qt, 512, 128, None, 2, None, out, 1, 4096, 1 << 30,  # noqa: E731
                                                               hq, 0.1, None)
    assert att(qt=0) == -2 and att(out=None) == -1 and att(hq=18) == -5
    assert lib.sphkv_blocks_decode_scratch_bytes(0, 4, 2, 128) < 0 and lib.sphkv_blocks_decode_scratch_bytes(2, 5, 2, 128) < 0
    assert lib.sphkv_blocks_attend_scratch_bytes(2, -1, 4, 2, 128) < 0 and lib.sphkv_blocks_attend_scratch_bytes(2, 4, 36, 2, 128) < 0


def test_wrappers_refuse_what_they_cannot_take(pkg):
    table = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError):
        pkg.new_block_cache(4, 2, 16, 128, table, torch.float16)
    with pytest.raises(ValueError):
        pkg.new_block_cache(4, 2, 24, 128, table)
    with pytest.raises(ValueError):
        pkg.new_block_cache(4, 2, 16, 80, table)
    cache = pkg.new_block_cache(4, 2, 16, 128, table, torch.float8_e4m3fn)
    assert cache.k_codes.shape == (4, 2, 16, 128) and cache.page_size == 16 and cache.dh == 128 and cache.Hkv == 2
    x = torch.zeros(2, 1, 2, 128)
    for call in (lambda: pkg.append_blocks(cache, x, x), lambda: pkg.read_blocks(cache, n=1),
                 lambda: pkg.decode_blocks(torch.zeros(2, 4, 128), cache), lambda: pkg.attend_blocks(torch.zeros(2, 1, 4, 128), cache)):
        with pytest.raises(pkg.SphKVError):  # host tensors: there is no CPU path
            call()


def test_oracle_rounds_to_the_nearest_code():
    # every e4m3 value is its own nearest, midpoints go to the even code
    vals = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(orc.nearest(vals, torch.float8_e4m3fn), vals) and torch.equal(orc.nearest(-vals, torch.float8_e4m3fn), -vals)
    mid = (vals[1:] + vals[:-1]) / 2
    even = torch.where(torch.arange(126) % 2 == 0, vals[:-1], vals[1:])
    assert torch.equal(orc.nearest(mid, torch.float8_e4m3fn), even)
    assert torch.equal(orc.nearest(mid * (1 + 2.0 ** -40), torch.float8_e4m3fn), vals[1:])
    assert torch.equal(orc.nearest(mid * (1 - 2.0 ** -40), torch.float8_e4m3fn), vals[:-1])
    x = torch.randn(1000, generator=torch.Generator().manual_seed(0)) * 30
    assert torch.equal(orc.nearest(x.double(), torch.float8_e4m3fn).float(), x.to(torch.float8_e4m3fn).float())
    assert orc.nearest(torch.tensor([2.5, -2.5, 3.5, 126.6], dtype=torch.float64), torch.int8).tolist() == [2, -2, 4, 127]
    assert math.isclose(float(orc.f32_quotient(torch.tensor(1.0), 127.0)), 1 / 127, rel_tol=2 ** -24)

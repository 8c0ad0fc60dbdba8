"""The 8-bit block cache on the GPU where it can go wrong: what the other tests of it do not reach."""
import math
import random

import pytest
import torch

from test_gpu_blocks import DEV, E4M3, I8, _cache, _check, _cu, _filled, _random, _same, _sides
import blocks_oracle as orc

pytestmark = pytest.mark.gpu
HALF16 = torch.finfo(torch.float16).eps / 2  # a weight of the many-query kernel is off by this, relative


@pytest.mark.parametrize("store,N,dh", [(I8, 16, 128), (E4M3, 64, 64)])
def test_attend_repeats_itself(pkg, store, N, dh):
    """Many short segments a worker: every warp of a block reads the same ones, in every pass."""
    H, Hq = 4, 16
    lens = [37 + 61 * (b % 7) for b in range(60)]
    cache = _filled(pkg, lens, H, N, dh, store, 13)
    news = [min(n, 3 + 29 * (b % 5)) for b, n in enumerate(lens)]
    q = _random((sum(news), Hq, dh), 3, torch.bfloat16).to(DEV)
    want = pkg.attend_blocks(q, cache, cu_new=_cu(news))
    assert want.isfinite().all()
    for _ in range(20):
        assert torch.equal(pkg.attend_blocks(q, cache, cu_new=_cu(news)), want)
    sides, table = _sides(cache), cache.block_table.cpu()
    for b in (0, 6, 33, 59):
        at, n = sum(news[:b]), news[b]
        kk, vv = (s.rows(table[b], 0, lens[b]) for s in sides)
        exact, _, _, off, size, _ = orc.attend(q[at:at + n].cpu(), kk, vv, 0, list(range(lens[b] - n, lens[b])), 1 / math.sqrt(dh))
        _check(want[at:at + n], exact, off + HALF16 * size, torch.bfloat16)
    pkg.check_status(cache)


@pytest.mark.parametrize("store,N,dh", [(I8, 16, 128), (E4M3, 32, 64)])
def test_references_move_inside_an_edge_tile(pkg, store, N, dh):
    """Logits that grow by more than the reference's slack from one group of 16 keys to the next, in tiles that `first` or the queries' own
    positions cut: the weights before are scaled down in front of every group, odd ones among them."""
    H, Hq, ctx, n = 1, 8, 250, 130
    cache = _cache(pkg, [ctx], H, N, dh, store, 17)
    steps = (torch.arange(ctx) // 16 + 1.0)[:, None, None]
    direction = torch.sign(_random((1, 1, dh), 9, torch.float32))
    k = direction * steps * (24.0 / dh ** 0.5) + 0.01 * _random((ctx, H, dh), 5, torch.float32)  # logits about 24 apart, in units of log2 e
    v = _random((ctx, H, dh), 6, torch.float32)
    pkg.append_blocks(cache, k.to(DEV), v.to(DEV), cu_new=_cu([ctx]))
    q = (direction + 0.01 * _random((n, Hq, dh), 3, torch.float32)).to(torch.float16)
    sides, table = _sides(cache), cache.block_table.cpu()
    for first in (0, 5, 100):
        kk, vv = (s.rows(table[0], first, ctx) for s in sides)
        want, _, _, off, size, _ = orc.attend(q, kk, vv, first, list(range(ctx - n, ctx)), 1 / math.sqrt(dh))
        f = torch.tensor([first], dtype=torch.int32, device=DEV)
        got = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu([n]), first=f, out_dtype=torch.float32)
        # a weight below 2^-14 is off by 2^-25, and again in each of the 15 times that it may be scaled down, where the largest is 2^6 or more
        tiny = 16 * ctx * 2.0 ** -31 * float(vv.abs().max())
        _check(got, want, off + HALF16 * size + tiny, torch.float32)
    pkg.check_status(cache)


@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("lead", [1, 5, 700])
def test_rows_before_the_first_sequence(pkg, group, lead):
    """cu[0] above 0: the rows before it are no sequence's, in every operator and in both of attend's kernels."""
    H, N, dh = 2, 16, 64
    lens, Hq = [900, 40], 2 * group
    cache = _filled(pkg, lens, H, N, dh, I8, 23)
    other = _cache(pkg, lens, H, N, dh, I8, 23)
    sides, table = _sides(cache), cache.block_table.cpu()
    for news in ([1, 1], [500, 33]):
        rows = lead + sum(news) + 2
        cu = _cu(news) + lead
        q = _random((rows, Hq, dh), 3, torch.bfloat16).to(DEV)
        out = torch.full((rows, Hq, dh), 7.0, dtype=torch.bfloat16, device=DEV)
        pkg.attend_blocks(q, cache, cu_new=cu, out=out)
        assert (out[:lead] == 7.0).all() and (out[-2:] == 7.0).all()
        at = lead
        for b, n in enumerate(news):
            kk, vv = (s.rows(table[b], 0, lens[b]) for s in sides)
            want, _, _, off, size, _ = orc.attend(q[at:at + n].cpu(), kk, vv, 0, list(range(lens[b] - n, lens[b])), 1 / math.sqrt(dh))
            _check(out[at:at + n], want, off + HALF16 * size, torch.bfloat16)
            at += n
        k, v = pkg.read_blocks(cache, cu_rows=_cu(news), rows=sum(news))
        got = tuple(torch.full((rows, H, dh), 7.0, device=DEV) for _ in range(2))
        pkg.read_blocks(cache, cu_rows=cu, out=got)
        for a, b in zip(got, (k, v)):
            assert (a[:lead] == 7.0).all() and torch.equal(a[lead:-2], b) and (a[-2:] == 7.0).all()
    new = [torch.full((lead + sum(lens), H, dh), math.nan, device=DEV) for _ in range(2)]
    for x, s in zip(new, (5, 6)):
        x[lead:] = _random((sum(lens), H, dh), 23 + s, torch.bfloat16).to(DEV)
    pkg.append_blocks(other, *new, cu_new=_cu(lens) + lead)
    for a, b in zip(pkg.read_blocks(other, cu_rows=_cu(lens), rows=sum(lens)), pkg.read_blocks(cache, cu_rows=_cu(lens), rows=sum(lens))):
        assert torch.equal(a, b)
    pkg.check_status(cache)
    pkg.check_status(other)


def test_read_without_a_type(pkg):
    """out_dtype=None is read_blocks' default, and is not looked at where outputs are given."""
    cache = _filled(pkg, [40, 20], 2, 16, 64, I8, 29)
    want = pkg.read_blocks(cache, n=20)
    for got in (pkg.read_blocks(cache, n=20, out_dtype=None), pkg.read_blocks(cache, cu_rows=_cu([20, 20]), rows=40, out_dtype=None)):
        for a, b in zip(got, want):
            assert a.dtype == torch.float32 and torch.equal(a.view_as(b), b)
    out = tuple(torch.empty(2, 20, 2, 64, dtype=torch.float16, device=DEV) for _ in range(2))
    got = pkg.read_blocks(cache, n=20, out=out, out_dtype=None)
    for a, b in zip(got, want):
        assert torch.equal(a, b.half())


@pytest.mark.parametrize("store,N,dh", [(I8, 16, 128), (E4M3, 16, 64), (E4M3, 32, 128), (E4M3, 128, 64), (I8, 64, 64)])
def test_nothing_before_first_is_looked_at(pkg, store, N, dh):
    """Pages before first's have been given away (the table names none), and the slots before first hold any bytes."""
    H, Hq = 2, 8
    lens, first = [300, 140, 700], [100, 139, 517]
    cache = _filled(pkg, lens, H, N, dh, store, 33)
    sides, table = _sides(cache), cache.block_table.cpu()
    for b, f in enumerate(first):
        page = int(table[b, f // N])
        for codes in (cache.k_codes, cache.v_codes):
            codes.view(torch.uint8)[page, :, :f % N] = 0x7f  # NaN in e4m3
        cache.block_table[b, :f // N] = -1
    fs = torch.tensor(first, dtype=torch.int32, device=DEV)
    for news in ([1, 1, 1], [2, 1, 0], [20, 1, 3], [250, 130, 300]):
        q = _random((sum(news), Hq, dh), 3, torch.bfloat16)
        got = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu(news), first=fs)
        pkg.check_status(cache)
        at = 0
        for b, n in enumerate(news):
            kk, vv = (s.rows(table[b], first[b], lens[b]) for s in sides)
            want, _, _, off, size, _ = orc.attend(q[at:at + n], kk, vv, first[b], list(range(lens[b] - n, lens[b])), 1 / math.sqrt(dh))
            if n:
                _check(got[at:at + n], want, off + HALF16 * size, torch.bfloat16)
            at += n
    q = _random((3, Hq, dh), 3, torch.float32)
    got = pkg.decode_blocks(q.to(DEV), cache, first=fs)
    for b in range(3):
        kk, vv = (s.rows(table[b], first[b], lens[b]) for s in sides)
        want, _, _, off, _, _ = orc.attend(q[b:b + 1], kk, vv, first[b], [lens[b] - 1], 1 / math.sqrt(dh))
        _check(got[b:b + 1], want, off, torch.float32)
    pkg.check_status(cache)


def _scales(side, table, lo, hi):
    """Of the pages of keys lo .. hi - 1: [keys, H]."""
    return side.scale[table[torch.arange(lo, hi) // side.N].long()]


def _least(q, k, scale, pos, scales, top, key0=0):
    """What weights may be off that are below f16's normal numbers, per query row and head: 2^-25 of each where the row's largest weight (times
    value scale) is put at 2^5 at least, that is 2^-30 of the largest, for every key; times the largest code.  scales: [keys, H], of the keys' pages."""
    n, Hq, dh = q.shape
    H = k.shape[1]
    out = torch.zeros(n, Hq, 1, dtype=torch.float64)
    if k.shape[0] == 0:
        return out
    for h in range(Hq):
        x = q[:, h].double() @ k[:, h // (Hq // H)].T * scale
        x = x.masked_fill(torch.arange(key0, key0 + k.shape[0])[None] > torch.as_tensor(pos)[:, None], -math.inf)
        out[:, h, 0] = (torch.softmax(x, 1).nan_to_num(0.0) * scales[:, h // (Hq // H)].double()).amax(1) * (k.shape[0] * top * 2.0 ** -30)
    return out


@pytest.mark.parametrize("sm_scale", [0.4, 1.0])
@pytest.mark.parametrize("store,N,dh,Hq,H,dtype", [(I8, 16, 128, 8, 2, torch.bfloat16), (E4M3, 64, 64, 6, 2, torch.float16)])
def test_large_sm_scales(pkg, store, N, dh, Hq, H, dtype, sm_scale):
    """Logits far apart: weights stand beside ones 2^20 times as large, and were scaled down where those came in behind them."""
    lens = [5, 333, 200, 0]
    cache = _filled(pkg, lens, H, N, dh, store, 51)
    sides, table = _sides(cache), cache.block_table.cpu()
    for news, first in (([1, 2, 1, 0], None), ([5, 150, 129, 0], None), ([5, 150, 129, 0], [3, 190, 130, 0])):
        q = _random((sum(news), Hq, dh), 3, dtype)
        f = None if first is None else torch.tensor(first, dtype=torch.int32, device=DEV)
        out = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu(news), first=f, sm_scale=sm_scale, out_dtype=torch.float32)
        at = 0
        for b, n in enumerate(news):
            lo = min(lens[b], 0 if first is None else first[b])
            k, v = (s.rows(table[b], lo, lens[b]).reshape(-1, H, dh) for s in sides)
            pos = list(range(lens[b] - n, lens[b]))
            want, _, _, off, size, _ = orc.attend(q[at:at + n], k, v, lo, pos, sm_scale)
            if n:
                least = _least(q[at:at + n], k, sm_scale, pos, _scales(sides[1], table[b], lo, lens[b]), orc.TOP[store], lo)
                _check(out[at:at + n], want, off + HALF16 * size + least, torch.float32)
            at += n
    q = _random((4, Hq, dh), 3, dtype)
    out = pkg.decode_blocks(q.to(DEV), cache, sm_scale=sm_scale, out_dtype=torch.float32)
    for b, n in enumerate(lens):
        k, v = (s.rows(table[b], 0, n).reshape(-1, H, dh) for s in sides)
        want, _, _, off, _, _ = orc.attend(q[b:b + 1], k, v, 0, [n - 1], sm_scale)
        least = _least(q[b:b + 1], k, sm_scale, [n - 1], _scales(sides[1], table[b], 0, n), orc.TOP[store])
        _check(out[b:b + 1], want, off + least, torch.float32)
    pkg.check_status(cache)


@pytest.mark.parametrize("sm_scale", [-0.3, -1.0, 0.0])
@pytest.mark.parametrize("store,N,dh,Hq,H,dtype", [(I8, 16, 128, 8, 2, torch.bfloat16), (E4M3, 64, 64, 6, 2, torch.float16)])
def test_any_finite_sm_scale(pkg, store, N, dh, Hq, H, dtype, sm_scale):
    """Negative scales and zero, in both of attend's kernels and in decode."""
    lens = [5, 333, 200, 0]
    cache = _filled(pkg, lens, H, N, dh, store, 51)
    sides, table = _sides(cache), cache.block_table.cpu()
    sign = -1 if sm_scale < 0 else 1
    for news, first in (([1, 2, 1, 0], None), ([5, 150, 129, 0], None), ([5, 150, 129, 0], [3, 190, 130, 0])):
        q = _random((sum(news), Hq, dh), 3, dtype)
        f = None if first is None else torch.tensor(first, dtype=torch.int32, device=DEV)
        out = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu(news), first=f, sm_scale=sm_scale, out_dtype=torch.float32)
        at = 0
        for b, n in enumerate(news):
            lo = min(lens[b], 0 if first is None else first[b])
            k, v = (s.rows(table[b], lo, lens[b]).reshape(-1, H, dh) for s in sides)
            pos = list(range(lens[b] - n, lens[b]))
            want, _, _, off, size, _ = orc.attend(sign * q[at:at + n], k, v, lo, pos, abs(sm_scale))
            if n:
                least = _least(q[at:at + n], k, sm_scale, pos, _scales(sides[1], table[b], lo, lens[b]), orc.TOP[store], lo)
                _check(out[at:at + n], want, off + HALF16 * size + least, torch.float32)
            at += n
    q = _random((4, Hq, dh), 3, dtype)
    out = pkg.decode_blocks(q.to(DEV), cache, sm_scale=sm_scale, out_dtype=torch.float32)
    for b, n in enumerate(lens):
        k, v = (s.rows(table[b], 0, n).reshape(-1, H, dh) for s in sides)
        want, _, _, off, _, _ = orc.attend(sign * q[b:b + 1], k, v, 0, [n - 1], abs(sm_scale))
        least = _least(q[b:b + 1], k, sm_scale, [n - 1], _scales(sides[1], table[b], 0, n), orc.TOP[store])
        _check(out[b:b + 1], want, off + least, torch.float32)
    pkg.check_status(cache)


def test_scales_that_are_no_number_are_refused(pkg):
    cache = _filled(pkg, [40, 20], 2, 16, 64, I8, 29)
    q = _random((2, 4, 64), 3, torch.bfloat16).to(DEV)
    for bad in (math.nan, math.inf, -math.inf, 1e300):
        for call in (lambda: pkg.decode_blocks(q, cache, sm_scale=bad), lambda: pkg.attend_blocks(q[:, None], cache, sm_scale=bad)):
            with pytest.raises(pkg.SphKVError, match="sm_scale"):
                call()
    assert torch.equal(pkg.decode_blocks(q, cache), pkg.decode_blocks(q, cache, sm_scale=0.125))


@pytest.mark.parametrize("power", [10, 20, 30, 70, 110])
@pytest.mark.parametrize("store,N,dh,q_dtype", [(I8, 128, 128, torch.float32), (E4M3, 16, 64, torch.float16)])
def test_decode_value_scales_far_apart(pkg, store, N, dh, q_dtype, power):
    """A page of large values that the softmax gives next to nothing takes no bits from the others, wherever it lies.  Every warp has several
    tiles: of the page, before and behind it."""
    H, Hq, ctx, B = 8, 16, 4000, 8
    direction = torch.sign(_random((1, 1, dh), 9, torch.float32))
    q = (direction + 0.05 * _random((B, Hq, dh), 3, torch.float32)).to(q_dtype)
    for at in (0, 2000):
        cache = _cache(pkg, [ctx] * B, H, N, dh, store, 61)
        k, v = 0.05 * _random((B, ctx, H, dh), 5, torch.float32), _random((B, ctx, H, dh), 6, torch.float32)
        page = torch.arange(ctx) // 128 == at // 128
        # logits of the page: lower by about `power` + 8 in units of log2 e
        k[:, page] -= direction * ((power + 8) * math.log(2) / dh ** 0.5)
        v[:, page] *= 2.0 ** power
        pkg.append_blocks(cache, k.to(DEV), v.to(DEV))
        sides, table = _sides(cache), cache.block_table.cpu()
        part = torch.empty(B, Hq, dh + 2, device=DEV)
        got = pkg.decode_blocks(q.to(DEV), cache, out_dtype=torch.float32, out_partial=part)
        for b in (0, 3, 7):
            kk, vv = (s.rows(table[b], 0, ctx) for s in sides)
            want, _, _, off, _, _ = orc.attend(q[b:b + 1], kk, vv, 0, [ctx - 1], 1 / math.sqrt(dh))
            least = _least(q[b:b + 1], kk, 1 / math.sqrt(dh), [ctx - 1], _scales(sides[1], table[b], 0, ctx), orc.TOP[store])
            _check(got[b:b + 1], want, off + least, torch.float32)
            _check((part[b:b + 1, :, 2:] / part[b:b + 1, :, 1:2]), want, off + least + want.abs() * 2.0 ** -22, torch.float32)
        pkg.check_status(cache)


@pytest.mark.parametrize("power", [20, 60, 110])
def test_few_tokens_and_values_that_they_do_not_see(pkg, power):
    """The last token's value is large: the token before it, in the same unit, does not see it."""
    H, Hq, N, dh, ctx, B = 8, 32, 16, 128, 4000, 8
    cache = _cache(pkg, [ctx - 1] * B, H, N, dh, I8, 65, max_len=[ctx] * B)
    k, v = _random((B, ctx, H, dh), 5, torch.float32), _random((B, ctx, H, dh), 6, torch.float32)
    v[:, -N:] *= 0  # the last page's scale will be the large value's
    pkg.append_blocks(cache, k[:, :-1].contiguous().to(DEV), v[:, :-1].contiguous().to(DEV))
    cache.seq_lens += 1
    v[:, -1] = 2.0 ** power
    pkg.append_blocks(cache, k[:, -1:].to(DEV), v[:, -1:].to(DEV))
    # tiles go round a unit's warps in order, and a warp has several: behind the first it starts with what it has
    first = torch.arange(B, dtype=torch.int32, device=DEV)
    sides, table = _sides(cache), cache.block_table.cpu()
    q = _random((B, 2, Hq, dh), 3, torch.float16)
    got = pkg.attend_blocks(q.to(DEV), cache, first=first, out_dtype=torch.float32)
    for b in (0, 1, 7):
        kk, vv = (s.rows(table[b], b, ctx) for s in sides)
        for i in (0, 1):
            n = ctx - 1 + i
            want, _, _, off, _, _ = orc.attend(q[b, i:i + 1], kk[:n - b], vv[:n - b], b, [n - 1], 1 / math.sqrt(dh))
            scales = _scales(sides[1], table[b], b, n).clone()
            if i == 0:
                scales[-(N - 1):] = 0  # its page's scale is large, its values there are zeros
            _check(got[b, i:i + 1], want, off + _least(q[b, i:i + 1], kk[:n - b], 1 / math.sqrt(dh), [n - 1], scales, 127.0, b), torch.float32)
    pkg.check_status(cache)


def test_decode_scales_at_both_ends(pkg):
    """Value scales from 2^-126 to 2^120, pages of zeros that outweigh all others by far, and a page of large values 2^100 lighter."""
    H, Hq, N, dh, ctx, B = 8, 16, 16, 64, 4000, 8
    direction = torch.sign(_random((1, 1, dh), 9, torch.float32))
    q = direction + 0.05 * _random((B, Hq, dh), 3, torch.float32)
    tile = torch.arange(ctx) // 128
    for small, large, light, zero in ((-119, 119, 250, 0), (-20, 100, 100, 60), (-118, -118, 0, 100), (0, 0, 0, 230), (-110, 0, 105, 20), (0, 112, 108, 0)):
        k, v = 0.05 * _random((B, ctx, H, dh), 5, torch.float32), _random((B, ctx, H, dh), 6, torch.float32).clamp(-4, 4)
        v = v.double() * 2.0 ** small
        lift = torch.zeros(ctx)
        big, none = tile % 4 == 1, tile % 4 == 2
        v[:, big] *= 2.0 ** (large - small)
        v[:, none] = 0
        lift[big], lift[none] = -light, zero  # log2 of how much heavier a page's tokens are
        k += direction * (lift * math.log(2) / dh ** 0.5)[:, None, None]
        v = v.float()
        assert v.isfinite().all()
        cache = _cache(pkg, [ctx] * B, H, N, dh, I8, 67)
        pkg.append_blocks(cache, k.to(DEV), v.to(DEV))
        sides, table = _sides(cache), cache.block_table.cpu()
        got = pkg.decode_blocks(q.to(DEV), cache)
        for b in (0, 7):
            kk, vv = (s.rows(table[b], 0, ctx) for s in sides)
            want, _, _, off, _, _ = orc.attend(q[b:b + 1], kk, vv, 0, [ctx - 1], 1 / math.sqrt(dh))
            least = _least(q[b:b + 1], kk, 1 / math.sqrt(dh), [ctx - 1], _scales(sides[1], table[b], 0, ctx), 127.0)
            # p and the factors between parts are fp32 numbers: below 2^-126 of the row's largest p (its reference may be one power of two above
            # that) they are 0, whatever they are multiplied by
            x = torch.einsum("hgd,thd->hgt", q[b].double().view(H, Hq // H, dh), kk).reshape(Hq, ctx) / math.sqrt(dh)
            w = torch.exp(x - x.amax(1, keepdim=True))
            lost = torch.einsum("ht,thd->hd", w.masked_fill(w > 2.0 ** -125, 0.0), vv.abs().repeat_interleave(2, 1)) / w.sum(1, keepdim=True)
            least = least + lost + 2.0 ** -149
            _check(got[b:b + 1], want, off + least, torch.float32)
        pkg.check_status(cache)


@pytest.mark.parametrize("store", [I8, E4M3])
def test_nearest_codes_of_the_smallest_scales(pkg, store):
    """Scales a few powers of two above 2^-126, tokens a unit of 2^-149 beside the borders between codes: differences that fp32 has no
    number for."""
    top, dh, n = orc.TOP[store], 64, 48
    unit = 2.0 ** -149
    rows = []
    for i in range(n):
        scale = (2 ** 23 + 2 * (3 * i * i * 7919 % (2 ** 22)) + 1) * 2 ** (i // 16)
        largest = torch.tensor(scale * top, dtype=torch.float64).mul(unit).float()
        s = orc.f32_quotient(largest, top).double() / unit
        codes = torch.arange(0, 127, dtype=torch.uint8).view(E4M3).double() if store is E4M3 else torch.arange(0, 127).double()
        border = (codes[1:] + codes[:-1]) / 2 * s
        border = border[border < 2 ** 24][:31 * (2 if store is E4M3 else 1)]
        pick = border[torch.randperm(border.numel(), generator=torch.Generator().manual_seed(i))[:31]]
        x = torch.cat([torch.floor(pick), torch.ceil(pick)])
        x = torch.cat([torch.tensor([float(largest) / unit], dtype=torch.float64), x, torch.zeros(dh - 1 - x.numel(), dtype=torch.float64)])
        rows.append((x * unit).float())
    rows = torch.stack(rows)[:, None]
    cache = _cache(pkg, [1] * n, 1, 16, dh, store, 3, max_len=[1] * n)
    table, sides = cache.block_table.cpu(), _sides(cache)
    pkg.append_blocks(cache, rows[:, None].to(DEV), -rows[:, None].to(DEV))
    for b in range(n):
        sides[0].append(table[b], 1, rows[b:b + 1])
        sides[1].append(table[b], 1, -rows[b:b + 1])
    _same(cache, sides, table, [1] * n)
    pkg.check_status(cache)


def test_value_scale_reference_moves_row_by_row(pkg):
    """Thirty-two rows of a warp: the first see only values of 2^-75, so that their sums cannot follow the value scales' reference when it grows
    by 2^40 for a page that none of them sees; the last, which see that tile's first keys, keep their bits all the same."""
    B, H, N, dh, n = 20, 16, 16, 64, 64
    ctx = 100 + n
    cache = _cache(pkg, [ctx] * B, H, N, dh, I8, 97)
    k, v = _random((B, ctx, H, dh), 5, torch.float32), _random((B, ctx, H, dh), 6, torch.float32)
    v[:, :112] *= 2.0 ** -75
    v[:, 144:] *= 2.0 ** 40
    pkg.append_blocks(cache, k.to(DEV), v.to(DEV))
    sides, table = _sides(cache), cache.block_table.cpu()
    q = _random((B, n, H, dh), 3, torch.float16)
    got = pkg.attend_blocks(q.to(DEV), cache, out_dtype=torch.float32)
    for b in range(0, B, 5):
        kk, vv = (s.rows(table[b], 0, ctx) for s in sides)
        for lo, hi in ((0, 12), (12, 44), (44, 64)):
            last = 100 + hi
            want, _, _, off, size, _ = orc.attend(q[b, lo:hi], kk[:last], vv[:last], 0, list(range(100 + lo, last)), 0.125)
            least = _least(q[b, lo:hi], kk[:last], 0.125, list(range(100 + lo, last)), _scales(sides[1], table[b], 0, last), 127.0)
            _check(got[b, lo:hi], want, off + HALF16 * size + least, torch.float32)
    pkg.check_status(cache)


@pytest.mark.parametrize("power", [20, 40, 70])
def test_attend_zeros_beside_small_values(pkg, power):
    """Values far below the sequence's largest, which only later rows see, between pages of zeros: the zeros take no bits from them."""
    H, N, dh, Hq, ctx, n = 1, 16, 64, 8, 384, 150
    cache = _cache(pkg, [ctx], H, N, dh, I8, 97)
    k, v = _random((ctx, H, dh), 5, torch.float32), _random((ctx, H, dh), 6, torch.float32)
    page = torch.arange(ctx) // N
    v[page % 3 == 1] = 0
    v[ctx - N:] *= 2.0 ** power  # seen by the last 16 rows
    pkg.append_blocks(cache, k.to(DEV), v.to(DEV), cu_new=_cu([ctx]))
    sides, table = _sides(cache), cache.block_table.cpu()
    kk, vv = (s.rows(table[0], 0, ctx) for s in sides)
    q = _random((n, Hq, dh), 3, torch.float16)
    got = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu([n]), out_dtype=torch.float32)
    for lo, hi in ((0, n - N), (n - N, n)):
        want, _, _, off, size, _ = orc.attend(q[lo:hi], kk, vv, 0, list(range(ctx - n + lo, ctx - n + hi)), 0.125)
        last = ctx - n + hi
        # weights below 2^-14 are off by 2^-25 where the row's largest weight times scale is 2^6 at least: 2^-31 of the largest, for each key
        tiny = last * 2.0 ** -31 * float(vv[:last].abs().max())
        _check(got[lo:hi], want, off + HALF16 * size + tiny, torch.float32)
    pkg.check_status(cache)


def test_nan_reaches_the_merge_with_another_cache(pkg):
    """A page that reads back as NaN makes its decode's rows NaN, with however few keys, and so the rows of both caches together."""
    H, N, dh, Hq, ctx = 2, 16, 128, 4, 2000
    cache = _filled(pkg, [ctx, ctx, 16, ctx], H, N, dh, I8, 71)
    q = _random((4, Hq, dh), 3, torch.float32).to(DEV)
    other = torch.randn(4, Hq, dh + 2, device=DEV)
    other[..., 1] = 2.0
    for scales in (cache.k_scale, cache.v_scale):
        clean = scales.clone()
        scales[cache.block_table[1, 77].long(), 0] = math.nan
        scales[cache.block_table[2, 0].long(), 0] = math.nan
        parts = torch.empty(2, 4, Hq, dh + 2, device=DEV)
        parts[0] = other
        out = pkg.decode_blocks(q, cache, out_partial=parts[1])
        merged = pkg.merge_partials(parts.view(2, 4 * Hq, dh + 2)).view(4, Hq, dh)
        for x in (out, merged):
            for b in range(4):
                assert x[b, 2:].isfinite().all(), b
                assert x[b, :2].isnan().all() if b in (1, 2) else x[b].isfinite().all(), b
        # nothing in the other one
        parts[0, ..., 0], parts[0, ..., 1:] = -math.inf, 0.0
        merged = pkg.merge_partials(parts.view(2, 4 * Hq, dh + 2)).view(4, Hq, dh)
        assert torch.equal(merged.isnan(), out.isnan())
        scales.copy_(clean)
    pkg.check_status(cache)


def test_negative_first_is_none(pkg):
    cache = _filled(pkg, [40, 700], 2, 16, 64, I8, 29)
    first = torch.tensor([-5, -2 ** 31], dtype=torch.int32, device=DEV)
    q = _random((2, 100, 4, 64), 3, torch.bfloat16).to(DEV)
    for n in (1, 30):
        assert torch.equal(pkg.attend_blocks(q[:, :n].contiguous(), cache, first=first), pkg.attend_blocks(q[:, :n].contiguous(), cache))
    assert torch.equal(pkg.decode_blocks(q[:, 0], cache, first=first), pkg.decode_blocks(q[:, 0], cache))
    pkg.check_status(cache)


def test_two_threads(pkg):
    """Calls from two threads at once, each on a stream and a cache of its own."""
    import threading
    caches = [_filled(pkg, [40, 700], 2, 16, 64, I8, 29 + i) for i in (0, 1)]
    q = _random((2, 40, 4, 64), 3, torch.bfloat16).to(DEV)
    want = [(pkg.attend_blocks(q, c), pkg.decode_blocks(q[:, 0], c), pkg.read_blocks(c, n=40)[1]) for c in caches]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                got = (pkg.attend_blocks(q, caches[i]), pkg.decode_blocks(q[:, 0], caches[i]), pkg.read_blocks(caches[i], n=40)[1])
                bad.extend(i for a, b in zip(got, want[i]) if not torch.equal(a, b))
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    for c in caches:
        pkg.check_status(c)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(pkg):
    import copy
    cache = _filled(pkg, [40, 700], 2, 16, 64, I8, 29)
    other = pkg.BlockCache(**{k: t.to("cuda:1") for k, t in copy.copy(cache.__dict__).items()})
    q = _random((2, 30, 4, 64), 3, torch.bfloat16).to(DEV)
    assert torch.equal(pkg.attend_blocks(q.to("cuda:1"), other).to(DEV), pkg.attend_blocks(q, cache))
    assert torch.cuda.current_device() == 0
    pkg.check_status(other)


@pytest.mark.parametrize("seed", [1998, 5876, 6861, 10839] + list(range(40)))
def test_drawn_batches(pkg, seed):
    """Batches of any lengths, groups, pages, rows before and behind, firsts whose older pages are gone, scales of either sign and values over up
    to forty powers of two: attend and decode within the bounds of fp32 sums and of weights that are rounded once (attend: to f16)."""
    r = random.Random(seed)
    H, group = r.choice([1, 2, 3, 4]), r.choice([1, 2, 3, 4, 5, 6, 7, 8])
    Hq, N, dh, store = H * group, r.choice([16, 32, 64, 128]), r.choice([64, 128]), r.choice([I8, E4M3])
    B = r.choice([1, 1, 2, 3, 5, 9, 40, 150])
    top = r.choice([40, 300, 900]) if B < 20 else r.choice([20, 90])
    lens = [r.choice([0, 1, r.randint(0, top), r.randint(0, top), r.randint(top // 2, top)]) for _ in range(B)]
    dtype = r.choice([torch.bfloat16, torch.float16])
    out_dtype = r.choice([dtype, torch.float32])
    most = r.choice([1, 3, 8, 40, 300])
    news = [min(x, r.choice([0, 1, r.randint(0, most), most])) for x in lens]
    first = [r.choice([0, -1, x, x + 5, r.randint(0, max(x, 1))]) for x in lens] if r.random() < 0.5 else None
    sm_scale = r.choice([None, None, 0.05, -0.2, 0.3])
    powers = r.choice([0, 0, 6, 20])
    cache = _cache(pkg, lens, H, N, dh, store, seed + 1)
    total = sum(lens)
    k, v = _random((total, H, dh), seed + 6, torch.float32), _random((total, H, dh), seed + 7, torch.float32)
    if powers and total:
        spread = torch.rand(total // 16 + 1, 1, 1, generator=torch.Generator().manual_seed(seed + 1)).repeat_interleave(16, 0)[:total]
        v = v * torch.exp2(powers * (2 * spread - 1))
    pkg.append_blocks(cache, k.to(DEV), v.to(DEV), cu_new=_cu(lens))
    sides, table = _sides(cache), cache.block_table.cpu()
    if first and r.random() < 0.5:
        for b in range(B):
            if first[b] < lens[b]:
                cache.block_table[b, :max(0, first[b]) // N] = -1
    f = None if first is None else torch.tensor(first, dtype=torch.int32, device=DEV)
    lead, tail = r.choice([0, 0, 3, 77]), r.choice([0, 2])
    rows = lead + sum(news) + tail
    wide = _random((rows, Hq + 1, dh + 8), seed + 8, dtype).to(DEV)
    off = r.choice([0, 1, 8])
    head = r.choice([0, 1])
    q = wide[:, head:head + Hq, off:off + dh]
    out = torch.full((rows, Hq, dh), 7.0, dtype=out_dtype, device=DEV)
    pkg.attend_blocks(q, cache, cu_new=_cu(news) + lead, first=f, sm_scale=sm_scale, out=out)
    q1 = _random((B, Hq, dh), seed + 9, r.choice([torch.float32, dtype]))
    got1 = pkg.decode_blocks(q1.to(DEV), cache, first=f, sm_scale=sm_scale, out_dtype=torch.float32)
    pkg.check_status(cache)
    assert (out[:lead] == 7.0).all() and (out[rows - tail:] == 7.0).all()
    at, scale, largest = lead, 1 / math.sqrt(dh) if sm_scale is None else sm_scale, torch.finfo(out_dtype).max
    sign = -1 if scale < 0 else 1
    for b in range(B):
        n, end, lo = news[b], lens[b], 0 if first is None else min(max(first[b], 0), lens[b])
        at += n
        if B > 9 and b % 29:
            continue
        kk, vv = (s.rows(table[b], lo, end).reshape(-1, H, dh) for s in sides)
        scales = _scales(sides[1], table[b], lo, end).reshape(-1, H)
        qs = q[at - n:at].cpu()
        for qq, pos, got, half in ((qs, list(range(end - n, end)), out[at - n:at], HALF16), (q1[b:b + 1], [end - 1], got1[b:b + 1], 0.0)):
            if not pos:
                continue
            want, _, _, bound, size, _ = orc.attend(sign * qq, kk, vv, lo, pos, abs(scale))
            fits = want.abs() < 0.99 * largest  # beyond, f16 has infinities
            least = _least(qq, kk, scale, pos, scales, orc.TOP[store], lo)
            _check(torch.where(fits.to(DEV), got.double(), want.to(DEV)), want, bound + half * size + least, got.dtype)


@pytest.mark.parametrize("times", [1, 37])
@pytest.mark.parametrize("cu", [[0, 7, 3, 10], [5, 2, 9], [0, 4, 12, 8], [0, 9, 1, 2, 3, 4, 12], [0, 13], [-1, 4], "long"])
def test_offsets_that_do_not_ascend_are_reported(pkg, cu, times):
    """In every operator, wherever the bad pair stands and whichever sequences its neighbours' rows go to."""
    if cu == "long":
        cu = list(range(0, 140, 2))
        cu[50] = 3
    B, rows, H, N, dh = len(cu) - 1, 12 * times if len(cu) < 9 else 140 * times, 2, 16, 64
    ctx = 16 * times + 300
    cache = _filled(pkg, [ctx] * B, H, N, dh, I8, 23)
    c = torch.tensor([x * times for x in cu], dtype=torch.int32, device=DEV)
    k = _random((rows, H, dh), 5, torch.bfloat16).to(DEV)
    q = _random((rows, 4, dh), 6, torch.bfloat16).to(DEV)
    for call in (lambda: pkg.read_blocks(cache, cu_rows=c, rows=rows), lambda: pkg.attend_blocks(q, cache, cu_new=c),
                 lambda: pkg.append_blocks(cache, k, k, cu_new=c)):
        pkg.check_status(cache)
        call()
        with pytest.raises(pkg.SphKVError, match="do not fit"):
            pkg.check_status(cache)


def test_recorded_calls_follow_lengths_and_offsets(pkg):
    """More sequences than a block deals by itself, recorded once in two graphs that replay in turn while lengths, offsets and firsts change on the
    device, in front of a bound of rows that is never reached."""
    B, H, N, dh, Hq, rows = 150, 2, 16, 64, 4, 700
    steps = [[(7 * b + 3 * i) % 9 for b in range(B)] for i in range(3)]
    final = [sum(s[b] for s in steps) + 1 for b in range(B)]
    caches = [_cache(pkg, [0] * B, H, N, dh, I8, 31, max_len=final) for _ in range(2)]
    k, v, q = (_random((3, rows, h, dh), 40 + h + i, torch.bfloat16).to(DEV) for i, h in enumerate((H, H, Hq)))
    held = [torch.zeros_like(x[0]) for x in (k, v, q)]
    cu, first = torch.zeros(B + 1, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)

    def step(cache, kk, vv, qq, c, f):
        pkg.append_blocks(cache, kk, vv, cu_new=c)
        out = torch.full((rows, Hq, dh), 7.0, dtype=torch.bfloat16, device=DEV)
        pkg.attend_blocks(qq, cache, cu_new=c, first=f, out=out)
        back = tuple(torch.full((rows, H, dh), 7.0, device=DEV) for _ in range(2))
        pkg.read_blocks(cache, cu_rows=c, out=back)
        return (out, pkg.decode_blocks(qq[:B], cache, first=f)) + back
    step(caches[1], *held, cu, first)  # nothing to do, but loads the kernels
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(caches[1], *held, cu, first))
        graphs.append(graph)
    lens = [0] * B
    for i, news in enumerate(steps):
        lens = [a + b for a, b in zip(lens, news)]
        for c in caches:
            c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(_cu(news))
        first.copy_(torch.tensor([n // 3 for n in lens], dtype=torch.int32))
        for x, y in zip(held, (k, v, q)):
            x.copy_(y[i])
        want = step(caches[0], k[i], v[i], q[i], cu, first)
        graphs[i % 2].replay()
        for a, b in zip(outs[i % 2], want):
            assert torch.equal(a, b)
        assert (want[0][sum(news):] == 7.0).all() and want[0][:sum(news)].isfinite().all()
    for c in caches:
        pkg.check_status(c)

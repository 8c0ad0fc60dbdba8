"""The 8-bit block cache on the GPU against its definition in 64 bits."""
import math

import pytest
import torch

import blocks_oracle as orc

pytestmark = pytest.mark.gpu
I8, E4M3 = torch.int8, torch.float8_e4m3fn
DEV = "cuda"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _table(lens, N, seed, spare=3, holes=True):
    """Random pages for sequences of these lengths; entries past the end are rubbish."""
    blocks = [max(1, -(-n // N)) for n in lens]
    P = sum(blocks) + spare
    order = torch.randperm(P, generator=_gen(seed)).to(torch.int32)
    t = torch.full((len(lens), max(blocks) + 1), 2 ** 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(blocks):
        t[b, :n] = order[at:at + n]
        at += n
    return t, P


def _rubbish(P, H, N, dh, store, seed):
    """Codes of every byte value (NaN codes among them), scales of the size of random data."""
    c = torch.randint(0, 256, (P, H, N, dh), generator=_gen(seed), dtype=torch.int32).to(torch.uint8)
    return c.view(store)


def _cache(pkg, lens, H, N, dh, store, seed, max_len=None):
    table, P = _table(max_len or lens, N, seed)
    nan = torch.full((P, H), math.nan)
    return pkg.BlockCache(_rubbish(P, H, N, dh, store, seed + 1).to(DEV), _rubbish(P, H, N, dh, store, seed + 2).to(DEV),
                          nan.to(DEV), nan.clone().to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))


def _random(shape, seed, dtype):
    g = _gen(seed)
    scale = torch.exp(0.5 * torch.randn(shape[-1], generator=g))
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _cu(news):
    return torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device=DEV)


def _filled(pkg, lens, H, N, dh, store, seed, dtype=torch.bfloat16):
    """A cache whose sequences hold random tokens, and what the definition says about it (from its own codes)."""
    cache = _cache(pkg, lens, H, N, dh, store, seed)
    k, v = _random((sum(lens), H, dh), seed + 5, dtype), _random((sum(lens), H, dh), seed + 6, dtype)
    pkg.append_blocks(cache, k.to(DEV), v.to(DEV), cu_new=_cu(lens))
    return cache


def _sides(cache):
    return orc.Cache(cache.k_codes, cache.k_scale), orc.Cache(cache.v_codes, cache.v_scale)


def _same(cache, sides, table, lens):
    for o, codes, scale in ((sides[0], cache.k_codes, cache.k_scale), (sides[1], cache.v_codes, cache.v_scale)):
        got = codes.cpu().float().double() if codes.dtype != I8 else codes.cpu().double()
        for b, n in enumerate(lens):
            for i in range(-(-n // o.N)):
                p, c = int(table[b, i]), min(o.N, n - i * o.N)
                assert torch.equal(scale[p].cpu().nan_to_num(123.0), o.scale[p].nan_to_num(123.0)), (b, i)
                assert torch.equal(got[p, :, :c], o.codes[p, :, :c]), (b, i)


@pytest.mark.parametrize("store", [I8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,dh", [(16, 128), (32, 64), (64, 128), (128, 64), (128, 128), (16, 64)])
def test_append_and_read(pkg, store, dtype, N, dh):
    H = 3
    steps = [[37, 0, 200, 1], [1, 1, 1, 1], [5, 130, 0, 15], [1, 1, 1, 1], [0, 0, 1, 64]]
    final = [sum(s[b] for s in steps) for b in range(4)]
    cache = _cache(pkg, [0] * 4, H, N, dh, store, 11, max_len=final)
    table = cache.block_table.cpu()
    sides, lens = _sides(cache), [0] * 4
    for i, news in enumerate(steps):
        grow = 1.0 + 0.7 * i  # pages that were begun need larger scales
        k, v = [_random((sum(news) + 2, H, dh), 100 + 2 * i + s, torch.float32).mul(grow).to(dtype) for s in (0, 1)]
        k[sum(news):], v[sum(news):] = math.nan, math.inf  # padding
        lens = [a + b for a, b in zip(lens, news)]
        cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        if len(set(news)) == 1 and i == 1:
            pkg.append_blocks(cache, k[:4].view(4, 1, H, dh).to(DEV), v[:4].view(4, 1, H, dh).to(DEV))
        else:
            pkg.append_blocks(cache, k.to(DEV), v.to(DEV), cu_new=_cu(news))
        at = 0
        for b, n in enumerate(news):
            if n:
                sides[0].append(table[b], lens[b], k[at:at + n])
                sides[1].append(table[b], lens[b], v[at:at + n])
            at += n
        _same(cache, sides, table, lens)
    pkg.check_status(cache)
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        back = [max(0, n - 7 * (b + 1)) for b, n in enumerate(final)]
        out = tuple(torch.full((sum(back) + 3, H, dh), 7.0, dtype=out_dtype, device=DEV) for _ in range(2))
        pkg.read_blocks(cache, cu_rows=_cu(back), out=out)
        n = 9
        ends = torch.tensor([n + b for b in range(4)], dtype=torch.int32, device=DEV)
        even = pkg.read_blocks(cache, n=n, ends=ends, out_dtype=out_dtype)
        for o, got, dense in zip(sides, out, even):
            want = torch.cat([o.rows(table[b], final[b] - m, final[b]) for b, m in enumerate(back)])
            # code * scale has at most 8 + 24 bits: one rounding to fp32, one to the output's type
            assert torch.equal(got[:-3].cpu(), want.float().to(out_dtype))
            assert (got[-3:] == 7.0).all()
            for b in range(4):
                assert torch.equal(dense[b].cpu(), o.rows(table[b], b, n + b).float().to(out_dtype))
    pkg.check_status(cache)


@pytest.mark.parametrize("store", [I8, E4M3])
def test_append_ties_tiny_and_not_finite(pkg, store):
    """One token a page of 16: rows of exact ties, of the smallest numbers, of zeros, of infinities and NaN."""
    top = orc.TOP[store]
    H, dh = 1, 128
    ties = (torch.arange(dh).float() - 64) * 0.5
    ties[0] = top                                     # scale 1: halves are ties of whole numbers
    fine = torch.linspace(-1, 1, dh) * 2.0 ** -9 * 8  # multiples of half an e4m3 step below 2^-6
    fine[0] = top
    near = torch.nextafter(torch.arange(dh).float() * 0.5 + 0.5, torch.tensor(0.0))
    near[0] = top
    rows = [ties, fine, near, torch.zeros(dh), torch.full((dh,), 2.0 ** -149), torch.full((dh,), top * 2.0 ** -126),
            torch.full((dh,), 3e38), torch.arange(dh).float() * 2.0 ** -140]
    odd = [ties.clone() for _ in range(3)]
    odd[0][5], odd[1][5], odd[2][5] = math.inf, math.nan, -math.inf
    rows = torch.stack(rows + odd)
    n = rows.shape[0]
    cache = _cache(pkg, [1] * n, H, 16, dh, store, 3, max_len=[2] * n)
    table, sides = cache.block_table.cpu(), _sides(cache)
    x = rows.view(n, 1, 1, dh)
    pkg.append_blocks(cache, x.to(DEV), -x.to(DEV))
    for b in range(n):
        sides[0].append(table[b], 1, x[b])
        sides[1].append(table[b], 1, -x[b])
    _same(cache, sides, table, [1] * n)
    # a second token: larger for some (the first is re-quantised), an infinity where there was none
    cache.seq_lens += 1
    y = rows.flip(0).view(n, 1, 1, dh) * 0.75
    pkg.append_blocks(cache, y.to(DEV), y.to(DEV))
    for b in range(n):
        sides[0].append(table[b], 2, y[b])
        sides[1].append(table[b], 2, y[b])
    _same(cache, sides, table, [2] * n)
    k, _ = pkg.read_blocks(cache, n=2)
    want = torch.stack([sides[0].rows(table[b], 0, 2) for b in range(n)]).float()
    assert torch.equal(k.cpu().nan_to_num(5.0), want.nan_to_num(5.0))
    assert k[n - 1].isnan().all() and not k[3].isnan().all()
    pkg.check_status(cache)


def test_append_strides(pkg):
    """Slices of a fused projection, rows off a 16-byte boundary, heads that are not next to each other."""
    H, dh, N = 2, 64, 16
    for pad, off in ((0, 0), (8, 8), (3, 1), (2, 0)):
        base = _random((30, 1, 3 * H * dh + pad), 5, torch.bfloat16).to(DEV)
        k = base.as_strided((30, H, dh), (3 * H * dh + pad, dh, 1), off)
        v = base.as_strided((30, H, dh), (3 * H * dh + pad, 2 * dh, 1), off + H * dh // 2)
        got, want = (_cache(pkg, [30], H, N, dh, I8, 3) for _ in range(2))
        pkg.append_blocks(got, k, v, cu_new=_cu([30]))
        pkg.append_blocks(want, k.contiguous(), v.contiguous(), cu_new=_cu([30]))
        for a, b in zip(pkg.read_blocks(got, n=30), pkg.read_blocks(want, n=30)):
            assert torch.equal(a, b)


def _check(got, want, off, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    err = (got.detach().cpu().double() - want).abs()
    ratio = float((err / (off + half * (want.abs() + off) + tiny)).max()) if err.isfinite().all() else math.inf
    assert ratio <= 1.0, ratio


@pytest.mark.parametrize("store", [I8, E4M3])
@pytest.mark.parametrize("N,dh,Hq,H,q_dtype,out_dtype", [
    (16, 128, 8, 2, torch.bfloat16, torch.bfloat16), (64, 128, 16, 2, torch.float32, torch.float32),
    (128, 64, 6, 2, torch.float16, torch.float32), (32, 64, 3, 3, torch.float32, torch.float16),
    (16, 128, 7, 1, torch.bfloat16, torch.float32), (128, 128, 20, 4, torch.float16, torch.float16)])
def test_decode(pkg, store, N, dh, Hq, H, q_dtype, out_dtype):
    lens = [1, 777, 0, 16, 17, 2500, 33]
    cache = _filled(pkg, lens, H, N, dh, store, 21)
    q = _random((len(lens), Hq, dh), 3, q_dtype)
    sides, table = _sides(cache), cache.block_table.cpu()
    for first in (None, [0, 500, 0, 16, 3, 2499, 40]):
        f = None if first is None else torch.tensor(first, dtype=torch.int32, device=DEV)
        part = torch.full((len(lens), Hq, dh + 2), 9.0, device=DEV)
        out = pkg.decode_blocks(q.to(DEV), cache, first=f, out_dtype=out_dtype, out_partial=part)
        for b, n in enumerate(lens):
            lo = min(n, 0 if first is None else first[b])
            k, v = (s.rows(table[b], lo, n).reshape(-1, H, dh) for s in sides)
            want, m, l, off, _, err = orc.attend(q[b:b + 1], k, v, lo, [n - 1], 1 / math.sqrt(dh))
            _check(out[b:b + 1], want, off, out_dtype)
            p = part[b].cpu().double()
            if lo == n:
                assert (out[b] == 0).all() and (p[:, 0] == -math.inf).all() and (p[:, 1:] == 0).all()
                continue
            assert bool(((p[:, 0] - m[0]).abs() <= err[0] + m[0].abs() * 2.0 ** -22).all())
            joined = p[:, 2:] / p[:, 1:2]
            _check(joined[None], want, off + want.abs() * 2.0 ** -22, torch.float32)
    pkg.check_status(cache)


def test_decode_long_and_many(pkg):
    """One long sequence over all workers, and more sequences than a block plans by itself."""
    dh, Hq, H = 128, 8, 2
    cache = _filled(pkg, [20011], H, 16, dh, I8, 31)
    q = _random((1, Hq, dh), 3, torch.float32)
    sides, table = _sides(cache), cache.block_table.cpu()
    out = pkg.decode_blocks(q.to(DEV), cache)
    want, _, _, off, size, _ = orc.attend(q, sides[0].rows(table[0], 0, 20011), sides[1].rows(table[0], 0, 20011), 0, [20010], 1 / math.sqrt(dh))
    _check(out, want, off, torch.float32)
    lens = [1 + (7 * b) % 50 for b in range(700)]
    lens[5] = 0
    cache = _filled(pkg, lens, 1, 16, 64, E4M3, 41)
    q = _random((700, 4, 64), 3, torch.bfloat16)
    sides, table = _sides(cache), cache.block_table.cpu()
    out = pkg.decode_blocks(q.to(DEV), cache)
    for b in list(range(0, 700, 37)) + [5, 699]:
        k, v = (s.rows(table[b], 0, lens[b]).reshape(-1, 1, 64) for s in sides)
        want, _, _, off, size, _ = orc.attend(q[b:b + 1], k, v, 0, [lens[b] - 1], 0.125)
        _check(out[b:b + 1], want, off, torch.bfloat16)
    pkg.check_status(cache)


@pytest.mark.parametrize("store", [I8, E4M3])
@pytest.mark.parametrize("N,dh,Hq,H,dtype", [(16, 128, 8, 2, torch.bfloat16), (64, 64, 3, 1, torch.float16),
                                             (128, 128, 7, 1, torch.bfloat16), (32, 64, 4, 4, torch.float16)])
def test_attend(pkg, store, N, dh, Hq, H, dtype):
    lens = [5, 777, 300, 129, 1, 0, 640]
    news = [5, 1, 150, 129, 1, 0, 131]
    cache = _filled(pkg, lens, H, N, dh, store, 51)
    sides, table = _sides(cache), cache.block_table.cpu()
    q = _random((sum(news) + 4, Hq, dh), 3, dtype)
    q[sum(news):] = math.nan
    for first in (None, [2, 776, 200, 300, 1, 0, 0]):
        f = None if first is None else torch.tensor(first, dtype=torch.int32, device=DEV)
        out = torch.full((sum(news) + 4, Hq, dh), 7.0, dtype=dtype, device=DEV)
        pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu(news), first=f, out=out)
        assert (out[sum(news):] == 7.0).all()
        at = 0
        for b, n in enumerate(news):
            lo = min(lens[b], 0 if first is None else first[b])
            k, v = (s.rows(table[b], lo, lens[b]).reshape(-1, H, dh) for s in sides)
            want, _, _, off, size, _ = orc.attend(q[at:at + n], k, v, lo, list(range(lens[b] - n, lens[b])), 1 / math.sqrt(dh))
            if n:
                # weights in f16 are off by half a step, finfo.eps / 2 = 2^-11 of each, and so is their weighted sum of |v|
                _check(out[at:at + n], want, off + torch.finfo(torch.float16).eps / 2 * size, dtype)
            at += n
    pkg.check_status(cache)


@pytest.mark.parametrize("store,N,dh,Hq,H", [(I8, 16, 128, 16, 4), (E4M3, 64, 64, 8, 2)])
def test_references_move(pkg, store, N, dh, Hq, H):
    """Many key tiles a worker, logits that grow along the sequence and values over twenty powers of two: maxima and the value scales'
    reference move all the time, in front of every part of a tile."""
    ctx, n = 9001, 150
    cache = _cache(pkg, [ctx], H, N, dh, store, 61)
    ramp = torch.linspace(0.05, 3.0, ctx)[:, None, None]
    k, v = _random((ctx, H, dh), 5, torch.float32) * ramp, _random((ctx, H, dh), 6, torch.float32) * torch.exp2(20 * torch.linspace(-1, 0, ctx))[:, None, None]
    pkg.append_blocks(cache, k.to(DEV), v.to(DEV), cu_new=_cu([ctx]))
    sides, table = _sides(cache), cache.block_table.cpu()
    kk, vv = (s.rows(table[0], 0, ctx) for s in sides)
    q = _random((n, Hq, dh), 3, torch.float16)
    want, _, _, off, size, _ = orc.attend(q, kk, vv, 0, list(range(ctx - n, ctx)), 1 / math.sqrt(dh))
    # a weight below 2^-14 is off by up to 2^-25 in f16, of weights up to 2^14 (the reference's slack 2^8, times 2^6) and as low as 2^6: the sum
    # of 2^-31 |v| over keys, relative to the largest scale
    tiny = ctx * 2.0 ** -31 * float(vv.abs().max())
    got = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu([n]), out_dtype=torch.float32)
    _check(got, want, off + torch.finfo(torch.float16).eps / 2 * size + tiny, torch.float32)
    got = pkg.decode_blocks(q[-1:].to(DEV), cache, out_dtype=torch.float32)
    _check(got, want[-1:], off[-1:] + tiny, torch.float32)
    # the other way round: the largest come first
    cache = _cache(pkg, [ctx], H, N, dh, store, 61)
    pkg.append_blocks(cache, k.flip(0).to(DEV), v.flip(0).to(DEV), cu_new=_cu([ctx]))
    sides = _sides(cache)
    kk, vv = (s.rows(table[0], 0, ctx) for s in sides)
    want, _, _, off, size, _ = orc.attend(q, kk, vv, 0, list(range(ctx - n, ctx)), 1 / math.sqrt(dh))
    got = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu([n]), out_dtype=torch.float32)
    _check(got, want, off + torch.finfo(torch.float16).eps / 2 * size + tiny, torch.float32)
    pkg.check_status(cache)


def test_attend_shapes(pkg):
    """The even form, one token and the decode kernel's few, strided queries, outputs of other types, more blocks of queries than a CTA
    deals by itself, and a recorded call."""
    H, N, dh, Hq = 2, 32, 128, 8
    lens = [90, 200, 33]
    cache = _filled(pkg, lens, H, N, dh, I8, 71)
    sides, table = _sides(cache), cache.block_table.cpu()
    for n in (1, 2, 3, 20):
        base = _random((3, n, Hq + 2, dh + 8), 3, torch.bfloat16).to(DEV)
        for q in (base[:, :, :Hq, :dh], base[:, :, 1:Hq + 1, 3:dh + 3]):
            for out_dtype in (torch.bfloat16, torch.float32):
                out = pkg.attend_blocks(q, cache, out_dtype=out_dtype)
                assert out.shape == (3, n, Hq, dh) and out.dtype == out_dtype
                for b in range(3):
                    kk, vv = (s.rows(table[b], 0, lens[b]) for s in sides)
                    want, _, _, off, size, _ = orc.attend(q[b].cpu(), kk, vv, 0, list(range(lens[b] - n, lens[b])), 1 / math.sqrt(dh))
                    _check(out[b], want, off + torch.finfo(torch.float16).eps / 2 * size, out_dtype)
    q = _random((3, 20, Hq, dh), 3, torch.bfloat16).to(DEV)
    want = pkg.attend_blocks(q, cache)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = pkg.attend_blocks(q, cache)
    for _ in range(2):
        out.zero_()
        gr.replay()
        assert torch.equal(out, want)
    many = [40 + b % 3 for b in range(150)]
    cache = _filled(pkg, many, 1, 16, 64, E4M3, 81)
    sides, table = _sides(cache), cache.block_table.cpu()
    q = _random((sum(many), 4, 64), 3, torch.float16)
    out = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu(many))
    for b in range(0, 150, 13):
        kk, vv = (s.rows(table[b], 0, many[b]) for s in sides)
        at = sum(many[:b])
        want, _, _, off, size, _ = orc.attend(q[at:at + many[b]], kk, vv, 0, list(range(many[b])), 0.125)
        _check(out[at:at + many[b]], want, off + torch.finfo(torch.float16).eps / 2 * size, torch.float16)
    pkg.check_status(cache)


def test_padding_bad_tables_and_lengths(pkg):
    H, N, dh = 2, 16, 128
    cache = _filled(pkg, [40, 40, 40, 40], H, N, dh, I8, 61)
    good = pkg.read_blocks(cache, n=40)
    q = _random((4, 4, dh), 3, torch.bfloat16).to(DEV)
    want = pkg.decode_blocks(q, cache)
    pkg.check_status(cache)
    # a page number out of range: its tokens are absent
    before = cache.block_table.clone()
    cache.block_table[1, 1] = cache.k_codes.shape[0]
    cache.block_table[2, 0] = -1
    got = pkg.read_blocks(cache, n=40)
    with pytest.raises(pkg.SphKVError, match="block-table"):
        pkg.check_status(cache)
    for a, b in zip(got, good):
        assert torch.equal(a[0], b[0]) and torch.equal(a[3], b[3])
        assert (a[1, 16:32] == 0).all() and torch.equal(a[1, 32:], b[1, 32:]) and (a[2, :16] == 0).all()
    out = pkg.decode_blocks(q, cache)
    with pytest.raises(pkg.SphKVError, match="block-table"):
        pkg.check_status(cache)
    assert torch.equal(out[0], want[0]) and torch.equal(out[3], want[3]) and out.isfinite().all()
    cache.block_table.copy_(before)
    # lengths that the table has no room for, or that are shorter than the new tokens
    state = [t.clone() for t in (cache.k_codes, cache.k_scale)]
    cache.seq_lens.copy_(torch.tensor([40, 10 ** 6, -1, 2], dtype=torch.int32))
    k = _random((4, 3, H, dh), 5, torch.float32).to(DEV)
    pkg.append_blocks(cache, k, k)
    with pytest.raises(pkg.SphKVError, match="do not fit"):
        pkg.check_status(cache)
    kept = [int(p) for p in before[0, :3].tolist()]
    for t, s in zip((cache.k_codes, cache.k_scale), state):
        t = t.clone()
        t[kept] = s[kept]
        assert torch.equal(t.view(torch.uint8), s.view(torch.uint8))  # bytes: unused pages have NaN scales
    cache.seq_lens.fill_(40)
    out = torch.full((9, 4, dh), 7.0, dtype=torch.bfloat16, device=DEV)
    pkg.attend_blocks(_random((9, 4, dh), 3, torch.bfloat16).to(DEV), cache, out=out,
                      cu_new=torch.tensor([0, 2, 1, 4, 9], dtype=torch.int32, device=DEV))
    with pytest.raises(pkg.SphKVError, match="do not fit"):
        pkg.check_status(cache)
    assert out.isfinite().all()


def test_refusals(pkg):
    H, N, dh = 2, 16, 128
    cache = _filled(pkg, [40, 20], H, N, dh, I8, 61)
    q, k = _random((2, 4, dh), 3, torch.bfloat16).to(DEV), _random((2, 1, H, dh), 3, torch.bfloat16).to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    bad = [lambda: pkg.decode_blocks(q, cache, first=[0, 0]), lambda: pkg.decode_blocks(q, cache, first=torch.zeros(2, device=DEV)),
           lambda: pkg.decode_blocks(q, cache, first=torch.zeros(3, **i32)), lambda: pkg.decode_blocks(q, cache, first=torch.zeros(2, dtype=torch.int32)),
           lambda: pkg.decode_blocks(q[:1], cache), lambda: pkg.decode_blocks(q[..., :64], cache), lambda: pkg.decode_blocks(q.double(), cache),
           lambda: pkg.decode_blocks(q.transpose(1, 2).contiguous().transpose(1, 2), cache), lambda: pkg.decode_blocks(q[:, :3], cache),
           lambda: pkg.decode_blocks(torch.cat([q] * 5, 1), cache), lambda: pkg.decode_blocks(q, cache, out=q[:, :2]),
           lambda: pkg.decode_blocks(q, cache, out_dtype=torch.int8), lambda: pkg.decode_blocks(q, cache, out_partial=torch.zeros(2, 4, dh, device=DEV)),
           lambda: pkg.decode_blocks(q, cache, want_out=False), lambda: pkg.decode_blocks(q.cpu(), cache),
           lambda: pkg.append_blocks(cache, k, k.float()), lambda: pkg.append_blocks(cache, k[:, 0], k[:, 0]), lambda: pkg.append_blocks(cache, k[:, :, :1], k[:, :, :1]),
           lambda: pkg.append_blocks(cache, k[:, 0], k[:, 0], cu_new=torch.zeros(2, **i32)), lambda: pkg.append_blocks(cache, k, [1, 2]),
           lambda: pkg.append_blocks(cache, k.expand(2, 3, H, dh)[:, ::2].contiguous()[:, :1].expand(2, 2, H, dh), k.expand(2, 2, H, dh)),
           lambda: pkg.read_blocks(cache), lambda: pkg.read_blocks(cache, n=2, cu_rows=torch.zeros(3, **i32)), lambda: pkg.read_blocks(cache, n=-1),
           lambda: pkg.read_blocks(cache, cu_rows=torch.zeros(3, **i32)), lambda: pkg.read_blocks(cache, n=2, out=(q, q)),
           lambda: pkg.read_blocks(cache, n=2, out_dtype=torch.float64), lambda: pkg.attend_blocks(q[:, None].float(), cache),
           lambda: pkg.attend_blocks(q, cache), lambda: pkg.attend_blocks(q, cache, cu_new=torch.zeros(2, **i32))]
    for n, call in enumerate(bad):
        with pytest.raises(pkg.SphKVError):
            call()
            print("call", n, "was taken")
    for field, wrong in (("k_scale", cache.k_scale.half()), ("v_codes", cache.v_codes[:, :, :, :64].contiguous()), ("block_table", cache.block_table.long()),
                         ("k_codes", cache.k_codes.transpose(0, 1)), ("seq_lens", cache.seq_lens.long()), ("status", torch.zeros(1, device=DEV))):
        other = pkg.BlockCache(**{**cache.__dict__, field: wrong})
        with pytest.raises(pkg.SphKVError):
            pkg.decode_blocks(q, other)
    # nothing to do is no error
    assert pkg.read_blocks(cache, n=0)[0].shape == (2, 0, H, dh)
    pkg.append_blocks(cache, k[:, :0], k[:, :0])
    assert pkg.attend_blocks(q[:, None][:, :0], cache).shape == (2, 0, 4, dh)
    pkg.check_status(cache)


def test_nan_pages_stay_where_they_are_seen(pkg):
    """A page that reads back as NaN reaches the rows that see it, and no others."""
    H, N, dh = 1, 16, 64
    lens = [200, 200]
    cache = _filled(pkg, lens, H, N, dh, I8, 71)
    for scales in (cache.k_scale, cache.v_scale):
        clean = scales.clone()
        q = _random((2, 100, 4, dh), 3, torch.bfloat16).to(DEV)
        want = pkg.attend_blocks(q, cache)
        scales[int(cache.block_table[1, 9])] = math.nan  # tokens 144 .. 159 of the second sequence
        got = pkg.attend_blocks(q, cache)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1, :44], want[1, :44]) and got[1, 44:].isnan().all()
        first = torch.tensor([0, 160], dtype=torch.int32, device=DEV)
        got = pkg.attend_blocks(q, cache, first=first)
        assert got.isfinite().all() and (got[1, :60] == 0).all()
        assert pkg.decode_blocks(q[:, -1], cache)[1].isnan().all()
        assert pkg.decode_blocks(q[:, -1], cache, first=first).isfinite().all()
        scales.copy_(clean)


@pytest.mark.parametrize("big", [2.0 ** 30, 2.0 ** 70, 1e36])
def test_scales_that_are_not_seen(pkg, big):
    """Rows do not lose bits to a larger value that only later rows see (down to 2^-80 of it), and pages whose value scale is smaller still
    keep their part in the sums of weights."""
    H, N, dh, Hq, ctx, n = 1, 16, 128, 8, 700, 150
    cache = _cache(pkg, [ctx], H, N, dh, I8, 91)
    k, v = _random((ctx, H, dh), 5, torch.float32), _random((ctx, H, dh), 6, torch.float32)
    v[ctx - 30] *= big
    v[:600] *= 2.0 ** -60 if big == 1e36 else 1.0
    pkg.append_blocks(cache, k.to(DEV), v.to(DEV), cu_new=_cu([ctx]))
    sides, table = _sides(cache), cache.block_table.cpu()
    kk, vv = (s.rows(table[0], 0, ctx) for s in sides)
    q = _random((n, Hq, dh), 3, torch.float16)
    got = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu([n]), out_dtype=torch.float32)
    # the page's 16 tokens share the large scale
    see = (ctx - 30) // N * N - (ctx - n)
    for lo, hi in ((0, see), (see, n))[big == 1e36:]:
        want, _, _, off, size, _ = orc.attend(q[lo:hi], kk, vv, 0, list(range(ctx - n + lo, ctx - n + hi)), 1 / math.sqrt(dh))
        last = ctx - n + hi
        # weights below 2^-14 are off by 2^-25 where the row's largest weight times scale is 2^6 at least, and that is no more than what
        # the row's values, scale by scale, weigh: keys * 2^-31 * the largest scale * 127 that the row sees
        tiny = last * 2.0 ** -31 * float(vv[:last].abs().max())
        _check(got[lo:hi], want, off + torch.finfo(torch.float16).eps / 2 * size + tiny, torch.float32)
    pkg.check_status(cache)


def test_value_scales_of_zero(pkg):
    """A value is code * scale: pages of scale 0 are zeros whatever their codes, and count in the sum of weights."""
    H, N, dh, Hq, ctx = 2, 16, 64, 8, 400
    cache = _filled(pkg, [ctx], H, N, dh, I8, 95)
    table = cache.block_table.cpu()
    for zero in ([3, 4, 20], list(range(25)), list(range(0, 16))):
        cache.v_scale[table[0, zero].long().to(DEV)] = 0
        sides = _sides(cache)
        kk, vv = (s.rows(table[0], 0, ctx) for s in sides)
        for n in (1, 200):
            q = _random((n, Hq, dh), 3, torch.bfloat16)
            want, _, _, off, size, _ = orc.attend(q, kk, vv, 0, list(range(ctx - n, ctx)), 0.125)
            got = pkg.attend_blocks(q.to(DEV), cache, cu_new=_cu([n]), out_dtype=torch.float32)
            _check(got, want, off + torch.finfo(torch.float16).eps / 2 * size, torch.float32)
            got = pkg.decode_blocks(q[-1:].to(DEV), cache, out_dtype=torch.float32)
            _check(got, want[-1:], off[-1:], torch.float32)
        cache.v_scale[:] = 0.01
    pkg.check_status(cache)


def test_streams_and_graphs(pkg):
    """A decode step recorded into two graphs that replay over growing lengths, and the same on another stream."""
    H, N, dh, Hq = 2, 16, 128, 8
    lens = [30, 100]
    steps = 5
    caches = [_cache(pkg, lens, H, N, dh, I8, 81, max_len=[n + steps for n in lens]) for _ in range(3)]
    k0 = _random((sum(lens), H, dh), 5, torch.bfloat16).to(DEV)
    for c in caches:
        pkg.append_blocks(c, k0, k0, cu_new=_cu(lens))
    q, k = _random((steps, 2, Hq, dh), 3, torch.bfloat16).to(DEV), _random((steps, 2, 1, H, dh), 4, torch.bfloat16).to(DEV)
    want = []
    for i in range(steps):
        caches[0].seq_lens += 1
        pkg.append_blocks(caches[0], k[i], k[i])
        want.append(pkg.decode_blocks(q[i], caches[0]))
    qs, ks = q[0].clone(), k[0].clone()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            caches[1].seq_lens += 1
            pkg.append_blocks(caches[1], ks, ks)
            outs.append(pkg.decode_blocks(qs, caches[1]))
        graphs.append(gr)
    for i in range(steps):
        qs.copy_(q[i])
        ks.copy_(k[i])
        graphs[i % 2].replay()
        assert torch.equal(outs[i % 2], want[i])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(steps):
            caches[2].seq_lens += 1
            pkg.append_blocks(caches[2], k[i], k[i])
            got = pkg.decode_blocks(q[i], caches[2])
    side.synchronize()
    assert torch.equal(got, want[-1])
    for c in caches:
        pkg.check_status(c)


def test_merged_with_spherical_pages(pkg):
    """The oldest tokens move into bit-packed pages, the rest stays in 8 bits; both decodes merge to attention over all."""
    B, Hq, H, dh, N, ctx, old = 2, 8, 2, 128, 16, 500, 300
    cache = _filled(pkg, [ctx] * B, H, N, dh, I8, 91, torch.float32)
    ends = torch.full((B,), old, dtype=torch.int32, device=DEV)
    k, v = pkg.read_blocks(cache, n=old, ends=ends)
    tiers = pkg.TierSet(dh, pkg.REFERENCE_TIERS[:1])
    books = pkg.synth.make_codebooks(H, dh, pkg.REFERENCE_TIERS[:1])
    assign = torch.ones(B, H, old, dtype=torch.uint8, device=DEV)
    pages = pkg.encode_pages(k.view(B * old, H, dh), v.view(B * old, H, dh), pkg.build_page_lists(assign, tiers, N),
                             tiers.pack_codebooks(books).to(DEV), tiers)
    q = _random((B, Hq, dh), 3, torch.float32).to(DEV)
    parts = torch.empty(2, B, Hq, dh + 2, device=DEV)
    a = pkg.decode_paged(q, pages, None, out_partial=parts[0])
    pkg.decode_blocks(q, cache, first=ends, out_partial=parts[1], want_out=False)
    got = pkg.merge_partials(parts.view(2, B * Hq, dh + 2)).view(B, Hq, dh)
    # attention over both sets, from the paged decode's own partial and the definition of the 8-bit one
    sides, table = _sides(cache), cache.block_table.cpu()
    p = parts[0].cpu().double()
    assert torch.allclose(p[..., 2:] / p[..., 1:2], a.cpu().double(), rtol=0, atol=1e-5)
    for b in range(B):
        kk, vv = (s.rows(table[b], old, ctx) for s in sides)
        want, m, l, off, _, _ = orc.attend(q[b:b + 1], kk, vv, old, [ctx - 1], 1 / math.sqrt(dh))
        top = torch.maximum(m[0], p[b, :, 0])
        wa, wb = torch.exp(p[b, :, 0] - top) * p[b, :, 1], torch.exp(m[0] - top) * l[0]
        whole = (torch.exp(p[b, :, 0] - top)[:, None] * p[b, :, 2:] + wb[:, None] * want[0]) / (wa + wb)[:, None]
        # relative weight of the two sets: exp of maxima in fp32 (2^-22 of up to |max|), and the parts' own bounds
        slack = (off[0] + (m[0].abs()[:, None] + 1) * 2.0 ** -20 * (want[0].abs() + a[b].cpu().double().abs()))
        _check(got[b], whole, slack, torch.float32)
    pkg.check_status(cache)
    pkg.check_status(pages)

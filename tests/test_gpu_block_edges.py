"""The 8-bit block cache on the GPU where it can go wrong: what the other tests of it do not reach."""
import math

import pytest
import torch

from test_gpu_blocks import DEV, E4M3, I8, _cache, _check, _cu, _filled, _random, _sides
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

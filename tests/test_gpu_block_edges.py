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

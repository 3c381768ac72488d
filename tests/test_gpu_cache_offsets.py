"""Offsets that reach past the rows of a call are cut to them, and the rows'
positions follow from what is left, in every form of the streams' operators."""
import pytest
import torch

import trispconv.pytorch as spconv
from cache_oracle import attend_pages64, ints, offsets_of, scatter, tables
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import check

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.float32, 64), (torch.bfloat16, 32)])
@pytest.mark.parametrize("lq", [[2], [1, 2], [7, 1, 31], [100, 40]])
@pytest.mark.parametrize("unseen", [1.0, float("nan")])
@pytest.mark.parametrize("prefix", [0, 2])
def test_attention(prefix, unseen, lq, dtype, dim):
    """The last sample's offset is past the last row, the first one's before the
    first: with a prefix (read for all rows at once) and without, what those of
    the rows that there are say."""
    page = 64
    # (windows reach back over the prefix's end)
    lk = [page * prefix + n + 3 * b for b, n in enumerate(lq)]
    g = torch.Generator().manual_seed(3)
    table, pages = tables(lk, page, prefix)
    q = torch.randn(sum(lq), 4, dim, generator=g).to(dtype)
    k, v = (torch.randn(pages, page, 2, dim, generator=g).to(dtype) for _ in range(2))
    if prefix:
        k[table[0, 1], 80 - page], v[table[0, 1], 80 - page] = unseen, unseen
    want = attend_pages64(q, k, v, table, lq, lk, (40, 0), 3)
    for past in (0, 3, 1 << 20):
        off = offsets_of(lq)
        off[-1] += past
        off[0] -= past
        say("cache_attention, offsets", off.tolist(), lk, prefix, dtype, dim)
        got = spconv.cache_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), off.to(DEV), ints(lk).to(DEV),
                                     prefix=table[0, :prefix].to(DEV) if prefix else None, window=(40, 0), sinks=3)
        check(got, *want, what=f"{past}")


@pytest.mark.parametrize("dim", [32, 6])
def test_append(dim):
    lq, lk, page = [3, 12], [3, 20], 4
    g = torch.Generator().manual_seed(4)
    table, pages = tables(lk, page)
    q, k, v = (torch.randn(15, 2, dim, generator=g) for _ in range(3))
    pos = torch.randint(0, 99, (15, 3), generator=g, dtype=torch.int32)
    want = torch.zeros(pages, page, 2, dim)
    scatter(want, table, 0, v[:3], 0)
    scatter(want, table, 1, v[3:], 8)
    keys = None
    for past in (0, 3, 1 << 20):
        off = offsets_of(lq)
        off[-1] += past
        off[0] -= past
        say("norm_rotate_append, offsets", off.tolist(), dim)
        kp, vp = (torch.zeros(pages, page, 2, dim, device=DEV) for _ in range(2))
        spconv.norm_rotate_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), kp, vp, table.to(DEV),
                                  off.to(DEV), ints(lk).to(DEV))
        assert torch.equal(vp.cpu(), want), past
        keys = kp if keys is None else keys
        assert torch.equal(kp, keys), past

"""cache_attention's steps of many rows, over long and scattered caches: single
rows of the results against the 64-bit form."""
import pytest
import torch

import trispconv.pytorch as spconv
from cache_oracle import gather, ints, offsets_of, tables
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import attend64, check

pytestmark = [pytest.mark.gpu, needs_gpu]


def _rows_of(q, k, v, table, lq, lk, left, sinks, rows, got):
    """Rows (sample, row of it), which see the positions up to their own."""
    at = offsets_of(lq).tolist()
    for b, i in rows:
        i %= lq[b]
        n = lk[b] - lq[b] + i + 1
        t = at[b] + i
        ref, tol = attend64(q[t:t + 1], gather(k, table, b, n), gather(v, table, b, n), [1], [n],
                            (left, 0), sinks)
        check(got[t:t + 1], ref, tol, what=f"sample {b} row {i}")


def _case(lq, lk, hq, hk, dim, dtype, page, prefix=0):
    g = torch.Generator().manual_seed(1)
    table, pages = tables(lk, page, prefix)
    q = torch.randn(sum(lq), hq, dim, generator=g).to(dtype)
    k, v = (torch.randn(pages, hk, page, dim, generator=g).to(dtype).transpose(1, 2) for _ in range(2))
    return q, k, v, table


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq,lk,hq,hk,dim,page,left,sinks,prefix", [
    ([2048, 2008], [9000, 8003], 16, 4, 64, 64, None, 0, 0),      # 64 rows a wave, in parts
    ([2048, 2008], [9000, 8003], 16, 4, 64, 16, 3000, 70, 0),
    ([2048, 2008], [9000, 8003], 16, 4, 64, 20, None, 0, 0),
    ([129] * 16, [5000 + 3 * b for b in range(16)], 16, 4, 64, 64, None, 0, 0),  # parts that are not made
    ([129] * 16, [5000 + 3 * b for b in range(16)], 16, 4, 40, 64, 700, 5, 0),
    ([512, 342, 172, 2], [6000, 5000, 4001, 3002], 16, 4, 64, 64, None, 0, 16),
    ([300, 1, 77], [4000, 3900, 3777], 8, 2, 128, 32, None, 0, 0),
    ([300, 1, 77], [4000, 3900, 3777], 8, 2, 96, 64, 2000, 9, 31),
    ([300, 1, 77], [2000, 1900, 1777], 4, 2, 256, 64, None, 0, 0),
    ([100] * 3, [9000, 8000, 8500], 32, 1, 32, 64, None, 0, 100),
])
def test_against_single_rows(lq, lk, hq, hk, dim, page, left, sinks, prefix, dtype):
    say("many rows:", lq, lk, hq, hk, dim, page, left, sinks, prefix, dtype)
    q, k, v, table = _case(lq, lk, hq, hk, dim, dtype, page, prefix)
    got = spconv.cache_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), offsets_of(lq).to(DEV),
                                 ints(lk).to(DEV), prefix=table[0, :prefix].to(DEV) if prefix else None,
                                 window=(left, 0), sinks=sinks).cpu()
    assert torch.isfinite(got).all()
    last = len(lq) - 1
    rows = [(0, 0), (0, 63), (0, 64), (0, -1), (last // 2, 0), (last // 2, 100), (last, 0), (last, -1)]
    _rows_of(q, k, v, table, lq, lk, left, sinks, rows, got)


@pytest.mark.parametrize("lq", [[1, 1], [300, 200]])
def test_rows_of_2_to_the_31_elements_and_more(lq):
    """Pages whose rows lie past 2^31 elements and 2^32 bytes."""
    rows, hk, dim, lk = 64, 4, 256, [500, 400]
    pages = (1 << 31) // (rows * hk * dim) + 40
    k, v = (torch.empty(pages, rows, hk, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.randperm(24)[:16].view(2, 8).to(torch.int32) + pages - 24
    table[0, 0] = 3
    q = torch.randn(sum(lq), 4, dim).to(torch.bfloat16)
    new = [torch.randn(sum(lk), hk, dim).to(torch.bfloat16) for _ in range(2)]
    pos = torch.zeros(sum(lk), 1, device=DEV)
    args = [table.to(DEV), offsets_of(lk).to(DEV), ints(lk).to(DEV)]
    spconv.norm_rotate_append(new[0].to(DEV), new[0].to(DEV), new[1].to(DEV), pos, k, v, *args)
    _, kn = spconv.norm_rotate_heads(new[0].to(DEV), new[0].to(DEV), pos)
    got = spconv.cache_attention(q.to(DEV), k, v, args[0], offsets_of(lq).to(DEV), args[2], window=(None, 0))
    at_q, at_k = offsets_of(lq).tolist(), offsets_of(lk).tolist()
    for b, i in ((0, 0), (0, -1), (1, 0), (1, -1)):
        i %= lq[b]
        n, t = lk[b] - lq[b] + i + 1, at_q[b] + i
        s = slice(at_k[b], at_k[b] + n)
        ref, tol = attend64(q[t:t + 1], kn[s].cpu(), new[1][s], [1], [n], (None, 0), 0)
        check(got[t:t + 1], ref, tol, what=f"{b} {i}")


@pytest.mark.parametrize("lq", [[1] * 4, [700, 600, 1, 30]])
def test_two_streams_at_once(lq):
    """Calls that run beside each other, each with a workspace of its own."""
    lk = [9000, 4000, 5000, 800]
    cases = []
    for seed in range(2):
        q, k, v, table = (t.to(DEV) for t in _case(lq, lk, 8, 2, 64, torch.float16, 64))
        args = (q + seed, k, v, table, offsets_of(lq).to(DEV), ints(lk).to(DEV))
        cases.append((args, spconv.cache_attention(*args, window=(None, 0))))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        outs = []
        for stream, (args, _) in zip(streams, cases):
            with torch.cuda.stream(stream):
                outs.append(spconv.cache_attention(*args, window=(None, 0)))
        torch.cuda.synchronize()
        for out, (_, want) in zip(outs, cases):
            assert torch.equal(out, want)


def test_offsets_that_decrease_stay_inside():
    """Results unspecified, nothing outside the tensors is touched."""
    q, k, v, table = (t.to(DEV) for t in _case([40, 40, 40], [300, 200, 250], 4, 2, 64, torch.float16, 64))
    n = ints([300, 200, 250]).to(DEV)
    for off in ([0, 120, 3, 90], [120, 0, 120, 0], [-5, 500, -9, 1 << 30], [0, 0, 0, 1 << 30]):
        off = ints(off).to(DEV)
        for prefix in (None, table[0, :2].clone()):
            out = spconv.cache_attention(q, k, v, table, off, n, prefix=prefix, window=(None, 0))
            torch.cuda.synchronize()
            assert out.shape == q.shape
        for lk in ([1 << 30, -1, 0], [0, 0, 0]):
            spconv.cache_attention(q, k, v, table, off, ints(lk).to(DEV))
        torch.cuda.synchronize()

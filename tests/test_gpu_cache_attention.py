"""cache_attention against the 64-bit form: pages, rows a step, masks, prefixes."""
import pytest
import torch

import trispconv.pytorch as spconv
from cache_oracle import attend_pages64, gather, ints, offsets_of, tables
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import check, seen

pytestmark = [pytest.mark.gpu, needs_gpu]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _case(lq, lk, hq, hk, dim, dtype, page, prefix=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    table, pages = tables(lk, page, prefix, seed=seed)
    q = torch.randn(sum(lq), hq, dim, generator=g).to(dtype)
    k, v = (torch.randn(pages, page, hk, dim, generator=g).to(dtype) for _ in range(2))
    # what no sample keeps: rows of free pages and those past the last positions
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lk):
        j = torch.arange(n)
        used[table[b].long()[j // page], j % page] = True
    k[~used], v[~used] = float("nan"), float("inf")
    return q, k, v, table


def _run(q, k, v, table, lq, lk, window, sinks=0, prefix=0, scale=None, head_major=True):
    if head_major:
        k, v = (t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    return spconv.cache_attention(
        q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), offsets_of(lq).to(DEV), ints(lk).to(DEV),
        prefix=table[0, :prefix].to(DEV) if prefix else None, window=window, sinks=sinks, scale=scale)


def _check(lq, lk, hq, hk, dim, dtype, page, window=(None, 0), sinks=0, prefix=0, **more):
    say("cache_attention", lq, lk, hq, hk, dim, dtype, page, window, sinks, prefix)
    q, k, v, table = _case(lq, lk, hq, hk, dim, dtype, page, prefix)
    got = _run(q, k, v, table, lq, lk, window, sinks, prefix, **more)
    check(got, *attend_pages64(q, k, v, table, lq, lk, window, sinks), what=f"{lq} {lk}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 2, 7, 16, 20, 32, 48, 64, 96, 128, 300])
def test_pages(page, dtype):
    _check([1, 1, 1, 1], [1, 63, 290, 641], 4, 2, 64, dtype, page)
    _check([40, 1, 25], [300, 130, 25], 4, 2, 64, dtype, page, head_major=False)
    _check([150, 0, 70], [400, 13, 70], 4, 4, 32, dtype, page, window=(90, 10), sinks=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,dim", [(1, 1, 1), (2, 1, 7), (3, 3, 16), (6, 2, 24), (5, 1, 40),
                                       (2, 2, 48), (4, 4, 72), (2, 1, 80), (3, 1, 96), (2, 2, 100),
                                       (8, 2, 128), (2, 1, 136), (1, 1, 200), (2, 1, 256),
                                       (17, 1, 64), (32, 1, 64), (48, 1, 32), (80, 2, 64)])
def test_heads(hq, hk, dim, dtype):
    for lq, lk, window, sinks in (([1, 1, 1], [1, 77, 300], (None, 0), 0),
                                  ([5, 3], [200, 90], (60, 0), 3),
                                  ([150, 77], [200, 77], (50, 20), 3)):
        _check(lq, lk, hq, hk, dim, dtype, 32, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 8, 15, 16, 17, 31, 40, 64, 65, 129, 300])
def test_rows_a_step(rows, dtype):
    """From one new row to many, for samples that kept much, little and nothing."""
    for window, sinks in (((None, 0), 0), ((100, 5), 4), ((None, None), 0)):
        _check([rows] * 3, [rows + 500, rows + 1, rows], 4, 2, 64, dtype, 64, window, sinks)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.float16, 32), (torch.bfloat16, 64),
                                       (torch.bfloat16, 128), (torch.float32, 256)])
@pytest.mark.parametrize("lq,lk,prefix", [([1, 1, 1, 1, 0], [2600, 1, 700, 257, 300], 0),
                                          ([3, 0, 16], [513, 20, 1500], 0), ([1, 2], [900, 300], 4)])
def test_tables_with_far_more_room(dtype, dim, lq, lk, prefix):
    """Parts follow what is kept, not the 40,000 positions that the table has room for."""
    q, k, v, table = _case(lq, lk, 4, 2, dim, dtype, 32, prefix)
    wide = torch.full((len(lk), 1250), 1 << 30, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    for window, sinks in (((None, 0), 0), ((400, 0), 5)):
        say("cache_attention, room", lq, lk, dim, dtype, prefix, window, sinks)
        check(_run(q, k, v, wide, lq, lk, window, sinks, prefix),
              *attend_pages64(q, k, v, table, lq, lk, window, sinks), what=f"{lq} {lk} {window}")


@pytest.mark.parametrize("samples,rows,keys,hq,hk,dim", [(1, 16, 5000, 16, 4, 64), (4, 4, 900, 16, 4, 64),
                                                         (4, 2, 700, 32, 2, 96), (3, 16, 600, 16, 4, 128),
                                                         (2, 32, 600, 4, 2, 256), (9, 5, 333, 24, 3, 32)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tiles_of_some_rows(samples, rows, keys, hq, hk, dim, dtype):
    """Tiles of 16, 32 and 64 rows, whole and not, of one sample and of several."""
    _check([rows] * samples, [keys - 7 * b for b in range(samples)], hq, hk, dim, dtype, 64)
    _check([rows, *[1] * (samples - 1)], [keys] * samples, hq, hk, dim, dtype, 64, window=(300, 2), sinks=9)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [((None, None), 0), ((0, 0), 0), ((63, 0), 0), ((64, 0), 16),
                                          ((100, 0), 70), ((100, 0), 1000), ((5, None), 2),
                                          ((0, 0), 1), ((1000, 0), 600)])
def test_windows(window, sinks, dtype):
    _check([1, 1, 1], [700, 64, 3], 4, 1, 64, dtype, 64, window, sinks)
    _check([1, 30, 4], [700, 690, 300], 4, 1, 64, dtype, 16, window, sinks)
    _check([260, 3], [700, 300], 4, 4, 64, dtype, 64, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,prefix", [(64, 1), (64, 9), (16, 20), (20, 13), (1, 5)])
def test_prefix(page, prefix, dtype):
    first = page * prefix
    for lq, own in (([1] * 5, [1, 2, 70, 130, 1]), ([1] * 70, [1 + i for i in range(70)]),
                    ([7, 1, 20], [7, 100, 33]), ([200, 0, 30], [230, 0, 30])):
        lk = [first + n for n in own]
        for window, sinks in (((None, 0), 0), ((90, 0), 5)):
            _check(lq, lk, 4, 2, 64, dtype, page, window, sinks, prefix)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,dim", [(1, 1, 7), (5, 1, 40), (8, 8, 32), (8, 2, 128), (2, 1, 256),
                                       (16, 1, 96)])
def test_prefix_heads(hq, hk, dim, dtype):
    _check([1] * 9, [512 + 3 * i + 1 for i in range(9)], hq, hk, dim, dtype, 32, prefix=16)
    _check([30, 2], [512 + 33, 512 + 2], hq, hk, dim, dtype, 32, prefix=16)


def test_prefix_of_samples_shorter_than_it():
    """A sample may end within the prefix, or keep nothing."""
    lq, lk = [1, 2, 1, 0], [40, 150, 130, 0]
    q, k, v, table = _case(lq, lk, 4, 2, 64, torch.float16, 32, prefix=0)
    table[:] = table[1].clone()  # 150 positions in five pages, the same for all
    want = attend_pages64(q, k, v, table, lq, lk, (None, 0), 0)
    for prefix in (0, 1, 4):
        check(_run(q, k, v, table, lq, lk, (None, 0), prefix=prefix), *want, what=f"{prefix}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_long(dtype):
    """Keys split over many workgroups, and joined."""
    _check([1], [9001], 2, 1, 64, dtype, 64)
    _check([1, 2], [5000, 9001], 8, 2, 64, dtype, 16, window=(6000, 0), sinks=4)
    _check([1] * 3, [8192 + 5, 8192 + 64, 8192 + 1], 4, 1, 32, dtype, 64, prefix=128)
    _check([33], [6000], 2, 2, 64, dtype, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_and_scale(dtype):
    """Scores of some hundreds, rising and falling along the keys; a scale of the
    caller's, negative too."""
    for lq, lk in (([1, 1], [700, 300]), ([200], [700])):
        q, k, v, table = _case(lq, lk, 2, 2, 64, dtype, 64)
        ramp = torch.linspace(-1, 1, 64)[None, :, None, None]
        for factor in (ramp * 20, -ramp * 20, 20 * torch.sin(20 * ramp)):
            kk = (k.float() * factor).to(dtype)
            check(_run(q, kk, v, table, lq, lk, (None, 0)),
                  *attend_pages64(q, kk, v, table, lq, lk, (None, 0), 0))
        for scale in (0.0, 0.5, -0.3):
            check(_run(q, k, v, table, lq, lk, (50, 0), scale=scale),
                  *attend_pages64(q, k, v, table, lq, lk, (50, 0), 0, scale), what=f"scale {scale}")


def test_scores_beyond_exact_exponents():
    """Scores of 2^24 and more in exponents of two: finite weights."""
    for lq, lk in (([1], [300]), ([4], [300]), ([150], [300])):
        q, k, v, table = _case(lq, lk, 1, 1, 32, torch.float32, 64)
        k = torch.where(torch.isnan(k), k, torch.ones_like(k) * 2.0 ** 22)
        q = torch.ones_like(q)
        got = _run(q, k, v, table, lq, lk, (None, None)).cpu().double()
        rows = gather(v, table, 0, 300).double()  # all scores are the same: the mean of v
        check(got.float(), rows.mean(0, keepdim=True).expand(lq[0], 1, 32),
              torch.full((lq[0], 1, 32), 310 * 2.0 ** -24 * float(rows.abs().max()), dtype=torch.float64))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq,lk,prefix", [([1, 1], [500, 300], 0), ([3], [900], 0), ([12, 1], [300, 300], 2),
                                          ([200, 90], [400, 300], 0), ([200, 90], [400, 300], 2)])
def test_unseen_keys_may_hold_anything(lq, lk, prefix, dtype):
    """NaN and infinities at keys: those that do not see them are right, those
    that do are not finite."""
    window, sinks = (20, 0), 2
    q, k, v, table = _case(lq, lk, 4, 2, 64, dtype, 64, prefix)
    want, tol = attend_pages64(q, k, v, table, lq, lk, window, sinks)
    bad = [0, 70, 130, lk[0] - 25, lk[0] - 1]
    for j, x in zip(bad, ("nan", "inf", "-inf", "nan", "inf")):
        at = int(table[0, j // 64]), j % 64
        k[at], v[at] = float(x), float(x)
    got = _run(q, k, v, table, lq, lk, window, sinks, prefix).cpu()
    hit = []
    for b, (n, end) in enumerate(zip(lq, lk)):
        ok = seen(n, end, *window, sinks)
        there = [j for j in bad if b == 0 or j < 64 * prefix]
        hit.append(ok[:, there].any(1))
    hit = torch.cat(hit)
    assert hit.any()
    check(got[~hit], want[~hit], tol[~hit])
    assert not torch.isfinite(got[hit]).all(-1).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_no_sample_are_zero(dtype):
    for lq, lk in (([1, 1], [400, 300]), ([90, 40], [400, 300])):
        q, k, v, table = _case(lq, lk, 4, 2, 64, dtype, 64)
        want, tol = attend_pages64(q, k, v, table, lq, lk, (None, 0), 0)
        wide = torch.cat([torch.full((3, 4, 64), float("nan"), dtype=dtype), q,
                          torch.full((5, 4, 64), float("inf"), dtype=dtype)]).to(DEV)
        torch.full((1 << 20,), float("nan"), device=DEV)  # (what the output's memory held)
        got = spconv.cache_attention(wide, k.to(DEV), v.to(DEV), table.to(DEV), offsets_of(lq).to(DEV) + 3,
                                     ints(lk).to(DEV), window=(None, 0))
        check(got[3:-5], want, tol)
        assert not got[:3].any() and not got[-5:].any()


def test_lengths_that_do_not_fit():
    """Lengths below the new rows, negative or over the table's room are cut; no
    page, no key: zeros."""
    q, k, v, table = _case([3, 2, 2, 1], [3, 128, 128, 5], 2, 1, 32, torch.float32, 64)
    off = offsets_of([3, 2, 2, 1]).to(DEV)
    got = spconv.cache_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), off,
                                 ints([1, -5, 1 << 30, 0]).to(DEV), window=(None, 0)).cpu()
    lk = [1, 0, 128, 0]
    ref, tol = attend_pages64(q, k, v, table, [3, 2, 2, 1], lk, (None, 0), 0)
    check(got, ref, tol)
    assert not got[:2].any() and not got[3:5].any() and not got[7].any()
    none = torch.zeros(0, 64, 1, 32, device=DEV)
    got = spconv.cache_attention(q.to(DEV), none, none, table.to(DEV), off, ints([3, 9, 9, 5]).to(DEV))
    assert got.shape == q.shape and not got.any()


def test_strides_and_alignment():
    lq, lk = [1, 1, 1], [400, 64, 65]
    for lq in ([1, 1, 1], [60, 64, 60]):
        q, k, v, table = _case(lq, lk, 4, 2, 64, torch.float16, 64)
        want = _run(q, k, v, table, lq, lk, (None, 0))
        args = [table.to(DEV), offsets_of(lq).to(DEV), ints(lk).to(DEV)]
        for pad in (1, 8):
            room = [torch.zeros(*t.shape[:3], 64 + pad, dtype=t.dtype, device=DEV) for t in (q[None], k, v)]
            for r, t in zip(room, (q, k, v)):
                r[..., pad:] = t.to(DEV)
            got = spconv.cache_attention(room[0][0][..., pad:], room[1][..., pad:], room[2][..., pad:],
                                         *args, window=(None, 0))
            assert torch.equal(got, want), pad
        wide = torch.full((3, 3 * table.shape[1]), -1, dtype=torch.int32, device=DEV)
        wide[:, ::3] = args[0]
        got = spconv.cache_attention(q.to(DEV), k.to(DEV), v.to(DEV), wide[:, ::3], *args[1:], window=(None, 0))
        assert torch.equal(got, want)


def test_samples_by_the_hundred():
    n = 200
    lk = [1 + (37 * b) % 150 for b in range(n)]
    for lq in ([1] * n, [b % 3 for b in range(n)]):
        lk2 = [max(a, b) for a, b in zip(lq, lk)]
        _check(lq, lk2, 2, 1, 32, torch.bfloat16, 16)
        _check(lq, [64 + m for m in lk2], 2, 1, 32, torch.bfloat16, 16, prefix=4)


def test_no_rows_no_samples():
    k = torch.zeros(2, 8, 1, 32, device=DEV)
    table, off = ints([[0]]).to(DEV), ints([0, 0]).to(DEV)
    q = torch.zeros(0, 2, 32, device=DEV)
    assert spconv.cache_attention(q, k, k, table, off, ints([3]).to(DEV)).shape == q.shape
    q = torch.ones(4, 2, 32, device=DEV)
    got = spconv.cache_attention(q, k, k, table[:0], off[:1], off[:0])
    assert got.shape == q.shape and not got.any()


def test_refusals():
    q, k, v, table = (t.to(DEV) for t in _case([2], [100], 4, 2, 32, torch.float16, 64))
    off, n = offsets_of([2]).to(DEV), ints([100]).to(DEV)

    def refused(match, **change):
        a = dict(q=q, k_pages=k, v_pages=v, table=table, offsets=off, lengths=n)
        with pytest.raises(ValueError, match=match):
            spconv.cache_attention(**{**a, **change})

    refused("Nq, Hq, D", q=q[0])
    refused("pages", q=q[..., :16])
    refused("evenly", q=q[:, :3])
    refused("k_pages is", k_pages=k.float())
    refused("pages", k_pages=k[:1])
    refused("behind the other", v_pages=v.transpose(1, 3).contiguous().transpose(1, 3))
    refused("table", lengths=n[:0])
    refused("int32", offsets=off.long())
    refused("int32", table=table.cpu())
    refused("prefix", prefix=table)
    refused("prefix", prefix=table[0].long())
    refused("prefix", prefix=table[0].repeat(2))
    refused("negative", window=(-1, 0))
    refused("negative", sinks=-1)
    refused("finite", scale=float("nan"))
    big = torch.zeros(2, 2, 300, device=DEV, dtype=torch.float16)
    with pytest.raises(ValueError, match="head size"):
        spconv.cache_attention(big, big[None], big[None], table, off, n)
    with pytest.raises(TypeError):
        spconv.cache_attention(q.double(), k, v, table, off, n)


@pytest.mark.parametrize("lq", [[1, 1, 1], [3, 1, 40]])
@pytest.mark.parametrize("prefix", [0, 3])
def test_graph_replays(prefix, lq):
    """Captured once over a table with room to spare, replayed as the samples
    grow, with eager work between: every replay equals the eager result.  Two
    graphs over the same tensors do not disturb each other."""
    lk = [400, 900, 300]
    q, k, v, table = (t.to(DEV) for t in _case(lq, lk, 8, 2, 64, torch.bfloat16, 64, prefix))
    off, n = offsets_of(lq).to(DEV), ints(lk).to(DEV)
    head = table[0, :prefix].clone() if prefix else None

    def step():
        return spconv.cache_attention(q, k, v, table, off, n, prefix=head, window=(None, 0))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for i in range(4):
        q.copy_(torch.randn_like(q))
        n.copy_(ints([m - 31 * i for m in lk]))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), i


def test_repeats_give_the_same_bits():
    lq, lk = [1, 2, 1], [5000, 300, 2000]
    q, k, v, table = (t.to(DEV) for t in _case(lq, lk, 8, 2, 64, torch.bfloat16, 64))
    args = (q, k, v, table, offsets_of(lq).to(DEV), ints(lk).to(DEV))
    want = spconv.cache_attention(*args, window=(None, 0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        assert torch.equal(spconv.cache_attention(*args, window=(None, 0)), want)
        with torch.cuda.stream(side):
            again = spconv.cache_attention(*args, window=(None, 0))
        side.synchronize()
        assert torch.equal(again, want)

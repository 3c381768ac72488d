"""norm_rotate_append against the 64-bit form, and what it must leave alone."""
import pytest
import torch

import trispconv.pytorch as spconv
from cache_oracle import ints, offsets_of, scatter, tables
from gpu_util import DEV, needs_gpu, say
from sequence_oracle import check, rotate64

pytestmark = [pytest.mark.gpu, needs_gpu]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _case(lq, lk, hq, hk, dim, dtype, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = sum(lq)
    q, k, v = (torch.randn(n, h, dim, generator=g).mul(2).to(dtype) for h in (hq, hk, hk))
    pos = torch.randint(0, 1500, (n, 3), generator=g, dtype=torch.int32)
    table, pages = tables(lk, page)
    k_pages, v_pages = (torch.randn(pages, page, hk, dim, generator=g).to(dtype) for _ in range(2))
    return q, k, v, pos, k_pages, v_pages, table


def _expected(pages, rows, table, lq, lk):
    out, at = pages.clone(), 0
    for b, (n, end) in enumerate(zip(lq, lk)):
        scatter(out, table, b, rows[at:at + n], end - n)
        at += n
    return out


def _check(lq, lk, hq, hk, dim, dtype, page, weights=False, interleaved=False):
    q, k, v, pos, k_pages, v_pages, table = _case(lq, lk, hq, hk, dim, dtype, page)
    g = torch.Generator().manual_seed(9)
    qw = torch.randn(dim, generator=g).to(dtype) if weights else None
    kw = torch.randn(hk, dim, generator=g).to(dtype) if weights else None
    kp, vp = k_pages.to(DEV), v_pages.to(DEV)
    got = spconv.norm_rotate_append(
        q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), kp, vp, table.to(DEV),
        offsets_of(lq).to(DEV), ints(lk).to(DEV), None if qw is None else qw.to(DEV),
        None if kw is None else kw.to(DEV), base=100.0, interleaved=interleaved)
    check(got, *rotate64(q, pos, qw, base=100.0, interleaved=interleaved), what="q")
    ref, tol = rotate64(k, pos, kw, base=100.0, interleaved=interleaved)
    want = _expected(k_pages.double(), ref, table, lq, lk)
    room = _expected(torch.zeros_like(want), tol, table, lq, lk)
    check(kp, want, room, what="k")
    written = _expected(torch.zeros_like(want), torch.ones_like(ref), table, lq, lk).bool()
    assert torch.equal(kp.cpu()[~written], k_pages[~written])
    assert torch.equal(vp.cpu(), _expected(v_pages, v, table, lq, lk))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 3, 16, 20, 64])
def test_pages(page, dtype):
    say("append pages", page, dtype)
    _check([1, 1, 1], [1, 40, 129], 4, 2, 64, dtype, page)
    _check([33, 0, 7, 100], [33, 5, 70, 164], 2, 2, 32, dtype, page, weights=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,dim", [(1, 1, 2), (3, 1, 6), (2, 2, 8), (6, 6, 24), (5, 1, 40),
                                       (4, 4, 72), (2, 1, 96), (8, 2, 128), (2, 1, 250), (4, 1, 256),
                                       (0, 3, 16), (3, 0, 16)])
def test_heads(hq, hk, dim, dtype):
    say("append heads", hq, hk, dim, dtype)
    for interleaved in (False, True):
        _check([9, 17], [40, 17], hq, hk, dim, dtype, 16, weights=True, interleaved=interleaved)


@pytest.mark.parametrize("dim", [64, 6])
def test_same_queries_and_keys_as_norm_rotate_heads(dim):
    q, k, v, pos, k_pages, v_pages, table = _case([50], [50], 4, 2, dim, torch.float16, 64)
    kp, vp = k_pages.to(DEV), v_pages.to(DEV)
    a = spconv.norm_rotate_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), kp, vp,
                                  table.to(DEV), offsets_of([50]).to(DEV), ints([50]).to(DEV))
    b, c = spconv.norm_rotate_heads(q.to(DEV), k.to(DEV), pos.to(DEV))
    assert torch.equal(a, b)
    assert torch.equal(kp[int(table[0, 0]), :50], c)


@pytest.mark.parametrize("dim", [32, 6])
def test_rows_without_a_place(dim):
    """Rows of no sample, positions before the first or past the table's room,
    pages that there are not: written nowhere, their queries computed."""
    lq = [4, 6, 5, 3]
    q, k, v, pos, k_pages, v_pages, _ = _case([20], [20], 2, 1, dim, torch.float32, 4)
    k_pages, v_pages = k_pages[:6].clone(), v_pages[:6].clone()
    table = ints([[0, 1], [2, 3], [-1, 6], [4, 1 << 30]])
    # sample 0: two of its four rows before its first position; 1: its last two
    # past the room; 2: no page is there; 3: its last row's is not
    lk = [2, 10, 5, 5]
    off = offsets_of(lq) + 1  # a row before the first sample, one behind the last
    kp, vp = k_pages.to(DEV), v_pages.to(DEV)
    got = spconv.norm_rotate_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), kp, vp,
                                    table.to(DEV), off.to(DEV), ints(lk).to(DEV))
    check(got, *rotate64(q, pos), what="q")
    want = v_pages.clone()
    want[0, 0], want[0, 1] = v[3], v[4]                       # sample 0
    for i, t in enumerate(range(4, 8)):                       # sample 1, positions 4 to 7
        want[3, t - 4] = v[5 + i]
    want[4, 2], want[4, 3] = v[16], v[17]                     # sample 3, positions 2 and 3
    assert torch.equal(vp.cpu(), want)
    same = (vp.cpu() == v_pages).all(-1)
    assert torch.equal(kp.cpu()[same], k_pages[same])


def test_strides_and_views():
    """A packed projection's parts, head-major and row-major pages, spread tables
    and lengths: the bits of contiguous ones."""
    lq, lk = [30, 11], [70, 11]
    q, k, v, pos, k_pages, v_pages, table = _case(lq, lk, 4, 2, 64, torch.bfloat16, 16)
    args = [table.to(DEV), offsets_of(lq).to(DEV), ints(lk).to(DEV)]
    kp, vp = k_pages.to(DEV), v_pages.to(DEV)
    want = spconv.norm_rotate_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), kp, vp, *args)
    packed = torch.cat([q, k, v], 1).to(DEV)
    coords = torch.cat([torch.zeros(41, 1, dtype=torch.int32), pos], 1).to(DEV)
    kh, vh = (t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for t in (k_pages, v_pages))
    wide = torch.full((2, 2 * table.shape[1]), -1, dtype=torch.int32, device=DEV)
    wide[:, ::2] = args[0]
    spread = torch.zeros(2, 5, dtype=torch.int32, device=DEV)
    spread[:, 3] = args[2]
    got = spconv.norm_rotate_append(packed[:, :4], packed[:, 4:6], packed[:, 6:], coords[:, 1:], kh,
                                    vh, wide[:, ::2], args[1], spread[:, 3])
    assert torch.equal(got, want) and torch.equal(kh, kp) and torch.equal(vh, vp)
    # pages aligned to their elements only
    room = [torch.zeros(*t.shape[:3], 65, dtype=t.dtype, device=DEV) for t in (kp, vp)]
    ku, vu = (r[..., 1:] for r in room)
    ku.copy_(k_pages), vu.copy_(v_pages)
    got = spconv.norm_rotate_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), ku, vu, *args)
    assert torch.equal(got, want) and torch.equal(ku, kp) and torch.equal(vu, vp)
    assert not any(r[..., 0].any() for r in room)


def test_nothing_to_append():
    q = torch.zeros(0, 4, 32, device=DEV)
    kp = torch.ones(2, 8, 2, 32, device=DEV)
    none = torch.zeros(0, 2, 32, device=DEV)
    pos = torch.zeros(0, 3, device=DEV)
    table, off, n = ints([[0]]).to(DEV), ints([0, 0]).to(DEV), ints([5]).to(DEV)
    assert spconv.norm_rotate_append(q, none, none, pos, kp, kp.clone(), table, off, n).shape == q.shape
    # rows, and no samples: queries only
    q, k = torch.randn(3, 4, 32, device=DEV), torch.randn(3, 2, 32, device=DEV)
    got = spconv.norm_rotate_append(q, k, k, torch.zeros(3, 3, device=DEV), kp, kp.clone(), table[:0],
                                    off[:1], n[:0])
    check(got, *rotate64(q.cpu(), torch.zeros(3, 3)))
    assert (kp == 1).all()


def test_refusals():
    q, k, v, pos, kp, vp, table = (t.to(DEV) for t in _case([4], [4], 2, 1, 32, torch.float16, 8))
    off, n = offsets_of([4]).to(DEV), ints([4]).to(DEV)

    def refused(match, **change):
        a = dict(q=q, k=k, v=v, positions=pos, k_pages=kp, v_pages=vp, table=table, offsets=off,
                 lengths=n)
        with pytest.raises(ValueError, match=match):
            spconv.norm_rotate_append(**{**a, **change})

    refused("not \\(N, Hq, D\\)", v=v[:2])
    refused("not \\(N, Hq, D\\)", k=k[..., :16])
    refused("v is", v=v.float())
    refused("pages", k_pages=kp[0])
    refused("pages", v_pages=vp[:, :4])
    refused("k_pages is", k_pages=kp.float())
    refused("key heads", k_pages=kp.repeat(1, 1, 2, 1), v_pages=vp.repeat(1, 1, 2, 1))
    refused("behind the other", k_pages=kp.transpose(1, 3).contiguous().transpose(1, 3))
    refused("expanded", v_pages=vp[:1].expand(vp.shape))
    refused("table", table=table[0])
    refused("table", lengths=n.repeat(2))
    refused("table", offsets=off[:1])
    refused("int32", table=table.long())
    refused("int32", lengths=n.cpu())
    refused("positions", positions=pos.long())
    refused("q_weight", q_weight=torch.ones(5, device=DEV, dtype=torch.float16))
    refused("base", base=0.5)
    with pytest.raises(TypeError):
        spconv.norm_rotate_append(q.double(), k, v, pos, kp, vp, table, off, n)


def test_graph_and_streams():
    """A captured step, replayed with other rows, lengths and tables between eager
    work, on a stream of its own."""
    page, dim = 16, 64
    table, pages = tables([200, 200], page, seed=3)
    table = table.to(DEV)
    shape = (pages, page, 2, dim)
    q = torch.randn(2, 4, dim, device=DEV).half()
    k, v = (torch.randn(2, 2, dim, device=DEV).half() for _ in range(2))
    pos = torch.randint(0, 99, (2, 3), device=DEV, dtype=torch.int32)
    off, n = offsets_of([1, 1]).to(DEV), ints([5, 9]).to(DEV)
    kp, vp = (torch.zeros(shape, device=DEV).half() for _ in range(2))

    def step(kp, vp):
        return spconv.norm_rotate_append(q, k, v, pos, kp, vp, table, off, n)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kp, vp)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(kp, vp)
    ke, ve = kp.clone(), vp.clone()
    for i in range(4):
        q.copy_(torch.randn_like(q)), k.copy_(torch.randn_like(k)), v.copy_(torch.randn_like(v))
        n.add_(37)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(ke, ve)), i
        assert torch.equal(kp, ke) and torch.equal(vp, ve), i

"""Page copies and token compaction of the paged cache: bit-exact against the
same moves on the host, bad lists reported and left alone."""
import numpy as np
import pytest
import torch

from kvm_b200 import ops
from kvm_b200._lib import KvmError
from kvm_b200.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu


def _i32(a, dev):
    return torch.tensor(np.asarray(a, dtype=np.int32), device=dev)


def _cache(cuda, **kw):
    c = PagedKVCache(device=cuda, **kw)
    c.pool.view(torch.int16).copy_(
        torch.randint(-2 ** 15, 2 ** 15, c.pool.shape, device=cuda, dtype=torch.int16))
    return c


def _view(c):
    """int16 bits as [page, layer, kv, slot, width]."""
    p = c.pool.view(torch.int16)
    if c.layout == "page_first":
        return p.view(c.pages, c.layers, 2, c.block_size, c.width)
    return p.view(c.layers, c.pages, 2, c.block_size, c.width).transpose(0, 1)


SHAPES = [dict(pages=9, layers=1, block_size=16, heads_kv=1, layout="page_first"),
          dict(pages=12, layers=3, block_size=1, heads_kv=3, layout="layer_first"),
          dict(pages=40, layers=5, block_size=17, heads_kv=2, layout="page_first"),
          dict(pages=30, layers=2, block_size=256, heads_kv=8, layout="layer_first")]


@pytest.mark.parametrize("shape", SHAPES)
def test_copy_pages(cuda, shape):
    c = _cache(cuda, **shape)
    rng = np.random.default_rng(shape["pages"])
    ids = rng.permutation(c.pages)
    n = c.pages // 3
    src, dst = rng.choice(ids[:n], n), ids[n:2 * n]     # sources repeat
    want = _view(c).clone()
    want[torch.tensor(dst)] = want[torch.tensor(src)]
    c.copy_pages(_i32(src, cuda), _i32(dst, cuda))
    ops.device_status()
    assert torch.equal(_view(c), want)


def test_copy_pages_skips_and_reports_what_would_race(cuda):
    c = _cache(cuda, pages=12, layers=2, block_size=16, heads_kv=1)
    before = _view(c).clone()
    # 0 -> 5 and 1 -> 5 (twice a destination), 2 -> 3 and 3 -> 6 (3 is read),
    # bad ids, 7 -> 7 (nothing to do), 8 -> 9 (fine)
    pairs = [(0, 5), (1, 5), (2, 3), (3, 6), (12, 10), (10, -1), (7, 7), (8, 9)]
    c.copy_pages(_i32([a for a, _ in pairs], cuda), _i32([b for _, b in pairs], cuda))
    with pytest.raises(KvmError):
        ops.device_status()
    want = before.clone()
    want[9], want[6] = before[8], before[3]
    assert torch.equal(_view(c), want)


def test_copy_pages_many_small_pages(cuda):
    c = _cache(cuda, pages=2500, layers=1, block_size=16, heads_kv=1)
    perm = torch.randperm(2500, device=cuda).to(torch.int32)
    want = _view(c).clone()
    want[perm[1250:].long()] = want[perm[:1250].long()]
    c.copy_pages(perm[:1250].contiguous(), perm[1250:].contiguous())
    ops.device_status()
    assert torch.equal(_view(c), want)


def _compact_ref(c, view, kept, ctx, bt, bt_off):
    out = view.clone()
    for s, ks in enumerate(kept):
        def place(p):
            return int(bt[bt_off[s] + p // c.block_size]), p % c.block_size
        rows = [view[place(ctx[s] + j)[0], :, :, place(ctx[s] + j)[1]].clone() for j in ks]
        for i, row in enumerate(rows):
            p, slot = place(ctx[s] + i)
            out[p, :, :, slot] = row
    return out


def _tables(rng, pages, bs, lens):
    need = [(n + bs - 1) // bs for n in lens]
    return rng.permutation(pages)[:sum(need)], np.concatenate([[0], np.cumsum(need)])


@pytest.mark.parametrize("shape,ctx,nodes", [
    (dict(layers=1, block_size=16, heads_kv=1, layout="page_first"), [0], 5),
    (dict(layers=4, block_size=16, heads_kv=2, layout="page_first"), [15, 16, 33, 0], 40),
    (dict(layers=3, block_size=1, heads_kv=1, layout="layer_first"), [7, 2], 9),
    (dict(layers=2, block_size=64, heads_kv=8, layout="layer_first"), [100, 63, 1], 200),
    (dict(layers=2, block_size=17, heads_kv=3, layout="page_first"), [50, 16], 70),
])
def test_compact(cuda, shape, ctx, nodes):
    rng = np.random.default_rng(nodes)
    lens = [c + nodes for c in ctx]
    pages = sum((n + shape["block_size"] - 1) // shape["block_size"] for n in lens) + 2
    c = _cache(cuda, pages=pages, **shape)
    bt, bt_off = _tables(rng, pages, c.block_size, lens)
    # all, none, a random half, one, and a long run shifted by one
    kinds = [list(range(1, nodes)), [], list(range(nodes)),
             sorted(rng.choice(nodes, nodes // 2, replace=False).tolist()), [nodes - 1]]
    kinds = kinds[3:] + kinds[:3] if len(ctx) == 1 else kinds
    for turn in range(len(kinds)):
        kept = [kinds[(s + turn) % len(kinds)] for s in range(len(ctx))]
        if not sum(kept, []):
            continue
        off = np.concatenate([[0], np.cumsum([len(k) for k in kept])])
        want = _compact_ref(c, _view(c), kept, ctx, bt, bt_off)
        c.compact(_i32(sum(kept, []), cuda), _i32(off, cuda), _i32(ctx, cuda), _i32(bt, cuda),
                  _i32(bt_off, cuda))
        ops.device_status()
        assert torch.equal(_view(c), want), turn


@pytest.mark.parametrize("kept", [[2, 1], [1, 1], [-1, 2], [0, 31], [0, 10 ** 9]])
def test_compact_leaves_a_bad_sequence_alone(cuda, kept):
    """A list that is not strictly increasing or leaves the table: the sequence
    stays as it is and is reported, its neighbour is served."""
    c = _cache(cuda, pages=6, layers=2, block_size=16, heads_kv=1)
    ctx, bt, bt_off = [3, 3], [4, 1, 0, 2], [0, 2, 4]
    good = [1, 4]
    want = _compact_ref(c, _view(c), [[], good], ctx, bt, bt_off)
    c.compact(_i32(kept + good, cuda), _i32([0, 2, 4], cuda), _i32(ctx, cuda), _i32(bt, cuda),
              _i32(bt_off, cuda))
    with pytest.raises(KvmError):
        ops.device_status()
    assert torch.equal(_view(c), want)


def test_compact_reports_bad_pages_and_offsets(cuda):
    c = _cache(cuda, pages=4, layers=1, block_size=16, heads_kv=1)
    want = _view(c).clone()
    for bt, off, pos in (([9, 1], [0, 1], [3]), ([0, -2], [0, 1], [15]),
                         ([0, 1], [0, 2], [3]), ([0, 1], [1, 0], [3]), ([0, 1], [0, 1], [-4])):
        c.compact(_i32([2], cuda), _i32(off, cuda), _i32(pos, cuda), _i32(bt, cuda),
                  _i32([0, 2], cuda))
        with pytest.raises(KvmError):
            ops.device_status()
        assert torch.equal(_view(c), want)


def test_page_calls_refuse(cuda):
    c = _cache(cuda, pages=4, layers=1, block_size=16, heads_kv=1)
    one = _i32([0], cuda)
    with pytest.raises(ValueError):
        c.copy_pages(one, _i32([1, 2], cuda))
    with pytest.raises(TypeError):
        c.copy_pages(one.long(), one.long())
    with pytest.raises(ValueError):
        c.copy_pages(one.cpu(), one)
    with pytest.raises(ValueError):
        c.compact(one, one, one, one, _i32([0, 1], cuda))
    c.copy_pages(one[:0], one[:0])
    c.compact(one[:0], _i32([0, 0], cuda), one, one, _i32([0, 1], cuda))
    ops.device_status()


def test_compact_refuses_tables_outside_the_list(cuda):
    c = _cache(cuda, pages=4, layers=1, block_size=16, heads_kv=1)
    want = _view(c).clone()
    for bt_off in ([0, 9], [-1, 1], [2, 1]):
        c.compact(_i32([2], cuda), _i32([0, 1], cuda), _i32([3], cuda), _i32([0, 1], cuda),
                  _i32(bt_off, cuda))
        with pytest.raises(KvmError):
            ops.device_status()
        assert torch.equal(_view(c), want)


def test_compact_empty_block_table(cuda):
    """No sequence has a page: one that keeps nothing is served, one that keeps
    a token is reported."""
    c = _cache(cuda, pages=4, layers=1, block_size=16, heads_kv=1)
    want = _view(c).clone()
    none, two = _i32([], cuda), _i32([0, 0], cuda)
    c.compact(_i32([2], cuda), two, _i32([3], cuda), none, two)
    ops.device_status()
    c.compact(_i32([2], cuda), _i32([0, 1], cuda), _i32([3], cuda), none, two)
    with pytest.raises(KvmError):
        ops.device_status()
    assert torch.equal(_view(c), want)


def test_page_calls_in_a_graph(cuda):
    """Captured calls follow the lists and positions they find at replay."""
    c = _cache(cuda, pages=20, layers=2, block_size=16, heads_kv=2)
    src, dst = _i32([0, 1], cuda), _i32([5, 6], cuda)
    kept, off, ctx = _i32([1, 3, 0, 7], cuda), _i32([0, 2, 4], cuda), _i32([14, 3], cuda)
    bt, bt_off = [8, 9, 10, 11], [0, 2, 4]
    args = (kept, off, ctx, _i32(bt, cuda), _i32(bt_off, cuda))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.copy_pages(src, dst)
        c.compact(*args)
    for s, d, k, p in (([0, 1], [5, 6], [1, 3, 0, 7], [14, 3]),
                       ([6, 6], [2, 19], [0, 9, 2, 3], [0, 20])):
        src.copy_(torch.tensor(s)), dst.copy_(torch.tensor(d))
        kept.copy_(torch.tensor(k)), ctx.copy_(torch.tensor(p))
        want = _view(c).clone()
        want[torch.tensor(d)] = want[torch.tensor(s)]
        want = _compact_ref(c, want, [k[:2], k[2:]], p, bt, bt_off)
        graph.replay()
        ops.device_status()
        assert torch.equal(_view(c), want)

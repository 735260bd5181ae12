"""Attention of drafted trees over the paged cache against its formula in 64
bits (the tolerance is test_packed_attention_gpu's)."""
import math

import numpy as np
import pytest
import torch

from kvm_b200 import ops
from kvm_b200._lib import KvmError
from kvm_b200.kvcache import PagedKVCache, tree_mask
from test_packed_attention_gpu import check

pytestmark = pytest.mark.gpu


def _i32(a, dev):
    return torch.tensor(np.asarray(a, dtype=np.int64).astype(np.int32), device=dev)


class Case:
    """A filled cache with `nodes` drafted tokens after `ctx` cached ones."""

    def __init__(self, cuda, ctx, nodes, hq, hkv, bs, layout="page_first", layers=2, layer=1,
                 stale="nan", seed=0, density=0.5, empty=()):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.nodes, self.hq, self.hkv, self.layer = ctx, nodes, hq, hkv, layer
        total = [c + n for c, n in zip(ctx, nodes)]
        need = [(t + bs - 1) // bs for t in total]
        self.cache = PagedKVCache(pages=sum(need) + 3, layers=layers, block_size=bs,
                                  heads_kv=hkv, layout=layout, device=cuda)
        if stale == "nan":
            self.cache.pool.fill_(float("nan"))
        self.off = np.concatenate([[0], np.cumsum(nodes)])
        rows = int(self.off[-1])
        self.bt = _i32(rng.permutation(sum(need) + 3)[:sum(need)], cuda)
        self.bt_off = _i32(np.concatenate([[0], np.cumsum(need)]), cuda)
        self.q_off, self.q_pos = _i32(self.off, cuda), _i32(ctx, cuda)
        W = hkv * 128
        all_off = np.concatenate([[0], np.cumsum(total)])
        self.k, self.v = (torch.randn((int(all_off[-1]), W), generator=g, device=cuda)
                          .to(torch.bfloat16) for _ in range(2))
        self.all_off = all_off
        self.write()
        self.q = torch.randn((rows, hq * 128), generator=g, device=cuda).to(torch.bfloat16)
        self.words = (max(nodes) + 31) // 32 + (seed % 2)
        self.see = []
        for n in nodes:
            m = rng.random((n, n)) < density
            np.fill_diagonal(m, True)
            self.see.append(m)
        for s, i in empty:
            self.see[s][i] = False
        bits = np.zeros((rows, self.words * 32), dtype=bool)
        bits[:, :] = rng.random(bits.shape) < 0.5      # bits behind the last node mean nothing
        for s, m in enumerate(self.see):
            bits[self.off[s]:self.off[s + 1], :nodes[s]] = m
        packed = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
        self.mask = torch.tensor(packed.view(np.int32), device=cuda)

    def write(self):
        dev = self.q_off.device
        zeros = _i32([0] * len(self.ctx), dev)
        self.cache.write(self.layer, self.k, self.v, _i32(self.all_off, dev), zeros, self.bt,
                         self.bt_off)

    def run(self, **kw):
        args = dict(heads_q=self.hq, max_q_rows=max(self.nodes),
                    max_keys=max(c + n for c, n in zip(self.ctx, self.nodes)))
        return self.cache.tree_decode(self.layer, self.q, self.q_off, self.q_pos, self.mask,
                                      self.bt, self.bt_off, **{**args, **kw})

    def exact(self, scale=None):
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=self.q.device)
        mag = torch.zeros_like(out)
        g = self.hq // self.hkv
        for s, (c, n) in enumerate(zip(self.ctx, self.nodes)):
            if n == 0:
                continue
            r = slice(int(self.off[s]), int(self.off[s + 1]))
            Q = self.q[r].double().view(n, self.hkv, g, 128)
            kr = slice(int(self.all_off[s]), int(self.all_off[s + 1]))
            K, V = (t[kr].double().view(c + n, self.hkv, 128) for t in (self.k, self.v))
            z = torch.einsum("nhgd,mhd->hgnm", Q, K) * (scale or 1 / math.sqrt(128))
            seen = torch.cat((torch.ones((n, c), dtype=torch.bool),
                              torch.tensor(self.see[s]).reshape(n, n)), 1).to(z.device)
            p = torch.softmax(z.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
            out[r] = torch.einsum("hgnm,mhd->nhgd", p, V).reshape(n, -1)
            mag[r] = torch.einsum("hgnm,mhd->nhgd", p, V.abs()).reshape(n, -1)
        return out, mag


CASES = [
    dict(ctx=[0], nodes=[1], hq=1, hkv=1, bs=16),
    dict(ctx=[1], nodes=[1], hq=8, hkv=1, bs=16),
    dict(ctx=[0, 5, 127, 128, 129], nodes=[3, 1, 9, 16, 2], hq=8, hkv=2, bs=16),
    dict(ctx=[1030, 200, 0], nodes=[6, 0, 3], hq=16, hkv=2, bs=32),
    dict(ctx=[2100, 77], nodes=[1, 40], hq=4, hkv=4, bs=256, layout="layer_first"),
    dict(ctx=[900, 3000, 64], nodes=[33, 65, 20], hq=12, hkv=4, bs=64),     # 3 heads a group
    dict(ctx=[300], nodes=[300], hq=8, hkv=1, bs=128),                       # three node tiles
    dict(ctx=[100, 50], nodes=[130, 7], hq=2, hkv=2, bs=16),
    dict(ctx=[6000], nodes=[5], hq=64, hkv=1, bs=16),                        # 64 heads a group
    dict(ctx=[700, 31], nodes=[4, 4], hq=100, hkv=1, bs=16),                 # 100: 1 token a tile
    dict(ctx=[255, 256, 257, 1], nodes=[1, 1, 1, 1], hq=40, hkv=8, bs=32),   # 5 heads a group
    dict(ctx=[20000], nodes=[16], hq=8, hkv=1, bs=16),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_tree(cuda, i):
    c = Case(cuda, seed=i, **CASES[i])
    out = c.run()
    ops.device_status()
    check(out, *c.exact(), max(c.ctx) + max(c.nodes))


def test_tree_rows_that_see_nothing_are_zero(cuda):
    """Rows without a key, alone, beside others, and in an item that is cut
    between CTAs."""
    c = Case(cuda, ctx=[0, 0], nodes=[12, 700], hq=8, hkv=1, bs=16, seed=20, density=0.3,
             empty=[(0, 0), (0, 5), (1, 0), (1, 3), (1, 699)])
    out = c.run()
    ops.device_status()
    ref, mag = c.exact()
    check(out, ref, mag, 700)
    for s, i in ((0, 0), (0, 5), (1, 0), (1, 3), (1, 699)):
        assert bool((out[int(c.off[s]) + i] == 0).all())


def test_tree_chain_is_decode(cuda):
    """A chain's mask gives what the causal decode kernel gives."""
    c = Case(cuda, ctx=[1000, 40, 333], nodes=[4, 4, 4], hq=16, hkv=2, bs=16, seed=21)
    c.see = [np.tril(np.ones((4, 4), dtype=bool))] * 3
    c.mask = tree_mask([-1, 0, 1, 2], "cuda").repeat(3, 1)
    out = c.run()
    ref, mag = c.exact()
    check(out, ref, mag, 1004)
    dec = c.cache.decode(c.layer, c.q, c.q_off, c.q_pos, c.bt, c.bt_off, heads_q=16,
                         max_q_rows=4, max_keys=1004)
    ops.device_status()
    check(dec, ref, mag, 1004)


def test_tree_broken_nodes_reach_only_who_sees_them(cuda):
    c = Case(cuda, ctx=[250, 30], nodes=[20, 9], hq=8, hkv=2, bs=16, seed=22, density=0.4)
    ref, mag = c.exact()
    nan, inf = float("nan"), float("inf")
    a = int(c.all_off[1])
    c.v[250 + 7, :128] = inf
    c.k[250 + 11, 128:] = nan
    c.v[a + 30 + 2, 130] = -inf
    c.write()
    out = c.run()
    ops.device_status()
    o, ok = out.view(-1, 2, 4, 128), torch.ones((29, 2, 4, 128), dtype=torch.bool, device="cuda")
    for i in range(20):
        if c.see[0][i, 7]:
            ok[i, 0] = False
            assert bool((o[i, 0] == inf).all())
        if c.see[0][i, 11]:
            ok[i, 1] = False
            assert bool(torch.isnan(o[i, 1]).all())
    for i in range(9):
        if c.see[1][i, 2]:
            ok[20 + i, 1, :, 2] = False
            assert bool((o[20 + i, 1, :, 2] == -inf).all())
    ok = ok.view(out.shape)
    check(out[ok], ref[ok], mag[ok], 270)


def test_tree_scale_out_workspace_and_rows_left_alone(cuda):
    c = Case(cuda, ctx=[1500, 70], nodes=[8, 3], hq=8, hkv=2, bs=16, seed=23)
    rows = c.q.shape[0]
    wide = torch.full((rows + 4, 8 * 128 + 8), 5.0, dtype=torch.bfloat16, device=cuda)
    q = torch.cat((c.q, c.q[:4]))
    mask = torch.cat((c.mask, c.mask[:4]))
    n = c.cache.tree_workspace(2, heads_q=8, max_q_rows=8, max_keys=2000)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda)
    c.cache.tree_decode(c.layer, q, c.q_off, c.q_pos, mask, c.bt, c.bt_off, heads_q=8,
                        max_q_rows=8, max_keys=2000, scale=0.3, out=wide[:, :1024], workspace=ws)
    ops.device_status()
    ref, mag = c.exact(scale=0.3)
    # scores are 0.3 * sqrt(128) = 3.4 times the usual ones
    check(wide[:rows, :1024], ref, mag * (1 + 4 * 2.0 ** -5), 1508)
    assert bool((wide[rows:] == 5).all()) and bool((wide[:, 1024:] == 5).all())
    with pytest.raises(KvmError):
        c.run(workspace=ws[:16], max_keys=2000)


@pytest.mark.parametrize("i", [3, 5, 6, 8, 11])
def test_tree_takes_nothing_from_the_workspace(cuda, i):
    """Whatever an earlier call or another tensor left there."""
    c = Case(cuda, seed=i, **CASES[i])
    want = c.run()
    n = c.cache.tree_workspace(len(c.ctx), heads_q=c.hq, max_q_rows=max(c.nodes),
                               max_keys=max(a + b for a, b in zip(c.ctx, c.nodes)))
    for fill in (0, 1, 0x7F, 0xFF):
        ws = torch.full((n,), fill, dtype=torch.uint8, device=cuda)
        assert torch.equal(c.run(workspace=ws), want)
    ws.copy_(torch.randint(0, 256, (n,), device=cuda, dtype=torch.uint8))
    assert torch.equal(c.run(workspace=ws), want)
    ops.device_status()


def test_tree_out_of_bounds_sequences_are_reported(cuda):
    """More nodes or keys than the bounds allow: that sequence is skipped."""
    for kw, skipped in ((dict(max_q_rows=5), 0), (dict(max_keys=200), 1)):
        c = Case(cuda, ctx=[100, 400], nodes=[9, 4], hq=4, hkv=1, bs=16, seed=24)
        out = torch.full_like(c.q, 9.0)
        c.run(out=out, **kw)
        with pytest.raises(KvmError):
            ops.device_status()
        ref, mag = c.exact()
        r = [slice(0, 9), slice(9, 13)]
        assert bool((out[r[skipped]] == 9).all())
        check(out[r[1 - skipped]], ref[r[1 - skipped]], mag[r[1 - skipped]], 404)


@pytest.mark.parametrize("ctx", [[300, 40, 200], [5000, 40, 200]])     # whole items, cut ones
def test_tree_after_bad_offsets_nothing_is_written(cuda, ctx):
    """Rows of a sequence after a descending pair of offsets can be another
    sequence's: that one keeps its result, the later ones are left out."""
    c = Case(cuda, ctx=ctx, nodes=[9, 0, 4], hq=8, hkv=2, bs=16, seed=32)
    ref, mag = c.exact()
    for off, served in (([0, 9, 4, 13], 9), ([0, 9, 20, 13], 9), ([0, -1, 9, 13], 0),
                        ([-4, 9, 9, 13], 0)):
        for turn in range(5):
            out = torch.full_like(c.q, 9.0)
            c.cache.tree_decode(c.layer, c.q, _i32(off, cuda), c.q_pos, c.mask, c.bt, c.bt_off,
                                heads_q=8, max_q_rows=9, max_keys=max(ctx) + 9, out=out)
            with pytest.raises(KvmError):
                ops.device_status()
            check(out[:served], ref[:served], mag[:served], max(ctx) + 9)
            assert bool((out[served:] == 9).all())


def test_tree_bad_offsets_far_down_the_list(cuda):
    """The first bad pair is the 36th of 70: the 35 before it are served."""
    n = 70
    c = Case(cuda, ctx=[(i * 13) % 90 for i in range(n)], nodes=[1 + i % 3 for i in range(n)],
             hq=4, hkv=1, bs=16, seed=33)
    off = c.off.copy()
    off[36] = off[30]                            # sequence 35 descends, 36 covers rows of 30..36
    out = torch.full_like(c.q, 9.0)
    c.cache.tree_decode(c.layer, c.q, _i32(off, cuda), c.q_pos, c.mask, c.bt, c.bt_off, heads_q=4,
                        max_q_rows=32, max_keys=130, out=out)
    with pytest.raises(KvmError):
        ops.device_status()
    ref, mag = c.exact()
    m = int(off[35])
    check(out[:m], ref[:m], mag[:m], 95)
    assert bool((out[m:] == 9).all())


def test_tree_bad_pages_are_reported(cuda):
    c = Case(cuda, ctx=[100, 300], nodes=[4, 4], hq=4, hkv=1, bs=16, seed=25)
    for bad in (-1, 10 ** 6, c.cache.pages):
        bt = c.bt.clone()
        bt[2] = bad
        out = c.cache.tree_decode(c.layer, c.q, c.q_off, c.q_pos, c.mask, bt, c.bt_off,
                                  heads_q=4, max_q_rows=4, max_keys=304)
        with pytest.raises(KvmError):
            ops.device_status()
        ref, mag = c.exact()
        check(out[4:], ref[4:], mag[4:], 304)      # the other sequence is served


def test_tree_tables_outside_the_list_are_reported(cuda):
    c = Case(cuda, ctx=[100, 300], nodes=[4, 4], hq=4, hkv=1, bs=16, seed=31)
    n = c.bt.numel()
    first = c.bt_off.tolist()[1]
    for off in ([-1, first, n], [first + 1, first, n]):
        out = c.cache.tree_decode(c.layer, c.q, c.q_off, c.q_pos, c.mask, c.bt, _i32(off, cuda),
                                  heads_q=4, max_q_rows=4, max_keys=304)
        with pytest.raises(KvmError):
            ops.device_status()
        ref, mag = c.exact()
        check(out[4:], ref[4:], mag[4:], 304)


def test_tree_empty_block_table(cuda):
    """A padded step in which no sequence has a node or a page: nothing to do,
    and nothing wrong. With nodes, their positions are outside their tables."""
    c = Case(cuda, ctx=[100, 300], nodes=[4, 4], hq=4, hkv=1, bs=16, seed=34)
    zero = _i32([0, 0, 0], cuda)
    for off, bad in ((zero, False), (c.q_off, True)):
        out = torch.full_like(c.q, 9.0)
        c.cache.tree_decode(c.layer, c.q, off, c.q_pos, c.mask, c.bt[:0], zero, heads_q=4,
                            max_q_rows=4, max_keys=304, out=out)
        if bad:
            with pytest.raises(KvmError):
                ops.device_status()
        else:
            ops.device_status()
            assert bool((out == 9).all())


def test_tree_graph_and_two_streams(cuda):
    """A captured call follows contexts that change; two calls at once with a
    workspace each."""
    c = Case(cuda, ctx=[2000, 500], nodes=[6, 6], hq=16, hkv=2, bs=16, seed=26)
    d = Case(cuda, ctx=[1700], nodes=[30], hq=16, hkv=2, bs=32, seed=27)
    n = c.cache.tree_workspace(2, heads_q=16, max_q_rows=6, max_keys=2006)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda)
    out = torch.zeros_like(c.q)
    c.run(out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=out, workspace=ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(5):
        graph.replay()
        with torch.cuda.stream(s):
            outs.append(d.run())
    torch.cuda.synchronize()
    ops.device_status()
    check(out, *c.exact(), 2006)
    for o in outs:
        check(o, *d.exact(), 1730)
    c.ctx = [1990, 11]
    c.q_pos.copy_(torch.tensor(c.ctx))
    # the nodes now follow the shorter contexts in the cache
    old = c.all_off
    c.k, c.v = (torch.cat((t[:1996], t[old[1]:old[1] + 17])) for t in (c.k, c.v))
    c.all_off = np.array([0, 1996, 2013])
    graph.replay()
    ops.device_status()
    check(out, *c.exact(), 2006)


def test_tree_same_bits_every_time(cuda):
    c = Case(cuda, ctx=[5000, 300, 2000], nodes=[16, 2, 40], hq=16, hkv=2, bs=16, seed=28)
    a = c.run()
    for _ in range(20):
        assert torch.equal(a, c.run())


def test_tree_refusals_and_empty(cuda):
    c = Case(cuda, ctx=[40], nodes=[4], hq=4, hkv=1, bs=16, seed=30)
    with pytest.raises(KvmError):
        c.run(max_q_rows=40)                     # the mask has 32 bits
    with pytest.raises(KvmError):
        c.run(max_q_rows=0)
    with pytest.raises((ValueError, KvmError)):
        c.run(heads_q=3)
    with pytest.raises(ValueError):
        c.cache.tree_decode(1, c.q, c.q_off, c.q_pos, c.mask[:3], c.bt, c.bt_off, heads_q=4,
                            max_q_rows=4, max_keys=44)
    with pytest.raises(ValueError):
        c.cache.tree_decode(1, c.q, c.q_off, c.q_pos, c.mask, c.bt, c.bt_off[:1], heads_q=4,
                            max_q_rows=4, max_keys=44)
    with pytest.raises(ValueError):
        c.cache.tree_decode(2, c.q, c.q_off, c.q_pos, c.mask, c.bt, c.bt_off, heads_q=4,
                            max_q_rows=4, max_keys=44)
    small = PagedKVCache(pages=4, layers=1, block_size=8, heads_kv=1, device=cuda)
    with pytest.raises(KvmError):
        small.tree_decode(0, c.q, c.q_off, c.q_pos, c.mask, c.bt, c.bt_off, heads_q=4,
                          max_q_rows=4, max_keys=44)
    none = c.cache.tree_decode(1, c.q[:0], c.q_off * 0, c.q_pos, c.mask[:0], c.bt, c.bt_off,
                               heads_q=4, max_q_rows=4, max_keys=44)
    assert none.shape == (0, 512)
    ops.device_status()

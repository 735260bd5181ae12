"""The serving operators run together as a server runs them - packed prompts,
the cache, a fork, drafted trees, their verification and compaction, plain
decoding - against attention over each sequence's own tokens in 64 bits."""
import math

import numpy as np
import pytest
import torch

from kvm_b200 import ops
from kvm_b200.kvcache import PagedKVCache, tree_mask

pytestmark = pytest.mark.gpu

HQ, HKV, HD, BS, LAYERS = 16, 2, 128, 16, 2


def _i32(a, dev):
    return torch.tensor(np.asarray(a, dtype=np.int32), device=dev)


class Tokens:
    """q, k, v of a token in a layer, from its id alone (before rotation)."""

    def __init__(self, cuda, n):
        g = torch.Generator(device="cuda").manual_seed(n)
        self.q = [torch.randn((n, HQ * HD), generator=g, device=cuda).to(torch.bfloat16)
                  for _ in range(LAYERS)]
        self.k, self.v = ([torch.randn((n, HKV * HD), generator=g, device=cuda)
                           .to(torch.bfloat16) for _ in range(LAYERS)] for _ in range(2))


def _exact(tok, layer, ids, positions, freq, rows):
    """Outputs of the last `rows` tokens of the chain `ids`, and sum p |v|."""
    def turn(x, heads):
        t = x.double().view(len(ids), heads, HD)
        ang = torch.tensor(positions, dtype=torch.float64, device=x.device)[:, None] * freq
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        a, b = t[..., :HD // 2], t[..., HD // 2:]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
        return y.to(torch.bfloat16).double()        # the rotated values are stored in bf16
    q = turn(tok.q[layer][ids], HQ).view(-1, HKV, HQ // HKV, HD)[-rows:]
    k = turn(tok.k[layer][ids], HKV)
    v = tok.v[layer][ids].double().view(-1, HKV, HD)
    n = len(ids)
    seen = torch.ones((n, n), dtype=torch.bool, device=q.device).tril()[-rows:]
    z = torch.einsum("nhgd,mhd->hgnm", q, k) / math.sqrt(HD)
    p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
    return (torch.einsum("hgnm,mhd->nhgd", p, v).reshape(rows, -1),
            torch.einsum("hgnm,mhd->nhgd", p, v.abs()).reshape(rows, -1))


def _close(got, ref, mag):
    # P and the result are rounded once each (2^-8); a rotated q or k that the
    # kernel rounds to the other neighbour (its angle is 2^-21 off) is 2^-7 off in
    # one of the 2 * 128 products of a score: 2^-7 * 16 / sqrt(128) at most for
    # values below 4, and rare; 2^-6 of P covers it.
    tol = 2.0 ** -8 * (mag + ref.abs()) * (1 + 2.0 ** -7) + 2.0 ** -6 * mag
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def _run(cuda):
    outs = []
    table = ops.rope_table(HD)
    freq = 10000.0 ** (-2 * torch.arange(HD // 2, dtype=torch.float64, device=cuda) / HD)
    tok = Tokens(cuda, 900)
    cache = PagedKVCache(pages=80, layers=LAYERS, block_size=BS, heads_kv=HKV, device=cuda)
    cache.pool.fill_(float("nan"))           # nothing may read what was not written
    free = list(np.random.default_rng(3).permutation(80))
    chains = [list(range(0, 130)), list(range(200, 237)), list(range(300, 577))]
    tables = [[free.pop() for _ in range(24)] for _ in chains]

    def bt():
        off = np.concatenate([[0], np.cumsum([len(t) for t in tables])])
        return _i32(sum(tables, []), cuda), _i32(off, cuda)

    def step(layer, ids, positions):
        """Rotated q, k and the values of these tokens."""
        i = torch.tensor(ids, device=cuda)
        q, k = ops.rope(tok.q[layer][i], _i32(positions, cuda), table, heads=HQ,
                        k=tok.k[layer][i], heads_kv=HKV)
        return q, k, tok.v[layer][i]

    # prompts, packed
    ids = sum(chains, [])
    off = _i32(np.concatenate([[0], np.cumsum([len(c) for c in chains])]), cuda)
    pos = sum([list(range(len(c))) for c in chains], [])
    start = _i32([0] * len(chains), cuda)
    for layer in range(LAYERS):
        q, k, v = step(layer, ids, pos)
        out = ops.attention_packed(q, k, v, off, heads_q=HQ, heads_kv=HKV)
        cache.write(layer, k, v, off, start, *bt())
        outs.append(out)
        at = 0
        for c in chains:
            _close(out[at:at + len(c)], *_exact(tok, layer, c, range(len(c)), freq, len(c)))
            at += len(c)

    # a fork of sequence 1 (37 tokens: two full pages shared, the third copied)
    fresh = [free.pop()] + tables[1][3:]
    cache.copy_pages(_i32([tables[1][2]], cuda), _i32(fresh[:1], cuda))
    tables.append(tables[1][:2] + fresh[:1] + [free.pop() for _ in range(4)])
    chains.append(list(chains[1]))

    # a drafted tree per sequence, checked, its accepted path kept
    parents = [[-1, 0, 0, 1, 1, 2, -1], [-1], [-1, -1, 1, 2, 3], [-1, 0, 1, 1]]
    accept = [[0, 2, 5], [0], [1, 2, 3, 4], [0, 1, 3]]
    draft, nid = [], 600
    for p in parents:
        draft.append(list(range(nid, nid + len(p))))
        nid += len(p)
    n_off = np.concatenate([[0], np.cumsum([len(d) for d in draft])])
    q_off = _i32(n_off, cuda)
    ctx = _i32([len(c) for c in chains], cuda)
    paths = []
    for s, p in enumerate(parents):
        for i in range(len(p)):
            path = [i]
            while p[path[0]] >= 0:
                path.insert(0, p[path[0]])
            paths.append((s, path))
    depth = [len(path) - 1 for _, path in paths]
    pos = [len(chains[s]) + d for (s, _), d in zip(paths, depth)]
    mask = torch.cat([tree_mask(p, cuda) for p in parents])
    most = max(len(c) + len(d) for c, d in zip(chains, draft))
    for layer in range(LAYERS):
        q, k, v = step(layer, sum(draft, []), pos)
        cache.write(layer, k, v, q_off, ctx, *bt())
        out = cache.tree_decode(layer, q, q_off, ctx, mask, *bt(), heads_q=HQ, max_q_rows=7,
                                max_keys=most)
        outs.append(out)
        for r, (s, path) in enumerate(paths):
            chain = chains[s] + [draft[s][i] for i in path]
            _close(out[r:r + 1], *_exact(tok, layer, chain, range(len(chain)), freq, 1))
    kept = _i32(sum(accept, []), cuda)
    k_off = _i32(np.concatenate([[0], np.cumsum([len(a) for a in accept])]), cuda)
    cache.compact(kept, k_off, ctx, *bt())
    chains = [c + [d[i] for i in a] for c, d, a in zip(chains, draft, accept)]

    # plain decoding of one more token: the causal kernel and a one-node tree
    new = list(range(700, 700 + len(chains)))
    ctx = _i32([len(c) for c in chains], cuda)
    one = _i32(range(len(chains) + 1), cuda)
    for layer in range(LAYERS):
        q, k, v = step(layer, new, [len(c) for c in chains])
        cache.write(layer, k, v, one, ctx, *bt())
        kw = dict(heads_q=HQ, max_q_rows=1, max_keys=max(len(c) for c in chains) + 1)
        a = cache.decode(layer, q, one, ctx, *bt(), **kw)
        b = cache.tree_decode(layer, q, one, ctx, torch.ones((len(new), 1), dtype=torch.int32,
                                                             device=cuda), *bt(), **kw)
        outs += [a, b]
        for s, c in enumerate(chains):
            ref = _exact(tok, layer, c + [new[s]], range(len(c) + 1), freq, 1)
            _close(a[s:s + 1], *ref)
            _close(b[s:s + 1], *ref)
    ops.device_status()
    return outs


def test_prompt_fork_tree_compact_decode(cuda):
    _run(cuda)


def test_the_same_run_gives_the_same_bits(cuda):
    """Kernel after kernel with programmatic dependent launch, busy or not."""
    first = _run(cuda)
    for _ in range(5):
        noise = [torch.randn(1 << 22, device=cuda) for _ in range(3)]
        for n in noise:
            n.mul_(2.0)
        for a, b in zip(first, _run(cuda)):
            assert torch.equal(a, b)


def test_one_row_has_no_row_stride(cuda):
    """torch leaves the stride of a dimension of one entry free; the calls take
    such a row, whatever its stride says, and give what they give for a plain one."""
    def odd(x):
        return x.as_strided(x.shape, (1, 1))
    tok = Tokens(cuda, 1)
    q, k, v = tok.q[0], tok.k[0], tok.v[0]
    table, pos = ops.rope_table(HD), _i32([5], cuda)
    kw = dict(heads=HQ, heads_kv=HKV)
    outs = []
    for f in (lambda x: x, odd):
        rq, rk = ops.rope(f(q), pos, table, k=f(k), out=f(torch.empty_like(q)),
                          out_k=f(torch.empty_like(k)), **kw)
        a = ops.attention_packed(f(rq), f(rk), f(v), _i32([0, 1], cuda), heads_q=HQ,
                                 heads_kv=HKV, out=f(torch.empty_like(q)))
        cache = PagedKVCache(pages=1, layers=1, block_size=BS, heads_kv=HKV, device=cuda)
        one, zero = _i32([0, 1], cuda), _i32([0], cuda)
        cache.write(0, rk.view(-1)[None], v, one, zero, zero, one)
        mask = torch.ones((1, 1), dtype=torch.int32, device=cuda)
        b = cache.tree_decode(0, f(rq), one, zero, mask, zero, one, heads_q=HQ, max_q_rows=1,
                              max_keys=1, out=f(torch.empty_like(q)))
        outs.append([t.contiguous().view(-1) for t in (rq, rk, a, b)])
    ops.device_status()
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    assert torch.equal(outs[0][2], v.view(HKV, 1, HD).expand(-1, HQ // HKV, -1).reshape(-1))

"""Rotary positions, packed prompt attention, tree attention over the paged
cache, and the cache's page copies and token compaction: the cases they are
measured at, their inputs, their plain forms and the framework's calls.

Every operator is defined by its formula:
  rope     y = x rotated by the angle positions[r] * f_i in the plane of the pair i
  packed   out[r] = sum_j softmax_j(scale q_r . k_j) v_j over the keys j <= r of r's sequence
  tree     the same over the cached context and the drafted tokens that the row's mask names
  copy     page dst[i] of the pool becomes page src[i], all layers, K and V
  compact  token slot ctx + i of a sequence becomes slot ctx + kept[i], all layers, K and V
"""
import math
import random

import torch

own = False

HD = 128          # head width of the paged cache
ELEM = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases ---

def listed():
    return [
        # one decode step of eight sequences: the rotation is all latency
        dict(name="rope_decode", op="rope", rows=8, heads_q=64, heads_kv=8, hd=128, rot=128,
             inter=False, dtype="bf16", scaling="none", max_pos=8192),
        # a prompt batch of the decoder layer's heads, positions far beyond the trained length
        dict(name="rope_prompt", op="rope", rows=8192, heads_q=64, heads_kv=8, hd=128, rot=64,
             inter=True, dtype="bf16", scaling="yarn", max_pos=131072),
        # a few short questions admitted together
        dict(name="packed_short", op="packed", seqs=6, lo=3, hi=90, heads_q=16, heads_kv=2,
             hd=128, dtype="bf16", lens=1),
        # an ordinary prompt batch with the decoder layer's heads
        dict(name="packed_batch", op="packed", seqs=9, lo=130, hi=2048, heads_q=64, heads_kv=8,
             hd=128, dtype="bf16", lens=2),
        # one long document
        dict(name="packed_long", op="packed", seqs=1, lo=16383, hi=16383, heads_q=32, heads_kv=4,
             hd=128, dtype="bf16", lens=3),
        # narrow heads, three queries to a key head, many odd lengths
        dict(name="packed_narrow", op="packed", seqs=40, lo=1, hi=700, heads_q=24, heads_kv=8,
             hd=64, dtype="fp16", lens=4),
        # two users, a small draft each
        dict(name="tree_small", op="tree", seqs=2, lo=40, hi=600, nodes=7, heads_q=16,
             heads_kv=2, bs=16, layout="page_first", lens=5),
        # a serving batch at the decode benchmark's context, sixteen drafted tokens each
        dict(name="tree_batch", op="tree", seqs=32, lo=2000, hi=4096, nodes=16, heads_q=64,
             heads_kv=8, bs=16, layout="page_first", lens=6),
        # few long contexts, wide trees: the split along the keys carries it
        dict(name="tree_long", op="tree", seqs=3, lo=12000, hi=20000, nodes=60, heads_q=64,
             heads_kv=8, bs=64, layout="layer_first", lens=7),
        # forks that give each child its own copy of the parent's last page
        dict(name="copy_pages", op="copy", pairs=96, pages=256, layers=32, bs=16, heads_kv=8,
             layout="page_first"),
        # one sequence keeps a token or two of its draft
        dict(name="compact_one", op="compact", seqs=1, nodes=8, ctx=1000, layers=32, bs=16,
             heads_kv=8, layout="page_first"),
        # a batch keeps the accepted path of every tree
        dict(name="compact_batch", op="compact", seqs=48, nodes=24, ctx=300, layers=24, bs=32,
             heads_kv=8, layout="layer_first"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "packed", "packed", "tree", "tree", "copy", "compact"])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    lens = rng.randrange(1 << 20)
    if op == "rope":
        hd = rng.choice([64, 80, 128, 256])
        return dict(op=op, rows=_log(rng, 1, 8192), heads_q=min(64, hkv * group), heads_kv=hkv,
                    hd=hd, rot=rng.choice([hd, hd // 2, 32]), inter=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]) if hkv * group <= 32 else "bf16",
                    scaling=rng.choice(["none", "linear", "ntk", "bands", "yarn"]),
                    max_pos=_log(rng, 100, 1 << 20))
    if op == "packed":
        hi = _log(rng, 8, 6000)
        lo = rng.randint(0, hi)
        return dict(op=op, seqs=max(1, min(_log(rng, 1, 64), 12000 // hi)), lo=lo, hi=hi,
                    heads_q=hkv * group if hkv * group <= 64 else hkv * 8, heads_kv=hkv,
                    hd=rng.choice([64, 128]), dtype=rng.choice(["bf16", "fp16"]), lens=lens)
    if op == "tree":
        hi = _log(rng, 16, 20000)
        return dict(op=op, seqs=max(1, min(_log(rng, 1, 64), 60000 // hi)),
                    lo=rng.randint(0, hi), hi=hi, nodes=_log(rng, 1, 100),
                    heads_q=hkv * group if hkv * group <= 64 else hkv * 8, heads_kv=hkv,
                    bs=rng.choice([16, 32, 64, 128, 256]),
                    layout=rng.choice(["page_first", "layer_first"]), lens=lens)
    bs, layers = rng.choice([16, 32, 64]), rng.choice([1, 4, 24, 32])
    layout = rng.choice(["page_first", "layer_first"])
    if op == "copy":
        pairs = max(1, min(_log(rng, 1, 96), 96 * 16 * 32 * 8 // (bs * layers * hkv)))
        return dict(op=op, pairs=pairs, pages=2 * pairs + rng.randint(1, 64), layers=layers,
                    bs=bs, heads_kv=hkv, layout=layout)
    return dict(op=op, seqs=_log(rng, 1, 48), nodes=rng.randint(2, 24), ctx=rng.randint(1, 300),
                layers=min(layers, 24), bs=bs, heads_kv=hkv, layout=layout)


def _lens(case):
    """The sequences' lengths (or contexts), the same for every seed."""
    r = random.Random(case["lens"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    return lens if any(lens) or case["op"] == "tree" else [case["hi"]] * len(lens)


def _nodes(case):
    """Drafted tokens per sequence: the last one has the most."""
    r = random.Random(case["lens"] + 1)
    return [r.randint(1, case["nodes"]) for _ in range(case["seqs"] - 1)] + [case["nodes"]]


def _kept(case):
    """Contexts, and how many of its drafted tokens each sequence keeps (a third at most)."""
    r = random.Random(case["ctx"] * 64 + case["seqs"])
    ctx = [case["ctx"] - r.randint(0, case["ctx"] // 2) for _ in range(case["seqs"])]
    return ctx, [r.randint(1, max(1, case["nodes"] // 3)) for _ in ctx]


# ---------------------------------------------------------------- inputs ---

def _scaling(case):
    """Arguments of the rotary table: what stretches the trained 4096 positions."""
    kind = case["scaling"]
    more = dict(none={}, linear=dict(factor=8.0), ntk=dict(factor=8.0),
                bands=dict(factor=8.0, original_len=4096, low=1.0, high=4.0),
                yarn=dict(factor=32.0, original_len=4096, low=1.0, high=32.0))[kind]
    return dict(base=10000.0, scaling=kind, **more)


def _randn(g, shape, dtype, std=1.0):
    t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return t.mul_(std).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(counts):
    off = [0]
    for n in counts:
        off.append(off[-1] + n)
    return off


def _parents(rng, n):
    """A drafted tree in topological order: parent of each node, -1 for the roots."""
    return [-1] + [rng.choice([-1] + list(range(max(0, i - 6), i))) for i in range(1, n)]


def _pool(case, g, layers, pages):
    """A cache with every slot filled; the framework's own class where it is measured."""
    if own:
        from kvm_b200.kvcache import PagedKVCache
        cache = PagedKVCache(pages=pages, layers=layers, block_size=case["bs"],
                             heads_kv=case["heads_kv"], layout=case["layout"], device="cuda")
        pool = cache.pool
    else:
        cache = None
        pool = torch.zeros(pages * layers * 2 * case["bs"] * case["heads_kv"] * HD,
                           dtype=torch.bfloat16, device="cuda")
    pool.normal_(generator=g)
    return cache, pool


def _view(case, pool, layers, pages):
    """The pool as [page, layer, kv, slot, width] whatever its layout."""
    W = case["heads_kv"] * HD
    if case["layout"] == "page_first":
        return pool.view(pages, layers, 2, case["bs"], W)
    return pool.view(layers, pages, 2, case["bs"], W).transpose(0, 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = random.Random(seed)
    op = case["op"]
    st = dict(case=case)
    if op == "rope":
        dt, hd = ELEM[case["dtype"]], case["hd"]
        R, nq, nk = case["rows"], case["heads_q"] * hd, case["heads_kv"] * hd
        qkv = _randn(g, (R, nq + 2 * nk), dt)
        st.update(q=qkv[:, :nq], k=qkv[:, nq:nq + nk],
                  positions=torch.randint(0, case["max_pos"], (R,), generator=g, device="cuda",
                                          dtype=torch.int32),
                  out_q=torch.empty((R, nq), dtype=dt, device="cuda"),
                  out_k=torch.empty((R, nk), dtype=dt, device="cuda"))
        if own:
            from kvm_b200 import ops
            st["table"] = ops.rope_table(case["rot"], **_scaling(case))
    elif op == "packed":
        dt, hd = ELEM[case["dtype"]], case["hd"]
        lens = _lens(case)
        rows, nq, nk = sum(lens), case["heads_q"] * hd, case["heads_kv"] * hd
        qkv = _randn(g, (rows, nq + 2 * nk), dt)
        qkv[:, :nq] *= 1.5
        st.update(q=qkv[:, :nq], k=qkv[:, nq:nq + nk], v=qkv[:, nq + nk:], lens=lens,
                  offsets=_i32(_offsets(lens)),
                  out=torch.empty((rows, nq), dtype=dt, device="cuda"))
    elif op == "tree":
        ctx, nodes = _lens(case), _nodes(case)
        need = [(c + n + case["bs"] - 1) // case["bs"] for c, n in zip(ctx, nodes)]
        pages, layers, bt_off = sum(need) + 3, 2, _offsets(need)
        cache, pool = _pool(case, g, layers, pages)
        q_off, most = _offsets(nodes), case["nodes"]
        words = (most + 31) // 32
        mask = []
        for n in nodes:  # bit j of row i: drafted token j is i itself or an ancestor
            seen = []
            for i, p in enumerate(_parents(rng, n)):
                seen.append((seen[p] if p >= 0 else 0) | (1 << i))
            mask += [[(m >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for m in seen]
        mask = [[b - (1 << 32) if b >> 31 else b for b in row] for row in mask]
        st.update(cache=cache, pool=pool, layers=layers, pages=pages, layer=1,
                  ctx=ctx, nodes=nodes, q_offsets=_i32(q_off), q_positions=_i32(ctx),
                  table=torch.randperm(pages, generator=g, device="cuda")[:bt_off[-1]].to(torch.int32),
                  bt_offsets=_i32(bt_off), need=need, mask=_i32(mask),
                  q=_randn(g, (q_off[-1], case["heads_q"] * HD), torch.bfloat16, 1.5),
                  out=torch.empty((q_off[-1], case["heads_q"] * HD), dtype=torch.bfloat16,
                                  device="cuda"))
        if own:
            st["workspace"] = torch.empty(
                cache.tree_workspace(len(ctx), heads_q=case["heads_q"], max_q_rows=most,
                                     max_keys=case["hi"] + most),
                dtype=torch.uint8, device="cuda")
    elif op == "copy":
        cache, pool = _pool(case, g, case["layers"], case["pages"])
        ids = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
        n = case["pairs"]
        # a parent may have several children: sources repeat, destinations do not
        src = ids[torch.randint(0, n, (n,), generator=g, device="cuda")]
        st.update(cache=cache, pool=pool, src=src, dst=ids[n:2 * n].contiguous())
    else:
        S, n, bs = case["seqs"], case["nodes"], case["bs"]
        ctx, counts = _kept(case)
        need = [(c + n + bs - 1) // bs for c in ctx]
        first = [c // bs for c in ctx]    # pages before the first drafted token are elsewhere
        bt_off = _offsets(need)
        used = [j >= f for f, m in zip(first, need) for j in range(m)]
        pages = sum(used) + 1
        cache, pool = _pool(case, g, case["layers"], pages)
        perm = torch.randperm(pages, generator=g, device="cuda").tolist()
        table, at = [], 0
        for u in used:
            table.append(perm[at] if u else perm[pages - 1])
            at += 1 if u else 0
        kept = [sorted(rng.sample(range(n), m)) for m in counts]
        k_off = _offsets([len(k) for k in kept])
        st.update(cache=cache, pool=pool, pages=pages, ctx=ctx, kept_list=kept,
                  kept=_i32([i for k in kept for i in k]), kept_offsets=_i32(k_off),
                  q_positions=_i32(ctx), table=_i32(table), bt_offsets=_i32(bt_off),
                  host_table=table, host_bt=bt_off)
    return st


# ------------------------------------------------------------ plain forms ---

def _freqs(case):
    """Rotary frequencies in 64 bits and the factor on cos and sin."""
    sc = _scaling(case)
    d, base, f = case["rot"], sc["base"], sc.get("factor", 1.0)
    i = torch.arange(d // 2, dtype=torch.float64, device="cuda")
    kind = sc["scaling"]
    if kind == "ntk":
        base = base * f ** (d / (d - 2))
    inv = base ** (-2.0 * i / d)
    if kind == "linear":
        return inv / f, 1.0
    if kind == "bands":
        turns = sc["original_len"] * inv / (2 * math.pi)
        s = ((turns - sc["low"]) / (sc["high"] - sc["low"])).clamp(0, 1)
        return inv * ((1 - s) / f + s), 1.0
    if kind == "yarn":
        at = [d * math.log(sc["original_len"] / (2 * math.pi * b)) / (2 * math.log(base))
              for b in (sc["high"], sc["low"])]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv * (1 - ramp) + inv / f * ramp, 0.1 * math.log(f) + 1.0
    return inv, 1.0


def _plain_rope(case, x, heads, cos, sin, out):
    d, hd = case["rot"], case["hd"]
    t = x.reshape(x.shape[0], heads, hd).float()
    r = t[..., :d]
    a, b = (r[..., 0::2], r[..., 1::2]) if case["inter"] else (r[..., :d // 2], r[..., d // 2:])
    c, s = cos[:, None, :], sin[:, None, :]
    ya, yb = a * c - b * s, b * c + a * s
    y = torch.stack((ya, yb), -1).flatten(-2) if case["inter"] else torch.cat((ya, yb), -1)
    return out.copy_(torch.cat((y, t[..., d:]), -1).reshape(x.shape))


def _plain_attend(q, k, v, seen):
    """q [n, Hq, hd], k/v [m, Hkv, hd], seen [n, m]; 32 bits, one key head's queries at a
    time where all the scores together would not fit."""
    n, hq, hd = q.shape
    hkv = k.shape[1]
    qs = q.float().view(n, hkv, hq // hkv, hd).permute(1, 2, 0, 3)   # [Hkv, g, n, hd]
    ks, vs = k.float().transpose(0, 1), v.float().transpose(0, 1)    # [Hkv, m, hd]
    step = max(1, (1 << 31) // max(1, n * k.shape[0] * (hq // hkv)))
    parts = []
    for h in range(0, hkv, step):
        s = torch.einsum("hgnd,hmd->hgnm", qs[h:h + step], ks[h:h + step])
        s = s.mul_(1.0 / math.sqrt(hd)).masked_fill_(~seen, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        parts.append(torch.einsum("hgnm,hmd->hgnd", p / p.sum(-1, keepdim=True), vs[h:h + step]))
    return torch.cat(parts).permute(2, 0, 1, 3).reshape(n, hq * hd)


def _bits(mask, n):
    """[rows, words] masks as truth values [rows, n]."""
    j = torch.arange(n, device=mask.device)
    return (mask[:, j // 32] >> (j % 32)) & 1 == 1


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "rope":
        inv, m = _freqs(case)
        angle = st["positions"].double()[:, None] * inv
        cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
        return [_plain_rope(case, st["q"], case["heads_q"], cos, sin, st["out_q"]),
                _plain_rope(case, st["k"], case["heads_kv"], cos, sin, st["out_k"])]
    if op == "packed":
        hd, at = case["hd"], 0
        for n in filter(None, st["lens"]):
            r = slice(at, at + n)
            i = torch.arange(n, device="cuda")
            st["out"][r] = _plain_attend(st["q"][r].reshape(n, -1, hd), st["k"][r].reshape(n, -1, hd),
                                         st["v"][r].reshape(n, -1, hd), i[:, None] >= i[None, :])
            at += n
        return st["out"]
    if op == "tree":
        pool = _view(case, st["pool"], st["layers"], st["pages"])[:, st["layer"]]
        at = page = 0
        for c, n, m in zip(st["ctx"], st["nodes"], st["need"]):
            kv = pool[st["table"][page:page + m].long()].transpose(0, 1)   # [2, m, bs, W]
            k, v = kv.reshape(2, m * case["bs"], -1, HD)[:, :c + n]
            seen = torch.cat((torch.ones((n, c), dtype=torch.bool, device="cuda"),
                              _bits(st["mask"][at:at + n], n)), 1)
            st["out"][at:at + n] = _plain_attend(st["q"][at:at + n].view(n, -1, HD), k, v, seen)
            at, page = at + n, page + m
        return st["out"]
    if op == "copy":
        view = _view(case, st["pool"], case["layers"], case["pages"])
        view[st["dst"].long()] = view[st["src"].long()]
        return st["pool"]
    # compact: every kept token's page and slot, before and after, in one gather and one store
    bs, ko, bo = case["bs"], st["kept_offsets"].long(), st["bt_offsets"].long()
    view = _view(case, st["pool"], case["layers"], st["pages"])
    row = torch.arange(st["kept"].numel(), device="cuda")
    s = torch.searchsorted(ko, row, right=True) - 1
    old = st["q_positions"].long()[s] + st["kept"].long()
    new = st["q_positions"].long()[s] + row - ko[s]
    page = lambda p: st["table"].long()[bo[s] + p // bs]  # noqa: E731
    view[page(new), :, :, new % bs] = view[page(old), :, :, old % bs]
    return st["pool"]


# ------------------------------------------------------- the framework's ---

def _run_own(st):
    from kvm_b200 import ops
    case = st["case"]
    op = case["op"]
    if op == "rope":
        q, k = ops.rope(st["q"], st["positions"], st["table"], heads=case["heads_q"],
                        head_dim=case["hd"], interleaved=case["inter"], k=st["k"],
                        heads_kv=case["heads_kv"], out=st["out_q"], out_k=st["out_k"])
        return [q, k]
    if op == "packed":
        return ops.attention_packed(st["q"], st["k"], st["v"], st["offsets"],
                                    heads_q=case["heads_q"], heads_kv=case["heads_kv"],
                                    head_dim=case["hd"], out=st["out"])
    if op == "tree":
        return st["cache"].tree_decode(
            st["layer"], st["q"], st["q_offsets"], st["q_positions"], st["mask"], st["table"],
            st["bt_offsets"], heads_q=case["heads_q"], max_q_rows=case["nodes"],
            max_keys=case["hi"] + case["nodes"], out=st["out"], workspace=st["workspace"])
    if op == "copy":
        st["cache"].copy_pages(st["src"], st["dst"])
    else:
        st["cache"].compact(st["kept"], st["kept_offsets"], st["q_positions"], st["table"],
                            st["bt_offsets"])
    return st["pool"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -------------------------------------------------------------- the floor ---

def work(case):
    op = case["op"]
    if op == "rope":
        n = case["rows"] * (case["heads_q"] + case["heads_kv"]) * case["hd"]
        rotated = case["rows"] * (case["heads_q"] + case["heads_kv"]) * case["rot"]
        return dict(bytes=2 * n * ELEM[case["dtype"]].itemsize + 4 * case["rows"],
                    flops=3 * rotated)
    if op == "packed":
        lens = _lens(case)
        rows, hd = sum(lens), case["hd"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        return dict(bytes=2 * rows * hd * (2 * case["heads_q"] + 2 * case["heads_kv"]),
                    flops=4 * pairs * hd * case["heads_q"])
    if op == "tree":
        ctx, nodes = _lens(case), _nodes(case)
        keys, rows = sum(c + n for c, n in zip(ctx, nodes)), sum(nodes)
        pairs = sum(n * (c + n) for c, n in zip(ctx, nodes))
        return dict(bytes=2 * HD * (2 * keys * case["heads_kv"] + 2 * rows * case["heads_q"]),
                    flops=4 * pairs * HD * case["heads_q"])
    slot = case["heads_kv"] * HD * 2 * 2 * case["layers"]   # one token, all layers, K and V
    if op == "copy":
        return dict(bytes=2 * case["pairs"] * case["bs"] * slot, flops=0)
    return dict(bytes=2 * sum(_kept(case)[1]) * slot, flops=0)


# ------------------------------------------------- the definition, 64 bits ---

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        f, m = _freqs(case)
        outs = []
        for x, heads in ((st["q"], case["heads_q"]), (st["k"], case["heads_kv"])):
            z = x.double().reshape(x.shape[0], heads, case["hd"]).clone()
            for i in range(case["rot"] // 2):
                a, b = (2 * i, 2 * i + 1) if case["inter"] else (i, i + case["rot"] // 2)
                turn = torch.polar(torch.full_like(st["positions"], 1, dtype=torch.float64) * m,
                                   st["positions"].double() * f[i])
                pair = torch.complex(z[..., a], z[..., b]) * turn[:, None]
                z[..., a], z[..., b] = pair.real, pair.imag
            outs.append(z.reshape(x.shape))
        return outs
    if op in ("packed", "tree"):
        hd = case.get("hd", HD)
        group = case["heads_q"] // case["heads_kv"]
        q = st["q"].double()
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        at = page = 0
        counts = st["lens"] if op == "packed" else st["nodes"]
        for s, n in enumerate(counts):
            if op == "packed":
                k, v = st["k"][at:at + n].double(), st["v"][at:at + n].double()
                seen = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
            else:
                c, m = st["ctx"][s], st["need"][s]
                pool = _view(case, st["pool"], st["layers"], st["pages"])
                rows = [pool[p, st["layer"]] for p in st["table"][page:page + m].tolist()]
                k = torch.cat([r[0] for r in rows])[:c + n].double()
                v = torch.cat([r[1] for r in rows])[:c + n].double()
                seen = torch.ones((n, c + n), dtype=torch.bool, device="cuda")
                for i, words in enumerate(st["mask"][at:at + n].tolist()):
                    seen[i, c:] = torch.tensor([words[j // 32] >> (j % 32) & 1 == 1
                                                for j in range(n)], device="cuda")
                page += m
            for h in range(case["heads_q"]):
                kh = h // group
                qc, kc = slice(h * hd, (h + 1) * hd), slice(kh * hd, (kh + 1) * hd)
                for r in range(0, n, 4096):
                    e = min(n, r + 4096)
                    z = (q[at + r:at + e, qc] @ k[:, kc].T) / math.sqrt(hd)
                    w = torch.softmax(z.masked_fill(~seen[r:e], -math.inf), -1)
                    out[at + r:at + e, qc] = w @ v[:, kc]
            at += n
        return out
    if op == "copy":
        view = _view(case, st["pool"], case["layers"], case["pages"])
        before = view.clone()
        for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
            view[b] = before[a]
        return st["pool"].double()
    view = _view(case, st["pool"], case["layers"], st["pages"])
    bs = case["bs"]
    for s, kept in enumerate(st["kept_list"]):
        place = lambda p: (st["host_table"][st["host_bt"][s] + p // bs], p % bs)  # noqa: E731
        moved = [view[place(st["ctx"][s] + j)[0], :, :, place(st["ctx"][s] + j)[1]].clone()
                 for j in kept]
        for i, row in enumerate(moved):
            p, slot = place(st["ctx"][s] + i)
            view[p, :, :, slot] = row
    return st["pool"].double()

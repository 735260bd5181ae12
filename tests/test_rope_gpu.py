"""Rotary embedding with a position per row against the rotation in 64 bits.

Tolerance. The kernel's angle is off by at most pi 2^-25 (a fraction of a turn
rounded to 24 bits; the 64-bit product adds less than 2^-31), sincospif by
2^-22 at most (two units in the last place of values up to 1), the factor m
and the products by a few 2^-24: together below 2^-21 (|a| + |b|) m. The result
is then rounded once to the tensor's type: eps / 2 of its value."""
import math

import pytest
import torch

from kvm_b200 import ops
from kvm_b200._lib import KvmError

pytestmark = pytest.mark.gpu


def _freqs(d, base=10000.0, scaling="none", factor=1.0, original_len=0.0, low=1.0, high=32.0,
           magnitude=0.0, divisors=None):
    i = torch.arange(d // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (d / (d - 2))
    f = base ** (-2 * i / d)
    m = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":
        t = original_len * f / (2 * math.pi)
        keep = ((t - low) / (high - low)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    elif scaling == "yarn":
        lo, hi = (d * math.log(original_len / (2 * math.pi * b)) / (2 * math.log(base))
                  for b in (high, low))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), d - 1)
        keep = 1 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        m = 0.1 * math.log(factor) + 1
    elif scaling == "divisors":
        f = f / torch.tensor(divisors, dtype=torch.float64)
    return f, magnitude or m


def _ref(x, pos, heads, hd, f, m, inter, backward=False):
    """(rotated, |a| + |b| of each element's pair), in 64 bits on the CPU."""
    d = 2 * len(f)
    t = x.double().cpu().reshape(x.shape[0], heads, hd)
    ang = pos.cpu().double()[:, None] * f
    c, s = (ang.cos() * m)[:, None], (ang.sin() * m * (-1 if backward else 1))[:, None]
    ia = torch.arange(0, d, 2) if inter else torch.arange(d // 2)
    ib = ia + 1 if inter else ia + d // 2
    a, b = t[..., ia], t[..., ib]
    y, size = t.clone(), torch.zeros_like(t)
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * m
    return y.reshape(x.shape), size.reshape(x.shape)


def _close(got, ref, size):
    tol = size * 2.0 ** -21 + ref.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -20)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25      # half a step of the subnormal numbers
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


YARN = dict(scaling="yarn", factor=16.0, original_len=4096)
BANDS = dict(scaling="bands", factor=8.0, original_len=8192, low=1.0, high=4.0, base=500000.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rows,heads,kvh,hd,rot,cfg", [
    (1, 8, 1, 128, 128, {}),
    (1, 64, 8, 128, 128, YARN),
    (37, 5, 5, 64, 32, dict(scaling="linear", factor=4.0)),
    (130, 12, 3, 80, 80, dict(scaling="ntk", factor=8.0)),
    (33, 3, 0, 96, 36, BANDS),                 # 36 columns: no 16-byte units
    (9, 1, 1, 256, 256, YARN),
    (5, 40, 8, 10, 6, {}),                     # rows that are not 16-byte aligned
    (7, 2, 1, 128, 2, {}),
])
def test_rope(cuda, dtype, inter, rows, heads, kvh, hd, rot, cfg):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + heads)
    f, m = _freqs(rot, **cfg)
    table = ops.rope_table(rot, **cfg)
    q = torch.randn((rows, heads * hd), generator=g, device=cuda).to(dtype)
    pos = torch.randint(0, 200000, (rows,), generator=g, device=cuda, dtype=torch.int32)
    pos[0] = 0
    if kvh:
        k = torch.randn((rows, kvh * hd), generator=g, device=cuda).to(dtype)
        yq, yk = ops.rope(q, pos, table, heads=heads, head_dim=hd, interleaved=inter, k=k,
                          heads_kv=kvh)
        _close(yk, *_ref(k, pos, kvh, hd, f, m, inter))
    else:
        yq = ops.rope(q, pos, table, heads=heads, head_dim=hd, interleaved=inter)
    ref, size = _ref(q, pos, heads, hd, f, m, inter)
    _close(yq, ref, size)
    kept = size == 0                            # columns that only pass through
    assert torch.equal(yq.cpu().double()[kept], ref[kept])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("heads,kvh,hd,rot", [
    (64, 8, 128, 128),      # one to three blocks a row
    (64, 8, 128, 64),
    (37, 5, 128, 128),      # a last pass that is not full
    (50, 3, 80, 32),
    (31, 2, 96, 36),        # units of one pair, many blocks a row
    (1, 70, 64, 64),        # the border of q and k within the first pass
])
def test_rope_many_rows(cuda, dtype, inter, heads, kvh, hd, rot):
    """More rows than two blocks an SM, where blocks take their heads in two or
    three passes; in place the same bits."""
    rows = 300
    g = torch.Generator(device="cuda").manual_seed(heads + hd + rot)
    f, m = _freqs(rot, **YARN)
    table = ops.rope_table(rot, **YARN)
    qkv = torch.randn((rows, (heads + kvh) * hd + 8), generator=g, device=cuda).to(dtype)
    q, k = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kvh) * hd]
    pos = torch.randint(0, 100000, (rows,), generator=g, device=cuda)
    kw = dict(heads=heads, head_dim=hd, interleaved=inter, k=k, heads_kv=kvh)
    yq, yk = ops.rope(q, pos, table, **kw)
    for got, x, n in ((yq, q, heads), (yk, k, kvh)):
        ref, size = _ref(x, pos, n, hd, f, m, inter)
        _close(got, ref, size)
        kept = size == 0
        assert torch.equal(got.cpu().double()[kept], ref[kept])
    tail = qkv[:, (heads + kvh) * hd:].clone()
    ops.rope(q, pos, table, out=q, out_k=k, **kw)
    assert torch.equal(q, yq) and torch.equal(k, yk)
    assert torch.equal(qkv[:, (heads + kvh) * hd:], tail)


def test_rope_far_and_negative_positions(cuda):
    """int64 positions up to 2^40 and negative ones. The 64-bit reference angle
    is itself rounded (2^40 * 2^-53 = 2^-13), so the far rows are checked with
    frequencies that are exact fractions of a turn."""
    hd = 64
    table = ops.rope_table(hd)
    for i in range(hd // 2):
        table.turns[i] = ((i + 1) << 58) + (i << 20)   # (i+1)/64 turn + i 2^-44
    pos = torch.tensor([0, 1, -1, 2 ** 40 + 5, -(2 ** 40) - 3, 2 ** 62 + 7, -2 ** 63],
                       dtype=torch.int64, device=cuda)
    q = torch.randn((len(pos), hd), device=cuda)
    y = ops.rope(q, pos, table, heads=1, head_dim=hd)
    t = q.double().cpu()
    for r, p in enumerate(pos.tolist()):
        for i in range(hd // 2):
            turn = (p * table.turns[i]) % 2 ** 64 / 2 ** 64
            c, s = math.cos(2 * math.pi * turn), math.sin(2 * math.pi * turn)
            a, b = float(t[r, i]), float(t[r, i + hd // 2])
            tol = (abs(a) + abs(b)) * 2.0 ** -20
            assert abs(float(y[r, i]) - (a * c - b * s)) <= tol
            assert abs(float(y[r, i + hd // 2]) - (b * c + a * s)) <= tol


def test_rope_in_place_on_views_of_one_matrix(cuda):
    """q and k as column slices of a fused matrix, rotated in place: same bits
    as out of place, value columns untouched."""
    rows, hq, hkv, hd = 50, 8, 2, 128
    qkv = torch.randn((rows, (hq + 2 * hkv) * hd), device=cuda).to(torch.bfloat16)
    before = qkv.clone()
    q, k = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hkv) * hd]
    pos = torch.arange(rows, device=cuda, dtype=torch.int64) * 3
    table = ops.rope_table(64)
    yq, yk = ops.rope(q, pos, table, heads=hq, k=k, heads_kv=hkv)
    assert torch.equal(qkv, before)
    rq, rk = ops.rope(q, pos, table, heads=hq, k=k, heads_kv=hkv, out=q, out_k=k)
    assert rq is q and torch.equal(q, yq) and torch.equal(k, yk)
    assert torch.equal(qkv[:, (hq + hkv) * hd:], before[:, (hq + hkv) * hd:])


def test_rope_matches_the_row_index_form(cuda):
    """rope_ (position = row index) gives the same rotation."""
    x = torch.randn((64, 4 * 128), device=cuda).to(torch.bfloat16)
    y = ops.rope(x, torch.arange(64, device=cuda), ops.rope_table(128), heads=4)
    ops.rope_(x, seq_len=64, heads=4)
    diff = (y.double() - x.double()).abs()
    # Each side rounds once, by at most eps / 2 = 2^-8 of its value: 2 * 2^-8 between them,
    # of a value that is itself 2^-8 off. rope_'s angle is a product of up to 63 with a
    # powf that is a few 2^-23 off: 2^-16, times |a| + |b| < 12: below 2^-12.
    assert bool((diff <= x.double().abs() * 2.0 ** -7 * (1 + 2.0 ** -7) + 2.0 ** -12).all())


@pytest.mark.parametrize("inter", [False, True])
def test_rope_backward(cuda, inter):
    """backward=True is the gradient of <g, rope(x)>: against the transposed
    rotation in 64 bits, and against central differences of the forward call
    (linear in x, so their only error is the rounding of the two results)."""
    rows, hd = 6, 32
    cfg = dict(scaling="yarn", factor=4.0, original_len=256)
    f, m = _freqs(24, **cfg)
    table = ops.rope_table(24, **cfg)
    pos = torch.tensor([0, 1, 5, 300, 4000, 100000], device=cuda)
    x, g = torch.randn((2, rows, hd), device=cuda)
    kw = dict(heads=1, head_dim=hd, interleaved=inter)
    dx = ops.rope(g, pos, table, backward=True, **kw)
    _close(dx, *_ref(g, pos, 1, hd, f, m, inter, backward=True))
    for j in (0, 1, 11, 12, 23, 24, 31):
        e = torch.zeros_like(x)
        e[:, j] = 0.5
        up = ops.rope(x + e, pos, table, **kw).double()
        dn = ops.rope(x - e, pos, table, **kw).double()
        num = ((up - dn) * g.double()).sum(1)
        tol = g.double().abs().sum(1) * 2.0 ** -18   # |x| < 8: 2 * 16 * 2^-21 m / (2 * 0.5) and more
        assert bool(((num - dx[:, j].double()).abs() <= tol).all())


def test_rope_refusals_and_empty(cuda):
    table = ops.rope_table(128)
    q = torch.zeros((4, 256), dtype=torch.bfloat16, device=cuda)
    pos = torch.zeros(4, dtype=torch.int32, device=cuda)
    e = ops.rope(q[:0], pos[:0], table, heads=2)
    assert e.shape == (0, 256)
    for kw in (dict(heads=3), dict(heads=4, head_dim=64), dict(heads=2, k=q),
               dict(heads=2, k=q[:3], heads_kv=2)):
        with pytest.raises((ValueError, KvmError)):
            ops.rope(q, pos, table, **kw)
    with pytest.raises(ValueError):
        ops.rope(q, pos[:3], table, heads=2)
    with pytest.raises(TypeError):
        ops.rope(q, pos.float(), table, heads=2)
    with pytest.raises(TypeError):
        ops.rope(q.to(torch.float64), pos, table, heads=2)
    big = torch.zeros((4, 512), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(KvmError):                       # in place with two row strides
        ops.rope(big[:, :256], pos, table, heads=2, out=torch.as_strided(big, (4, 256), (256, 1)))


def test_rope_on_a_side_stream_and_in_a_graph(cuda):
    table = ops.rope_table(128)
    q = torch.randn((16, 512), device=cuda).to(torch.bfloat16)
    pos = torch.arange(16, device=cuda)
    want = ops.rope(q, pos, table, heads=4)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.rope(q, pos, table, heads=4, out=out)
    s.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rope(q, pos, table, heads=4, out=out)
    pos += 7
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.rope(q, pos, table, heads=4))

"""Packed causal attention against its formula in 64 bits.

Tolerance, per element, with A = sum_j p_j |v_j| of the exact softmax: each
P value is rounded once to the type (eps / 2 of it: eps / 2 * A), the result
once (eps / 2 of it). Scores are fp32 sums of hd products of 16-bit numbers,
scaled: for the normal data here |q . k| scale stays below 64, so a score is
off by less than 64 * 2^-24 * sqrt(hd) and P by less than 2^-13 of itself;
ex2, the sum l and the division add a few 2^-22. Below 2^-14 a half-precision
P is subnormal: half its step, 2^-25, per key, divided by l >= 1/2."""
import math

import pytest
import torch

from kvm_b200 import ops
from kvm_b200._lib import KvmError

pytestmark = pytest.mark.gpu


def exact(q, k, v, lens, hq, hkv, hd, start=0, scale=None):
    """(out, A) in 64 bits; rows outside the sequences are zero."""
    scale = scale or 1 / math.sqrt(hd)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    at, g = start, hq // hkv
    for n in lens:
        r = slice(at, at + n)
        Q = q[r].double().view(n, hkv, g, hd)
        K, V = (t[r].double().view(n, hkv, hd) for t in (k, v))
        s = torch.einsum("nhgd,mhd->hgnm", Q, K) * scale
        seen = torch.ones((n, n), dtype=torch.bool, device=q.device).tril()
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        # a value that a row does not see takes no part, whatever it is
        out[r] = torch.einsum("hgnm,mhd->nhgd", p, V).reshape(n, hq * hd)
        mag[r] = torch.einsum("hgnm,mhd->nhgd", p, V.abs()).reshape(n, hq * hd)
        at += n
    return out, mag


def check(got, out, mag, n_keys, vmax=6.0):
    half = torch.finfo(got.dtype).eps / 2
    tol = half * (mag * (1 + 2 * half) + out.abs()) + 2.0 ** -13 * mag
    if got.dtype == torch.float16:
        tol = tol + 2 * n_keys * vmax * 2.0 ** -25 + 2.0 ** -25
    err = (got.double() - out).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def make(cuda, lens, hq, hkv, hd, dtype, seed=0, extra=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(lens) + extra
    q, k, v = (torch.randn((rows, h * hd), generator=g, device=cuda).to(dtype)
               for h in (hq, hkv, hkv))
    off = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=cuda)
    return q * std, k, v, off


@pytest.mark.parametrize("lens,hq,hkv", [
    ([1], 1, 1),
    ([128], 1, 1),
    ([1, 0, 127, 128, 129, 3, 0], 4, 2),
    ([300, 17, 256, 255, 257], 8, 1),
    ([5, 64, 640, 33], 3, 1),
    ([77, 513], 10, 2),              # 5 heads a group
    ([130, 1, 1, 2], 14, 2),         # 7
    ([200, 31, 90], 32, 2),          # 16
    ([50, 3], 128, 1),               # 128: one token a tile
    ([20, 9], 100, 1),               # 100
    ([700, 1100], 2, 2),
])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed(cuda, lens, hq, hkv, hd, dtype):
    q, k, v, off = make(cuda, lens, hq, hkv, hd, dtype, seed=len(lens) + hq)
    out = ops.attention_packed(q, k, v, off, heads_q=hq, heads_kv=hkv, head_dim=hd)
    ops.device_status()
    check(out, *exact(q, k, v, lens, hq, hkv, hd), max(lens))


def test_packed_long_and_peaked(cuda):
    """5000 keys, scores of standard deviation 4: a few keys dominate."""
    lens = [5003, 1200]
    q, k, v, off = make(cuda, lens, 8, 2, 128, torch.bfloat16, seed=5, std=4.0)
    out = ops.attention_packed(q, k, v, off, heads_q=8, heads_kv=2)
    ops.device_status()
    check(out, *exact(q, k, v, lens, 8, 2, 128), 5003)


def test_packed_many_sequences(cuda):
    lens = [(i * 37) % 61 for i in range(1024)]
    q, k, v, off = make(cuda, lens, 4, 1, 64, torch.bfloat16, seed=6)
    out = ops.attention_packed(q, k, v, off, heads_q=4, heads_kv=1, head_dim=64)
    ops.device_status()
    check(out, *exact(q, k, v, lens, 4, 1, 64), 61)
    with pytest.raises(KvmError):
        ops.attention_packed(q, k, v, torch.zeros(1026, dtype=torch.int32, device=cuda),
                             heads_q=4, heads_kv=1, head_dim=64)


def test_packed_later_keys_dominate(cuda):
    """Growing keys raise each row's maximum by far more than 2^8 in every tile,
    so the accumulator is rescaled again and again."""
    lens = [900, 400]
    q, k, v, off = make(cuda, lens, 4, 2, 128, torch.bfloat16, seed=7)
    k = (k.float() * (1 + torch.arange(1300, device=cuda)[:, None] // 100)).to(torch.bfloat16)
    out = ops.attention_packed(q, k, v, off, heads_q=4, heads_kv=2)
    ops.device_status()
    # scores reach 13 times 64: P is off by 13 * 2^-13 more
    ref, mag = exact(q, k, v, lens, 4, 2, 128)
    check(out, ref, mag * (1 + 13 * 2.0 ** -5), 900)


def test_packed_views_scale_and_foreign_rows(cuda):
    """Column slices of one matrix, a first sequence that does not begin at row
    0, rows behind the last one: those stay as they were."""
    lens, hq, hkv, hd = [70, 260], 4, 2, 128
    rows = 9 + sum(lens) + 30
    qkv = torch.randn((rows, (hq + 2 * hkv) * hd), device=cuda).to(torch.bfloat16)
    q, k, v = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hkv) * hd], qkv[:, (hq + hkv) * hd:]
    off = torch.tensor([9, 79, 339], dtype=torch.int32, device=cuda)
    big = torch.full((rows, hq * hd + 64), 7.0, dtype=torch.bfloat16, device=cuda)
    res = ops.attention_packed(q, k, v, off, heads_q=hq, heads_kv=hkv, scale=0.2,
                               out=big[:, :hq * hd])
    ops.device_status()
    ref, mag = exact(q, k, v, lens, hq, hkv, hd, start=9, scale=0.2)
    check(res[9:339], ref[9:339], mag[9:339], 260)
    assert bool((big[:9] == 7).all()) and bool((big[339:] == 7).all())
    assert bool((big[:, hq * hd:] == 7).all())


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_packed_broken_values_reach_only_who_sees_them(cuda, dtype, hd, group):
    """NaN and infinities in keys and values: rows before them and other
    sequences come out as if they were not there; rows that see an infinite
    value get it."""
    lens, hkv = [100, 300, 40], 2
    hq = group * hkv
    q, k, v, off = make(cuda, lens, hq, hkv, hd, dtype, seed=8)
    clean, mag = exact(q, k, v, lens, hq, hkv, hd)
    nan, inf = float("nan"), float("inf")
    k[100 + 150] = nan                  # sequence 1 from its row 150 on
    v[100 + 140, :hd] = inf             # kv head 0, from row 140 on
    v[100 + 145, 3] = nan
    v[60, hd] = -inf                    # sequence 0, head 1, column 0, from row 60 on
    q[139 + 100 + 161 + 20] = nan       # sequence 2: row 20 alone
    out = ops.attention_packed(q, k, v, off, heads_q=hq, heads_kv=hkv, head_dim=hd)
    ops.device_status()
    o = out.view(-1, hkv, group, hd)
    ok = torch.ones_like(o, dtype=torch.bool)
    ok[100 + 140:400, 0] = False
    ok[100 + 150:400] = False
    ok[60:100, 1, :, 0] = False
    ok[420] = False
    ok = ok.view(out.shape)
    err = (out.double() - clean).abs()
    half = torch.finfo(dtype).eps / 2
    tol = half * (mag * (1 + 2 * half) + clean.abs()) + 2.0 ** -13 * mag + 300 * 2.0 ** -20
    assert bool((err[ok] <= tol[ok]).all())
    assert bool((o[240:245, 0] == inf).all())                 # infinity, nothing undefined
    assert bool(torch.isnan(o[245:250, 0, :, 3]).all())
    assert bool((o[60:100, 1, :, 0] == -inf).all())
    assert bool(torch.isnan(o[250:400]).all()) and bool(torch.isnan(o[420]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_infinite_value_of_no_weight(cuda, dtype):
    """An infinite value under a weight that P cannot hold, in a key tile that a
    row sees whole and in one that it sees in part: the column is not finite in
    the rows that see it, and nothing else changes."""
    lens, hd = [400], 64
    q, k, v, off = make(cuda, lens, 1, 1, hd, dtype, seed=12)
    q[:, 0] = 40
    k[:, 0] = 20                        # each score is 100, give or take a few,
    for j in (20, 290):
        k[j, 0] = -20                   # but these keys' is -100: weight e^-190
    clean, mag = exact(q, k, v, lens, 1, 1, hd)
    v[20, 3] = float("inf")
    v[290, 5] = -float("inf")
    out = ops.attention_packed(q, k, v, off, heads_q=1, heads_kv=1, head_dim=hd)
    ops.device_status()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[20:, 3] = bad[290:, 5] = True
    assert bool((~torch.isfinite(out[bad])).all())
    # scores are 100 instead of at most 64: P is off by twice as much
    check(out[~bad], clean[~bad], 2 * mag[~bad], 400)


def test_packed_bad_offsets_are_reported(cuda):
    q, k, v, _ = make(cuda, [64], 2, 1, 128, torch.bfloat16)
    out = torch.full_like(q, 3.0)
    off = torch.tensor([0, 20, 10, 200, 64], dtype=torch.int32, device=cuda)
    ops.attention_packed(q, k, v, off, heads_q=2, heads_kv=1, out=out)
    with pytest.raises(KvmError):
        ops.device_status()
    check(out[:20], *(t[:20] for t in exact(q, k, v, [20], 2, 1, 128)), 20)
    assert bool((out[20:] == 3).all())
    # what comes after a bad pair could cover rows twice: left out too
    off = torch.tensor([0, 30, 10, 64], dtype=torch.int32, device=cuda)
    out.fill_(3.0)
    ops.attention_packed(q, k, v, off, heads_q=2, heads_kv=1, out=out)
    with pytest.raises(KvmError):
        ops.device_status()
    check(out[:30], *(t[:30] for t in exact(q, k, v, [30], 2, 1, 128)), 30)
    assert bool((out[30:] == 3).all())


def test_packed_graph_and_stream(cuda):
    """The lengths are read on the device: a captured call serves other ones."""
    lens, other = [90, 200, 10], [1, 150, 149]
    q, k, v, off = make(cuda, lens, 8, 2, 128, torch.bfloat16, seed=9)
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.attention_packed(q, k, v, off, heads_q=8, heads_kv=2, out=out)
    s.synchronize()
    check(out, *exact(q, k, v, lens, 8, 2, 128), 200)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_packed(q, k, v, off, heads_q=8, heads_kv=2, out=out)
    off.copy_(torch.tensor([0, 1, 151, 300]))
    graph.replay()
    ops.device_status()
    check(out, *exact(q, k, v, other, 8, 2, 128), 150)


def test_packed_same_bits_every_time(cuda):
    lens = [500, 33, 129, 1000]
    q, k, v, off = make(cuda, lens, 16, 2, 128, torch.bfloat16, seed=10)
    a = ops.attention_packed(q, k, v, off, heads_q=16, heads_kv=2)
    for _ in range(20):
        assert torch.equal(a, ops.attention_packed(q, k, v, off, heads_q=16, heads_kv=2))


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (12, 4, 64), (5, 1, 128)])
def test_packed_a_sequence_is_the_same_in_any_batch(cuda, hq, hkv, hd):
    """Bit for bit: alone, and between others whose rows share its tiles."""
    lens = [333, 50, 1, 700]
    q, k, v, off = make(cuda, lens, hq, hkv, hd, torch.bfloat16, seed=11, std=3.0)
    kw = dict(heads_q=hq, heads_kv=hkv, head_dim=hd)
    out = ops.attention_packed(q, k, v, off, **kw)
    for s in range(4):
        r = slice(int(off[s]), int(off[s + 1]))
        one = torch.tensor([0, lens[s]], dtype=torch.int32, device=cuda)
        assert torch.equal(out[r], ops.attention_packed(q[r], k[r], v[r], one, **kw))


def test_packed_refusals_and_empty(cuda):
    q, k, v, off = make(cuda, [8], 4, 2, 128, torch.bfloat16)
    kw = dict(heads_q=4, heads_kv=2)
    assert ops.attention_packed(q[:0], k[:0], v[:0], off * 0, **kw).shape == (0, 512)
    assert bool((ops.attention_packed(q, k, v, off[:1], **kw) == 0).all())
    assert bool((ops.attention_packed(q, k, v, off * 0, **kw) == 0).all())
    for bad in (dict(heads_q=4, heads_kv=1), dict(heads_q=3, heads_kv=2),
                dict(heads_q=8, heads_kv=4, head_dim=64, scale=float("nan")),
                dict(heads_q=16, heads_kv=8, head_dim=32)):
        with pytest.raises((ValueError, KvmError)):
            ops.attention_packed(q, k, v, off, **bad)
    with pytest.raises(ValueError):
        ops.attention_packed(q, k, v, off.cpu(), **kw)
    with pytest.raises(TypeError):
        ops.attention_packed(q, k, v, off.long(), **kw)
    with pytest.raises(TypeError):
        ops.attention_packed(q.float(), k.float(), v.float(), off, **kw)
    with pytest.raises(ValueError):
        ops.attention_packed(q, k[:7], v, off, **kw)

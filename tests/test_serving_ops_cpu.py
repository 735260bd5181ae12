"""Host side of the serving operators: the rotary table against 50-digit
arithmetic, and the refusals of the C ABI (no GPU)."""
import ctypes as C
from decimal import Decimal, getcontext

import pytest
import torch

from kvm_b200 import _lib, ops
from kvm_b200._lib import KvmError

PI = Decimal("3.14159265358979323846264338327950288419716939937510")


def _turns(d, base=10000, factor=1, kind="none", orig=0, low=1, high=32, div=None):
    """f_i / 2 pi in 50 digits."""
    getcontext().prec = 50
    D = Decimal
    base = D(base)
    if kind == "ntk":
        base *= D(factor) ** (D(d) / D(d - 2))
    fs = [base ** (D(-2 * i) / D(d)) for i in range(d // 2)]
    if kind == "linear":
        fs = [f / D(factor) for f in fs]
    if kind == "bands":
        keep = [min(max((D(orig) * f / (2 * PI) - D(low)) / (D(high) - D(low)), D(0)), D(1))
                for f in fs]
        fs = [f * k + f / D(factor) * (1 - k) for f, k in zip(fs, keep)]
    if kind == "yarn":
        lo, hi = (D(d) * (D(orig) / (2 * PI * D(b))).ln() / (2 * base.ln()) for b in (high, low))
        lo = max(lo.to_integral_value("ROUND_FLOOR"), D(0))
        hi = min(hi.to_integral_value("ROUND_CEILING"), D(d - 1))
        keep = [1 - min(max((i - lo) / max(hi - lo, D("1e-3")), D(0)), D(1))
                for i in range(d // 2)]
        fs = [f * k + f / D(factor) * (1 - k) for f, k in zip(fs, keep)]
    if kind == "divisors":
        fs = [f / D(x) for f, x in zip(fs, div)]
    return [f / (2 * PI) for f in fs]


@pytest.mark.parametrize("d,kw,ref", [
    (128, {}, {}),
    (64, dict(base=500000.0), dict(base=500000)),
    (256, dict(scaling="linear", factor=7.0), dict(kind="linear", factor=7)),
    (80, dict(scaling="ntk", factor=4.0), dict(kind="ntk", factor=4)),
    (128, dict(scaling="bands", factor=8.0, original_len=8192, low=1.0, high=4.0,
               base=500000.0), dict(kind="bands", factor=8, orig=8192, low=1, high=4, base=500000)),
    (64, dict(scaling="yarn", factor=32.0, original_len=4096),
     dict(kind="yarn", factor=32, orig=4096)),
    (8, dict(scaling="divisors", divisors=[1.0, 2.0, 3.5, 64.0]),
     dict(kind="divisors", div=["1", "2", "3.5", "64"])),
])
def test_rope_table(d, kw, ref):
    """Turns as 64-bit fractions: long double arithmetic has 64 bits, a dozen
    roundings of a value below 2^62, so a few dozen units at most."""
    t = ops.rope_table(d, **kw)
    assert t.pairs == d // 2
    for got, want in zip(t.turns, _turns(d, **ref)):
        assert abs(int(want * 2 ** 64) - got) <= 64, (got, want)
    if kw.get("scaling") == "yarn":
        assert abs(t.magnitude - (0.1 * float(Decimal(32).ln()) + 1)) < 1e-6
    else:
        assert t.magnitude == 1.0
    assert ops.rope_table(d, magnitude=1.25, **kw).magnitude == 1.25


@pytest.mark.parametrize("d,kw", [
    (0, {}), (7, {}), (258, {}), (64, dict(base=1.0)), (64, dict(base=float("nan"))),
    (64, dict(scaling="linear", factor=0.5)), (64, dict(scaling="linear", factor=float("inf"))),
    (64, dict(scaling="bands", factor=2.0)), (2, dict(scaling="ntk", factor=2.0)),
    (64, dict(scaling="yarn", factor=2.0, original_len=100, low=4.0, high=4.0)),
    (64, dict(magnitude=-1.0)), (4, dict(scaling="divisors", divisors=[1.0, 0.0])),
])
def test_rope_table_refuses(d, kw):
    with pytest.raises(KvmError) as e:
        ops.rope_table(d, **kw)
    assert e.value.code == _lib.KVM_ERR_INVALID_ARG


@pytest.mark.parametrize("magnitude", [1e39, 1e-50, float("inf"), float("nan")])
def test_rope_table_refuses_a_magnitude_that_fp32_cannot_hold(magnitude):
    """The table holds it in fp32, where these are infinity, zero or not numbers."""
    with pytest.raises(KvmError) as e:
        ops.rope_table(64, magnitude=magnitude)
    assert e.value.code == _lib.KVM_ERR_INVALID_ARG


def test_rope_table_python_refusals():
    with pytest.raises(ValueError):
        ops.rope_table(64, scaling="other")
    with pytest.raises(ValueError):
        ops.rope_table(64, scaling="divisors", divisors=[1.0])
    with pytest.raises(ValueError):
        ops.rope_table(64, divisors=[1.0] * 32)


def _rc(name, *args):
    return getattr(_lib.lib(), "kvm_sm100_" + name)(*args)


def test_rope_refuses_without_a_gpu():
    t = C.byref(ops.rope_table(64))
    P = 4096   # an aligned address that is never read
    ok = [t, P, 128, P, 128, 2, None, 0, None, 0, 0, 4, 64, 0, 0, 0, P, 0, None]

    def bad(**at):
        args = list(ok)
        for i, v in at.items():
            args[int(i[1:])] = v
        return _rc("rope", *args)
    INV = _lib.KVM_ERR_INVALID_ARG
    assert bad(a0=None) == INV and bad(a1=None) == INV and bad(a16=None) == INV
    assert bad(a2=100) == INV            # row stride below heads * head_dim
    assert bad(a5=0) == INV and bad(a12=62) == INV and bad(a12=65) == INV and bad(a12=258) == INV
    assert bad(a15=3) == INV and bad(a1=P + 1) == INV and bad(a16=P + 2) == INV
    assert bad(a4=192) == INV            # in place with two row strides
    assert bad(a10=1) == INV             # key heads without a key tensor
    assert bad(a11=-1) == INV and bad(a11=0) == _lib.KVM_OK


def test_page_calls_refuse_without_a_gpu():
    L = _lib.KvLayout(4096, 2048, 1024, 64, 16, 0, 64, 4)
    P = 4096
    INV = _lib.KVM_ERR_INVALID_ARG
    copy = lambda *a: _rc("kvcache_copy_pages", *a)  # noqa: E731
    assert copy(P, None, 1, P, P, 1, None) == INV
    assert copy(None, C.byref(L), 1, P, P, 1, None) == INV
    assert copy(P, C.byref(L), 0, P, P, 1, None) == INV
    assert copy(P, C.byref(L), 1, P, P, -1, None) == INV
    assert copy(P, C.byref(L), 1, None, P, 1, None) == INV
    assert copy(P, C.byref(L), 1, None, None, 0, None) == _lib.KVM_OK
    wide = _lib.KvLayout(8192, 4096, 2048, 128, 16, 0, 64, 4)
    assert copy(P, C.byref(wide), 1, P, P, 1, None) in (_lib.KVM_ERR_UNSUPPORTED,
                                                        _lib.KVM_ERR_CUDA)
    comp = lambda *a: _rc("kvcache_compact", *a)  # noqa: E731
    assert comp(P, C.byref(L), 1, None, 1, P, P, P, 4, P, 1, None) == INV
    assert comp(P, C.byref(L), 1, P, -1, P, P, P, 4, P, 1, None) == INV
    assert comp(P + 8, C.byref(L), 1, P, 1, P, P, P, 4, P, 1, None) == INV
    assert comp(P, C.byref(L), 1, P, 1, P, P, P, -1, P, 1, None) == INV
    assert comp(P, C.byref(L), 1, None, 0, None, None, None, 0, None, 1, None) == _lib.KVM_OK


def test_tree_mask():
    from kvm_b200.kvcache import tree_mask
    m = tree_mask([-1, 0, 0, 1, -1])
    assert m.tolist() == [[1], [3], [5], [11], [16]]
    chain = tree_mask(range(-1, 69))
    assert chain.shape == (70, 3)
    got = [sum((w & 0xFFFFFFFF) << (32 * i) for i, w in enumerate(r)) for r in chain.tolist()]
    assert got == [(1 << (i + 1)) - 1 for i in range(70)]
    assert tree_mask([]).shape == (0, 1)
    for bad in ([0], [-1, 1], [-1, -2], [-1, 5]):
        with pytest.raises(ValueError):
            tree_mask(bad)


def test_attention_packed_refuses_without_a_gpu():
    P, INV, UNS = 4096, _lib.KVM_ERR_INVALID_ARG, _lib.KVM_ERR_UNSUPPORTED
    ok = [P, 512, P, 256, P, 256, P, 512, P, 3, 100, 4, 2, 128, 0, 0.0, None]

    def rc(**at):
        args = list(ok)
        for i, v in at.items():
            args[int(i[1:])] = v
        return _rc("attention_packed", *args)
    assert rc(a9=-1) == INV and rc(a10=-1) == INV and rc(a11=3) == INV and rc(a12=0) == INV
    assert rc(a13=32) == UNS and rc(a14=1) == UNS and rc(a9=1025) == UNS
    assert rc(a11=258, a1=1 << 20, a7=1 << 20) == UNS       # 129 query heads a kv head
    assert rc(a15=float("inf")) == INV
    assert rc(a0=None) == INV and rc(a4=P + 2) == INV and rc(a8=None) == INV
    assert rc(a1=504) == INV and rc(a3=260) == INV and rc(a7=500) == INV
    assert rc(a9=0) == _lib.KVM_OK and rc(a10=0) == _lib.KVM_OK


def test_attention_tree_refuses_without_a_gpu():
    P, INV, UNS = 4096, _lib.KVM_ERR_INVALID_ARG, _lib.KVM_ERR_UNSUPPORTED
    lay = dict(page_stride=8192, layer_stride=8192, kv_stride=4096, token_stride=256,
               block_size=16, layer=0, width=256, num_pages=9)

    def rc(layout=None, **at):
        L = _lib.KvLayout(*{**lay, **(layout or {})}.values())
        args = [P, 1024, P, C.byref(L), P, 1024, P, P, P, 1, P, 9, P, 2, 10, 8, 5, 100, 0.0, P,
                1 << 40, None]
        for i, v in at.items():
            args[int(i[1:])] = v
        return _rc("attention_tree_paged", *args)
    assert rc(a3=None) == INV and rc(layout=dict(width=192)) == INV and rc(a15=7) == INV
    assert rc(layout=dict(block_size=8)) == UNS and rc(layout=dict(block_size=48)) == UNS
    assert rc(layout=dict(kv_stride=4096 + 8)) == INV
    assert rc(a13=1025) == UNS and rc(a16=0) == INV and rc(a16=1025, a9=64) == INV
    assert rc(a16=33) == INV and rc(a17=0) == INV and rc(a18=float("nan")) == INV
    assert rc(a0=None) == INV and rc(a4=P + 4) == INV and rc(a8=None) == INV and rc(a1=1000) == INV
    assert rc(a19=None, a17=2000) == INV and rc(a20=100, a17=2000) == INV
    assert rc(layout=dict(num_pages=1 << 30, page_stride=1 << 20)) == UNS
    assert rc(a13=0) == _lib.KVM_OK and rc(a14=0) == _lib.KVM_OK
    assert rc(a11=-1) == INV
    ws = _lib.lib().kvm_sm100_attention_tree_workspace
    assert ws(0, 8, 2, 5, 100) == 0 and ws(2, 7, 2, 5, 100) == 0 and ws(2, 8, 2, 0, 100) == 0
    assert ws(2, 8, 2, 5, (1 << 30) + 1) == 0
    assert rc(a17=(1 << 30) + 1) == INV
    assert ws(2, 8, 2, 5, 1024) == 0      # four short items are not cut
    assert ws(2, 8, 2, 5, 1025) == 9 * (2 * 256 * 130 * 4 + 32)    # 36 key tiles, four to a CTA
    assert ws(64, 64, 8, 16, 5000) == 148 * (2 * 256 * 130 * 4 + 32)


class _OnGpu(torch.Tensor):
    """A tensor without storage (meta) that says it is on GPU 0."""

    def get_device(self):
        return 0


def _huge(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta").as_subclass(_OnGpu)


def test_sizes_beyond_32_bits_are_refused(monkeypatch):
    """The C calls take 32-bit counts and bounds: what does not fit is refused
    instead of cut off to its low 32 bits (2^32 + 3 rows would run as 3)."""
    from kvm_b200.kvcache import PagedKVCache
    monkeypatch.setattr(ops, "_call_on", lambda *a: pytest.fail("the call went out"))
    monkeypatch.setattr("kvm_b200.kvcache._call_on", lambda *a: pytest.fail("the call went out"))
    n = 2 ** 32 + 3
    pos = _huge(n, dtype=torch.int32)
    with pytest.raises(ValueError, match="32 bits"):
        ops.rope(_huge(n, 4), pos, ops.rope_table(4), heads=1, head_dim=4, out=_huge(n, 4))
    few = _huge(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="32 bits"):
        ops.attention_packed(_huge(n, 64), _huge(n, 64), _huge(n, 64), few, heads_q=1, heads_kv=1,
                             head_dim=64, out=_huge(n, 64))
    with pytest.raises(ValueError, match="32 bits"):
        ops.attention_packed(_huge(5, 64), _huge(5, 64), _huge(5, 64), pos, heads_q=1, heads_kv=1,
                             head_dim=64, out=_huge(5, 64))
    cache = PagedKVCache(pages=4, layers=1, block_size=16, heads_kv=1, device="cpu")
    cache.pool = _huge(4)
    with pytest.raises(ValueError, match="32 bits"):
        cache.copy_pages(pos, pos)
    with pytest.raises(ValueError, match="32 bits"):
        cache.compact(pos, few, few[:1], few, few)
    one = _huge(1, dtype=torch.int32)
    for bounds in (dict(max_keys=n, max_q_rows=3), dict(max_keys=9, max_q_rows=n),
                   dict(max_keys=9 - 2 ** 32, max_q_rows=3)):
        with pytest.raises(ValueError, match="32 bits"):
            cache.tree_workspace(1, heads_q=1, **bounds)
        for ws in (None, _huge(99, dtype=torch.uint8)):
            with pytest.raises(ValueError, match="32 bits"):
                cache.tree_decode(0, _huge(3, 128), few, one, _huge(3, 1, dtype=torch.int32), few,
                                  few, heads_q=1, out=_huge(3, 128), workspace=ws, **bounds)


def test_what_is_no_tensor_is_refused():
    from kvm_b200.kvcache import PagedKVCache
    q = _huge(3, 128)
    one, few = _huge(1, dtype=torch.int32), _huge(2, dtype=torch.int32)
    cache = PagedKVCache(pages=4, layers=1, block_size=16, heads_kv=1, device="cpu")
    cache.pool = _huge(4)
    kw = dict(heads_q=1, max_q_rows=3, max_keys=9)
    with pytest.raises(TypeError):
        ops.rope(q, [0, 1, 2], ops.rope_table(4), heads=1, out=q)
    with pytest.raises(TypeError):
        cache.tree_decode(0, None, few, one, _huge(3, 1, dtype=torch.int32), few, few, **kw)
    with pytest.raises(TypeError):
        cache.tree_decode(0, q, few, one, [[1]], few, few, **kw)
    with pytest.raises(TypeError):
        cache.tree_decode(0, q, few, one, _huge(3, 1, dtype=torch.int32), few, few, out=q,
                          workspace=4096, **kw)

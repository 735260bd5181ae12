"""Paged KV cache and decode attention on the sm_100a kernels.

A pool holds K and V for `layers` layers in pages of `block_size` token
slots; a slot is one token's K (or V) row of width HKV * 128 bf16. KVMeta's
two layouts (src/ir/graph_config.h:20-39):
    page_first   [page][layer][kv][slot][width]
    layer_first  [layer][page][kv][slot][width]
Sequences own pages through a block table (AttnMetaImpl's kv block_table,
src/ir/dialect/kernel/values.h:83-117), flattened as `block_table` with
`bt_offsets` [S+1]. kvcache.write / kvcache.read / attn.decode are the ops of
src/ir/dialect/kernel/dialect.cpp:39,69-70.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import call
from .ops import _call_on, _check, _list, _mat, _rowmajor, _stream


def kv_strides(layout: str, pages: int, layers: int, block_size: int, width: int):
    """Element strides (page, layer, kv, token) of a pool in `layout`."""
    kv = block_size * width
    if layout == "page_first":
        layer = 2 * kv
        page = layers * layer
    elif layout == "layer_first":
        page = 2 * kv
        layer = pages * page
    else:
        raise ValueError(f"unknown KV layout {layout!r}")
    return page, layer, kv, width


def tree_mask(parents, device=None) -> torch.Tensor:
    """The masks of a drafted tree for `tree_decode`: parents[i] is the index of
    node i's parent (below i), or -1 for a child of the last cached token. Row
    i has the bits of i and of its ancestors: int32 [len(parents), words]."""
    rows = []
    for i, p in enumerate(int(p) for p in parents):
        if not -1 <= p < i:
            raise ValueError(f"parents[{i}] must be -1 or the index of an earlier node")
        rows.append((rows[p] if p >= 0 else 0) | (1 << i))
    words = max(1, (len(rows) + 31) // 32)
    data = b"".join(r.to_bytes(4 * words, "little") for r in rows)
    t = torch.frombuffer(bytearray(data), dtype=torch.int32) if rows else \
        torch.empty(0, dtype=torch.int32)
    return t.view(len(rows), words).to(device)


def _check_bounds(max_q_rows: int, max_keys: int) -> None:
    """What the C calls would cut off to its low 32 bits is refused."""
    if max_q_rows >> 31 not in (0, -1) or max_keys >> 31 not in (0, -1):
        raise ValueError("max_q_rows and max_keys must fit 32 bits")


class PagedKVCache:
    """A device pool of KV pages (bf16, zero-initialised)."""

    def __init__(self, *, pages: int, layers: int, block_size: int, heads_kv: int,
                 layout: str = "page_first", device=None):
        self.pages, self.layers, self.block_size = pages, layers, block_size
        self.heads_kv, self.width, self.layout = heads_kv, heads_kv * 128, layout
        self.strides = kv_strides(layout, pages, layers, block_size, self.width)
        self._layouts: dict = {}
        n = pages * layers * 2 * block_size * self.width
        self.pool = torch.zeros(n, dtype=torch.bfloat16, device=device)

    def layout_struct(self, layer: int) -> _lib.KvLayout:
        if not 0 <= layer < self.layers:
            raise ValueError("layer out of range")
        ps, ls, ks, ts = self.strides
        return _lib.KvLayout(ps, ls, ks, ts, self.block_size, layer, self.width, self.pages)

    def _layout(self, layer: int):
        """layout_struct(layer) by reference, made once per layer."""
        ref = self._layouts.get(layer)
        if ref is None:
            ref = self._layouts[layer] = C.byref(self.layout_struct(layer))
        return ref

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor,
              q_positions: torch.Tensor, block_table: torch.Tensor,
              bt_offsets: torch.Tensor) -> None:
        """kvcache.write: rows of k/v [rows, width] to their page slots."""
        _check(k, "k", torch.bfloat16, 2)
        _check(v, "v", torch.bfloat16, 2)
        for t, n in ((q_offsets, "q_offsets"), (q_positions, "q_positions"),
                     (block_table, "block_table"), (bt_offsets, "bt_offsets")):
            _check(t, n, torch.int32, 1)
        L = self.layout_struct(layer)
        call("kvm_sm100_kvcache_write", self.pool.data_ptr(), C.byref(L), k.data_ptr(),
             _rowmajor(k, "k"), v.data_ptr(), _rowmajor(v, "v"), q_offsets.data_ptr(),
             q_positions.data_ptr(), block_table.data_ptr(), bt_offsets.data_ptr(),
             q_offsets.numel() - 1, k.shape[0], _stream())

    def read(self, layer: int, kv_offsets: torch.Tensor, block_table: torch.Tensor,
             bt_offsets: torch.Tensor, rows: int):
        """kvcache.read: (k, v) [rows, width], each sequence's tokens in order."""
        L = self.layout_struct(layer)
        k = torch.empty((rows, self.width), dtype=torch.bfloat16, device=self.pool.device)
        v = torch.empty_like(k)
        call("kvm_sm100_kvcache_read", self.pool.data_ptr(), C.byref(L), k.data_ptr(),
             v.data_ptr(), kv_offsets.data_ptr(), block_table.data_ptr(),
             bt_offsets.data_ptr(), kv_offsets.numel() - 1, rows, _stream())
        return k, v

    def decode(self, layer: int, q: torch.Tensor, q_offsets: torch.Tensor,
               q_positions: torch.Tensor, block_table: torch.Tensor,
               bt_offsets: torch.Tensor, *, heads_q: int, max_q_rows: int, max_keys: int,
               scale: float = 0.0, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
        """attn.decode: causal attention of the new rows q [rows, HQ*128] over
        the cached positions up to their own."""
        _check(q, "q", torch.bfloat16, 2)
        L = self.layout_struct(layer)
        S = q_offsets.numel() - 1
        if out is None:
            out = torch.empty((q.shape[0], heads_q * 128), dtype=torch.bfloat16,
                              device=q.device)
        need = int(_lib.lib().kvm_sm100_attention_decode_workspace(
            S, heads_q, self.heads_kv, max_q_rows, max_keys))
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
        call("kvm_sm100_attention_decode_paged", q.data_ptr(), _rowmajor(q, "q"),
             self.pool.data_ptr(), C.byref(L), out.data_ptr(), _rowmajor(out, "out"),
             q_offsets.data_ptr(), q_positions.data_ptr(), block_table.data_ptr(),
             bt_offsets.data_ptr(), S, heads_q, max_q_rows, max_keys, float(scale),
             workspace.data_ptr(), workspace.numel(), _stream())
        return out

    def tree_workspace(self, sequences: int, *, heads_q: int, max_q_rows: int,
                       max_keys: int) -> int:
        """Bytes of workspace `tree_decode` needs for these bounds."""
        _check_bounds(max_q_rows, max_keys)
        return int(_lib.lib().kvm_sm100_attention_tree_workspace(
            sequences, heads_q, self.heads_kv, max_q_rows, max_keys))

    def tree_decode(self, layer: int, q: torch.Tensor, q_offsets: torch.Tensor,
                    q_positions: torch.Tensor, tree_mask: torch.Tensor,
                    block_table: torch.Tensor, bt_offsets: torch.Tensor, *, heads_q: int,
                    max_q_rows: int, max_keys: int, scale: float = 0.0,
                    out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of trees of drafted tokens q [rows, HQ*128], written with
        `write` at positions q_positions[s] + i: row i of sequence s attends to
        the q_positions[s] tokens before the tree and to the drafted tokens
        named by its tree_mask row (int32 [rows, words], bit j % 32 of word
        j / 32 for token j; see tree_mask()). A row that sees nothing is zero.
        Two calls that overlap in time need a workspace each."""
        dev = self.pool.get_device()
        S = _list(q_positions, "q_positions", dev)
        if _list(q_offsets, "q_offsets", dev) != S + 1 or \
                _list(bt_offsets, "bt_offsets", dev) != S + 1:
            raise ValueError("q_offsets and bt_offsets must have one more entry than "
                             "q_positions")
        table = _list(block_table, "block_table", dev)
        if not isinstance(q, torch.Tensor) or not isinstance(tree_mask, torch.Tensor):
            raise TypeError("q and tree_mask must be tensors")
        if q.dim() != 2 or tree_mask.dim() != 2:
            raise ValueError("q and tree_mask must be 2-D")
        _check_bounds(max_q_rows, max_keys)
        rows, words = q.shape[0], tree_mask.shape[1]
        ldq = _mat(q, "q", torch.bfloat16, rows, heads_q * 128, dev)
        if _mat(tree_mask, "tree_mask", torch.int32, rows, words, dev) != words:
            raise ValueError("tree_mask must be contiguous")
        if out is None:
            out = torch.zeros((rows, heads_q * 128), dtype=q.dtype, device=q.device)
        ldo = _mat(out, "out", torch.bfloat16, rows, heads_q * 128, dev)
        if workspace is None:
            need = self.tree_workspace(S, heads_q=heads_q, max_q_rows=max_q_rows,
                                       max_keys=max_keys)
            workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
        elif not isinstance(workspace, torch.Tensor):
            raise TypeError("workspace must be a tensor")
        elif workspace.get_device() != dev or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous on the pool's device")
        _call_on(dev, "kvm_sm100_attention_tree_paged", q.data_ptr(), ldq,
                 self.pool.data_ptr(), self._layout(layer), out.data_ptr(), ldo,
                 q_offsets.data_ptr(), q_positions.data_ptr(), tree_mask.data_ptr(), words,
                 block_table.data_ptr(), table, bt_offsets.data_ptr(), S, rows, heads_q, max_q_rows,
                 max_keys, scale, workspace.data_ptr(), workspace.nbytes)
        return out

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page dst[i] := page src[i] in every layer, K and V (device int32
        lists): a fork's own copy of the page it goes on writing, or pages
        moved within the pool. Sources may repeat; a pair that would race with
        another one (a destination named twice, or also a source) is skipped
        and raises at the next ops.device_status(), as does a bad page id."""
        dev = self.pool.get_device()
        n = _list(src, "src", dev)
        if _list(dst, "dst", dev) != n:
            raise ValueError("src and dst must have the same length")
        _call_on(dev, "kvm_sm100_kvcache_copy_pages", self.pool.data_ptr(),
                 self._layout(0), self.layers, src.data_ptr(), dst.data_ptr(), n)

    def compact(self, kept: torch.Tensor, kept_offsets: torch.Tensor,
                q_positions: torch.Tensor, block_table: torch.Tensor,
                bt_offsets: torch.Tensor) -> None:
        """Keep the tokens kept[kept_offsets[s]:kept_offsets[s+1]] (strictly
        increasing) of those written from position q_positions[s] on: token
        kept[i] moves to position q_positions[s] + i in every layer. A sequence
        with a bad list or page stays as it is and raises at the next
        ops.device_status()."""
        dev = self.pool.get_device()
        S, n = _list(q_positions, "q_positions", dev), _list(kept, "kept", dev)
        if _list(kept_offsets, "kept_offsets", dev) != S + 1 or \
                _list(bt_offsets, "bt_offsets", dev) != S + 1:
            raise ValueError("kept_offsets and bt_offsets must have one more entry than "
                             "q_positions")
        table = _list(block_table, "block_table", dev)
        _call_on(dev, "kvm_sm100_kvcache_compact", self.pool.data_ptr(),
                 self._layout(0), self.layers, kept.data_ptr(), n,
                 kept_offsets.data_ptr(), q_positions.data_ptr(), block_table.data_ptr(), table,
                 bt_offsets.data_ptr(), S)

"""Pages of a cache copied to other pages, and page tables rewritten, in one launch for all layers and pools (``csrc/kernels/page_moves.cu``): what a fork of a row or a
compaction of the pool does to the device.  The page numbers are the host's, whose ledger (``inference.pages``) gives them."""
from __future__ import annotations

import ctypes
from array import array
from typing import Optional, Sequence, Tuple

import torch

from . import library as L

Span = Tuple[int, int, Sequence[int]]          # (row, first column, pages): a piece of a row's table

_REFUSED = {-11: "a page number outside the pool", -12: "a page that is written twice", -13: "a page that is both read and written", -14: "an entry outside the page table",
            -16: "an entry of the page table that is written twice"}


class _Pool(ctypes.Structure):
    _fields_ = [("base", ctypes.c_void_p), ("layer_stride", ctypes.c_longlong), ("layers", ctypes.c_int), ("page_bytes", ctypes.c_int)]


def _refuse(rc: int) -> None:
    if rc in _REFUSED:
        raise ValueError(f"move_pages: {_REFUSED[rc]}")


def _check(src: Sequence[int], dst: Sequence[int], pages: int, table: Optional[torch.Tensor], tables: Sequence[Span]) -> None:
    if any(not 0 <= p < pages for ps in (src, dst, *(s[2] for s in tables)) for p in ps):
        _refuse(-11)
    if len(set(dst)) < len(dst):
        _refuse(-12)
    if not set(src).isdisjoint(dst):
        _refuse(-13)
    for row, first, ps in tables:
        if not (0 <= row < table.shape[0] and 0 <= first <= table.shape[1] - len(ps)):
            _refuse(-14)
    places = [row * table.shape[1] + first + i for row, first, ps in tables for i in range(len(ps))]
    if len(set(places)) < len(places):
        _refuse(-16)


def _no_gradient() -> None:
    raise NotImplementedError("move_pages has no gradient: pages of a cache are moved between steps of generation")


def _pool(t: torch.Tensor, pages: int, device) -> _Pool:
    if t.requires_grad and torch.is_grad_enabled():
        _no_gradient()
    if t.dim() < 2 or t.shape[1] != pages or t.device != device:
        raise ValueError(f"move_pages: pools of one device and [layers, {pages}, ...], got {tuple(t.shape)} on {t.device}")
    shape, strides, size, by = t.shape, t.stride(), 1, t.element_size()
    for i in range(len(shape) - 1, 0, -1):
        if shape[i] != 1 and strides[i] != size:
            raise ValueError("move_pages: the pages of a layer have to be one piece of memory, one behind another")
        size *= shape[i]
    size //= max(1, pages)
    if size * by >= 1 << 31:
        raise ValueError("move_pages: pages of 2 GB and more are not built")
    return _Pool(t.data_ptr(), strides[0] * by, shape[0], size * by)


def move_pages(pools: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int], table: Optional[torch.Tensor] = None, tables: Sequence[Span] = ()) -> None:
    """``pool[:, dst[i]] = pool[:, src[i]]`` in every pool ``[layers, pages, ...]`` (any types; all of as many pages), and ``table[row, first:first + len(pages)] = pages`` for
    every ``(row, first, pages)`` of ``tables`` (``table`` int32 ``[rows, columns]``).

    The numbers are lists of the host's.  A page may be read several times; it is refused to write one (or an entry) twice, to write one that is
    read, and to name one outside the pools, and then nothing has been written.  Everything happens on the current stream, in place; a captured call repeats these very moves."""
    if len(src) != len(dst):
        raise ValueError(f"move_pages: {len(src)} pages to {len(dst)}")
    if not pools:
        raise ValueError("move_pages: no pools")
    if tables and (table is None or table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous() or table.device != pools[0].device):
        raise ValueError("move_pages: the table is int32 [rows, columns] in one piece on the pools' device")
    if L.transformed(*pools):
        _no_gradient()
    pages = pools[0].shape[1] if pools[0].dim() > 1 else 0
    made = (_Pool * len(pools))(*(_pool(t, pages, pools[0].device) for t in pools))
    if not L.use_cuda(pools[0]):
        _check(src, dst, pages, table, tables)
        if len(src):
            s, d = (torch.tensor(list(x), dtype=torch.long, device=pools[0].device) for x in (src, dst))
            for t in pools:
                t = t.view(torch.uint8) if t.element_size() == 1 else t          # (8-bit floats have no indexing of their own)
                t.index_copy_(1, d, t.index_select(1, s))
        for row, first, ps in tables:
            if len(ps):
                table[row, first:first + len(ps)] = torch.tensor(list(ps), dtype=torch.int32, device=table.device)
        return
    if not L.device_is_current(pools[0]):
        with L.on_device_of(pools[0]):
            return move_pages(pools, src, dst, table, tables)
    # (the quickest way from lists to integers; they are held until the call is over)
    numbers = array("i")
    take = numbers.fromlist
    try:
        for ps in (src, dst):
            take(ps) if type(ps) is list else numbers.extend(ps)
        if tables:
            rows, firsts, named = zip(*tables)
            numbers.extend(rows)
            numbers.extend(firsts)
            numbers.extend(map(len, named))
            for ps in named:
                take(ps) if type(ps) is list else numbers.extend(ps)
    except OverflowError as e:
        raise ValueError(f"move_pages: {e}") from None
    n, spans_n = len(src), len(tables)
    start = numbers.buffer_info()[0]
    spans = start + 8 * n
    launches = ctypes.c_int(0)
    rc = L.load().dewb_move_pages(ctypes.addressof(made), len(made), pages, start, start + 4 * n, n, table.data_ptr() if tables else 0, table.shape[0] if tables else 0,
                                  table.shape[1] if tables else 0, spans, spans + 4 * spans_n, spans + 8 * spans_n, spans + 12 * spans_n, spans_n, ctypes.addressof(launches), L.stream())
    _refuse(rc)
    L.check(rc, "move_pages")
    L.count_launches(launches.value)
    torch.autograd.graph.increment_version((*pools, table) if tables else pools)         # (autograd is to know, as it does of what torch writes)

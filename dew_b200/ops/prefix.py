"""A decode step of rows that share prefixes (``csrc/kernels/shared_prefix_sm100.cu``; ``shared_prefix.cu`` for types and
widths that it does not take): the keys and values of a group's shared pages are read once for all of its rows, not once a row."""
from __future__ import annotations

import ctypes
import math
from typing import Dict, List, NamedTuple, Optional, Sequence, Tuple

import torch

from . import library as L


class Shared(NamedTuple):
    """Which rows of a batch share a prefix, as int32 tensors on the device (their values may change under a captured step): group ``g`` is rows ``order[first[g]:first[g + 1]]``,
    whose tables name the same pages for their first ``tokens[g]`` keys.  ``order`` holds every row once; a row that shares nothing is a group of its own."""
    order: torch.Tensor        # [rows]
    first: torch.Tensor        # [groups + 1]
    tokens: torch.Tensor       # [groups]


def _common(a: Sequence[int], b: Sequence[int]) -> int:
    """Pages that both begin with (halving: comparing pieces of lists is quick)."""
    lo, hi = 0, min(len(a), len(b))
    while lo < hi:
        mid = (lo + hi + 1) // 2
        if a[lo:mid] == b[lo:mid]:
            lo = mid
        else:
            hi = mid - 1
    return lo


def _families(rows: Sequence[int], tables: Sequence[Optional[Sequence[int]]], least: int) -> List[Tuple[List[int], int]]:
    """``rows``, which begin with the same page, in groups of (rows, pages that all of them begin with and that are read once for them): those that save the most pages,
    (rows of a group - 1) x its pages, over all groups; no group of fewer than ``least`` pages.

    The tables form a tree that branches where they part.  A row counts the pages of the group that it is in, and a group costs its pages once.  So what is saved below a node, if
    the group around it has d pages, is the larger of: the sum over its branches with that d (a row: d), or the sum with the node's own depth, less that depth."""
    tables = {r: list(tables[r]) for r in rows}
    at = sorted(rows, key=tables.get)
    # nodes [depth, branches], a branch a row's number or a node: those open from the root on, in the order of the tables
    open_, last = [], at[0]
    for before, row in zip(at, at[1:]):
        depth = _common(tables[before], tables[row])
        while open_ and open_[-1][0] > depth:
            open_[-1][1].append(last)
            last = open_.pop()
        if open_ and open_[-1][0] == depth:
            open_[-1][1].append(last)
        else:
            open_.append([depth, [last]])
        last = row
    while open_:
        open_[-1][1].append(last)
        last = open_.pop()
    # every node with the depths of the groups that may be around it (0: none), its own last where it may be one
    nodes, todo = [], [(last, (0,))]
    while todo:
        node, around = todo.pop()
        inside = around + (node[0],) if node[0] >= max(1, least) else around
        nodes.append((node, around, inside))
        todo += [(branch, inside) for branch in node[1] if type(branch) is list]
    sums, saved = {}, {}
    for node, around, inside in reversed(nodes):
        lists, n = [saved[id(x)] for x in node[1] if type(x) is list], sum(type(x) is int for x in node[1])
        total = [n * d + sum(x[i] for x in lists) for i, d in enumerate(inside)]
        sums[id(node)] = total
        saved[id(node)] = [max(x, total[-1] - inside[-1]) for x in total[:len(around)]] if len(inside) > len(around) else total
    groups, alone, todo = [], [], [(last, 0, None)]
    place = {id(node): (around, inside) for node, around, inside in nodes}
    while todo:
        branch, i, group = todo.pop()
        if type(branch) is int:
            alone.append(([branch], 0)) if group is None else group.append(branch)
            continue
        (around, inside), total = place[id(branch)], sums[id(branch)]
        if len(inside) > len(around) and total[-1] - inside[-1] > total[i]:
            i, group = len(around), []
            groups.append((group, branch[0]))
        todo += [(x, i, group) for x in branch[1]]
    return [(sorted(group), pages) for group, pages in groups] + alone


def group_rows(tables: Sequence[Optional[Sequence[int]]], page_size: int, least: int = 1) -> Tuple[List[int], List[int], List[int]]:
    """``order, first, tokens`` of ``Shared`` for rows of these pages (None: an empty row), as lists of as many groups as rows: rows that begin with the same pages, in the groups
    that leave the fewest tokens to read.  Fewer than ``least`` tokens are not worth a group."""
    starts: Dict[object, List[int]] = {}
    for r, pages in enumerate(tables):
        starts.setdefault(pages[0] if pages else ("alone", r), []).append(r)
    groups: List[Tuple[List[int], int]] = []
    for rows in starts.values():
        groups += [(rows, 0)] if len(rows) == 1 else _families(rows, tables, -(-least // page_size))
    order, first, tokens = [], [0], []
    for rows, pages in sorted(groups):
        order += rows
        first.append(len(order))
        tokens.append(pages * page_size)
    empty = len(order) - len(tokens)
    return order, first + [len(order)] * empty, tokens + [0] * empty


def shared_decode_reference(q, k, v, table, lengths, scale, window=None, softcap=0.0, sinks=None, k_scale=None, v_scale=None) -> torch.Tensor:
    """Every row by its own table, in fp32: what sharing does not change."""
    R, H, D = q.shape
    page, G = k.shape[1:3]
    n = max(int(lengths.max()), 1) if R else 1
    key = torch.arange(n, device=q.device)
    slots = (table.long()[:, key // page] * page + key % page).clamp(0, k.shape[0] * page - 1)
    seen = key < lengths[:, None]
    if window:
        seen = seen & (key >= lengths[:, None] - window)

    def rows(t, by):
        t = t.reshape(-1, G, D)[slots].float()
        t = t if by is None else t * by.reshape(-1, G)[slots][..., None]
        return torch.where(seen[..., None, None], t, torch.zeros_like(t))           # (what a row does not see may be anything)
    kr, vr = rows(k, k_scale), rows(v, v_scale)
    s = torch.einsum("rghd,rngd->rghn", q.float().reshape(R, G, H // G, D), kr) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    if sinks is not None:
        s = torch.cat([s, sinks.float().view(1, G, H // G, 1).expand(R, -1, -1, 1)], -1)
    p = torch.softmax(s, -1)
    p = torch.where((s == -math.inf).all(-1, keepdim=True), torch.zeros_like(p), p)          # (nothing to see; a score that is no number shows)
    p = p if sinks is None else p[..., :-1]
    return torch.einsum("rghn,rngd->rghd", p, vr).reshape(R, H, D).to(q.dtype)


LEAST_TILES = 1          # 128-key tiles that an engine of the tensor cores' kernel takes at least (with 2: 4 rows behind 448 shared tokens 17.7 us instead of 15, 8 behind 1024 23.4 instead of 22)
MOST_ROWS = 448          # rows, and groups, that its lists hold
_ENGINES: Dict[Tuple[int, int], int] = {}


def _engines(lib, device, D: int) -> int:
    key = (device.index or 0, D)
    if key not in _ENGINES:
        _ENGINES[key] = lib.dewb_shared_mma_engines(ctypes.c_int(D))
    return _ENGINES[key]


def on_tensor_cores(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, columns: int, groups: int) -> bool:
    """Whether the call is one of ``shared_prefix_sm100.cu``'s: bf16 throughout, heads of 64, 128 or 256, pages of whole sixteens of tokens, 16-byte rows, tables whose tiles
    can be counted in 32 bits."""
    (R, H, D), (pages, page, G, _) = q.shape, k.shape
    return (q.dtype is torch.bfloat16 and k.dtype is torch.bfloat16 and _counted(R, H, D, pages, page, G, columns, groups)
            and (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15 == 0 and (R == 1 or q.stride(0) % 8 == 0))


def _counted(R: int, H: int, D: int, pages: int, page: int, G: int, columns: int, groups: int) -> bool:
    return (D in (64, 128, 256) and page % 16 == 0 and R <= MOST_ROWS and groups <= MOST_ROWS and pages * page < 0x7fffff00
            and (2 * R * -(-H // G // 32) + groups) * G * (columns * page // 64 + 8) < 1 << 30)


def _splits(most: int, lists: int) -> int:
    """Parts of the keys in the kernel for other types: of 128 keys as long as there are no more than 2048 CTAs (rows times key heads times parts), then of 512.
    (Parts of 512, 128, 64 keys: 24 rows of 500, two key heads, 48, 30, 35 us; four rows of 400 56, 28, 26.)"""
    return max(1, min(32, -(-most // 128), max(-(-most // 512), 2048 // lists)))


_POOLS = {torch.int8: 1, torch.float8_e4m3fn: 2}


def _device(t: torch.Tensor) -> torch.device:
    return t.device


def _check(q, k, v, table, lengths, shared: Shared, window, softcap, sinks, k_scale, v_scale) -> None:
    order, first, tokens = shared
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 3 or len(k_shape) != 4 or k_shape != v.shape or q_shape[2] != k_shape[3] or k_shape[2] == 0 or q_shape[1] % k_shape[2]:
        raise ValueError(f"shared_decode: queries [rows, heads, dim] and pools [pages, page, kv heads, dim], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    own, pool = q.dtype, k.dtype
    if (own is not torch.bfloat16 and own is not torch.float32) or pool != v.dtype or (pool is not own and pool not in _POOLS):
        raise TypeError(f"shared_decode: bf16 or fp32 queries and pools of their type, int8 or float8_e4m3fn, got {q.dtype}, {k.dtype}, {v.dtype}")
    R, H, D = q_shape
    scaled = pool is not own
    if (k_scale is not None) != scaled or (v_scale is not None) != scaled:
        raise ValueError("shared_decode: scales belong to int8 and float8 pools")
    if not 0 < D <= 256:
        raise ValueError(f"shared_decode: heads of up to 256, got {D}")
    groups = len(tokens) if tokens.dim() == 1 else -1
    if groups < (R > 0) or order.shape != (R,) or first.shape != (groups + 1,):
        raise ValueError(f"shared_decode: order [rows], first [groups + 1] and tokens [groups] for {R} rows, got {[tuple(t.shape) for t in shared]}")
    if table.dim() != 2 or len(table) != R or lengths.shape != (R,):
        raise ValueError(f"shared_decode: a table [rows, columns] and lengths [rows] for {R} rows, got {tuple(table.shape)}, {tuple(lengths.shape)}")
    if R and (k_shape[0] == 0 or k_shape[1] == 0 or table.shape[1] == 0):
        raise ValueError(f"shared_decode: pools and tables of a page or more, got {tuple(k_shape)}, {tuple(table.shape)}")
    where = torch.Tensor.get_device if q.is_cuda else _device          # (the quicker question)
    device = where(q)
    apart = where(k) != device or where(v) != device
    for t in (table, lengths, order, first, tokens):
        if t.dtype is not torch.int32 or not t.is_contiguous():
            raise TypeError("shared_decode: table, lengths, order, first and tokens are int32 in one piece")
        apart = apart or where(t) != device
    if scaled:
        for t in (k_scale, v_scale):
            if t.shape != k_shape[:3] or t.dtype is not torch.float32 or not t.is_contiguous():
                raise ValueError("shared_decode: fp32 scales [pages, page, kv heads]")
            apart = apart or where(t) != device
    if sinks is not None:
        if sinks.shape != (H,) or sinks.dtype is not torch.float32 or not sinks.is_contiguous():
            raise ValueError("shared_decode: fp32 sinks, one a head")
        apart = apart or where(sinks) != device
    if (window is not None and window < 1) or softcap < 0:
        raise ValueError(f"shared_decode: a window of 1 or more and a cap of 0 or more, got {window}, {softcap}")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("shared_decode: pools in one piece")
    if apart:
        raise ValueError("shared_decode: tensors of one device")
    if L.transformed(q, k, v, sinks, k_scale, v_scale) or (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                                                                        or (sinks is not None and sinks.requires_grad))):
        raise NotImplementedError("shared_decode has no gradient: it is a step of generation")


def shared_decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, shared: Shared, scale: float, *,
                  window: Optional[int] = None, softcap: float = 0.0, sinks: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None,
                  v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query token of every row, ``q [rows, heads, dim]`` (a view with other rows between will do), against the first ``lengths[r]`` keys of its pages -> ``[rows, heads,
    dim]``; rows of length 0 give zeros.  Pools ``[pages, page, kv heads, dim]``, ``table [rows, columns]``.  A ``window`` leaves a row its last keys, ``softcap`` and ``sinks`` are
    those of ``ops.attention``.  ``shared`` says what is read once for several rows; it does not change what is computed.

    Page numbers, lengths and rows that lie outside their tensors, rows that ``order`` names twice, places that no group holds and groups that begin behind their end are
    reported by the status word (``library.check_status``) and read nothing."""
    _check(q, k, v, table, lengths, shared, window, softcap, sinks, k_scale, v_scale)
    R, H, D = q.shape
    if R == 0:
        return q.new_empty(q.shape)
    if not L.use_cuda(q):
        return shared_decode_reference(q, k, v, table, lengths, scale, window, softcap, sinks, k_scale, v_scale)
    if not L.device_is_current(q):
        with L.on_device_of(q):
            return shared_decode(q, k, v, table, lengths, shared, scale, window=window, softcap=softcap, sinks=sinks, k_scale=k_scale, v_scale=v_scale)
    strides = q.stride()
    if strides[2] != 1 or (H > 1 and strides[1] != D):
        q = q.contiguous()
        strides = q.stride()
    out = torch.empty(R, H, D, dtype=q.dtype, device=q.device)
    pages, page, G, _ = k.shape
    seen = window if window is not None and window < 1 << 30 else 0         # (a row's keys are counted in 30 bits: a wider window leaves it all)
    columns, groups, fp32, lib = table.shape[1], len(shared.tokens), torch.float32, L.load()
    at_q, at_k, at_v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    numbers = (table.data_ptr(), lengths.data_ptr(), shared.order.data_ptr(), shared.first.data_ptr(), shared.tokens.data_ptr(), L.at(sinks))
    err, stream = L.status(q.device).data_ptr(), L.stream()
    if (q.dtype is torch.bfloat16 and k.dtype is torch.bfloat16 and (at_q | at_k | at_v) & 15 == 0 and (R == 1 or strides[0] % 8 == 0)
            and _counted(R, H, D, pages, page, G, columns, groups)):
        engines = _engines(lib, q.device, D)
        rows = 2 * R * H + 320 * engines
        # one piece of scratch a call: sums, maxima and sums of weights, the plan
        scratch = torch.empty(rows * (D + 2) + 8 * R, dtype=fp32, device=q.device)
        at = scratch.data_ptr()
        L.check(lib.dewb_shared_decode_mma(at_q, strides[0] if R > 1 else H * D, at_k, at_v, *numbers, at, at + 4 * rows * D, at + 4 * rows * (D + 2),
                                           out.data_ptr(), R, H, G, D, page, columns, pages, groups, seen, LEAST_TILES, engines, scale, softcap, err, stream), "shared_decode_mma")
        L.count_launches(2)
        return out
    splits = _splits(columns * page, R * G)
    parts = torch.empty(2 * splits * R * H * (D + 2), dtype=fp32, device=q.device)
    at = parts.data_ptr()
    one = 2 * splits * R * H * 4
    L.check(lib.dewb_shared_decode(at_q, strides[0], at_k, at_v, L.at(k_scale), L.at(v_scale), *numbers, at, at + one, at + 2 * one, out.data_ptr(),
                                   R, H, G, D, page, columns, pages, groups, splits, seen, scale, softcap, int(q.dtype is fp32), _POOLS.get(k.dtype, 0), err, stream),
            "shared_decode")
    L.count_launches(2)
    return out

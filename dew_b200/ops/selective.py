"""The selective state space scan (``csrc/kernels/selective_scan.cu``, ``selective_grad.cu``, ``selective_heads.cu``; the equations stand in ``csrc/common/selective.cuh``): a rate per channel and state
(Mamba-1) over whole rows with every gradient, and over a call's ``Rows`` with the states that a store keeps; and the same with a decay per head (Mamba-2) for such a call.  The plain
forms go token by token (``selective_tokens_reference``, ``ssd_tokens_reference``) or in chunks (``ops.scan.selective_scan_chunked``).
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from . import library as L
from .token_mix import Rows, kernel_ok, whole

MOST_STATES, MOST_HEAD_STATES = 128, 256
OUTSIDE = 6              # the status word's code of a row outside the store
EVERY = 16               # tokens between two states that the forward keeps for the backward

# ``dewb_selective_args`` of ``csrc/common/selective.cuh`` and ``dewb_selective_grad_args`` of ``csrc/kernels/selective_grad.cu``, packed in one call (a ctypes structure of 42 fields takes five
# microseconds to fill, a step's call of one token all in all 20)
_ARGS, _GRAD = struct.Struct("@5P10q12P14iP"), struct.Struct("@P2q12P")


def _padded(C: int, N: int, groups: int = 1, heads: int = 0):
    """Channels (of all groups) and states as the workspaces pad them, and the channels that a warp takes with four states a lane."""
    lanes = 4 if N <= 16 else 8 if N <= 32 else 16 if N <= 64 else 32
    block = 256 if heads else 128
    return -(-(C // groups) // block) * block * groups, lanes * 4 if N <= 128 else 256, block // lanes


def _split(R: int, T: int, C: int, N: int, groups: int, heads: int = 0, backward: bool = False, fp32: bool = False):
    """Tokens of a piece of a row (the pieces run side by side), and states of a lane (of up to 16).  Pieces cost a pass of their own over the tokens (about half of the other) and are put
    together one after another, so there are no more than fill the GPU, or than the square root of half the tokens; fewer states a lane fill it without them, at the price of more sums over lanes.

    What it was measured on: rows of 2048 tokens of 16 states in bf16, gated, in us, by the warps that the channels of all rows make.  Forwards, whole with 1, 2, 4 states a lane, and in
    pieces (their number, states a lane):

        64     259  338  538   (16, 2) 80         448    426  398  538   (5, 4) 376, (4, 2) 400     1024   841  607  663   (2, 4) 732
        128    254  340  538   (9, 2) 138         512    427  396  539   (8, 4) 404                 1280  1113  868  829   (5, 4) 899
        256    294  342  537   (6, 2) 261         640    698  490  657   (8, 4) 495                 1536  1174  947  828   (3, 4) 1050
        384    350  398  545   (4, 2) 352         768    711  492  664   (3, 4) 551

    so pieces of two states a lane up to 448 warps (within a tenth of the best there, but for up to a quarter below 256 in other numbers of pieces), whole rows from there on, with four states a
    lane from 1536 on.  Backwards, whole with 2, 4 states a lane, and in pieces of 4:

        64    1099 1399   (16) 202     384   1367 1400   (11) 826     896   2566 1823   (5) 1763
        256   1115 1398   (16) 577     512   1370 1418   (8) 1059     1024  2609 1832   (4) 1971
        128   1089 1401   (9) 334      768   1668 1830   (6) 1500     1280  2905 3030   (6) 2396

    so pieces up to 1024 warps; behind 1184, as many as two blocks an SM are, whole rows make a second wave, and pieces would be faster again for some way.  512 tokens: forwards 512 warps whole
    106, in pieces 118; 384 whole with one state 93, in pieces 101; backwards 1024 whole 507, in pieces 547; 512 whole 390, in 5 and 8 pieces 318, 323.  One row of 512 of 1024 channels
    in 16 pieces of 2, 11 of 1: 19, 20; one of 2048 of 2048 channels backwards in 16 pieces of 4, 22 of 2: 154, 177."""
    warps = max(1, R * groups * -(-(C // groups) // _padded(C, N, groups, heads)[2]))
    most = max(1, min(-(-T // EVERY), int((T / 2) ** 0.5)))
    narrow = N <= 16 and not heads
    if warps >= 1024 or (narrow and not backward and warps >= 448):
        pieces = 1
    elif narrow:
        # all blocks on the GPU at once (two an SM backwards, four with two states a lane forwards) where that leaves eight pieces or more
        pieces = 1184 // warps if backward else 592 // -(-warps // 2)
        pieces = min(most, pieces if pieces >= 8 else -(-(4096 if backward else 1536) // warps))
    else:
        pieces = min(most, -(-4096 // warps))
    each = 4
    if narrow:
        each = (4 if warps * pieces >= 1024 and not fp32 else 2) if backward else 4 if warps >= 1536 else 2 if warps * pieces >= 384 else 1
    return -(-(-(-T // pieces)) // EVERY) * EVERY, each


def _rows_each(R: int, C: int) -> int:
    """Rows of a step whose rates a block of 128 channels reads once: so many that all blocks are on the GPU together, five an SM (128 rows of 8192 channels, 1, 4, 8, 12, 16 rows: 37, 28,
    30, 27, 30 us; 32 rows of 4096, 1, 2, 4 rows: 8.0, 6.8, 8.3; 256 of 2048, 2, 6, 8 rows: 18, 16, 17)."""
    return max(1, min(32, -(-R * -(-C // 128) // 740)))


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """``t [R, T, n]`` with its last axis in one piece."""
    return t if t is None or t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _strides(t: torch.Tensor):
    """Row and token strides (0 where there is one of them)."""
    shape, (row, token, _) = t.shape, t.stride()
    return row if shape[0] > 1 else 0, token if shape[1] > 1 else 0


class _Call(NamedTuple):
    """A launch's arguments, how it cuts rows and deals states, and the workspace that has to live until it is issued."""
    packed: bytes
    segments: int
    each: int
    work: Optional[torch.Tensor]


def _args(x, dt, z, b, c, a, dt_bias, d, initial, last, y, checkpoints, rows: Optional[Rows], N: int, groups: int, heads: int, softplus: bool, log_a: bool, stored: int = 0,
          token: bool = False, backward: bool = False, whole: bool = False) -> _Call:
    R, T, C = x.shape
    at, starts, sums, segments, work = L.at, 0, 0, 1, None
    channels, states, _ = _padded(C, N, groups, heads)
    if token:
        segment, each = EVERY, _rows_each(R, C)
        strides = [0] * 10
        if R > 1:
            strides[::2] = x.stride(0), dt.stride(0), 0 if z is None else z.stride(0), b.stride(0), c.stride(0)
    else:
        segment, each = (-(-T // EVERY) * EVERY, 4) if whole else _split(R, T, C, N, groups, heads, backward, x.dtype is torch.float32)
        segments = -(-T // segment)
        if segments > 1:
            work = torch.empty(R * segments * channels * (states + 1), dtype=torch.float32, device=x.device)
            starts = work.data_ptr()
            sums = starts + 4 * R * segments * channels * states
        strides = *_strides(x), *_strides(dt), *((0, 0) if z is None else _strides(z)), *_strides(b), *_strides(c)
    positions, lengths, ids = (0, 0, 0) if rows is None else (rows.positions.data_ptr(), rows.lengths.data_ptr(), at(rows.row_ids))
    packed = _ARGS.pack(x.data_ptr(), dt.data_ptr(), at(z), b.data_ptr(), c.data_ptr(), *strides, a.data_ptr(), at(dt_bias), at(d), at(initial), at(last), at(y), at(checkpoints), starts, sums,
                        positions, lengths, ids, R, T, C, N, groups, heads, segments, segment, channels // groups, each, softplus, log_a, dt.dtype is torch.float32, stored,
                        L.status(x.device).data_ptr())
    return _Call(packed, segments, each, work)


def _launch(call: _Call, heads: bool, fp32: bool, token: bool, stream: int) -> None:
    lib = L.load()
    if heads:
        L.check(lib.dewb_head_scan(call.packed, fp32, token, stream), "head_scan")
    elif token:
        L.check(lib.dewb_selective_token(call.packed, fp32, stream), "selective_token")
    else:
        L.check(lib.dewb_selective_scan(call.packed, fp32, stream), "selective_scan")
    L.count_launches(1 if call.segments == 1 else 2)


# ---------------------------------------------------------------------------------------------------------------
# whole rows, with gradients


def _forward(x, dt, a, b, c, d, z, initial, softplus: bool, keep: bool):
    if not L.device_is_current(x):
        with L.on_device_of(x):
            return _forward(x, dt, a, b, c, d, z, initial, softplus, keep)
    R, T, C = x.shape
    N = a.shape[1]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    last = torch.empty(R, C, N, dtype=torch.float32, device=x.device)
    channels, states, _ = _padded(C, N)
    kept = torch.empty(R, -(-T // EVERY), channels, states, dtype=torch.float32, device=x.device) if keep else None
    _launch(_args(x, dt, z, b, c, a, None, d, initial, last, y, kept, None, N, 1, 0, softplus, False), False, x.dtype is torch.float32, False, L.stream())
    return y, last, kept


def _backward(x, dt, a, b, c, d, z, initial, kept, softplus: bool, dy, dlast):
    """-> dx, ddt, da, db, dc, dd, dz, dinitial."""
    if not L.device_is_current(x):
        with L.on_device_of(x):
            return _backward(x, dt, a, b, c, d, z, initial, kept, softplus, dy, dlast)
    L.ensure_device(x)                                       # (a thread of autograd's may come here first)
    R, T, C = x.shape
    N, dev = a.shape[1], x.device
    channels, states, wide = _padded(C, N)
    like = lambda t: None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)
    dx, ddt, dz, db, dc, da, dd, dinitial = like(x), like(dt), like(z), like(b), like(c), like(a), like(d), like(initial)
    call = _args(x, dt, z, b, c, a, None, d, initial, None, None, kept, None, N, 1, 0, softplus, False, backward=True)
    # one piece of scratch: parts of dB and dC per channel block, of dA and of dD per row and piece
    of_bc, of_a = -(-C // (wide * call.each)) * R * T * 2 * states, R * call.segments * channels * states
    scratch = torch.empty(of_bc + of_a + R * call.segments * channels, dtype=torch.float32, device=dev)
    parts = scratch.data_ptr()
    grad = _GRAD.pack(dy.data_ptr(), *_strides(dy), *(L.at(t) for t in (dlast, dx, ddt, dz, db, dc, da, dd, dinitial)), parts, parts + 4 * of_bc, parts + 4 * (of_bc + of_a))
    L.check(L.load().dewb_selective_grad(call.packed + grad, x.dtype is torch.float32, L.stream()), "selective_grad")
    L.count_launches(2 if call.segments == 1 else 3)
    return dx, ddt, da, db, dc, dd, dz, dinitial


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, a, b, c, d, z, initial, softplus):
        ctx.set_materialize_grads(False)
        ctx.softplus = softplus
        y, last, kept = _forward(x, dt, a, b, c, d, z, initial, softplus, True)
        ctx.save_for_backward(x, dt, a, b, c, d, z, initial, kept)
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        *ins, kept = ctx.saved_tensors
        x = ins[0]
        if torch.is_grad_enabled():                          # (create_graph: the kernel's results would have no history)
            return (*_plain_gradients(ins, ctx.softplus, dy, dlast, ctx.needs_input_grad), None)
        dy = torch.zeros_like(x) if dy is None else _dense(dy.to(x.dtype))
        dx, ddt, da, db, dc, dd, dz, dinitial = _backward(*ins, kept, ctx.softplus, dy, None if dlast is None else dlast.float().contiguous())
        return dx, ddt, da, db, dc, dd, dz, dinitial, None


def _plain_gradients(ins, softplus, dy, dlast, needed):
    from .scan import selective_scan_chunked
    out = selective_scan_chunked(*ins, softplus=softplus)
    # (the last state depends neither on C, D nor the gate, and needs no gradient where nothing else does)
    pairs = [(o, g) for o, g in zip(out, (dy, dlast)) if g is not None and o.requires_grad]
    if not pairs:
        return [None] * len(ins)
    at = [i for i, t in enumerate(ins) if t is not None and needed[i]]
    grads = torch.autograd.grad([o for o, _ in pairs], [ins[i] for i in at], [g for _, g in pairs], create_graph=True, allow_unused=True)
    return [grads[at.index(i)] if i in at else None for i in range(len(ins))]


def kernel_available(x: torch.Tensor, *others: Optional[torch.Tensor]) -> bool:
    """Whether the scan of whole rows runs on the kernels: a GPU's tensors of up to 32 bits, nothing that has to be seen through."""
    given = [t for t in (x, *others) if t is not None]
    return (x.is_cuda and x.dim() == 3 and all(t.dtype in (torch.bfloat16, torch.float16, torch.float32) for t in given) and not L.transformed(*given)
            and L.use_cuda(x))


def fits(x, dt, A, Bm, Cm, D=None, z=None, initial_state=None) -> bool:
    """Whether everything expands to its size beside ``x [R, T, C]``."""
    R, T, C = x.shape
    tokens, narrow, rates = (R, T, C), (R, T, A.shape[-1]), (C, A.shape[-1])
    return all(t is None or t.shape == size or (t.dim() <= len(size) and all(n == m or n == 1 for n, m in zip(reversed(t.shape), reversed(size))))
               for t, size in ((dt, tokens), (A, rates), (Bm, narrow), (Cm, narrow), (D, (C,)), (z, tokens), (initial_state, (R, *rates))))


def selective_scan(x, dt, A, Bm, Cm, D=None, z=None, initial_state=None, softplus: bool = False):
    """``ops.scan.selective_scan`` on the kernels."""
    R, T, C = x.shape
    N = A.shape[-1]
    given = [t for t in (dt, A, Bm, Cm, D, z, initial_state) if t is not None]
    if any(t.dim() and t.device != x.device for t in given):
        raise ValueError("selective_scan: tensors of one device")
    out_type = x.dtype
    # one type for what is per token: where they differ (or are fp16) in fp32, which holds every value of each
    one = out_type is not torch.float16 and all(t is None or t.dtype is out_type for t in (Bm, Cm, z)) and dt.dtype in (out_type, torch.float32)

    def fit(t, *size):
        if t is None:
            return None
        t = (t if one else t.float()).to(x.device)                                       # (a number may lie elsewhere)
        return _dense(t if t.shape == size else t.expand(size))

    def fp32(t, *size):
        if t is None or (t.dtype is torch.float32 and t.shape == size and t.is_contiguous()):
            return t
        return t.to(x.device).float().expand(size).contiguous()
    ins = (fit(x, R, T, C), fit(dt, R, T, C), fp32(A, C, N), fit(Bm, R, T, N), fit(Cm, R, T, N), fp32(D, C), fit(z, R, T, C), fp32(initial_state, R, C, N))
    y, last = _forward(*ins, softplus, False)[:2] if L.unrecorded(*ins) else _SelectiveScan.apply(*ins, softplus)
    return y.to(out_type), last


# ---------------------------------------------------------------------------------------------------------------
# a call's rows, with the states of a store


_TYPES = (torch.bfloat16, torch.float32, torch.float16, torch.float64)         # (the last two in the plain form)


def _check(what: str, x, dt, b, c, z, weights, state, rows: Optional[Rows], state_shape, wide, steps, narrow) -> None:
    if x.dim() != 3:
        raise ValueError(f"{what}: x [rows, tokens, channels], got {tuple(x.shape)}")
    R, S, _ = shape = x.shape
    own, where = x.dtype, torch.Tensor.get_device if x.is_cuda else _device          # (the quicker question)
    if own not in _TYPES or b.dtype is not own or c.dtype is not own or (z is not None and z.dtype is not own) or (dt.dtype is not own and dt.dtype is not torch.float32):
        raise TypeError(f"{what}: floating-point tokens of one type and steps of that type or fp32, got {[t.dtype for t in (x, dt, b, c, z) if t is not None]}")
    if dt.shape != (R, S, steps) or b.shape != (R, S, narrow) or c.shape != b.shape or (z is not None and z.shape != shape):
        raise ValueError(f"{what}: steps [.., {steps}], B and C [.., {narrow}] and z [.., {wide}] beside x {tuple(shape)}, got {[tuple(t.shape) for t in (dt, b, c, z) if t is not None]}")
    device = where(x)
    apart = where(dt) != device or where(b) != device or where(c) != device or (z is not None and where(z) != device)
    for t in weights:
        apart = apart or (t is not None and where(t) != device)
    if rows is not None:
        positions, lengths, ids = rows
        if positions.shape != (R, S) or lengths.shape != (R,) or (ids is not None and ids.shape != (R,)):
            raise ValueError(f"{what}: positions [rows, tokens], lengths and row ids [rows] of {R} rows of {S} tokens")
        for t in rows:
            if t is not None:
                if t.dtype is not torch.int32 or not t.is_contiguous():
                    raise TypeError(f"{what}: positions, lengths and row ids are int32 in one piece")
                apart = apart or where(t) != device
    if state is not None:
        if state.shape[1:] != state_shape or state.dtype is not torch.float32 or not state.is_contiguous():
            raise ValueError(f"{what}: an fp32 state [store rows, {', '.join(map(str, state_shape))}] in one piece, got {tuple(state.shape)}, {state.dtype}")
        if (rows is None or rows.row_ids is None) and state.shape[0] < R:
            raise ValueError(f"{what}: {R} rows against a store of {state.shape[0]}")
        apart = apart or where(state) != device
    if apart:
        raise ValueError(f"{what}: tensors of one device")


def _device(t: torch.Tensor) -> torch.device:
    return t.device


def _fp32(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or (t.dtype is torch.float32 and t.is_contiguous()) else t.detach().float().contiguous()


def _moved(state: Optional[torch.Tensor]) -> None:
    """A state went on in place: autograd is to know, as it does of what torch writes (inference tensors have no version)."""
    if state is not None and not state.is_inference():
        torch.autograd.graph.increment_version(state)


def _tokens(x, dt, z, b, c, a, dt_bias, d, rows: Rows, state, N: int, groups: int, heads: int) -> torch.Tensor:
    if not L.device_is_current(x):
        with L.on_device_of(x):
            return _tokens(x, dt, z, b, c, a, dt_bias, d, rows, state, N, groups, heads)
    x, dt, z, b, c = _dense(x), _dense(dt), _dense(z), _dense(b), _dense(c)
    a, dt_bias, d = _fp32(a), _fp32(dt_bias), _fp32(d)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    token = x.shape[1] == 1 and state is not None
    call = _args(x, dt, z, b, c, a, dt_bias, d, state, state, y, None, rows, N, groups, heads, True, True, 0 if state is None else state.shape[0], token)
    _launch(call, heads > 0, x.dtype is torch.float32, token, L.stream())
    _moved(state)
    return y


# From here on a call of heads of 64 over 128 states in bf16 goes through the tensor cores' scan in chunks.  64 heads, in us, chunks and token by token: one row of 16 tokens 32, 12; of 32 37, 23;
# of 64 25, 33; of 2048 94, 395; eight of 32 40, 42; of 512 151, 485; eight of 37 to 512 149, 301; 32 of 32 98, 139; 24 heads, one row of 33 30, 25, of 64 28, 29, of 512 40, 100.  Chunks
# are formed for a call's longest row and all others, so one long row beside single tokens is slower so: 64 tokens and seven rows of one 42, 33; 512 and 31 rows of one 497, 209.  The states
# are as exact; y is formed of states and weights that were rounded to bf16 once (0.0022 of y instead of 0.0017), as scan.ssd forms it of whole rows.  Heads come in pairs, as ops/ssd.py has them.
CHUNKED_TOKENS = 32


def _suits_chunks(x, heads: int, groups: int, N: int, state: Optional[torch.Tensor] = None) -> bool:
    """(The chunks read and write states in pairs of floats; the kernels of tokens take them from any float on.)"""
    return (x.dtype is torch.bfloat16 and x.shape[1] >= CHUNKED_TOKENS and x.shape[2] == 64 * heads and N == 128 and heads % 2 == 0 and heads // groups % 2 == 0
            and x.shape[0] <= 65535 and (state is None or state.data_ptr() % 8 == 0) and hasattr(L.load(), "dewb_ssd_rows"))


def _chunks(x, dt, b, c, a, dt_bias, d, rows: Rows, state, heads: int, groups: int) -> torch.Tensor:
    """``_tokens`` by the chunked scan of ``csrc/kernels/ssd_sm100.cu``."""
    if not L.device_is_current(x):
        with L.on_device_of(x):
            return _chunks(x, dt, b, c, a, dt_bias, d, rows, state, heads, groups)
    R, T, C = x.shape
    whole16 = lambda t: t if t.stride(2) == 1 and all(n == 1 or s % 8 == 0 for n, s in zip(t.shape[:2], t.stride())) and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
    x, b, c, dt = whole16(x), whole16(b), whole16(c), _dense(dt)
    a, dt_bias, d = _fp32(a), _fp32(dt_bias), _fp32(d)
    dev, stream, lib = x.device, L.stream(), L.load()
    y = torch.empty(R, T, C, dtype=x.dtype, device=dev)
    scratch = torch.empty(R * T * heads + heads + 3 * R, dtype=torch.float32, device=dev)
    states = torch.empty(R * heads * -(-T // 64) * 64 * 128, dtype=torch.bfloat16, device=dev)
    steps = scratch.data_ptr()
    rates, places = steps + 4 * R * T * heads, steps + 4 * (R * T * heads + heads)
    call = _args(x, dt, None, b, c, a, dt_bias, d, state, state, y, None, rows, 128, groups, heads, True, True, 0 if state is None else state.shape[0], whole=True)
    L.check(lib.dewb_head_steps(call.packed, steps, rates, places, stream), "head_steps")
    strides = (ctypes.c_longlong * 6)(*_strides(x), *_strides(b), *_strides(c))
    L.check(lib.dewb_ssd_rows(x.data_ptr(), steps, rates, b.data_ptr(), c.data_ptr(), L.at(d), L.at(state), states.data_ptr(), y.data_ptr(), places, places + 4 * R, places + 8 * R,
                              R, T, heads, groups, ctypes.addressof(strides), stream), "ssd_rows")
    L.count_launches(3)
    _moved(state)
    return y


def _inside(rows: Rows, state: Optional[torch.Tensor]) -> Rows:
    """The plain forms' rows, of which those outside the store rest: on a GPU the status word tells of them, as the kernels have it (there an index outside would end the process); on the
    CPU they are an error."""
    if state is None or rows.row_ids is None:
        return rows
    there = (rows.row_ids >= 0) & (rows.row_ids < state.shape[0])
    if state.is_cuda:
        word = L.status(state.device)
        word.copy_(torch.where(there.all(), word, torch.full_like(word, OUTSIDE)))
    elif not bool((there | (rows.positions[:, 0] < 0)).all()):
        raise IndexError(f"rows {rows.row_ids.tolist()} of a store of {state.shape[0]}")
    return Rows(torch.where(there[:, None], rows.positions, -1), rows.lengths, torch.where(there, rows.row_ids, 0))


def selective_tokens_reference(x, dt, A_log, Bm, Cm, D=None, z=None, rows: Optional[Rows] = None, state=None):
    from .recurrence import _tokens as walk
    R, S, C = x.shape
    rows = whole(R, S, x.device) if rows is None else _inside(rows, state)
    step, A = F.softplus(dt.float(), threshold=60.0), -torch.exp(A_log.float())
    xf, Bf, Cf = x.float(), Bm.float(), Cm.float()

    def body(t, now):
        h = torch.exp(step[:, t].unsqueeze(-1) * A) * now[0] + (step[:, t] * xf[:, t]).unsqueeze(-1) * Bf[:, t].unsqueeze(1)
        y = torch.einsum("rcn,rn->rc", h, Cf[:, t])
        y = y if D is None else y + xf[:, t] * D.float()
        return [h], y if z is None else y * F.silu(z[:, t].float())
    return walk(rows, [state], [xf.new_zeros(R, *A.shape)], body, (R, S, C), x.dtype)


def selective_tokens(x: torch.Tensor, dt: torch.Tensor, A_log: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                     rows: Optional[Rows] = None, state: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A call's tokens ``x [R, S, C]`` through the selective scan: the steps' logits ``dt [R, S, C]``, ``A_log [C, N]`` (rates ``-exp(A_log)``), ``Bm, Cm [R, S, N]``, ``D [C]``, the gate's
    input ``z [R, S, C]`` (columns of wider rows will do) -> ``[R, S, C]``.  ``state [store rows, C, N]`` goes on in place (none: whole rows from nothing, nothing kept); a store row
    belongs to one row of a call.  Rows outside the store are reported by the status word (``library.check_status``) and give zeros."""
    N = A_log.shape[-1]
    C = x.shape[-1]
    _check("selective_tokens", x, dt, Bm, Cm, z, (A_log, D), state, rows, (C, N), C, C, N)
    if A_log.shape != (C, N) or (D is not None and D.shape != (C,)):
        raise ValueError(f"selective_tokens: A_log [{C}, states] and D [{C}], got {tuple(A_log.shape)}, {None if D is None else tuple(D.shape)}")
    if N > MOST_STATES or N == 0 or 0 in x.shape or not kernel_ok(x, dt, A_log, Bm, Cm, D, z) or L.transformed(x, dt, A_log, Bm, Cm, D, z):
        return selective_tokens_reference(x, dt, A_log, Bm, Cm, D, z, rows, state) if 0 not in x.shape else torch.zeros_like(x)
    return _tokens(x, dt, z, Bm, Cm, A_log, None, D, whole(*x.shape[:2], x.device) if rows is None else rows, state, N, 1, 0)


def ssd_tokens_reference(x, dt, dt_bias, A_log, Bm, Cm, D, H: int, G: int, rows: Optional[Rows] = None, state=None):
    from .recurrence import _tokens as walk
    R, S, _ = x.shape
    rows = whole(R, S, x.device) if rows is None else _inside(rows, state)
    xf = x.float().view(R, S, H, -1)
    Bf, Cf = (t.float().reshape(R, S, G, -1).repeat_interleave(H // G, 2) for t in (Bm, Cm))
    step = F.softplus(dt.float() if dt_bias is None else dt.float() + dt_bias.float(), threshold=60.0)
    decay = torch.exp(-step * torch.exp(A_log.float()))

    def body(t, now):
        h = decay[:, t, :, None, None] * now[0] + (step[:, t, :, None] * xf[:, t]).unsqueeze(-1) * Bf[:, t].unsqueeze(2)
        y = torch.einsum("rhpn,rhn->rhp", h, Cf[:, t])
        return [h], y if D is None else y + xf[:, t] * D.float()[:, None]
    return walk(rows, [state], [xf.new_zeros(R, H, xf.shape[-1], Bf.shape[-1])], body, x.shape, x.dtype)


def ssd_tokens(x: torch.Tensor, dt: torch.Tensor, dt_bias: Optional[torch.Tensor], A_log: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, D: Optional[torch.Tensor], H: int, G: int,
               rows: Optional[Rows] = None, state: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A call's tokens through the state space scan with a decay per head: ``x [R, S, H P]``, the steps' logits ``dt [R, S, H]`` and their bias ``[H]``, ``A_log [H]``, ``Bm, Cm [R, S, G N]``
    (head h uses those of group ``h // (H // G)``), ``D [H]`` -> ``[R, S, H P]``.  ``state [store rows, H, P, N]`` as in ``selective_tokens``."""
    if H < 1 or G < 1 or H % G or x.shape[-1] % H or Bm.shape[-1] % G or x.shape[-1] == 0:
        raise ValueError(f"ssd_tokens: {H} heads in {G} groups of x {tuple(x.shape)}, B {tuple(Bm.shape)}")
    P, N = x.shape[-1] // H, Bm.shape[-1] // G
    _check("ssd_tokens", x, dt, Bm, Cm, None, (A_log, dt_bias, D), state, rows, (H, P, N), H * P, H, G * N)
    if A_log.shape != (H,) or (dt_bias is not None and dt_bias.shape != (H,)) or (D is not None and D.shape != (H,)):
        raise ValueError(f"ssd_tokens: a number per head, {H}, for A_log, the steps' bias and D")
    if N > MOST_HEAD_STATES or 0 in x.shape or N == 0 or not kernel_ok(x, dt, dt_bias, A_log, Bm, Cm, D) or L.transformed(x, dt, dt_bias, A_log, Bm, Cm, D):
        return ssd_tokens_reference(x, dt, dt_bias, A_log, Bm, Cm, D, H, G, rows, state) if 0 not in x.shape else torch.zeros_like(x)
    rows = whole(*x.shape[:2], x.device) if rows is None else rows
    if _suits_chunks(x, H, G, N, state):
        return _chunks(x, dt, Bm, Cm, A_log, dt_bias, D, rows, state, H, G)
    return _tokens(x, dt, None, Bm, Cm, A_log, dt_bias, D, rows, state, N, G, H)

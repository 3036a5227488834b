"""Importable ``mk_sequences`` module: a ctypes shim over ``libmkb200_sequences.so``.

What happens to sequences between two decoding steps (``include/mkb200_sequences.h``): beam search's
selection and the reordering of states, the attention weight that cached keys receive, and the
eviction of the others.  No counterpart in the reference.  As the other shims it marshals pointers and
sizes; a missing library is an ImportError, never a fallback.

Every function enqueues its work on ``stream`` (a stream, a handle, or None for the current one) of the
current device, where all tensors must live, and neither synchronises nor reads anything back, so all of
them can be captured into a CUDA graph.  Arguments that the library does not take raise ``ValueError`` /
``TypeError`` here or ``SequenceError`` from its own checks, before anything is launched.  A wait on the device that
gives up is recorded there, and :func:`raise_status` looks.
"""

from __future__ import annotations

import ctypes
import math
import threading
from pathlib import Path

import torch
from torch import Tensor

_HERE = Path(__file__).resolve().parent
LIB_PATH = _HERE / "libmkb200_sequences.so"

MKBS_ABI_VERSION = 1
MAX_BEAMS, MAX_BEST, MAX_REGIONS, MAX_SLOTS = 64, 128, 48, 256
ERROR_NAMES = {0: "MKBS_OK", 1: "MKBS_ERR_INVALID_ARGUMENT", 2: "MKBS_ERR_CUDA", 3: "MKBS_ERR_DEVICE_TIMEOUT", 5: "MKBS_ERR_UNSUPPORTED"}

_i32, _f32, _ptr, _i64, _u32, _size = ctypes.c_int32, ctypes.c_float, ctypes.c_void_p, ctypes.c_int64, ctypes.c_uint32, ctypes.c_size_t


class MkbsBeams(ctypes.Structure):
    _fields_ = [
        ("struct_bytes", _u32), *[(n, _i32) for n in ("dtype", "groups", "beams", "vocab", "k")], ("row_stride", _i64),
        ("logits", _ptr), ("scores", _ptr), ("done", _ptr), ("eos", _i32), ("reserved", _i32),
        *[(n, _ptr) for n in ("out_scores", "out_parents", "out_tokens", "out_done", "workspace")], ("workspace_bytes", _size),
    ]


class MkbsRegion(ctypes.Structure):
    _fields_ = [("base", _ptr), ("outer", _i32), ("rows", _i32), ("outer_stride", _i64), ("slot_stride", _i64), ("row_bytes", _i64)]


class MkbsReorder(ctypes.Structure):
    _fields_ = [
        ("struct_bytes", _u32), ("slots", _i32), ("num_regions", _i32), ("first", _i32), ("regions", ctypes.POINTER(MkbsRegion)),
        ("parents", _ptr), ("lengths", _ptr), ("status", _ptr),
    ]


class MkbsKeyWeights(ctypes.Structure):
    _fields_ = [
        ("struct_bytes", _u32),
        *[(n, _i32) for n in ("layers", "sequences", "queries", "heads", "kv_heads", "dim", "positions", "length")],
        ("scale", _f32), ("lengths", _ptr), ("q", _ptr), ("q_layer", _i64), ("q_sequence", _i64),
        ("k", _ptr), ("k_layer", _i64), ("k_sequence", _i64), ("weights", _ptr), ("w_layer", _i64), ("w_sequence", _i64), ("w_head", _i64),
        ("workspace", _ptr), ("workspace_bytes", _size), ("status", _ptr), ("wait_timeout_ms", _u32), ("reserved", _u32),
    ]


class MkbsSelect(ctypes.Structure):
    _fields_ = [
        ("struct_bytes", _u32),
        *[(n, _i32) for n in ("layers", "sequences", "kv_heads", "positions", "length", "keep", "sinks", "recent", "reserved")],
        ("lengths", _ptr), ("weights", _ptr), ("w_layer", _i64), ("w_sequence", _i64), ("w_head", _i64), ("rows", _ptr), ("kept", _ptr),
    ]


class MkbsMove(ctypes.Structure):
    _fields_ = [
        ("struct_bytes", _u32), *[(n, _i32) for n in ("layers", "sequences", "kv_heads", "positions", "length", "keep", "head_bytes")],
        ("lengths", _ptr), ("rows", _ptr), ("caches", _ptr * 2), ("c_layer", _i64), ("c_sequence", _i64),
    ]


STRUCTS = (MkbsBeams, MkbsRegion, MkbsReorder, MkbsKeyWeights, MkbsSelect, MkbsMove)


class SequenceError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"{ERROR_NAMES.get(code, code)}: {message}")
        self.code = code


_lib = None


def load_library() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise ImportError(f"{LIB_PATH} is missing: build it with `python -m megakernels_b200.build sequences`. "
                          "There is no CPU fallback.")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, struct in (("beam_select", MkbsBeams), ("reorder_slots", MkbsReorder), ("key_weights", MkbsKeyWeights),
                         ("select_rows", MkbsSelect), ("move_rows", MkbsMove)):
        fn = getattr(lib, f"mkb_{name}")
        fn.argtypes, fn.restype = [ctypes.POINTER(struct), _ptr], ctypes.c_int
    for name, struct in (("beam", MkbsBeams), ("key_weights", MkbsKeyWeights)):
        fn = getattr(lib, f"mkb_{name}_bytes")
        fn.argtypes, fn.restype = [ctypes.POINTER(struct)], _size
    lib.mkb_sequences_last_error.restype = ctypes.c_char_p
    lib.mkb_sequences_struct_bytes.argtypes, lib.mkb_sequences_struct_bytes.restype = [_i32], _size
    if lib.mkb_sequences_abi_version() != MKBS_ABI_VERSION:
        raise ImportError(f"{LIB_PATH.name} has ABI {lib.mkb_sequences_abi_version()}, expected {MKBS_ABI_VERSION}")
    sizes = [lib.mkb_sequences_struct_bytes(i) for i in range(len(STRUCTS))]
    if sizes != [ctypes.sizeof(s) for s in STRUCTS]:
        raise ImportError(f"struct layouts of {LIB_PATH.name} {sizes} differ from this shim")
    _lib = lib
    return lib


def _refuse_host(name: str, t: Tensor):
    if not t.is_cuda:  # (before anything asks for a current device, which there may not be)
        raise ValueError(f"{name} must live on a CUDA device")


def _refuse(name: str, t, dtype, device: int, shape, inner: int | None):
    """Why a tensor is not what a call needs."""
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on a CUDA device")
    if t.get_device() != device:  # (the launch goes to the current device)
        raise ValueError(f"{name} lives on cuda:{t.get_device()} but the current device is cuda:{device} (wrap the call in torch.cuda.device(...))")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    raise ValueError(f"{name} must be contiguous" + ("" if inner is None else f" in its last {inner} dimensions"))


def _check(name: str, t, dtype, device: int, shape=None, inner: int | None = None) -> int:
    """Address of a tensor on the current device.  ``shape``: what it must be; ``inner``: how many of its last dimensions
    must lie one behind the other (None: all)."""
    # (a call's checks cost more than its launch, so what is right passes through one condition)
    if (isinstance(t, Tensor) and t.dtype is dtype and t.get_device() == device and (shape is None or t.shape == shape)
            and (t.is_contiguous() or (inner is not None and t.numel() and t[(0,) * (t.ndim - inner)].is_contiguous()))):
        return t.data_ptr()
    _refuse(name, t, dtype, device, shape, inner)


def _entry_points(c):
    """The current stream's handle, memory of a stream and its return.  torch has entry points of little host time for these that it does
    not document; without them its public ones serve."""
    return (getattr(c, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream),
            getattr(c, "_cuda_cudaCachingAllocator_raw_alloc", None) or (lambda size, handle: torch.cuda.caching_allocator_alloc(size, stream=handle)),
            getattr(c, "_cuda_cudaCachingAllocator_raw_delete", None) or torch.cuda.caching_allocator_delete)


_raw_stream, _raw_alloc, _raw_free = _entry_points(torch._C)


class _Where:
    """The stream of a call, and the tensors that it allocates there: given back when the call returns they go to
    that stream alone, whose later work runs after the kernels."""

    def __init__(self, stream, of: Tensor):
        self.device, self.where = torch.cuda.current_device(), of.device
        if stream is None:
            self.other, self.handle = None, _raw_stream(self.device)  # (0.1 us; as an object 1.3)
        elif isinstance(stream, int):  # (an external stream of handle 0 would be another one from torch's pool)
            self.other = torch.cuda.ExternalStream(stream, device=self.device) if stream else torch.cuda.default_stream(self.device)
            self.handle = stream
        else:
            if stream.device_index != self.device:  # (a launch goes to the current device)
                raise ValueError(f"the stream is cuda:{stream.device_index}'s but the current device is cuda:{self.device}")
            self.other, self.handle = stream, stream.cuda_stream

    def empty(self, shape: tuple[int, ...], strides: tuple[int, ...], dtype) -> Tensor:
        if self.other is None:  # (with its strides given a tensor takes 1.5 us, without them 2.4)
            return torch.empty_strided(shape, strides, dtype=dtype, device=self.where)
        with torch.cuda.stream(self.other):
            return torch.empty_strided(shape, strides, dtype=dtype, device=self.where)

    def launch_with(self, size: int, name: str, struct, *used) -> None:
        """A launch with ``size`` bytes of workspace, which go back to the stream behind it (as a tensor's would, in half the time)."""
        struct.workspace, struct.workspace_bytes = _raw_alloc(size, self.handle), size
        try:
            self.launch(name, struct, *used)
        finally:
            _raw_free(struct.workspace)

    def launch(self, name: str, struct, *used) -> None:
        """``used``: tensors that are not given out again before this stream has used them."""
        code = getattr(_lib, name)(ctypes.byref(struct), self.handle)
        if code:
            raise SequenceError(code, _lib.mkb_sequences_last_error().decode())
        if self.other is not None and self.other != torch.cuda.current_stream(self.device):
            for t in used:
                if t is not None:
                    t.record_stream(self.other)


def _fit(*numbers: int) -> None:
    """What goes into a struct's 32 bits: ctypes cuts other numbers without a word.  (Asked only where some number is negative or large.)"""
    if min(numbers) < -(2**31) or max(numbers) >= 2**31:
        raise ValueError(f"a number or a size does not fit 32 bits: {max(numbers, key=abs)}")


def _struct(kind):
    s = kind()
    s.struct_bytes = ctypes.sizeof(kind)
    return s


def _check_status(status, device: int) -> int:
    at = _check("status", status, torch.int32, device)
    if status.numel() < 16:
        raise ValueError("status must hold 16 words")
    return at


_records: dict[int, Tensor] = {}  # of the calls that are given no status, by device
_making = threading.Lock()


def _record(device: int) -> int:
    record = _records.get(device)
    if record is None:
        with _making:
            if device not in _records:
                record = torch.empty(16, dtype=torch.int32, device=torch.device("cuda", device))
                with torch.cuda.stream(torch.cuda.Stream(device)):  # (the current one may be under capture, and a replay shall not clear the record)
                    record.zero_()
                _records[device] = record
        record = _records[device]
    return record.data_ptr()


def raise_status(status: Tensor | None = None) -> None:
    """Synchronise, and raise if a wait of the calls that were given ``status`` has given up (None: of the calls on the current
    device that were given none); it is cleared then."""
    if status is None:
        status = _records.get(torch.cuda.current_device())
        if status is None:
            return
    if status.is_cuda:
        torch.cuda.synchronize(status.device)  # (all streams: the calls may have had others than the current one)
    code, block = status[:2].tolist()
    if code:
        with torch.inference_mode():  # (a record that was made there can be written nowhere else)
            status.zero_()
        raise SequenceError(code, f"a wait on the device gave up (block {block})")


def _set_lengths(s, lengths, device: int, sequences: int, positions: int):
    """Rows that each sequence holds: an int32 tensor on the device, or one number for all."""
    if isinstance(lengths, Tensor):
        s.lengths = _check("lengths", lengths, torch.int32, device, (sequences,))
        return lengths
    if not 0 <= int(lengths) <= positions:
        raise ValueError(f"length {lengths} outside a cache of {positions} rows")
    s.length = int(lengths)
    return None


def beam_select(logits: Tensor, scores: Tensor | None = None, *, beams: int, k: int, done: Tensor | None = None, eos: int | None = None,
                stream=None) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """The ``k`` best continuations of every group of ``beams`` rows of ``logits`` (``[groups * beams, vocab]`` bf16 or
    float32, rows any stride apart), best first: ``scores[b] + log_softmax(logits[b])[v]``, ties to the lowest ``(b, v)``.

    ``scores`` float32 ``[groups, beams]`` (None: zero); ``done`` uint8 ``[groups, beams]``: beams whose only
    continuation is ``eos``, at their score.  Returns scores float32, parents int32 (rows of ``logits``), tokens int32
    and done uint8, each ``[groups, k]``.
    """
    if not isinstance(logits, Tensor) or logits.ndim != 2:
        raise ValueError("logits must be [groups * beams, vocab]")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"logits must be bfloat16 or float32, got {logits.dtype}")
    rows, vocab = logits.shape
    if beams < 1 or rows < 1 or rows % beams:
        raise ValueError(f"{rows} rows of logits are no groups of {beams}")
    if (rows | vocab | k | (eos or 0)) >> 31:
        _fit(rows, vocab, k, eos or 0)
    _refuse_host("logits", logits)
    lib, where, groups = load_library(), _Where(stream, logits), rows // beams
    s, device = _struct(MkbsBeams), where.device
    s.groups, s.beams, s.vocab, s.k, s.dtype = groups, beams, vocab, k, int(logits.dtype is torch.float32)
    s.row_stride = logits.stride(0) if rows > 1 else vocab
    s.logits = _check("logits", logits, logits.dtype, device, inner=1)
    if scores is not None:
        s.scores = _check("scores", scores, torch.float32, device, (groups, beams))
    if done is not None:
        s.done = _check("done", done, torch.uint8, device, (groups, beams))
    s.eos = -1 if eos is None else int(eos)
    size = lib.mkb_beam_bytes(s)
    if not size:
        where.launch("mkb_beam_select", s)  # (says what is wrong)
    out = [where.empty((groups, k), (k, 1), t) for t in (torch.float32, torch.int32, torch.int32, torch.uint8)]
    s.out_scores, s.out_parents, s.out_tokens, s.out_done = (t.data_ptr() for t in out)
    where.launch_with(size, "mkb_beam_select", s, logits, scores, done)
    return tuple(out)


def reorder_slots(tensors: list[Tensor], parents: Tensor, *, dim: int = 0, first: int = 0, lengths: Tensor | None = None, status: Tensor | None = None,
                  stream=None) -> None:
    """``t[..., slot, ...] <- t[..., parents[slot], ...]`` for every slot at once and in place, ``dim`` being the slots'
    dimension (0, or 1 behind the layers') of every tensor.

    With ``lengths`` (int32 ``[slots]``) the dimension behind it is rows: a slot takes its parent's rows ``first ..
    lengths[parent] - 1``; the others stay.  ``parents`` int32 ``[slots]``; one outside the slots leaves its slot as it is.
    ``status``: int32 ``[16]``, zero, for a wait that gives up, after which not all rows have moved (:func:`raise_status`).
    """
    tensors = list(tensors)
    if not tensors:
        raise ValueError("no tensors to reorder")
    if dim not in (0, 1):
        raise ValueError("the slots' dimension is 0 or 1")
    if first < 0 or (first and lengths is None):
        raise ValueError("first counts rows: it is not negative and needs lengths")
    if not isinstance(parents, Tensor) or parents.ndim != 1:
        raise ValueError("parents must be int32 [slots]")
    if (first | parents.shape[0]) >> 31:
        _fit(first, parents.shape[0])
    _refuse_host("parents", parents)
    load_library()
    slots, where = parents.shape[0], _Where(stream, parents)
    base, device = _struct(MkbsReorder), where.device
    base.slots, base.first = slots, first
    base.parents = _check("parents", parents, torch.int32, device)
    by_rows = lengths is not None
    base.status = _record(device) if status is None else _check_status(status, device)
    if by_rows:
        base.lengths = _check("lengths", lengths, torch.int32, device, (slots,))
    regions = (MkbsRegion * len(tensors))()
    like = strides = None
    for i, t in enumerate(tensors):
        if like is not None and isinstance(t, Tensor) and t.shape == shape and t.dtype is like.dtype and t.get_device() == device and t.stride() == strides:
            regions[i] = regions[i - 1]  # (a layer's states are mostly as the one's before)
            regions[i].base = t.data_ptr()
            continue
        if not isinstance(t, Tensor):
            raise TypeError(f"tensor {i} must be a torch.Tensor")
        like, shape, strides, r = t, t.shape, t.stride(), regions[i]
        if len(shape) < dim + 1 + by_rows or shape[dim] != slots:
            raise ValueError(f"tensor {i} {list(shape)} does not have {slots} slots in dimension {dim}" + (" and rows behind it" if by_rows else ""))
        if t.numel() == 0:
            raise ValueError(f"tensor {i} is empty")
        if (shape[0] | shape[dim + by_rows]) >> 31:
            _fit(shape[0], shape[dim + by_rows])
        r.base = _check(f"tensor {i}", t, t.dtype, device, inner=len(shape) - dim - 1)
        size = t.element_size()
        slot_bytes = math.prod(shape[dim + 1 :]) * size
        r.outer, r.outer_stride = (shape[0], strides[0] * size) if dim else (1, 0)
        r.slot_stride = strides[dim] * size if slots > 1 else slot_bytes
        r.rows = shape[dim + 1] if by_rows else 1
        r.row_bytes = slot_bytes // r.rows
    if len(tensors) > MAX_REGIONS and len({r.base for r in regions}) < len(tensors):  # (the library sees those of a call)
        raise ValueError("a tensor is listed twice")
    for at in range(0, len(tensors), MAX_REGIONS):
        base.num_regions = min(MAX_REGIONS, len(tensors) - at)
        base.regions = ctypes.cast(ctypes.byref(regions, at * ctypes.sizeof(MkbsRegion)), ctypes.POINTER(MkbsRegion))
        where.launch("mkb_reorder_slots", base, parents, lengths, status, *tensors)


def key_weights(q: Tensor, keys: Tensor, weights: Tensor, lengths: Tensor | int, *, scale: float, status: Tensor | None = None, wait_timeout_ms: int = 0,
                stream=None) -> None:
    """Add to ``weights`` (float32 ``[layers, sequences, kv_heads, positions]``) the softmax weight that each cached key
    receives from the queries, summed over them and over the query heads that share the key.  ``status``: as in :func:`reorder_slots`
    (not all weights have been added then).

    ``q`` bf16 ``[layers, sequences, queries, heads, dim]``: the queries of the sequences' last rows; ``keys`` bf16 ``[layers,
    sequences, positions, kv_heads, dim]``, dim 64 or 128; ``lengths``: rows that each sequence holds, an int32 tensor
    ``[sequences]`` or one number for all.  Query t sees the rows up to its own, ``length - queries + t``.
    """
    if not all(isinstance(t, Tensor) for t in (q, keys, weights)) or q.ndim != 5 or keys.ndim != 5:
        raise ValueError("q must be [layers, sequences, queries, heads, dim], keys [layers, sequences, positions, kv_heads, dim]")
    layers, sequences, queries, heads, dim = q.shape
    positions, kv_heads = keys.shape[2:4]
    if (layers | sequences | queries | heads | positions | kv_heads) >> 31:
        _fit(*q.shape, *keys.shape)
    if wait_timeout_ms >> 32:
        raise ValueError(f"a limit of {wait_timeout_ms} ms does not fit 32 bits")
    _refuse_host("q", q)
    lib, where, bf16 = load_library(), _Where(stream, q), torch.bfloat16
    s, device = _struct(MkbsKeyWeights), where.device
    s.layers, s.sequences, s.queries, s.heads, s.dim, s.positions, s.kv_heads = layers, sequences, queries, heads, dim, positions, kv_heads
    s.q = _check("q", q, bf16, device, inner=3)
    s.k = _check("keys", keys, bf16, device, (layers, sequences, positions, kv_heads, dim), inner=3)
    s.weights = _check("weights", weights, torch.float32, device, (layers, sequences, kv_heads, positions), inner=1)
    s.q_layer, s.q_sequence = q.stride()[:2]
    s.k_layer, s.k_sequence = keys.stride()[:2]
    s.w_layer, s.w_sequence, s.w_head = weights.stride()[:3]
    lengths = _set_lengths(s, lengths, device, sequences, positions)
    s.scale, s.wait_timeout_ms = scale, wait_timeout_ms
    s.status = _record(device) if status is None else _check_status(status, device)
    size = lib.mkb_key_weights_bytes(s)
    if not size:
        where.launch("mkb_key_weights", s)  # (says what is wrong)
    where.launch_with(size, "mkb_key_weights", s, q, keys, weights, lengths, status)


def select_rows(weights: Tensor, lengths: Tensor | int, *, keep: int, sinks: int = 0, recent: int = 0, kept: Tensor | None = None, stream=None) -> Tensor:
    """Rows that stay when sequences are cut to ``keep`` rows: all of a sequence that has no more, else its first
    ``sinks``, its last ``recent`` and the heaviest others by ``weights`` (float32 ``[layers, sequences, kv_heads, positions]``;
    equal weights: the lowest row).

    Returns int32 ``[layers, sequences, kv_heads, keep]``: the rows, ascending, and -1 behind them.  ``kept`` (shape and strides of
    ``weights``, or ``weights`` itself) receives the weights of these rows in their new places.
    """
    if not isinstance(weights, Tensor) or weights.ndim != 4:
        raise ValueError("weights must be [layers, sequences, kv_heads, positions]")
    layers, sequences, kv_heads, positions = weights.shape
    if (keep | sinks | recent | layers | sequences | kv_heads | positions) >> 31:
        _fit(keep, sinks, recent, *weights.shape)
    _refuse_host("weights", weights)
    load_library()
    s, where = _struct(MkbsSelect), _Where(stream, weights)
    device = where.device
    s.layers, s.sequences, s.kv_heads, s.positions = layers, sequences, kv_heads, positions
    s.weights = _check("weights", weights, torch.float32, device, inner=1)
    s.w_layer, s.w_sequence, s.w_head = weights.stride()[:3]
    s.keep, s.sinks, s.recent = keep, sinks, recent
    lengths = _set_lengths(s, lengths, device, sequences, positions)
    if kept is not None:
        s.kept = _check("kept", kept, torch.float32, device, weights.shape, inner=1)
        if kept.stride() != weights.stride():
            raise ValueError("kept must have the strides of weights")
    n = max(keep, 1)  # (the library refuses less)
    rows = where.empty((layers, sequences, kv_heads, n), (sequences * kv_heads * n, kv_heads * n, n, 1), torch.int32)
    s.rows = rows.data_ptr()
    where.launch("mkb_select_rows", s, weights, lengths, kept)
    return rows


def move_rows(keys: Tensor, values: Tensor | None, rows: Tensor, lengths: Tensor | int, *, stream=None) -> None:
    """Row r of every key/value head <- its row ``rows[..., r]``, in place, in caches ``[layers, sequences, positions,
    kv_heads, dim]`` of one shape; ``rows`` as :func:`select_rows` returns them, ``lengths`` as it was given there.  An entry below r or
    outside the sequence's rows leaves row r as it is."""
    if not all(isinstance(t, Tensor) for t in (keys, rows)) or keys.ndim != 5 or rows.ndim != 4:
        raise ValueError("caches must be [layers, sequences, positions, kv_heads, dim], rows [layers, sequences, kv_heads, keep]")
    layers, sequences, positions, kv_heads, dim = keys.shape
    keep, size = rows.shape[3], keys.element_size()
    if (layers | sequences | positions | kv_heads | dim * size | keep) >> 31:
        _fit(*keys.shape, dim * size, keep)
    _refuse_host("keys", keys)
    load_library()
    s, where = _struct(MkbsMove), _Where(stream, keys)
    device = where.device
    s.layers, s.sequences, s.positions, s.kv_heads = layers, sequences, positions, kv_heads
    s.caches[0] = _check("keys", keys, keys.dtype, device, inner=3)
    if values is not None:
        s.caches[1] = _check("values", values, keys.dtype, device, keys.shape, inner=3)
        if values.stride() != keys.stride():
            raise ValueError("keys and values must have the same strides")
    s.head_bytes, s.c_layer, s.c_sequence = dim * size, keys.stride(0) * size, keys.stride(1) * size
    s.keep = keep
    s.rows = _check("rows", rows, torch.int32, device, (layers, sequences, kv_heads, keep))
    lengths = _set_lengths(s, lengths, device, sequences, positions)
    where.launch("mkb_move_rows", s, keys, values, rows, lengths)

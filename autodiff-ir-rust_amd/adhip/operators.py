"""Operators on device arrays: rotary positions, attention with masks, capped scores, distance bias and shared heads
(forward, backward, single tokens against a cache), and AdamW over many tensors.  The kernels and the checks of arguments
are behind the C ABI (`adhip_rotary`, `adhip_attention`, `adhip_attention_backward`, `adhip_adamw` in include/adhip.h,
where the formulas stand); they have no counterpart in the reference.

An array is a `DeviceArray` (`DeviceArray.empty`, `DeviceArray.of`, `program_array`) or anything on the device's memory with
`data_ptr()`, `shape`, `stride()` and `dtype` (for AdamW also `numel()` and `is_contiguous()`), such as a torch tensor; one that says by
`is_cuda` that it is elsewhere is refused.  Every call queues its kernels on `stream`
(a hipStream_t as an integer, for instance `torch.cuda.current_stream().cuda_stream`; the device's own stream where it is
not given) and returns: results are there when the stream has got to them, and arrays and workspaces must live and keep
still until then.  Nothing is allocated and nothing is kept between calls.
"""
from __future__ import annotations

import ctypes
import math
import struct
from array import array
from typing import List, Optional, Sequence

import numpy as np

F32, BF16, I32, E4M3 = 0, 1, 2, 3
_TYPES = {"float32": F32, "torch.float32": F32, "bfloat16": BF16, "torch.bfloat16": BF16, "int32": I32, "torch.int32": I32,
          "float8_e4m3fn": E4M3, "torch.float8_e4m3fn": E4M3}
_WIDTH = {F32: 4, BF16: 2, I32: 4, E4M3: 1}
ADAMW_BLOCK = 256  # elements that share a scale where states are held in 8 bits


def _host_values(values, dtype: str) -> np.ndarray:
    """Packed float32 or int32; whole numbers are not cut off to 32 bits."""
    values = np.ascontiguousarray(values)
    out = values.astype(dtype, copy=False)
    if dtype == "int32" and not np.array_equal(out, values):
        raise ValueError("values that are no whole numbers of 32 bits")
    return out


class DeviceArray:
    """Packed device memory of a `HipDevice`; freed with the object where the object allocated it."""

    is_cuda = True  # what torch calls memory of a GPU

    def __init__(self, dev, shape: Sequence[int], dtype: str = "float32", data: Optional[int] = None, owner=None):
        if dtype not in _TYPES:
            raise ValueError(f"{dtype!r} is not a type of device arrays (float32, bfloat16, int32, float8_e4m3fn)")
        self._dev, self.shape, self.dtype = dev, tuple(int(n) for n in shape), dtype
        self._own, self._owner = data is None, owner
        self._data = data
        if data is None:
            h = ctypes.c_void_p()
            _check(dev, _lib(dev).adhip_alloc(dev._ctx, max(1, self.nbytes), ctypes.byref(h)), "adhip_alloc")
            self._data = h.value

    @classmethod
    def empty(cls, dev, shape, dtype: str = "float32") -> "DeviceArray":
        return cls(dev, shape, dtype)

    @classmethod
    def of(cls, dev, values) -> "DeviceArray":
        """A copy of host values: float32 or int32."""
        values = np.asarray(values)
        values = _host_values(values, "int32" if values.dtype.kind in "iub" else "float32")
        a = cls(dev, values.shape, str(values.dtype))
        a.set(values)
        return a

    @property
    def nbytes(self) -> int:
        return math.prod(self.shape) * _WIDTH[_TYPES[self.dtype]]

    def data_ptr(self) -> int:
        return self._data

    def numel(self) -> int:
        return math.prod(self.shape)

    def is_contiguous(self) -> bool:
        return True

    def stride(self):
        out, n = [], 1
        for d in reversed(self.shape):
            out.append(n)
            n *= d
        return tuple(reversed(out))

    def reshape(self, *shape) -> "DeviceArray":
        """The same memory under another shape (it lives as long as either)."""
        shape = tuple(shape[0]) if len(shape) == 1 and not isinstance(shape[0], int) else shape
        if math.prod(shape) != math.prod(self.shape):
            raise ValueError(f"cannot see {list(self.shape)} as {list(shape)}")
        return DeviceArray(self._dev, shape, self.dtype, self._data, owner=self)

    def set(self, values) -> None:
        """Copies host values in (waits)."""
        if self.dtype not in ("float32", "int32"):
            raise ValueError(f"host values of type {self.dtype} are not supported")
        values = _host_values(values, self.dtype)
        if values.size != math.prod(self.shape):
            raise ValueError(f"{values.size} values for {list(self.shape)}")
        _check(self._dev, _lib(self._dev).adhip_copy_in(self._dev._ctx, self._data, values.ctypes.data, values.nbytes), "adhip_copy_in")

    def clear(self) -> None:
        """Zeros in every byte (waits)."""
        zeros = np.zeros(self.nbytes, np.uint8)
        _check(self._dev, _lib(self._dev).adhip_copy_in(self._dev._ctx, self._data, zeros.ctypes.data, zeros.nbytes), "adhip_copy_in")

    def numpy(self) -> np.ndarray:
        """A copy on the host (waits); bfloat16 as float32, 8-bit codes as uint8."""
        kind = {F32: np.float32, BF16: np.uint16, I32: np.int32, E4M3: np.uint8}[_TYPES[self.dtype]]
        out = np.empty(self.shape, kind)
        _check(self._dev, _lib(self._dev).adhip_copy_out(self._dev._ctx, out.ctypes.data, self._data, out.nbytes), "adhip_copy_out")
        return (out.astype(np.uint32) << 16).view(np.float32) if self.dtype == "bfloat16" else out

    def close(self) -> None:
        if self._own and self._data is not None and getattr(self._dev, "_ctx", None):
            _lib(self._dev).adhip_free(self._dev._ctx, self._data)
        self._data = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def program_array(program, id: str, shape: Optional[Sequence[int]] = None) -> DeviceArray:
    """The device buffer of a kept id of a resident program (`HipDevice.compile`), under `shape` where it is given: the
    value a run left there, and for a tensor made from host values what the next run reads."""
    lib, data, dims, n = program._lib, ctypes.c_void_p(), ctypes.POINTER(ctypes.c_uint64)(), ctypes.c_size_t()
    rc = _declared(lib).adhip_program_buffer(program._h, id.encode("utf-8"), ctypes.byref(data), ctypes.byref(dims), ctypes.byref(n))
    if rc == 1:
        raise KeyError(f"{id!r} is not a kept id of the program")
    _check(program._dev, rc, "adhip_program_buffer")
    a = DeviceArray(program._dev, [int(dims[i]) for i in range(n.value)], "float32", data.value, owner=program)
    return a if shape is None else a.reshape(*shape)


def synchronize(dev) -> None:
    """Waits for everything queued on the device's own stream."""
    _check(dev, _lib(dev).adhip_sync(dev._ctx), "adhip_sync")


# ---- the C structs, packed without a ctypes object per field: a call's own cost counts where one token is decoded ----

_ARRAY = struct.Struct("=Qii8q")
_PACK_ARRAY = _ARRAY.pack
_NONE = bytes(_ARRAY.size)
_ZEROS = (0, 0, 0, 0)
_PADS = [(0,) * (4 - n) for n in range(5)]
_ROTARY_TAIL = struct.Struct("=ii")
_ATTENTION_TAIL = struct.Struct("=ffiiqQQ")
_ADAMW = struct.Struct("=Qqiiii6d")
_SIZE = struct.Struct("=q").unpack_from
_NO_GRADIENTS = _NONE * 4
_NO_MORE = _NONE * 11 + bytes(_ATTENTION_TAIL.size)


_kinds = {}  # type objects met so far -> our number of the type


def _kind(dtype) -> int:
    kind = _kinds.get(dtype)
    if kind is None:
        kind = _TYPES.get(str(dtype))
        if kind is None:
            raise ValueError(f"arrays of type {dtype} are not supported")
        _kinds[dtype] = kind
    return kind


def _array(a, shape_alone: bool = False) -> bytes:
    if a is None:
        return _NONE
    try:
        if not (a.is_cuda or shape_alone):
            raise ValueError(f"an array of shape {list(a.shape)} is not in device memory")
    except AttributeError:  # an array that does not say
        pass
    shape = a.shape
    n = len(shape)
    kind = _kinds.get(a.dtype)
    if kind is None:
        kind = _kind(a.dtype)
    if n == 4:
        return _PACK_ARRAY(a.data_ptr(), kind, 4, *shape, *a.stride())
    if n > 4:
        raise ValueError(f"arrays of {n} dims are not supported")
    pad = _PADS[n]
    return _PACK_ARRAY(a.data_ptr(), kind, n, *shape, *pad, *a.stride(), *pad)


def _declared(lib):
    if getattr(lib, "_adhip_operators", False):
        return lib
    c = ctypes
    vp, sz, i32 = c.c_void_p, c.c_size_t, c.c_int
    lib.adhip_alloc.argtypes = [vp, sz, c.POINTER(vp)]
    lib.adhip_free.argtypes = [vp, vp]
    lib.adhip_copy_in.argtypes = [vp, vp, vp, sz]
    lib.adhip_copy_out.argtypes = [vp, vp, vp, sz]
    lib.adhip_sync.argtypes = [vp]
    lib.adhip_program_buffer.argtypes = [vp, c.c_char_p, c.POINTER(vp), c.POINTER(c.POINTER(c.c_uint64)), c.POINTER(sz)]
    lib.adhip_attention_workspace.argtypes = [vp, c.c_char_p, i32, c.POINTER(sz)]
    for name in ("adhip_rotary", "adhip_attention", "adhip_attention_backward", "adhip_adamw"):
        getattr(lib, name).argtypes = [vp, c.c_char_p, vp]
    for name in ("adhip_alloc", "adhip_free", "adhip_copy_in", "adhip_copy_out", "adhip_sync", "adhip_program_buffer",
                 "adhip_attention_workspace", "adhip_rotary", "adhip_attention", "adhip_attention_backward", "adhip_adamw"):
        getattr(lib, name).restype = i32
    lib.adhip_stream.argtypes = [vp]
    lib.adhip_stream.restype = vp
    lib._adhip_operators = True
    return lib


def _lib(dev):
    lib = dev._lib
    return lib if getattr(lib, "_adhip_operators", False) else _declared(lib)


def _check(dev, rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed: " + dev.last_error())


def _stream(dev, stream: Optional[int]) -> int:
    return _lib(dev).adhip_stream(dev._ctx) if stream is None else stream


# ---- rotary positions -----------------------------------------------------------------------------------------------


def rotary_table(rows: int, features: int, base: float = 10000.0, factor: float = 1.0, scaling: Optional[str] = None,
                 trained: int = 0, slow: float = 1.0, fast: float = 32.0):
    """(cos, sin), float32 [rows, features / 2], of the angles position * base^(-2 i / features), computed in 64 bits.

    For contexts `factor` times as long as the `trained` positions: scaling "linear" divides all angles by the factor,
    "base" raises the base so that the slowest pair turns as far as it did (base * factor^(features / (features - 2))),
    "parts" leaves pairs that turn more than `fast` times over the trained positions as they are, divides those that turn
    less than `slow` times by the factor, and goes from one to the other in proportion between (the method of YaRN, Peng
    et al. 2023, whose factor on the scores, (0.1 ln factor + 1)^2, is the caller's to put into the attention's scale)."""
    if rows < 1 or features < 2 or features % 2 or base <= 0 or factor <= 0:
        raise ValueError("a table has at least one row, an even number of features, a positive base and a positive factor")
    i = np.arange(0, features, 2, dtype=np.float64)
    if scaling == "base":
        if features == 2:
            raise ValueError("scaling by the base wants more than one pair")
        base = base * factor ** (features / (features - 2))
    per = base ** (-i / features)
    if scaling == "linear":
        per = per / factor
    elif scaling == "parts":
        if trained < 1 or not 0 <= slow < fast:
            raise ValueError("scaling in parts wants the trained length and 0 <= slow < fast")
        turns = trained * per / (2.0 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
        per = per * keep + per / factor * (1.0 - keep)
    elif scaling not in (None, "base"):
        raise ValueError(f"scaling is 'linear', 'base' or 'parts', not {scaling!r}")
    angles = np.arange(rows, dtype=np.float64)[:, None] * per
    return np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)


def rotary(dev, x, out, cos, sin, positions, *, second=None, second_out=None, interleaved: bool = False, inverse: bool = False,
           stream: Optional[int] = None) -> None:
    """Turns the feature pairs of x [batch, length, heads, size] by the angles of `positions` [batch, length] into out
    (x itself is allowed); `second` [batch, length, other heads, size] by the same angles in the same launch.  cos and sin
    are tables [rows, pairs]; features behind 2 pairs are copied.  `inverse` is the gradient's rule."""
    args = b"".join((_array(x), _array(out), _array(second), _array(second_out), _array(cos), _array(sin), _array(positions),
                     _ROTARY_TAIL.pack(bool(interleaved), bool(inverse))))
    _check(dev, _lib(dev).adhip_rotary(dev._ctx, args, _stream(dev, stream)), "adhip_rotary")


# ---- attention ------------------------------------------------------------------------------------------------------


def _attention_tail(q: bytes, scale, causal, window, cap, workspace) -> bytes:
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, _SIZE(q, 40)[0]))  # (the last extent of four)
    room, room_bytes = 0, 0
    if workspace is not None:
        if not getattr(workspace, "is_cuda", True):
            raise ValueError("the workspace is not in device memory")
        room, room_bytes = workspace.data_ptr(), workspace.nbytes
    return _ATTENTION_TAIL.pack(scale, cap, bool(causal), 0, window, room, room_bytes)


def _masks(slopes, lengths, prefix, query_documents, key_documents) -> bytes:
    if slopes is lengths is prefix is query_documents is key_documents is None:
        return _NONE * 5
    return b"".join([_array(a) for a in (slopes, lengths, prefix, query_documents, key_documents)])


def attention_workspace(dev, q, k, v, *, backward: bool = False) -> int:
    """Bytes of workspace that `attention`, and with `backward` also `attention_backward`, take on arrays of these shapes."""
    need = ctypes.c_size_t()
    args = _array(q, True) + _array(k, True) + _array(v, True) + _NO_MORE
    _check(dev, _lib(dev).adhip_attention_workspace(dev._ctx, args, bool(backward), ctypes.byref(need)), "adhip_attention_workspace")
    return need.value


def attention(dev, q, k, v, out, lse, *, scale: Optional[float] = None, causal: bool = False, window: int = 0, cap: float = 0.0,
              slopes=None, lengths=None, prefix=None, query_documents=None, key_documents=None, workspace=None,
              stream: Optional[int] = None) -> None:
    """out = softmax(scores) v over the keys that each query sees, lse = log of the sum of the scores' exponentials.

    q, out [batch, queries, heads, size]; k, v [batch, keys, key heads, size]; lse f32 [batch, queries, heads].  Scores are
    cap tanh(scale q.k / cap) - slopes[head] |distance|; what a query sees is said by causal, window, lengths [batch],
    prefix [batch] and documents [batch, queries] / [batch, keys].  scale is 1 / sqrt(size) where it is not given."""
    first = _array(q)
    args = b"".join((first, _array(k), _array(v), _array(out), _array(lse), _masks(slopes, lengths, prefix, query_documents, key_documents),
                     _NO_GRADIENTS, _attention_tail(first, scale, causal, window, cap, workspace)))
    _check(dev, _lib(dev).adhip_attention(dev._ctx, args, _stream(dev, stream)), "adhip_attention")


def attention_backward(dev, q, k, v, out, lse, out_grad, q_grad, k_grad, v_grad, *, scale: Optional[float] = None,
                       causal: bool = False, window: int = 0, cap: float = 0.0, slopes=None, lengths=None, prefix=None,
                       query_documents=None, key_documents=None, workspace=None, stream: Optional[int] = None) -> None:
    """Gradients of q, k and v from `attention`'s out and lse and the gradient of out; the other arguments as there."""
    first = _array(q)
    args = b"".join((first, _array(k), _array(v), _array(out), _array(lse), _masks(slopes, lengths, prefix, query_documents, key_documents),
                     _array(out_grad), _array(q_grad), _array(k_grad), _array(v_grad),
                     _attention_tail(first, scale, causal, window, cap, workspace)))
    _check(dev, _lib(dev).adhip_attention_backward(dev._ctx, args, _stream(dev, stream)), "adhip_attention_backward")


# ---- AdamW ----------------------------------------------------------------------------------------------------------


def _one_kind(name, arrays, allowed) -> int:
    kinds = {a.dtype for a in arrays}
    if len(kinds) == 1 and _kinds.get(*kinds) in allowed:
        return _kinds[kinds.pop()]
    kinds = {_kind(t) for t in kinds}
    if len(kinds) != 1 or not kinds <= allowed:
        raise ValueError(f"{name} must all have one supported type, not {sorted({str(a.dtype) for a in arrays})}")
    return kinds.pop()


def _addresses(name, arrays, counts) -> List[int]:
    """Where the packed arrays begin, of these numbers of elements."""
    if len(arrays) != len(counts):
        raise ValueError(f"{len(arrays)} {name} for {len(counts)} parameters")
    try:
        if all([a.is_cuda and a.is_contiguous() and a.numel() == n for a, n in zip(arrays, counts)]):
            return [a.data_ptr() for a in arrays]
    except AttributeError:  # arrays that do not say where they are
        pass
    for i, (a, n) in enumerate(zip(arrays, counts)):
        if a.numel() != n or not a.is_contiguous():
            raise ValueError(f"{name}[{i}] is {list(a.shape)}: {n} packed elements are wanted")
        if not getattr(a, "is_cuda", True):
            raise ValueError(f"{name}[{i}] is not in device memory")
    return [a.data_ptr() for a in arrays]


def adamw(dev, parameters: List, gradients: List, first: List, second: List, *, step: int, rate: float, beta1: float = 0.9,
          beta2: float = 0.999, eps: float = 1e-8, decay: float = 0.01, grad_scale: float = 1.0, first_scales: Optional[List] = None,
          second_scales: Optional[List] = None, parameters_out: Optional[List] = None, first_out: Optional[List] = None,
          second_out: Optional[List] = None, first_scales_out: Optional[List] = None, second_scales_out: Optional[List] = None,
          stream: Optional[int] = None) -> None:
    """One AdamW step on every tensor of the list: parameters and gradients f32 or bf16, moments `first` and `second` f32 of
    the parameters' sizes, or float8_e4m3fn codes [blocks, 256] with f32 scales [blocks] (`adamw_blocks`).  In place where
    no *_out list is given.  Arrays are packed."""
    n = len(parameters)
    if n == 0:
        return
    counts = [p.numel() for p in parameters]
    p_type = _one_kind("parameters", parameters, {F32, BF16})
    g_type = _one_kind("gradients", gradients, {F32, BF16})
    state = _one_kind("moments", [*first, *second], {F32, E4M3})
    blocks = [-(-c // ADAMW_BLOCK) for c in counts]
    held = counts if state == F32 else [b * ADAMW_BLOCK for b in blocks]
    none = [0] * n
    columns = [_addresses("parameters", parameters, counts), _addresses("gradients", gradients, counts),
               _addresses("first", first, held), _addresses("second", second, held)]
    scales = [none, none]
    if state == E4M3:
        if first_scales is None or second_scales is None:
            raise ValueError("moments in 8 bits want first_scales and second_scales")
        _one_kind("scales", [*first_scales, *second_scales], {F32})
        scales = [_addresses("first_scales", first_scales, blocks), _addresses("second_scales", second_scales, blocks)]
    outs = []
    for name, arrays, own, size, kind in (("parameters_out", parameters_out, columns[0], counts, p_type),
                                          ("first_out", first_out, columns[2], held, state), ("second_out", second_out, columns[3], held, state),
                                          ("first_scales_out", first_scales_out if state == E4M3 else None, scales[0], blocks, F32),
                                          ("second_scales_out", second_scales_out if state == E4M3 else None, scales[1], blocks, F32)):
        if arrays is not None:
            _one_kind(name, arrays, {kind})
            own = _addresses(name, arrays, size)
        outs.append(own)
    flat = [x for row in zip(*columns, *scales, *outs, counts) for x in row]
    tensors = array("q", flat)  # n of the C struct; read before the call returns
    args = _ADAMW.pack(tensors.buffer_info()[0], n, p_type, g_type, state, step, rate, beta1, beta2, eps, decay, grad_scale)
    _check(dev, _lib(dev).adhip_adamw(dev._ctx, args, _stream(dev, stream)), "adhip_adamw")


def adamw_blocks(count: int) -> int:
    """Blocks of 256 elements, one scale each, that a tensor of `count` elements has where its states are held in 8 bits."""
    return -(-count // ADAMW_BLOCK)

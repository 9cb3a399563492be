"""8-bit serving operators on torch CUDA tensors, over
include/denoiser_b200_quant.h (which has the exact definitions):

``RowCache``  rows quantised to 8 or 4 bits as they are written (a scale for
              each row or group of columns) and read back through row numbers
              or page tables;
``FrameStore`` encoded frames of a temporal model in RowCaches, so that one
              model decodes several sequences in turn (``sharding.
              denoise_streams``);
``Linear8``   the product of tokens with a weight matrix in 8-bit integers,
              a scale for each token and each output channel: over token rows,
              over the pixels of NCHW planes (a 1x1 convolution), or straight
              from the rows of an 8-bit RowCache.

The reference has no counterpart. Calls are asynchronous on ``stream``
(default: torch's current stream on the operator's device) and may be captured
into a CUDA graph. Wrong arguments raise ``InvalidArgumentError`` (or
``DenoiserError`` with DN_ERR_DTYPE for a type that is neither FP16 nor FP32).
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import DN_ERR_DEVICE, DN_ERR_DTYPE, DN_ERR_INVALID_ARG, DenoiserError, InvalidArgumentError, Weights, check, lib


def _bad(msg: str):
    raise InvalidArgumentError(DN_ERR_INVALID_ARG, msg)


def _code(dtype, what: str) -> int:
    """The C-ABI's number of a torch dtype."""
    if dtype is torch.float16:
        return 1
    if dtype is torch.float32:
        return 0
    raise DenoiserError(DN_ERR_DTYPE, f"{what}: expected FP16 or FP32, got {dtype}")


def _device_of(device) -> int:
    d = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    if d.type != "cuda":
        _bad("the operators run on CUDA devices")
    return torch.cuda.current_device() if d.index is None else d.index


@contextlib.contextmanager
def _on(device: int, stream):
    """`device` and `stream` made current, so that what a call allocates
    belongs to them. The methods below come back through here when they are
    not on their device, or were given a stream."""
    with torch.cuda.device(device):
        s = stream if stream is not None else torch.cuda.current_stream(device)
        if s.device.index != device:
            _bad(f"the stream is of device {s.device.index}, the operator of device {device}")
        with torch.cuda.stream(s):
            yield


def _elsewhere(device: int, stream) -> bool:
    return stream is not None or torch.cuda.current_device() != device


try:  # the current stream's handle without a Stream object: a microsecond of a call's eight
    from torch._C import _cuda_getCurrentRawStream as _stream
except ImportError:
    def _stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream


def _on_device(t, device: int, what: str) -> None:
    if t.get_device() != device:
        _bad(f"{what} must be a tensor on cuda:{device}")


def _matrix(t, rows: int | None, cols: int, device: int, what: str) -> int:
    """Row stride of a 2-D tensor with unit column stride."""
    if t.get_device() != device:
        _bad(f"{what} must be a tensor on cuda:{device}")
    shape = t.shape
    if len(shape) != 2 or shape[1] != cols or (rows is not None and shape[0] != rows):
        _bad(f"{what} must be ({'rows' if rows is None else rows}, {cols}), got {tuple(shape)}")
    ld, one = t.stride()
    if one != 1 and cols > 1 and shape[0] > 0:
        _bad(f"{what}: the columns must be adjacent (stride 1)")
    return ld if shape[0] > 1 else cols


class RowCache:
    """``pages * page_rows`` rows of ``cols`` values held in ``bits`` bits (8
    or 4), with a scale for every ``group`` columns (0: one a row). ``codes``
    and ``scales`` are the tensors it is held in; new rows read as zeros, on any
    stream once the cache is made. Whoever uses one cache on several streams
    orders writes and reads of the same rows, and keeps the cache until they are
    done, as with any tensor."""

    def __init__(self, pages: int, page_rows: int, cols: int, bits: int = 8, group: int = 0, device=0):
        if pages < 0 or page_rows < 1 or cols < 1:
            _bad("RowCache: pages >= 0, page_rows >= 1 and cols >= 1 are needed")
        if bits not in (8, 4):
            _bad("RowCache: bits must be 8 or 4")
        group = group or cols
        if group < 0 or cols % group or (group != cols and group % 8):
            _bad("RowCache: group must divide cols, and be a multiple of 8 where it is smaller than a row")
        if pages * page_rows >= 1 << 31:
            _bad("RowCache: fewer than 2^31 rows")
        self.pages, self.page_rows, self.cols, self.bits, self.group = pages, page_rows, cols, bits, group
        self.capacity = pages * page_rows
        self.device = _device_of(device)
        d = torch.device("cuda", self.device)
        row = ((cols * bits + 7) // 8 + 15) // 16 * 16
        self._codes = torch.zeros(self.capacity, row, dtype=torch.uint8, device=d)
        self._scales = torch.zeros(self.capacity, cols // group, dtype=torch.float32, device=d)
        self._err = torch.zeros(1, dtype=torch.int32, device=d)
        # The zeros are there before any call, whatever stream it is on. (In a
        # capture they are part of the graph, in front of what uses them.)
        with torch.cuda.device(d):
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream(d).synchronize()
        self._bind()

    def _bind(self) -> None:
        """The addresses that the calls take, of the tensors that this cache holds."""
        self.device = self._codes.get_device()
        self._held = (self._codes.data_ptr(), self._codes.shape[1], self._scales.data_ptr(), self.capacity)
        self._err_ptr = self._err.data_ptr()

    def __setstate__(self, state) -> None:  # a copy or a loaded cache has tensors of its own
        self.__dict__.update(state)
        self._bind()

    # Tensors to look at or write into; another one cannot take their place.
    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)

    def _slots(self, slots, rows: int | None):
        _on_device(slots, self.device, "RowCache: slots")
        if slots.dtype is not torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
            _bad("RowCache: slots must be a contiguous 1-D int64 tensor")
        if rows is not None and slots.shape[0] != rows:
            _bad(f"RowCache: {slots.shape[0]} slots for {rows} rows")
        return slots.data_ptr()

    def write(self, x, slots=None, row0: int = 0, stream=None) -> None:
        """Rows x (rows, cols), FP16 or FP32, any row stride that holds a row,
        into the cache rows ``slots`` (int64 CUDA tensor), or ``row0``, ``row0 + 1``, ...
        Rows with a negative slot are skipped; a slot at or behind the capacity
        is skipped and reported by ``sync``. Of rows with the same slot the
        last one is held."""
        if _elsewhere(self.device, stream):
            with _on(self.device, stream):
                return self.write(x, slots, row0)
        dtype = _code(x.dtype, "RowCache.write")
        ldx = _matrix(x, None, self.cols, self.device, "RowCache.write: x")
        rows = x.shape[0]
        codes, ld, scales, cap = self._held
        if slots is None and not 0 <= row0 <= cap:  # ctypes would cut a number that 64 bits do not hold
            _bad(f"RowCache.write: row0 {row0} outside a cache of {cap} rows")
        check(lib().dn_launch_cache_write(
            x.data_ptr(), dtype, ldx, rows, self.cols, None if slots is None else self._slots(slots, rows), row0, codes,
            ld, scales, cap, self.bits, self.group, self._err_ptr, _stream(self.device)))

    def read_rows(self, slots=None, row0: int = 0, rows: int | None = None, out=None, dtype=None, stream=None):
        """Cache rows ``slots`` (int64 CUDA tensor), or the ``rows`` rows from
        ``row0`` on -> (rows, cols) in ``dtype`` (default FP16) or into
        ``out``. Out rows of a skipped slot (see ``write``) stay as they were;
        without ``out`` they are zeros."""
        if _elsewhere(self.device, stream):
            with _on(self.device, stream):
                return self.read_rows(slots, row0, rows, out, dtype)
        if slots is None:
            if rows is None or rows < 0:
                _bad("RowCache.read_rows: slots, or rows >= 0, is needed")
            p, n = None, rows
        else:
            p, n = self._slots(slots, rows), slots.shape[0]
        if out is None:
            out = torch.zeros(n, self.cols, dtype=dtype or torch.float16, device=self._codes.device)
        code = _code(out.dtype, "RowCache.read_rows")
        ldo = _matrix(out, n, self.cols, self.device, "RowCache.read_rows: out")
        codes, ld, scales, cap = self._held
        if slots is None and not 0 <= row0 <= cap:
            _bad(f"RowCache.read_rows: row0 {row0} outside a cache of {cap} rows")
        check(lib().dn_launch_cache_read_rows(codes, ld, scales, cap, self.cols, self.bits, self.group, p, row0, n,
                                              out.data_ptr(), code, ldo, self._err_ptr, _stream(self.device)))
        return out

    def read(self, table, lengths=None, out=None, dtype=None, stream=None):
        """Sequences through a page table (batch, n) (int32 CUDA tensor; a page
        may occur more than once) -> (batch, n * page_rows, cols) in ``dtype``
        (default FP16), or into ``out`` (batch, max_rows, cols). Row i of
        sequence b is row i % page_rows of page table[b, i // page_rows] for
        i < lengths[b] (int32 CUDA tensor; default: all). What lies behind a
        sequence's length, and rows of a negative page, stay as they were;
        without ``out`` they are zeros."""
        if _elsewhere(self.device, stream):
            with _on(self.device, stream):
                return self.read(table, lengths, out, dtype)
        _on_device(table, self.device, "RowCache.read: table")
        if table.dtype is not torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
            _bad("RowCache.read: table must be a 2-D int32 tensor with adjacent columns")
        b, n = table.shape
        if lengths is not None:
            _on_device(lengths, self.device, "RowCache.read: lengths")
            if lengths.dtype is not torch.int32 or lengths.shape != (b,) or not lengths.is_contiguous():
                _bad(f"RowCache.read: lengths must be a contiguous int32 tensor ({b},)")
        if out is None:
            out = torch.zeros(b, n * self.page_rows, self.cols, dtype=dtype or torch.float16, device=self._codes.device)
        code = _code(out.dtype, "RowCache.read")
        _on_device(out, self.device, "RowCache.read: out")
        if out.dim() != 3 or out.shape[0] != b or out.shape[2] != self.cols:
            _bad(f"RowCache.read: out must be ({b}, rows, {self.cols}), got {tuple(out.shape)}")
        step, ldo, one = out.stride()
        if one != 1 and self.cols > 1 and out.numel():
            _bad("RowCache.read: out's columns must be adjacent (stride 1)")
        codes, ld, scales, cap = self._held
        check(lib().dn_launch_cache_read_pages(
            codes, ld, scales, cap, self.cols, self.bits, self.group, self.page_rows, table.data_ptr(),
            table.stride(0) if b > 1 else n, n, None if lengths is None else lengths.data_ptr(), b, out.shape[1],
            out.data_ptr(), code, step, ldo if out.shape[1] > 1 else self.cols, self._err_ptr, _stream(self.device)))
        return out

    def sync(self, stream=None) -> None:
        """Synchronise the stream and raise if a call met a slot or page
        behind the cache since the last check."""
        with _on(self.device, stream):
            torch.cuda.current_stream(self.device).synchronize()
            word = int(self._err.item())
            if word:
                self._err.zero_()
        if word:
            raise DenoiserError(DN_ERR_DEVICE, f"RowCache: a slot or page lies behind the cache (error word {word:#x})")


class FrameStore:
    """``frames`` encoded h x w frames of a temporal Model in 8 (or 4) bits, a
    RowCache per level: ``park`` quantises a frame's features out of the model's
    cache slot, ``restore`` puts them back into a slot (any one, any number of
    times). A slot holds them in FP16; the store takes half of that (or a
    quarter), and the model's T slots can serve many sequences."""

    def __init__(self, model, h: int, w: int, frames: int, bits: int = 8, group: int = 0):
        self.model, self.h, self.w, self.frames = model, h, w, frames
        self.caches = []
        for level in range(model.num_levels + 1):
            rows, cols = model.feature_shape(h, w, level)
            self.caches.append(RowCache(frames, rows, cols, bits=bits, group=group, device=model.device))

    def _entry(self, entry: int) -> int:
        if not 0 <= entry < self.frames:
            _bad(f"FrameStore: entry {entry} outside [0, {self.frames})")
        return entry

    def park(self, slot: int, entry: int, stream=None) -> None:
        """The h x w frame in the model's cache slot `slot` into `entry`."""
        self._entry(entry)
        held = self.model.slot_frame(slot)
        if held != (self.h, self.w):
            _bad(f"FrameStore.park: slot {slot} holds " + (f"a {held[0]}x{held[1]} frame" if held[0] else "no frame") +
                 f", the store {self.h}x{self.w} ones")
        for level, c in enumerate(self.caches):
            c.write(self.model.frame_features(self.h, self.w, slot, level), row0=entry * c.page_rows, stream=stream)

    def restore(self, entry: int, slot: int, stream=None) -> None:
        """The frame of `entry` into the model's cache slot `slot` (where the
        model was used with another frame size last, its other slots are
        dropped, as by ``encode_frame``)."""
        self._entry(entry)
        for level, c in enumerate(self.caches):
            c.read_rows(row0=entry * c.page_rows, rows=c.page_rows,
                        out=self.model.frame_features(self.h, self.w, slot, level), stream=stream)

    @property
    def bytes(self) -> int:
        """Device bytes of the held codes and scales."""
        return sum(c.codes.numel() + 4 * c.scales.numel() for c in self.caches)


class Linear8:
    """The 8-bit product layer with weights (Cout, Cin) or (Cout, Cin, 1, 1)
    and optional bias from a WeightStore, quantised when the layer is made.
    ``gate`` ends it with SimpleGate (half the output channels); ``segments``
    > 1 makes the layer of ``forward_cached`` over that many pages. A layer
    may be used by any number of calls at once."""

    def __init__(self, store: Weights, weight_name: str, bias_name: str | None = None, gate: bool = False,
                 segments: int = 1, device=0):
        self._h = ctypes.c_void_p()
        self.device = _device_of(device)
        check(lib().dn_linear8_create(store._h, weight_name.encode(), bias_name.encode() if bias_name else None,
                                      int(gate), segments, self.device, ctypes.byref(self._h)))
        self._info()

    @classmethod
    def from_tensors(cls, weight, bias=None, gate: bool = False, segments: int = 1, stream=None):
        """A layer of CUDA tensors: weight (Cout, Cin) and bias (Cout) of the
        same type, FP16 or FP32, both copied."""
        self = cls.__new__(cls)
        self._h = ctypes.c_void_p()
        if weight.dim() == 4 and weight.shape[2:] == (1, 1):
            weight = weight.reshape(weight.shape[:2])
        if not weight.is_cuda:
            _bad("Linear8: the weight must be a CUDA tensor")
        self.device = weight.device.index
        dtype = _code(weight.dtype, "Linear8: weight")
        ldw = _matrix(weight, None, weight.shape[-1], self.device, "Linear8: weight")
        if bias is not None:
            _on_device(bias, self.device, "Linear8: bias")
            if bias.dtype != weight.dtype or bias.shape != (weight.shape[0],) or not bias.is_contiguous():
                _bad(f"Linear8: bias must be a contiguous ({weight.shape[0]},) tensor of the weight's type")
        with _on(self.device, stream):
            check(lib().dn_linear8_create_device(weight.data_ptr(), dtype, ldw,
                                                 None if bias is None else bias.data_ptr(), weight.shape[0],
                                                 weight.shape[1], int(gate), segments, self.device,
                                                 _stream(self.device),
                                                 ctypes.byref(self._h)))
        self._info()
        return self

    def _info(self):
        vals = [ctypes.c_int() for _ in range(4)]
        check(lib().dn_linear8_info(self._h, *[ctypes.byref(v) for v in vals]))
        self.out_channels, self.in_channels = vals[0].value, vals[1].value
        self.gate, self.segments = bool(vals[2].value), vals[3].value
        self._need = {}  # workspace bytes of the sizes met

    def __reduce_ex__(self, protocol):  # two objects would destroy the one layer
        raise TypeError("a Linear8 cannot be copied or pickled: make another one of its weights")

    def close(self) -> None:
        h = getattr(self, "_h", None)
        if h:
            lib().dn_linear8_destroy(h)
        self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _workspace(self, rows: int, dtype: int, nchw: int = 0):
        """(address, bytes, tensor) of a call's workspace, from torch's
        allocator on the current stream, which keeps it from others until the
        stream is past the call."""
        need = self._need.get((rows, dtype, nchw))
        if need is None:
            n = ctypes.c_int64()
            check(lib().dn_linear8_workspace(self._h, rows, dtype, nchw, ctypes.byref(n)))
            if len(self._need) > 256:
                self._need.clear()
            need = self._need[rows, dtype, nchw] = n.value
        if need == 0:
            return None, 0, None
        t = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", self.device))
        return t.data_ptr(), need, t

    def forward(self, x, out=None, out_dtype=None, stream=None):
        """Token rows x (rows, in_channels), FP16 or FP32, any row stride that
        holds a row -> (rows, out_channels) in ``out_dtype`` (default: x's) or into
        ``out``, which may not share memory with x."""
        if _elsewhere(self.device, stream):
            with _on(self.device, stream):
                return self.forward(x, out, out_dtype)
        dtype = _code(x.dtype, "Linear8.forward")
        ldx = _matrix(x, None, self.in_channels, self.device, "Linear8.forward: x")
        rows = x.shape[0]
        if out is None:
            out = x.new_empty((rows, self.out_channels), dtype=out_dtype)
        code = _code(out.dtype, "Linear8.forward: out")
        ldo = _matrix(out, rows, self.out_channels, self.device, "Linear8.forward: out")
        ws, n, _keep = self._workspace(rows, dtype)
        check(lib().dn_linear8_forward(self._h, x.data_ptr(), dtype, ldx, rows, out.data_ptr(), code, ldo, ws, n,
                                       _stream(self.device)))
        return out

    __call__ = forward

    def forward_nchw(self, x, out=None, stream=None):
        """A 1x1 convolution: x (N, in_channels, H, W) FP16 contiguous ->
        (N, out_channels, H, W) FP16, a scale for every pixel; ``out`` may not
        share memory with x."""
        if _elsewhere(self.device, stream):
            with _on(self.device, stream):
                return self.forward_nchw(x, out)
        if x.dtype is not torch.float16:
            raise DenoiserError(DN_ERR_DTYPE, "Linear8.forward_nchw: expected FP16 input")
        _on_device(x, self.device, "Linear8.forward_nchw: x")
        if x.dim() != 4 or x.shape[1] != self.in_channels or not x.is_contiguous():
            _bad(f"Linear8.forward_nchw: x must be a contiguous (N, {self.in_channels}, H, W) tensor")
        n, _, h, w = x.shape
        shape = (n, self.out_channels, h, w)
        if out is None:
            out = torch.empty(shape, dtype=torch.float16, device=x.device)
        _on_device(out, self.device, "Linear8.forward_nchw: out")
        if out.dtype is not torch.float16 or tuple(out.shape) != shape or not out.is_contiguous():
            _bad(f"Linear8.forward_nchw: out must be a contiguous FP16 tensor {shape}")
        ws, nb, _keep = self._workspace(n * h * w, 1, 1)
        check(lib().dn_linear8_forward_nchw(self._h, x.data_ptr(), n, h, w, out.data_ptr(), ws, nb,
                                            _stream(self.device)))
        return out

    def forward_cached(self, cache: RowCache, pages, rows: int | None = None, out=None, out_dtype=None, stream=None):
        """Straight from an 8-bit cache: ``segments`` pages (ints) side by
        side, the first ``rows`` rows of each (default: all) -> (rows,
        out_channels) in ``out_dtype`` (default FP16) or into ``out``."""
        if _elsewhere(self.device, stream):
            with _on(self.device, stream):
                return self.forward_cached(cache, pages, rows, out, out_dtype)
        if cache.device != self.device:
            _bad("Linear8.forward_cached: cache and layer are on different devices")
        if cache.bits != 8 or cache.group != cache.cols:
            _bad("Linear8.forward_cached: an 8-bit cache with one scale a row is needed")
        if cache.cols * self.segments != self.in_channels:
            _bad(f"Linear8.forward_cached: {self.segments} segments of {cache.cols} columns for "
                 f"{self.in_channels} channels")
        if rows is None:
            rows = cache.page_rows
        if not 0 <= rows <= cache.page_rows:
            _bad(f"Linear8.forward_cached: {rows} rows of pages of {cache.page_rows}")
        if out is None:
            out = torch.empty(rows, self.out_channels, dtype=out_dtype or torch.float16, device=cache._codes.device)
        code = _code(out.dtype, "Linear8.forward_cached: out")
        ldo = _matrix(out, rows, self.out_channels, self.device, "Linear8.forward_cached: out")
        codes, ld, scales, cap = cache._held
        for p in pages:
            if not 0 <= p < cache.pages:  # ctypes would cut a number that 64 bits do not hold
                _bad(f"Linear8.forward_cached: page {p} of a cache of {cache.pages}")
        check(lib().dn_linear8_forward_cached(self._h, codes, ld, scales, cap, cache.page_rows,
                                              (ctypes.c_int64 * len(pages))(*pages), len(pages), rows, out.data_ptr(),
                                              code, ldo, _stream(self.device)))
        return out

    def sync(self, stream=None) -> None:
        """Synchronise the stream and raise if a kernel flagged a device error."""
        with _on(self.device, stream):
            check(lib().dn_linear8_sync(self._h, _stream(self.device)))

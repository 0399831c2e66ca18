"""``CoefCache``: the newest slices of a set of streams, held in 8 bits.

What ``SlicedCQT`` / ``SliceStream`` give per slice goes in with ``append``
(quantised as it is written, ``csrc/coefcache.cu``); ``window(n)`` gives the
last n slices of every stream back in the layout of ``SlicedCQT.fwd``, in 32 or
in 16 bits.  A slice takes 2.06 bytes a coefficient instead of 8.

    cache = CoefCache(sliced, (B, C), capacity=64)
    blocks, side = stream.fwd(chunk)          # one slice of every stream
    cache.append(blocks, side)
    past, past_side = cache.window(32, dtype=torch.bfloat16)
"""
import ctypes

import torch

from . import _native
from .engine import _cuda_device, _raw_stream_of

RUN = 16   # coefficients that share a scale
FORMATS = {"int8": (torch.int8, _native.CQT_CACHE_INT8),
           "e4m3": (torch.float8_e4m3fn, _native.CQT_CACHE_E4M3)}
_OUT = {torch.complex64: _native.CQT_F32, torch.float32: _native.CQT_F32,
        torch.bfloat16: _native.CQT_BF16, torch.float16: _native.CQT_F16}


def _layout(cqt):
    """the heap layout behind an OctCQT, TrainableCQT, SlicedCQT or the like"""
    for c in (cqt, getattr(cqt, "cqt", None), getattr(cqt, "_fused_cqt", None)):
        heap = getattr(c, "heap", None)
        if heap is not None:
            return heap
    raise TypeError(f"{type(cqt).__name__} has no coefficient layout (an OctCQT, TrainableCQT "
                    "or SlicedCQT is needed)")


class CoefCache:
    """Rings of ``capacity`` slices for ``lead`` streams.

    cqt: the transform that the coefficients come from; lead: the leading
    dimensions of its blocks, e.g. (B, C).  ``fmt`` is "int8" (steps of 1/127
    to 1/64 of the largest of 16 neighbours: the scale is a power of two) or
    "e4m3" (3 bits behind the leading one, down to about 2^-14 of it).  Slice k of a stream lies in slot k mod capacity.

    ``length`` (int64 [*lead], on the device) counts the slices that each
    stream has been given; ``codes`` [*lead, capacity, ncoef, 2] and ``scales``
    [*lead, capacity, ncoef / 16] are the store, in heap order.  A coefficient
    is code * scale; a value that is not finite is held, and read, as NaN.  To
    restore a store that was saved, copy into the three.

    No gradient flows through the cache.  Calls on one cache must be ordered on
    one stream at a time; all of them may be captured into a graph.
    """

    def __init__(self, cqt, lead, capacity, fmt="int8", device=None):
        heap = _layout(cqt)
        self.lead = (int(lead),) if isinstance(lead, int) else tuple(int(d) for d in lead)
        self.capacity = int(capacity)
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        if self.capacity < 1 or any(d < 0 for d in self.lead):
            raise ValueError(f"bad capacity {capacity} or lead {self.lead}")
        self.gspec = [(b, M) for b, M, _ in heap.gspec]
        self.ngroups = len(heap.groups)
        for b, M in self.gspec:
            if M < RUN or M & (M - 1):
                raise ValueError(f"band lengths must be powers of two from {RUN}, got {M}")
        if len(self.gspec) > 16:
            raise ValueError(f"at most 16 coefficient groups, got {len(self.gspec)}")
        self.ncoef = heap.ncoef
        self.fmt = fmt
        dt, self._format = FORMATS[fmt]
        self.dev = _cuda_device(device if device is not None else getattr(cqt, "device", None))
        self.rows = 1
        for d in self.lead:
            self.rows *= d
        store = (*self.lead, self.capacity)
        z = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=self.dev)  # noqa: E731
        self._codes = z(*store, self.ncoef, 2).view(dt)
        self._scales = z(*store, self.ncoef // RUN).fill_(1).view(torch.float8_e8m0fnu)
        self._length = torch.zeros(self.lead, dtype=torch.int64, device=self.dev)
        self._ws = z(max(4 * self.rows, 16))
        # the same storage, kept whatever is done to the public tensors: a captured
        # call addresses it
        self._own = [t.detach() for t in (self.codes, self.scales, self.length)]
        i32 = ctypes.c_int32 * len(self.gspec)
        self._bands, self._lens = i32(*[b for b, _ in self.gspec]), i32(*[M for _, M in self.gspec])
        self._desc = _native.CqtCache(
            self.codes.data_ptr(), self.scales.data_ptr(), self.length.data_ptr(),
            self._ws.data_ptr(), self.rows, self.capacity, self._format, len(self.gspec),
            ctypes.cast(self._bands, _native._i32p), ctypes.cast(self._lens, _native._i32p))

        mod = _native.torch_ops()   # the same calls from C++ (None: ctypes)
        self._h = None if mod is None else mod.CacheHandle(
            *[_native.fn_address(n) for n in ("cqt_cache_append", "cqt_cache_window",
                                              "cqt_last_error")],
            self.codes, self.scales, self.length, self._ws, self.capacity, self._format,
            [b for b, _ in self.gspec], [M for _, M in self.gspec], self.ngroups)

    @property
    def codes(self):
        return self._codes

    @property
    def scales(self):
        return self._scales

    @property
    def length(self):
        return self._length

    def nbytes(self):
        """bytes of the store"""
        return self.codes.numel() + self.scales.numel()

    def reset(self):
        """forget every slice (the store is not cleared: no call reads it)"""
        self.length.zero_()

    # ------------------------------------------------------------------ checks
    def _slices(self, blocks, side):
        """slices in (blocks, side), whose shapes must be those of SlicedCQT.fwd
        or of one slice"""
        if side is None:
            raise ValueError("the cache holds the DC and Nyquist blocks too: side is needed")
        blocks, side = list(blocks), list(side)
        if len(blocks) != self.ngroups or len(side) != len(self.gspec) - self.ngroups:
            raise ValueError(f"{self.ngroups} blocks and {len(self.gspec) - self.ngroups} side "
                             f"blocks are needed, got {len(blocks)} and {len(side)}")
        S = blocks[0].shape[-1] // self.gspec[0][1] if blocks[0].dim() else 0
        for k, (c, (b, M)) in enumerate(zip(blocks + side, self.gspec)):
            if not torch.is_tensor(c) or c.device != self.dev:
                raise ValueError(f"coefficients must be tensors on {self.dev}")
            if c.dtype != torch.complex64:
                raise TypeError(f"coefficients must be complex64, got {c.dtype}")
            shape = tuple(c.shape)
            want = [(*self.lead, b, S * M)] if k < self.ngroups else [(*self.lead, S, b, M)]
            if k >= self.ngroups and S == 1:
                want.append((*self.lead, b, M))
            if shape not in want:
                raise ValueError(f"coefficient group {k} must be {want[0]}, got {shape}")
        return blocks, side, S

    def _check_store(self):
        d = self._desc
        if [t.data_ptr() or None for t in (self.codes, self.scales, self.length)] != [
                d.codes, d.scales, d.length]:
            raise ValueError("the cache's codes, scales or length have another storage than they "
                             "were made with (copy into them instead)")

    def _numbers(self, t, name):
        if t is None:
            return None
        if not torch.is_tensor(t) or t.device != self.dev or t.dtype != torch.int64 \
                or tuple(t.shape) != self.lead:
            raise ValueError(f"{name} must be an int64 tensor {self.lead} on {self.dev}")
        return t.contiguous()

    # ------------------------------------------------------------------- calls
    def append(self, blocks, side, counts=None):
        """the slices of (blocks, side) -- blocks [*lead, b, S * M], side
        [*lead, S, 1, M], as ``SlicedCQT.fwd`` returns them, or one slice with
        side [*lead, 1, M] -- behind those that the streams have.  counts (int64
        [*lead] on the device): how many of the S slices each stream has
        (padded batches); the others are left out."""
        if side is not None:
            blocks, side = list(blocks), list(side)   # looked at more than once
        if self._h is not None and side is not None and self._h.append(blocks + side, counts):
            return
        blocks, side, S = self._slices(blocks, side)   # refuses what does not fit
        counts = self._numbers(counts, "counts")
        self._check_store()
        parts = (_native.CqtCachePart * len(self.gspec))()
        keep = []
        for k, (c, (b, M)) in enumerate(zip(blocks + side, self.gspec)):
            c = c.resolve_conj().resolve_neg()
            v = c.reshape(self.rows, b, S * M) if k < self.ngroups else c.reshape(self.rows, S, b, M)
            if (v.stride(-1) != 1 and v.shape[-1] > 1) or v.data_ptr() % 8:
                v = v.clone(memory_format=torch.contiguous_format)
            keep.append(v)
            if k < self.ngroups:
                parts[k] = _native.CqtCachePart(v.data_ptr(), v.stride(0), M, v.stride(1))
            else:
                parts[k] = _native.CqtCachePart(v.data_ptr(), v.stride(0), v.stride(1), v.stride(2))
        with torch.cuda.device(self.dev):
            _native._check(_native.lib().cqt_cache_append(
                ctypes.byref(self._desc), parts, S, counts.data_ptr() if counts is not None else None,
                _raw_stream_of(self.dev.index)), "cqt_cache_append")
        torch.autograd.graph.increment_version(
            [t for t in (self.codes, self.scales, self.length) if not t.is_inference()])

    def window(self, n, dtype=torch.complex64, end=None):
        """slices [end - n, end) of every stream as (blocks, side) in the layout
        of ``SlicedCQT.fwd``: blocks [*lead, b, n * M], side [*lead, n, 1, M].
        end (int64 [*lead] on the device) is the stream's length unless given.
        Slices before a stream's first one, behind its last one, or too old for
        the ring read as zeros.  dtype: complex64, or float32, bfloat16 or
        float16 for pairs (re, im) in one more dimension at the end."""
        n = int(n)
        if n < 0:
            raise ValueError(f"the window must not be negative, got {n}")
        if dtype not in _OUT:
            raise TypeError("dtype must be complex64, float32, bfloat16 or float16, "
                            f"got {dtype}")
        if self._h is not None:
            return self._h.window(n, dtype, _OUT[dtype], end)
        end = self._numbers(end, "end")
        self._check_store()
        cplx = dtype == torch.complex64
        tail = () if cplx else (2,)
        out = torch.empty((self.rows * n * self.ncoef, *tail), dtype=dtype, device=self.dev)
        parts = (_native.CqtCachePart * len(self.gspec))()
        sizes = [self.rows * n * b * M for b, M in self.gspec]
        views = []
        for k, (v, (b, M)) in enumerate(zip(out.split(sizes), self.gspec)):
            row = n * b * M
            if k < self.ngroups:
                parts[k] = _native.CqtCachePart(v.data_ptr(), row, M, n * M)
                views.append(v.view(*self.lead, b, n * M, *tail))
            else:
                parts[k] = _native.CqtCachePart(v.data_ptr(), row, b * M, M)
                views.append(v.view(*self.lead, n, b, M, *tail))
        with torch.cuda.device(self.dev):
            _native._check(_native.lib().cqt_cache_window(
                ctypes.byref(self._desc), parts, n, end.data_ptr() if end is not None else None,
                _OUT[dtype], _raw_stream_of(self.dev.index)), "cqt_cache_window")
        return views[:self.ngroups], views[self.ngroups:]

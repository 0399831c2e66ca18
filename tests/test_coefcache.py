"""CPU checks of CoefCache: refusals, the C entries' argument checks, the plain
model that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

import plain_cache as pc
from flash_cqt_b200 import CoefCache, OctCQT, _native


@pytest.fixture(scope="module")
def cqt():
    return OctCQT([3, 4, 2], [8, 16, 32], fs=44100, audio_len=65536)


def test_constructor_refuses(cqt):
    with pytest.raises(ValueError, match="fmt"):
        CoefCache(cqt, (2,), 4, fmt="int4")
    for cap in (0, -1):
        with pytest.raises(ValueError, match="capacity"):
            CoefCache(cqt, (2,), cap)
    with pytest.raises(ValueError, match="lead"):
        CoefCache(cqt, (2, -1), 4)
    with pytest.raises(TypeError, match="layout"):
        CoefCache(object(), (2,), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        CoefCache(cqt, (2,), 4, device="cpu")


@pytest.fixture
def shell(cqt):
    """a cache without its store, for the argument checks"""
    c = CoefCache.__new__(CoefCache)
    c.lead, c.rows, c.capacity, c.dev = (2, 1), 2, 4, torch.device("cpu")
    c.gspec = [(b, M) for b, M, _ in cqt.heap.gspec]
    c.ngroups, c.ncoef = 9, cqt.heap.ncoef
    return c


def blocks_of(c, S, dtype=torch.complex64):
    out = [torch.zeros(*c.lead, b, S * M, dtype=dtype) for b, M in c.gspec[:9]]
    side = [torch.zeros(*c.lead, S, b, M, dtype=dtype) for b, M in c.gspec[9:]]
    return out, side


def test_shapes(shell):
    c = shell
    for S in (0, 1, 3):
        assert c._slices(*blocks_of(c, S))[2] == S
    b, s = blocks_of(c, 1)
    assert c._slices(b, [x[:, :, 0] for x in s])[2] == 1
    with pytest.raises(ValueError, match="side is needed"):
        c._slices(b, None)
    with pytest.raises(ValueError, match="9 blocks"):
        c._slices(b[:-1], s)
    with pytest.raises(TypeError, match="complex64"):
        c._slices(*blocks_of(c, 1, torch.complex128))
    b[3] = b[3][..., :-1]
    with pytest.raises(ValueError, match="group 3"):
        c._slices(b, s)
    b, s = blocks_of(c, 2)
    with pytest.raises(ValueError, match="group 9"):
        c._slices(b, [x[:, :, :1] for x in s])
    with pytest.raises(ValueError, match="tensors"):
        c._slices([b[0].to("meta")] + b[1:], s)


def test_numbers(shell):
    c = shell
    assert c._numbers(None, "counts") is None
    c._numbers(torch.zeros(2, 1, dtype=torch.int64), "counts")
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(2, 1), [1, 2],
                torch.zeros(2, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="counts"):
            c._numbers(bad, "counts")
    with pytest.raises(ValueError, match="negative"):
        c.window(-1)
    with pytest.raises(TypeError, match="dtype"):
        c.window(1, dtype=torch.float64)


def test_c_entries_refuse():
    L = _native.lib()
    i32 = ctypes.c_int32 * 2
    bands, lens = i32(2, 1), i32(32, 16)
    ptr = lambda a: ctypes.cast(a, ctypes.POINTER(ctypes.c_int32))  # noqa: E731

    def call(slices=1, parts=((64, 80, 32, 32), (64, 80, 16, 16)), name="append", dtype=0, **kw):
        c = _native.CqtCache(64, 64, 64, 64, 1, 4, 0, 2, ptr(bands), ptr(lens))
        for k, v in kw.items():
            setattr(c, k, v)
        p = (_native.CqtCachePart * 2)(*(_native.CqtCachePart(*x) for x in parts))
        rc = L.cqt_cache_append(ctypes.byref(c), p, slices, None, None) if name == "append" else \
            L.cqt_cache_window(ctypes.byref(c), p, slices, None, dtype, None)
        return rc, L.cqt_last_error().decode()

    # addresses that are never read: every call is refused on the host
    assert L.cqt_cache_append(None, None, 1, None, None) == -1
    for bad in (dict(rows=-1), dict(capacity=0), dict(slices=-1), dict(format=2), dict(ngroups=0),
                dict(ngroups=17), dict(group_len=None), dict(workspace=None), dict(workspace=72),
                dict(codes=None), dict(codes=72), dict(scales=None), dict(length=None),
                dict(length=68), dict(group_len=ptr(i32(32, 8))), dict(group_len=ptr(i32(32, 24))),
                dict(group_count=ptr(i32(0, 1))), dict(group_count=ptr(i32(513, 1))),
                dict(parts=((None, 80, 32, 32), (64, 80, 16, 16))),
                dict(parts=((68, 80, 32, 32), (64, 80, 16, 16))),
                dict(slices=2 ** 31 - 1, rows=2 ** 20)):
        for name in ("append", "window"):
            rc, msg = call(name=name, **bad)
            assert rc == -1 and msg, (name, bad)
    assert call(name="window", dtype=3)[1] == "unknown output type"
    for parts in (((72, 80, 32, 32), (64, 80, 16, 16)), ((64, 81, 32, 32), (64, 80, 16, 16))):
        assert "16-byte" in call(name="window", parts=parts)[1]
    # no slices, no streams: no work
    assert call(slices=0)[0] == 0 and call(rows=0)[0] == 0
    assert call(slices=0, name="window")[0] == 0 and call(rows=0, name="window")[0] == 0


@pytest.mark.parametrize("fmt, top", [("int8", 127.0), ("e4m3", 448.0)])
def test_plain_quantiser(fmt, top):
    """within half a step, the largest value is kept to a step, scales least"""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 64)) * np.exp(3 * rng.standard_normal((50, 1)))).astype(np.float32)
    x[3] = 0
    c, s = pc.quantise(x, fmt)
    sc = np.repeat(s, pc.RUN, axis=1)
    assert np.abs(c).max() <= top
    peak = np.abs(x).reshape(50, 2, 32).max(-1)
    assert np.all((peak <= top * s) & ((peak > top * s / 2) | (peak == 0)))
    y = np.abs(x) / sc
    step = np.ones_like(y) if fmt == "int8" else np.exp2(np.maximum(np.frexp(y)[1] - 4, -9.0))
    assert np.all(np.abs(c - x / sc) <= step / 2)
    if fmt == "e4m3":   # torch's conversion agrees with the arithmetic
        t = torch.tensor(x / sc).to(torch.float8_e4m3fn).double().numpy()
        assert np.array_equal(t, c)


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("what", ["codes", "scales", "length"])
def test_exchanged_store_is_refused(cqt, monkeypatch, what, python):
    """kernels address the store that the cache was made with"""
    import flash_cqt_b200.coefcache as module
    monkeypatch.setattr(module, "_cuda_device", lambda d: torch.device("cpu"))
    if python:
        monkeypatch.setattr(_native, "_torchops", None)
        monkeypatch.setattr(_native, "_torchops_tried", True)
    c = CoefCache(cqt, (2, 1), 3)
    with pytest.raises(AttributeError):
        setattr(c, what, torch.zeros(1))
    t = getattr(c, what)
    t.data = t.data.clone()
    with pytest.raises(ValueError, match="another storage"):
        c.append(*blocks_of(c, 1))
    with pytest.raises(ValueError, match="another storage"):
        c.window(1)
    assert CoefCache(cqt, (0,), 3).codes.numel() == 0


def test_blocks_from_an_iterator(cqt, monkeypatch):
    """any iterable of blocks, also where the fast path leaves them to the other"""
    import flash_cqt_b200.coefcache as module
    monkeypatch.setattr(module, "_cuda_device", lambda d: torch.device("cpu"))
    c = CoefCache(cqt, (2, 1), 3)
    b, s = blocks_of(c, 1)
    b[3] = b[3][..., :-1]
    with pytest.raises(ValueError, match="group 3"):
        c.append(iter(b), (x for x in s))
    with pytest.raises(ValueError, match="side is needed"):
        c.append(iter(b), None)

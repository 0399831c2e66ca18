"""CoefCache on the GPU: codes, scales and what is read back equal the plain
model exactly (a value is rounded once, by arithmetic that both do exactly)."""
import numpy as np
import pytest
import torch

import plain_cache as pc
from flash_cqt_b200 import CoefCache, OctCQT, SlicedCQT

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def banks():
    return {"default": OctCQT([3, 4, 2], [8, 16, 32], fs=44100, audio_len=65536),
            "short": OctCQT([3, 4, 2], [8, 16, 32], fs=44100, audio_len=32768),
            "other": OctCQT([2, 2, 2, 3], [8, 12, 16, 32], fs=44100, audio_len=65536)}


def heaps(rows, S, ncoef, seed):
    """complex64 [rows, S, ncoef]: three decades, silence, extremes"""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, S, ncoef // 16, 32)) * np.exp(
        2.5 * rng.standard_normal((rows, S, ncoef // 16, 1)))
    x[..., ::7, :] = 0
    return np.ascontiguousarray(x.astype(np.float32)).reshape(rows, S, 2 * ncoef).view(np.complex64)


def to_blocks(h, cqt, lead):
    """[rows, S, ncoef] -> (blocks, side) in SlicedCQT.fwd's layout"""
    S = h.shape[1]
    h = torch.from_numpy(h).to(DEV)
    out = []
    for k, (b, M, off) in enumerate(cqt.heap.gspec):
        x = h[:, :, off:off + b * M].reshape(h.shape[0], S, b, M)
        if k < len(cqt.heap.groups):
            out.append(x.permute(0, 2, 1, 3).reshape(*lead, b, S * M))
        else:
            out.append(x.reshape(*lead, S, b, M))
    n = len(cqt.heap.groups)
    return out[:n], out[n:]


def from_blocks(blocks, side, cqt, S):
    """the way back, as float64 [rows, S, ncoef, 2]"""
    out = []
    rows = int(np.prod(blocks[0].shape[:-2 if blocks[0].is_complex() else -3]))
    for k, (c, (b, M, _)) in enumerate(zip(list(blocks) + list(side), cqt.heap.gspec)):
        x = torch.view_as_real(c) if c.is_complex() else c
        x = x.double()
        if k < len(cqt.heap.groups):
            x = x.reshape(rows, b, S, M, 2).permute(0, 2, 1, 3, 4)
        out.append(x.reshape(rows, S, b * M, 2))
    return torch.cat(out, 2).cpu().numpy()


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def check_store(cache, ring):
    c = cache.codes.double().cpu().numpy().reshape(ring.codes.shape)
    if cache.fmt == "int8":
        c = np.where(c == -128, np.nan, c)
    assert same(c, ring.codes)
    assert same(cache.scales.double().cpu().numpy().reshape(ring.scales.shape), ring.scales)
    assert same(cache.length.cpu().numpy().reshape(-1), ring.length)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bank", ["default", "short", "other"])
def test_append_and_window(banks, bank, fmt):
    cqt = banks[bank]
    nc = cqt.heap.ncoef
    cache = CoefCache(cqt, (3, 1), 5, fmt=fmt, device=DEV)
    ring = pc.Ring(3, 5, nc, fmt)
    for k, (S, counts) in enumerate([(1, None), (2, [2, 0, 1]), (3, [-4, 3, 99]), (0, None),
                                     (4, None), (9, [9, 7, 1])]):
        h = heaps(3, S, nc, seed=k)
        ring.append(h, counts)
        c = None if counts is None else torch.tensor(counts, device=DEV)[:, None]
        cache.append(*to_blocks(h, cqt, (3, 1)), c)
        check_store(cache, ring)
    for n in (0, 1, 4, 5, 8, 30):
        for dt in (torch.complex64, torch.float32):
            got = from_blocks(*cache.window(n, dtype=dt), cqt, n)
            assert same(got, ring.window(n))
        # bf16 holds every code, float16 rounds once
        got = from_blocks(*cache.window(n, dtype=torch.bfloat16), cqt, n)
        assert same(got, ring.window(n))
        got = from_blocks(*cache.window(n, dtype=torch.float16), cqt, n)
        with np.errstate(over="ignore"):
            assert same(got, ring.window(n).astype(np.float32).astype(np.float16).astype(np.float64))
    for end in ([0, 0, 0], [3, 14, 4], [18, -5, 10 ** 12], [14, 15, 16]):
        e = torch.tensor(end, device=DEV)[:, None]
        got = from_blocks(*cache.window(6, end=e), cqt, 6)
        assert same(got, ring.window(6, end))


def test_python_path(banks, monkeypatch):
    """the calls through ctypes, as where the torch fast path is not built"""
    from flash_cqt_b200 import _native
    monkeypatch.setattr(_native, "_torchops", None)
    monkeypatch.setattr(_native, "_torchops_tried", True)
    test_append_and_window(banks, "short", "int8")
    test_append_and_window(banks, "short", "e4m3")
    test_views_and_orders(banks)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_special_values(banks, fmt):
    """not finite, tiny, huge, exact borders and ties"""
    cqt = banks["short"]
    nc = cqt.heap.ncoef
    x = heaps(1, 2, nc, seed=9).view(np.float32).reshape(2, -1, 32)
    x[0, 0, 3], x[0, 0, 4], x[0, 1, 31] = np.nan, np.inf, -np.inf
    x[0, 2] = np.nan
    x[0, 3] = 1e-42                       # subnormal: under the least scale's steps
    x[0, 4, 0] = 3.4e38
    x[0, 5] = 2.0 ** -126 * np.arange(32)
    for i, top in enumerate((127.0, 127.5, 128.0, 448.0, 449.0, 447.99997, 1.0)):
        x[1, 2 * i] = np.linspace(-1, 1, 32) * top
        x[1, 2 * i, 5] = top
        x[1, 2 * i + 1] = np.arange(32) / 2.0 - 8     # ties at half a step
        x[1, 2 * i + 1, 0] = top
    x[1, 20] = -0.0
    h = np.ascontiguousarray(x.reshape(1, 2, -1)).view(np.complex64)
    cache, ring = CoefCache(cqt, (1,), 2, fmt=fmt, device=DEV), pc.Ring(1, 2, nc, fmt)
    cache.append(*to_blocks(h, cqt, (1,)))
    ring.append(h)
    check_store(cache, ring)
    assert same(from_blocks(*cache.window(2), cqt, 2), ring.window(2))
    assert np.isnan(ring.window(2)).sum() == 35


def test_views_and_orders(banks):
    """inputs that are views: channels last, slices of longer blocks, lazily
    conjugated, at places that are not 16-byte aligned"""
    cqt = banks["short"]
    nc = cqt.heap.ncoef
    h = heaps(2, 3, nc, seed=3)
    blocks, side = to_blocks(h, cqt, (2,))
    ring = pc.Ring(2, 4, nc, "int8")
    ring.append(h)
    longer = [torch.cat([torch.zeros_like(b[..., :1]), b], -1)[..., 1:] for b in blocks]
    assert all(b.data_ptr() % 16 == 8 for b in longer)
    swapped = [b.transpose(1, 2).contiguous().transpose(1, 2) for b in blocks]
    lazy = [b.conj().resolve_conj().conj() for b in blocks]
    negated = [torch._neg_view(-b) for b in blocks]
    rows = [torch.stack([b, b], 1)[:, 1] for b in blocks]
    assert negated[0].is_neg()
    for v in (longer, swapped, lazy, negated, rows):
        cache = CoefCache(cqt, (2,), 4, device=DEV)
        cache.append(v, [s.transpose(0, 1).contiguous().transpose(0, 1) for s in side])
        check_store(cache, ring)
    assert lazy[0].is_conj()


@pytest.mark.parametrize("lead", [(), (0,), (2, 0), (3,), (2, 1, 2)])
def test_leading_dimensions(banks, lead):
    """no dimensions, no streams, several dimensions"""
    cqt = banks["short"]
    rows = int(np.prod(lead))
    cache, ring = CoefCache(cqt, lead, 2, device=DEV), pc.Ring(rows, 2, cqt.heap.ncoef, "int8")
    for seed in range(3):
        h = heaps(rows, 1, cqt.heap.ncoef, seed)
        cache.append(*to_blocks(h, cqt, lead))
        ring.append(h)
    check_store(cache, ring)
    b, s = cache.window(3)
    assert b[0].shape[:len(lead)] == lead and s[0].shape[len(lead)] == 3
    assert same(from_blocks(b, s, cqt, 3), ring.window(3))


def test_many_slices_and_streams(banks):
    """more streams, and more slices, than a grid's extents hold"""
    cqt = banks["short"]
    nc = cqt.heap.ncoef
    h = heaps(1, 1, nc, 0)
    b, s = to_blocks(h, cqt, (1,))
    rows = 65537
    cache = CoefCache(cqt, (rows,), 1, device=DEV)
    cache.append([x.expand(rows, *x.shape[1:]) for x in b], [x.expand(rows, *x.shape[1:]) for x in s])
    assert (cache.length == 1).all()
    assert torch.equal(cache.codes[0], cache.codes[rows - 1])
    assert (cache.codes[::8191] == cache.codes[:1]).all()
    ring = pc.Ring(1, 1, nc, "int8")
    ring.append(h)
    assert same(cache.codes[rows - 1].double().cpu().numpy().reshape(1, 1, -1), ring.codes)
    # a window far longer than the ring: zeros but for its end
    one = CoefCache(cqt, (1,), 1, device=DEV)
    one.append(b, s)
    blocks, _ = one.window(65540, dtype=torch.bfloat16)
    M = cqt.heap.gspec[0][1]
    assert same(blocks[0][0, 0, -M:].double().cpu().numpy(), ring.window(1)[0, 0, :M])
    assert not blocks[0][0, 0, :-M].any() and not blocks[5][0, :, :M].any()


def test_rows_left_alone(banks):
    """no call touches the slots of slices that it does not bring"""
    cqt = banks["short"]
    nc = cqt.heap.ncoef
    cache = CoefCache(cqt, (3,), 6, device=DEV)
    cache.codes.random_(-127, 128)
    cache.scales.view(torch.uint8).random_(100, 140)
    codes, scales = cache.codes.clone(), cache.scales.view(torch.uint8).clone()
    cache.length.copy_(torch.tensor([4, 5, 6]))
    cache.append(*to_blocks(heaps(3, 3, nc, seed=1), cqt, (3,)), torch.tensor([0, 1, 3], device=DEV))
    touched = torch.zeros(3, 6, dtype=torch.bool, device=DEV)
    touched[1, 5] = touched[2, 0] = touched[2, 1] = touched[2, 2] = True
    assert torch.equal(cache.codes[~touched], codes[~touched])
    assert torch.equal(cache.scales.view(torch.uint8)[~touched], scales[~touched])
    assert (cache.codes[touched] != codes[touched]).any(-1).any(-1).all()


def test_far_offsets(banks):
    """a store over 4 GB and slice numbers beyond 32 bits"""
    cqt = banks["default"]
    nc = cqt.heap.ncoef
    cap = 16200
    assert cap * nc * 2 > 2 ** 32
    cache = CoefCache(cqt, (1,), cap, device=DEV)
    h = heaps(1, 3, nc, seed=5)
    for start in (cap - 1, 5 * 2 ** 32 + cap - 2 - (5 * 2 ** 32) % cap):
        cache.length.fill_(start)
        cache.append(*to_blocks(h, cqt, (1,)))
        ring = pc.Ring(1, 3, nc, "int8")
        ring.append(h)
        assert same(from_blocks(*cache.window(3), cqt, 3), ring.window(3))
        for k in range(3):
            slot = (start + k) % cap
            c = cache.codes[0, slot].double().cpu().numpy().reshape(-1)
            assert same(c, ring.codes[0, k])
    cache.length.fill_(-3)   # no such length: counted from 0
    cache.append(*to_blocks(h, cqt, (1,)))
    assert int(cache.length) == 3


def test_capture_and_streams(banks):
    """two captured graphs over one cache, replayed in turn, and a side stream"""
    cqt = banks["short"]
    nc = cqt.heap.ncoef
    h = [heaps(2, 1, nc, seed=s) for s in range(5)]
    a, ring = CoefCache(cqt, (2,), 3, device=DEV), pc.Ring(2, 3, nc, "int8")
    src = to_blocks(h[0], cqt, (2,))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    a.append(*src)
    a.window(3)
    a.reset()
    with torch.cuda.graph(g1):
        a.append(*src)
    with torch.cuda.graph(g2):
        out = a.window(3, dtype=torch.bfloat16)
    for x in h:
        for d, s in zip(src[0] + src[1], sum(to_blocks(x, cqt, (2,)), [])):
            d.copy_(s)
        g1.replay()
        g2.replay()
        ring.append(x)
        assert same(from_blocks(*out, cqt, 3), ring.window(3))
    check_store(a, ring)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.append(*src)
        got = a.window(2)
    torch.cuda.current_stream().wait_stream(s)
    ring.append(h[-1])
    assert same(from_blocks(*got, cqt, 2), ring.window(2))


def test_signal_through_the_cache():
    """analysis -> cache -> synthesis: what comes back differs from the signal
    by the quantisation, each value's error at most half a step of its run"""
    sl = SlicedCQT([3, 4, 2], [8, 16, 32], fs=44100, sl_len=32768, device=DEV)
    x = torch.randn(2, 1, 70000, device=DEV)
    blocks, side = sl.fwd(x)
    S = side[0].shape[2]
    for fmt in ("int8", "e4m3"):
        cache = CoefCache(sl, (2, 1), S, fmt=fmt)
        cache.append(blocks, side)
        b2, s2 = cache.window(S)
        for p, q in zip(list(blocks) + list(side), list(b2) + list(s2)):
            assert p.shape == q.shape
            r = lambda c: torch.view_as_real(c).reshape(-1, 32)  # noqa: E731
            top = r(p).abs().amax(-1, keepdim=True)
            # int8: half of a step of top / 63.5 at the most; e4m3: 2^-4 of it
            assert ((r(q) - r(p)).abs() <= top * (1 / 127 if fmt == "int8" else 1 / 16)).all()
        y = sl.bwd(b2, s2, length=70000)
        assert y.shape == x.shape and torch.isfinite(y).all()


def test_refusals(banks):
    cqt = banks["short"]
    cache = CoefCache(cqt, (2,), 3, device=DEV)
    blocks, side = to_blocks(heaps(2, 1, cqt.heap.ncoef, 0), cqt, (2,))
    with pytest.raises(ValueError, match="tensors on"):
        cache.append([b.cpu() for b in blocks], side)
    with pytest.raises(ValueError, match="counts"):
        cache.append(blocks, side, torch.ones(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="end"):
        cache.window(1, end=torch.ones(1, dtype=torch.int64, device=DEV))
    assert int(cache.length.sum()) == 0


@pytest.mark.parametrize("python", [False, True])
def test_store_is_restored_by_copying(banks, python, monkeypatch):
    """what was saved is copied into another cache; other storage is refused, and
    a captured call goes on with the cache's own"""
    if python:
        from flash_cqt_b200 import _native
        monkeypatch.setattr(_native, "_torchops", None)
        monkeypatch.setattr(_native, "_torchops_tried", True)
    cqt = banks["short"]
    a, b = (CoefCache(cqt, (2,), 3, device=DEV) for _ in range(2))
    src = to_blocks(heaps(2, 2, cqt.heap.ncoef, seed=6), cqt, (2,))
    a.append(*src)
    for k in ("codes", "scales", "length"):
        x, y = getattr(a, k), getattr(b, k)
        y.copy_(x)
    want = from_blocks(*a.window(3), cqt, 3)
    assert same(from_blocks(*b.window(3), cqt, 3), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.window(3)
    keep = b.codes.data
    b.codes.data = torch.zeros_like(keep)
    with pytest.raises(ValueError, match="another storage"):
        b.window(3)
    with pytest.raises(ValueError, match="another storage"):
        b.append(*src)
    del keep
    torch.cuda.synchronize()
    graph.replay()
    assert same(from_blocks(*out, cqt, 3), want)


@pytest.mark.parametrize("python", [False, True])
def test_append_is_seen_by_autograd(banks, python, monkeypatch):
    """a backward pass through a store that has been appended to is refused"""
    if python:
        from flash_cqt_b200 import _native
        monkeypatch.setattr(_native, "_torchops", None)
        monkeypatch.setattr(_native, "_torchops_tried", True)
    cqt = banks["short"]
    cache = CoefCache(cqt, (2,), 3, device=DEV)
    src = to_blocks(heaps(2, 1, cqt.heap.ncoef, seed=7), cqt, (2,))
    cache.append(*src)
    w = torch.ones(5, device=DEV, requires_grad=True)
    y = w[cache.length].sum()          # the index is saved
    cache.window(2)                    # (reading changes nothing)
    y.backward()
    assert w.grad.tolist() == [0, 2, 0, 0, 0]
    y = w[cache.length].sum()
    versions = [t._version for t in (cache.codes, cache.scales, cache.length)]
    cache.append(*src)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    assert all(t._version > v for t, v in zip((cache.codes, cache.scales, cache.length), versions))


def test_lazy_views_from_an_iterator(banks):
    """what the fast path does not take is appended all the same"""
    cqt = banks["short"]
    h = heaps(2, 1, cqt.heap.ncoef, seed=8)
    blocks, side = to_blocks(h, cqt, (2,))
    cache, ring = CoefCache(cqt, (2,), 2, device=DEV), pc.Ring(2, 2, cqt.heap.ncoef, "int8")
    cache.append((b.conj().resolve_conj().conj() for b in blocks), iter(side))
    ring.append(h)
    check_store(cache, ring)

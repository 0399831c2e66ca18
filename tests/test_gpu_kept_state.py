"""The optimizer and the coefficient cache together with the transform, as a
streaming or training program uses them."""
import numpy as np
import pytest
import torch

import plain_cache as pc
from flash_cqt_b200 import AdamW, CoefCache, SlicedCQT
from test_gpu_coefcache import from_blocks, same
from test_gpu_optim import check_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def sliced():
    return SlicedCQT([3, 4, 2], [8, 16, 32], fs=44100, sl_len=32768, device=DEV)


def heap_of(blocks, side, cqt, S):
    """SlicedCQT's (blocks, side) as complex64 [rows, S, ncoef]"""
    x = from_blocks(blocks, side, cqt, S).astype(np.float32)
    return np.ascontiguousarray(x).view(np.complex64)[..., 0]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_stream_history(sliced, fmt):
    """every hop's slice is in the history; a new stream starts an empty one"""
    cqt, hop, n = sliced.cqt, sliced.hop, 5
    st = sliced.streamer((2, 1), history=4, history_format=fmt)
    for seed in (0, 1):
        torch.manual_seed(seed)
        x = torch.randn(2, 1, hop * n, device=DEV)
        whole = sliced.fwd(x)
        S = whole[1][0].shape[2]
        h = heap_of(*whole, cqt, S)
        ring = pc.Ring(2, 4, cqt.heap.ncoef, fmt)
        assert same(from_blocks(*st.past(3), cqt, 3), ring.window(3))   # none yet: zeros
        for k in range(S):
            got = st.fwd(x[..., k * hop:(k + 1) * hop]) if k < n else st.flush()
            ring.append(h[:, k:k + 1])
            # the slice itself is what it is without a history
            assert same(heap_of(*got, cqt, 1), h[:, k:k + 1])
            for dt in (torch.complex64, torch.bfloat16):
                assert same(from_blocks(*st.past(4, dtype=dt), cqt, 4), ring.window(4))
        assert st.cache.length.flatten().tolist() == [S, S]
        st.reset()
    with pytest.raises(RuntimeError, match="no history"):
        sliced.streamer((1, 1)).past(1)
    with pytest.raises(ValueError, match="history"):
        sliced.streamer((1, 1), history=-1)


def test_history_changes_no_coefficient(sliced):
    a, b = sliced.streamer((1, 2)), sliced.streamer((1, 2), history=2)
    torch.manual_seed(2)
    for _ in range(4):
        chunk = torch.randn(1, 2, sliced.hop, device=DEV)
        for p, q in zip(sum(a.fwd(chunk), []), sum(b.fwd(chunk), [])):
            assert torch.equal(torch.view_as_real(p), torch.view_as_real(q))


@pytest.mark.parametrize("bits", [32, 8])
def test_training_on_a_cache(sliced, bits):
    """batches that were written once are read back, weighted by learned gains
    and synthesised; each step moves the gains as the formulas say, and the
    gradient agrees with differences of the loss"""
    torch.manual_seed(3)
    cqt = sliced.cqt
    L = 4 * sliced.hop
    x = torch.randn(2, 1, L, device=DEV)
    blocks, side = sliced.fwd(x)
    S = side[0].shape[2]
    cache = CoefCache(sliced, (2, 1), S)
    cache.append(blocks, side)
    target = 0.5 * x
    gains = [torch.ones(b, 1, device=DEV, requires_grad=True) for b, _, _ in cqt.heap.gspec]
    opt = AdamW(gains, lr=1e-2, weight_decay=0.0, state_bits=bits, max_norm=0.05)

    def loss_of():
        b, s = cache.window(S)
        n = len(b)
        y = sliced.bwd([c * g for c, g in zip(b, gains)],
                       [c * g for c, g in zip(s, gains[n:])], length=L)
        return (y - target).square().mean()
    kw = dict(lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=0.0)
    for step in (1, 2, 3):
        opt.zero_grad()
        loss_of().backward()
        check_step(opt, gains, step, kw, bits, max_norm=0.05)
    opt.zero_grad()
    loss_of().backward()
    g, h = gains[7], 0.25
    k = int(g.grad.abs().argmax())
    with torch.no_grad():
        g[k] += h
        hi = float(loss_of())
        g[k] -= 2 * h
        lo = float(loss_of())
        g[k] += h
    # the loss is quadratic in one gain: the difference is exact up to the
    # rounding of the two means (of 131072 squares: a few steps of float32)
    assert abs((hi - lo) / (2 * h) - float(g.grad[k])) <= 8 * 2.0 ** -23 * max(hi, lo) / (2 * h)


def test_whole_step_in_a_graph(sliced):
    """window, synthesis, loss, gradients and step captured once and replayed
    give the bits of the same steps run one by one"""
    cqt = sliced.cqt
    L = 2 * sliced.hop
    torch.manual_seed(4)
    x = torch.randn(1, 1, L, device=DEV)

    def setup():
        cache = CoefCache(sliced, (1, 1), 4)
        cache.append(*sliced.fwd(x))
        gains = [torch.ones(b, 1, device=DEV, requires_grad=True) for b, _, _ in cqt.heap.gspec]
        opt = AdamW(gains, lr=1e-2, state_bits=8, max_norm=0.05)
        opt.init_state()

        def step():
            b, s = cache.window(3)
            n = len(b)
            y = sliced.bwd([c * g for c, g in zip(b, gains)],
                           [c * g for c, g in zip(s, gains[n:])], length=L)
            for g, d in zip(gains, torch.autograd.grad((y - 0.5 * x).square().mean(), gains)):
                g.grad = d
            opt.step()
        return gains, opt, step
    gains, _, step = setup()
    for _ in range(4):
        step()
    want = [g.detach().clone() for g in gains]
    gains, opt, step = setup()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()   # the first one eagerly (it also warms the engines up)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        graph.replay()
    for g, w in zip(gains, want):
        assert torch.equal(g.detach(), w)
    assert int(opt.state[gains[0]]["step"]) == 4


def test_history_is_the_streams_own(sliced):
    """the graphs write to the cache that they were captured with"""
    st = sliced.streamer((1, 1), history=2)
    with pytest.raises(AttributeError):
        st.cache = CoefCache(sliced, (1, 1), 2)
    assert sliced.streamer((1, 1)).cache is None
    x = torch.randn(1, 1, sliced.hop, device=DEV)
    st.fwd(x)
    assert int(st.cache.length) == 1 and st.past(1)[0][0].abs().max() > 0

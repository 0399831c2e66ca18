"""AdamW's step on the GPU against the formulas in 64 bits.

Tolerances: tests/plain_optim.py counts the roundings of each output; 16-bit
parameters are rounded once more, by half a step of their type."""
import copy
import gc
import weakref

import numpy as np
import pytest
import torch

import plain_optim as po
from flash_cqt_b200 import AdamW, OctCQT, TrainableCQT

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
        torch.complex64: 0.0}


def flat(t):
    """a tensor's real elements in memory order, float64 on the host"""
    t = t.detach()
    if t.is_complex():
        t = torch.view_as_real(t)
    order = sorted(range(t.dim()), key=lambda d: (-t.stride(d), -t.shape[d]))
    return t.permute(order).reshape(-1).to(torch.float64).cpu().numpy()


def make(shapes, seed=0, grad_scale=0.1):
    """[(shape, dtype)] -> leaves with gradients"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    ps = []
    for shape, dt in shapes:
        real = (*shape, 2) if dt == torch.complex64 else shape
        x, y = (torch.randn(real, generator=g, device=DEV) for _ in range(2))
        if dt == torch.complex64:
            x, y = torch.view_as_complex(x), torch.view_as_complex(y)
        p = x.to(dt).requires_grad_()
        p.grad = (grad_scale * y).to(dt)
        ps.append(p)
    return ps


def values8(s, k):
    """an 8-bit moment's values"""
    c = s[k].double().cpu().numpy()
    return c * po.spread(s[k + "_scale"].double().cpu().numpy(), c.size)


def check_step(opt, ps, t, kw, bits=32, master=False, max_norm=None, seed=0):
    """one step of `opt`, compared with the formulas from the state before it"""
    def state(p):
        s = opt.state.get(p) or {}
        if not s:
            z = np.zeros(flat(p).size)
            return flat(p), z, z
        q = flat(s["master"]) if "master" in s else flat(p)
        return (q, values8(s, "exp_avg"), values8(s, "exp_avg_sq")) if bits == 8 else \
            (q, flat(s["exp_avg"]), flat(s["exp_avg_sq"]))
    before = [state(p) for p in ps]
    grads = [flat(p.grad) for p in ps]
    clip = 1.0
    if max_norm is not None:
        norm = np.sqrt(sum((g ** 2).sum() for g in grads))
        clip = min(1.0, max_norm / (norm + 1e-6))
    opt.step()
    torch.cuda.synchronize()
    if max_norm is not None:
        # summed in 64 bits, rounded once
        assert abs(float(opt.grad_norm) - norm) <= norm * (po.U + 1e-12)
    for i, (p, g, (q, m, v)) in enumerate(zip(ps, grads, before)):
        s = opt.state[p]
        p1, m1, v1, (ep, em, ev) = po.step(q, g, m, v, t, clip=clip, **kw)
        half = HALF[p.dtype]
        small = 2.0 ** -25 if p.dtype == torch.float16 else 0.0   # fp16's own subnormals
        assert np.all(np.abs(flat(p) - p1) <= ep + half * (np.abs(p1) + ep) + small), i
        if master and half:
            assert np.all(np.abs(flat(s["master"]) - p1) <= ep), i
            assert torch.equal(p.detach(), s["master"].to(p.dtype)), i
        assert int(s["step"]) == t
        if bits == 32:
            assert np.all(np.abs(flat(s["exp_avg"]) - m1) <= em), i
            assert np.all(np.abs(flat(s["exp_avg_sq"]) - v1) <= ev), i
            continue
        h = po.noise(seed, t, i, m1.size)
        for k, x, e, top, rnd in (("exp_avg", m1, em, 448.0, po.round_m),
                                  ("exp_avg_sq", v1, ev, 57344.0, po.round_v)):
            sc = s[k + "_scale"].double().cpu().numpy()
            lo, hi = (po.scales(np.abs(x) + d * e, top) for d in (-1, 1))
            assert np.all((lo <= sc) & (sc <= hi)), (i, k)
            # rounding with the same noise is monotonic: what is computed from
            # x +- e bounds what may come out (with either scale: a scale that
            # may be one binade off changes no value but the smallest)
            got = values8(s, k)
            a, b = rnd(x - e if k == "exp_avg" else np.maximum(x - e, 0), sc, h), rnd(x + e, sc, h)
            assert np.all((a <= got) & (got <= b)), (i, k)


ODD = [((1,), torch.float32), ((7,), torch.float32), ((8,), torch.float32), ((255,), torch.float32),
       ((256,), torch.float32), ((257,), torch.float32), ((3, 683), torch.float32),
       ((2048,), torch.float32), ((2049,), torch.float32), ((), torch.float32),
       ((5, 1000), torch.float32)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype, master", [(torch.float32, False), (torch.complex64, False),
                                           (torch.bfloat16, False), (torch.bfloat16, True),
                                           (torch.float16, False), (torch.float16, True)])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_steps(bits, dtype, master, max_norm):
    ps = make([(s, dtype) for s, _ in ODD], seed=1)
    kw = dict(lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=0.1)
    opt = AdamW(ps, lr=1e-2, weight_decay=0.1, state_bits=bits, master=master, max_norm=max_norm,
                seed=11)
    assert opt.grad_norm is None
    for t in range(1, 4):
        for k, p in enumerate(ps):   # other gradients every step
            p.grad = torch.roll(p.grad, 1) * (1 + 0.5 * k % 3)
        check_step(opt, ps, t, kw, bits, master, max_norm, seed=11)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """more tensors than one launch takes, mixed types and sizes, among them
    none and empty ones"""
    dts = [torch.float32, torch.bfloat16, torch.complex64, torch.float16]
    shapes = [((k * 37 % 91 + (k % 50 == 3) * 3000,), dts[k % 4]) for k in range(400)]
    ps = make(shapes, seed=2)
    opt = AdamW(ps, lr=3e-3, weight_decay=0.0, state_bits=bits, max_norm=1.0, seed=5)
    full = [p for p in ps if p.numel()]
    assert len(full) < len(ps)
    kw = dict(lr=3e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0)
    # check_step numbers the tensors itself: only the values are compared here
    before = [flat(p) for p in full]
    opt.step()
    norm = np.sqrt(sum((flat(p.grad) ** 2).sum() for p in full))
    clip = min(1.0, 1.0 / (norm + 1e-6))
    for p, q in zip(full, before):
        z = np.zeros(q.size)
        p1, _, _, (ep, _, _) = po.step(q, flat(p.grad), z, z, 1, clip=clip, **kw)
        assert np.all(np.abs(flat(p) - p1) <= ep + HALF[p.dtype] * (np.abs(p1) + ep) + 2.0 ** -25)
        assert int(opt.state[p]["step"]) == 1
    assert abs(float(opt.grad_norm) - norm) <= norm * (po.U + 1e-12)


def test_moments_have_the_bits_of_separate_roundings():
    """m = fl(fl(b1 m) + fl((1 - b1) g)), v alike: nothing is fused"""
    p = make([((4099,), torch.float32)], seed=20)[0]
    opt = AdamW([p], lr=1e-3)
    f = np.float32
    m = v = np.zeros(4099, f)
    for k in range(3):
        p.grad = p.grad * 1.25 + 0.01 * k
        g = p.grad.cpu().numpy()
        opt.step()
        m = m * f(0.9) + g * f(1 - 0.9)
        v = v * f(0.999) + (g * g) * f(1 - 0.999)
        assert np.array_equal(opt.state[p]["exp_avg"].cpu().numpy(), m)
        assert np.array_equal(opt.state[p]["exp_avg_sq"].cpu().numpy(), v)


def test_same_bits_every_time_and_across_lists():
    """no atomics order anything: two runs agree in every bit"""
    def run():
        ps = make([((70001,), torch.float32), ((33, 129), torch.bfloat16)] * 8, seed=3)
        opt = AdamW(ps, lr=1e-2, state_bits=8, max_norm=0.1)
        for _ in range(3):
            opt.step()
        return [p.detach() for p in ps] + [t for p in ps for t in opt.state[p].values()] + [opt.grad_norm]
    for a, b in zip(run(), run()):
        assert torch.equal(a.view(torch.uint8) if a.dim() else a, b.view(torch.uint8) if b.dim() else b)


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_have_their_own_count(bits):
    ps = make([((300,), torch.float32), ((20,), torch.float32)], seed=4)
    opt = AdamW(ps, lr=1e-2, weight_decay=0.0, state_bits=bits)
    kw = dict(lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=0.0)
    g = ps[1].grad
    ps[1].grad = None
    was = ps[1].detach().clone()
    check_step(opt, ps[:1], 1, kw, bits)
    check_step(opt, ps[:1], 2, kw, bits)
    assert torch.equal(ps[1].detach(), was) and ps[1] not in opt.state
    ps[1].grad = g
    q = flat(ps[1])
    opt.step()
    z = np.zeros(q.size)
    p1, _, _, (ep, _, _) = po.step(q, flat(g), z, z, 1, **kw)
    assert np.all(np.abs(flat(ps[1]) - p1) <= ep)
    assert [int(opt.state[p]["step"]) for p in ps] == [3, 1]
    opt.zero_grad()
    opt.step()   # nothing has a gradient
    assert [int(opt.state[p]["step"]) for p in ps] == [3, 1]


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(bits):
    """other orders of dimensions, gradients in another order, views at odd
    places: element by element the same as contiguous ones"""
    g = torch.Generator(device=DEV).manual_seed(6)
    base = torch.randn(6, 10, 14, 4, generator=g, device=DEV)
    grad = torch.randn(6, 10, 14, 4, generator=g, device=DEV)
    room = torch.zeros(base.numel() + 3, device=DEV)
    odd = room[3:].view_as(base).copy_(base)
    variants = [
        (base.clone(), grad.clone()),
        (base.clone(), grad.to(memory_format=torch.channels_last)),
        (base.clone(), torch.stack([grad, grad], -1)[..., 0]),
        (odd, grad.clone()),
    ]
    got = []
    for p, q in variants:
        p = p.detach().requires_grad_()
        p.grad = q
        opt = AdamW([p], lr=1e-2, state_bits=bits)
        opt.step()
        opt.step()
        got.append(p.detach().clone(memory_format=torch.contiguous_format))
    assert torch.equal(room[:3], torch.zeros(3, device=DEV))
    for p in got[1:]:
        assert torch.equal(p, got[0])
    # a parameter in another order: its own memory order, so 32 bits agree
    if bits == 32:
        p = base.to(memory_format=torch.channels_last).requires_grad_()
        p.grad = grad.clone()
        opt = AdamW([p], lr=1e-2)
        opt.step()
        opt.step()
        assert torch.equal(p.detach().contiguous(), got[0])
        assert opt.state[p]["exp_avg"].stride() == p.stride()


def test_broadcast_gradient():
    """an expanded gradient (stride 0), as the sum of a parameter gives"""
    p = torch.ones(5, 7, device=DEV, requires_grad=True)
    p.sum().backward()
    opt = AdamW([p], lr=0.1, weight_decay=0.0)
    opt.step()
    # m / (1 - b1) = 1, sqrt(v / (1 - b2)) = 1: p - 0.1 within the roundings
    assert torch.allclose(p, torch.full_like(p, 0.9), rtol=0, atol=2e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite(bits):
    """NaN and infinite gradients spoil their own elements and no other"""
    p = torch.ones(600, device=DEV, requires_grad=True)
    p.grad = torch.full((600,), 0.5, device=DEV)
    q = p.detach().clone().requires_grad_()
    q.grad = p.grad.clone()
    bad = [3, 300, 599]
    p.grad[3], p.grad[300], p.grad[599] = float("nan"), float("inf"), -float("inf")
    a, b = (AdamW([x], lr=1e-2, state_bits=bits) for x in (p, q))
    for _ in range(2):
        a.step()
        b.step()
        p.grad = q.grad.clone()   # finite from now on: the state remembers
    fine = torch.ones(600, dtype=torch.bool, device=DEV)
    fine[bad] = False
    assert torch.equal(p[fine], q[fine])
    assert not torch.isfinite(p[bad]).any()
    for k in ("exp_avg", "exp_avg_sq"):
        x, y = a.state[p][k].float(), b.state[q][k].float()
        assert torch.equal(x[fine], y[fine])
        assert not torch.isfinite(x[bad]).any()


def test_not_finite_norm():
    p = torch.ones(40, device=DEV, requires_grad=True)
    p.grad = torch.ones(40, device=DEV)
    p.grad[7] = float("nan")
    opt = AdamW([p], max_norm=1.0)
    opt.step()
    assert torch.isnan(opt.grad_norm) and torch.isnan(p).all()


def test_zero_and_tiny_gradients():
    """zero moments in 8 bits stay zero; small v never becomes zero"""
    p = torch.ones(512, device=DEV, requires_grad=True)
    p.grad = torch.zeros(512, device=DEV)
    p.grad[1] = 1.0
    p.grad[2] = 1e-9     # 2^-30 of the block's largest, v 2^-60 of it
    p.grad[300] = 1e-30  # v underflows in 32 bits
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8, eps=1e-8)
    for _ in range(3):
        opt.step()
        assert torch.isfinite(p).all()
    s = opt.state[p]
    v = s["exp_avg_sq"].float()
    zero = torch.ones(512, dtype=torch.bool, device=DEV)
    zero[[1, 2, 300]] = False
    assert (v[zero] == 0).all() and (s["exp_avg"].float()[zero] == 0).all()
    assert v[2] == 2.0 ** -14 and v[1] > 0
    assert torch.equal(p[zero], torch.ones_like(p[zero]))


def test_largest_gradients():
    """the 8-bit moments stay finite where the 32-bit ones do"""
    p = torch.ones(300, device=DEV, requires_grad=True)
    p.grad = torch.full((300,), 1.0, device=DEV)
    p.grad[5] = 3.4028e38    # m near 0.1 of the largest float; v overflows, as in 32 bits
    p.grad[299] = 5.8e20     # g^2 = 3.4e41 overflows before it is scaled by 0.001
    opt = AdamW([p], lr=1e-3, state_bits=8, betas=(0.0, 0.999))
    opt.step()
    s = opt.state[p]
    m, v = s["exp_avg"].float(), s["exp_avg_sq"].float()
    m, v = (x * s[k].float().repeat_interleave(256)[:300]
            for x, k in ((m, "exp_avg_scale"), (v, "exp_avg_sq_scale")))
    assert torch.isfinite(m).all() and torch.isfinite(p).all()
    assert torch.isinf(v[[5, 299]]).all() and torch.isinf(v).sum() == 2
    # v next to the largest float is held as less, never as more
    p.grad = torch.full((300,), 1.83e19, device=DEV)   # v = g^2 = 3.35e38
    opt = AdamW([p], lr=1e-3, state_bits=8, betas=(0.0, 0.0))
    opt.step()
    s = opt.state[p]
    v = s["exp_avg_sq"].float() * s["exp_avg_sq_scale"].float().repeat_interleave(256)[:300]
    assert torch.isfinite(v).all() and (v > 2.0 ** 127).all()


def test_learning_rate_tensor_and_groups():
    """a device rate is read at every step, groups keep their own options"""
    ps = make([((500,), torch.float32), ((500,), torch.float32)], seed=8)
    qs = [p.detach().clone().requires_grad_() for p in ps]
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    lr = torch.tensor(0.0, device=DEV)
    a = AdamW([dict(params=[ps[0]], lr=lr, weight_decay=0.5),
               dict(params=[ps[1]], state_bits=8, betas=(0.8, 0.9))], lr=2e-3)
    b = AdamW([dict(params=[qs[0]], weight_decay=0.5),
               dict(params=[qs[1]], state_bits=8, betas=(0.8, 0.9))], lr=2e-3)
    for v in (0.25, 0.125, 0.5):   # exact in float32: the same number either way
        lr.fill_(v)
        b.param_groups[0]["lr"] = v
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    assert a.state[ps[1]]["exp_avg"].dtype == torch.float8_e4m3fn


@pytest.mark.parametrize("bits, dtype, master", [(32, torch.float32, False), (8, torch.bfloat16, True),
                                                 (8, torch.complex64, False)])
def test_state_dict(bits, dtype, master):
    """a run that is saved and resumed gives the bits of one that went on"""
    shapes = [((3, 5), dtype), ((700,), dtype)]
    a_ps, b_ps = make(shapes, seed=9), make(shapes, seed=9)
    kw = dict(lr=1e-2, state_bits=bits, master=master, max_norm=0.3)
    a = AdamW(a_ps, **kw)
    for _ in range(2):
        a.step()
    saved = copy.deepcopy(a.state_dict())
    with torch.no_grad():
        for p, q in zip(a_ps, b_ps):
            q.copy_(p)
    b = AdamW(b_ps, **kw)
    b.load_state_dict(saved)
    for _ in range(2):
        a.step()
        b.step()
    for p, q in zip(a_ps, b_ps):
        assert torch.equal(p, q)
        for k, x in a.state[p].items():
            assert x.dtype == b.state[q][k].dtype
            assert torch.equal(x.float() if "float8" in str(x.dtype) else x,
                               b.state[q][k].float() if "float8" in str(x.dtype) else b.state[q][k])
    with pytest.raises(ValueError, match="state"):
        AdamW(b_ps, lr=1e-2, state_bits=40 - bits).load_state_dict(
            dict(saved, param_groups=[dict(g, state_bits=40 - bits) for g in saved["param_groups"]]))


def test_state_of_torch_adamw():
    """the state of torch's own AdamW is taken over"""
    ps = make([((4, 9), torch.float32), ((33,), torch.float32)], seed=10)
    qs = [p.detach().clone().requires_grad_() for p in ps]
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    a, b = torch.optim.AdamW(ps, lr=1e-2), AdamW(qs, lr=1e-2)
    a.step()
    b.load_state_dict(a.state_dict())
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    kw = dict(lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2)
    check_step(b, qs, 2, kw)


def test_refused_state_changes_nothing():
    p, q = make([((40,), torch.float32), ((30,), torch.float32)], seed=22)
    opt = AdamW([p, q], lr=1e-2)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    opt.step()
    m = opt.state[p]["exp_avg"].clone()
    bad = copy.deepcopy(saved)
    bad["state"][1]["exp_avg"] = torch.zeros(31, device=DEV)
    bad["param_groups"][0]["lr"] = 7.0
    with pytest.raises(ValueError, match="exp_avg"):
        opt.load_state_dict(bad)
    bad = copy.deepcopy(saved)
    bad["param_groups"][0]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(bad)
    assert torch.equal(opt.state[p]["exp_avg"], m) and opt.param_groups[0]["lr"] == 1e-2
    assert int(opt.state[q]["step"]) == 2
    opt.step()
    assert int(opt.state[p]["step"]) == 3


def test_moments_of_16_bit_parameters_from_torch():
    """torch keeps them in the parameter's type; here they are 32-bit"""
    p = make([((50,), torch.bfloat16)], seed=23)[0]
    q = p.detach().clone().requires_grad_()
    q.grad = p.grad.clone()
    a, b = torch.optim.AdamW([p], lr=1e-2), AdamW([q], lr=1e-2)
    a.step()
    b.load_state_dict(a.state_dict())
    assert b.state[q]["exp_avg"].dtype == torch.float32
    assert torch.equal(b.state[q]["exp_avg"], a.state[p]["exp_avg"].float())
    with torch.no_grad():
        q.copy_(p)
    check_step(b, [q], 2, dict(lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2))


def test_schedule_and_closure():
    p = make([((64,), torch.float32)], seed=12)[0]
    opt = AdamW([p], lr=0.1)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)

    def closure():
        opt.zero_grad()
        loss = (p ** 2).sum()
        loss.backward()
        return loss
    assert torch.is_tensor(opt.step(closure))
    sched.step()
    assert opt.param_groups[0]["lr"] == 0.05
    opt.step(closure)
    assert int(opt.state[p]["step"]) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """replays advance the counts, follow the gradients and a device rate"""
    def setup():
        ps = make([((1000,), torch.float32), ((77,), torch.bfloat16)], seed=13)
        lr = torch.tensor(1e-2, device=DEV)
        return ps, lr, AdamW(ps, lr=lr, state_bits=bits, max_norm=0.5)
    ps, lr, opt = setup()
    qs, lq, ref = setup()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="init_state"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.init_state()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        opt.step()
    for k in range(3):
        for p, q in zip(ps, qs):
            p.grad.mul_(0.5 + k)
            q.grad.mul_(0.5 + k)
        lr.fill_(0.01 * (k + 1))
        lq.fill_(0.01 * (k + 1))
        graph.replay()
        ref.step()
    torch.cuda.synchronize()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and int(opt.state[p]["step"]) == 3
    assert torch.equal(opt.grad_norm, ref.grad_norm)


def test_other_stream():
    p, q = (make([((300000,), torch.float32)], seed=14)[0] for _ in range(2))
    a, b = AdamW([p], lr=1e-2, max_norm=1.0), AdamW([q], lr=1e-2, max_norm=1.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            a.step()
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        b.step()
    assert torch.equal(p, q)


@pytest.fixture
def python_path(monkeypatch):
    """the calls through ctypes, as where the torch fast path is not built"""
    from flash_cqt_b200 import _native
    monkeypatch.setattr(_native, "_torchops", None)
    monkeypatch.setattr(_native, "_torchops_tried", True)


@pytest.mark.parametrize("bits", [32, 8])
def test_python_path(bits, request):
    def run():
        ps = make([((300,), torch.float32), ((5, 77), torch.bfloat16), ((9,), torch.complex64)], seed=15)
        opt = AdamW([dict(params=ps[:2], weight_decay=0.1), dict(params=ps[2:], lr=1e-3)], lr=1e-2,
                    state_bits=bits, master=True, max_norm=0.5)
        for _ in range(3):
            opt.step()
        return [p.detach() for p in ps] + [opt.grad_norm]
    a = run()
    request.getfixturevalue("python_path")
    for x, y in zip(a, run()):
        assert torch.equal(x, y)


def test_replaced_state_is_seen():
    """states, options and parameters that are exchanged between steps"""
    def fresh():
        p = make([((50,), torch.float32)], seed=16)[0]
        return p, AdamW([p], lr=1e-2)
    p, opt = fresh()
    q, ref = fresh()
    first = p.detach().clone()
    opt.step()
    for forget in (lambda: opt.state.clear(), lambda: opt.state.pop(p),
                   lambda: opt.state.__setitem__(p, {})):
        forget()
        with torch.no_grad():
            p.copy_(first)
        opt.step()
        assert int(opt.state[p]["step"]) == 1
    opt.state[p]["exp_avg"] = torch.zeros_like(p)
    opt.state[p]["exp_avg_sq"] = torch.zeros_like(p)
    opt.state[p]["step"] = torch.zeros((), dtype=torch.int64, device=DEV)
    with torch.no_grad():
        p.copy_(first)
    opt.step()
    ref.step()
    assert torch.equal(p, q)
    p.data = torch.zeros(50, device=DEV)    # another storage of the same size
    opt.step()
    assert p.abs().max() > 0
    opt.param_groups[0]["state_bits"] = 8   # does not fit the states
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()
    opt.param_groups[0].update(state_bits=32, lr=-1.0)
    with pytest.raises((ValueError, RuntimeError), match="lr"):
        opt.step()


@pytest.mark.parametrize("python", [False, True])
def test_refused_options_change_nothing(python, request):
    if python:
        request.getfixturevalue("python_path")
    ps = make([((50,), torch.float32), ((60,), torch.float32)], seed=24)
    opt = AdamW([dict(params=[ps[0]]), dict(params=[ps[1]])], lr=1e-2, max_norm=1.0)
    opt.step()
    was = [p.detach().clone() for p in ps]
    for k, v in (("lr", -1.0), ("lr", float("nan")), ("betas", (0.9, 1.0)), ("eps", -1.0),
                 ("weight_decay", -1.0)):
        keep = opt.param_groups[1][k]
        opt.param_groups[1][k] = v
        with pytest.raises(ValueError):
            opt.step()
        opt.param_groups[1][k] = keep
    assert all(torch.equal(p, q) for p, q in zip(ps, was))
    assert [int(opt.state[p]["step"]) for p in ps] == [1, 1]
    # another type in the same parameter: the state is 32-bit and stays
    ps[0].data = ps[0].data.bfloat16()
    ps[0].grad = torch.ones(50, device=DEV, dtype=torch.bfloat16)
    opt.step()
    assert int(opt.state[ps[0]]["step"]) == 2 and torch.isfinite(ps[0]).all()
    assert (ps[0].float() - was[0]).abs().max() < 0.1


def test_step_hooks_are_served():
    p, calls = make([((5,), torch.float32)], seed=17)[0], []
    opt = AdamW([p])
    a = opt.register_step_pre_hook(lambda *_: calls.append("pre"))
    opt.register_step_post_hook(lambda *_: calls.append("post"))
    opt.step()
    assert calls == ["pre", "post"] and int(opt.state[p]["step"]) == 1
    a.remove()
    opt.step()
    assert calls == ["pre", "post", "post"] and int(opt.state[p]["step"]) == 2


def test_deepcopy_and_save():
    import io
    p = make([((70,), torch.float32)], seed=18)[0]
    opt = AdamW([p], lr=1e-2, max_norm=0.2, seed=3, state_bits=8)
    opt.step()
    f = io.BytesIO()   # (plain pickle cannot hold 8-bit tensors, torch.save can)
    torch.save(opt, f)
    f.seek(0)
    for other in (copy.deepcopy(opt), torch.load(f, weights_only=False)):
        q = other.param_groups[0]["params"][0]
        if q.grad is None:
            q.grad = p.grad.clone()
        assert other.max_norm == 0.2 and other.seed == 3
        other.step()
        assert int(other.state[q]["step"]) == 2
    q2 = q.detach().clone()
    opt.step()
    assert torch.equal(p, q2)


def test_load_into_a_captured_step():
    """a captured step goes on from a state that is loaded later"""
    def setup():
        p = make([((600,), torch.float32)], seed=21)[0]
        return p, AdamW([p], lr=1e-2, state_bits=8, max_norm=0.5)
    p, opt = setup()
    q, ref = setup()
    for _ in range(2):
        ref.step()
    saved = copy.deepcopy(ref.state_dict())
    opt.init_state()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.load_state_dict(saved)
    with torch.no_grad():
        p.copy_(q)
    graph.replay()
    ref.step()
    assert torch.equal(p, q) and int(opt.state[p]["step"]) == 3


def test_first_step_of_a_process_in_a_capture():
    """nothing that has to happen outside of a capture is left to a first launch"""
    import subprocess
    import sys
    code = """
import torch
from flash_cqt_b200 import AdamW
p = torch.ones(1000, device="cuda", requires_grad=True)
p.grad = torch.ones_like(p)
opt = AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8, max_norm=1e9)
opt.init_state()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    opt.step()
g.replay()
torch.cuda.synchronize()
assert abs(float(p[0]) - 0.5) < 1e-5 and int(opt.state[p]["step"]) == 1
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_more_than_2_32_elements():
    """offsets and noise beyond 32 bits"""
    far, tail = 2 ** 32, 3001
    p = torch.zeros(far + tail, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    p.grad = torch.zeros(far + tail, dtype=torch.bfloat16, device=DEV)
    p.grad[-tail:] = torch.randn(tail, device=DEV)
    p.grad[:5] = 1.0
    g = p.grad[-tail:].double().cpu().numpy()
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=8, max_norm=1e3, seed=4)
    opt.step()
    assert abs(float(opt.grad_norm) - np.sqrt((g ** 2).sum() + 5)) <= float(opt.grad_norm) * po.U * 1.01
    z = np.zeros(tail)
    p1, m1, _, (ep, em, _) = po.step(z, g, z, z, 1, 1e-2, 0.9, 0.999, 1e-8, 0.0)
    assert np.all(np.abs(flat(p[-tail:]) - p1) <= ep + 2.0 ** -8 * (np.abs(p1) + ep))
    s = opt.state[p]
    sc = s["exp_avg_scale"][far // 256:].double().cpu().numpy()
    got = s["exp_avg"][-tail:].double().cpu().numpy() * po.spread(sc, tail)
    h = po.noise(4, 1, 0, tail, start=far)
    assert np.all((po.round_m(m1 - em, sc, h) <= got) & (got <= po.round_m(m1 + em, sc, h)))
    assert float(s["exp_avg"][5:4096].float().abs().max()) == 0 and float(p[:5].float().max()) < 0


def test_refusals():
    p = torch.zeros(8, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="share memory"):
        AdamW([p, p.detach()[2:4].requires_grad_()])
    with pytest.raises(ValueError, match="share memory"):
        AdamW([p, p])
    with pytest.raises(TypeError, match="set"):
        AdamW([dict(params={p})])
    opt = AdamW([p])
    with pytest.raises(ValueError, match="share memory"):
        opt.add_param_group(dict(params=[p]))
    with pytest.raises(TypeError, match="device lr"):
        AdamW([p], lr=torch.tensor(1e-3, device=DEV, dtype=torch.float64))
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1), (8,)).to(DEV)
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    p.grad = torch.ones(8, device=DEV)
    opt.step()
    s = opt.state[p]
    s["exp_avg"] = s["exp_avg"][:4]
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()


def test_train_step_with_the_transform():
    """analysis, learned gains, synthesis, fused loss, gradients and step: the
    parameters move as the formulas say for the gradients that autograd gives,
    and the gains' gradients agree with differences of the loss"""
    torch.manual_seed(0)
    cqt = OctCQT([3, 4, 2], [8, 16, 32], fs=44100, audio_len=65536, device=DEV)
    t = TrainableCQT(cqt, DEV)
    x = torch.randn(2, 65536, device=DEV)
    target = torch.randn(2, 65536, device=DEV)
    gains = [torch.ones(b, 1, device=DEV, dtype=torch.complex64, requires_grad=True)
             for b, _, _ in cqt.heap.gspec]
    sig = x.clone().requires_grad_()
    opt = AdamW(gains + [sig], lr=1e-3, weight_decay=0.0, max_norm=1e-3)

    def loss_of():
        blocks, side = t.fwd(sig)
        every = [c * g for c, g in zip(list(blocks) + list(side), gains)]
        return t.mse_loss(every[:len(blocks)], every[len(blocks):], target)
    kw = dict(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0)
    for step in (1, 2):
        opt.zero_grad()
        loss_of().backward()
        check_step(opt, gains + [sig], step, kw, max_norm=1e-3)
    # a difference over 2 h of a loss that is quadratic in one gain is its
    # slope up to the loss's own rounding: 2^-23 of a mean near 2, over 2 h
    opt.zero_grad()
    loss_of().backward()
    g, h = gains[6], 0.25
    with torch.no_grad():
        k = int(g.grad.real.abs().argmax())
        up, down = g.detach().clone(), g.detach().clone()
        up[k] += h
        down[k] -= h
        keep = g.detach().clone()
        g.copy_(up)
        hi = float(loss_of())
        g.copy_(down)
        lo = float(loss_of())
        g.copy_(keep)
    slope = (hi - lo) / (2 * h)
    # the loss is a mean of 131072 squares: a few steps of float32
    assert abs(slope - float(g.grad[k].real)) <= 8 * 2.0 ** -23 * max(hi, lo) / (2 * h)


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_step_is_seen_by_autograd(bits, python, request):
    """a backward pass through values that were saved before a step is refused,
    as behind any operation in place"""
    if python:
        request.getfixturevalue("python_path")
    ps = make([((50,), torch.float32), ((7, 3), torch.float32), ((4,), torch.float32)], seed=30)
    opt = AdamW(ps, lr=1e-2, state_bits=bits, max_norm=1.0)
    ps[2].grad = None
    opt.step()
    x = torch.ones((), device=DEV, requires_grad=True)
    ys = [(p * p).sum() for p in ps] + [x * opt.grad_norm]
    state = [t for k, t in opt.state[ps[0]].items() if k != "order"]   # (never written)
    seen = [t._version for t in state]
    opt.step()
    for y in (ys[0], ys[1], ys[3]):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    ys[2].backward()   # that one has not been stepped
    assert torch.equal(ps[2].grad, 2 * ps[2].detach())
    assert all(t._version > v for t, v in zip(state, seen))
    # a refused step marks nothing
    was = [p._version for p in ps]
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError):
        opt.step()
    assert [p._version for p in ps] == was


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_exchanged_storage_is_refused(bits, python, request):
    """a state whose storage was moved away or replaced behind the same object
    is refused before anything is launched"""
    if python:
        request.getfixturevalue("python_path")
    ps = make([((4, 130), torch.bfloat16), ((300,), torch.bfloat16)], seed=31)
    opt = AdamW(ps, lr=1e-2, state_bits=bits, master=True, max_norm=1.0)
    opt.step()
    was = [p.detach().clone() for p in ps]
    for k in [k for k in opt.state[ps[1]] if k != "order"]:   # (no kernel takes that)
        t = opt.state[ps[1]][k]
        for other in (t.data.cpu(), t.data.double() if k != "step" else t.data.int()):
            keep = t.data
            t.data = other
            with pytest.raises(ValueError, match=k):
                opt.step()
            t.data = keep
    p = ps[1]
    keep, grad = p.data, p.grad
    for other in (keep.cpu(), torch.zeros(300, 2, dtype=torch.bfloat16, device=DEV)[:, 0]):
        p.grad = None
        p.data = other
        p.grad = torch.ones_like(p)
        with pytest.raises((RuntimeError, ValueError), match="CUDA devices only|dense"):
            opt.step()
    p.grad = None
    p.data = keep
    p.grad = grad
    norm = opt.grad_norm
    opt.grad_norm = norm.cpu()
    with pytest.raises(ValueError, match="grad_norm"):
        opt.step()
    opt.grad_norm = norm
    assert all(torch.equal(p.detach(), q) for p, q in zip(ps, was))
    opt.step()
    assert [int(opt.state[p]["step"]) for p in ps] == [2, 2]


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("bits, master", [(32, False), (32, True), (8, False), (8, True)])
def test_changed_order_is_refused(bits, master, python, request):
    """a parameter that is moved to another memory order behind the same object"""
    if python:
        request.getfixturevalue("python_path")
    p = make([((4, 6, 3, 5), torch.bfloat16)], seed=32)[0]
    opt = AdamW([p], lr=1e-2, state_bits=bits, master=master)
    opt.step()
    was, m = p.detach().clone(), opt.state[p]["exp_avg"].clone()
    p.data = p.data.to(memory_format=torch.channels_last)
    with pytest.raises(ValueError, match="order" if bits == 8 and not master else "state"):
        opt.step()
    assert torch.equal(p.detach(), was) and int(opt.state[p]["step"]) == 1
    assert torch.equal(opt.state[p]["exp_avg"].float(), m.float())
    p.data = p.data.contiguous()
    check_step(opt, [p], 2, dict(lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2), bits, master)


@pytest.mark.parametrize("dtype, master", [(torch.float32, False), (torch.complex64, False),
                                           (torch.bfloat16, True)])
def test_state_of_another_order(dtype, master):
    """8-bit moments saved from a contiguous parameter go on with one in another
    order, and the way back"""
    kw = dict(lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2)
    p = make([((4, 6, 3, 50), dtype)], seed=33)[0]
    other = p.detach().permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    q = other.requires_grad_()
    a = AdamW([p], lr=1e-2, state_bits=8, master=master)
    a.step()
    b = AdamW([q], lr=1e-2, state_bits=8, master=master)
    b.load_state_dict(a.state_dict())
    with torch.no_grad():
        q.copy_(p)
    q.grad = p.grad.clone()   # in the other order: copied for the step

    def moments(opt, x):
        """element by element, in the order of the indices"""
        shape = (*x.shape, 2) if x.is_complex() else tuple(x.shape)
        strides = (*(2 * t for t in x.stride()), 1) if x.is_complex() else x.stride()
        return [torch.from_numpy(values8(opt.state[x], k)).as_strided(shape, strides)
                for k in ("exp_avg", "exp_avg_sq")]
    for x, y, small in zip(moments(a, p), moments(b, q), (2.0 ** -6, 2.0 ** -14)):
        # what is small beside its new neighbours rounds: a scale is at most 2^-8
        # (2^-15) of the largest value over 0.875
        top = float(x.abs().max())
        assert ((x - y).abs() <= (top / 0.875 * 2.0 ** (-8 if small > 1e-3 else -15)) * small).all()
        assert ((x - y).abs() == 0).double().mean() > 0.5
    q.grad = torch.empty_like(q).copy_(p.grad)
    check_step(b, [q], 2, kw, 8, master)
    c = AdamW([p], lr=1e-2, state_bits=8, master=master)
    c.load_state_dict(b.state_dict())
    with torch.no_grad():
        p.copy_(q)
    check_step(c, [p], 3, kw, 8, master)


@pytest.mark.parametrize("where", ["cuda", "cpu"])
def test_captured_step_follows_a_loaded_rate(where):
    """and what is put into the group's tensor after the dictionary was loaded"""
    def setup():
        p = make([((600,), torch.float32)], seed=34)[0]
        return p, AdamW([p], lr=torch.tensor(1e-2, device=DEV))
    p, opt = setup()
    q, ref = setup()
    ref.step()
    ref.param_groups[0]["lr"].fill_(0.25)
    saved = copy.deepcopy(ref.state_dict())
    saved["param_groups"][0]["lr"] = saved["param_groups"][0]["lr"].to(where)
    opt.init_state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.load_state_dict(saved)
    with torch.no_grad():
        p.copy_(q)
    for rate in (None, 0.5):
        if rate:
            opt.param_groups[0]["lr"].fill_(rate)
            ref.param_groups[0]["lr"].fill_(rate)
        graph.replay()
        ref.step()
        assert torch.equal(p, q)
    assert int(opt.state[p]["step"]) == 3


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_goes_on_from_an_empty_state(bits, python, request):
    """a dictionary that was saved before the first step"""
    if python:
        request.getfixturevalue("python_path")
    def setup():
        p = make([((600,), torch.float32)], seed=35)[0]
        return p, AdamW([p], lr=1e-2, state_bits=bits)
    p, opt = setup()
    q, ref = setup()
    empty = copy.deepcopy(opt.state_dict())
    opt.step()
    at = {k: t.data_ptr() for k, t in opt.state[p].items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.load_state_dict(empty)
    with torch.no_grad():
        p.copy_(q)
    for _ in range(2):
        graph.replay()
        ref.step()
    assert torch.equal(p, q) and int(opt.state[p]["step"]) == 2
    assert {k: t.data_ptr() for k, t in opt.state[p].items()} == at
    opt.step()   # a step of its own goes on from there
    ref.step()
    assert torch.equal(p, q) and int(opt.state[p]["step"]) == 3


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("capture", [False, True])
def test_what_a_graph_writes_to_stays(capture, python, request):
    """tensors that are replaced live on if, and only if, a graph addresses them"""
    if python:
        request.getfixturevalue("python_path")
    p = make([((600,), torch.float32)], seed=36)[0]
    # (a rate of the group's own: the constructor's default is kept by the class)
    opt = AdamW([dict(params=[p], lr=torch.tensor(1e-2, device=DEV))], state_bits=8)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    if capture:
        with torch.cuda.graph(graph):
            opt.step()
    old = [weakref.ref(t) for k, t in opt.state[p].items() if k != "order"]
    old.append(weakref.ref(opt.param_groups[0]["lr"]))
    other = AdamW([make([((600,), torch.float32)], seed=37)[0]], lr=2e-2)
    other.step()
    opt.param_groups[0]["lr"] = 3e-2
    opt.load_state_dict(other.state_dict())   # 32-bit moments
    opt.step()
    gc.collect()
    assert opt.state[p]["exp_avg"].dtype == torch.float32 and opt.param_groups[0]["lr"] == 2e-2
    # (the count has the same form in both and is used again)
    assert [r() is not None for r in old] == [capture or k == 0 for k in range(len(old))]
    if capture:
        was = [t.clone() for t in opt.state[p].values()]
        graph.replay()   # the old state's step, of the same parameter
        assert torch.isfinite(p).all()
        assert all(torch.equal(a, b) for a, b in zip(was[1:], list(opt.state[p].values())[1:]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("eps, size", [(0.0, 1e-17), (1e-30, 1e-17), (1e-18, 1e-17), (9e-10, 1e-17),
                                       (1e-9, 1e-17), (1e-8, 1e-17), (0.0, 1.0), (1e-30, 1e-3),
                                       (2e38, 1e17)])
def test_any_eps(eps, size, dtype, bits):
    """the formula's denominator for every eps that is accepted, and gradients as
    small: v and g^2 stay normal numbers of float32, so every rounding is counted"""
    if dtype == torch.float16 and size not in (1.0, 1e-3):
        return   # (not numbers of that type)
    ps = make([((700,), dtype), ((9, 31), dtype)], seed=38)
    for p in ps:
        with torch.no_grad():
            p.zero_()   # the update is all there is
        y = p.grad.float()
        p.grad = (torch.sign(y) * (0.5 + y.abs()) * size).to(dtype)
        assert (p.grad.float().abs() >= 0.49 * size).all()
    opt = AdamW(ps, lr=1e-2, weight_decay=0.0, eps=eps, state_bits=bits, seed=2)
    kw = dict(lr=1e-2, b1=0.9, b2=0.999, eps=eps, wd=0.0)
    for t in (1, 2, 3):
        check_step(opt, ps, t, kw, bits, seed=2)


@pytest.mark.parametrize("bits", [32, 8])
def test_no_eps_at_the_border(bits):
    """eps 0: a subnormal v, and 0 / 0 where there has been no gradient"""
    p = torch.zeros(600, device=DEV, requires_grad=True)
    p.grad = torch.full((600,), 1e-19, device=DEV)
    p.grad[5] = p.grad[400] = 0.0
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, eps=0.0, state_bits=bits)
    opt.step()
    none = torch.zeros(600, dtype=torch.bool, device=DEV)
    none[[5, 400]] = True
    assert torch.isnan(p[none]).all()
    # m / (1 - b1) = g and sqrt(v / (1 - b2)) = |g|: the update is the rate.  v =
    # 1e-41 is rounded to a multiple of 2^-149, its root is off by half of that
    off = (p.detach()[~none].double() / -1e-2 - 1).abs().max()
    assert float(off) <= 0.5 * 2.0 ** -150 / 1e-41 * 1.01 + 31 * po.U


@pytest.mark.parametrize("python", [False, True])
def test_refused_host_rate_changes_nothing(python, request):
    if python:
        request.getfixturevalue("python_path")
    ps = make([((50,), torch.float32), ((60,), torch.float32)], seed=39)
    rate = torch.tensor(1e-2)
    opt = AdamW([dict(params=[ps[0]]), dict(params=[ps[1]], lr=rate)], lr=1e-2)
    opt.step()
    was = [p.detach().clone() for p in ps]
    rate.fill_(-1.0)
    with pytest.raises(ValueError, match="lr"):
        opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, was))
    assert [int(opt.state[p]["step"]) for p in ps] == [1, 1]


@pytest.mark.parametrize("bits", [32, 8])
def test_state_through_a_file(bits):
    """saved and loaded to the device, the record of the order with it, into a
    parameter in another order"""
    import io
    p = make([((4, 6, 70), torch.bfloat16)], seed=40)[0]
    a = AdamW([p], lr=1e-2, state_bits=bits, master=True)
    a.step()
    f = io.BytesIO()
    torch.save(a.state_dict(), f)
    q = p.detach().transpose(0, 2).contiguous().transpose(0, 2).requires_grad_()
    q.grad = torch.empty_like(q).copy_(p.grad)
    b = AdamW([q], lr=1e-2, state_bits=bits, master=True)
    for where in (DEV, "cpu"):
        f.seek(0)
        b.load_state_dict(torch.load(f, map_location=where, weights_only=True))
    assert torch.equal(b.state[q]["master"], a.state[p]["master"])
    assert b.state[q]["master"].stride() == q.stride()
    check_step(b, [q], 2, dict(lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2), bits, True)

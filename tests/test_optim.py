"""CPU checks of AdamW: refusals, the C entries' argument checks, the rounding
noise of the 8-bit moments."""
import copy
import ctypes

import numpy as np
import pytest
import torch

import plain_optim as po
from flash_cqt_b200 import AdamW, _native


def leaf(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, requires_grad=True)


@pytest.mark.parametrize("kw, what", [
    (dict(lr=-1.0), "lr"), (dict(lr=float("nan")), "lr"), (dict(betas=(1.0, 0.9)), "betas"),
    (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1e-8), "eps"), (dict(weight_decay=-1.0), "eps"),
    (dict(state_bits=16), "state_bits"), (dict(max_norm=0.0), "max_norm"),
    (dict(max_norm=float("nan")), "max_norm"), (dict(lr=torch.ones(2)), "lr")])
def test_bad_options(kw, what):
    with pytest.raises(ValueError, match=what):
        AdamW([leaf(3)], **kw)


def test_bad_parameters():
    with pytest.raises(TypeError, match="float32"):
        AdamW([leaf(3, dtype=torch.float64)])
    with pytest.raises(TypeError, match="float32"):
        AdamW([leaf(3, dtype=torch.complex128)])
    with pytest.raises(ValueError, match="dense"):
        AdamW([torch.zeros(4, 6)[:, ::2].requires_grad_()])
    with pytest.raises(ValueError, match="dense"):
        AdamW([torch.zeros(1, 4).expand(3, 4).requires_grad_()])
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        AdamW([leaf(3)])
    with pytest.raises(ValueError):
        AdamW([])


def test_dense_orders():
    from flash_cqt_b200.optim import _dense, _same_order
    a = torch.zeros(2, 3, 4, 5)
    assert _dense(a) and _dense(a.permute(2, 0, 3, 1)) and _dense(torch.zeros(()))
    assert _dense(a.to(memory_format=torch.channels_last))
    assert not _dense(a[:, 1:]) and not _dense(a[..., ::2])
    assert _dense(torch.zeros(3, 1)[:, :1]) and _dense(torch.zeros(0, 4))
    assert not _same_order(torch.zeros(3, 4), torch.zeros(4, 3).t())
    assert _same_order(torch.zeros(1, 4), torch.zeros(4, 1).t())


def test_c_entries_refuse():
    L = _native.lib()
    T = _native.CqtAdamwTensor
    ws = ctypes.create_string_buffer(1 << 16)
    at = (ctypes.addressof(ws) + 15) & ~15
    need = L.cqt_adamw_workspace_bytes(1)
    assert need < 1 << 15 and L.cqt_adamw_workspace_bytes(-1) == 0
    assert L.cqt_adamw_workspace_bytes(361) > need
    good = _native.CqtAdamwArgs(1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0, None, 0, 0)

    def step(t, args=good, bits=32, count=1, w=at, size=need):
        rc = L.cqt_adamw_step(ctypes.byref(t) if t is not None else None, count, bits,
                              ctypes.byref(args), w, size, None)
        return rc, L.cqt_last_error().decode()

    # addresses that are never read: every call is refused on the host
    ok = dict(param=64, grad=64, exp_avg=64, exp_avg_sq=64, step=64, numel=4)
    assert step(T(**ok), w=None) == (-1, "workspace missing or smaller than cqt_adamw_workspace_bytes")
    assert step(T(**ok), size=need - 1)[0] == -1
    assert step(T(**ok), w=at + 4)[1] == "workspace not 16-byte aligned"
    assert step(T(**ok), count=-1)[1] == "negative tensor count"
    assert step(None)[1] == "null tensors or arguments"
    assert step(T(**ok), bits=16)[1] == "state_bits must be 8 or 32"
    for bad in (dict(grad=None), dict(grad=66), dict(param=None), dict(param=65), dict(exp_avg=None),
                dict(exp_avg_sq=None), dict(exp_avg_sq=66), dict(step=None), dict(step=68),
                dict(master=64), dict(numel=-1), dict(dtype=3), dict(numel=1 << 43)):
        rc, msg = step(T(**{**ok, **bad}))
        assert rc == -1 and msg, bad
    assert step(T(**ok), bits=8)[1] == "null scales or misaligned moments"
    for k, v in (("beta1", 1.0), ("beta2", -0.1), ("beta1", float("nan")), ("eps", -1.0)):
        a = _native.CqtAdamwArgs(1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0, None, 0, 0)
        setattr(a, k, v)
        assert "betas" in step(T(**ok), a)[1]
    a = _native.CqtAdamwArgs(1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0, None, 1, 0)
    assert step(T(**ok), a)[1] == "max_norm must be positive"
    a = _native.CqtAdamwArgs(1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None, 3, 0)
    assert "use_norm" in step(T(**ok), a)[1]
    a = _native.CqtAdamwArgs(-1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None, 0, 0)
    assert step(T(**ok), a)[1] == "lr must not be negative"
    assert L.cqt_grad_norm(ctypes.byref(T(numel=3)), 1, None, at, need, None) == -1
    assert L.cqt_grad_norm(None, 1, None, at, need, None) == -1
    # a list without elements is no work
    assert step(T(numel=0))[0] == 0 and step(None, count=0)[0] == 0


def test_noise_is_uniform_and_independent():
    n = 1 << 16
    h = po.noise(7, 3, 2, n)
    for bits in (h & np.uint32(0xffff), h >> np.uint32(16)):
        # 64 classes of 1024 expected: chi square of 63 degrees of freedom is
        # below 63 + 6 sqrt(126) = 130 but for one in a million
        c = np.bincount(bits >> np.uint32(10), minlength=64)
        assert ((c - 1024.0) ** 2 / 1024).sum() < 130
    # neighbours, steps, tensors and seeds: correlations of n pairs are below
    # 6 / sqrt(n)
    f = lambda x: (x & np.uint32(0xffff)) / 65536.0 - 0.5  # noqa: E731
    a = f(h)
    for b in (f(h >> np.uint32(16)), np.roll(a, 1), f(po.noise(7, 4, 2, n)), f(po.noise(7, 3, 3, n)),
              f(po.noise(8, 3, 2, n))):
        assert abs((a * b).mean() * 12) < 6 / np.sqrt(n)


def test_rounding_is_unbiased():
    """the mean over many draws is the value itself (within 6 deviations)"""
    n = 1 << 15
    for x in (0.3, 1.0, 447.0, 2.0 ** -5):
        v = np.full(n, x)
        v[::po.BLOCK] = 448.0
        s = po.scales(v, 448.0)
        r = po.round_m(v, s, po.noise(1, 1, 0, n))[v == x]
        step = 2.0 ** (np.floor(np.log2(x)) - 3)
        assert abs(r.mean() - x) < 6 * step / 2 / np.sqrt(r.size) + step * 2.0 ** -17
    v = np.full(n, 3.3)
    v[::po.BLOCK] = 57344.0
    r = po.round_v(v, po.scales(v, 57344.0), po.noise(1, 1, 0, n))[v == 3.3]
    assert abs(r.mean() - 3.3) < 6 * 0.25 / np.sqrt(r.size)


def plans():
    mod = _native.torch_ops()
    if mod is None:
        pytest.skip("the torch fast path is not built")
    return mod


def state_of(p, bits, master=False):
    """a state as the kernels take it, on the parameter's device"""
    n = p.numel() * (2 if p.is_complex() else 1)
    s = dict(step=torch.zeros((), dtype=torch.int64, device=p.device))
    if bits == 8:
        z = lambda n, dt: torch.ones(n, dtype=torch.uint8, device=p.device).view(dt)  # noqa: E731
        s.update(exp_avg=z(n, torch.float8_e4m3fn), exp_avg_sq=z(n, torch.float8_e5m2),
                 exp_avg_scale=z(-(-n // 256), torch.float8_e8m0fnu),
                 exp_avg_sq_scale=z(-(-n // 256), torch.float8_e8m0fnu))
    else:
        dt = torch.complex64 if p.is_complex() else torch.float32
        s.update(exp_avg=torch.zeros_like(p, dtype=dt, requires_grad=False),
                 exp_avg_sq=torch.zeros_like(p, dtype=dt, requires_grad=False))
    if master:
        s["master"] = p.detach().float()
    return s


def exchanges(bits, master):
    """(entry, what is put in its place): another type, size or order"""
    every = ["exp_avg", "exp_avg_sq", "step"] + (["master"] if master else []) \
        + (["exp_avg_scale", "exp_avg_sq_scale"] if bits == 8 else [])
    out = []
    for k in every:
        out.append((k, lambda x: x.float().double() if x.dtype != torch.int64 else x.int()))
        out.append((k, lambda x: torch.cat([x.reshape(-1).view(torch.uint8)] * 2).view(x.dtype)))
        if k == "master" or (bits == 32 and k != "step"):
            out.append((k, lambda x: x.t().contiguous().t()))
            out.append((k, lambda x: x.bfloat16()))
            out.append((k, lambda x: x.t()))
        elif k != "step":
            out.append((k, lambda x: x[:-1]))
            out.append((k, lambda x: x.view(torch.uint8)))
            out.append((k, lambda x: torch.cat([x.view(torch.uint8)] * 2).view(x.dtype)[::2]))
    return out


@pytest.mark.parametrize("bits, master", [(32, False), (32, True), (8, False), (8, True)])
def test_exchanged_states_are_refused(bits, master):
    """every tensor of a state is looked at again before a step: its storage
    can be exchanged behind the same object"""
    mod = plans()
    dt = torch.bfloat16 if master else torch.float32
    p, q = (torch.zeros(5, 120, dtype=dt, requires_grad=True) for _ in range(2))
    for x in (p, q):
        x.grad = torch.ones_like(x)
    group = dict(params=[p, q], state_bits=bits, master=master)
    state = {x: state_of(x, bits, master) for x in (p, q)}
    plan = mod.AdamWPlan(-1, 0, 0, 0, [group], state)
    assert plan.fits([group], state)
    for k, change in exchanges(bits, master):
        was = state[q][k].data
        state[q][k].data = change(was)
        assert not plan.fits([group], state), k
        with pytest.raises(ValueError, match=k):
            AdamW._check_state(state[q], q, group)
        state[q][k].data = was
        assert plan.fits([group], state)
    # the parameter's own
    was = p.data
    for other in (was.double(), was[:, :7], was.t().contiguous().t(), was.t()):
        p.data = other
        p.grad = None
        assert plan.fits([group], state)   # nothing is done with it
        p.grad = torch.ones_like(p)
        assert not plan.fits([group], state)
    p.data, p.grad = was, None
    p.grad = torch.ones_like(p)
    assert plan.fits([group], state)
    AdamW._check_state(state[p], p, group)


@pytest.fixture
def on_host(monkeypatch):
    """optimizers over host tensors: everything but the step itself"""
    monkeypatch.setattr(AdamW, "_check_param", lambda self, p: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def values(s, p):
    """an 8-bit state's moments as float64, element by element of the parameter"""
    out = []
    for k in ("exp_avg", "exp_avg_sq"):
        x = s[k].double() * s[k + "_scale"].double().repeat_interleave(256)[:s[k].numel()]
        shape, strides = list(p.shape), list(p.stride())
        if p.is_complex():
            shape, strides = [*shape, 2], [*(2 * t for t in strides), 1]
        out.append(x.as_strided(shape, strides))
    return out


def random_codes(s, seed):
    """normal values (and zero) of both formats, scales of a few binades"""
    g = torch.Generator().manual_seed(seed)
    n = s["exp_avg"].numel()
    r = lambda lo, hi, m=n: torch.randint(lo, hi, (m,), generator=g, dtype=torch.uint8)  # noqa: E731
    s["exp_avg"].view(torch.uint8).copy_(r(64, 127) | r(0, 2) << 7)     # 2 to 448
    s["exp_avg"].view(torch.uint8)[::17] = 0
    s["exp_avg_sq"].view(torch.uint8).copy_(r(60, 124))                 # 1 to 57344
    for k in ("exp_avg_scale", "exp_avg_sq_scale"):
        s[k].view(torch.uint8).copy_(r(100, 106, s[k].numel()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.complex64])
def test_codes_are_laid_out_anew(on_host, dtype):
    """8-bit moments that were saved in another memory order keep their elements"""
    a = torch.zeros(3, 5, 7, 4, dtype=dtype, requires_grad=True)
    b = torch.zeros(3, 5, 7, 4, dtype=dtype).permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    b.requires_grad_()
    assert a.shape == b.shape and a.stride() != b.stride()
    for p, q in ((a, b), (b, a), (a, a), (b, b)):
        one, two = AdamW([p], state_bits=8), AdamW([q], state_bits=8)
        one.init_state()
        random_codes(one.state[p], seed=5)
        two.load_state_dict(one.state_dict())
        for x, y in zip(values(one.state[p], p), values(two.state[q], q)):
            assert torch.equal(x, y)   # no value is 2^-6 (m) or 2^-14 (v) of a neighbour's scale
        AdamW._check_state(two.state[q], q, two.param_groups[0])
        assert two.state[q]["order"].tolist() == [list(q.shape), list(q.stride())]


def test_codes_small_beside_new_neighbours(on_host):
    """what falls under its new block's scale: m goes to the nearest value, v never
    to zero; infinite and undefined values stay what they are"""
    p = torch.zeros(256, 2, requires_grad=True)
    q = torch.zeros(2, 256).t().requires_grad_()
    one, two = AdamW([p], state_bits=8), AdamW([q], state_bits=8)
    one.init_state()
    s = one.state[p]
    s["exp_avg"].view(torch.uint8).fill_(0x38)       # 1
    s["exp_avg_sq"].view(torch.uint8).fill_(0x3c)    # 1
    for k in ("exp_avg_scale", "exp_avg_sq_scale"):
        s[k].view(torch.uint8)[:] = torch.tensor([127, 87], dtype=torch.uint8)   # 1 and 2^-40
    s["exp_avg"].view(torch.uint8)[3] = 0x7f         # NaN
    s["exp_avg_sq"].view(torch.uint8)[5] = 0x7c      # inf
    s["exp_avg_sq"].view(torch.uint8)[300] = 0
    two.load_state_dict(one.state_dict())
    (m0, v0), (m1, v1) = values(s, p), values(two.state[q], q)
    big = torch.arange(256) < 128
    assert torch.equal(m1[~big], torch.zeros(128, 2).double())
    assert torch.equal(torch.nan_to_num(m1[big], 9.0), torch.nan_to_num(m0[big], 9.0))
    assert m1.isnan().sum() == 1 and v1.isinf().sum() == 1
    assert torch.equal(v1[big], v0[big])
    # the columns' largest value is 1: scales 2^-15, their smallest normal value 2^-29
    assert v1[150, 0] == 0 and (v1[~big] == 2.0 ** -29).sum() == 255


def test_order_refusals(on_host):
    p = torch.zeros(6, 40, requires_grad=True)
    q = torch.zeros(40, 6).t().requires_grad_()
    one, two = AdamW([p], state_bits=8), AdamW([q], state_bits=8)
    one.init_state()
    saved = one.state_dict()

    def without(key, value=None):
        s = {k: v for k, v in saved["state"][0].items() if k != key}
        return dict(saved, state={0: s if value is None else dict(s, **{key: value})})
    one.load_state_dict(without("order"))            # a contiguous parameter: fine
    AdamW._check_state(one.state[p], p, one.param_groups[0])
    with pytest.raises(ValueError, match="order"):
        two.load_state_dict(without("order"))
    for bad in (torch.tensor([[6, 40], [40, 2]]), torch.tensor([[40, 6], [6, 1]]),
                torch.tensor([[6, 40, 1], [40, 1, 1]]), torch.tensor([[6, 40], [1 << 40, 1]])):
        with pytest.raises(ValueError, match="order"):
            one.load_state_dict(without("order", bad))
    # a parameter that was moved to another order after its state was made
    group = one.param_groups[0]
    plan = plans().AdamWPlan(-1, 0, 0, 0, one.param_groups, one.state)
    p.grad = torch.ones(6, 40)
    assert plan.fits(one.param_groups, one.state)
    p.data = p.data.t().contiguous().t()
    assert not plan.fits(one.param_groups, one.state)
    with pytest.raises(ValueError, match="order"):
        AdamW._check_state(one.state[p], p, group)


def torch_state(*shapes, dtype=torch.float32, **kw):
    """the state of torch's own AdamW after a step"""
    ps = [torch.ones(*s, dtype=dtype, requires_grad=True) for s in shapes]
    opt = torch.optim.AdamW(ps, **kw)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    return opt.state_dict()


def test_loaded_dictionary_leaves_a_groups_own_options(on_host):
    """what a dictionary does not name stays as the group has it"""
    p, q = leaf(5, dtype=torch.bfloat16), leaf(6)
    groups = [dict(params=[p], master=True, eps=1e-6), dict(params=[q], state_bits=8)]
    opt = AdamW(groups, lr=1e-2)
    saved = torch_state((5,), dtype=torch.bfloat16, lr=3e-4)
    saved["param_groups"].append(dict(params=[1], lr=7e-4))
    opt.load_state_dict(saved)
    a, b = opt.param_groups
    assert a["master"] is True and a["state_bits"] == 32 and a["lr"] == 3e-4 and a["eps"] == 1e-8
    assert opt.state[p]["master"].dtype == torch.float32
    assert b["state_bits"] == 8 and b["master"] is False and b["lr"] == 7e-4 and b["eps"] == 1e-8
    # 32-bit moments for a group that keeps 8 bits: refused, not turned over
    saved["state"][1] = torch_state((6,))["state"][0]
    with pytest.raises(ValueError, match="exp_avg"):
        opt.load_state_dict(saved)
    assert opt.param_groups[1]["state_bits"] == 8


def test_loaded_rate_goes_into_the_tensor(on_host):
    """a rate on the optimizer's device stays the same tensor"""
    p, q = leaf(5), leaf(6)
    one, two = (torch.tensor(x) for x in (0.5, 0.25))
    opt = AdamW([dict(params=[p], lr=one), dict(params=[q], lr=two)])
    saved = copy.deepcopy(opt.state_dict())
    for a, b in ((0.125, 0.0625), (torch.tensor(2.0), torch.tensor([4.0], dtype=torch.float64))):
        saved["param_groups"][0]["lr"], saved["param_groups"][1]["lr"] = a, b
        opt.load_state_dict(saved)
        assert opt.param_groups[0]["lr"] is one and opt.param_groups[1]["lr"] is two
        assert (float(one), float(two)) == (float(a), float(b))
        saved["param_groups"][0]["lr"] = 9.0
        assert float(one) == float(a)
    # a number takes what comes
    opt.param_groups[0]["lr"] = 0.5
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 9.0
    # refused: nothing is written
    saved["param_groups"][1]["lr"] = torch.ones(2)
    with pytest.raises(ValueError, match="one number"):
        opt.load_state_dict(saved)
    assert float(two) == 4.0
    shared = torch.tensor(1.0)
    opt = AdamW([dict(params=[p]), dict(params=[q])], lr=shared)
    saved["param_groups"][1]["lr"] = 8.0
    with pytest.raises(ValueError, match="share one lr"):
        opt.load_state_dict(saved)
    assert float(shared) == 1.0 and opt.param_groups[1]["lr"] is shared
    saved["param_groups"][1]["lr"] = 9.0
    opt.load_state_dict(saved)
    assert float(shared) == 9.0 and opt.param_groups[0]["lr"] is shared


@pytest.mark.parametrize("bits", [32, 8])
def test_state_that_is_not_loaded_goes_back_to_zeros(on_host, bits):
    """in the tensors that are there: a captured step writes to them"""
    p, q = leaf(300, dtype=torch.bfloat16), leaf(40)
    opt = AdamW([p, q], state_bits=bits, master=True)
    empty = opt.state_dict()
    assert not empty["state"]
    opt.load_state_dict(empty)
    assert not opt.state          # nothing was there
    opt.init_state()
    fresh = copy.deepcopy(opt.state[p])
    for t in opt.state[p].values():
        if t is not opt.state[p].get("order"):
            t.view(torch.uint8).random_(0, 100) if t.dim() else t.fill_(7)
    was = dict(opt.state[p])
    with torch.no_grad():
        p.fill_(1.5)
    opt.load_state_dict(empty)
    assert set(opt.state) == {p, q}
    for k, t in opt.state[p].items():
        assert t is was[k]
        want = torch.full((300,), 1.5) if k == "master" else fresh[k]
        assert torch.equal(t.float(), want.float()), k


def test_load_hooks(on_host):
    """hooks before a load may change what is loaded, those behind it see it"""
    p = leaf(8)
    opt = AdamW([p], lr=1e-2)
    saved = torch_state((8,), lr=0.5)
    m = saved["state"][0]["exp_avg"].clone()
    seen = []

    def returns(_, d):
        state = {0: dict(d["state"][0], exp_avg=2 * d["state"][0]["exp_avg"])}
        return dict(d, state=state, param_groups=[dict(d["param_groups"][0], lr=0.25)])

    def changes(_, d):
        d["state"] = {0: dict(d["state"][0], step=torch.tensor(40.0))}

    def behind(o):
        seen.append((float(o.state[p]["exp_avg"][0]), int(o.state[p]["step"]), o.param_groups[0]["lr"]))
    handles = [opt.register_load_state_dict_pre_hook(returns),
               opt.register_load_state_dict_pre_hook(changes, prepend=True),
               opt.register_load_state_dict_post_hook(behind)]
    for _ in range(2):
        opt.load_state_dict(saved)
    assert seen == [(2 * float(m[0]), 40, 0.25)] * 2
    assert torch.equal(saved["state"][0]["exp_avg"], m) and saved["param_groups"][0]["lr"] == 0.5
    bad = copy.deepcopy(saved)
    bad["state"][0]["exp_avg_sq"] = torch.zeros(9)
    with pytest.raises(ValueError, match="exp_avg_sq"):
        opt.load_state_dict(bad)
    handles[0].remove()   # (it gives one group for any number)
    with pytest.raises(ValueError):
        opt.load_state_dict(dict(saved, param_groups=saved["param_groups"] * 2))
    assert len(seen) == 2   # nothing was loaded
    for h in handles[1:]:
        h.remove()
    opt.load_state_dict(saved)
    assert float(opt.state[p]["exp_avg"][0]) == float(m[0]) and opt.param_groups[0]["lr"] == 0.5


def test_refused_load_keeps_the_objects(on_host):
    """a group or a state that a program holds is still the optimizer's own"""
    p, q = leaf(8), leaf(9)
    opt = AdamW([dict(params=[p], lr=0.5), dict(params=[q], state_bits=8)])
    opt.init_state()
    groups, state, own = opt.param_groups, opt.state, list(opt.param_groups)
    options, entries = [dict(g) for g in own], {x: dict(s) for x, s in state.items()}
    bad = copy.deepcopy(opt.state_dict())
    bad["param_groups"][0]["lr"] = 0.125
    bad["state"][1]["exp_avg_scale"] = torch.zeros(1)
    with pytest.raises(ValueError, match="exp_avg_scale"):
        opt.load_state_dict(bad)
    assert opt.param_groups is groups and opt.state is state
    assert all(a is b for a, b in zip(groups, own)) and [dict(g) for g in own] == options
    assert state.keys() == entries.keys()
    for x, s in state.items():
        assert all(t is entries[x][k] for k, t in s.items())
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert opt.param_groups[0]["lr"] == 0.5 and opt.state[p]["exp_avg"] is entries[p]["exp_avg"]


@pytest.mark.parametrize("lr", [-1.0, float("nan")])
def test_rate_in_a_host_tensor_is_checked(lr):
    """like a number: before anything is changed, not between two groups"""
    with pytest.raises(ValueError, match="lr must not be negative"):
        AdamW([leaf(3)], lr=torch.tensor(lr))
    with pytest.raises(ValueError, match="lr must not be negative"):
        AdamW._check_options(dict(lr=torch.tensor([lr], dtype=torch.float64), betas=(0.9, 0.9)))


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_without_gradients_are_checked_too(on_host, bits):
    """a plan that is made while a parameter has none does not take it as it is
    then: its order may have changed since its state was made"""
    p, q = leaf(6, 40), leaf(5)
    opt = AdamW([p, q], state_bits=bits)
    opt.init_state()
    q.grad = torch.ones(5)
    was = p.data
    for other in (was.t().contiguous().t(), torch.zeros(6, 80)[:, ::2], torch.zeros(1).expand(6, 40),
                  was.t().contiguous(), was.double()):
        p.data = other
        plan = plans().AdamWPlan(-1, 0, 0, 0, opt.param_groups, opt.state)
        assert plan.fits(opt.param_groups, opt.state)        # nothing is done with it
        p.grad = torch.empty_strided(p.shape, p.stride(), dtype=p.dtype)
        assert not plan.fits(opt.param_groups, opt.state)
        p.grad = None
        p.data = was
    plan = plans().AdamWPlan(-1, 0, 0, 0, opt.param_groups, opt.state)
    p.grad = torch.ones(6, 40)
    assert plan.fits(opt.param_groups, opt.state)
    if bits == 8:   # without the record: a contiguous parameter's
        del opt.state[p]["order"]
        plan = plans().AdamWPlan(-1, 0, 0, 0, opt.param_groups, opt.state)
        assert plan.fits(opt.param_groups, opt.state)
        for bad in (torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 2), torch.zeros(4).long()):
            opt.state[p]["order"] = bad
            plan = plans().AdamWPlan(-1, 0, 0, 0, opt.param_groups, opt.state)
            assert not plan.fits(opt.param_groups, opt.state)

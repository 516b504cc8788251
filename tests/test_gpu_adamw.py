"""``training.AdamW`` against the update written out: to the bit where it is a sequence of fp32 operations (the moments, and what 8 bits
hold of them), and in 64 bits for the parameters.

Tolerances.  A parameter's change is a product of a quotient: five roundings and the scalars' own, less than 16 * 2^-24 of its size; the
parameter is scaled and rounded to its type: half a step, or with stochastic rounding a whole one."""
import collections
import copy
import gc
import io
import math
import threading

import pytest
import torch

from torchtune_amd import _lib
from torchtune_amd.training import AdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
BLOCK = 128


def _tensors(shapes, dtype, seed=0, scale=1e-3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    params = []
    for shape in shapes:
        p = torch.nn.Parameter((torch.randn(shape, generator=g, device=DEV) * 0.05).to(dtype))
        size = torch.exp(torch.randn((), generator=g, device=DEV) * 2)
        p.grad = (torch.randn(shape, generator=g, device=DEV) * scale * size).to(dtype)
        params.append(p)
    return params


def _numbers(seed, step, tensor, n):
    """(for the second moment, for the first and the parameter): a small n through the library's own function"""
    lib = _lib.load()
    key = lib.ttamd_adamw_key(seed, step, tensor)
    r = torch.tensor([lib.ttamd_adamw_number(key, i) for i in range(n)], dtype=torch.int64)
    return r >> 16, r & 0xFFFF


def _padded(x):
    return torch.cat([x, x.new_zeros(-x.numel() % BLOCK)]).view(-1, BLOCK)


def _hold(x, numbers, mantissa):
    """codes and exponents of fp32 numbers, from the description of the format"""
    drop = 23 - mantissa
    size = x.view(torch.int32).to(torch.int64) & 0x7FFFFFFF
    k = (size.clamp(max=0x7F800000) + numbers * 2 ** (drop - 16) + 2 ** (drop - 17)) >> drop
    exponent = (_padded(k).amax(-1) >> mantissa).clamp(min=16)
    c = k - ((exponent - 15) << mantissa).repeat_interleave(BLOCK)[:x.numel()]
    if mantissa == 3:
        return torch.where(c < 1, 0, c + 128 * torch.signbit(x)).to(torch.uint8), exponent.to(torch.uint8)
    return torch.where(size == 0, 0, c.clamp(min=1)).to(torch.uint8), exponent.to(torch.uint8)


def _value(code, exponent, mantissa):
    code, field = code.to(torch.int64), exponent.to(torch.int64).repeat_interleave(BLOCK)[:code.numel()]
    size = code & (127 if mantissa == 3 else 255)
    bits = torch.where(size == 0, 0, (size + ((field - 15) << mantissa)) << (23 - mantissa)).to(torch.int32)
    v = bits.view(torch.float32)
    return torch.where(code > 127, -v, v) if mantissa == 3 else v


class _Reference:
    """One tensor's step on the CPU, fp32 moments to the bit and the parameter in 64 bits."""

    def __init__(self, p, number, bits, seed, **group):
        self.n, self.number, self.bits, self.seed, self.group = p.numel(), number, bits, seed, group
        self.step, self.m, self.v = 0, torch.zeros(self.n), torch.zeros(self.n)

    def take(self, p, g):
        c = self.group
        b1, b2 = c["betas"]
        self.step += 1
        p, g = p.detach().cpu().reshape(-1).double(), g.cpu().reshape(-1).float()
        m = self.m * b1 + g * (1 - b1)
        v = self.v * b2 + (g * g) * (1 - b2)
        change = c["lr"] / (1 - b1 ** self.step) * m.double() / (v.double().sqrt() / math.sqrt(1 - b2 ** self.step) + c["eps"])
        self.want, self.size = p * (1 - c["lr"] * c["weight_decay"]) - change, p.abs() + change.abs()
        if self.bits == 8:
            high, low = _numbers(self.seed, self.step, self.number, self.n)
            self.mc, self.vc = _hold(m, low, 3), _hold(v, high, 4)
            m, v = _value(*self.mc, 3), _value(*self.vc, 4)
        self.m, self.v = m, v

    def check(self, p, state, whole_step=False):
        eps = torch.finfo(p.dtype).eps
        off = (p.detach().cpu().reshape(-1).double() - self.want).abs()
        bound = self.want.abs() * eps / (1 if whole_step else 2) + 16 * U * self.size
        assert bool((off <= bound).all()), float((off / bound).max())
        assert int(state["step"]) == self.step
        if self.bits == 8:
            for name, (code, exponent) in (("exp_avg", self.mc), ("exp_avg_sq", self.vc)):
                assert torch.equal(state[name].cpu().reshape(-1), code), name
                assert torch.equal(state[name + "_exponent"].cpu(), exponent), name
        else:
            assert torch.equal(state["exp_avg"].cpu().reshape(-1), self.m) and torch.equal(state["exp_avg_sq"].cpu().reshape(-1), self.v)


SHAPES = [(1,), (7,), (128,), (129,), (16, 256), (4095,), (4097,), (33, 65), (0,), (2, 3, 2048)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("stochastic", [False, True])
def test_steps_over_many_tensors(dtype, bits, stochastic):
    params = _tensors(SHAPES, dtype)
    group = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    opt = AdamW(params, **group, state_bits=bits, stochastic_rounding=stochastic, seed=7)
    refs = [_Reference(p, i, bits, 7, **group) for i, p in enumerate(params)]
    for step in range(3):
        before = [p.detach().clone() for p in params]
        if step:
            for p in params:
                p.grad = torch.randn_like(p) * 1e-3 * 10 ** step
        opt.step()
        for p, b, r in zip(params, before, refs):
            r.take(b, p.grad)
            r.check(p, opt.state[p], stochastic and dtype == torch.bfloat16)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_holds_some_without_gradients(bits):
    """Groups with their own rates, tensors that join later and so count their own steps, two types."""
    params = _tensors([(5 + i % 97,) for i in range(500)], torch.float32) + _tensors([(64,), (65,)], torch.bfloat16, 1)
    gone = [p.grad for p in params]
    groups = [{"params": params[:300], "lr": 1e-2}, {"params": params[300:], "weight_decay": 0.0}]
    opt = AdamW(groups, lr=1e-3, betas=(0.8, 0.9), state_bits=bits, seed=3)
    scalars = [dict(lr=1e-2 if i < 300 else 1e-3, betas=(0.8, 0.9), eps=1e-8, weight_decay=0.01 if i < 300 else 0.0) for i in range(len(params))]
    refs = [_Reference(p, i, bits, 3, **c) for i, (p, c) in enumerate(zip(params, scalars))]
    for step in range(3):
        used = [i for i in range(len(params)) if step == 2 or i % 5 != step]
        for i, p in enumerate(params):
            p.grad = gone[i] if i in used else None
        before = [p.detach().clone() for p in params]
        opt.step()
        for i, (p, b, r) in enumerate(zip(params, before, refs)):
            if i in used:
                r.take(b, p.grad)
                r.check(p, opt.state[p])
            else:
                assert torch.equal(p.detach(), b) and (p in opt.state) == (r.step > 0)
    m, v = opt.moments()
    assert torch.equal(m.float().cpu(), torch.cat([r.m for r in refs])) and torch.equal(v.float().cpu(), torch.cat([r.v for r in refs]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_and_other_orders_in_memory(dtype, bits):
    """Parameters at odd places, transposed ones, ones with gaps; gradients that lie differently: the elements' own results."""
    g = torch.Generator(device=DEV).manual_seed(2)
    base = (torch.randn(4000, generator=g, device=DEV) * 0.1).to(dtype)
    wide = (torch.randn(40, 50, generator=g, device=DEV) * 0.1).to(dtype)
    guard = base.clone(), wide.clone()
    params = [torch.nn.Parameter(t) for t in (base[1:400], base[401:401 + 33 * 9].view(9, 33).t(), wide[:, 3:20], base[1000:3000].view(2, 1000))]
    grads = [torch.randn(p.shape, generator=g, device=DEV).to(dtype) * 1e-2 for p in params]
    grads[0] = torch.stack([grads[0], grads[0]], -1)[:, 0]  # with gaps
    grads[3] = grads[3].t().contiguous().t()
    for p, x in zip(params, grads):
        p.grad = x
    group = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    opt = AdamW(params, **group, state_bits=bits, seed=1)
    flat = [p.t() if i == 1 else p for i, p in enumerate(params)]  # in the order in memory
    refs = [_Reference(p, i, bits, 1, **group) for i, p in enumerate(params)]
    for _ in range(2):
        before = [p.detach().clone() for p in flat]
        opt.step()
        for i, (p, b, r) in enumerate(zip(flat, before, refs)):
            r.take(b, (grads[i].t() if i == 1 else grads[i]).contiguous())
            state = dict(opt.state[params[i]])
            assert state["exp_avg"].shape == params[i].shape
            if i == 1:
                state["exp_avg"], state["exp_avg_sq"] = state["exp_avg"].t(), state["exp_avg_sq"].t()
            r.check(p, state)
    same = torch.ones(4000, dtype=torch.bool, device=DEV)
    for lo, hi in ((1, 400), (401, 401 + 297), (1000, 3000)):
        same[lo:hi] = False
    assert torch.equal(base[same], guard[0][same])
    assert torch.equal(wide[:, :3], guard[1][:, :3]) and torch.equal(wide[:, 20:], guard[1][:, 20:])


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_whose_memory_moves(bits):
    """``p.data = ..`` between steps, as offloading and resharding do: the new memory is stepped, the old left alone."""
    results = []
    for move in (False, True):
        params = _tensors([(300,), (4096,), (5000,)], torch.bfloat16)
        opt = AdamW(params, lr=1e-2, state_bits=bits)
        opt.step()
        old = params[1].data
        kept = old.clone()
        if move:
            params[1].data = old.clone()
        for _ in range(2):
            opt.step()
        assert not move or torch.equal(old, kept)
        results.append([p.detach().clone() for p in params] + list(opt.moments()))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_zero_tiny_and_huge_size(bits):
    n = 8 * BLOCK
    p = torch.nn.Parameter(torch.randn(n, device=DEV))
    grad = torch.zeros(n, device=DEV)
    grad[BLOCK:2 * BLOCK] = torch.logspace(-30, 3, BLOCK, device=DEV)   # a block over many powers
    grad[2 * BLOCK:3 * BLOCK] = 1e-22                                   # squares below the smallest normal number
    grad[3 * BLOCK:4 * BLOCK] = 1e18
    grad[4 * BLOCK] = -5.0
    grad[5 * BLOCK:6 * BLOCK] = torch.linspace(-1, 1, BLOCK, device=DEV)
    group = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    opt, r = AdamW([p], **group, state_bits=bits, seed=9), None
    r = _Reference(p, 0, bits, 9, **group)
    for sign in (1, -1, 0.5, 0):
        p.grad = grad * sign
        before = p.detach().clone()
        opt.step()
        r.take(before, p.grad)
        r.check(p, opt.state[p])
    assert torch.equal(p.detach()[:BLOCK].isfinite().cpu(), torch.ones(BLOCK, dtype=torch.bool))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_gradient_that_is_not_finite(bits, bad):
    p = torch.nn.Parameter(torch.randn(4 * BLOCK, device=DEV))
    opt = AdamW([p], lr=1e-2, state_bits=bits)
    p.grad = torch.randn_like(p)
    opt.step()
    p.grad = torch.randn_like(p)
    p.grad[BLOCK + 5] = bad
    opt.step()
    for _ in range(2):
        p.grad = torch.randn_like(p)
        opt.step()
    here = torch.zeros(4 * BLOCK, dtype=torch.bool, device=DEV)
    here[BLOCK + 5] = True
    assert bool(torch.isnan(p.detach()[here]).all()) and bool(torch.isfinite(p.detach()[~here]).all())


def test_eight_bits_are_right_on_average():
    """4096 elements with the same gradient: their held moments scatter around the fp32 ones.  A rounding's standard deviation is
    at most half a step (2^-4 of the size for exp_avg, 2^-5 for exp_avg_sq), its mean's a 64th of that; four of those are allowed, and the
    steps before add up: exp_avg remembers 10, exp_avg_sq up to all 200 of them, but in quadrature.  Rounding to nearest would leave exp_avg_sq
    where a step of 0.1 % is lost, at less than a tenth of its value."""
    n = 4096
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8, seed=11)
    g = 0.37
    for step in range(1, 201):
        p.grad = torch.full((n,), g, device=DEV)
        opt.step()
    m, v = (x.double() for x in opt.moments())
    want_m, want_v = g * (1 - 0.9 ** 200), g * g * (1 - 0.999 ** 200)
    assert abs(float(m.mean()) / want_m - 1) < 4 / 64 * 2 ** -4 * math.sqrt(10)
    assert abs(float(v.mean()) / want_v - 1) < 4 / 64 * 2 ** -5 * math.sqrt(200)
    assert float(v.std()) > 0  # the elements' numbers differ


def test_stochastic_rounding_keeps_small_updates():
    """Changes of a hundredth of bf16's step: lost to the nearest, kept on average.  100 steps of the same sign move each of
    65536 elements by about one step, with a standard deviation of at most sqrt(100) / 2 steps; the mean's is a 256th of it."""
    n, steps = 65536, 100
    change = 2.0 ** -8 / 100
    results = []
    for stochastic in (False, True):
        p = torch.nn.Parameter(torch.full((n,), 1.0, device=DEV, dtype=torch.bfloat16))
        opt = AdamW([p], lr=change, betas=(0.0, 0.0), eps=0.0, weight_decay=0.0, stochastic_rounding=stochastic, seed=5)
        for _ in range(steps):
            p.grad = -torch.ones_like(p)
            opt.step()
        results.append(p.detach().double())
    assert bool((results[0] == 1).all())
    assert abs(float(results[1].mean()) - 1 - steps * change) < 4 * 2 ** -7 * math.sqrt(steps) / 2 / 256


def test_runs_repeat_and_seeds_differ():
    def run(seed):
        params = _tensors(SHAPES, torch.bfloat16)
        opt = AdamW(params, lr=1e-2, state_bits=8, stochastic_rounding=True, seed=seed)
        for _ in range(2):
            opt.step()
        return [p.detach().clone() for p in params] + list(opt.moments())

    a, b, c = run(1), run(1), run(2)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and not all(torch.equal(x, y) for x, y in zip(a, c))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["state_dict", "file", "pickle", "deepcopy"])
def test_saved_and_continued(bits, how):
    def fresh():
        return _tensors(SHAPES, torch.bfloat16)

    def grads(params, step):
        g = torch.Generator(device=DEV).manual_seed(step)
        for p in params:
            p.grad = (torch.randn(p.shape, generator=g, device=DEV) * 1e-3).to(p.dtype)

    make = lambda params: AdamW([{"params": params[:4], "lr": 1e-3}, {"params": params[4:]}], lr=1e-2, state_bits=bits, stochastic_rounding=True, seed=2)
    params = fresh()
    opt = make(params)
    for step in range(2):
        grads(params, step)
        opt.step()
    if how == "deepcopy":
        other, again = copy.deepcopy((params, opt))
    else:
        other = [torch.nn.Parameter(p.detach().clone()) for p in params]
        again = make(other)
        saved = opt.state_dict()
        if how == "file":
            f = io.BytesIO()
            torch.save(saved, f)
            f.seek(0)
            saved = torch.load(f, weights_only=True)
        if how == "pickle":
            f = io.BytesIO()
            torch.save(opt, f)
            f.seek(0)
            saved = torch.load(f, weights_only=False).state_dict()  # written four lines above
        again.load_state_dict(saved)
    for step in range(2, 4):
        for ps, o in ((params, opt), (other, again)):
            grads(ps, step)
            o.step()
    for p, q in zip(params, other):
        assert torch.equal(p.detach(), q.detach())
        for name in opt.state[p]:
            assert torch.equal(opt.state[p][name], again.state[q][name]), name
            assert opt.state[p][name].dtype == again.state[q][name].dtype
    assert again.param_groups[0]["lr"] == 1e-3


def test_a_state_dict_of_torchs_optimizer():
    params = _tensors([(33, 7), (100,)], torch.float32)
    theirs = torch.optim.AdamW(params, lr=1e-2, fused=True)
    theirs.step()
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    ours = AdamW(other, lr=1.0)
    ours.load_state_dict(theirs.state_dict())
    for p, q in zip(params, other):
        q.grad = p.grad.clone()
    theirs.step()
    ours.step()
    for p, q in zip(params, other):
        assert float((p - q).detach().abs().max()) < 1e-2 * 64 * U + 2 * U * float(p.detach().abs().max())
        assert int(ours.state[q]["step"]) == 2
    with pytest.raises(ValueError, match="expected"):
        AdamW(other, state_bits=8).load_state_dict(theirs.state_dict())


def test_states_of_the_other_width_are_refused_and_nothing_changes():
    params = _tensors([(300,)], torch.float32)
    eight, wide = AdamW(params, state_bits=8), AdamW(params, state_bits=32)
    eight.step()
    wide.step()
    kept = wide.state[params[0]]["exp_avg"].clone()
    with pytest.raises(ValueError, match="bits"):
        wide.load_state_dict(eight.state_dict())
    short = wide.state_dict()
    short["state"] = {0: {**short["state"][0], "exp_avg": torch.zeros(299)}}
    with pytest.raises(ValueError, match="elements"):
        wide.load_state_dict(short)
    assert torch.equal(wide.state[params[0]]["exp_avg"], kept)


def test_moments_of_transposed_parameters_are_in_the_order_of_their_memory():
    """Also where not all parameters have states yet."""
    p = torch.nn.Parameter(torch.randn(6, 5, device=DEV).t())
    late = torch.nn.Parameter(torch.randn(7, device=DEV))
    q = torch.nn.Parameter(torch.randn(3, device=DEV))
    opt = AdamW([p, late, q], betas=(0.0, 0.0))
    p.grad, q.grad = torch.randn(5, 6, device=DEV), torch.randn(3, device=DEV)
    opt.step()
    m, _ = opt.moments()
    assert torch.equal(m, torch.cat([p.grad.t().reshape(-1), q.grad]))
    late.grad = torch.randn(7, device=DEV)
    opt.step()
    m, _ = opt.moments()
    assert torch.equal(m, torch.cat([p.grad.t().reshape(-1), late.grad, q.grad]))
    alone = AdamW([p], betas=(0.0, 0.0))
    alone.step()
    assert torch.equal(alone.moments()[0], p.grad.t().reshape(-1)) and torch.equal(alone.state[p]["exp_avg"], p.grad)
    p.data = p.data.contiguous()
    with pytest.raises(RuntimeError, match="order"):
        alone.step()
    assert int(alone.state[p]["step"]) == 1


def test_a_refused_step_leaves_its_states_visible_and_uncounted():
    a, b = (torch.nn.Parameter(torch.ones(4, device=DEV)) for _ in range(2))
    opt = AdamW([a, b], lr=0.1)
    a.grad, b.grad = torch.ones(4, device=DEV), torch.ones(4, device=DEV)
    opt.param_groups[0]["betas"] = (1.5, 0.9)
    with pytest.raises(ValueError, match="beta"):
        opt.step()
    assert len(opt.state) == 2 and int(opt.state[a]["step"]) == 0 and bool((a == 1).all())
    opt.param_groups[0]["betas"] = (0.9, 0.9)
    opt.step()
    assert int(opt.state[b]["step"]) == 1 and bool((b != 1).all())


def test_threads_may_step_their_own_and_the_same_optimizer():
    """Ten steps from each of four threads: as many steps as asked for, of one constant gradient in whatever order."""
    p = torch.nn.Parameter(torch.ones(5000, device=DEV))
    mine = [torch.nn.Parameter(torch.ones(5000, device=DEV)) for _ in range(4)]
    shared, own = AdamW([p], lr=1e-3, state_bits=8), [AdamW([x], lr=1e-3, state_bits=8) for x in mine]
    p.grad = torch.ones_like(p)
    shared.step()
    torch.cuda.synchronize()

    def work(x, opt):
        x.grad = torch.ones_like(x)
        for _ in range(10):
            opt.step()
            shared.step()

    threads = [threading.Thread(target=work, args=args) for args in zip(mine, own)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert int(shared.state[p]["step"]) == 41 and all(int(o.state[x]["step"]) == 10 for o, x in zip(own, mine))
    assert all(torch.equal(mine[0], x) for x in mine[1:])


def test_more_than_2_to_the_31_elements():
    """The first, the middle and the last of a parameter of 2^31 + 5000 elements: the steps of a small one."""
    n = 2 ** 31 + 5000
    p = torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=torch.bfloat16))
    p.grad = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(0)
    small = []
    for at in (0, 2 ** 31 - 2048, n - 2048):
        part = slice(at, at + 2048)
        p.data[part] = torch.randn(2048, generator=g, device=DEV).to(torch.bfloat16)
        p.grad[part] = torch.randn(2048, generator=g, device=DEV).to(torch.bfloat16)
        small.append((part, torch.nn.Parameter(p.detach()[part].clone())))
        small[-1][1].grad = p.grad[part].clone()
    opt = AdamW([p], lr=1e-2)
    others = AdamW([q for _, q in small], lr=1e-2)
    for _ in range(2):
        opt.step()
        others.step()
    for part, q in small:
        assert torch.equal(p.detach()[part], q.detach()) and torch.equal(opt.state[p]["exp_avg_sq"][part], others.state[q]["exp_avg_sq"])
    assert not bool(p.detach()[4096:2 ** 31 - 4096].any())
    del opt, others
    opt = AdamW([p], lr=0.0, betas=(0.0, 0.0), state_bits=8)  # the moments are the gradient and its square, rounded
    opt.step()
    m, v = opt.moments()
    for part, q in small:
        assert bool(((m[part].float() - q.grad.float()).abs() <= q.grad.float().abs() / 8 + 2.0 ** -14 * q.grad.float().abs().max()).all())
        assert bool(((v[part].float() - q.grad.float() ** 2).abs() <= q.grad.float() ** 2 / 16 + 2.0 ** -14 * q.grad.float().abs().max() ** 2).all())
    assert not bool(m[4096:2 ** 31 - 4096].any()) and not bool(v[4096:2 ** 31 - 4096].any())


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(10, device=DEV))
    opt = AdamW([p])
    p.grad = torch.sparse_coo_tensor([[1]], [1.0], (10,), device=DEV)
    with pytest.raises(RuntimeError, match="dense"):
        opt.step()
    half = torch.nn.Parameter(torch.zeros(10, device=DEV, dtype=torch.float16))
    half.grad = torch.zeros_like(half)
    with pytest.raises(TypeError, match="not supported"):
        AdamW([half]).step()
    wide = torch.nn.Parameter(torch.zeros(1, device=DEV).expand(10))
    wide.grad = torch.ones(10, device=DEV)
    with pytest.raises(RuntimeError, match="single memory location"):
        AdamW([wide]).step()
    q = torch.nn.Parameter(torch.zeros(10, device=DEV))
    q.grad = torch.ones_like(q)
    opt = AdamW([q], lr=0.5)
    opt.step()
    after = q.detach().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="graph"):
            opt.step()
    assert int(opt.state[q]["step"]) == 1 and torch.equal(q.detach(), after)
    opt.param_groups[0]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        opt.step()


def test_closures_hooks_schedulers_and_versions():
    w = torch.nn.Parameter(torch.ones(3, device=DEV))
    opt = AdamW([w], lr=0.1, weight_decay=0.0)
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, lambda step: 1.0 / (1 + step))
    seen = []
    opt.register_step_post_hook(lambda *a: seen.append(1))

    def closure():
        opt.zero_grad()
        loss = (w * w).sum()
        loss.backward()
        return loss

    assert float(opt.step(closure)) == 3.0 and seen == [1]
    assert float((w.detach() - 0.9).abs().max()) < 1e-6
    schedule.step()
    assert opt.param_groups[0]["lr"] == 0.05
    before = w._version
    out = (w * w).sum()
    w.grad = torch.ones_like(w)
    opt.step()
    assert w._version > before
    with pytest.raises(RuntimeError, match="inplace"):
        out.backward()
    opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(2, device=DEV))]})
    opt.param_groups[1]["params"][0].grad = torch.ones(2, device=DEV)
    opt.step()
    assert len(opt.state) == 2 and int(opt.state[opt.param_groups[1]["params"][0]]["step"]) == 1


def test_on_another_stream():
    """The states made on one stream, steps on another, the optimizer gone while they run."""
    results = []
    for streams in (1, 2):
        params = _tensors([(1 << 20,)] * 4, torch.float32)
        opt = AdamW(params, lr=1e-2, state_bits=8, seed=4)
        opt.step()
        side = torch.cuda.Stream() if streams == 2 else torch.cuda.current_stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(5):
                opt.step()
        del opt
        junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV) for _ in range(8)]
        torch.cuda.current_stream().wait_stream(side)
        results.append(torch.cat([p.detach() for p in params]))
        del junk
    assert torch.equal(*results)


def test_eight_bit_states_are_not_loaded_into_another_order():
    """A block's exponent is that of neighbours in memory.  Rows of very different sizes, so that another block's exponent would show."""
    g = torch.Generator(device=DEV).manual_seed(0)
    grad = torch.randn(64, 64, generator=g, device=DEV) * torch.exp(4 * torch.randn(64, 1, generator=g, device=DEV))
    p = torch.nn.Parameter(torch.zeros(64, 64, device=DEV).t())
    p.grad = grad
    opt = AdamW([p], state_bits=8)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    moments = [x.clone() for x in opt.moments()]
    rows = torch.nn.Parameter(p.detach().contiguous())
    with pytest.raises(ValueError, match="another order"):
        AdamW([rows], state_bits=8).load_state_dict(saved)
    again = AdamW([torch.nn.Parameter(torch.zeros(64, 64, device=DEV).t())], state_bits=8)
    again.load_state_dict(saved)
    assert all(torch.equal(a, b) for a, b in zip(again.moments(), moments))
    # the same parameter, laid out anew: its own states are refused, by a load and by a group that has grown, and are still there
    p.data = p.data.contiguous()
    with pytest.raises(ValueError, match="another order"):
        opt.load_state_dict(saved)
    late = torch.nn.Parameter(torch.zeros(5, device=DEV))
    late.grad = torch.ones(5, device=DEV)
    opt.param_groups[0]["params"].append(late)
    with pytest.raises(ValueError, match="another order"):
        opt.step()
    assert int(opt.state[p]["step"]) == 1 and torch.equal(opt.state[p]["exp_avg"], saved["state"][0]["exp_avg"]) and bool((late == 0).all())
    p.data = p.data.t().contiguous().t()
    opt.step()
    assert int(opt.state[p]["step"]) == 2 and int(opt.state[late]["step"]) == 1


def test_a_run_continued_by_an_optimizer_built_with_another_seed():
    params = _tensors([(3000,), (200,)], torch.bfloat16)
    opt = AdamW(params, lr=1e-3, state_bits=8, stochastic_rounding=True, seed=9)
    opt.step()
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = AdamW(other, lr=1.0, state_bits=8, seed=1)
    again.load_state_dict(opt.state_dict())
    for p, q in zip(params, other):
        q.grad = p.grad.clone()
    for _ in range(2):
        opt.step()
        again.step()
    for p, q in zip(params, other):
        assert torch.equal(p.detach(), q.detach()) and all(torch.equal(opt.state[p][name], again.state[q][name]) for name in opt.state[p])


def test_options_of_the_groups_own():
    """Width, seed and rounding of each group, as an optimizer of its own would have them."""
    def groups(params):
        return [{"params": params[:2], "state_bits": 8, "seed": 5}, {"params": params[2:4], "seed": 6, "stochastic_rounding": True},
                {"params": params[4:], "state_bits": 8, "seed": 7, "stochastic_rounding": True}]

    shapes = [(300,), (129,)] * 3
    params = _tensors(shapes, torch.bfloat16)
    opt = AdamW(groups(params), lr=1e-2)
    scalars = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)
    refs = [_Reference(p, i, (8, 32, 8)[i // 2], 5 + i // 2, **scalars) for i, p in enumerate(params)]
    for _ in range(2):
        before = [p.detach().clone() for p in params]
        opt.step()
        for i, (p, b, r) in enumerate(zip(params, before, refs)):
            r.take(b, p.grad)
            r.check(p, opt.state[p], whole_step=i >= 2)
    m, v = opt.moments()
    assert torch.equal(m.float().cpu(), torch.cat([r.m for r in refs])) and torch.equal(v.float().cpu(), torch.cat([r.v for r in refs]))
    # stochastic rounding shows: some parameters are not the nearest to what they should be
    off = torch.cat([(p.detach().cpu().double() - r.want).abs() / (r.want.abs() * torch.finfo(p.dtype).eps / 2 + 16 * U * r.size) for p, r in zip(params[2:], refs[2:])])
    assert bool((off > 1).any())
    # the width of states that are there does not change
    opt.param_groups[0]["state_bits"] = 32
    with pytest.raises(ValueError, match="bits"):
        opt.step()
    assert all(int(opt.state[p]["step"]) == 2 for p in params)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("with_states", [False, True])
def test_a_parameter_replaced_in_its_group(bits, with_states):
    """``param_groups[0]["params"][i] = other``, as resizing and pruning do: the new one is stepped, from states given for it, and the old
    one is left alone; the neighbours go on."""
    params = _tensors([(300,), (129,), (40,)], torch.float32)
    group = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    opt = AdamW(params, **group, state_bits=bits, seed=4)
    refs = [_Reference(p, i, bits, 4, **group) for i, p in enumerate(params)]

    def step(used):
        before = [p.detach().clone() for p in used]
        opt.step()
        for p, b, r in zip(used, before, refs):
            r.take(b, p.grad)
            r.check(p, opt.state[p])

    step(params)
    old, new = params[1], _tensors([(129,) if with_states else (200,)], torch.float32, 7)[0]
    kept = old.detach().clone()
    opt.param_groups[0]["params"][1] = new
    if with_states:
        opt.state[new] = {name: t.clone() for name, t in opt.state.pop(old).items()}
    else:
        refs[1] = _Reference(new, 1, bits, 4, **group)
    for _ in range(2):
        step([params[0], new, params[2]])
    assert torch.equal(old.detach(), kept) and int(opt.state[new]["step"]) == (3 if with_states else 2)


@pytest.mark.parametrize("how", ["clear", "replace", "pop"])
def test_states_taken_out_begin_anew(how):
    """As an optimizer made at that point would go on, for the parameters whose states are gone."""
    params = _tensors([(300,), (129,)], torch.float32)
    group = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    opt = AdamW([{"params": params[:1]}, {"params": params[1:]}], **group, state_bits=8, seed=4)
    refs = [_Reference(p, i, 8, 4, **group) for i, p in enumerate(params)]
    for step in range(4):
        if step == 2:
            if how == "clear":
                opt.state.clear()
            elif how == "replace":
                opt.state = collections.defaultdict(dict)
            else:
                opt.state.pop(params[0])
            for i, p in enumerate(params[:1 if how == "pop" else 2]):
                refs[i] = _Reference(p, i, 8, 4, **group)
        before = [p.detach().clone() for p in params]
        opt.step()
        for p, b, r in zip(params, before, refs):
            r.take(b, p.grad)
            r.check(p, opt.state[p])
    assert len(opt.state_dict()["state"]) == 2


def _blocks_of_all_kinds():
    """Two groups; the first with two types and a parameter that joined later: four blocks in all."""
    params = _tensors([(300,), (8, 16)], torch.float32) + _tensors([(129,)], torch.bfloat16, 1) + _tensors([(9, 16)], torch.float32, 2) + _tensors([(70,), (6, 5)], torch.float32, 3)
    opt = AdamW([{"params": params[:4]}, {"params": params[4:]}], lr=1e-2)
    late, params[3].grad = params[3].grad, None
    opt.step()
    params[3].grad = late
    opt.step()
    return params, opt


@pytest.mark.parametrize("which", [1, 3, 5])
@pytest.mark.parametrize("why", ["order", "size", "gone"])
def test_a_step_refused_for_one_parameter_moves_none(which, why):
    params, opt = _blocks_of_all_kinds()
    before, counts = [p.detach().clone() for p in params], [int(opt.state[p]["step"]) for p in params]
    moments = [x.clone() for x in opt.moments()]
    p, kept = params[which], params[which].data
    if why == "order":
        p.data = kept.t().contiguous().t()
    elif why == "size":
        p.grad = None
        p.data = torch.zeros(3, device=DEV)
        p.grad = torch.ones(3, device=DEV)
    else:
        g = p.grad
        p.grad = None
        p.data = kept.cpu()
        p.grad = g.cpu()
    with pytest.raises(RuntimeError, match="order" if why == "order" else "size" if why == "size" else "AMD GPU"):
        opt.step()
    p.data = kept
    assert all(torch.equal(q.detach(), b) for q, b in zip(params, before)) and [int(opt.state[q]["step"]) for q in params] == counts
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), moments))


@pytest.mark.parametrize("name,bad", [("betas", (0.9, 1.5)), ("betas", (math.nan, 0.9)), ("eps", -1.0), ("eps", math.nan), ("amsgrad", True), ("maximize", True)])
def test_a_step_refused_for_one_group_moves_none(name, bad):
    params, opt = _blocks_of_all_kinds()
    before, counts = [p.detach().clone() for p in params], [int(opt.state[p]["step"]) for p in params]
    kept = opt.param_groups[1].get(name)
    opt.param_groups[1][name] = bad
    with pytest.raises(ValueError, match="eps|amsgrad"):
        opt.step()
    assert all(torch.equal(q.detach(), b) for q, b in zip(params, before)) and [int(opt.state[q]["step"]) for q in params] == counts
    opt.param_groups[1][name] = kept
    opt.step()
    assert [int(opt.state[q]["step"]) for q in params] == [n + 1 for n in counts]


def test_a_parameter_with_gaps_whose_memory_and_shape_change():
    """As many elements in the same order, laid out with other gaps."""
    g = torch.Generator(device=DEV).manual_seed(5)
    wide, other = torch.randn(12, 10, generator=g, device=DEV), torch.zeros(8, 30, device=DEV)
    group = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    p = torch.nn.Parameter(wide[:, 1:9])
    opt, r = AdamW([p], **group), _Reference(p, 0, 32, 0, **group)
    for shape in ((12, 8), (8, 12), (8, 12)):
        if tuple(p.shape) != shape:
            other[:, 3:15] = p.detach().reshape(8, 12)
            p.grad = None
            p.data = other[:, 3:15]
        p.grad = torch.randn(shape, generator=g, device=DEV)
        before = p.detach().clone()
        opt.step()
        r.take(before, p.grad)
        r.check(p, opt.state[p])
    assert bool((other[:, :3] == 0).all()) and bool((other[:, 15:] == 0).all())


@pytest.mark.parametrize("what", ["parameter", "gradient"])
def test_memory_that_was_given_up_and_came_back(what):
    """After the first step, so that the table of addresses is there: refused while it is away, and nothing moves."""
    params = _tensors([(300,), (129,)], torch.float32)
    opt = AdamW(params, lr=1e-2)
    opt.step()
    t = params[1] if what == "parameter" else params[1].grad
    kept, first, size = t.detach().clone(), params[0].detach().clone(), t.untyped_storage().nbytes()
    torch.cuda.synchronize()
    t.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match=f"memory of a {what}"):
        opt.step()
    t.untyped_storage().resize_(size)
    t.detach().copy_(kept)
    assert torch.equal(params[0].detach(), first) and [int(opt.state[p]["step"]) for p in params] == [1, 1]
    opt.step()
    assert bool((params[0].detach() != first).any()) and [int(opt.state[p]["step"]) for p in params] == [2, 2]


def test_parameters_that_share_memory_are_refused():
    """In one launch they would be stepped at the same time.  Columns of one matrix share none; one of two that share may go alone."""
    base = torch.ones(40, 50, device=DEV)
    a, b, c = (torch.nn.Parameter(t) for t in (base[:, 3:20], base[:, 20:33], base[4:6, 10:25]))
    opt = AdamW([a, b, c], lr=0.1)
    for p in (a, b, c):
        p.grad = torch.ones(p.shape, device=DEV)
    with pytest.raises(RuntimeError, match="parameters 0 and 2.* share memory"):
        opt.step()
    assert bool((base == 1).all()) and all(int(opt.state[p]["step"]) == 0 for p in (a, b, c))
    c.grad = None
    opt.step()
    assert [int(opt.state[p]["step"]) for p in (a, b, c)] == [1, 1, 0]
    assert bool((base[:, 3:33] != 1).all()) and bool((base[:, :3] == 1).all()) and bool((base[:, 33:] == 1).all())
    # memory that moves into a neighbour's
    x, y = (torch.nn.Parameter(torch.ones(100, device=DEV)) for _ in range(2))
    x.grad, y.grad = torch.ones(100, device=DEV), torch.ones(100, device=DEV)
    opt = AdamW([x, y], lr=0.1)
    opt.step()
    after = x.detach().clone()
    kept, both = y.data, torch.ones(150, device=DEV)
    x.data, y.data = both[:100], both[50:]
    with pytest.raises(RuntimeError, match="share memory"):
        opt.step()
    assert bool((both == 1).all())
    x.data, y.data = after, kept
    opt.step()
    assert int(opt.state[x]["step"]) == 2


def test_threads_take_the_first_step_of_one_optimizer():
    """Four threads at once, no states before: as many steps as asked for, in one set of states, which another thread reads meanwhile."""
    for _ in range(5):
        params = _tensors([(5000,)] * 20, torch.float32)
        opt, alone = AdamW(params, lr=1e-3, state_bits=8), None
        torch.cuda.synchronize()
        start = threading.Barrier(5)

        def work():
            start.wait()
            for _ in range(5):
                opt.step()

        def read():
            start.wait()
            for _ in range(20):
                opt.state_dict()

        threads = [threading.Thread(target=work) for _ in range(4)] + [threading.Thread(target=read)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        other = _tensors([(5000,)] * 20, torch.float32)
        alone = AdamW(other, lr=1e-3, state_bits=8)
        for _ in range(20):
            alone.step()
        for p, q in zip(params, other):
            assert int(opt.state[p]["step"]) == 20 and torch.equal(p.detach(), q.detach())
            assert all(torch.equal(opt.state[p][name], alone.state[q][name]) for name in opt.state[p])


@pytest.mark.parametrize("bits", [32, 8])
def test_hooks_of_a_load(bits):
    """Hooks before it may change the states; hooks after it find them in place, and what they write there counts."""
    params = _tensors([(300,), (33, 7)], torch.bfloat16)
    opt = AdamW(params, lr=1e-2, state_bits=bits)
    for _ in range(2):
        opt.step()
    saved = opt.state_dict()
    kept = copy.deepcopy(saved["state"])
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = AdamW(other, lr=1e-2, state_bits=bits)

    def count_from_seven(o, d):
        return {**d, "state": {k: {**s, "step": torch.tensor(7)} for k, s in d["state"].items()}}

    def after(o):
        for i, q in enumerate(other):
            assert int(o.state[q]["step"]) == 7 and o.state[q]["exp_avg"].data_ptr() != saved["state"][i]["exp_avg"].data_ptr()
            assert all(torch.equal(o.state[q][name], kept[i][name]) for name in kept[i] if name != "step")
        o.state[other[0]]["exp_avg"].zero_()

    again.register_load_state_dict_pre_hook(count_from_seven)
    again.register_load_state_dict_post_hook(after)
    again.load_state_dict(saved)
    assert bool((again.state[other[0]]["exp_avg"] == 0).all()) and torch.equal(again.state[other[1]]["exp_avg"], kept[1]["exp_avg"])
    assert all(torch.equal(saved["state"][i][name], kept[i][name]) for i in kept for name in kept[i])  # what was loaded is not touched
    for q in other:
        q.grad = torch.zeros_like(q)
    again.step()
    assert bool((again.state[other[0]]["exp_avg"] == 0).all()) and [int(again.state[q]["step"]) for q in other] == [8, 8]


def test_a_group_that_cannot_take_over_its_states_keeps_them():
    """A group that has grown, one of whose states has been spoilt: an error, and no other state is lost."""
    params = _tensors([(300,), (129,)], torch.float32)
    opt = AdamW(params, lr=1e-2)
    opt.step()
    kept = [opt.state[p]["exp_avg"].clone() for p in params]
    opt.state[params[1]] = {**opt.state[params[1]], "step": "seven"}
    opt.param_groups[0]["params"].append(torch.nn.Parameter(torch.zeros(5, device=DEV)))
    with pytest.raises(ValueError, match="seven"):
        opt.step()
    assert int(opt.state[params[0]]["step"]) == 1 and all(torch.equal(opt.state[p]["exp_avg"], k) for p, k in zip(params, kept))
    opt.state[params[1]]["step"] = 1
    opt.step()
    assert [int(opt.state[p]["step"]) for p in params] == [2, 2]


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_holds_all_with_gradients(bits):
    """700 of one group in a step: a launch that is full, and the rest in another."""
    params = _tensors([(5 + i % 97,) for i in range(1000)], torch.float32)
    scalars = dict(lr=1e-2, betas=(0.8, 0.9), eps=1e-8, weight_decay=0.01)
    opt = AdamW([{"params": params[:700]}, {"params": params[700:]}], **scalars, state_bits=bits, seed=3)
    refs = [_Reference(p, i, bits, 3, **scalars) for i, p in enumerate(params)]
    for _ in range(2):
        before = [p.detach().clone() for p in params]
        opt.step()
        for p, b, r in zip(params, before, refs):
            r.take(b, p.grad)
            r.check(p, opt.state[p])


@pytest.mark.parametrize("b2", [0.95, 0.999])
def test_a_run_with_eight_bits_beside_one_with_32(b2):
    """200 steps on the same gradients, which change: blocks of different scale, a drift with noise half as large.

    An error of a held moment is ``b`` times the one before, plus that of the holding: ``e' = b e + d``.  ``d`` is 0 on average and within a step
    ``u`` of the number that is held, so that its variance is at most u^2 / 4; beside it a bias of at most 2^-16 u (numbers of 16 bits), the
    smallest code where the range ends (0 or that code is held), and four roundings of either run.  Variances of the elements add up; the sum
    of all errors, each over its block's scale, stays within six standard deviations and the bias.
    The change of a parameter is linear in the first moment.  In the second, of relative variance V <= 2^-10 min(steps, 1 / (1 - b2^2)), it
    is larger by 3/8 V on average, to second order; twice that is allowed, and 1 % for the first order over 65536 elements."""
    n, steps, b1 = 1 << 16, 200, 0.9
    g = torch.Generator(device=DEV).manual_seed(11)
    scale = torch.exp(3 * torch.randn(n // BLOCK, generator=g, device=DEV)).repeat_interleave(BLOCK)
    params = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for _ in range(2)]
    opts = [AdamW([p], lr=1e-3, betas=(b1, b2), weight_decay=0.0, state_bits=bits, seed=2) for p, bits in zip(params, (8, 32))]
    variance, bias = [torch.zeros(n, dtype=torch.float64, device=DEV) for _ in range(2)], [torch.zeros(n, dtype=torch.float64, device=DEV) for _ in range(2)]
    for _ in range(steps):
        grad = scale * (1 + 0.5 * torch.randn(n, generator=g, device=DEV))
        for p, opt in zip(params, opts):
            p.grad = grad
            opt.step()
        held, exact = ([x.double() for x in opt.moments()] for opt in opts)
        for k, (b, mantissa, name) in enumerate(((b1, 3, "exp_avg_exponent"), (b2, 4, "exp_avg_sq_exponent"))):
            field = opts[0].state[params[0]][name].double().repeat_interleave(BLOCK)
            least = torch.exp2(field - 142) * (1 + 2.0 ** -mantissa)
            h = held[k].abs()
            u = torch.where(h == 0, least, torch.exp2(torch.floor(torch.log2(h.clamp(min=1e-300)))) * 2.0 ** -mantissa)
            variance[k] = b * b * variance[k] + u * u / 4
            bias[k] = b * bias[k] + 2.0 ** -16 * u + torch.where(h <= least, least, 0.0) + 4 * U * (h + u + exact[k].abs())
    for k, unit in enumerate((scale.double(), scale.double() ** 2)):
        off = float(((held[k] - exact[k]) / unit).sum())
        bound = 6 * math.sqrt(float((variance[k] / unit ** 2).sum())) + float((bias[k] / unit).sum())
        assert abs(off) <= bound, (k, off, bound)
        assert bound < 0.05 * float((exact[k] / unit).sum().abs())  # a bound that says something
    far, wide = (float(p.detach().double().mean()) for p in params)
    tolerance = 0.75 * 2.0 ** -10 * min(steps, 1 / (1 - b2 * b2)) + 0.01
    assert wide < 0 and abs(far / wide - 1) <= tolerance, (far, wide, tolerance)


def test_small_elements_beside_a_large_one_in_eight_bits():
    """What a block's range of 2^15 leaves of them, as the format is described: first moments 0, second moments the smallest code, and so
    smaller changes than with 32 bits from the second step on (the first one's moments have not been held before they are used).  The next block
    is not touched by it.

    Of a gradient g = 1e-6: step 1 changes it by lr g / (g + eps).  In steps 2 and 3 the first moment is 0.1 g, over 1 - 0.9^t at most
    5.3e-7; the second at least 2^-16 of the large one's, 0.9e-3, so that its root over that of 1 - 0.999^3 is at least 2.1e-3: each changes
    it by at most 2.6e-4 lr."""
    p = torch.nn.Parameter(torch.zeros(2 * BLOCK, device=DEV))
    p.grad = torch.full((2 * BLOCK,), 1e-6, device=DEV)
    p.grad[0] = 1.0
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=8)
    for _ in range(3):
        opt.step()
    m, v = (x.float() for x in opt.moments())
    field = opt.state[p]["exp_avg_sq_exponent"].double()
    assert bool((m[1:BLOCK] == 0).all()) and bool((v[1:BLOCK].double() == 2.0 ** (float(field[0]) - 142) * 17 / 16).all())
    assert float(v[1]) > 2.0 ** -16 * float(v[0]) and bool((m[BLOCK:] > 0).all()) and bool((v[BLOCK:] < 1e-11).all())
    change, first = -p.detach().double(), 1e-2 * 1e-6 / (1e-6 + 1e-8)
    assert bool((change[1:BLOCK] > first * (1 - 16 * U)).all()) and bool((change[1:BLOCK] < first * (1 + 16 * U) + 2 * 2.6e-4 * 1e-2).all())
    assert float(change[BLOCK:].min()) > 2e-2


@pytest.mark.parametrize("bits", [32, 8])
def test_no_eps_and_no_gradient(bits):
    """0 / 0 where eps is 0: such an element keeps its place, but for the decay."""
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    p.grad = torch.zeros(300, device=DEV)
    p.grad[7] = 1.0
    opt = AdamW([p], lr=0.5, eps=0.0, weight_decay=0.25, state_bits=bits)
    opt.step()
    idle = torch.ones(300, dtype=torch.bool, device=DEV)
    idle[7] = False
    assert bool((p.detach()[idle] == 0.875).all()) and abs(float(p.detach()[7]) - 0.375) < 16 * U


def test_looking_for_states_moves_none():
    """An empty entry, made by asking for one that is not there, is no reason to make the states anew; one that is put in is."""
    params = _tensors([(300,), (129,), (40,)], torch.float32)
    params[1].grad, params[2].grad, kept = None, None, params[1].grad
    opt = AdamW(params, lr=1e-2)
    opt.step()
    at = opt.state[params[0]]["exp_avg"].data_ptr()
    assert not opt.state[params[1]]
    opt.step()
    assert opt.state[params[0]]["exp_avg"].data_ptr() == at and int(opt.state[params[0]]["step"]) == 2
    params[1].grad = kept
    opt.step()
    assert opt.state[params[0]]["exp_avg"].data_ptr() == at and [int(opt.state[p]["step"]) for p in params[:2]] == [3, 1]
    # given states for one that has none yet
    opt.state[params[2]] = {"step": 6, "exp_avg": torch.ones(40, device=DEV), "exp_avg_sq": torch.ones(40, device=DEV)}
    params[2].grad = torch.zeros(40, device=DEV)
    opt.step()
    assert [int(opt.state[p]["step"]) for p in params] == [4, 2, 7] and bool((opt.state[params[2]]["exp_avg"] - 0.9).abs().max() < 4 * U)


def test_memory_of_states_that_were_replaced():
    """New native sides do not keep the buffers of those before them."""
    params = _tensors([(1 << 20,), (1 << 20,)], torch.float32)
    opt = AdamW(params, lr=1e-2)
    opt.step()
    torch.cuda.synchronize()
    gc.collect()
    before = torch.cuda.memory_allocated()
    for seed in range(4):
        new = _tensors([(1 << 20,)], torch.float32, seed)[0]
        opt.state[new] = {name: t.clone() for name, t in opt.state.pop(params[0]).items()}
        opt.param_groups[0]["params"][0] = params[0] = new
        opt.step()
        opt.load_state_dict(copy.deepcopy(opt.state_dict()))
        opt.step()
    del new
    torch.cuda.synchronize()
    gc.collect()
    assert torch.cuda.memory_allocated() < before + (1 << 20) and int(opt.state[params[0]]["step"]) == 9

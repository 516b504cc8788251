"""Microscaled linears as a program uses them: modules, groups, a decoder's training step, graphs, streams, views, and the
calls at the edges.  Bounds as in ``test_gpu_mx.py``: a half step of bf16 for each rounding, 7 * 2^-13 of the terms' magnitudes for
the sums of fp8 products, 2^-16 for other sums."""
import pytest
import torch
from torch import nn

from oracle import mx_oracle as ox
from torchtune_amd import FrozenMXLinear, MXLoRALinear, MXTensor, harness, linear_mx, lora_linear_mx, to_mx
from torchtune_amd.modules.peft import (disable_adapter, get_adapter_params, get_merged_lora_ckpt, lora_linear_group, lora_swiglu_group,
                                        set_trainable_params)

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda"
HALF, SUMS, SUMS_FP8 = 2.0 ** -8, 2.0 ** -16, 7 * 2.0 ** -13


def _gen(n):
    return torch.Generator().manual_seed(n)


def _randn(*shape, seed, scale=1.0):
    return (torch.randn(*shape, generator=_gen(seed)) * scale).to(BF).to(DEV)


def _layer(k, n, r=8, seed=0, bias=False, dropout=0.0):
    with torch.device(DEV):
        m = MXLoRALinear(k, n, r, 2.0 * r, dropout=dropout, use_bias=bias).to(BF)
    with torch.no_grad():
        m.set_weight(_randn(n, k, seed=seed, scale=0.05))
        m.lora_a.weight.copy_(_randn(r, k, seed=seed + 1, scale=k ** -0.5))
        m.lora_b.weight.copy_(_randn(n, r, seed=seed + 2, scale=0.05))
        if bias:
            m.bias.copy_(_randn(n, seed=seed + 3))
    return m


def _dense(m):
    """the layer's weight in float64, from its buffers by the oracle"""
    return ox.values(ox.unpack(m.weight_codes.cpu(), "mxfp4"), m.weight_scales.cpu(), "mxfp4")


def _within(got, want, lost):
    err = (got.detach().double().cpu() - want).abs()
    worst = (err / (HALF * want.abs() + lost + 1e-38)).max().item()
    assert worst <= 1.0, f"{worst} of the bound"


# ---- modules ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("bias", [False, True])
def test_frozen_linear(act, bias):
    with torch.device(DEV):
        m = FrozenMXLinear(128, 96, bias=bias, activation=act)
    assert not list(p for p in m.parameters() if p.requires_grad) and set(m.state_dict()) == {"weight_codes", "weight_scales"} | ({"bias"} if bias else set())
    x = _randn(3, 5, 128, seed=1)
    y = m(x)
    assert torch.equal(y, linear_mx(x, m.mx_weight, m.bias, act)) and tuple(y.shape) == (3, 5, 96)
    with torch.device(DEV):
        other = FrozenMXLinear(128, 96, bias=bias, activation=act)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), y)


@pytest.mark.parametrize("dtype", [BF, torch.float32, torch.float16])
def test_a_dense_checkpoint_is_quantised_while_it_is_loaded(dtype):
    w = _randn(128, 64, seed=2).to(dtype)
    outer = nn.Sequential(_layer(64, 128), nn.Identity())
    state = {"0.weight": w, "0.lora_a.weight": outer[0].lora_a.weight.detach().clone(), "0.lora_b.weight": outer[0].lora_b.weight.detach().clone()}
    keys = set(state)
    outer.load_state_dict(state)
    assert set(state) == keys  # the caller's dictionary stays as it was
    want = to_mx(w.float())
    assert torch.equal(outer[0].weight_codes, want.codes) and torch.equal(outer[0].weight_scales, want.scales)
    with pytest.raises(RuntimeError, match="size mismatch"):
        outer.load_state_dict({**state, "0.weight": w[:64]})
    with pytest.raises(RuntimeError, match="Missing key"):
        outer.load_state_dict({k: v for k, v in state.items() if k != "0.weight"})
    with pytest.raises(ValueError):
        outer[0].set_weight(w[:, :32])


def test_lora_layer_is_the_functional_call_and_its_switches():
    m = _layer(256, 192, 16, seed=3, bias=True)
    x = _randn(40, 256, seed=4)
    y = m(x)
    assert torch.equal(y, lora_linear_mx(x, [m.mx_weight], [m.lora_a.weight], [m.lora_b.weight], [2.0], [m.bias])[0])
    base = linear_mx(x, m.mx_weight, m.bias)
    with disable_adapter(m):
        assert torch.equal(m(x), base)
    assert torch.equal(m(x), y)
    set_trainable_params(m, get_adapter_params(m))
    assert sorted(n for n, p in m.named_parameters() if p.requires_grad) == ["lora_a.weight", "lora_b.weight"]
    m(x).sum().backward()  # a gradient of ones, expanded from one element
    ones = torch.ones_like(y)
    ga, gb = torch.autograd.grad(m(x), [m.lora_a.weight, m.lora_b.weight], ones)
    assert torch.equal(m.lora_a.weight.grad, ga) and torch.equal(m.lora_b.weight.grad, gb) and m.bias.grad is None


def test_dropout_composes_the_same_sum():
    m = _layer(128, 64, 8, seed=5, dropout=0.5)
    x = _randn(300, 128, seed=6)
    m.eval()
    assert torch.equal(m(x), lora_linear_mx(x, [m.mx_weight], [m.lora_a.weight], [m.lora_b.weight], [2.0])[0])
    m.train()
    torch.manual_seed(0)
    y = m(x)
    torch.manual_seed(0)
    dropped = m.dropout(x)
    assert torch.equal(y, linear_mx(x, m.mx_weight) + 2.0 * m.lora_b(m.lora_a(dropped)))


@pytest.mark.parametrize("where", ["cuda", "cpu"])
def test_merged_checkpoint(where):
    m = _layer(128, 64, 8, seed=7)
    x, a, b = _dense(m), m.lora_a.weight.detach(), m.lora_b.weight.detach()
    merged = get_merged_lora_ckpt({f"l.{k}": v.to(where) for k, v in m.state_dict().items()}, rank=8, alpha=16.0)
    assert set(merged) == {"l.weight"} and merged["l.weight"].device.type == where
    delta = 2.0 * (b.double() @ a.double()).cpu()
    # bf16: the product, its factor and the sum are rounded, two of them before the sum
    _within(merged["l.weight"], x + delta, 3 * HALF * delta.abs() + SUMS * 2.0 * (b.double().abs() @ a.double().abs()).cpu())


# ---- layers with a common input, and a decoder ------------------------------------------------------
def _check_lora(m_list, x, ys, gys, gx):
    """outputs, input gradient and the accumulated adapter gradients of layers over the same input against the formulas"""
    x2, gy2 = x.detach().cpu().reshape(-1, x.shape[-1]), [g.detach().cpu().reshape(-1, g.shape[-1]) for g in gys]
    xq = ox.nearest(x2, "mxfp8")
    dense, s = [_dense(m) for m in m_list], [m.alpha / m.rank for m in m_list]
    a, b = [m.lora_a.weight.detach().cpu() for m in m_list], [m.lora_b.weight.detach().cpu() for m in m_list]
    wy, wgx, wga, wgb = ox.lora(xq, dense, a, b, s, gy2)
    my, mgx, mga, mgb = ox.lora(xq.abs(), [d.abs() for d in dense], [t.abs() for t in a], [t.abs() for t in b], s, [t.abs() for t in gy2])
    ghs = 0.0
    for i, m in enumerate(m_list):
        h = (xq @ a[i].double().T).abs()
        gh = (s[i] * (gy2[i].double() @ b[i].double())).abs()
        ghs = ghs + gh @ a[i].double().abs()
        _within(ys[i].reshape(-1, ys[i].shape[-1]), wy[i], SUMS_FP8 * my[i] + 2 * HALF * s[i] * (h @ b[i].double().abs().T))
        _within(m.lora_a.weight.grad, wga[i], SUMS * mga[i] + HALF * (gh.T @ xq.abs()))
        _within(m.lora_b.weight.grad, wgb[i], SUMS * mgb[i] + HALF * s[i] * (gy2[i].double().abs().T @ h))
    if gx is not None:
        _within(gx.reshape(-1, gx.shape[-1]), wgx, SUMS * mgx + HALF * ghs)


@pytest.mark.parametrize("outs,rank", [((128,), 64), ((256, 64), 24), ((192, 64, 64), 16), ((64, 64, 128, 64), 16), ((64, 128, 64), 32)])
def test_group(outs, rank):
    """The last one has ranks beyond what a call takes together: its layers run one after the other."""
    layers = [_layer(320, n, rank, seed=10 * i) for i, n in enumerate(outs)]
    x = _randn(2, 70, 320, seed=8).requires_grad_()
    ys = lora_linear_group(x, layers)
    gys = [_randn(*y.shape, seed=60 + i) for i, y in enumerate(ys)]
    gx, = torch.autograd.grad(ys, [x], gys, retain_graph=True)
    torch.autograd.backward(ys, gys)
    if sum(l.rank for l in layers) <= 64:
        _check_lora(layers, x, ys, gys, gx)
    else:
        for l, y, g in zip(layers, ys, gys):
            _check_lora([l], x, [y], [g], None)
    assert len(layers) != 2 or lora_swiglu_group(x, *layers) is None  # the caller multiplies


def test_decoder_training_step(monkeypatch):
    """A QLoRA decoder over an mxfp4 base: every adapter gradient of a step is that of its layer's formula over what the layer
    read and got back; the grouped step is near the ungrouped one; checkpointed, it is the same; and an optimiser step moves it."""
    model = harness.build_qlora_decoder("tiny", rank=8, alpha=16.0, device=DEV, seed=0, base="mxfp4")
    layers = [m for m in model.modules() if isinstance(m, MXLoRALinear)]
    assert len(layers) == 14 and all("lora_" in n for n, p in model.named_parameters() if p.requires_grad)
    tokens = torch.randint(0, 1024, (2, 96), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    loss = harness.train_step(model, tokens, tokens)
    grouped = {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}
    assert torch.isfinite(loss) and 6.0 < float(loss) < 8.0  # ~ln(1024)
    model.zero_grad(set_to_none=True)

    monkeypatch.setattr(harness, "GROUP_SHARED_INPUT", False)
    seen = {}
    for m in layers:
        m.register_forward_hook(lambda m, args, y: seen.update({m: [args[0].detach(), y.detach()]}))
        m.register_full_backward_hook(lambda m, gi, go: seen[m].append(go[0].detach()))
    harness.train_step(model, tokens, tokens)
    for m in layers:
        x, y, gy = seen[m]
        _check_lora([m], x, [y], [gy], None)
    for n, p in model.named_parameters():
        if p.grad is not None:  # some ten roundings of 2^-8 differ on the way: 5 % of a gradient's norm
            assert (p.grad.float() - grouped[n].float()).norm() <= 0.05 * grouped[n].float().norm(), n
    monkeypatch.setattr(harness, "GROUP_SHARED_INPUT", True)
    again = harness.build_qlora_decoder("tiny", rank=8, alpha=16.0, device=DEV, seed=0, base="mxfp4", activation_checkpointing=True)
    assert torch.equal(harness.train_step(again, tokens, tokens), loss)
    for n, p in again.named_parameters():
        assert p.grad is None or torch.equal(p.grad, grouped[n]), n
    torch.optim.SGD([p for p in again.parameters() if p.requires_grad], lr=0.1).step()
    assert not torch.equal(again.loss(tokens, tokens), loss)


# ---- gradients against differences ------------------------------------------------------------------
def test_gradients_against_differences():
    """The adapters enter linearly, one at a time, so a step of their own size has the exact difference <gradient, step>; and the
    rounding of the input scales with it, so that <gx, x^> is <gy, y>.  y's own rounding (a half step of each value, both
    times) and the sums' loss, against a step along the gradient's signs, which adds up all of its magnitudes."""
    m, k, n, r = 130, 192, 128, 16
    w, x, gy = to_mx(_randn(n, k, seed=1, scale=0.05)), _randn(m, k, seed=2).requires_grad_(), _randn(m, n, seed=3)
    a, b = _randn(r, k, seed=4, scale=k ** -0.5).requires_grad_(), _randn(n, r, seed=5, scale=0.05).requires_grad_()
    f = lambda a, b: lora_linear_mx(x, [w], [a], [b], [2.0])[0]
    y = f(a, b)
    gx, ga, gb = torch.autograd.grad(y, [x, a, b], gy)

    def total(t):
        return (gy.double() * t.double()).sum().item()

    def slack(*ts):  # of the totals: each value's half step and, no more than that, what its sums and its rounded h lose
        return sum((gy.double().abs() * t.double().abs()).sum().item() for t in ts) * (HALF + SUMS_FP8) \
            + 4 * HALF * (gy.double().abs() * 2.0 * ((x.double() @ a.double().T).abs() @ b.double().abs().T)).sum().item()

    for which, (p, g) in enumerate(((a, ga), (b, gb))):
        step = (g.sign() * p.abs().mean() * 4).to(BF)
        moved = (p.detach() + step).to(BF)
        step = moved.double() - p.detach().double()
        y2 = f(*((moved, b) if which == 0 else (a, moved)))
        expect = (g.double() * step).sum().item()
        lim = slack(y, y2, y2) + 2 * HALF * (g.double() * step).abs().sum().item()
        assert abs(total(y2) - total(y) - expect) <= lim and abs(expect) > lim / 4
    xq = ox.nearest(x.detach().cpu(), "mxfp8").to(DEV)
    assert abs(total(y) - (gx.double() * xq).sum().item()) <= slack(y) + 2 * HALF * (gx.double() * xq).abs().sum().item()


# ---- graphs, streams, threads -----------------------------------------------------------------------
@pytest.mark.parametrize("m,k,outs", [(1, 256, (128,)), (200, 4160, (64, 128)), (2100, 256, (192,))])
def test_captured_and_replayed(m, k, outs):
    """Forward and backward recorded once and replayed on other inputs, with eager calls between the replays; two graphs whose
    replays alternate."""
    layers = [_layer(k, n, 16, seed=20 * i) for i, n in enumerate(outs)]
    frozen = [l.mx_weight for l in layers]
    params = [p for l in layers for p in (l.lora_a.weight, l.lora_b.weight)]
    xs = [_randn(m, k, seed=30 + i).requires_grad_() for i in range(2)]
    gys = [_randn(m, n, seed=40 + i) for i, n in enumerate(outs)]

    def run(x):
        ys = lora_linear_group(x, layers)
        z = linear_mx(x, frozen[0], activation="mxfp4")
        grads = torch.autograd.grad([*ys, z], [x, *params], [*gys, gys[0]])
        return [*(y.detach() for y in ys), z.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            run(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs_of = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs_of.append(run(x))
        graphs.append(graph)
    for turn in range(4):
        for i, (x, graph) in enumerate(zip(xs, graphs)):
            with torch.no_grad():
                x.copy_(_randn(m, k, seed=50 + 2 * turn + i))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs_of[i]]
            for t, want in zip(got, run(x)):
                assert torch.equal(t, want)


def test_other_stream():
    layer, x, gy = _layer(2048, 256, 16, seed=60), _randn(500, 2048, seed=61).requires_grad_(), _randn(500, 256, seed=62)
    run = lambda: torch.autograd.grad(layer(x), [x, layer.lora_a.weight, layer.lora_b.weight], gy)
    want = run()
    q = to_mx(x.detach(), "mxfp8")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, q2 = run(), to_mx(x.detach(), "mxfp8")
        back = q2.to(torch.float32)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(q.codes, q2.codes) and torch.equal(q.scales, q2.scales) and torch.equal(back, q.to(torch.float32))


def test_trace():
    layer, x = _layer(64, 128, 8, seed=63), _randn(20, 64, seed=64)
    w = layer.mx_weight
    traced = torch.jit.trace(lambda t: linear_mx(t, w), (x,), check_trace=False)

    class Two(nn.Module):  # the trace holds a module's parameters
        def __init__(self):
            super().__init__()
            self.layer = layer

        def forward(self, t):
            return lora_linear_group(t, [self.layer, self.layer])

    two = torch.jit.trace(Two(), (x,), check_trace=False)
    y, one = _randn(20, 64, seed=65), layer(x)
    assert torch.equal(traced(y), linear_mx(y, w))
    a, b = two(x)
    assert torch.equal(a, b) and tuple(a.shape) == tuple(one.shape)
    assert torch.equal(two(y)[0], lora_linear_group(y, [layer, layer])[0])
    xr, gy = y.clone().requires_grad_(), _randn(20, 128, seed=66)
    for f, g in ((traced, lambda t: linear_mx(t, w)), (lambda t: two(t)[1], lambda t: lora_linear_group(t, [layer, layer])[1])):
        assert torch.equal(torch.autograd.grad(f(xr), [xr], gy)[0], torch.autograd.grad(g(xr), [xr], gy)[0])


# ---- views, alignment, edges ------------------------------------------------------------------------
def _shapes_of(t):
    """the same values in other places: transposed, off by one element, every second row, expanded views of t"""
    base = torch.zeros(t.numel() + 8, dtype=t.dtype, device=t.device)
    off = base[1:1 + t.numel()].view(t.shape).copy_(t)
    rows = torch.zeros(2 * t.shape[0], *t.shape[1:], dtype=t.dtype, device=t.device)
    rows[::2] = t
    return [t.t().contiguous().t(), off, rows[::2]]


def test_views_and_unaligned_operands():
    layer, x, gy = _layer(128, 192, 8, seed=70, bias=True), _randn(50, 128, seed=71), _randn(50, 192, seed=72)
    run = lambda x, gy: torch.autograd.grad(layer(x), [x, layer.lora_a.weight, layer.lora_b.weight], gy)
    want = run(x.clone().requires_grad_(), gy)
    base = linear_mx(x, layer.mx_weight, layer.bias)
    for v, g in zip(_shapes_of(x), _shapes_of(gy)):
        assert all(torch.equal(a, b) for a, b in zip(run(v.requires_grad_(), g), want))
        assert torch.equal(linear_mx(v.detach(), layer.mx_weight, layer.bias), base)
    w = layer.mx_weight
    for codes, scales in zip(_shapes_of(w.codes), _shapes_of(w.scales)):
        v = MXTensor(codes, scales)
        assert torch.equal(linear_mx(x, v, layer.bias), base) and torch.equal(v.to(torch.float32), w.to(torch.float32))
    odd_bias = torch.zeros(193, dtype=BF, device=DEV)[1:].copy_(layer.bias.detach())
    assert torch.equal(linear_mx(x, w, odd_bias), base)
    one = x[0].clone()
    assert torch.equal(linear_mx(one, w, layer.bias), linear_mx(x[:1], w, layer.bias)[0]) and tuple(layer(one).shape) == (192,)


def test_no_tokens():
    layer = _layer(64, 128, 8, seed=73, bias=True)
    x = torch.zeros(2, 0, 64, dtype=BF, device=DEV, requires_grad=True)
    for y in (layer(x), linear_mx(x, layer.mx_weight, layer.bias), linear_mx(x.detach(), layer.mx_weight)):
        assert tuple(y.shape) == (2, 0, 128)
    grads = torch.autograd.grad(layer(x), [x, layer.lora_a.weight, layer.lora_b.weight, layer.bias], torch.zeros(2, 0, 128, dtype=BF, device=DEV))
    assert tuple(grads[0].shape) == (2, 0, 64) and all(not g.any() for g in grads[1:])
    gx, = torch.autograd.grad(linear_mx(x, layer.mx_weight), [x], torch.zeros(2, 0, 128, dtype=BF, device=DEV))
    assert tuple(gx.shape) == (2, 0, 64)


def test_no_outputs():
    w = MXTensor(torch.zeros(0, 64, dtype=torch.uint8, device=DEV), torch.zeros(0, 4, dtype=torch.uint8, device=DEV))
    x = _randn(5, 128, seed=77).requires_grad_()
    y = linear_mx(x, w)
    gx, = torch.autograd.grad(y, [x], torch.zeros_like(y))
    assert tuple(y.shape) == (5, 0) and tuple(gx.shape) == (5, 128) and not gx.any()
    assert tuple(w.to().shape) == (0, 128)


def test_only_the_gradients_that_are_asked_for():
    layer, x, gy = _layer(128, 64, 8, seed=74, bias=True), _randn(30, 128, seed=75), _randn(30, 64, seed=76)
    every = torch.autograd.grad(layer(x.clone().requires_grad_()), [layer.lora_a.weight, layer.lora_b.weight, layer.bias], gy)
    assert torch.equal(every[2], gy.sum(0))
    for p, want in zip((layer.lora_a.weight, layer.lora_b.weight, layer.bias), every):
        for q in layer.parameters():
            q.requires_grad_(q is p)
        got, = torch.autograd.grad(layer(x), [p], gy)
        assert torch.equal(got, want)
    layer.requires_grad_(False)
    xr = x.clone().requires_grad_()
    gx, = torch.autograd.grad(layer(xr), [xr], gy)
    layer.requires_grad_(True)
    assert torch.equal(gx, torch.autograd.grad(layer(xr), [xr], gy)[0])
    with torch.no_grad():
        assert not layer(xr).requires_grad
    # the same tensor in two members, one output unused: its share of the gradients is zero
    layers = [_layer(128, 64, 8, seed=80), _layer(128, 64, 8, seed=90)]
    ys = lora_linear_group(xr, layers)
    got = torch.autograd.grad(ys[0], [xr, layers[0].lora_b.weight, layers[1].lora_a.weight], gy)
    full = torch.autograd.grad(lora_linear_group(xr, layers), [xr, layers[0].lora_b.weight, layers[1].lora_a.weight], [gy, torch.zeros_like(gy)])
    assert all(torch.equal(a, b) for a, b in zip(got, full)) and not got[2].any()


def test_saved_tensors_are_the_eight_bit_input():
    """What a layer keeps of its input: codes and scales, 8.25 bits an element (rows padded to 256), and the rank-wide product."""
    layer, x = _layer(1024, 64, 8, seed=95), _randn(2048, 1024, seed=96)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        layer(x)
    frozen = {t.data_ptr() for t in (layer.weight_codes, layer.weight_scales, layer.lora_a.weight, layer.lora_b.weight)}
    assert sum(t.numel() * t.element_size() for t in kept if t.data_ptr() not in frozen) == 2048 * (1024 + 32 + 2 * 8)


def test_transforms_and_second_derivatives_are_refused():
    """None of them may drop a tangent, a batch or a second derivative without saying so."""
    layer, x = _layer(64, 64, 8, seed=110), _randn(6, 64, seed=111).requires_grad_()
    w = layer.mx_weight
    for f in (layer, lambda t: linear_mx(t, w)):
        with pytest.raises(RuntimeError, match="differentiated"):
            torch.autograd.grad(f(x).sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x.detach())
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (x.detach(),), (torch.ones_like(x),))
        f(x).sum().backward()  # and what is asked for in earnest still works


def test_changed_in_place_after_the_forward_pass():
    layer, x = _layer(64, 64, 8, seed=97), _randn(10, 64, seed=98).requires_grad_()
    y = layer(x)
    with torch.no_grad():
        layer.lora_b.weight.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("k,n", [(16448, 64), (64, 16448)])
def test_offsets_beyond_32_bits(k, n):
    """More than 2^31 elements of input, or of output: the last tokens against the same tokens by themselves."""
    m, tail = 131072 + 77, 45
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GiB of free device memory")
    layer = _layer(k, n, 8, seed=100)
    x = torch.empty(m, k, dtype=BF, device=DEV)
    x.view(-1, 64)[:] = _randn(1, 64, seed=101)
    x[-tail:] = _randn(tail, k, seed=102)
    q, end = to_mx(x, "mxfp8"), to_mx(x[-tail:], "mxfp8")
    assert torch.equal(q.codes[-tail:], end.codes) and torch.equal(q.scales[-tail:], end.scales)
    assert torch.equal(q.to(BF)[-tail:], end.to(BF))
    del q
    gy = torch.zeros(m, n, dtype=BF, device=DEV)
    gy[-tail:] = _randn(tail, n, seed=103)
    x.requires_grad_()
    y = layer(x)
    gx, = torch.autograd.grad(y, [x], gy, retain_graph=True)
    torch.autograd.backward(y, gy, inputs=[layer.lora_a.weight, layer.lora_b.weight])
    _check_lora([layer], x[-tail:], [y[-tail:]], [gy[-tail:]], gx[-tail:])
    assert not gx[:-tail].any()

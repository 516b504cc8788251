"""``layer_ops.token_logprobs`` against a plain implementation in 64 bits: log probabilities, entropy, alternatives, gradients.

Tolerances.  With d the distance from the row's largest logit in powers of two, a term 2^d of the sum is off by |d| 2^-24 twice (the product
with log2(e) / temperature, the rounding of d) and by 2^-23 (the hardware's exp2); weighted by the terms themselves |d| is below 40.
A thread adds at most 1024 terms one after another, then 14 partial sums.  So the sum is off by less than
(2 * 40 + 2 + 1024 + 14) * 2^-24 < 1200 * 2^-24 of itself; its logarithm by that number.  A log probability adds 4 roundings of its own
parts, the entropy a second such sum, weighted by |d|."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from torchtune_amd.modules import layer_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
SUM = 1200 * U
INF = math.inf


def _plain(logits, tokens, temperature, top):
    z = logits.double().cpu() / temperature
    tokens = tokens.cpu()
    lp = z - torch.logsumexp(z, -1, keepdim=True)
    p = lp.exp()
    entropy = -(p * lp.masked_fill(p == 0, 0)).sum(-1)
    at = tokens if tokens.dim() == z.dim() else tokens[..., None]
    chosen = lp.gather(-1, at.clamp(min=0)).masked_fill(at < 0, 0).view(tokens.shape)
    order = torch.sort(logits.float().cpu(), dim=-1, descending=True, stable=True).indices[..., :top]
    return lp, p, entropy, chosen, order


def _check(logits, tokens, temperature=1.0, top=0, entropy=True, seed=0):
    r = layer_ops.token_logprobs(logits, tokens, temperature=temperature, entropy=entropy, top=top)
    lp, p, ent, chosen, order = _plain(logits.detach(), tokens, temperature, top)
    size = (logits.detach().double().cpu() / temperature).masked_fill(p == 0, 0).abs().amax(-1, keepdim=True)  # of the parts of a difference
    scale = size if tokens.dim() == logits.dim() else size[..., 0]
    off = (r.logprobs.detach().double().cpu() - chosen).abs().nan_to_num(0, 0, 0)
    assert bool((off <= SUM + 8 * U * (chosen.abs().nan_to_num(0, 0, 0) + scale)).all()), float(off.max())
    assert bool((torch.isinf(r.logprobs.detach().cpu()) == torch.isinf(chosen)).all())
    if entropy:
        off = (r.entropy.detach().double().cpu() - ent).abs()
        assert bool((off <= 2 * SUM * (1 + ent) + 8 * U * size[..., 0]).all()), float(off.max())
    if top:
        assert torch.equal(r.top_tokens.cpu(), order)
        want = lp.gather(-1, order)
        off = (r.top_logprobs.double().cpu() - want).abs().nan_to_num(0, 0, 0)
        assert bool((off <= SUM + 8 * U * (want.abs().nan_to_num(0, 0, 0) + size)).all())
    else:
        assert r.top_logprobs is None and r.top_tokens is None
    if not logits.requires_grad:
        return
    g = torch.Generator().manual_seed(seed)
    gl, gh = torch.randn(tokens.shape, generator=g), torch.randn(logits.shape[:-1], generator=g)
    outs, gs = ([r.logprobs, r.entropy], [gl, gh]) if entropy else ([r.logprobs], [gl])
    (got,) = torch.autograd.grad(outs, logits, [x.to(DEV) for x in gs])
    at = tokens.cpu() if tokens.dim() == logits.dim() else tokens.cpu()[..., None]
    gl = gl.double().view(at.shape) * (at >= 0)
    total = gl.sum(-1, keepdim=True)
    own = torch.zeros_like(p).scatter_add_(-1, at.clamp(min=0), gl)
    own_size = torch.zeros_like(p).scatter_add_(-1, at.clamp(min=0), gl.abs())
    want, parts = own - p * total, own_size + p * gl.abs().sum(-1, keepdim=True)
    if entropy:
        surprise = -lp.masked_fill(p == 0, 0)
        want = want + gh.double()[..., None] * p * (surprise - ent[..., None])
        parts = parts + gh.double().abs()[..., None] * p * (1 + surprise + ent[..., None])
    want, parts = want / temperature, parts / temperature
    assert got.dtype == logits.dtype and got.shape == logits.shape and got.is_contiguous()
    bound = want.abs() * torch.finfo(got.dtype).eps / 2 + 4 * SUM * parts + 1e-38  # below the smallest normal number
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


def _logits(rows, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(rows, V, generator=g, device=DEV) * spread).to(dtype)


def _tokens(rows, V, n=0, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, V, (rows, n) if n else (rows,), generator=g, device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,n,top,temperature", [
    (1, 1, 0, 1, 1.0), (1, 7, 0, 7, 0.5), (3, 8, 2, 8, 1.0), (5, 33, 0, 3, 2.0), (2, 4096, 0, 64, 1.0), (1, 4097, 3, 64, 1.0),
    (1, 128256, 0, 20, 0.7), (7, 50257, 16, 5, 2.0), (48, 32000, 0, 50, 1.0), (600, 1025, 0, 10, 1.0), (513, 4100, 70, 0, 1.0),
    (300, 8191, 1, 1, 1.3), (1, 262144, 0, 2, 1.0),
])
def test_rows_of_all_sizes(dtype, rows, V, n, top, temperature):
    logits, tokens = _logits(rows, V, dtype).requires_grad_(), _tokens(rows, V, n)
    if rows > 2:
        tokens[1] = -100
    _check(logits, tokens, temperature, top)
    _check(logits.detach(), tokens, temperature, top, entropy=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [2, 600])
def test_ruled_out_tokens(dtype, rows):
    """-inf and the type's lowest value in part of a row, in all but a few places, and fewer places than alternatives."""
    V = 5000
    for fill in (-INF, torch.finfo(dtype).min):
        for left in (3000, 40, 3):
            logits, tokens = _logits(rows, V, dtype, seed=left), _tokens(rows, left)
            logits[:, left:] = fill
            order = torch.randperm(V, generator=torch.Generator(device=DEV).manual_seed(left), device=DEV)
            logits = logits[:, order].contiguous().requires_grad_()
            tokens = torch.argsort(order)[tokens]
            _check(logits, tokens, 1.0, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [2, 600])
def test_rows_without_a_difference(dtype, rows):
    """All logits equal: at 0, at the lowest and at the highest value of the type, where a product with log2(e) overflows."""
    V = 9000
    for value in (0.0, torch.finfo(dtype).min, torch.finfo(dtype).max, -1e4):
        for temperature in (1.0, 0.01):
            logits = torch.full((rows, V), value, dtype=dtype, device=DEV, requires_grad=True)
            r = layer_ops.token_logprobs(logits, _tokens(rows, V), temperature=temperature, entropy=True, top=4)
            want = math.log(V)
            assert float((r.logprobs + want).abs().max()) < SUM + 8 * U * want
            assert float((r.entropy - want).abs().max()) < 2 * SUM * (1 + want)
            assert torch.equal(r.top_tokens.cpu(), torch.arange(4).expand(rows, 4))
            (g,) = torch.autograd.grad(r.entropy.sum(), logits)
            assert float(g.abs().max()) < 4 * SUM * (1 + 2 * want) / V / temperature


@pytest.mark.parametrize("rows,V", [(2, 9000), (600, 5000), (40, 1000)])
@pytest.mark.parametrize("size", [1e6, 3e8, 1.2e9, 1.9e9, 4e9, 1e12, -2e9])
def test_logits_of_enormous_size(rows, V, size):
    """fp32 logits whose neighbours are up to 65536 apart: the row's distribution is even over its largest ones, apart from differences
    of one where the numbers are that fine.  The difference from the largest is exact; then the sums' error."""
    g = torch.Generator(device=DEV).manual_seed(3)
    logits = (size + torch.randint(-40, 40, (rows, V), generator=g, device=DEV).double() * max(1.0, abs(size) * 2.0 ** -24)).float()
    z = logits.double()
    lp = torch.log_softmax(z - z.amax(-1, keepdim=True), -1)
    ent = -(lp.exp() * lp).sum(-1)
    tokens = z.argmax(-1)
    leaf = logits.clone().requires_grad_()
    r = layer_ops.token_logprobs(leaf, tokens, entropy=True, top=40)
    assert float((r.logprobs.double() - lp.gather(1, tokens[:, None])[:, 0]).abs().max()) < SUM + 8 * U * math.log(V)
    assert float((r.entropy.double() - ent).abs().max()) < 2 * SUM * (1 + math.log(V))
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :40]
    assert torch.equal(r.top_tokens, order)
    (grad,) = torch.autograd.grad(r.logprobs.sum(), leaf)
    want = torch.zeros_like(lp).scatter_(1, tokens[:, None], 1.0) - lp.exp()
    assert float((grad.double() - want).abs().max()) < 4 * SUM


@pytest.mark.parametrize("rows", [1, 600])
def test_a_row_of_nothing(rows):
    logits = _logits(rows, 6000, torch.bfloat16)
    logits[0] = -INF
    logits.requires_grad_()
    r = layer_ops.token_logprobs(logits, _tokens(rows, 6000), entropy=True, top=3)
    assert float(r.logprobs[0]) == -INF and float(r.entropy[0]) == 0 and bool((r.top_logprobs[0] == -INF).all())
    assert r.top_tokens[0].tolist() == [0, 1, 2]
    (g,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), logits)
    assert not bool(g[0].any()) and (rows == 1 or bool(g[1:].any(-1).all()))


@pytest.mark.parametrize("rows", [2, 600])
@pytest.mark.parametrize("bad", [math.nan, INF])
def test_what_is_not_a_number_stays_in_its_row(rows, bad):
    clean = _logits(rows, 6000, torch.float32)
    logits = clean.clone()
    logits[1, 4321] = bad
    tokens = _tokens(rows, 6000)
    a = layer_ops.token_logprobs(clean, tokens, entropy=True, top=3)
    b = layer_ops.token_logprobs(logits, tokens, entropy=True, top=3)
    other = torch.arange(rows, device=DEV) != 1
    for x, y in zip(a, b):
        assert torch.equal(x[other], y[other])
    assert math.isnan(float(b.logprobs[1])) and math.isnan(float(b.entropy[1])) and bool(torch.isnan(b.top_logprobs[1]).all())
    assert bool(((b.top_tokens >= 0) & (b.top_tokens < 6000)).all())
    every = torch.full((rows, 100), math.nan, device=DEV)
    r = layer_ops.token_logprobs(every, tokens % 100, entropy=True, top=3)
    assert bool(torch.isnan(r.logprobs).all()) and bool(((r.top_tokens >= 0) & (r.top_tokens < 100)).all())


def test_equal_logits_give_the_lower_token_first():
    for rows in (1, 600):
        for V in (5000, 20000):
            g = torch.Generator(device=DEV).manual_seed(V + rows)
            logits = torch.randint(-2, 3, (rows, V), generator=g, device=DEV).to(torch.bfloat16) * 0.5  # more at the top than a list holds
            logits[:, ::7] *= -0.0
            _check(logits, _tokens(rows, V), 1.0, 64)


def test_tokens_outside_the_vocabulary():
    logits = _logits(4, 900, torch.float32).requires_grad_()
    tokens = torch.tensor([[5, -100], [900, 7], [-1, -100], [2 ** 40, 899]], device=DEV)
    r = layer_ops.token_logprobs(logits, tokens)
    bad = torch.tensor([[False, False], [True, False], [True, False], [True, False]], device=DEV)
    assert bool((torch.isnan(r.logprobs) == bad).all()) and float(r.logprobs[0, 1]) == 0
    (g,) = torch.autograd.grad(r.logprobs[~bad].sum(), logits)
    assert bool(torch.isfinite(g).all()) and not bool(g[2].any())
    r = layer_ops.token_logprobs(logits, tokens[:, 0] * 0 + 7, ignore_index=7)
    assert not bool(r.logprobs.any())


def test_the_same_token_twice_adds_up():
    logits = _logits(3, 300, torch.float32).requires_grad_()
    twice = torch.tensor([[4, 4, 9], [9, 9, 9], [0, 1, 0]], device=DEV)
    g = torch.randn(3, 3, device=DEV)
    (got,) = torch.autograd.grad(layer_ops.token_logprobs(logits, twice).logprobs, logits, g)
    want = sum(torch.autograd.grad(layer_ops.token_logprobs(logits, twice[:, i].contiguous()).logprobs, logits, g[:, i])[0] for i in range(3))
    assert float((got - want).abs().max()) < 64 * U * float(g.abs().sum(-1).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views(dtype):
    """Shifted sequences, part of the vocabulary, transposed batches: read where they are, or copied; the same bits."""
    whole = _logits(6 * 9, 1003, dtype).view(6, 9, 1003)
    for view in (whole[:, :-1], whole[:, 1:, 3:1000], whole.transpose(0, 1), whole[::2, ::3], whole[:1].expand(5, 9, 1003), whole[2, 4],
                 whole.view(2, 3, 9, 1003)[:, :2, 1:7:2], whole.transpose(1, 2)[:, :900].transpose(1, 2)):
        tokens = _tokens(int(view.numel() // view.shape[-1]), view.shape[-1]).view(view.shape[:-1])
        leaf = view.detach().requires_grad_()
        a = layer_ops.token_logprobs(leaf, tokens, entropy=True, top=2)
        dense = view.detach().clone().contiguous().requires_grad_()
        b = layer_ops.token_logprobs(dense, tokens, entropy=True, top=2)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert a.logprobs.shape == view.shape[:-1] and a.top_tokens.shape == (*view.shape[:-1], 2)
        ga, gb = (torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), t)[0] for r, t in ((a, leaf), (b, dense)))
        assert torch.equal(ga, gb)


def test_parts_of_the_gradient_and_empty_batches():
    logits, tokens = _logits(5, 2000, torch.float32).requires_grad_(), _tokens(5, 2000)
    r = layer_ops.token_logprobs(logits, tokens, entropy=True)
    a = torch.autograd.grad(r.logprobs.sum(), logits, retain_graph=True)[0]
    b = torch.autograd.grad(r.entropy.sum(), logits, retain_graph=True)[0]
    both = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), logits)[0]
    assert float((a + b - both).abs().max()) < 64 * U
    e = torch.zeros(0, 50, device=DEV, requires_grad=True)
    r = layer_ops.token_logprobs(e, torch.zeros(0, dtype=torch.long, device=DEV), entropy=True, top=2)
    assert r.logprobs.shape == (0,) and r.entropy.shape == (0,) and r.top_tokens.shape == (0, 2)
    assert torch.autograd.grad(r.logprobs.sum(), e)[0].shape == (0, 50)


def test_gradient_against_differences():
    """Central differences along a direction, step h: h^2 of the third derivative, and the sum's error over h."""
    logits, tokens = _logits(4, 500, torch.float32, spread=1.0).requires_grad_(), _tokens(4, 500, 2)
    g, gh, h = torch.randn(4, 2, device=DEV), torch.randn(4, device=DEV), 2.0 ** -5

    def total(x):
        r = layer_ops.token_logprobs(x, tokens, temperature=1.5, entropy=True)
        return (r.logprobs.double() * g).sum() + (r.entropy.double() * gh).sum()

    grad = torch.autograd.grad(total(logits), logits)[0]
    way = torch.randn(4, 500, device=DEV)
    way = way / way.norm()
    with torch.no_grad():
        slope = (total(logits + h * way) - total(logits - h * way)) / (2 * h)
    size = float(g.abs().sum() + gh.abs().sum()) * 8
    assert abs(float(slope - (grad * way).sum())) < size * (h * h + SUM / h)


def test_more_than_2_to_the_31_logits():
    """The last rows of 2^31 and more logits: what they give by themselves."""
    rows, V = 2 ** 14 + 40, 2 ** 17
    logits = torch.zeros(rows, V, device=DEV, dtype=torch.bfloat16)
    logits[-30:] = _logits(30, V, torch.bfloat16)
    tokens = _tokens(rows, V)
    logits.requires_grad_()
    r = layer_ops.token_logprobs(logits, tokens, entropy=True, top=3)
    (g,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), logits)
    few = torch.cat([logits.detach()[-30:]] * 40).requires_grad_()  # as many rows as are not cut into segments
    q = layer_ops.token_logprobs(few, tokens[-30:].repeat(40), entropy=True, top=3)
    (h,) = torch.autograd.grad(q.logprobs.sum() + q.entropy.sum(), few)
    for a, b in zip(r, q):
        assert torch.equal(a[-30:], b[-30:])
    assert torch.equal(g[-30:], h[-30:])
    assert float((r.logprobs.detach()[:-30] + math.log(V)).abs().max()) < SUM + 8 * U * math.log(V)


def test_agrees_with_the_chunk_loss():
    logits, tokens = _logits(40, 4096, torch.bfloat16), _tokens(40, 4096)
    tokens[3] = -100
    a = layer_ops.cross_entropy_sum(logits.clone().requires_grad_(), tokens)
    assert abs(float(a + layer_ops.token_logprobs(logits, tokens).logprobs.sum())) < 40 * 2 * SUM * 20


def test_recorded_into_graphs():
    """Two graphs that share nothing, and one's replays between eager calls."""
    sizes = [(3, 128256, 5), (700, 3000, 0)]
    graphs = []
    for rows, V, top in sizes:
        logits, tokens = _logits(rows, V, torch.bfloat16).requires_grad_(), _tokens(rows, V)

        def call(logits=logits, tokens=tokens, top=top):
            r = layer_ops.token_logprobs(logits, tokens, entropy=True, top=top)
            gs = torch.autograd.grad([r.logprobs, r.entropy], logits, [torch.ones_like(r.logprobs), torch.full_like(r.entropy, 0.1)])
            return [t for t in r if t is not None] + list(gs)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = call()
        graphs.append((graph, kept, call, logits, tokens))
    for i in range(3):
        for graph, kept, call, logits, tokens in graphs:
            with torch.no_grad():
                logits.copy_(torch.randn_like(logits) * 3)
                tokens.copy_(torch.randint_like(tokens, logits.shape[1]))
        for graph, *_ in graphs:
            graph.replay()
        for graph, kept, call, *_ in graphs:
            got = [t.clone() for t in kept]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, call()))


def test_second_derivatives_are_refused_and_written_logits_noticed():
    logits, tokens = _logits(2, 100, torch.float32).requires_grad_(), _tokens(2, 100)
    r = layer_ops.token_logprobs(logits, tokens, top=2)
    assert not r.top_logprobs.requires_grad
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(r.logprobs.sum(), logits, create_graph=True)
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        layer_ops.token_logprobs(fwAD.make_dual(logits.detach(), logits.detach()), tokens)
    r = layer_ops.token_logprobs(logits, tokens)
    with torch.no_grad():
        logits.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        r.logprobs.sum().backward()


def test_a_trace_keeps_the_gradients():
    logits, tokens = _logits(3, 400, torch.float32).requires_grad_(), _tokens(3, 400)

    def f(x, t):
        r = layer_ops.token_logprobs(x, t, entropy=True, top=2)
        return r.logprobs, r.entropy, r.top_tokens

    traced = torch.jit.trace(f, (logits, tokens), check_trace=False)
    other = (logits.detach() + 1 + torch.randn_like(logits)).requires_grad_()
    got, want = traced(other, tokens), f(other, tokens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    a, b = (torch.autograd.grad(o[0].sum() + o[1].sum(), other)[0] for o in (got, want))
    assert torch.equal(a, b)

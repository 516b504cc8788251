"""Microscaled tensors on the GPU against the 64-bit oracle: codec to the bit, products and gradients within bounds that are
derived beside them."""
import pytest
import torch

from oracle import mx_oracle as ox
from torchtune_amd import MXTensor, linear_mx, lora_linear_mx, to_mx

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
# Half a step of bf16, and what the sums of products lose.  bf16 and fp4 operands: fp32 sums, 2^-24 of the running sum's
# magnitude for each of at most 2^14 / 64 instructions.  fp8 operands: the matrix cores align eight products at a time to the
# largest of them and drop what lies below 2^-13 of it (measured with one large and one small product), so of eight products
# at most 7 * 2^-13 of the largest is lost, which is at most that share of their magnitudes' sum.
HALF, SUMS, SUMS_FP8 = 2.0 ** -8, 2.0 ** -16, 7 * 2.0 ** -13


def _seed(n):
    return torch.Generator().manual_seed(n)


def _special(shape, seed, dtype=torch.float32):
    """Values over the whole range: ordinary, tiny, subnormal, huge, ties, zeros, blocks at the top of the formats."""
    g = _seed(seed)
    x = torch.randn(shape, generator=g)
    rows = x.view(-1, shape[-1])
    n = rows.shape[0]
    for i, f in enumerate([1e-30, 1e-38, 1e-41, 1e30, 1e38, 448.0, 6.0, 2.0 ** -120]):
        if i < n:
            rows[i] *= f
    if n > 9:
        rows[8] = torch.randint(-16, 17, (shape[-1],), generator=g) / 4.0
        rows[9] = 0.0
    if n > 10:
        rows[10] = torch.randint(-255, 256, (shape[-1],), generator=g).float()
    return x.clamp(-3e38, 3e38).to(dtype)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("shape", [(32,), (1, 32), (13, 96), (3, 5, 64), (257, 1056), (64, 4096), (0, 64)])
def test_codec_is_the_oracle_to_the_bit(fmt, dtype, shape):
    x = _special(shape, 1, dtype) if shape[0] else torch.zeros(shape, dtype=dtype)
    q = to_mx(x.cuda(), fmt)
    codes, scales = ox.quantize(x, fmt) if x.numel() else (None, None)
    assert tuple(q.shape) == shape and q.dtype == dtype
    if x.numel():
        assert torch.equal(q.scales.cpu(), scales)
        assert torch.equal(q.codes.cpu(), ox.pack(codes, fmt))
        want = ox.values(codes, scales, fmt)
        for out in (torch.float32, BF):
            got = q.to(out).cpu()
            # the conversion to bf16 is the format's own: below bf16's normal range it may flush
            tiny = want.abs() < 2.0 ** -126
            assert torch.equal(got[~tiny], want.to(out)[~tiny])
            assert (got[tiny].double() - want[tiny]).abs().le(2.0 ** -126).all()
    assert q.to().dtype == dtype and q.to().shape == x.shape


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_codec_non_finite_blocks(fmt):
    for dtype in (BF, torch.float32):
        x = torch.randn(5, 128, generator=_seed(2)).to(dtype)
        x[0, 3], x[1, 70], x[2, 127], x[4] = float("inf"), float("nan"), -float("inf"), float("nan")
        q = to_mx(x.cuda(), fmt)
        codes, scales = ox.quantize(x, fmt)
        assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), ox.pack(codes, fmt))
        got, want = q.to(torch.float32).cpu(), ox.values(codes, scales, fmt).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_codec_of_views_and_unaligned_tensors():
    base = torch.randn(40, 200, generator=_seed(3)).cuda()
    for x in (base[:, 8:136], base.t()[:64, :32], base.flatten()[3:3 + 640].view(5, 128), base.to(BF).flatten()[1:1 + 640].view(5, 128)):
        q = to_mx(x, "mxfp4")
        codes, scales = ox.quantize(x, "mxfp4")
        assert torch.equal(q.codes.cpu(), ox.pack(codes, "mxfp4")) and torch.equal(q.scales.cpu(), scales)
        assert torch.equal(q.to(torch.float32).cpu(), ox.values(codes, scales, "mxfp4").float())


def _weight(n, k, seed):
    w = torch.randn(n, k, generator=_seed(seed)) * 0.02
    codes, scales = ox.quantize(w, "mxfp4")
    return MXTensor(ox.pack(codes, "mxfp4").cuda(), scales.cuda()), ox.values(codes, scales, "mxfp4")


def _close(got, want, lost, norm=HALF):
    """got bf16, want float64, lost: what the sums (and inner roundings) may lose of each output; norm: a bound on the whole
    error's 2-norm relative to the result's - a half step of every output is the most that one rounding makes of it, and
    what the sums lose is far from its worst in most outputs"""
    err = (got.double().cpu() - want).abs()
    worst = (err / (HALF * want.abs() + lost + 1e-38)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst} of the bound"
    if err.numel() >= 64:
        rel = (err.norm() / want.norm()).item()
        assert rel <= norm, f"2-norm of the error is {rel} of the result's"


LINEAR = [(1, 64, 32), (1, 1, 4096), (2, 4096, 160), (5, 100, 512), (13, 33, 1056), (16, 256, 4096), (17, 257, 608), (33, 1024, 2048),
          (64, 129, 96), (100, 384, 5632), (128, 128, 128), (129, 640, 544), (333, 1000, 1024), (1000, 2049, 640), (2000, 4096, 256)]


@pytest.mark.parametrize("act", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear(m, n, k, act):
    w, dense = _weight(n, k, 4)
    g = _seed(5)
    x = (torch.randn(m, k, generator=g) * torch.where(torch.rand(k, generator=g) < 0.02, 10.0, 1.0)).to(BF)
    bias = torch.randn(n, generator=g).to(BF) if m % 2 else None
    y = linear_mx(x.cuda(), w, None if bias is None else bias.cuda(), activation=act)
    xq = ox.nearest(x, act)
    want = xq @ dense.T + (0.0 if bias is None else bias.double())
    assert y.dtype == BF and tuple(y.shape) == (m, n)
    magnitude = xq.abs() @ dense.abs().T + (0.0 if bias is None else bias.double().abs())
    _close(y, want, (SUMS_FP8 if act == "mxfp8" else SUMS) * magnitude)


@pytest.mark.parametrize("r", [8, 16, 24, 64])
@pytest.mark.parametrize("m,k,outs", [(1, 64, [64]), (24, 128, [192]), (77, 1024, [256]), (350, 2048, [2048]), (513, 320, [64, 128, 64]),
                                      (300, 1024, [1024, 256, 256]),
                                      (33, 4160, [64]), (20, 8256, [128]), (2500, 320, [128, 64]), (1030, 64, [8192]), (1100, 4096, [1024, 512, 512])])
def test_lora(m, k, outs, r):
    if len(outs) > 1 and r > 16:
        r = 16
    g = _seed(7)
    x = torch.randn(m, k, generator=g).to(BF)
    both = [_weight(n, k, 8 + i) for i, n in enumerate(outs)]
    a = [((torch.rand(r, k, generator=g) * 2 - 1) / k ** 0.5).to(BF) for _ in outs]
    b = [(torch.randn(n, r, generator=g) * 0.05).to(BF) for n in outs]
    gy = [torch.randn(m, n, generator=g).to(BF) for n in outs]
    s = [2.0 if i % 2 == 0 else 0.75 for i in range(len(outs))]
    xd = x.cuda().requires_grad_()
    ad, bd = [t.cuda().requires_grad_() for t in a], [t.cuda().requires_grad_() for t in b]
    ys = lora_linear_mx(xd, [w for w, _ in both], ad, bd, s)
    grads = torch.autograd.grad(ys, [xd, *ad, *bd], [t.cuda() for t in gy])
    xq = ox.nearest(x, "mxfp8")
    dense = [d for _, d in both]
    wy, wgx, wga, wgb = ox.lora(xq, dense, a, b, s, gy)
    # magnitudes: the same formulas over absolute values
    my, mgx, mga, mgb = ox.lora(xq.abs(), [d.abs() for d in dense], [t.abs() for t in a], [t.abs() for t in b], s, [t.abs() for t in gy])
    for i in range(len(outs)):
        # y: h is rounded, and rounded again with its factor, before it meets lora_b: two half steps of the adapter's part
        adapter = s[i] * ((xq @ a[i].double().T).abs() @ b[i].double().abs().T)
        _close(ys[i].detach(), wy[i], SUMS_FP8 * my[i] + 2 * HALF * adapter, 2 * HALF)
        # gA, gB: gh (h) is rounded to bf16 before the product: half a step of every term
        gh = s[i] * (gy[i].double() @ b[i].double())
        _close(grads[1 + i], wga[i], SUMS * mga[i] + HALF * (gh.abs().T @ xq.abs()), 2 * HALF)
        _close(grads[1 + len(outs) + i], wgb[i], SUMS * mgb[i] + HALF * (s[i] * (gy[i].double().abs().T @ (xq @ a[i].double().T).abs())), 2 * HALF)
    ghs = sum((s[i] * (gy[i].double() @ b[i].double())).abs() @ a[i].double().abs() for i in range(len(outs)))
    _close(grads[0], wgx, SUMS * mgx + HALF * ghs, 2 * HALF)


@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (1, 64, 128), (20, 192, 128), (32, 4096, 256), (64, 640, 384), (65, 128, 1152), (167, 512, 1024), (700, 4096, 320),
                                   (1024, 1024, 1024), (1100, 64, 2048), (550, 2048, 4096)])
def test_linear_grad_input(m, n, k):
    w, dense = _weight(n, k, 11)
    g = _seed(12)
    x = torch.randn(2, m, k, generator=g).to(BF)
    gy = torch.randn(2, m, n, generator=g).to(BF)
    bias = torch.randn(n, generator=g).to(BF)
    xd, bd = x.cuda().requires_grad_(), bias.cuda().requires_grad_()
    y = linear_mx(xd, w, bd)
    gx, gb = torch.autograd.grad(y, [xd, bd], gy.cuda())
    _close(gx, gy.double() @ dense, SUMS * (gy.double().abs() @ dense.abs()))
    _close(gb, gy.double().sum((0, 1)), SUMS * gy.double().abs().sum((0, 1)))


@pytest.mark.parametrize("act", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m", [1, 3, 16, 17, 32, 47, 48, 49, 64, 65])
@pytest.mark.parametrize("n,k", [(70, 96), (8200, 1056), (8192 + 16, 4096)])
def test_linear_few_tokens(m, n, k, act):
    """Every shape of the kernels for a handful of tokens: one to four tiles of tokens, 16 and 32 outputs per workgroup, and
    inputs over the whole range."""
    w, dense = _weight(n, k, 20)
    x = _special((m, k), 21, torch.float32)
    x = torch.where(x.abs() > 1e20, x * 1e-20, x).to(BF)  # products stay in range
    y = linear_mx(x.cuda(), w, activation=act)
    xq = ox.nearest(x, act)
    _close(y, xq @ dense.T, (SUMS_FP8 if act == "mxfp8" else SUMS) * (xq.abs() @ dense.abs().T), 1.0)


@pytest.mark.parametrize("act", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m", [1, 16, 40, 300])
def test_linear_non_finite_inputs_stay_in_their_row(m, act):
    """A block of NaN (or with an infinity) makes its token NaN and no other; a NaN block of the weight its output."""
    w, dense = _weight(96, 256, 22)
    x = torch.randn(m, 256, generator=_seed(23)).to(BF)
    x[0, 200] = float("nan")
    if m > 2:
        x[2, 3] = -float("inf")
    w.scales[5, 7] = 255
    y = linear_mx(x.cuda(), w, activation=act).cpu()
    bad = torch.zeros(m, 96, dtype=torch.bool)
    bad[0], bad[:, 5] = True, True
    if m > 2:
        bad[2] = True
    assert torch.equal(torch.isnan(y), bad)
    xq = ox.nearest(x, act)
    want = (xq.nan_to_num() @ dense.T)[~bad]
    _close(y[~bad], want, (SUMS_FP8 if act == "mxfp8" else SUMS) * (xq.nan_to_num().abs() @ dense.abs().T)[~bad])

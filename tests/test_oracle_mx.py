"""Pins of the microscaled oracle (CPU), and what the public functions refuse before any kernel."""
import pytest
import torch

from oracle import mx_oracle as ox
from torchtune_amd import MXTensor, linear_mx, lora_linear_mx, to_mx


def test_tables():
    assert ox.FP4.tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    t = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(t, ox.fp8_table())


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_known_blocks(fmt):
    x = torch.zeros(4, 32)
    x[1, 0], x[1, 1] = 6.0 if fmt == "mxfp4" else 448.0, 0.25  # the top of the format: scale 1
    x[2, 3] = -1.0
    x[3, 0], x[3, 1] = 7.9, 1.0                                 # above the top: saturates
    codes, scales = ox.quantize(x, fmt)
    assert scales[0].item() == 0 and not codes[0].any()
    assert scales[1].item() == 127
    v = ox.values(codes, scales, fmt)
    if fmt == "mxfp4":
        assert v[1, :2].tolist() == [6.0, 0.0]                  # 0.25 is half way between 0 and 0.5: the even code
        assert v[3, 0].item() == 6.0
    else:
        assert v[1, :2].tolist() == [448.0, 0.25]
        assert v[3, 0].item() == 7.0
    assert v[2, 3].item() == -1.0
    assert torch.equal(ox.unpack(ox.pack(codes, fmt), fmt), codes)


def test_rounding_is_torch_fp8_rounding_inside_the_range():
    x = (torch.rand(64, 32, dtype=torch.float64, generator=torch.Generator().manual_seed(0)) * 2 - 1) * 440
    x[:, 0] = 400.0  # scale 1
    codes, scales = ox.quantize(x.float(), "mxfp8")
    assert (scales == 127).all()
    assert torch.equal(codes.view(torch.float8_e4m3fn).float(), x.float().to(torch.float8_e4m3fn).float())


def test_non_finite_blocks():
    x = torch.ones(3, 64)
    x[0, 5], x[1, 40], x[2, 63] = float("inf"), float("nan"), -float("inf")
    v = ox.nearest(x, "mxfp8")
    assert torch.isnan(v[0, :32]).all() and (v[0, 32:] == 1).all() and torch.isnan(v[1, 32:]).all() and torch.isnan(v[2, 32:]).all()


def _weight(n=64, k=64, fmt="mxfp4"):
    per = 2 if fmt == "mxfp4" else 1
    return MXTensor(torch.zeros(n, k // per, dtype=torch.uint8), torch.full((n, k // 32), 127, dtype=torch.uint8), format=fmt)


def test_mx_tensor_checks():
    u8 = torch.uint8
    w = _weight(3, 64)
    assert tuple(w.shape) == (3, 64) and w.device.type == "cpu" and "mxfp4" in repr(w)
    assert tuple(_weight(3, 64, "mxfp8").shape) == (3, 64)
    with pytest.raises(TypeError):
        MXTensor(torch.zeros(3, 32), torch.zeros(3, 2, dtype=u8))
    with pytest.raises(ValueError):
        MXTensor(torch.zeros(3, 32, dtype=u8), torch.zeros(3, 3, dtype=u8))
    with pytest.raises(ValueError):
        MXTensor(torch.zeros(3, 32, dtype=u8), torch.zeros(4, 2, dtype=u8))
    with pytest.raises(ValueError):
        MXTensor(torch.zeros(3, 32, dtype=u8), torch.zeros(3, 2, dtype=u8), format="mxfp6")


def test_refusals_come_before_the_device_is_asked_for():
    """CPU tensors throughout: what is wrong with shapes, types and formats is said first."""
    bf = torch.bfloat16
    x, w = torch.zeros(4, 64, dtype=bf), _weight(128, 64)
    a, b = torch.zeros(8, 64, dtype=bf), torch.zeros(128, 8, dtype=bf)
    with pytest.raises(TypeError):
        to_mx(torch.zeros(4, 64, dtype=torch.float16))
    for bad in (torch.zeros(4, 48), torch.zeros(()), torch.zeros(4, 0)):
        with pytest.raises(ValueError):
            to_mx(bad)
    with pytest.raises(ValueError):
        to_mx(torch.zeros(4, 64), "nf4")
    with pytest.raises(TypeError):
        w.to(torch.float16)
    with pytest.raises(TypeError):
        linear_mx(x.float(), w)
    with pytest.raises(TypeError):
        linear_mx(x, _weight(128, 64, "mxfp8"))
    with pytest.raises(RuntimeError, match="shapes cannot be multiplied"):
        linear_mx(torch.zeros(4, 96, dtype=bf), w)
    with pytest.raises(ValueError, match="inputs"):
        linear_mx(torch.zeros(4, 0, dtype=bf), _weight(0, 0))
    with pytest.raises(ValueError):
        linear_mx(x, w, activation="int8")
    with pytest.raises(ValueError):
        linear_mx(x, w, torch.zeros(127, dtype=bf))
    with pytest.raises(TypeError):
        linear_mx(x, w, torch.zeros(128))
    with pytest.raises(ValueError, match="multiples of 64"):
        linear_mx(x.clone().requires_grad_(), _weight(100, 64))
    ok = (x, [w], [a], [b], [2.0])
    cases = [
        (ValueError, (x, [], [], [], [])),
        (ValueError, (x, [w] * 5, [a] * 5, [b] * 5, [1.0] * 5)),
        (ValueError, (x, [w], [a], [b], [])),
        (ValueError, (x, [w], [a[:, :32]], [b], [2.0])),
        (ValueError, (x, [w], [a[:4]], [b[:, :4]], [2.0])),
        (ValueError, (x, [w], [a], [b[:64]], [2.0])),
        (ValueError, (x, [_weight(72, 64)], [a], [b[:72]], [2.0])),
        (ValueError, (x, [w], [a], [b], [2.0], [torch.zeros(64, dtype=bf)])),
        (ValueError, (x, [w] * 2, [torch.zeros(40, 64, dtype=bf)] * 2, [torch.zeros(128, 40, dtype=bf)] * 2, [1.0] * 2)),
        (TypeError, (x, [w], [a.float()], [b], [2.0])),
        (TypeError, (x.float(), *ok[1:])),
        (RuntimeError, (torch.zeros(4, 128, dtype=bf), *ok[1:])),
    ]
    for err, args in cases:
        with pytest.raises(err):
            lora_linear_mx(*args)


def test_cpu_tensors_are_refused():
    w = _weight()
    with pytest.raises(RuntimeError, match="AMD GPU"):
        to_mx(torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match="AMD GPU"):
        w.to()
    with pytest.raises(RuntimeError, match="AMD GPU"):
        linear_mx(torch.zeros(4, 64, dtype=torch.bfloat16), w)
    bf = torch.bfloat16
    with pytest.raises(RuntimeError, match="AMD GPU"):
        lora_linear_mx(torch.zeros(4, 64, dtype=bf), [w], [torch.zeros(8, 64, dtype=bf)], [torch.zeros(64, 8, dtype=bf)], [1.0])


def test_module_refusals():
    from torchtune_amd import FrozenMXLinear, MXLoRALinear, harness

    for args in ((100, 64, 8, 16.0), (64, 96, 8, 16.0), (64, 64, 12, 16.0), (64, 64, 0, 16.0), (64, 64, 72, 16.0)):
        with pytest.raises(ValueError):
            MXLoRALinear(*args)
    with pytest.raises(ValueError, match="multiple of 32"):
        FrozenMXLinear(48, 64)
    with pytest.raises(ValueError, match="unknown format"):
        FrozenMXLinear(64, 64, activation="int8")
    with pytest.raises(RuntimeError, match="AMD GPU"):
        FrozenMXLinear(64, 64)
    with pytest.raises(ValueError, match="unknown base"):
        harness.build_qlora_decoder("tiny", 8, 16.0, base="int4")
    with torch.device("meta"):
        m = MXLoRALinear(128, 64, 8, 16.0, use_bias=True)
    assert tuple(m.weight_codes.shape) == (64, 64) and tuple(m.weight_scales.shape) == (64, 4) and m.adapter_params() == ["lora_a.weight", "lora_b.weight"]
    assert tuple(m.mx_weight.shape) == (64, 128)


def test_c_entries_refuse_before_they_launch():
    """Addresses that are never read: every call below is turned away by its checks."""
    import ctypes

    from torchtune_amd import _lib

    lib = _lib.load()
    EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -3  # the header's codes
    p, odd, none = ctypes.c_void_p(1 << 12), ctypes.c_void_p((1 << 12) + 2), None

    def member(**kw):
        f = dict(codes=1 << 12, scales=1 << 12, lora_a=1 << 12, lora_b=1 << 12, bias=None, y=1 << 12, grad_lora_a=1 << 12, grad_lora_b=1 << 12,
                 N=128, rank=8, scale=1.0)
        f.update(kw)
        return _lib.MxLoraMember(**f)

    def ptr(*ms):
        arr = (_lib.MxLoraMember * len(ms))(*ms)
        return ctypes.cast(arr, ctypes.c_void_p), len(ms)

    fwd = lambda ms, x=p, m=4, k=64, ws=p, n=1 << 40: lib.ttamd_mx_lora_fwd_bf16(x, *ptr(*ms), p, p, p, m, k, ws, n, None)
    bwd = lambda ms, gx=p, m=4, k=64, ws=p, n=1 << 40: lib.ttamd_mx_lora_bwd_bf16(p, p, p, *ptr(*ms), p, gx, m, k, ws, n, None)
    lin = lambda x=p, f=8, m=4, n=128, k=64, ws=p, size=1 << 40, w=p, y=p, bias=none: lib.ttamd_mx_linear_bf16(x, f, w, p, bias, y, m, n, k, ws, size, None)
    dx = lambda m=4, n=128, k=64, ws=p, size=1 << 40, gy=p, s=p: lib.ttamd_mx_linear_dx_bf16(gy, p, s, p, m, n, k, ws, size, None)
    cases = [
        (EINVAL, lambda: lib.ttamd_mx_quantize(p, 99, 4, 64, 4, p, p, None)),
        (EINVAL, lambda: lib.ttamd_mx_quantize(p, _lib.TTAMD_BF16, 4, 48, 4, p, p, None)),
        (EINVAL, lambda: lib.ttamd_mx_quantize(p, _lib.TTAMD_BF16, 4, 64, 5, p, p, None)),
        (EINVAL, lambda: lib.ttamd_mx_quantize(odd, _lib.TTAMD_BF16, 4, 64, 4, p, p, None)),
        (EINVAL, lambda: lib.ttamd_mx_dequantize(p, none, 4, 4, 64, _lib.TTAMD_BF16, p, None)),
        (EINVAL, lambda: lin(f=5)), (EINVAL, lambda: lin(k=48)), (EINVAL, lambda: lin(m=0)), (EINVAL, lambda: lin(x=odd)), (EINVAL, lambda: lin(y=none)),
        (EINVAL, lambda: lin(bias=ctypes.c_void_p(4097))), (EUNSUPPORTED, lambda: lin(k=1 << 23)), (EWORKSPACE, lambda: lin(m=400, size=0)),
        (EWORKSPACE, lambda: lin(m=400, ws=none)), (EWORKSPACE, lambda: lin(m=400, ws=odd)),
        (EINVAL, lambda: dx(n=96)), (EINVAL, lambda: dx(k=96)), (EINVAL, lambda: dx(gy=odd)), (EINVAL, lambda: dx(s=odd)), (EUNSUPPORTED, lambda: dx(n=1 << 23)), (EUNSUPPORTED, lambda: dx(n=1 << 22)),
        (EWORKSPACE, lambda: dx(m=4096, n=4096, k=4096, size=16)),
        (EINVAL, lambda: lib.ttamd_mx_lora_fwd_bf16(p, None, 1, p, p, p, 4, 64, p, 1 << 40, None)),
        (EINVAL, lambda: fwd([member()] * 5)), (EINVAL, lambda: fwd([member()], k=96)), (EINVAL, lambda: fwd([member()], m=0)),
        (EINVAL, lambda: fwd([member(N=96)])), (EINVAL, lambda: fwd([member(rank=4)])), (EINVAL, lambda: fwd([member(rank=40), member(rank=32)])),
        (EINVAL, lambda: fwd([member(lora_b=None)])), (EINVAL, lambda: fwd([member(scales=4098)])), (EINVAL, lambda: fwd([member()], x=odd)),
        (EUNSUPPORTED, lambda: fwd([member(N=1 << 22)])), (EUNSUPPORTED, lambda: fwd([member(N=(1 << 22) - 64)] * 3)), (EWORKSPACE, lambda: fwd([member()], n=16)), (EWORKSPACE, lambda: fwd([member()], ws=none)),
        (EINVAL, lambda: bwd([member(grad_lora_a=None)])), (EINVAL, lambda: bwd([member()], gx=odd)), (EWORKSPACE, lambda: bwd([member()], n=16)),
    ]
    for i, (want, call) in enumerate(cases):
        assert call() == want, (i, lib.ttamd_last_error())
    assert lib.ttamd_mx_linear_workspace_bytes(0, 1, 64, 8) == 0 and lib.ttamd_mx_lora_fwd_workspace_bytes(*ptr(member(rank=4)), 4, 64) == 0
    assert lib.ttamd_mx_kept_codes_bytes(3, 320) == 3 * 512 and lib.ttamd_mx_kept_scales_bytes(3, 320) == 3 * 16


def test_backward_entry_refuses_adapter_gradients_that_are_null_for_some():
    """All of them null: not wanted.  One of them: a mistake, of whichever member."""
    import ctypes

    from torchtune_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(1 << 12)

    def bwd(size, *grads):
        arr = (_lib.MxLoraMember * len(grads))(*(_lib.MxLoraMember(codes=1 << 12, scales=1 << 12, lora_a=1 << 12, lora_b=1 << 12, y=1 << 12, grad_lora_a=a,
                                                                    grad_lora_b=b, N=128, rank=8, scale=1.0) for a, b in grads))
        return lib.ttamd_mx_lora_bwd_bf16(p, p, p, ctypes.cast(arr, ctypes.c_void_p), len(grads), p, p, 4, 64, p, size, None)

    q = 1 << 12
    for grads in (((None, q),), ((q, None),), ((q, q), (None, None)), ((None, None), (q, q)), ((q, q), (q, None)), ((q + 2, q),)):
        assert bwd(1 << 40, *grads) == -1, grads
    for grads in (((None, None),), ((None, None), (None, None))):
        assert bwd(0, *grads) == -3 and b"workspace" in lib.ttamd_last_error()  # past the members' checks

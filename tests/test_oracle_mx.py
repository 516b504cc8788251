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

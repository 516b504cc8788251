"""What the calls around a post-training step refuse before any kernel is launched, and what needs no GPU (all on the CPU)."""
import ctypes

import pytest
import torch

from torchtune_amd import AdamW, _lib
from torchtune_amd.modules import layer_ops


def _rope(q=(2, 3, 4, 32), k=(2, 3, 2, 32), cache=(8, 16, 2), dtype=torch.bfloat16, k_dtype=None, cache_dtype=torch.float32, scales=None, **more):
    w = [None, None] if scales is None else [None if s is None else torch.ones(s, dtype=dtype) for s in scales]
    return layer_ops.qk_norm_rope(torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=k_dtype or dtype), torch.zeros(cache, dtype=cache_dtype), *w, **more)


@pytest.mark.parametrize("error,match,call", [
    (RuntimeError, "AMD GPU", lambda: _rope()),
    (TypeError, "not supported", lambda: _rope(dtype=torch.float16)),
    (TypeError, "k ", lambda: _rope(k_dtype=torch.float32)),
    (ValueError, "expected", lambda: _rope(k=(2, 4, 2, 32))),
    (ValueError, "expected", lambda: _rope(q=(6, 4, 32))),
    (ValueError, "multiple of 16", lambda: _rope(q=(2, 3, 4, 24), k=(2, 3, 2, 24), cache=(8, 12, 2))),
    (ValueError, "multiple of 16", lambda: _rope(q=(2, 3, 4, 528), k=(2, 3, 2, 528), cache=(8, 264, 2))),
    (TypeError, "float32", lambda: _rope(cache_dtype=torch.bfloat16)),
    (ValueError, "cache must", lambda: _rope(cache=(8, 8, 2))),
    (ValueError, "the sequence", lambda: _rope(cache=(2, 16, 2))),
    (ValueError, "neither", lambda: _rope(scales=[32, None])),
    (ValueError, "a scale must", lambda: _rope(scales=[32, 16])),
    (ValueError, "need positions", lambda: _rope(sections=[8, 8])),
    (ValueError, "need positions", lambda: _rope(sections=[8, 8], positions=torch.zeros(2, 3, dtype=torch.long))),
    (ValueError, "add up", lambda: _rope(sections=[8, 9], positions=torch.zeros(2, 2, 3, dtype=torch.long))),
    (ValueError, "section of", lambda: _rope(sections=[20, -4], positions=torch.zeros(2, 2, 3, dtype=torch.long))),
    (ValueError, "add up", lambda: _rope(sections=[16], positions=torch.zeros(1, 2, 3, dtype=torch.long))),
    (TypeError, "int64", lambda: _rope(positions=torch.zeros(2, 3))),
    (ValueError, "do not fit", lambda: _rope(positions=torch.zeros(2, 4, dtype=torch.long))),
    (ValueError, "do not fit", lambda: _rope(positions=torch.zeros(3, 2, 3, dtype=torch.long))),
])
def test_qk_norm_rope_refuses(error, match, call):
    with pytest.raises(error, match=match):
        call()


def _logprobs(logits=(2, 3, 9), tokens=(2, 3), dtype=torch.float32, token_dtype=torch.long, **more):
    return layer_ops.token_logprobs(torch.zeros(logits, dtype=dtype), torch.zeros(tokens, dtype=token_dtype), **more)


@pytest.mark.parametrize("error,match,call", [
    (RuntimeError, "AMD GPU", lambda: _logprobs()),
    (TypeError, "not supported", lambda: _logprobs(dtype=torch.float64)),
    (TypeError, "int64", lambda: _logprobs(token_dtype=torch.int32)),
    (ValueError, "do not fit", lambda: _logprobs(tokens=(2, 4))),
    (ValueError, "do not fit", lambda: _logprobs(tokens=(6,))),
    (ValueError, "do not fit", lambda: _logprobs(tokens=(2, 3, 0))),
    (ValueError, "expected logits", lambda: _logprobs(logits=(2, 3, 0))),
    (ValueError, "temperature", lambda: _logprobs(temperature=0.0)),
    (ValueError, "temperature", lambda: _logprobs(temperature=-1.0)),
    (ValueError, "temperature", lambda: _logprobs(temperature=float("nan"))),
    (ValueError, "top must", lambda: _logprobs(top=10)),
    (ValueError, "top must", lambda: _logprobs(logits=(2, 3, 100), top=65)),
    (ValueError, "top must", lambda: _logprobs(top=-1)),
])
def test_token_logprobs_refuses(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_adamw_refuses():
    p = torch.nn.Parameter(torch.zeros(4))
    for error, more in ((ValueError, dict(lr=-1.0)), (ValueError, dict(eps=-1.0)), (ValueError, dict(weight_decay=-0.1)), (ValueError, dict(betas=(0.9, 1.0))),
                        (ValueError, dict(betas=(-0.1, 0.9))), (ValueError, dict(state_bits=16)), (TypeError, dict(lr=torch.tensor(0.1))),
                        (ValueError, dict(lr=float("nan")))):
        with pytest.raises(error):
            AdamW([p], **more)
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="twice"):
        AdamW([p, p]).step()
    opt = AdamW([p])
    opt.step()  # no gradient, nothing to do
    assert not opt.state
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        opt.step()
    assert not opt.state
    with pytest.raises(RuntimeError, match="no parameter"):
        opt.moments()


def test_the_c_entries_check_their_arguments():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) & ~255
    heads = (_lib.RopeHeads * 2)()
    at = _lib.RopePositions(p, 8, None, (ctypes.c_int64 * 3)(), 1, (ctypes.c_int * 4)(), 1)

    def rope(bwd=False, D=32, B=1, S=4, dtype=0, eps=1e-6, ws=0):
        args = [heads, ctypes.byref(at), dtype, eps, B, S, D]
        rc = lib.ttamd_qk_norm_rope_bwd(*args, p if ws else None, ws, None) if bwd else lib.ttamd_qk_norm_rope_fwd(*args, None)
        return rc, lib.ttamd_last_error().decode()

    assert rope()[0] == -1 and "no heads" in rope()[1]
    heads[0].heads = 2
    assert rope()[0] == -1 and "null" in rope()[1]
    heads[0].x = heads[0].out = p
    assert rope(D=24)[0] == -1 and rope(D=528)[0] == -1 and rope(B=0)[0] == -1 and rope(dtype=5)[0] == -1
    assert rope(S=9)[0] == -1 and "table" in rope(S=9)[1]
    at.n_axes = 3
    assert rope()[0] == -1 and "axes" in rope()[1]
    at.positions = p
    assert rope()[0] == -1 and "sections" in rope()[1]
    at.section[0], at.section[1], at.section[2] = 20, -4, 0
    assert rope()[0] == -1
    at.n_axes = 1
    heads[1].heads, heads[1].x, heads[1].out, heads[1].scale = 1, p, p, p
    assert rope()[0] == -1 and "neither" in rope()[1]
    heads[0].scale, heads[1].x = p, p + 1
    assert rope()[0] == -1 and "misaligned" in rope()[1]
    heads[1].x = p
    heads[0].gy = heads[1].gy = heads[0].gscale = p
    assert rope(bwd=True)[0] == -1 and "workspace" in rope(bwd=True)[1]
    assert rope(bwd=True, ws=64)[0] == -3
    heads[0].heads = 1 << 19
    assert rope(B=1 << 12, S=1)[0] == -1 and "2^31" in rope(B=1 << 12, S=1)[1]

    logits = _lib.Logits(p, 1, 2, 9, 2, 0, 9)

    def logprobs(top=0, temperature=1.0, n=1, ws=0, out=p):
        rc = lib.ttamd_token_logprobs_fwd(ctypes.byref(logits), p, n, -100, temperature, out, None, top, p if top else None, p if top else None, None,
                                          p if ws else None, ws, None)
        return rc, lib.ttamd_last_error().decode()

    assert logprobs(out=None)[0] == -1 and logprobs(top=10)[0] == -1 and logprobs(top=65)[0] == -1 and logprobs(temperature=0.0)[0] == -1
    assert logprobs(temperature=float("nan"))[0] == -1 and logprobs(n=-1)[0] == -1 and logprobs(n=1 << 17)[0] == -1
    logits.V = 100000
    need = lib.ttamd_token_logprobs_workspace_bytes(2, 100000, 5)
    assert need > 0 and logprobs(top=5)[0] == -1 and logprobs(top=5, ws=need - 1)[0] == -3
    logits.data = p + 2
    assert logprobs()[0] == -1 and "misaligned" in logprobs()[1]
    logits.data = p
    logits.dtype = 3
    assert logprobs()[0] == -1
    assert lib.ttamd_token_logprobs_workspace_bytes(0, 5, 1) == 0 and lib.ttamd_token_logprobs_workspace_bytes(5, 5, 65) == 0
    assert lib.ttamd_token_logprobs_bwd(ctypes.byref(logits), p, 1, -100, 1.0, p, p, None, p, None) == -1
    logits.dtype = 1
    assert lib.ttamd_token_logprobs_bwd(ctypes.byref(logits), p, 1, -100, 1.0, None, p, None, p, None) == -1
    assert lib.ttamd_token_logprobs_bwd(ctypes.byref(logits), p, 1, -100, 1.0, p, None, None, p, None) == -1

    states = _lib.AdamWStates(p, p, p, None, None, 32)
    scalars = _lib.AdamWScalars(1e-3, 0.9, 0.999, 1e-8, 0.01, 1, 0, 0)
    ptrs = (ctypes.c_void_p * 1)(p)

    def adamw(n=1, dtype=1, chunks=1):
        rc = lib.ttamd_adamw_step(ptrs, n, dtype, ctypes.byref(states), 0, 0, chunks, ctypes.byref(scalars), None)
        return rc, lib.ttamd_last_error().decode()

    assert adamw(n=0)[0] == -1 and adamw(n=481)[0] == -1 and adamw(dtype=4)[0] == -1 and adamw(chunks=0)[0] == -1
    for name, value in (("step", 0), ("beta1", 1.0), ("beta2", -0.5), ("eps", -1.0), ("stochastic", 1)):
        keep = getattr(scalars, name)
        setattr(scalars, name, value)
        assert adamw()[0] == -1, name
        setattr(scalars, name, keep)
    states.state_bits = 8
    assert adamw()[0] == -1 and "null" in adamw()[1]
    states.state_bits = 16
    assert adamw()[0] == -1 and "bits" in adamw()[1]
    states.state_bits = 32
    for bad in (None, p + 2):
        ptrs[0] = bad
        assert adamw()[0] == -1 and "pointer" in adamw()[1]
    assert lib.ttamd_adamw_moments_bf16(ctypes.byref(states), 1, p, p, None) == -1


def test_the_numbers_of_the_stochastic_rounding():
    """Uniform, and without a pattern along a tensor, from tensor to tensor or from step to step: means and correlations of n numbers
    within five of their standard deviations, 1 / sqrt(n)."""
    lib = _lib.load()
    n = 20000
    rows = []
    for step in (1, 2):
        for tensor in (0, 1):
            key = lib.ttamd_adamw_key(3, step, tensor)
            r = torch.tensor([lib.ttamd_adamw_number(key, i) for i in range(n)], dtype=torch.int64)
            for half in (r >> 16, r & 0xFFFF):
                rows.append((half.double() + 0.5) / 65536 - 0.5)
    bound = 5 / n ** 0.5
    unit = [x * 12 ** 0.5 for x in rows]
    for i, x in enumerate(unit):
        assert abs(float(x.mean())) < bound and abs(float((x * x).mean()) - 1) < bound
        for lag in (1, 2, 8, 128):
            assert abs(float((x[:-lag] * x[lag:]).mean())) < bound * 1.01
        for y in unit[:i]:
            assert abs(float((x * y).mean())) < bound
    key = lib.ttamd_adamw_key(3, 1, 0)
    far = [lib.ttamd_adamw_number(key, i + (1 << 32)) for i in range(64)]
    assert far != [lib.ttamd_adamw_number(key, i) for i in range(64)]

"""What surrounds the linears of a post-training step: the rotation of queries and keys, the log probabilities that a loss or a
sampler reads, and the step of the optimizer.

* ``rotate``: every query and key head is normalised by its root mean square, scaled, and rotated by the angles of its token's
  position; or rotated alone.  A position has one axis, or three (time, height, width of images and video) that share out the
  frequencies in sections.  A frequency turns two neighbouring elements (interleaved) or an element of the first half with
  its counterpart in the second.
* ``logprobs``: ``z = logits / temperature``; log softmax at one or several given tokens of each row, the entropy of the
  row, its largest log probabilities with their tokens; and the gradient of the first two.  A token of -100 has a log probability
  of 0 and no gradient.
* ``adamw``: one step over many tensors.  ``m' = b1 m + (1 - b1) g``, ``v' = b2 v + (1 - b2) g^2``,
  ``p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)``.  The moments are held in 32 bits or in 8.

The 8-bit form: 128 consecutive elements of a tensor are a block with one exponent ``E`` for each moment.  A first moment has a
sign, four bits of exponent below E and three of mantissa; a second moment four and four; 0 is 0, and what is below the range is
0 for the first and the smallest number for the second moment.  From the 32-bit moment the mantissa is cut after a number has
been added to the bits behind it that is uniform over them, so that it is right on average: a second moment changes by a
thousandth in a step, which rounding to the nearest would never show.  The numbers come from the optimizer's seed, the step, the
tensor's place and the element's, by ``_numbers`` below: 16 bits for each moment; those of the first also round a bfloat16
parameter where that is asked for.
"""
import math

import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
_IGNORED = -100
_BLOCK = 128
_TABLE = 32768  # positions in the table of angles
_BETAS, _EPS, _LR, _DECAY, _SEED, _STEPS = (0.9, 0.999), 1e-8, 3e-4, 0.01, 1234, 100


# ---------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------
def _rotate(batch, seq, heads, kv, dim, norm, axes, interleaved, train, dtype="bfloat16", given=True, joined=False):
    return {"kind": "rotate", "batch": batch, "seq": seq, "heads": heads, "kv": kv, "dim": dim, "norm": norm, "axes": axes,
            "interleaved": interleaved, "train": train, "dtype": dtype, "given": given or axes > 1, "joined": joined}


def _logprobs(rows, vocab, tokens, top, entropy, train, temperature=1.0, masked=False, dtype="bfloat16"):
    return {"kind": "logprobs", "rows": rows, "vocab": vocab, "tokens": tokens, "top": top, "entropy": entropy, "train": train,
            "temperature": temperature, "masked": masked, "dtype": dtype}


def _adamw(sizes, bits, dtype, stochastic=False):
    return {"kind": "adamw", "sizes": sizes, "bits": bits, "dtype": dtype, "stochastic": stochastic}


def _sizes(case):
    """"65536*2 77" -> [65536, 65536, 77]"""
    out = []
    for part in case["sizes"].split():
        n, _, times = part.partition("*")
        out += [int(n)] * int(times or 1)
    return out


_ADAPTERS_8B = "65536*288 16384*64 229376*96"  # rank 16 on the seven linears of 32 layers


def listed():
    """The cases, kind by kind from the smallest calls to the largest."""
    return [
        # generation: one token of one sequence
        {"name": "rotate_generate_1", **_rotate(1, 1, 32, 8, 128, True, 1, False, False)},
        # a prompt of ragged length with an image in it; queries and keys are parts of one projection's output
        {"name": "rotate_prompt_333_axes", **_rotate(1, 333, 32, 8, 128, True, 3, False, False, joined=True)},
        # a training batch of the larger shape with images, full precision, rotation alone
        {"name": "rotate_train_2x700_axes_fp32", **_rotate(2, 700, 64, 8, 128, False, 3, False, True, dtype="float32")},
        # a full training batch
        {"name": "rotate_train_4x2048", **_rotate(4, 2048, 32, 8, 128, True, 1, True, True, given=False)},
        # generation: what is reported for the token of one sequence
        {"name": "logprobs_generate_1", **_logprobs(1, 128256, 1, 20, False, False, temperature=0.7)},
        # generation for many sequences, part of the vocabulary ruled out
        {"name": "logprobs_sample_48", **_logprobs(48, 128256, 1, 5, True, False, masked=True)},
        # distillation on a teacher's 16 alternatives; rows that start at odd places, full precision
        {"name": "logprobs_distill_700_odd", **_logprobs(700, 50257, 16, 0, False, True, temperature=2.0, dtype="float32")},
        # a policy's log probabilities with a bonus for their entropy
        {"name": "logprobs_train_2048", **_logprobs(2048, 128256, 1, 0, True, True)},
        # the norms and biases of a small model
        {"name": "adamw_small_fp32", **_adamw("2048*33 77*3 1 5000", 32, "float32")},
        # the adapters of the 8B shape
        {"name": "adamw_adapters", **_adamw(_ADAPTERS_8B, 32, "bfloat16")},
        {"name": "adamw_adapters_8bit", **_adamw(_ADAPTERS_8B, 8, "bfloat16")},
        # one whole layer of the 8B shape
        {"name": "adamw_layer_8bit", **_adamw("16777216*2 4194304*2 58720256*3 4096*2", 8, "bfloat16", True)},
    ]


def _log_between(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["rotate", "logprobs", "adamw"])
    if kind == "rotate":
        heads, kv = rng.choice([(32, 8), (64, 8), (32, 32), (16, 4), (28, 4), (14, 2), (8, 1)])
        dim, dtype = rng.choice([64, 64, 80, 112, 128, 128, 256]), rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        most = 4 * 2048 * 40 * 128 // ((heads + kv) * dim * (2 if dtype == "float32" else 1))
        tokens, axes = _log_between(rng, 1, most), rng.choice([1, 1, 3])
        batch = rng.choice([1, 1, 2, 3, 4, 8])
        return _rotate(batch, max(1, tokens // batch), heads, kv, dim, rng.random() < 0.7, axes, rng.random() < 0.5, rng.random() < 0.6,
                       dtype, given=rng.random() < 0.6, joined=rng.random() < 0.4)
    if kind == "logprobs":
        vocab = rng.choice([1024, 32000, 32064, 50257, 65024, 128256, 151936, _log_between(rng, 300, 262144)])
        dtype, train = rng.choice(["bfloat16", "bfloat16", "float32"]), rng.random() < 0.5
        most = 2048 * 128256 // vocab // (2 if dtype == "float32" else 1)
        rows = _log_between(rng, 1, min(8192, most if train else most // 4))
        return _logprobs(rows, vocab, rng.choice([1, 1, 1, 2, 8, 20]), 0 if train else rng.choice([0, 1, 5, 20, 50]), rng.random() < 0.5, train,
                         rng.choice([1.0, 1.0, 0.6, 2.0]), rng.random() < 0.3, dtype)
    count, dtype = _log_between(rng, 1, 300), rng.choice(["bfloat16", "bfloat16", "float32"])
    total = _log_between(rng, 1000, 50000000)
    sizes, each = [], max(1, total // count)
    while len(sizes) < count:
        times = min(rng.randrange(1, 12), count - len(sizes))
        n = _log_between(rng, max(1, each // 8), each * 2)
        n = n if rng.random() < 0.3 else max(64, n // 64 * 64)
        sizes += [n] * times
    text = " ".join(str(n) for n in sizes)
    return _adamw(text, rng.choice([8, 32]), dtype, dtype == "bfloat16" and rng.random() < 0.4)


# ---------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------
def _axis_of(case):
    """Which axis of the positions turns each frequency."""
    half = case["dim"] // 2
    out = torch.zeros(half, dtype=torch.long, device="cuda")
    if case["axes"] > 1:
        first, second, _ = _sections(case)
        out[first:first + second] = 1
        out[first + second:] = 2
    return out


def _sections(case):
    half = case["dim"] // 2
    first = half // 4
    second = (half - first) // 2
    return [first, second, half - first - second]


def _angles(s):
    """cosines and sines [batch, seq, 1, dim / 2] of every token"""
    case, table = s["case"], s["cache"]
    pos = s["positions"]
    if pos is None:
        pos = torch.arange(case["seq"], device="cuda").expand(case["batch"], -1)
    if pos.dim() == 2:
        rows = table[pos]
    else:
        frequency = torch.arange(case["dim"] // 2, device="cuda")
        rows = table[pos[_axis_of(case)].permute(1, 2, 0), frequency]
    return rows[..., 0].unsqueeze(2), rows[..., 1].unsqueeze(2)


def _pairs(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)


def _join(a, b, interleaved):
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _plain_rotate(s):
    case, t = s["case"], s["q"].dtype
    cos, sin = _angles(s)
    out = {"out": []}
    grads, scales = [], []
    for x, w, gy in ((s["q"], s["q_scale"], s["gq"]), (s["k"], s["k_scale"], s["gk"])):
        x = x.float()
        n = x
        if w is not None:
            r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + s["eps"])
            n = x * r * w.float()
        a, b = _pairs(n, case["interleaved"])
        out["out"].append(_join(a * cos - b * sin, b * cos + a * sin, case["interleaved"]).to(t))
        if not case["train"]:
            continue
        a, b = _pairs(gy.float(), case["interleaved"])
        g = _join(a * cos + b * sin, b * cos - a * sin, case["interleaved"])
        if w is not None:
            scales.append((g * x * r).sum((0, 1, 2)).to(w.dtype))
            g = g * w.float()
            g = r * (g - x * (r * r * (g * x).mean(-1, keepdim=True)))
        grads.append(g.to(t))
    if case["train"]:
        out["grad"], out["grad_scale"] = grads, scales
    return out


def _plain_logprobs(s):
    case, tokens = s["case"], s["tokens"].reshape(s["case"]["rows"], -1)
    z = s["logits"].float() / case["temperature"]
    m = z.amax(-1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    kept = tokens != _IGNORED
    at = torch.where(kept, tokens, torch.zeros_like(tokens))
    out = {"logprobs": torch.where(kept, d.gather(1, at) - log_total, torch.zeros((), device="cuda")).view(s["tokens"].shape)}
    if case["entropy"]:
        mean = torch.where(e > 0, e * d, torch.zeros((), device="cuda")).sum(-1, keepdim=True) / total
        entropy = log_total - mean
        out["entropy"] = entropy.squeeze(-1)
    if case["top"]:
        # by the logits themselves, which division and difference may round together; of equal ones the first comes first
        order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_logprobs"] = d.gather(1, order) - log_total
        out["top_tokens"] = order
    if case["train"]:
        p = e / total
        g = torch.where(kept, s["g_logprobs"].reshape(case["rows"], -1), torch.zeros((), device="cuda"))
        grad = -p * g.sum(-1, keepdim=True)
        if case["entropy"]:
            log_p = torch.where(e > 0, d - log_total, torch.zeros((), device="cuda"))
            grad = grad - s["g_entropy"].unsqueeze(-1) * p * (log_p + entropy)
        grad.scatter_add_(1, at, g)
        out["grad"] = (grad / case["temperature"]).to(s["logits"].dtype)
    return out


_MASK32, _MASK64 = (1 << 32) - 1, (1 << 64) - 1


def _key(seed, step, tensor):
    """32 bits for a tensor's numbers in a step"""
    z = (seed * 0x9E3779B97F4A7C15 + step * 0xBF58476D1CE4E5B9 + tensor * 0x94D049BB133111EB + 0x6A09E667F3BCC909) & _MASK64
    z = ((z ^ (z >> 32)) * 0xD6E8FEB86659FD93) & _MASK64
    z = ((z ^ (z >> 32)) * 0xD6E8FEB86659FD93) & _MASK64
    return (z ^ (z >> 32)) & _MASK32


def _numbers(n, key):
    """Two 16-bit numbers for each of n elements (n below 2^32): (for the second moment, for the first moment and the parameter)"""
    x = (torch.arange(n, dtype=torch.int64, device="cuda") * 0x9E3779B9 + key) & _MASK32
    for shift, factor in ((16, 0x6A09E667), (15, 0xBB67AE85)):
        x = x ^ (x >> shift)
        # 32 x 32 bits: in two halves, so that 63 bits hold them
        x = ((x & 0xFFFF) * factor + (((x >> 16) * factor & 0xFFFF) << 16)) & _MASK32
    x = x ^ (x >> 16)
    return x >> 16, x & 0xFFFF


def _blocks(x, fill=0):
    n = x.numel()
    padded = torch.full((-(-n // _BLOCK) * _BLOCK,), fill, dtype=x.dtype, device=x.device)
    padded[:n] = x.reshape(-1)
    return padded.view(-1, _BLOCK)


def _hold(x, numbers, mantissa):
    """(codes [n], exponents [blocks]) of 32-bit moments: ``mantissa`` is 3 with a sign or 4 without"""
    n, drop = x.numel(), 23 - mantissa
    bits = x.reshape(-1).view(torch.int32).to(torch.int64)
    size = (bits & 0x7FFFFFFF).clamp(max=0x7F800000)
    k = (size + (numbers << (drop - 16)) + (1 << (drop - 17))) >> drop
    exponent = (_blocks(k).amax(-1) >> mantissa).clamp(min=16)
    base = ((exponent - 15) << mantissa).repeat_interleave(_BLOCK)[:n]
    code = k - base
    if mantissa == 3:
        code = torch.where(code < 1, torch.zeros_like(code), code + 128 * (bits < 0).to(torch.int64))
    else:
        code = torch.where(size == 0, torch.zeros_like(code), code.clamp(min=1))
    return code.to(torch.uint8), exponent.to(torch.uint8)


def _held(code, exponent, mantissa):
    """32-bit values of what is held"""
    n, drop = code.numel(), 23 - mantissa
    base = ((exponent.to(torch.int32) - 15) << mantissa).repeat_interleave(_BLOCK)[:n]
    code = code.to(torch.int32)
    size = code & (127 if mantissa == 3 else 255)
    value = torch.where(size == 0, torch.zeros_like(size), (size + base) << drop).view(torch.float32)
    return torch.where(code > 127, -value, value) if mantissa == 3 else value


def _scalars(step):
    (b1, b2) = _BETAS
    return {"b1": b1, "c1": 1 - b1, "b2": b2, "c2": 1 - b2, "keep": 1 - _LR * _DECAY, "rate": _LR / (1 - b1 ** step),
            "root": 1 / math.sqrt(1 - b2 ** step)}


def _plain_adamw(s):
    case, eight = s["case"], s["case"]["bits"] == 8
    s["step"] += 1
    c = _scalars(s["step"])
    moments = ([], [])
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        if eight:
            m, v = _held(s["m"][i], s["m_exponent"][i], 3), _held(s["v"][i], s["v_exponent"][i], 4)
        else:
            m, v = s["m"][i], s["v"][i]
        w, g = p.detach().float(), g.float()
        m = m * c["b1"] + g * c["c1"]
        v = v * c["b2"] + (g * g) * c["c2"]
        w = w * c["keep"] - c["rate"] * (m / (torch.sqrt(v) * c["root"] + _EPS))
        if eight or case["stochastic"]:
            high, low = _numbers(p.numel(), _key(_SEED, s["step"], i))
        if case["stochastic"]:
            bits = w.view(torch.int32).to(torch.int64) & _MASK32
            w = (((bits + low) >> 16) << 16).to(torch.int32).view(torch.float32)
        p.data.copy_(w)
        if not eight:
            s["m"][i].copy_(m)
            s["v"][i].copy_(v)
            continue
        for held, exponents, x, numbers, mantissa, values in ((s["m"], s["m_exponent"], m, low, 3, moments[0]),
                                                              (s["v"], s["v_exponent"], v, high, 4, moments[1])):
            code, exponent = _hold(x, numbers, mantissa)
            held[i].copy_(code)
            exponents[i].copy_(exponent)
            values.append(_held(code, exponent, mantissa).to(torch.bfloat16))  # five significant bits: nothing is lost
    if eight:
        return {"params": s["whole"], "exp_avg": torch.cat(moments[0]), "exp_avg_sq": torch.cat(moments[1])}
    return {"params": s["whole"], "exp_avg": s["m_whole"], "exp_avg_sq": s["v_whole"]}


# ---------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------
def _own_rotate(s):
    from torchtune_amd.modules import layer_ops

    case = s["case"]
    out = layer_ops.qk_norm_rope(s["q"], s["k"], s["cache"], s["q_scale"], s["k_scale"], eps=s["eps"], positions=s["positions"],
                                 sections=s["sections"], interleaved=case["interleaved"])
    if not case["train"]:
        return {"out": list(out)}
    wanted = [s["q"], s["k"]] + ([s["q_scale"], s["k_scale"]] if case["norm"] else [])
    grads = torch.autograd.grad(out, wanted, [s["gq"], s["gk"]])
    return {"out": [o.detach() for o in out], "grad": list(grads[:2]), "grad_scale": list(grads[2:])}


def _own_logprobs(s):
    from torchtune_amd.modules import layer_ops

    case = s["case"]
    r = layer_ops.token_logprobs(s["logits"], s["tokens"], temperature=case["temperature"], entropy=case["entropy"], top=case["top"])
    out = {"logprobs": r.logprobs.detach()}
    if case["entropy"]:
        out["entropy"] = r.entropy.detach()
    if case["top"]:
        out["top_logprobs"], out["top_tokens"] = r.top_logprobs, r.top_tokens
    if case["train"]:
        outs, gs = [r.logprobs], [s["g_logprobs"]]
        if case["entropy"]:
            outs.append(r.entropy)
            gs.append(s["g_entropy"])
        (out["grad"],) = torch.autograd.grad(outs, s["logits"], gs)
    return out


def _own_adamw(s):
    s["optimizer"].step()
    exp_avg, exp_avg_sq = s["optimizer"].moments()
    return {"params": s["whole"], "exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq}


# ---------------------------------------------------------------------------------------------------
# what the measurement calls
# ---------------------------------------------------------------------------------------------------
def _table(dim):
    theta = 500000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = torch.outer(torch.arange(_TABLE, device="cuda", dtype=torch.float64), theta)
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _positions(case, g):
    """Of packed documents, generation at a far place, or images among text."""
    b, s = case["batch"], case["seq"]
    if not case["given"]:
        return None
    start = torch.randint(0, _TABLE - s, (b, 1), generator=g, device="cuda")
    place = start + torch.arange(s, device="cuda")
    if case["axes"] == 1:
        return place
    width = max(1, int(math.sqrt(s)))
    inside = torch.arange(s, device="cuda") % (width * width)
    image = (torch.arange(s, device="cuda") // (width * width)).expand(b, s)
    return torch.stack([start + image, start + inside // width, start + inside % width])


def _prepare_rotate(case, g):
    b, s, nh, kv, d, t = case["batch"], case["seq"], case["heads"], case["kv"], case["dim"], _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["joined"]:
        whole = (normal(b, s, nh + kv, d) * 1.5).to(t)
        q, k = whole[:, :, :nh], whole[:, :, nh:]
    else:
        q, k = (normal(b, s, nh, d) * 1.5).to(t), (normal(b, s, kv, d) * 1.5).to(t)
    state = {"case": case, "eps": 1e-6, "q": q, "k": k, "q_scale": None, "k_scale": None, "gq": None, "gk": None,
             "cache": _table(d), "positions": _positions(case, g), "sections": _sections(case) if case["axes"] > 1 else None}
    if case["norm"]:
        state["q_scale"], state["k_scale"] = (normal(d) * 0.3 + 1).to(t), (normal(d) * 0.3 + 1).to(t)
    if case["train"]:
        state["gq"], state["gk"] = normal(b, s, nh, d).to(t), normal(b, s, kv, d).to(t)
        for name in ("q", "k", "q_scale", "k_scale"):
            if state[name] is not None:
                state[name] = state[name].detach().requires_grad_()
    return state


def _prepare_logprobs(case, g):
    rows, vocab, t = case["rows"], case["vocab"], _TYPES[case["dtype"]]
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
    # a few tokens stand out in each row, by more where the model is sure
    several = min(8, vocab)
    peaks = torch.randint(0, vocab, (rows, several), generator=g, device="cuda")
    logits.scatter_add_(1, peaks, torch.rand(rows, 1, generator=g, device="cuda") * 14 * torch.rand(rows, several, generator=g, device="cuda"))
    shape = (rows,) if case["tokens"] == 1 else (rows, case["tokens"])
    tokens = torch.randint(0, vocab, (rows, case["tokens"]), generator=g, device="cuda")
    frequent = torch.rand(rows, case["tokens"], generator=g, device="cuda") < 0.8
    tokens = torch.where(frequent, peaks[:, torch.arange(case["tokens"], device="cuda") % several], tokens)
    if case["masked"]:
        ruled_out = torch.rand(vocab, generator=g, device="cuda") < 0.3
        ruled_out[tokens[0, 0]] = False
        logits.masked_fill_(ruled_out, -math.inf)
        tokens = torch.where(ruled_out[tokens], tokens[0, 0], tokens)
    if rows > 1:  # padding
        tokens[torch.rand(rows, generator=g, device="cuda") < 0.1] = _IGNORED
    state = {"case": case, "logits": logits.to(t), "tokens": tokens.view(shape)}
    if case["train"]:
        state["logits"].requires_grad_()
        state["g_logprobs"] = torch.randn(shape, generator=g, device="cuda")
        state["g_entropy"] = torch.randn(rows, generator=g, device="cuda") * 0.1
    return state


def _prepare_adamw(case, g):
    t, eight = _TYPES[case["dtype"]], case["bits"] == 8
    state = {"case": case, "step": _STEPS, "params": [], "grads": [], "m": [], "v": [], "m_exponent": [], "v_exponent": []}
    half = torch.full((), 1 << 15, dtype=torch.int64, device="cuda")
    # the parameters lie one after another in one piece of memory, at odd places where sizes are odd
    sizes = _sizes(case)
    state["whole"] = torch.empty(sum(sizes), dtype=t, device="cuda")
    if not eight:
        state["m_whole"], state["v_whole"] = torch.empty(2, sum(sizes), device="cuda")
    for i, (n, part) in enumerate(zip(sizes, state["whole"].split(sizes))):
        part.copy_(torch.randn(n, generator=g, device="cuda") * 0.02)
        p = torch.nn.Parameter(part)
        # rows of a weight meet gradients of very different sizes
        size = torch.exp(torch.randn(-(-n // 512), generator=g, device="cuda") * 1.5 - 9).repeat_interleave(512)[:n]
        p.grad = (torch.randn(n, generator=g, device="cuda") * size).to(t)
        m = torch.randn(n, generator=g, device="cuda") * size * 0.3
        v = size * size * torch.rand(n, generator=g, device="cuda") * 0.2
        state["params"].append(p)
        state["grads"].append(p.grad)
        for name, x, mantissa in (("m", m, 3), ("v", v, 4)):
            if eight:
                x, exponent = _hold(x, half, mantissa)
                state[f"{name}_exponent"].append(exponent)
                state[name].append(x)
            else:
                state[name].append(state[f"{name}_whole"].split(sizes)[i].copy_(x))
    if own:
        _own_optimizer(state)
    return state


def _own_optimizer(s):
    from torchtune_amd.training import AdamW

    case = s["case"]
    opt = AdamW(s["params"], lr=_LR, betas=_BETAS, eps=_EPS, weight_decay=_DECAY, state_bits=case["bits"],
                stochastic_rounding=case["stochastic"], seed=_SEED)
    saved = opt.state_dict()
    saved["state"] = {}
    for i in range(len(s["params"])):
        saved["state"][i] = {"step": s["step"], "exp_avg": s["m"][i], "exp_avg_sq": s["v"][i]}
        if case["bits"] == 8:
            saved["state"][i].update(exp_avg_exponent=s["m_exponent"][i], exp_avg_sq_exponent=s["v_exponent"][i])
    opt.load_state_dict(saved)
    s["optimizer"] = opt


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"rotate": _prepare_rotate, "logprobs": _prepare_logprobs, "adamw": _prepare_adamw}[case["kind"]](case, g)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotate": _own_rotate, "logprobs": _own_logprobs, "adamw": _own_adamw}[kind](state)
    with torch.no_grad():
        return {"rotate": _plain_rotate, "logprobs": _plain_logprobs, "adamw": _plain_adamw}[kind](state)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "rotate":
        tokens, d = case["batch"] * case["seq"], case["dim"]
        n = tokens * (case["heads"] + case["kv"]) * d
        angles = (min(case["seq"], tokens) if not case["given"] else tokens) * d * 4
        # heads in and out, and with the backward pass their gradients out and in
        return {"bytes": n * size * (4 if case["train"] else 2) + angles + (8 * tokens * case["axes"] if case["given"] else 0),
                "flops": n * (3 + 4 * case["norm"]) * (3 if case["train"] else 1)}
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        results = case["rows"] * (12 * case["tokens"] + 4 * case["entropy"] + 12 * case["top"])
        return {"bytes": n * size * (2 if case["train"] else 1) + results * (2 if case["train"] else 1),
                "flops": n * (4 + 2 * case["entropy"]) * (2 if case["train"] else 1)}
    n = sum(_sizes(case))
    # parameter and moments in and out, gradient in; what is held in 8 bits is read out as numbers of 16 as well
    moments = 2 * 2 * 4 if case["bits"] == 32 else 2 * 2 * (1 + 1 / _BLOCK) + 2 * 2
    return {"bytes": n * (3 * size + moments), "flops": 15 * n}


# ---------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definition
# ---------------------------------------------------------------------------------------------------
def _exact_rotate(s):
    case = s["case"]
    b, n, d = case["batch"], case["seq"], case["dim"]
    axis = [0] * (d // 2)
    if s["sections"] is not None:
        axis = [a for a, count in enumerate(s["sections"]) for _ in range(count)]
    pos = s["positions"] if s["positions"] is not None else torch.arange(n, device="cuda").repeat(b, 1)
    pos = pos if pos.dim() == 3 else pos[None]
    # every pair as a complex number, and its turn as one
    turn = torch.stack([torch.complex(*(s["cache"][pos[axis[i]], i, part].double() for part in (0, 1))) for i in range(d // 2)], -1)[:, :, None]
    first = torch.arange(d // 2, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else d // 2)

    def turned(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        out = torch.empty_like(x)
        out[..., first], out[..., second] = z.real, z.imag
        return out

    out, grads, scales = [], [], []
    for x, w, gy in ((s["q"], s["q_scale"], s["gq"]), (s["k"], s["k_scale"], s["gk"])):
        x = x.detach().double()
        weight = torch.ones(d, dtype=torch.float64, device="cuda") if w is None else w.detach().double()
        length = torch.ones_like(x[..., :1]) if w is None else torch.sqrt((x * x).sum(-1, keepdim=True) / d + s["eps"])
        unit = x / length
        out.append(turned(unit * weight, turn))
        if case["train"]:
            g = turned(gy.double(), turn.conj())
            if w is None:
                grads.append(g)
                continue
            scales.append(torch.einsum("bshd,bshd->d", g, unit))
            along = (g * weight * unit).sum(-1, keepdim=True) / d
            grads.append((g * weight - unit * along) / length)
    return {"out": out, "grad": grads, "grad_scale": scales} if case["train"] else {"out": out}


def _exact_logprobs(s):
    case, rows = s["case"], s["case"]["rows"]
    tokens = s["tokens"].reshape(rows, -1)
    parts = {"logprobs": [], "entropy": [], "top_logprobs": [], "top_tokens": [], "grad": []}
    for lo in range(0, rows, 256):
        z = s["logits"][lo:lo + 256].detach().double() / case["temperature"]
        log_p = z - torch.logsumexp(z, -1, keepdim=True)
        p = log_p.exp()
        at = tokens[lo:lo + 256]
        valid = (at >= 0).double()
        parts["logprobs"].append(log_p.gather(1, at.clamp(min=0)).masked_fill(at < 0, 0.0))
        surprise = (-log_p).masked_fill(p == 0, 0.0)
        entropy = (p * surprise).sum(-1)
        parts["entropy"].append(entropy)
        if case["top"]:
            # logits are few distinct numbers: ranks by (value, then place)
            found = torch.sort(s["logits"][lo:lo + 256].detach().double(), dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            parts["top_tokens"].append(found)
            parts["top_logprobs"].append(log_p.gather(1, found))
        if case["train"]:
            g = s["g_logprobs"].reshape(rows, -1)[lo:lo + 256].double() * valid
            grad = torch.zeros_like(p).scatter_add_(1, at.clamp(min=0), g) - p * g.sum(-1, keepdim=True)
            if case["entropy"]:
                grad = grad + s["g_entropy"][lo:lo + 256, None].double() * p * (surprise - entropy[:, None])
            parts["grad"].append(grad / case["temperature"])
    whole = {name: torch.cat(part) for name, part in parts.items() if part}
    out = {"logprobs": whole["logprobs"].view(s["tokens"].shape)}
    if case["entropy"]:
        out["entropy"] = whole["entropy"]
    for name in ("top_logprobs", "top_tokens", "grad"):
        if name in whole:
            out[name] = whole[name]
    return out


def _exact_value(code, exponent, signed):
    """64-bit values of held moments, from the fields of a code"""
    mantissa = 3 if signed else 4
    code = code.double()
    sign = torch.where(code >= 128, -1.0, 1.0) if signed else torch.ones_like(code)
    code = torch.remainder(code, 128) if signed else code
    step = 2.0 ** mantissa
    power = exponent.double().repeat_interleave(_BLOCK)[:code.numel()] - 127 - 15 + torch.floor(code / step)
    return sign * torch.where(code == 0, 0.0, (1 + torch.remainder(code, step) / step) * torch.exp2(power))


def _exact_adamw(s):
    eight, t = s["case"]["bits"] == 8, _STEPS + 1
    (b1, b2) = _BETAS
    out = {"params": [], "exp_avg": [], "exp_avg_sq": []}
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        p, g, m, v = p.detach().double(), g.double(), s["m"][i], s["v"][i]
        if eight:
            m, v = _exact_value(m, s["m_exponent"][i], True), _exact_value(v, s["v_exponent"][i], False)
        m = b1 * m.double() + (1 - b1) * g
        v = b2 * v.double() + (1 - b2) * g ** 2
        corrected = torch.sqrt(v / (1 - b2 ** t)) + _EPS
        out["params"].append(p - _LR * _DECAY * p - _LR * (m / (1 - b1 ** t)) / corrected)
        out["exp_avg"].append(m)
        out["exp_avg_sq"].append(v)
    out = {name: torch.cat(parts) for name, parts in out.items()}
    if eight:
        # which way a moment of 32 bits is rounded to 8 is not for one of 64 to say
        out["exp_avg"] = out["exp_avg_sq"] = None
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotate": _exact_rotate, "logprobs": _exact_logprobs, "adamw": _exact_adamw}[case["kind"]](s)

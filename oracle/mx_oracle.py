"""CPU restatement of the microscaled formats and of the products over them, in 64 bits (test infrastructure).

A block is 32 consecutive elements of the last dimension; its scale is 2^e, e = max(floor(log2(max |v|)) - emax, -127); the
elements are the format's numbers nearest to v / 2^e, ties to the even code, saturated."""
import torch

BLOCK = 32
EMAX = {"mxfp4": 2, "mxfp8": 8}
FP4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def fp8_table() -> torch.Tensor:
    """The 127 finite magnitudes of e4m3, by code."""
    c = torch.arange(127, dtype=torch.float64)
    e, m = torch.floor(c / 8), torch.remainder(c, 8)
    return torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e - 7))


def table(fmt: str) -> torch.Tensor:
    return FP4 if fmt == "mxfp4" else fp8_table()


def quantize(x: torch.Tensor, fmt: str):
    """(codes uint8, one per element, scales uint8 [..., K / 32])"""
    b = x.detach().cpu().double().unflatten(-1, (-1, BLOCK))
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b)
    amax = b.abs().amax(-1)
    # frexp gives a mantissa in [0.5, 1)
    e = torch.where(amax > 0, torch.frexp(amax).exponent.double() - 1 - EMAX[fmt], torch.full_like(amax, -127.0)).clamp(min=-127)
    grid = table(fmt)
    size = b.abs() * torch.exp2(-e).unsqueeze(-1)
    hi = torch.searchsorted(grid, size.contiguous()).clamp(max=len(grid) - 1)  # first number >= size
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - size, size - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)) | (size >= grid[-1]), hi, lo)
    sign = torch.signbit(b).long() << (3 if fmt == "mxfp4" else 7)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code + sign)
    scale = torch.where(bad, torch.full_like(e, 255.0), e + 127)
    return code.flatten(-2).to(torch.uint8), scale.to(torch.uint8)


def pack(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    """Codes as a tensor holds them: mxfp4 two to a byte, the earlier element in the low half."""
    if fmt == "mxfp8":
        return codes
    p = codes.unflatten(-1, (-1, 2))
    return p[..., 0] | (p[..., 1] << 4)


def unpack(packed: torch.Tensor, fmt: str) -> torch.Tensor:
    return packed if fmt == "mxfp8" else torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def values(codes: torch.Tensor, scales: torch.Tensor, fmt: str) -> torch.Tensor:
    """float64 values of unpacked codes"""
    top = 8 if fmt == "mxfp4" else 128
    grid = table(fmt)
    if fmt == "mxfp8":
        grid = torch.cat([grid, torch.tensor([float("nan")], dtype=torch.float64)])
    v = grid[(codes % top).long()] * torch.where(codes >= top, -1.0, 1.0)
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (v.unflatten(-1, (-1, BLOCK)) * s.unsqueeze(-1)).flatten(-2)


def nearest(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """x replaced by the values its blocks hold, float64"""
    return values(*quantize(x, fmt), fmt)


def lora(x, weights, lora_a, lora_b, factors, gys):
    """(ys, gx, gas, gbs) in float64 of adapter linears over dense float64 weights; x already quantised"""
    ys, gas, gbs, gx = [], [], [], 0.0
    for w, a, b, s, gy in zip(weights, lora_a, lora_b, factors, gys):
        a, b, gy = a.double(), b.double(), gy.double()
        h = x @ a.T
        ys.append(x @ w.T + s * (h @ b.T))
        gh = s * (gy @ b)
        gx = gx + gy @ w + gh @ a
        gas.append(gh.T @ x)
        gbs.append(s * (gy.T @ h))
    return ys, gx, gas, gbs

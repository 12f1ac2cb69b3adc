"""Microscaled formats in 64 bits, for the tests: what elements stand for, and the quantiser's definition."""
import torch

FP4, FP8, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn, torch.float8_e8m0fnu
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
TOP = {FP4: 2, FP8: 8}            # exponents of the highest binades
LARGEST = {FP4: 6.0, FP8: 448.0}
LOWEST = {FP4: (0, 1), FP8: (-6, 3)}   # the lowest binade of normal numbers, bits behind the point


def blocks(extent, block=32):
    return -(-extent // block)


def width(dtype, k):
    """Extent of a row of k elements."""
    return k // 2 if dtype == FP4 else k


def elements(q):
    """The numbers that elements stand for before their scale, on the CPU."""
    if q.dtype == torch.int8:
        return q.cpu().double()
    if q.dtype == FP8:
        return q.cpu().double()
    pairs = q.cpu().view(torch.uint8).long()
    codes = torch.stack([pairs & 15, pairs >> 4], dim=-1).flatten(-2)
    return E2M1[codes & 7] * torch.where(codes >= 8, -1.0, 1.0).double()


def spread(scales, k, block=32):
    """Scales (e8m0 or fp32) as 64-bit numbers, one an element."""
    return scales.cpu().double().repeat_interleave(block, dim=-1)[..., :k]


def values(q, scales):
    e = elements(q)
    return e * spread(scales, e.shape[-1])


def nearest(y, dtype):
    """The element type's number nearest to y, ties to even, past the largest number that."""
    low, bits = LOWEST[dtype]
    exponent = torch.frexp(y.abs()).exponent - 1
    step = torch.exp2((exponent.clamp(min=low) - bits).double())
    return (torch.round(y / step) * step).clamp(-LARGEST[dtype], LARGEST[dtype])


def block_most(x, block=32):
    return torch.stack([part.abs().amax(dim=-1) for part in x.split(block, dim=-1)], dim=-1)


def scale_bytes(most, dtype):
    """The scales of blocks whose largest numbers are `most` (64 bits, finite)."""
    exponent = torch.where(most == 0, -1000, torch.frexp(most).exponent - 1 - TOP[dtype])
    return (exponent.clamp(min=-127) + 127).to(torch.uint8)


def quantized(x, dtype):
    """(numbers of the elements, bytes of the scales) of x [.., K] by the definition."""
    x = x.double().cpu()
    most = block_most(x)
    odd = ~torch.isfinite(most)
    bytes_ = scale_bytes(torch.where(odd, 0.0, most), dtype)
    wide = torch.exp2(bytes_.double() - 127).repeat_interleave(32, dim=-1)[..., :x.shape[-1]]
    q = nearest(torch.where(odd.repeat_interleave(32, dim=-1)[..., :x.shape[-1]], 0.0, x) / wide, dtype)
    return q, torch.where(odd, 255, bytes_).to(torch.uint8)


def room(lead, k, dtype, scale_dtype=E8M0, block=32, device="cuda", fill=0xA5):
    """(q, scales) for results of shape [*lead, k], filled with a pattern."""
    q = torch.full((*lead, width(dtype, k)), fill, dtype=torch.uint8, device=device).view(dtype)
    scales = torch.full((*lead, blocks(k, block)), 0x7B, dtype=torch.uint8, device=device).view(E8M0) if scale_dtype == E8M0 else \
        torch.full((*lead, blocks(k, block)), -1.0, device=device)
    return q, scales


def operands(rows, k, dtype, batch=(), seed=0, low=110, high=140):
    """Random elements (every finite number of the type) and scales, on the CPU."""
    g = torch.Generator().manual_seed(seed + rows * 31 + k)
    q = torch.randint(0, 256, (*batch, rows, width(dtype, k)), generator=g, dtype=torch.int64).to(torch.uint8)
    if dtype == FP8:
        q[(q & 0x7f) == 0x7f] = 0x38
    scales = torch.randint(low, high, (*batch, rows, blocks(k)), generator=g, dtype=torch.int64).to(torch.uint8)
    return q.view(dtype), scales.view(E8M0)

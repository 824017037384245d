"""The 8-bit block format in float64, written from its definition (include/hcmoco_hip.h): used by the tests of the operators
that read or write it."""
import torch


def _two(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _floor_log2(v):
    return torch.frexp(v)[1] - 1


def block_exponent(top):
    """Smallest E >= -126 with top <= 448 * 2^E (0 for top = 0), by trying the two candidates."""
    e = _floor_log2(torch.where(top > 0, top, torch.ones_like(top))) - 9
    for _ in range(2):
        e = torch.where(top > 448 * _two(e), e + 1, e)
    return torch.where(top > 0, e.clamp(min=-126), torch.zeros_like(e))


def e4m3(v):
    """Nearest e4m3 value, ties to even: 4 significant bits from 2^-6 up, multiples of 2^-9 below; not finite -> NaN."""
    step = _two((_floor_log2(torch.where((v != 0) & v.isfinite(), v.abs(), torch.ones_like(v))) - 3).clamp(min=-9))
    return torch.where(v.isfinite(), torch.round(v / step) * step, torch.full_like(v, float('nan')))


def held8(x, tall=1):
    """(values, exponents) of x [rows, cols] held in blocks of ``tall`` x 128."""
    x = x.detach().double().cpu()
    rows, cols = x.shape
    kb, rb = (cols + 127) // 128, (rows + tall - 1) // tall
    p = torch.zeros(rb * tall, kb * 128, dtype=torch.float64)
    p[:rows, :cols] = x
    p = p.view(rb, tall, kb, 128)
    top = torch.where(p.isfinite(), p.abs(), torch.zeros_like(p)).amax(dim=(1, 3), keepdim=True)
    e = block_exponent(top)
    val = e4m3(p * _two(-e)) * _two(e)
    return val.reshape(rb * tall, kb * 128)[:rows, :cols], e.reshape(rb, kb)

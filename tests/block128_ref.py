"""Plain 64-bit forms of the block-scaled FP8 operators, for the tests."""
import torch

E4M3 = torch.float8_e4m3fn


def blocks(n):
    return (n + 127) // 128


def e4m3_step(v):
    """Distance between neighbouring e4m3 values around v (64 bits): 2^(e-3) in [2^e, 2^(e+1)), 2^-9 below 2^-6."""
    _, ex = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), (ex - 1).clamp(min=-6) - 3)


def e4m3_of(v):
    step = e4m3_step(v)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def cast(x, group):
    """(codes before rounding, top) of 64-bit rows: 448 x / top for each `group` values."""
    rows, k = x.shape
    u = torch.empty_like(x)
    top = torch.empty((rows, (k + group - 1) // group), dtype=torch.float64, device=x.device)
    for j in range(top.shape[1]):
        part = x[:, j * group:(j + 1) * group]
        top[:, j] = part.abs().amax(1).clamp(min=float(torch.tensor(1e-4)))
        u[:, j * group:(j + 1) * group] = part * 448.0 / top[:, j:j + 1]
    return u, top


def random_operand(g, *shape):
    return (torch.randn(shape, generator=g) * 112.0).clamp(-448, 448).to(E4M3)


def random_scales(g, *shape):
    return torch.exp(0.5 * torch.randn(shape, generator=g)) * 0.01


def by_row(q, sf):
    return q.double() * sf.double().repeat_interleave(128, -1)[..., :q.shape[-1]]


def by_block(q, sf):
    return q.double() * sf.double().repeat_interleave(128, -2)[..., :q.shape[-2], :].repeat_interleave(128, -1)[..., :q.shape[-1]]


def product_and_bound(a, b):
    """64-bit product of 64-bit values and how far 32-bit sums may be from it.  A block of 128 products is summed by four MMAs of 32 each,
    in an order and with alignment of the hardware's choosing: each of the 128 additions may be off by a unit of the last place,
    2^-23, of a partial sum that is at most the sum of magnitudes.  Then one addition per block, and the multiplications by the scales."""
    kb = blocks(a.shape[-1])
    return a @ b.transpose(-1, -2), (128 + kb + 4) * 2.0 ** -23 * (a.abs() @ b.abs().transpose(-1, -2))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2

"""Plain 64-bit statements of the 8-bit block format, RMSNorm and the many-tensor AdamW with 8-bit moments (test infrastructure)."""
import torch

BLK = 128


def _pow2(e):
    return torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())


def block_exponent(amax):
    """Smallest e >= -127 with amax <= 448 * 2^e (amax finite, 64 bits)."""
    frac, e = torch.frexp(amax.double() / 448.0)
    return torch.where(frac == 0.5, e - 1, e).where(amax > 0, torch.full_like(e, -127)).clamp(min=-127)


def round_e4m3(z):
    """Nearest e4m3 value, ties to even; |z| <= 464."""
    step = _pow2(torch.frexp(z)[1].clamp(min=-5) - 4)
    return torch.round(z / step) * step


def quantize(x, square=False):
    """[R, C] -> (values as stored, exponents [R, blocks]) in 64 bits; non-finite values become NaN and do not enter the scale."""
    R, C = x.shape
    Cp = (C + BLK - 1) // BLK * BLK
    xp = torch.nn.functional.pad(x.double(), (0, Cp - C)).view(R, Cp // BLK, BLK)
    amax = torch.where(torch.isfinite(xp), xp.abs(), torch.zeros_like(xp)).amax(-1)
    if square:
        for r in range(0, R, BLK):
            amax[r:r + BLK] = amax[r:r + BLK].amax(0, keepdim=True)
    e = block_exponent(amax)
    v = round_e4m3(xp * _pow2(-e)[..., None]) * _pow2(e)[..., None]
    v = torch.where(torch.isfinite(xp), v, torch.full_like(v, float("nan")))
    return v.view(R, Cp)[:, :C], e


def decode(data, scale, K):
    """Codes and scale bytes (uint8, CPU) -> 64-bit values [rows, K]."""
    v = data.view(torch.float8_e4m3fn).float().double()
    e = scale.to(torch.int64).repeat_interleave(BLK, 1)[:, :v.shape[1]] - 127
    return (v * _pow2(e))[:, :K]


def rmsnorm(x, gamma, eps, dy=None, dh=None):
    """y [, dx, dgamma] of 64-bit rows."""
    x, gamma = x.double(), gamma.double()
    n = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y = x * n * gamma
    if dy is None:
        return y, n[:, 0]
    u = dy.double() * gamma
    dx = n * u - x * n ** 3 * (u * x).mean(-1, keepdim=True)
    return y, n[:, 0], dx if dh is None else dx + dh.double(), (dy.double() * x * n).sum(0)


def adamw(p, g, m, v, t, lr, betas, eps, wd):
    b1, b2 = betas
    p, g, m, v = (a.double() for a in (p, g, m, v))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p, m, v


def mix32(x):
    """Two multiply-xorshift rounds; shifts and factors from Chris Wellons' published search for 32-bit integer hashes of low bias (2018)."""
    low = 0xFFFFFFFF

    def mul(a, k):                                   # 32 x 32 -> low 32 bits without leaving 63
        return ((((a >> 16) * k) & 0xFFFF) << 16) + ((a & 0xFFFF) * k) & low
    x = mul((x ^ (x >> 16)) & low, 0x7FEB352D)
    x = mul(x ^ (x >> 15), 0x846CA68B)
    return x ^ (x >> 16)


def rounding_bits(index, seed, step):
    """The 32 random bits of element `index` (int64 tensor): low half rounds m, high half v."""
    key = mix32(torch.tensor(seed) ^ mix32(torch.tensor((step + 0x9E3779B9) & 0xFFFFFFFF)))
    return mix32((index & 0xFFFFFFFF) ^ key)


def _stochastic(z, lowest, bits):
    """z >= 0 rounded to 3 bits behind the leading one (steps of 2^(lowest - 3) below 2^lowest), up where frac + bits / 2^16 reaches 1
    -> (value, distance of that sum to the border, step)."""
    step = _pow2((torch.frexp(z)[1] - 1).clamp(min=lowest) - 3)
    pos = z / step
    s = pos - pos.floor() + bits.double() / 65536.0
    return (pos.floor() + (s >= 1.0).double()) * step, (s - 1.0).abs(), step


def store_m(m, bits):
    """First moments in blocks of 128 (last dim): (stored values, distance to the rounding border in steps, the step)."""
    e = block_exponent(m.abs().amax(-1, keepdim=True))
    q, d, s = _stochastic(m.double().abs() * _pow2(-e), -6, bits & 0xFFFF)
    return torch.sign(m.double()) * q * _pow2(e), d, s * _pow2(e)


def store_v(v, bits):
    """Second moments: 5 exponent and 3 mantissa bits; the scale is the smallest 2^e (e >= 0) under which the largest value's exponent
    field is at most 31 with a mantissa of at most 1.75; a positive value is never stored as 0."""
    frac, e = torch.frexp(v.double().amax(-1, keepdim=True) / 1.75)
    e = (torch.where(frac == 0.5, e - 1, e).clamp(min=-126) + 127 - 31).clamp(min=0)
    q, d, s = _stochastic(v.double() * _pow2(-e), -126, bits >> 16)
    q = torch.where(v > 0, q.clamp(min=2.0 ** -129), q)
    return q * _pow2(e), d, s * _pow2(e)

"""The stochastic rounding of 8-bit moments over many elements: codes differ from the 64-bit statement only where the deciding sum lies within the
arithmetic's own error of its border.

The sum is (value / step) + random / 2^16 against the next whole number.  In fp32 m is off by at most 3 * 2^-24 of its terms |b1 m0| + |(1 - b1) g|
and (b1 and 1 - b1 rounded to fp32) by another 2^-24 of each, v by at most 2^-22 of itself in all; 2^-22 of the terms covers both.  Lining the value up
with the code's exponent field is exact, but for the smallest codes, where fp32's subnormals round at 2^-21 of a step.  So a code is sure
outside 2^-22 terms / step + 2^-20 of the border; a random sum lies inside with a probability of twice that."""
import pytest
import torch

from oracle import blocks8 as ob

pytestmark = pytest.mark.gpu
H = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
N = 1 << 20


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from spn4cir_amd import ops as o
    return o


def test_codes_flip_only_at_their_border(ops):
    g = torch.Generator().manual_seed(0)
    p = (torch.randn(N, generator=g) * 0.05).cuda()
    plan = ops.AdamWPlan([p], state_bits=8)
    size = 10.0 ** (torch.rand(N // 128, 1, generator=g) * 3 - 5)
    for t in range(1, 5):
        grad = (torch.randn(N // 128, 128, generator=g) * size).view(-1)
        m0, v0 = (x.cpu().double() for x in plan.moments())
        ops.adamw_multi(plan, [grad.cuda()], t, H, seed=11)
        m1, v1 = (x.cpu().double().view(-1, 128) for x in plan.moments())
        _, rm, rv = ob.adamw(torch.zeros(N), grad, m0, v0, t, H["lr"], H["betas"], H["eps"], H["weight_decay"])
        bits = ob.rounding_bits(torch.arange(N), 11, t).view(-1, 128)
        terms = H["betas"][0] * m0.abs() + (1 - H["betas"][0]) * grad.double().abs()
        for name, got, ref, mag, store in (("m", m1, rm, terms, ob.store_m), ("v", v1, rv, rv, ob.store_v)):
            ref, mag = ref.view(-1, 128), mag.view(-1, 128)
            want, dist, unit = store(ref, bits)
            # blocks whose largest magnitude is not within its own error of the border between two scales
            top = ref.abs().amax(-1, keepdim=True)
            slack = 2.0 ** -22 * mag.amax(-1, keepdim=True) / top
            # (the step of a zero in the same block is that of the smallest codes: the scale)
            scale = [store(torch.cat([top * (1 + s * slack), torch.zeros_like(top)], 1), torch.zeros(1, dtype=torch.int64))[2][:, 1:] for s in (-1, 1)]
            one_scale = (scale[0] == scale[1]).expand_as(ref)
            near = 2.0 ** -22 * mag / unit + 2.0 ** -20
            flipped = (got != want) & one_scale
            assert not (flipped & (dist > near)).any(), (name, t, int((flipped & (dist > near)).sum()))
            expected = (2 * near.clamp(max=0.5) * one_scale).sum().item()
            assert int(flipped.sum()) <= expected + 6 * expected ** 0.5 + 6
            assert one_scale.double().mean() > 0.999


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-8])
def test_second_moments_below_the_smallest_normal_number(ops, eps):
    """Gradients of 1e-21 to 1e-17: v is subnormal, the step is lr * m / (sqrt(v) + eps) all the same, as with 32-bit moments.  v is off by at most 1.5 of
    fp32's smallest step (two roundings of its terms), its root by half of that share, the rest by the few-ulp instructions."""
    g = torch.Generator().manual_seed(1)
    grad = torch.randn(4096, generator=g).sign() * 10.0 ** (torch.rand(4096, generator=g) * 4 - 21)
    p0 = torch.randn(4096, generator=g)
    h = dict(lr=1e-2, betas=(0.9, 0.999), eps=eps, weight_decay=0.0)
    for bits in (8, 32):
        p = p0.cuda()
        ops.adamw_multi(ops.AdamWPlan([p], state_bits=bits), [grad.cuda()], 1, h)
        zero = torch.zeros(4096)
        ref, m, v = ob.adamw(p0, grad, zero, zero, 1, h["lr"], h["betas"], eps, 0.0)
        share = 1.5 * 2.0 ** -149 / v                               # of v; where it is not small nothing is left of v's value
        sure = share < 0.25
        assert sure.double().mean() > 0.5 and (v < 2.0 ** -126).double().mean() > 0.3 and torch.isfinite(p.cpu()[sure]).all()
        update = (ref - p0.double()).abs()
        off = (p.cpu().double() - ref).abs()
        assert (off <= update * (share + 2.0 ** -19) + 2.0 ** -22 * p0.double().abs())[sure].all(), bits

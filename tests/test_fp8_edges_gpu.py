"""8-bit blocks at the edges: batches without rows, padding behind a row of NaN, the ends of the number range."""
import pytest
import torch

from oracle import blocks8 as ob
from test_fp8_gpu import product, rnd, same, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from spn4cir_amd import ops as o
    return o


@pytest.mark.parametrize("form", ["numbers", "blocks"])
def test_linear_of_an_empty_batch(ops, form):
    """No rows: empty outputs, zero gradients of weight and bias (added to what is there with accumulate), in training and in serving."""
    w8, w8_t = ops.quantize_fp8(rnd((130, 200), 1).cuda(), block_rows=128, want="both")
    bias = rnd((130,), 2).cuda()
    x = torch.zeros(0, 200, dtype=torch.bfloat16, device="cuda")
    if form == "blocks":
        x = ops.rmsnorm_fwd(x, torch.ones(200, device="cuda"), out_dtype="fp8")[0]
    y, none = ops.linear_fp8_fwd(x, w8, bias)
    assert none is None and y.shape == (0, 130) and y.dtype == torch.bfloat16
    y, saved = ops.linear_fp8_fwd(x, w8, bias, w8_t=w8_t, out_dtype=torch.float32)
    assert y.shape == (0, 130) and y.dtype == torch.float32
    dy = torch.zeros(0, 130, device="cuda")
    dx, dw, db = ops.linear_fp8_bwd(saved, dy, dx_dtype=torch.float16, dw_dtype=torch.bfloat16)
    assert dx.shape == (0, 200) and dx.dtype == torch.float16
    assert dw.shape == (130, 200) and dw.dtype == torch.bfloat16 and not dw.any() and db.shape == (130,) and not db.any()
    into = torch.full((130, 207), 3.0, device="cuda")
    assert ops.linear_fp8_bwd(saved, dy, dw=into[:, :200], accumulate=True)[1].data_ptr() == into.data_ptr() and bool((into == 3.0).all())
    ops.linear_fp8_bwd(saved, dy, dw=into[:, :200])
    assert not into[:, :200].any() and bool((into[:, 200:] == 3.0).all())
    assert ops.linear_fp8_fwd(x, w8, w8_t=w8_t)[1]["bias"] is False
    for bad in (dict(dw=torch.zeros(130, 199, device="cuda")), dict(accumulate=True), dict(dw_dtype=torch.int32),
                dict(dw=torch.zeros(130, 200, dtype=torch.float16, device="cuda"), accumulate=True)):
        with pytest.raises(ValueError):
            ops.linear_fp8_bwd(saved, dy, **bad)
    with pytest.raises(ValueError):
        ops.linear_fp8_bwd(saved, torch.zeros(0, 131, device="cuda"))


def test_quantize_without_rows(ops):
    x = torch.zeros(0, 300, device="cuda")
    q, cs = ops.quantize_fp8(x, colsum=True)
    assert q.shape == (0, 300) and cs.shape == (300,) and not cs.any() and ops.quantize_fp8(q, block_rows=128).shape == (0, 300)
    for bad in (dict(want="cols"), dict(want="both")):
        with pytest.raises(ValueError, match="no rows"):
            ops.quantize_fp8(x, **bad)
    with pytest.raises(ValueError, match="no columns"):
        ops.quantize_fp8(torch.zeros(3, 0, device="cuda"))


@pytest.mark.parametrize("W", [1, 7, 120, 300, 520, 1001, 2056, 4100])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_codes_behind_a_row_of_nan_are_zero(ops, W, eps):
    """rstd of a row is NaN (a NaN in it) or infinite (all zeros, eps = 0): the row's values are NaN, the codes behind them zero all the same."""
    x = rnd((5, W), W)
    x[1, W // 2] = float("nan")
    x[2] = 0
    x[3, 0] = float("inf")
    y, _, rstd = ops.rmsnorm_fwd(x.cuda(), torch.ones(W, device="cuda"), eps=eps, out_dtype="fp8")
    assert torch.isnan(rstd[1]) and (eps > 0 or torch.isinf(rstd[2]))
    assert not y.data[:, W:].any()
    assert bool((y.data[1, :W] & 0x7F == 0x7F).all()) and bool((y.data[2, :W] & 0x7F == (0x7F if eps == 0 else 0)).all())


def test_the_largest_and_smallest_numbers(ops):
    """From 248 * 2^120 on (half way between two codes, ties to even) a magnitude is stored as 2^128: an infinity as a number, like bf16's own
    rounding of it.  Scale bytes 0..2 reach below bf16's smallest number; fp32 holds all of it."""
    top = 2.0 ** 120
    x = torch.zeros(9, 128)
    x[0, :4] = torch.tensor([torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max, 1e38, 3.0])
    x[1, :3] = torch.tensor([248.0 * top, 248.0 * top * (1 - 2.0 ** -24), -240.0 * top])
    for b in range(4):                                               # largest magnitude 448 * 2^(b - 127): scale byte b; then down to the smallest code
        x[2 + b] = torch.arange(128).double().mul(2.0 ** (b - 136)).float()
        x[2 + b, 0] = 448.0 * 2.0 ** (b - 127)
    x[6, 5], x[7, 5] = 2.0 ** -149, 2.0 ** -137                      # under half of the smallest code: zero; half of it: zero (even)
    x[8] = torch.finfo(torch.float32).tiny
    q = ops.quantize_fp8(x.cuda())
    ref, e = ob.quantize(x)
    assert same(values(q), ref) and torch.equal(q.scale.cpu()[:, :1].long() - 127, e.long())
    assert ref[0, 0] == 2.0 ** 128 and ref[1, 0] == 2.0 ** 128 and ref[1, 1] == 240.0 * top and q.scale.cpu()[2:6, 0].tolist() == [0, 1, 2, 3]
    full = q.dequantize(torch.float32).cpu()
    assert torch.equal(full, ref.float()) and bool(torch.isinf(full[0, :2]).all()) and torch.equal(full[1:].double()[1:], ref[2:])
    assert torch.equal(q.dequantize(torch.bfloat16).cpu(), ref.float().to(torch.bfloat16))
    assert torch.equal(q.dequantize(torch.bfloat16).cpu()[5].double(), ref[5]) and not torch.equal(q.dequantize(torch.bfloat16).cpu()[2].double(), ref[2])


@pytest.mark.parametrize("M", [5, 40, 300])
def test_product_at_the_ends_of_the_scale(ops, M):
    """Scale bytes 0 to 4 of one operand against 236 to 247 of the other (in both orders): results of ordinary size, each kernel."""
    N, K = 260, 640
    g = torch.Generator().manual_seed(M)
    mant = lambda r: torch.randn(r, K, generator=g).double().clamp(-3, 3) / 3  # noqa: E731
    each = lambda r, lo, hi: torch.randint(lo, hi, (r, 5), generator=g).double().repeat_interleave(128, 1)  # noqa: E731
    low = (mant(M) * 2.0 ** (each(M, 0, 4) - 118)).float()           # block maxima near 2^(b - 118): scale bytes 0..4
    high = (mant(N) * 2.0 ** (each(N, 116, 124) + 1)).float()
    a8, b8 = ops.quantize_fp8(low.cuda()), ops.quantize_fp8(high.cuda())
    assert int(a8.scale.cpu()[:, :5].min()) == 0 and int(a8.scale.cpu()[:, :5].max()) <= 4 and int(b8.scale.cpu()[:, :5].max()) >= 240
    ref, err = product(values(a8), values(b8))
    for p, q, r in ((a8, b8, ref), (b8, a8, ref.t())):
        got = ops.gemm_nt_fp8(p, q, out_dtype=torch.float32).cpu().double()
        assert ((got - r).abs() <= (err if r is ref else err.t())).all()


@pytest.mark.parametrize("M,N,K", [(4, 260, 4096), (300, 520, 640)])
def test_full_fp32_sums_from_the_decoded_operands(ops, M, N, K):
    """What a caller does who needs more than the 8-bit unit's 14 to 16 bits: bf16 holds the operands exactly, so K fp32 additions are all that rounds."""
    a8, b8 = ops.quantize_fp8(rnd((M, K), 1).cuda()), ops.quantize_fp8(rnd((N, K), 2, scale=K ** -0.5).cuda(), block_rows=128)
    a, b = values(a8), values(b8)
    exact = ops.gemm_nt(a8.dequantize(), b8.dequantize(), out_dtype=torch.float32).cpu().double()
    assert ((exact - a @ b.t()).abs() <= (K + 2) * 2.0 ** -24 * (a.abs() @ b.abs().t())).all()

"""The 8-bit operators against plain implementations in 64 bits.

Codes are whole numbers and have to be equal: a code is the number nearest to
127 y / max|y|, ties to even, and products of 16-bit values are exact in fp64.
Tolerances count half steps: 2^-24 for each fp32 operation, eps / 2 for the last
rounding to the output's type.
"""

from __future__ import annotations

import pytest
import torch

from helpers import announce, assert_bitwise_equal, captured_kernels, generator
from stateful_llm_compiler_hip import _native, backends

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF32 = 2.0**-24


# What squares summed in fp32, in chains of at most eight, would need: each step off by
# at most half a step of a growing sum, 8 * 2^-24 of the mean, half of that of its root;
# one more for the scale's own rounding.  test_norm_scales_are_rounded_once asks for the
# last alone.
NORM = 5


def q8(y):
    """Codes (float64) and scales of the rows of a float64 y."""

    amax = y.abs().amax(-1, keepdim=True)
    good = torch.isfinite(amax)
    codes = torch.where((amax > 0) & good, torch.round(y * 127 / amax), 0.0)
    return codes, torch.where(good, amax / 127, torch.nan).squeeze(-1)


def check_rows(codes, scales, y, factor=1.0, half_steps=1):
    """Codes of y and scales of y * factor [..., 1]; the scale is rounded once,
    after few fp64 operations, and a norm's by the five half steps of NORM."""

    want, want_scales = q8(y)
    want_scales = want_scales * (factor if isinstance(factor, float) else factor.squeeze(-1))
    assert codes.dtype == torch.int8 and codes.shape == y.shape and codes.is_contiguous()
    assert scales.dtype == torch.float32 and scales.shape == y.shape[:-1]
    codes, scales = codes.cpu().double(), scales.cpu().double()
    wrong = (codes != want).nonzero()
    assert not len(wrong), f"{len(wrong)} codes differ, first at {wrong[0].tolist()}"
    assert torch.equal(scales.isnan(), want_scales.isnan())
    fine = ~want_scales.isnan()
    # 2^-150 is half a step of the smallest fp32 numbers.
    bound = want_scales * (half_steps * HALF32 * 1.001) + 2.0**-150
    assert ((scales - want_scales).abs() <= bound)[fine].all()


def rows_of(rows, k, dtype, seed, scale=1.0):
    g = generator(seed)
    x = torch.randn(rows, k, generator=g) * (torch.rand(rows, 1, generator=g) * 3 + 0.1) * scale
    x[:, :: max(1, k // 3)] *= 6
    if rows > 2:
        x[2] = 0.0
    return x.to(dtype)


def swiglu_exact(gate, up):
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


# A vector's tail, one wave's and several waves' registers, and rows read twice.
WIDTHS = [1, 2, 7, 8, 9, 511, 512, 513, 896, 1001, 1024, 1030, 2048, 2055, 4096, 4864, 6144, 6150, 16384, 16390,
          32768, 33001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", WIDTHS)
def test_quantize(gpu, dtype, k):
    announce(f"quantize {dtype} {k}")
    x = rows_of(5, k, dtype, k)
    check_rows(*backends.hip_quantize_q8(x.to(gpu)), x.double())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("k", WIDTHS)
def test_norm(gpu, dtype, residual, k):
    announce(f"norm {dtype} {residual} {k}")
    x, r = rows_of(5, k, dtype, k), rows_of(5, k, dtype, k + 1, 3.0)
    w = (torch.randn(k, generator=generator(k + 2)) * 0.5 + 1).to(dtype)
    eps = 1e-6
    if residual:
        summed, codes, scales = backends.hip_add_rms_norm_q8(x.to(gpu), r.to(gpu), w.to(gpu), epsilon=eps)
        assert_bitwise_equal(summed, backends.hip_add(x.to(gpu), r.to(gpu)))
        assert_bitwise_equal(summed, (x.float() + r.float()).to(dtype))
        x = summed.cpu()
    else:
        codes, scales = backends.hip_rms_norm_q8(x.to(gpu), w.to(gpu), epsilon=eps)
    h = x.double()
    eps32 = float(torch.tensor(eps, dtype=torch.float32))
    check_rows(codes, scales, h * w.double(), torch.rsqrt(h.square().mean(-1, keepdim=True) + eps32), NORM)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", WIDTHS)
def test_swiglu(gpu, dtype, k):
    announce(f"swiglu {dtype} {k}")
    # The halves of one projection's output, whose rows are 2k apart.
    both = rows_of(5, 2 * k, dtype, k, 2.0)
    device = both.to(gpu)
    codes, scales = backends.hip_swiglu_q8(device[:, :k], device[:, k:])
    check_rows(codes, scales, swiglu_exact(both[:, :k], both[:, k:]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(gpu, dtype):
    announce(f"many rows {dtype}")
    x = rows_of(4099, 896, dtype, 3)
    check_rows(*backends.hip_quantize_q8(x.to(gpu)), x.double())
    up = rows_of(4099, 896, dtype, 4)
    check_rows(*backends.hip_swiglu_q8(x.to(gpu), up.to(gpu)), swiglu_exact(x, up))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_even(gpu, dtype):
    # Largest value 127 * 2^e: every odd half step is a tie.
    steps = torch.arange(-254, 255, dtype=torch.float64) / 2
    x = torch.stack([steps * 2.0**e for e in (-6, 0, 1, 5)]).to(dtype)
    assert torch.equal(x[1].double(), steps)  # no rounding in any of the types
    announce(f"ties {dtype}")
    codes, scales = backends.hip_quantize_q8(x.to(gpu))
    check_rows(codes, scales, x.double())
    assert torch.equal(codes[1].cpu().double(), torch.round(steps))
    # The same of products: a weight of 2^-3 moves every value alike.
    w = torch.full((steps.numel(),), 0.125, dtype=dtype)
    codes, _ = backends.hip_rms_norm_q8(x.to(gpu), w.to(gpu), epsilon=0.0)
    assert torch.equal(codes[1].cpu().double(), torch.round(steps))


def test_products_next_to_a_border(gpu):
    # amax 127 * 3 in 16-bit products: v * (127 / amax) rounds, ties do not.
    g = generator(5)
    odd = torch.randint(-127, 128, (64, 256), generator=g).double() * 1.5  # half steps of amax / 127 = 3
    x = odd.clone()
    x[:, 0] = 381.0
    w = torch.ones(256)
    announce("border products")
    for dtype in (torch.float16, torch.float32):
        codes, _ = backends.hip_rms_norm_q8(x.to(dtype).to(gpu), w.to(dtype).to(gpu), epsilon=1e-6)
        assert torch.equal(codes.cpu().double(), torch.round(x / 3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [40, 896, 4864, 33001])
def test_rows_without_a_value_and_extreme_rows(gpu, dtype, k):
    info = torch.finfo(dtype)
    x = rows_of(12, k, dtype, 11)
    x[0] = 0.0
    x[1, k // 2] = torch.nan
    x[3, k - 1] = torch.inf
    x[4, 0] = -torch.inf
    x[5] = 0.0
    x[5, k - 1] = info.max
    x[6] = info.tiny * 0.25  # below the normal numbers
    x[7, 3] = info.max
    x[8] *= info.tiny * 64
    announce(f"extreme rows {dtype} {k}")
    check_rows(*backends.hip_quantize_q8(x.to(gpu)), x.double())

    w = torch.full((k,), 100.0, dtype=dtype)  # products past fp32 in bf16 and fp32
    w[: k // 2] = 0.01
    h = x.double()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + float(torch.tensor(1e-6, dtype=torch.float32)))
    y = h * w.double()
    y[~torch.isfinite(y).all(-1) | ~torch.isfinite(rstd).squeeze(-1)] = torch.nan
    codes, scales = backends.hip_rms_norm_q8(x.to(gpu), w.to(gpu), epsilon=1e-6)
    check_rows(codes, scales, y, rstd, NORM)
    residual = torch.zeros_like(x)
    summed, codes2, scales2 = backends.hip_add_rms_norm_q8(x.to(gpu), residual.to(gpu), w.to(gpu), epsilon=1e-6)
    assert_bitwise_equal(codes2, codes)
    assert torch.equal(summed.cpu().nan_to_num(7.0), x.nan_to_num(7.0))

    up = rows_of(12, k, dtype, 12)
    up[9] = info.max
    gate = x.clone()
    gate[10] = -100.0  # exp(100) is past fp32, silu(-100) is not 0
    up[10] = min(info.max, 2.0**100)
    gate[11] = -30.0
    y = swiglu_exact(gate, up)
    y[(y.abs().amax(-1) / 127) > torch.finfo(torch.float32).max] = torch.nan
    y[~torch.isfinite(y).all(-1)] = torch.nan
    check_rows(*backends.hip_swiglu_q8(gate.to(gpu), up.to(gpu)), y)


def test_norm_of_zeros_without_epsilon_is_nan(gpu):
    announce("zeros, eps 0")
    codes, scales = backends.hip_rms_norm_q8(torch.zeros(3, 64, device=gpu), torch.ones(64, device=gpu), epsilon=0.0)
    assert scales.isnan().all() and not codes.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(gpu, dtype):
    announce(f"layouts {dtype}")
    base = rows_of(6 * 7, 104, dtype, 21)
    device = base.to(gpu)
    # A first element off the vectors' alignment, rows apart.
    check_rows(*backends.hip_quantize_q8(device[:, 1:98]), base[:, 1:98].double())
    w = torch.linspace(-1, 2, 98).to(dtype)
    codes, _ = backends.hip_rms_norm_q8(device[:, 1:98], w.to(gpu)[1:], epsilon=1e-6)
    check_codes = q8(base[:, 1:98].double() * w[1:].double())[0]
    assert torch.equal(codes.cpu().double(), check_codes)
    # Heads out of place (a copy), every other row, a column stride, one row twice.
    heads, host = device.view(6, 7, 104).permute(1, 0, 2), base.view(6, 7, 104).permute(1, 0, 2)
    check_rows(*backends.hip_quantize_q8(heads), host.double())
    check_rows(*backends.hip_quantize_q8(device[::2]), base[::2].double())
    check_rows(*backends.hip_quantize_q8(device[:, ::2]), base[:, ::2].double())
    check_rows(*backends.hip_quantize_q8(device[:1].expand(5, 104)), base[:1].expand(5, 104).double())
    check_rows(*backends.hip_quantize_q8(device[:, 5:6]), base[:, 5:6].double())
    check_rows(*backends.hip_quantize_q8(device[3]), base[3].double())
    check_rows(*backends.hip_swiglu_q8(device[:21], heads.reshape(42, 104)[21:]),
               swiglu_exact(base[:21], host.reshape(42, 104)[21:]))
    other = torch.randn(42, 104, generator=generator(1)).to(dtype)
    padded = torch.zeros(42, 300, dtype=dtype)
    padded[:, 3:107] = other
    summed, codes, _ = backends.hip_add_rms_norm_q8(device, padded.to(gpu)[:, 3:107], torch.ones(104, dtype=dtype,
                                                                                               device=gpu), epsilon=0.1)
    assert_bitwise_equal(summed, (base.float() + other.float()).to(dtype))
    assert torch.equal(codes.cpu().double(), q8(summed.cpu().double())[0])


def test_halves_of_a_padded_batch(gpu):
    # Gate and up as views of one projection [batch, tokens, 2 I]; the second sequence ends early.
    announce("halves of a batch")
    base = rows_of(3 * 5, 2 * 56, torch.bfloat16, 31).view(3, 5, 112)
    base[1, 3:] = 0.0
    gate, up = base.to(gpu).chunk(2, dim=-1)
    codes, scales = backends.hip_swiglu_q8(gate, up)
    check_rows(codes, scales, swiglu_exact(*base.chunk(2, dim=-1)))
    assert not scales[1, 3:].any() and not codes[1, 3:].any()
    # The first two sequences of it, and every second token: no view of evenly strided rows.
    for part in ((slice(0, 2),), (slice(None), slice(0, 5, 2))):
        check_rows(*backends.hip_swiglu_q8(gate[part], up[part]), swiglu_exact(*base[part].chunk(2, dim=-1)))


def test_empty_calls(gpu):
    announce("empty")
    x = torch.zeros(0, 3, 16, device=gpu)
    codes, scales = backends.hip_quantize_q8(x)
    assert codes.shape == (0, 3, 16) and scales.shape == (0, 3)
    w = torch.zeros(5, 16, dtype=torch.int8, device=gpu)
    y = backends.hip_linear_q8(codes, scales, w, torch.ones(5, device=gpu))
    assert y.shape == (0, 3, 5) and y.dtype == torch.bfloat16
    summed, codes, _ = backends.hip_add_rms_norm_q8(x, x, torch.ones(16, device=gpu), epsilon=1e-6)
    assert summed.shape == x.shape and codes.shape == x.shape


def test_refusals(gpu):
    x, w = torch.zeros(2, 16, device=gpu), torch.ones(16, device=gpu)
    codes, scales = torch.zeros(2, 16, dtype=torch.int8, device=gpu), torch.zeros(2, device=gpu)
    weight, weight_scales = torch.zeros(5, 16, dtype=torch.int8, device=gpu), torch.zeros(5, device=gpu)
    linear = backends.hip_linear_q8
    for call in (
        lambda: backends.hip_quantize_q8(codes),
        lambda: backends.hip_quantize_q8(x.double()),
        lambda: backends.hip_quantize_q8(x[0, 0]),
        lambda: backends.hip_quantize_q8(x[:, :0]),
        lambda: backends.hip_quantize_q8(torch.zeros(1, 131072, device=gpu)),
        lambda: backends.hip_rms_norm_q8(x, w.bfloat16(), epsilon=1e-6),
        lambda: backends.hip_rms_norm_q8(x, w[:15], epsilon=1e-6),
        lambda: backends.hip_rms_norm_q8(x, w.view(1, 16), epsilon=1e-6),
        lambda: backends.hip_rms_norm_q8(x, w, epsilon=-1e-6),
        lambda: backends.hip_rms_norm_q8(x, w, epsilon=float("nan")),
        lambda: backends.hip_rms_norm_q8(x, w, epsilon=float("inf")),
        lambda: backends.hip_add_rms_norm_q8(x, x[:1], w, epsilon=1e-6),
        lambda: backends.hip_add_rms_norm_q8(x, x.bfloat16(), w, epsilon=1e-6),
        lambda: backends.hip_add_rms_norm_q8(x, x.cpu(), w, epsilon=1e-6),
        lambda: backends.hip_swiglu_q8(x, x[:, :8]),
        lambda: backends.hip_swiglu_q8(x, x.half()),
        lambda: linear(x, scales, weight, weight_scales),
        lambda: linear(codes, scales.double(), weight, weight_scales),
        lambda: linear(codes, scales, weight.float(), weight_scales),
        lambda: linear(codes, scales, weight[:, :8], weight_scales),
        lambda: linear(codes, scales[:1], weight, weight_scales),
        lambda: linear(codes, scales, weight, weight_scales[:4]),
        lambda: linear(codes, scales, weight, weight_scales, torch.zeros(5, device=gpu)),  # fp32 bias, bf16 output
        lambda: linear(codes, scales, weight, weight_scales, torch.zeros(4, device=gpu, dtype=torch.bfloat16)),
        lambda: linear(codes, scales, weight, weight_scales, output_dtype=torch.float64),
        lambda: linear(codes, scales, weight.view(5, 4, 4), weight_scales),
        lambda: linear(codes.t().contiguous().t(), scales, weight, weight_scales),
        lambda: linear(codes.cpu(), scales, weight, weight_scales),
        lambda: linear(codes[:, :0], scales, weight[:, :0], weight_scales),
        lambda: linear(codes, scales, weight[:0], weight_scales[:0]),
    ):
        with pytest.raises(ValueError):
            call()


# ---- the product ---------------------------------------------------------------


def product_exact(codes, scales, weight, weight_scales, bias):
    """(result, magnitude of the product) in 64 bits."""

    sums = codes.double() @ weight.double().t()
    product = sums * scales.double().unsqueeze(-1) * weight_scales.double()
    return (product if bias is None else product + bias.double()), product.abs()


def check_product(y, codes, scales, weight, weight_scales, bias, dtype):
    want, size = product_exact(codes, scales, weight, weight_scales, bias)
    assert y.dtype == dtype and y.shape == want.shape
    # The sum's conversion and the token's scale, then the channel's scale and the
    # bias in one fma; then the output's type, whose subnormals' half step is last.
    half, fine = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
    bound = 2 * HALF32 * size * 1.001 + want.abs() * (HALF32 + half) * 1.001 + fine
    off = (y.cpu().double() - want).abs()
    assert (off <= bound).all(), f"off by {(off / bound).max().item():.3g} of the bound"


def operands(m, n, k, bias_dtype, seed, low=-128, high=128):
    g = generator(seed)
    codes = torch.randint(low, high, (m, k), generator=g, dtype=torch.int8)
    weight = torch.randint(low, high, (n, k), generator=g, dtype=torch.int8)
    scales, weight_scales = torch.rand(m, generator=g) * 0.02, torch.rand(n, generator=g) * 0.01
    bias = None if bias_dtype is None else torch.randn(n, generator=g).to(bias_dtype)
    return codes, scales, weight, weight_scales, bias


def run_product(gpu, m, n, k, dtype, bias=True, seed=0, **kw):
    announce(f"linear {m} x {n} x {k} {dtype}")
    ops = operands(m, n, k, dtype if bias else None, seed, **kw)
    y = backends.hip_linear_q8(*(None if t is None else t.to(gpu) for t in ops), output_dtype=dtype)
    check_product(y, *ops, dtype)
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 5, 16), (3, 7, 15), (2, 17, 17), (8, 1152, 896), (16, 896, 4864), (17, 100, 64), (31, 33, 1001),
    (33, 64, 128), (48, 896, 144), (64, 4864, 896), (65, 66, 130), (100, 200, 112), (129, 257, 1040), (300, 1003, 1001),
    (512, 896, 4864), (5, 20000, 80), (20, 18000, 896), (260, 4104, 272),
])
def test_linear(gpu, dtype, m, n, k):
    run_product(gpu, m, n, k, dtype, bias=(m + n) % 2 == 0, seed=m + n + k)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 1025])
def test_linear_rows(gpu, m):
    run_product(gpu, m, 192, 320, torch.bfloat16, seed=m)


@pytest.mark.parametrize("k", [1, 2, 3, 15, 16, 31, 32, 48, 63, 64, 65, 127, 128, 129, 144, 255, 256, 384, 511, 512,
                               528, 1024, 1040, 4096])
def test_linear_depths(gpu, k):
    for m in (4, 40, 200):
        run_product(gpu, m, 136, k, torch.float32, seed=k)


@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 255, 257, 300])
def test_linear_widths(gpu, n):
    for m in (4, 40, 200):
        run_product(gpu, m, n, 256, torch.float16, seed=n)


@pytest.mark.parametrize("m", [1, 100])
@pytest.mark.parametrize("sign", [-128, 127])
def test_linear_longest_sums(gpu, m, sign):
    # K = 131071 products of (-128)^2 are 2^31 - 2^14, the largest sum of 32 bits.
    announce(f"longest sums {m} {sign}")
    k, n = 131071, 40
    codes = torch.full((m, k), -128, dtype=torch.int8, device=gpu)
    weight = torch.full((n, k), sign, dtype=torch.int8, device=gpu)
    one = torch.ones(max(m, n), device=gpu)
    y = backends.hip_linear_q8(codes, one[:m], weight, one[:n], output_dtype=torch.float32)
    assert (y.double() == float(torch.tensor(-128.0 * sign * k, dtype=torch.float32))).all()


def test_linear_is_the_same_on_every_path(gpu):
    # The sums are exact, so a row's result does not depend on the rows beside it.
    announce("rows alone")
    codes, scales, weight, weight_scales, bias = (t.to(gpu) for t in operands(600, 904, 896, torch.bfloat16, 3))
    whole = backends.hip_linear_q8(codes, scales, weight, weight_scales, bias)
    for rows in (1, 8, 17, 40, 64, 100, 300):
        part = backends.hip_linear_q8(codes[:rows], scales[:rows], weight, weight_scales, bias)
        assert_bitwise_equal(part, whole[:rows])
    # Off the vectors' alignment.
    odd = torch.zeros(600 * 896 + 1, dtype=torch.int8, device=gpu)[1:].view(600, 896)
    odd.copy_(codes)
    assert_bitwise_equal(backends.hip_linear_q8(odd, scales, weight, weight_scales, bias), whole)
    odd_w = torch.zeros(904 * 896 + 3, dtype=torch.int8, device=gpu)[3:].view(904, 896)
    odd_w.copy_(weight)
    for rows in (5, 50, 600):
        y = backends.hip_linear_q8(codes[:rows], scales[:rows], odd_w, weight_scales, bias)
        assert_bitwise_equal(y, whole[:rows])


# The row kernel, each tile (with 16-byte stores and without), unaligned rows.
STRIDED = [(3, 200, 128), (30, 300, 144), (50, 96, 256), (50, 200, 256), (120, 500, 272), (3, 50001, 128),
           (200, 20000, 128), (500, 9728, 128), (1100, 9728, 128), (2300, 9728, 896), (2300, 9731, 896),
           (4000, 4096, 2048), (4000, 4090, 2048), (120, 9000, 272), (120, 9001, 272), (70, 130, 77),
           (1100, 9731, 33), (4100, 1030, 7)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", STRIDED)
def test_linear_writes_its_outputs_only(gpu, dtype, m, n, k):
    announce(f"strided {m} x {n} x {k} {dtype}")
    lib, tag = _native.library(), _native.dtype_tag(dtype)
    codes, scales, weight, weight_scales, bias = (t.to(gpu) for t in operands(m, n, k, dtype, m + n))
    x_rs, y_rs = k + 48, n + 24
    padded = torch.full((m + 2, x_rs), 99, dtype=torch.int8, device=gpu)
    padded[:m, :k] = codes
    out = torch.full((m + 3, y_rs), 7.0, dtype=dtype, device=gpu)
    want = backends.hip_linear_q8(codes, scales, weight, weight_scales, bias, output_dtype=dtype)
    _native.check(lib.slc_hip_linear_q8(
        padded.data_ptr(), scales.data_ptr(), weight.data_ptr(), weight_scales.data_ptr(), bias.data_ptr(),
        out.data_ptr(), tag, m, n, k, x_rs, y_rs, _native.current_stream(gpu)), "slc_hip_linear_q8")
    assert_bitwise_equal(out[:m, :n], want)
    assert (out[m:] == 7).all() and (out[:, n:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", STRIDED)
def test_linear_rounds_where_it_says(gpu, dtype, m, n, k):
    # Without a bias the bits follow: the sum is exact, float(sum) and its product with the
    # token's scale are fp32 roundings, the product with the channel's scale is exact in fp64
    # (24 x 24 bits), and then come one rounding to fp32 and one to the output's type.
    announce(f"roundings {m} x {n} x {k} {dtype}")
    codes, scales, weight, weight_scales, _ = (t.to(gpu) if t is not None else None for t in operands(m, n, k, None, 3))
    sums = codes.double() @ weight.double().t()
    want = ((sums.float() * scales.unsqueeze(-1)).double() * weight_scales.double()).float().to(dtype)
    assert_bitwise_equal(backends.hip_linear_q8(codes, scales, weight, weight_scales, output_dtype=dtype), want)


@pytest.mark.parametrize("n", [40, 9728, 20000])
def test_linear_of_one_row_takes_any_strides(gpu, n):
    announce(f"one row {n}")
    lib = _native.library()
    codes, scales, weight, weight_scales, bias = (t.to(gpu) for t in operands(1, n, 256, torch.bfloat16, 4))
    want = backends.hip_linear_q8(codes, scales, weight, weight_scales, bias)
    for x_rs, y_rs in ((0, 0), (7, 1), (-5, -5)):
        out = torch.full((70, n), 7.0, dtype=torch.bfloat16, device=gpu)
        _native.check(lib.slc_hip_linear_q8(
            codes.data_ptr(), scales.data_ptr(), weight.data_ptr(), weight_scales.data_ptr(), bias.data_ptr(),
            out.data_ptr(), _native.SLC_BF16, 1, n, 256, x_rs, y_rs, _native.current_stream(gpu)), "slc_hip_linear_q8")
        assert_bitwise_equal(out[:1], want)
        assert (out[1:] == 7).all()


def test_linear_of_a_repeated_row(gpu):
    # A row stride of 0: every row of X is the same one.
    announce("repeated row")
    lib = _native.library()
    codes, scales, weight, weight_scales, _ = operands(1, 512, 256, None, 6)
    for m in (20, 100, 600):
        tokens = torch.rand(m, generator=generator(m)).to(gpu)
        out = torch.empty(m, 512, device=gpu)
        row, w, ws = codes.to(gpu), weight.to(gpu), weight_scales.to(gpu)
        _native.check(lib.slc_hip_linear_q8(
            row.data_ptr(), tokens.data_ptr(), w.data_ptr(), ws.data_ptr(), None, out.data_ptr(), _native.SLC_F32, m,
            512, 256, 0, 512, _native.current_stream(gpu)), "slc_hip_linear_q8")
        assert_bitwise_equal(out, backends.hip_linear_q8(row.expand(m, 256).contiguous(), tokens, w, ws,
                                                         output_dtype=torch.float32))


def test_more_unaligned_rows_than_one_grid(gpu):
    # More than 65535 tiles of 128 rows.
    announce("8388485 rows")
    m = 65535 * 128 + 5
    codes = torch.ones(m, 3, dtype=torch.int8, device=gpu)
    codes[-1] = 5
    scales = torch.ones(m, device=gpu)
    weight = torch.tensor([[1, 2, 3], [-1, 0, 1]], dtype=torch.int8, device=gpu)
    y = backends.hip_linear_q8(codes, scales, weight, torch.ones(2, device=gpu), output_dtype=torch.float32)
    assert (y[:-1] == torch.tensor([6.0, 0.0], device=gpu)).all() and y[-1].tolist() == [30.0, 0.0]


def test_more_features_than_one_launch_has_threads(gpu):
    # 2^23 groups of 32 features and one more.
    n = (1 << 28) + 16
    announce(f"{n} features")
    weight = torch.empty(n, 16, dtype=torch.int8, device=gpu).random_(-128, 128)
    codes, scales, _, _, _ = (t.to(gpu) if t is not None else None for t in operands(2, 16, 16, None, 8))
    weight_scales = torch.full((n,), 0.5, device=gpu)
    y = backends.hip_linear_q8(codes, scales, weight, weight_scales)
    for at in (0, (1 << 27) - 64, n - 128):
        part = slice(at, at + 128)
        assert_bitwise_equal(y[:, part], backends.hip_linear_q8(codes, scales, weight[part], weight_scales[part]))


@pytest.mark.parametrize("at", [1, 2, 8])
def test_linear_of_operands_at_any_address(gpu, at):
    announce(f"address {at}")
    for m, n, k in ((5, 200, 128), (70, 130, 256), (70, 130, 37)):
        codes, scales, weight, weight_scales, _ = (t.to(gpu) if t is not None else None for t in operands(m, n, k, None, at))
        want = backends.hip_linear_q8(codes, scales, weight, weight_scales)
        moved = [torch.full((t.numel() + 16,), 99, dtype=torch.int8, device=gpu) for t in (codes, weight)]
        views = [b[at:at + t.numel()].view(t.shape) for b, t in zip(moved, (codes, weight))]
        for view, t in zip(views, (codes, weight)):
            view.copy_(t)
        for x, w in ((views[0], weight), (codes, views[1]), views):
            assert_bitwise_equal(backends.hip_linear_q8(x, scales, w, weight_scales), want)


def test_outputs_past_32_bits(gpu):
    m, n = 20000, 110000
    announce(f"{m} x {n} outputs")
    codes, scales, _, _, _ = (t.to(gpu) if t is not None else None for t in operands(m, 16, 64, None, 12))
    _, _, weight, weight_scales, _ = (t.to(gpu) if t is not None else None for t in operands(1, n, 64, None, 13))
    y = backends.hip_linear_q8(codes, scales, weight, weight_scales)
    for part in (slice(0, 300), slice(9700, 10000), slice(m - 300, m)):
        assert_bitwise_equal(y[part], backends.hip_linear_q8(codes[part], scales[part], weight, weight_scales))


def test_linear_leading_axes_and_nan_rows(gpu):
    announce("leading axes")
    codes, scales, weight, weight_scales, _ = operands(12, 64, 128, None, 9)
    scales[5] = torch.nan
    y = backends.hip_linear_q8(codes.view(3, 4, 128).to(gpu), scales.view(3, 4).to(gpu), weight.to(gpu),
                               weight_scales.to(gpu)).cpu()
    assert y.shape == (3, 4, 64)
    flat = y.view(12, 64)
    assert flat[5].isnan().all() and not flat[torch.arange(12) != 5].isnan().any()
    one = backends.hip_linear_q8(codes[0].to(gpu), scales[0].to(gpu), weight.to(gpu), weight_scales.to(gpu))
    assert one.shape == (64,)
    assert_bitwise_equal(one, flat[0])


def test_weight_rows_past_32_bits(gpu):
    # A weight of 2^31 bytes and more: its last rows are past 32-bit offsets.
    announce("weight past 2^31 bytes")
    n, k = 2**18 + 40, 8208
    g = torch.Generator(device=gpu).manual_seed(1)
    weight = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8, device=gpu)
    for m in (3, 70):
        codes = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8, device=gpu)
        scales = torch.rand(m, generator=g, device=gpu)
        weight_scales = torch.rand(n, generator=g, device=gpu)
        y = backends.hip_linear_q8(codes, scales, weight, weight_scales, output_dtype=torch.float32)
        for part in (slice(0, 40), slice(2**17, 2**17 + 40), slice(n - 40, n)):
            check_product(y[:, part], codes.cpu(), scales.cpu(), weight[part].cpu(), weight_scales[part].cpu(), None,
                          torch.float32)


def test_more_rows_than_one_grid(gpu):
    # 64 threads a row: 2^26 rows are 2^32 threads, one more than a grid holds.
    announce("2^26 + 5 rows")
    rows = 2**26 + 5
    x = torch.ones(rows, 1, dtype=torch.bfloat16, device=gpu)
    x[-1] = -2.0
    codes, scales = backends.hip_quantize_q8(x)
    assert int(codes[:-1].amin()) == 127 and int(codes[-1]) == -127
    one = torch.tensor(1.0, dtype=torch.float64) / 127
    assert (scales[:-1] == float(one.float())).all() and float(scales[-1]) == float((2 * one).float())


def test_rows_past_32_bits(gpu):
    announce("rows past 2^31 values")
    rows, k = 65540, 32770
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=gpu)
    x[:: rows - 1, ::7] = 3.0
    x[rows - 1, k - 1] = -4.0
    codes, scales = backends.hip_quantize_q8(x)
    last = x[rows - 1].cpu()
    check_rows(codes[rows - 1], scales[rows - 1], last.double())
    check_rows(codes[0], scales[0], x[0].cpu().double())
    assert not scales[1 : rows - 1].any()


# ---- as they are used ------------------------------------------------------------


def weights(n, k, seed):
    return torch.randn(n, k, generator=generator(seed)) * 0.05


def layer(x, residual, params):
    """Norm, gate/up, SwiGLU, down: an MLP block on 8-bit linears."""

    summed, codes, scales = backends.hip_add_rms_norm_q8(x, residual, params["norm"], epsilon=1e-6)
    both = backends.hip_linear_q8(codes, scales, *params["gate_up"])
    codes, scales = backends.hip_swiglu_q8(*both.chunk(2, dim=-1))
    return summed, backends.hip_linear_q8(codes, scales, *params["down"])


def layer_params(gpu):
    k, n = 896, 1216
    return {"norm": (torch.rand(k, generator=generator(1)) + 0.5).bfloat16().to(gpu),
            "gate_up": backends.hip_quantize_q8(weights(2 * n, k, 2).to(gpu)),
            "down": backends.hip_quantize_q8(weights(k, n, 3).to(gpu))}


@pytest.mark.parametrize("rows", [1, 30, 70, 300])
def test_mlp_block(gpu, rows):
    announce(f"mlp {rows}")
    params = layer_params(gpu)
    x, residual = rows_of(rows, 896, torch.bfloat16, 4), rows_of(rows, 896, torch.bfloat16, 5)
    summed, y = layer(x.to(gpu), residual.to(gpu), params)

    def plain(name):
        codes, scales = params[name]
        return codes.cpu().double() * scales.cpu().double().unsqueeze(-1)

    h = (x.float() + residual.float()).bfloat16().double()
    assert torch.equal(summed.cpu().double(), h)
    eps32 = float(torch.tensor(1e-6, dtype=torch.float32))
    codes, scales = q8(h * params["norm"].cpu().double())
    scales = scales * torch.rsqrt(h.square().mean(-1) + eps32)
    both = codes * scales.unsqueeze(-1) @ plain("gate_up").t()
    # The projection is stored in bf16; from the kernels' own values of it on, so
    # that a rounding's flip does not move the codes that follow.
    got = backends.hip_linear_q8(codes.to(torch.int8).to(gpu), scales.float().to(gpu), *params["gate_up"]).cpu().double()
    assert ((got - both).abs() <= both.abs() * 2.0**-8 + 1e-6 * both.abs().amax()).all()
    codes, scales = q8(swiglu_exact(*got.chunk(2, dim=-1)))
    want = codes * scales.unsqueeze(-1) @ plain("down").t()
    # Half a step of bf16, and the fp32 operations on the sums.
    assert ((y.cpu().double() - want).abs() <= want.abs() * 2.0**-8 * 1.001 + want.abs().amax() * 2.0**-20).all()


def test_side_stream_and_graph(gpu):
    announce("stream and graph")
    params = layer_params(gpu)
    inputs = [(rows_of(24, 896, torch.bfloat16, s).to(gpu), rows_of(24, 896, torch.bfloat16, s + 50).to(gpu))
              for s in range(4)]
    wants = [layer(x, r, params) for x, r in inputs]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = [layer(x, r, params) for x, r in inputs]
    stream.synchronize()
    for got, want in zip(side, wants):
        for a, b in zip(got, want):
            assert_bitwise_equal(a, b)
    x, r = inputs[0][0].clone(), inputs[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, r, params)
    for turn in range(3):
        for (new_x, new_r), want in zip(inputs, wants):
            x.copy_(new_x)
            r.copy_(new_r)
            graph.replay()
            eager = layer(new_x, new_r, params)
            torch.cuda.synchronize()
            for a, b, c in zip(out, want, eager):
                assert_bitwise_equal(a, b)
                assert_bitwise_equal(c, b)


def test_two_streams_at_once(gpu):
    announce("two streams")
    params = layer_params(gpu)
    inputs = [(rows_of(200, 896, torch.bfloat16, s).to(gpu), rows_of(200, 896, torch.bfloat16, s + 9).to(gpu))
              for s in (1, 2)]
    wants = [layer(x, r, params) for x, r in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(layer(*inputs[i], params))
    torch.cuda.synchronize()
    for i in range(2):
        for result in got[i]:
            for a, b in zip(result, wants[i]):
                assert_bitwise_equal(a, b)


# ---- every kernel, and past a workgroup's first tile ---------------------------------
# Which kernel takes a shape is a matter of speed and may change; these tests name the
# kernel that they mean, so that one which no longer runs it fails and its shape is moved.


# Vectors a lane (0: rows read twice) of many rows, few values past them in a row or none,
# the last row's end inside a vector.  SwiGLU of 2100 x 4864 is a prefill's.
ROW_VARIANTS = [
    (torch.bfloat16, 2100, 896, 2), (torch.bfloat16, 2100, 4864, 3), (torch.bfloat16, 2101, 4865, 3),
    (torch.bfloat16, 1100, 2063, 3), (torch.bfloat16, 300, 8192, 4), (torch.bfloat16, 701, 16390, 4),
    (torch.bfloat16, 300, 33001, 0), (torch.float16, 2101, 4864, 3), (torch.float16, 2100, 4867, 3),
    (torch.float16, 700, 16391, 4), (torch.float32, 1100, 896, 4), (torch.float32, 2101, 896, 2),
    (torch.float32, 2100, 4864, 3), (torch.float32, 2101, 4865, 3), (torch.float32, 701, 9001, 4),
    (torch.float32, 300, 16390, 0),
]


@pytest.mark.parametrize("source", ["plain", "norm", "add norm", "swiglu"])
@pytest.mark.parametrize("dtype,rows,k,vectors", ROW_VARIANTS)
def test_row_kernels_of_many_rows(gpu, dtype, rows, k, vectors, source):
    announce(f"{source} {rows} x {k} {dtype}")
    x, other = rows_of(rows, 2 * k, dtype, k, 2.0), rows_of(rows, k, dtype, k + 1, 3.0)
    w = (torch.randn(k, generator=generator(k + 2)) * 0.5 + 1).to(dtype)
    both, other_gpu, w_gpu = x.to(gpu), other.to(gpu), w.to(gpu)
    left, right = both[:, :k], both[:, k:]  # rows 2k apart
    x, y = x[:, :k], x[:, k:]
    call = {"plain": lambda: backends.hip_quantize_q8(left),
            "norm": lambda: backends.hip_rms_norm_q8(left, w_gpu, epsilon=1e-6),
            "add norm": lambda: backends.hip_add_rms_norm_q8(left, other_gpu, w_gpu, epsilon=1e-6),
            "swiglu": lambda: backends.hip_swiglu_q8(left, right)}[source]
    *summed, codes, scales = call()
    if source in ("plain", "swiglu"):
        check_rows(codes, scales, x.double() if source == "plain" else swiglu_exact(x, y))
    else:
        if summed:
            x = (x.float() + other.float()).to(dtype)
            assert_bitwise_equal(summed[0], x)
        h = x.double()
        eps32 = float(torch.tensor(1e-6, dtype=torch.float32))
        check_rows(codes, scales, h * w.double(), torch.rsqrt(h.square().mean(-1, keepdim=True) + eps32), NORM)
    (name, (_, nv, loop), _), = captured_kernels(call)
    assert (name, 0 if loop else nv) == ("quantize", vectors)


# Kernel, tile (or row blocks, feature blocks and depth), 16-byte stores or not.  The rings and
# the turns walk several output tiles a workgroup, of sizes that the tile divides and others;
# the 256 x 256 ones two each, and two or three.
LINEAR_VARIANTS = [
    (8, 1152, 896, "rows", (1, 1, 4)), (30, 300, 144, "rows", (2, 1, 2)), (3, 50001, 128, "rows", (1, 2, 2)),
    (20, 20000, 272, "stream", (64, 64, 1)), (20, 20001, 272, "stream", (64, 64, 0)),
    (37692, 24, 2960, "stream", (128, 64, 1)), (34001, 23, 512, "stream", (128, 64, 0)),
    (200, 20000, 128, "stream", (128, 128, 1)), (200, 20001, 128, "stream", (128, 128, 0)),
    (500, 9731, 128, "stream", (128, 128, 0)), (2300, 9728, 896, "stream", (256, 128, 1)),
    (2300, 9731, 896, "stream", (256, 128, 0)), (8192, 4096, 2048, "turns", (1,)), (8000, 4090, 2048, "turns", (0,)),
    (8192, 5632, 4096, "turns", (1,)), (8100, 5626, 4096, "turns", (0,)), (300, 1003, 1001, "tile", (64, 64)),
    (2200, 2051, 1001, "tile", (128, 128)), (4100, 1030, 263, "tile", (128, 128)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,kernel,variant", LINEAR_VARIANTS)
def test_linear_kernels_past_their_first_tile(gpu, dtype, m, n, k, kernel, variant):
    announce(f"{kernel} {variant} {m} x {n} x {k} {dtype}")
    g = torch.Generator(device=gpu).manual_seed(m + n + k)
    # Rows of codes are 48 bytes, those of outputs 24 elements longer than their contents.
    padded = torch.randint(-128, 128, (m, k + 48), generator=g, device=gpu, dtype=torch.int8)
    codes = padded[:, :k].contiguous()
    weight = torch.randint(-128, 128, (n, k), generator=g, device=gpu, dtype=torch.int8)
    scales, weight_scales = torch.rand(m, generator=g, device=gpu) * 0.02, torch.rand(n, generator=g, device=gpu) * 0.01
    bias = torch.randn(n, generator=g, device=gpu).to(dtype)
    (name, values, workgroups), = captured_kernels(
        lambda: backends.hip_linear_q8(codes, scales, weight, weight_scales, output_dtype=dtype))
    shown = values[:2] + values[-1:] if name == "stream" else values
    assert (name, shown) == (kernel, variant)
    if name in ("stream", "turns"):
        height, width = values[:2] if name == "stream" else (256, 256)
        assert -(-m // height) * -(-n // width) > workgroups

    # As in test_linear_rounds_where_it_says.
    sums = codes.double() @ weight.double().t()
    product = (sums.float() * scales.unsqueeze(-1)).double() * weight_scales.double()
    del sums
    y = backends.hip_linear_q8(codes, scales, weight, weight_scales, output_dtype=dtype)
    assert torch.equal(y, product.float().to(dtype))  # no NaN, and -0 == 0

    # With a bias: one rounding of the sum to fp32 and one to the output's type.
    lib, tag = _native.library(), _native.dtype_tag(dtype)
    out = torch.full((m + 3, n + 24), 7.0, dtype=dtype, device=gpu)
    _native.check(lib.slc_hip_linear_q8(
        padded.data_ptr(), scales.data_ptr(), weight.data_ptr(), weight_scales.data_ptr(), bias.data_ptr(),
        out.data_ptr(), tag, m, n, k, k + 48, n + 24, _native.current_stream(gpu)), "slc_hip_linear_q8")
    want = product.add_(bias.double())
    info = torch.finfo(dtype)
    bound = want.abs() * ((HALF32 + info.eps / 2) * 1.001) + info.tiny * info.eps / 2
    assert ((out[:m, :n].double() - want).abs() <= bound).all()
    assert (out[m:] == 7).all() and (out[:, n:] == 7).all()


def test_more_unaligned_features_than_one_grid(gpu):
    # More than 2^24 - 1 tiles of 64 features.
    n = (2**24 - 1) * 64 + 70
    announce(f"{n} features of one code")
    weight = torch.empty(n, 1, dtype=torch.int8, device=gpu).random_(-128, 128)
    weight_scales = torch.full((n,), 0.5, device=gpu)
    bias = torch.zeros(n, dtype=torch.float16, device=gpu)
    bias[-70:] = 3.0
    codes = torch.tensor([[7], [-3]], dtype=torch.int8, device=gpu)
    scales = torch.tensor([1.0, 0.25], device=gpu)
    call = lambda: backends.hip_linear_q8(codes, scales, weight, weight_scales, bias, output_dtype=torch.float16)  # noqa: E731
    assert [(name, groups) for name, _, groups in captured_kernels(call)] == [("tile", 2**24 - 1), ("tile", 2)]
    y = call()
    for row, factor in enumerate((3.5, -0.375)):  # exact in fp16: 8 bits of a code times 3
        for at in range(0, n, 2**28):
            part = slice(at, min(n, at + 2**28))
            assert torch.equal(y[row, part].float(), weight[part, 0] * factor + bias[part])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("k", [896, 1001, 4864, 16390, 33001])
def test_norm_scales_are_rounded_once(gpu, dtype, residual, k):
    # Squares of 2^-24 beside those of 1: sums in 24 bits lose every one that follows a 1.
    announce(f"norm scales {dtype} {residual} {k}")
    x = torch.full((96, k), 2.0**-12)
    x[:, :: 16 // dtype.itemsize] = 1.0
    x[:32] *= torch.ldexp(torch.tensor(1.0), -torch.arange(32) // 4).unsqueeze(-1)
    x[64:] = rows_of(32, k, torch.float32, k)
    x = x.to(dtype)
    # Every row has largest products of its own, and so a scale of its own.
    x[torch.arange(96), torch.arange(96) * 7 % k] *= torch.linspace(1.5, 9.5, 96).to(dtype)
    w = (torch.randn(k, generator=generator(k)) * 0.5 + 1).to(dtype)
    if residual:
        _, codes, scales = backends.hip_add_rms_norm_q8(x.to(gpu), torch.zeros_like(x, device=gpu), w.to(gpu),
                                                        epsilon=1e-6)
    else:
        codes, scales = backends.hip_rms_norm_q8(x.to(gpu), w.to(gpu), epsilon=1e-6)
    h = x.double()
    eps32 = float(torch.tensor(1e-6, dtype=torch.float32))
    want_codes, want = q8(h * w.double())
    assert torch.equal(codes.cpu().double(), want_codes)
    want = want * torch.rsqrt(h.square().mean(-1) + eps32)
    # Half a step of fp32, and 2^-44 for what comes before it: chains of at most 150 fp64
    # additions (2^-45.8 of a sum, half of it of its root) and a dozen operations more.
    half = torch.ldexp(torch.ones_like(want), torch.frexp(want)[1] - 25)
    live = want > 0
    assert ((scales.cpu().double() - want).abs() <= half + want * 2.0**-44)[live].all()
    assert not scales.cpu()[~live].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [7, 1001, 33001])
def test_sums_with_nans_are_those_of_hip_add(gpu, dtype, k):
    # Any bits at all; NaNs in one operand, in the other, in both, and infinities that cancel.
    announce(f"sums of any bits {dtype} {k}")
    whole = {2: torch.int16, 4: torch.int32}[dtype.itemsize]
    low, high = torch.iinfo(whole).min, torch.iinfo(whole).max
    g = generator(k)
    a, b = (torch.randint(low, high, (64, k), generator=g, dtype=whole).view(dtype) for _ in range(2))
    kind = torch.rand(64, k, generator=g)
    a[kind < 0.2] = torch.nan
    b[(kind > 0.1) & (kind < 0.3)] = -torch.nan
    a[(kind > 0.3) & (kind < 0.4)] = torch.inf
    b[(kind > 0.35) & (kind < 0.4)] = -torch.inf
    summed, _, scales = backends.hip_add_rms_norm_q8(a.to(gpu), b.to(gpu), torch.ones(k, dtype=dtype, device=gpu),
                                                     epsilon=1e-6)
    want = backends.hip_add(a.to(gpu), b.to(gpu))
    both = (a.isnan() & b.isnan()).to(gpu)
    assert torch.equal(summed.isnan(), want.isnan())
    assert_bitwise_equal(summed[~both], want[~both])
    assert scales[~want.isfinite().all(-1)].isnan().all()


@pytest.mark.parametrize("m,n,k", [(8, 1152, 896), (20, 20001, 272), (200, 20000, 128), (2300, 9731, 896),
                                   (8000, 4090, 2048), (300, 1003, 1001), (2200, 2051, 1001)])
def test_linear_adds_the_bias_before_it_rounds(gpu, m, n, k):
    # Row 0's outputs are what the bias, its rounded products negated, leaves of them: 0 if the
    # product were rounded before the addition.
    announce(f"bias {m} x {n} x {k}")
    codes, scales, weight, weight_scales, _ = (None if t is None else t.to(gpu) for t in operands(m, n, k, None, 17))
    sums = (codes[:1].double() @ weight.double().t())[0]
    product = (sums.float() * scales[0]).double() * weight_scales.double()  # exact: 24 x 24 bits
    bias = -product.float()
    y = backends.hip_linear_q8(codes, scales, weight, weight_scales, bias, output_dtype=torch.float32)
    want = product + bias.double()  # exact, and of at most 24 bits: fp32 holds it
    assert torch.equal(y[0].double(), want) and (want != 0).any()


def test_codes_of_the_norm_that_rounds_twice(gpu):
    # As documented: hip_rms_norm in Qwen2's order, then its codes.
    announce("norm in Qwen2's order")
    x, w = rows_of(40, 896, torch.bfloat16, 1), (torch.rand(896, generator=generator(2)) + 0.5).bfloat16()
    normed = backends.hip_rms_norm(x.to(gpu), w.to(gpu), epsilon=1e-6, round_before_weight=True)
    h = x.float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)
    # Two roundings to bf16, and fp32's in front of them.
    want = (h * rstd).bfloat16() * w
    assert ((normed.cpu().double() - want.double()).abs() <= want.double().abs() * 2.0**-7 * 1.01).all()
    check_rows(*backends.hip_quantize_q8(normed), normed.cpu().double())


@pytest.mark.parametrize("m,n,kernel", [(1, 40, "rows"), (100, 40, "stream"), (300, 9728, "stream"),
                                        (4096, 4096, "turns")])
def test_longest_aligned_sums(gpu, m, n, kernel):
    # The largest K that 16 divides: 1024 k-tiles, the last of them cut.
    k = 131056
    announce(f"longest aligned sums {m} x {n}")
    codes = torch.full((m, k), -128, dtype=torch.int8, device=gpu)
    weight = torch.full((n, k), -128, dtype=torch.int8, device=gpu)
    codes[-1], weight[-1, -16:] = 127, 1
    one = torch.ones(max(m, n), device=gpu)
    call = lambda: backends.hip_linear_q8(codes, one[:m], weight, one[:n], output_dtype=torch.float32)  # noqa: E731
    assert [name for name, _, _ in captured_kernels(call)] == [kernel]
    left = torch.full((m, 1), -128.0, dtype=torch.float64, device=gpu)
    left[-1] = 127.0
    right = torch.full((1, n), -128.0 * k, dtype=torch.float64, device=gpu)
    right[0, -1] = -128.0 * (k - 16) + 16
    assert torch.equal(call(), (left @ right).float())


# Row strides of the codes and of the outputs (elements): at the end of what 32-bit offsets
# within a 64-row tile reach, and past it.
@pytest.mark.parametrize("dtype,m,x_rs,y_rs,kernel", [
    (torch.bfloat16, 70, 2**25 - 2**15, 192, "stream"), (torch.bfloat16, 70, 2**25, 192, "tile"),
    (torch.bfloat16, 70, 320, 2**24 - 2**14, "stream"), (torch.bfloat16, 70, 320, 2**24, "tile"),
    (torch.float32, 70, 320, 2**23 - 2**13, "stream"), (torch.float32, 70, 320, 2**23, "tile"),
    (torch.float32, 20, 2**26 - 2**16, 2**25, "rows"), (torch.float32, 20, 2**26, 192, "tile"),
])
def test_linear_of_rows_far_apart(gpu, dtype, m, x_rs, y_rs, kernel):
    announce(f"rows {x_rs} and {y_rs} apart, {dtype}")
    n, k = (100, 320) if m > 32 else (192, 320)
    codes, scales, weight, weight_scales, bias = (t.to(gpu) for t in operands(m, n, k, dtype, 5))
    want = backends.hip_linear_q8(codes, scales, weight, weight_scales, bias, output_dtype=dtype)
    far = torch.empty((m - 1) * x_rs + k, dtype=torch.int8, device=gpu).as_strided((m, k), (x_rs, 1))
    far.copy_(codes)
    flat = torch.full((m * y_rs,), 7.0, dtype=dtype, device=gpu)
    call = lambda: _native.check(_native.library().slc_hip_linear_q8(  # noqa: E731
        far.data_ptr(), scales.data_ptr(), weight.data_ptr(), weight_scales.data_ptr(), bias.data_ptr(),
        flat.data_ptr(), _native.dtype_tag(dtype), m, n, k, x_rs, y_rs, _native.current_stream(gpu)),
        "slc_hip_linear_q8")
    assert [name for name, _, _ in captured_kernels(call)] == [kernel]
    call()
    out = flat.view(m, y_rs)
    assert_bitwise_equal(out[:, :n], want)
    assert (out[:, n:] == 7).all()

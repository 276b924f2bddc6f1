"""The 8-bit layer operators on the GPU against their definitions in 64 bits.

Tolerances.  A code is the nearest integer to q = 127 y / a; the kernel rounds y f once, f = 127 / a within half an ulp
(2^-24) and, for the norm, y and a times the row's rounded factor (three more), so |code - q| <= 1/2 + 127 * 5 * 2^-24.
The SwiGLU's y is within 8 ulps (exp2 1, its argument's compensation 1, the sum 1/2, the reciprocal 1, two products 1,
each doubled), so 127 * 2 * 8 * 2^-23.  A scale has the error of its row's maximum: 2^-24 twice for rows, the sum's for
the norm (at most 8 * 4 + 6 + 16 additions in a row of the order used: 64 * 2^-24, halved by the root, plus 5 roundings),
8 ulps for the SwiGLU.  A product's integer sum is exact: its conversion, the two scales' product, its use and two
additions round five times in fp32 (2^-24 of the terms' magnitudes each), and the output once (half its type's eps, and
half of fp16's smallest step)."""
from __future__ import annotations

import copy

import pytest
import torch

from triattention_amd.kernels import linear as Q

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = 2.0 ** -118
U = 2.0 ** -24


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def hidden(g, m, k, dtype, scale=1.0):
    x = torch.randn(m, k, generator=g, device=DEV) * torch.exp(torch.randn(m, 1, generator=g, device=DEV))
    x[:, :: max(1, k // 3)] *= 15
    return (x * scale).to(dtype)


def rand_codes(g, rows, k, low=-128, pad=None):
    """Codes inside a wider matrix whose other columns hold anything."""
    pad = -k % 16 if pad is None else pad
    x = torch.randint(low, 128, (rows, k + pad), generator=g, device=DEV, dtype=torch.int32).to(torch.int8)
    return x[:, :k]


def check_codes(codes, scales, y, delta, rel):
    """``codes`` and ``scales`` of the rows ``y`` (float64)."""
    top = y.abs().amax(-1).clamp(min=TINY)
    assert codes.dtype == torch.int8 and scales.dtype == torch.float32
    assert ((scales.double() - top / 127).abs() <= rel * top / 127).all()
    q = 127 * y / top.unsqueeze(-1)
    off = (codes.double() - q).abs()
    assert off.max() <= 0.5 + delta, off.max()


SHAPES = [(1, 1), (1, 3584), (3, 7), (5, 8), (4, 127), (9, 512), (2, 513), (7, 1025), (3, 2049), (6, 4096), (2, 4097),
          (2, 8200), (3, 18944), (2, 24577), (1, 32768), (2, 32777), (1000, 130)]


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_quantize_rows(module, m, k, dtype):
    x = hidden(gen(m * 7 + k), m, k, dtype)
    codes, scales = Q.quantize_rows(x)
    assert codes.shape == x.shape and scales.shape == (m,) and (m == 1 or codes.stride(0) % 16 == 0)
    check_codes(codes, scales, x.double(), 127 * 5 * U, 2 * U)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rms_norm_quant(module, m, k, dtype, residual):
    g = gen(m * 11 + k)
    x, r = hidden(g, m, k, dtype), hidden(g, m, k, dtype)
    w = (1 + 0.3 * torch.randn(k, generator=g, device=DEV)).to(dtype)
    codes, scales, h = Q.rms_norm_quant(x, w, 1e-6, residual=r if residual else None)
    if residual:
        assert h.dtype == dtype and torch.equal(h, (x.float() + r.float()).to(dtype))
    else:
        assert h is x
    hd = h.double()
    y = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    check_codes(codes, scales, y, 127 * 5 * U, (32 + 5) * U)


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_silu_mul_quant(module, m, k, dtype):
    g = gen(m * 13 + k)
    both = hidden(g, m, 2 * k, dtype)
    gate, up = both[:, :k], both[:, k:]
    codes, scales = Q.silu_mul_quant(gate, up)
    gd = gate.double()
    check_codes(codes, scales, gd * torch.sigmoid(gd) * up.double(), 127 * 16 * 2 * U, 16 * U)


@pytest.mark.parametrize("m,k", [(4200, 4100), (1100, 18945), (33000, 511), (520, 33001)])
def test_many_rows(module, m, k):
    """Millions of elements, rows at odd strides, and the memory around the outputs left alone."""
    g = gen(k)
    wide = hidden(g, m, k + 3, torch.bfloat16)
    x, w = wide[:, 1:1 + k], torch.ones(k, dtype=torch.bfloat16, device=DEV)
    codes = torch.full((m + 2, k + 5), 99, dtype=torch.int8, device=DEV)
    sums = torch.full((m + 2, k + 5), 7.0, dtype=torch.bfloat16, device=DEV)
    scales = torch.full((m + 2,), 5.0, device=DEV)
    module.rms_norm_quant(x, x, w, 1e-6, codes[1:-1, 2:2 + k], scales[1:-1], sums[1:-1, 2:2 + k])
    h = (x.float() * 2).bfloat16()
    assert torch.equal(sums[1:-1, 2:2 + k], h)
    hd = h.double()
    check_codes(codes[1:-1, 2:2 + k], scales[1:-1], hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6),
                127 * 5 * U, (32 + 5) * U)
    codes[1:-1, 2:2 + k], sums[1:-1, 2:2 + k], scales[1:-1] = 99, 7.0, 5.0
    assert (codes == 99).all() and (sums == 7.0).all() and (scales == 5.0).all()
    check_codes(*Q.quantize_rows(x), x.double(), 127 * 5 * U, 2 * U)


@pytest.mark.parametrize("k", [100, 512, 900, 2048, 2049, 4096, 9000, 18944, 30000, 33001])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_the_sum_may_take_its_operands_place(module, k, place):
    g = gen(k)
    for m in (1, 7):
        x, r = hidden(g, m, k, torch.bfloat16), hidden(g, m, k, torch.bfloat16)
        w = (1 + 0.3 * torch.randn(k, generator=g, device=DEV)).bfloat16()
        codes, scales, h = Q.rms_norm_quant(x, w, 1e-6, residual=r)
        c, s = torch.empty(m, k, dtype=torch.int8, device=DEV), torch.empty(m, device=DEV)
        module.rms_norm_quant(x, r, w, 1e-6, c, s, x if place == "x" else r)
        assert torch.equal(x if place == "x" else r, h) and torch.equal(c, codes) and torch.equal(s, scales)


def test_silu_of_far_negative_gates(module):
    # rows of negative gates alone: their own scale, down to where exp overflows (values of 0)
    gate = torch.stack([torch.linspace(-b, -b / 2, 300, device=DEV) for b in (1.0, 20.0, 60.0, 87.0, 300.0, 3e38)])
    up = torch.full_like(gate, 3.0)
    codes, scales = Q.silu_mul_quant(gate, up)
    gd = gate.double()
    y = gd * torch.sigmoid(gd) * 3
    check_codes(codes[:4], scales[:4], y[:4], 127 * 16 * 2 * U, 16 * U)
    assert torch.isfinite(scales).all() and (codes[5] == 0).all()


def test_rows_in_more_dimensions_and_views(module):
    g = gen(5)
    x = hidden(g, 2 * 3 * 5, 40, torch.bfloat16).view(2, 3, 5, 40)
    codes, scales = Q.quantize_rows(x)
    flat = Q.quantize_rows(x.reshape(30, 40))
    assert codes.shape == x.shape and scales.shape == (2, 3, 5)
    assert torch.equal(codes.reshape(30, 40), flat[0]) and torch.equal(scales.reshape(30), flat[1])
    one = Q.quantize_rows(x[0, 0, 0])
    assert one[0].shape == (40,) and one[1].shape == () and torch.equal(one[0], flat[0][0])
    wide = hidden(g, 9, 101, torch.float16)
    for view in (wide[:, 1:], wide[::2, 3:90], wide[4:5].expand(6, 101)):
        got = Q.quantize_rows(view)
        want = Q.quantize_rows(view.contiguous())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(RuntimeError, match="one stride"):
        Q.quantize_rows(x.transpose(0, 1))
    with pytest.raises(RuntimeError, match="contiguous features"):
        Q.quantize_rows(wide.t())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("k", [5, 600, 5000, 40000])
def test_rows_without_a_quantization(module, k, dtype):
    """Zero rows and rows with an infinity or a NaN, beside ordinary ones."""
    x = hidden(gen(k), 6, k, dtype)
    x[1] = 0
    x[2, k // 2] = float("inf")
    x[3, k - 1] = float("nan")
    x[4, 0] = float("-inf")
    w = torch.ones(k, dtype=dtype, device=DEV)
    ones = torch.ones_like(x)
    for codes, scales in (Q.quantize_rows(x), Q.rms_norm_quant(x, w, 1e-6)[:2], Q.silu_mul_quant(ones, x),
                          Q.rms_norm_quant(x, w, 1e-6, residual=torch.zeros_like(x))[:2]):
        assert torch.isnan(scales[2:5]).all() and torch.isfinite(scales[[0, 1, 5]]).all()
        assert (codes[1:5] == 0).all() and codes[0].abs().max() == 127 and codes[5].abs().max() == 127
        assert scales[1] > 0
    out = Q.int8_linear(*Q.quantize_rows(x), *Q.quantize_rows(hidden(gen(1), 20, k, dtype)))
    assert torch.isnan(out[2:5]).all() and torch.isfinite(out[[0, 1, 5]]).all() and (out[1] == 0).all()


def test_extreme_magnitudes(module):
    x = torch.tensor([[1e-44, -3e-40, 0.0], [1e-37, 1e-36, -1e-36], [3e38, -1e38, 1.0], [1e-30, 2e-30, 0.0]], device=DEV)
    codes, scales = Q.quantize_rows(x)
    check_codes(codes, scales, x.double(), 127 * 5 * U, 2 * U)
    # ties go to the even code: a = 127 makes the quotient the value
    t = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5]], device=DEV)
    assert Q.quantize_rows(t)[0].tolist() == [[127, 0, 2, 2, 0, -2, -2, 126]]


# ------------------------------------------------------------------ products
def check_linear(x, xs, w, ws, bias, residual, dtype, out):
    acc = x.double().cpu() @ w.double().cpu().t()
    y = acc * xs.double().cpu()[:, None] * ws.double().cpu()
    size = y.abs()
    for extra in (bias, residual):
        if extra is not None:
            y = y + extra.double().cpu()
            size = size + extra.double().cpu().abs()
    tol = 5 * U * size + torch.finfo(dtype).eps / 2 * (y.abs() + 5 * U * size)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    off = (out.double().cpu() - y).abs()
    assert out.dtype == dtype and out.shape == y.shape
    assert (off <= tol).all(), (off - tol).max()


def operands(seed, m, n, k, dtype, bias, residual):
    g = gen(seed)
    x, w = rand_codes(g, m, k), rand_codes(g, n, k)
    xs = torch.rand(m, generator=g, device=DEV) * 0.01
    ws = torch.rand(n, generator=g, device=DEV) * 0.01
    b = torch.randn(n, generator=g, device=DEV).to(dtype) if bias else None
    r = torch.randn(m, n, generator=g, device=DEV).to(dtype) if residual else None
    return x, xs, w, ws, b, r


# every form at its edges: token counts around the forms' limits, sums that end inside a 16-byte chunk, a step and a split
LINEAR = [(1, 1, 1), (1, 5, 15), (1, 4608, 3584), (2, 17, 16), (3, 64, 100), (4, 100, 1000), (5, 9, 127), (8, 513, 2049),
          (9, 1, 129), (9, 64, 128), (16, 63, 1000), (16, 200, 8192), (17, 65, 257), (32, 100, 4100), (33, 64, 64),
          (33, 40, 30000), (64, 130, 1), (64, 3, 2048), (65, 128, 100), (100, 300, 4097), (129, 127, 513), (257, 200, 384),
          (300, 1000, 640), (513, 2, 255), (2, 300, 131071), (70, 40, 20001),
          # few rows, where waves share K: fewer steps than waves, as many, one more; channels that end inside a block
          (1, 1283, 5120), (1, 20001, 300), (2, 20010, 1025), (3, 8192, 1000), (4, 30, 128), (7, 4611, 1024), (8, 700, 12000),
          (12, 20001, 640), (16, 9, 130), (16, 5120, 1152), (20, 5123, 1280), (24, 2000, 2048), (31, 513, 3584), (32, 17, 40),
          (17, 20001, 513), (30, 1000, 30001)]


@pytest.mark.parametrize("m,n,k", LINEAR)
def test_int8_linear(module, m, n, k):
    for i, dtype in enumerate(TYPES):
        bias, residual = (i + m) % 2 == 0, (i + n) % 2 == 0
        x, xs, w, ws, b, r = operands(m + n + k + i, m, n, k, dtype, bias, residual)
        out = Q.int8_linear(x, xs, w, ws, bias=b, residual=r, out_dtype=dtype)
        check_linear(x, xs, w, ws, b, r, dtype, out)


@pytest.mark.parametrize("m,n,k", [(2048, 4100, 300), (4100, 4097, 129), (8192, 2304, 256)])
def test_int8_linear_many_tiles(module, m, n, k):
    x, xs, w, ws, b, r = operands(m, m, n, k, torch.bfloat16, True, True)
    check_linear(x, xs, w, ws, b, r, torch.bfloat16, Q.int8_linear(x, xs, w, ws, b, r))


@pytest.mark.parametrize("m,n,k", [(1, 12500, 4000), (2, 12501, 4001), (3, 40001, 2600), (16, 30003, 3400), (17, 40001, 2600),
                                   (32, 30003, 3400)])
def test_few_rows_of_many_weights(module, m, n, k):
    """Products whose weights are loaded past the caches, and short of that."""
    x, xs, w, ws, b, r = operands(m, m, n, k, torch.bfloat16, True, True)
    check_linear(x, xs, w, ws, b, r, torch.bfloat16, Q.int8_linear(x, xs, w, ws, b, r))


@pytest.mark.parametrize("k", [64, 128, 160, 256, 384, 512, 640, 700])
@pytest.mark.parametrize("m,n", [(5, 300), (20, 2000), (40, 9000), (100, 4608), (300, 3000), (700, 5000), (1500, 6100),
                                 (4097, 5889)])
def test_few_steps(module, m, n, k):
    """Every tile form with fewer steps than buffers, as many, and a few more (sums below 2^24: fp32 products are exact)."""
    x, xs, w, ws, b, r = operands(m + k, m, n, k, torch.bfloat16, True, True)
    y = (x.float() @ w.float().t()).double()
    assert torch.equal(y, y.round())
    y = y * xs.double()[:, None] * ws.double()
    size = y.abs() + b.double().abs() + r.double().abs()
    y = y + b.double() + r.double()
    tol = 5 * U * size + torch.finfo(torch.bfloat16).eps / 2 * (y.abs() + 5 * U * size)
    assert ((Q.int8_linear(x, xs, w, ws, b, r).double() - y).abs() <= tol).all()


@pytest.mark.parametrize("m", [1, 4, 16, 40, 200])
def test_largest_sums(module, m):
    """Codes of -128 everywhere, at the longest K: sums of 2^31 - 16384."""
    k = 131071
    x = torch.full((m, k + 1), -128, dtype=torch.int8, device=DEV)[:, :k]
    w = torch.full((3, k + 1), -128, dtype=torch.int8, device=DEV)[:, :k]
    one = torch.ones
    out = Q.int8_linear(x, one(m, device=DEV), w, one(3, device=DEV), out_dtype=torch.float32)
    assert (out == float(128 * 128 * k)).all()


@pytest.mark.parametrize("m", [1, 6, 16, 33, 100, 600])
def test_nothing_outside_the_output_is_written(module, m):
    n, k = 77, 3000
    x, xs, w, ws, b, r = operands(m, m, n, k, torch.bfloat16, True, True)
    field = torch.full((m + 2, n + 9), 7.0, dtype=torch.bfloat16, device=DEV)
    out = field[1:-1, 4:4 + n]
    size = module.int8_linear_workspace(m, n, k, x.device)
    module.int8_linear(x, xs, w, ws, b, r, out, torch.empty(size, dtype=torch.uint8, device=DEV))
    check_linear(x, xs, w, ws, b, r, torch.bfloat16, out)
    field[1:-1, 4:4 + n] = 7.0
    assert (field == 7.0).all()


def test_the_residual_may_be_the_output(module):
    for m in (1, 20, 300):
        x, xs, w, ws, b, r = operands(m, m, 200, 4000, torch.bfloat16, True, True)
        want = Q.int8_linear(x, xs, w, ws, b, r)
        size = module.int8_linear_workspace(m, 200, 4000, x.device)
        module.int8_linear(x, xs, w, ws, b, r, r, torch.empty(size, dtype=torch.uint8, device=DEV))
        assert torch.equal(r, want)


def test_strided_and_repeated_codes(module):
    g = gen(3)
    big = rand_codes(g, 40, 256, pad=0)
    ws = torch.rand(40, generator=g, device=DEV)
    for rows in (big[::3, 16:200], big[:1].expand(20, 256)[:, :130], big[5:6, :100]):
        w = big[:, 32:32 + rows.size(1)]
        xs = torch.rand(rows.size(0), generator=g, device=DEV)
        out = Q.int8_linear(rows, xs, w, ws, out_dtype=torch.float32)
        check_linear(rows, xs, w, ws, None, None, torch.float32, out)


def test_a_layer_moved_and_copied(module):
    """Weights of 100 input channels (rows padded to 112 bytes) through the host and a deep copy."""
    torch.manual_seed(5)
    layer = torch.nn.Linear(100, 24).to(DEV, torch.bfloat16)
    layer = Q.Int8Linear(layer)
    x = torch.randn(3, 100, dtype=torch.bfloat16, device=DEV)
    with torch.no_grad():
        want = layer(x)
        assert torch.equal(copy.deepcopy(layer)(x), want)
        assert torch.equal(layer.cpu().to(DEV)(x), want)


def test_offsets_past_32_bits(module):
    """70,000 rows of 32,768: the last rows come out as they do alone (codes and integer sums are the same bits)."""
    m, k, tail = 70000, 32768, slice(-40, None)
    x = torch.empty(m, k, dtype=torch.bfloat16, device=DEV).normal_(generator=gen(9))
    codes, scales = Q.quantize_rows(x)
    for whole, alone in zip((codes, scales), Q.quantize_rows(x[tail])):
        assert torch.equal(whole[tail], alone)
    w = torch.ones(k, dtype=torch.bfloat16, device=DEV)
    for whole, alone in zip(Q.rms_norm_quant(x, w, 1e-6, residual=x), Q.rms_norm_quant(x[tail], w, 1e-6, residual=x[tail])):
        assert torch.equal(whole[tail], alone)
    for whole, alone in zip(Q.silu_mul_quant(x, x), Q.silu_mul_quant(x[tail], x[tail])):
        assert torch.equal(whole[tail], alone)
    del x, whole, alone
    # codes, then weights, then outputs and residual of more than 2^31 elements
    out = Q.int8_linear(codes, scales, codes[:300], scales[:300])
    assert torch.equal(out[tail], Q.int8_linear(codes[tail], scales[tail], codes[:300], scales[:300]))
    for rows in (1, 8, 32, 300):
        out = Q.int8_linear(codes[:rows], scales[:rows], codes, scales)
        assert torch.equal(out[:, tail], Q.int8_linear(codes[:rows], scales[:rows], codes[tail], scales[tail]))
    few = codes[:, :128]
    out = Q.int8_linear(few, scales, few[:k], scales[:k])
    assert torch.equal(out[tail], Q.int8_linear(few[tail], scales[tail], few[:k], scales[:k]))
    out = Q.int8_linear(few, scales, few[:k], scales[:k], residual=out)
    assert torch.equal(out[tail, :100], Q.int8_linear(few[tail], scales[tail], few[:100], scales[:100],
                                                      residual=Q.int8_linear(few[tail], scales[tail], few[:100], scales[:100])))


def test_no_rows(module):
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    codes, scales = Q.quantize_rows(x)
    assert codes.shape == (0, 64) and scales.shape == (0,)
    assert Q.rms_norm_quant(x, x.new_ones(64), 1e-6, residual=x)[2].shape == (0, 64)
    assert Q.silu_mul_quant(x, x)[0].shape == (0, 64)
    w = torch.ones(5, 64, dtype=torch.int8, device=DEV)
    assert Q.int8_linear(codes, scales, w, torch.ones(5, device=DEV)).shape == (0, 5)
    assert Q.int8_linear(codes.view(3, 0, 64), scales.view(3, 0), w, torch.ones(5, device=DEV)).shape == (3, 0, 5)


def mlp(x, r, w, up8, down8, keep=None):
    codes, scales, h = Q.rms_norm_quant(x, w, 1e-6, residual=r)
    both = Q.int8_linear(codes, scales, *up8)
    half = both.size(-1) // 2
    inner, inner_scales = Q.silu_mul_quant(both[..., :half], both[..., half:])
    if keep is not None:
        keep += [codes, scales, h, both, inner, inner_scales]
    return Q.int8_linear(inner, inner_scales, *down8, residual=h)


@pytest.mark.parametrize("m", [1, 12, 150])
def test_a_layer_together_eager_and_captured(module, m):
    """Norm, fused projection, SwiGLU, down projection with the residual: each step against 64 bits on what the step
    before gave it; and a captured pass replayed on new inputs, eager work between."""
    g = gen(m)
    d, f = 512, 1000
    w = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).bfloat16()
    up = (torch.randn(2 * f, d, generator=g, device=DEV) * d ** -0.5).bfloat16()
    down = (torch.randn(d, f, generator=g, device=DEV) * f ** -0.5).bfloat16()
    up8, down8 = Q.quantize_rows(up), Q.quantize_rows(down)
    xs = [hidden(g, m, d, torch.bfloat16) for _ in range(3)]
    r = hidden(g, m, d, torch.bfloat16)
    eager = []
    for x in xs:
        steps = []
        eager.append(mlp(x, r, w, up8, down8, steps))
        codes, scales, h, both, inner, inner_scales = steps
        assert torch.equal(h, (x.float() + r.float()).bfloat16())
        hd = h.double()
        check_codes(codes, scales, hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6) * w.double(),
                    127 * 5 * U, (32 + 5) * U)
        check_linear(codes, scales, *up8, None, None, torch.bfloat16, both)
        gd, ud = both[:, :f].double(), both[:, f:].double()
        check_codes(inner, inner_scales, gd * torch.sigmoid(gd) * ud, 127 * 16 * 2 * U, 16 * U)
        check_linear(inner, inner_scales, *down8, None, h, torch.bfloat16, eager[-1])
    buf = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlp(buf, r, w, up8, down8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(buf, r, w, up8, down8)
    for turn in range(2):
        for x, want in zip(xs, eager):
            buf.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert torch.equal(mlp(x, r, w, up8, down8), want)


def test_two_streams_at_once(module):
    """Products split over K take workspaces of their own: two streams' calls do not share one."""
    sets = [operands(s, 100, 300, 8192, torch.float32, True, False) for s in (1, 2)]
    want = [Q.int8_linear(x, xs, w, ws, b, out_dtype=torch.float32) for x, xs, w, ws, b, _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, xs, w, ws, b, _ = sets[i]
                got[i].append(Q.int8_linear(x, xs, w, ws, b, out_dtype=torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_refusals(module):
    g = gen(0)
    x, xs, w, ws, _, _ = operands(0, 20, 30, 100, torch.bfloat16, False, False)
    bad = [dict(codes=x.float()), dict(weight=w.int()), dict(weight=w[:, :50]), dict(scales=xs[:5]),
           dict(weight_scales=ws[:3]), dict(scales=xs.double()), dict(bias=torch.ones(30, device=DEV)),
           dict(bias=torch.ones(29, device=DEV).bfloat16()), dict(residual=torch.ones(20, 29, device=DEV).bfloat16()),
           dict(residual=torch.ones(20, 30, device=DEV)), dict(out_dtype=torch.float64), dict(weight=w.cpu()),
           dict(codes=torch.ones(20, 100, dtype=torch.int8, device=DEV)),   # rows at 100 bytes
           dict(codes=rand_codes(g, 20, 160, pad=0)[:, 1:101]),               # rows off the 16 bytes
           dict(codes=rand_codes(g, 100, 20).t())]
    for change in bad:
        call = dict(codes=x, scales=xs, weight=w, weight_scales=ws) | change
        with pytest.raises((RuntimeError, ValueError)):
            Q.int8_linear(**call)
    long = torch.ones(2, 131072, dtype=torch.int8, device=DEV)
    with pytest.raises(RuntimeError, match="at most 131071"):
        Q.int8_linear(long, torch.ones(2, device=DEV), long, torch.ones(2, device=DEV))
    h = torch.ones(3, 64, device=DEV, dtype=torch.bfloat16)
    for call in (lambda: Q.quantize_rows(h.double()), lambda: Q.quantize_rows(h.cpu()), lambda: Q.quantize_rows(h[:, :0]),
                 lambda: Q.rms_norm_quant(h, h[0].float(), 1e-6), lambda: Q.rms_norm_quant(h, h[0], 0.0),
                 lambda: Q.rms_norm_quant(h, h[0], float("nan")), lambda: Q.rms_norm_quant(h, h[0, :5], 1e-6),
                 lambda: Q.rms_norm_quant(h, h[0], 1e-6, residual=h[:2]),
                 lambda: Q.rms_norm_quant(h, h[0], 1e-6, residual=h.float()),
                 lambda: Q.silu_mul_quant(h, h[:, :32]), lambda: Q.silu_mul_quant(h, h.float()),
                 lambda: Q.quantize_rows(h.clone().requires_grad_())):
        with pytest.raises((RuntimeError, ValueError)):
            call()

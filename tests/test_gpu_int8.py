"""8-bit projections on the GPU against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import solvedelta_b200 as sd
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu
BF16_EPS, F32_EPS = 2.0 ** -7, 2.0 ** -23


def _rows(rows, width, seed, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, width, generator=gen, device="cuda")
    x[:, :: max(1, width // 3)] *= 6
    return x.to(dtype)


def _weight(columns, width, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed)
    return sd.quantize_rows(torch.randn(columns, width, generator=gen, device="cuda") / width ** 0.5)


def _check(y, q, scale, weight, weight_scale, bias=None, swiglu=False):
    want, size = ref.projection(q, scale, ref.as64(weight), ref.as64(weight_scale), None if bias is None else ref.as64(bias))
    want, bound = ref.projection_bound(want, size, BF16_EPS if y.dtype == torch.bfloat16 else F32_EPS, swiglu)
    got = ref.as64(y).reshape(want.shape)
    assert (np.abs(got - want) <= bound).all(), float(np.max(np.abs(got - want) / bound))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("rows,width", ((1, 1), (3, 7), (2, 16), (5, 130), (4, 1024), (7, 2049), (2, 8192), (1, 40001)))
def test_quantized_rows_are_the_nearest_whole_numbers(rows, width, dtype):
    x = _rows(rows, width, rows + width, dtype)
    q, scale = sd.quantize_rows(x)
    want, want_scale = ref.quantize(ref.as64(x))
    assert q.shape == x.shape and q.dtype == torch.int8 and q.stride(0) % 16 == 0
    assert np.array_equal(q.cpu().numpy(), want) and np.array_equal(ref.as64(scale), want_scale)


def test_halves_go_to_the_even_neighbour():
    # 127 x / 254 = x / 2: every odd entry is a half
    x = torch.arange(-254, 255, device="cuda").float()
    for rows in (x.to(torch.bfloat16)[None], x[None] * 2.0 ** -20, x[None] * 2.0 ** 90, x[None] * 2.0 ** -120):
        q, _ = sd.quantize_rows(rows)
        assert np.array_equal(q[0].cpu().numpy(), np.rint(np.arange(-254, 255) / 2))
    # and next to a half: one step of FP32 to either side decides
    half = torch.tensor([254.0, 3.0, np.nextafter(np.float32(3), np.float32(4)), np.nextafter(np.float32(3), np.float32(2)),
                         -5.0, np.nextafter(np.float32(-5), np.float32(-6)), np.nextafter(np.float32(-5), np.float32(-4))],
                        device="cuda", dtype=torch.float32)
    assert sd.quantize_rows(half)[0].tolist() == [127, 2, 2, 1, -2, -3, -2]
    odd = torch.tensor([3.0e-3, 1e-3, -1.7e-3, 2.9999e-3], device="cuda") * 0.37
    want, _ = ref.quantize(ref.as64(odd[None]))
    assert sd.quantize_rows(odd)[0].tolist() == want[0].tolist()


def test_rows_of_zeros_small_large_and_infinite_entries():
    x = torch.zeros(7, 33, device="cuda")
    x[1, 5], x[1, 6] = 1e-42, -3e-43          # below the smallest normal number
    x[2] = torch.linspace(-3.0e38, 3.0e38, 33, device="cuda")
    x[3, 2], x[4, 7], x[5, 0] = float("inf"), float("-inf"), float("nan")
    x[6, 1] = 2e-31
    q, scale = sd.quantize_rows(x)
    want, want_scale = ref.quantize(ref.as64(x))
    assert np.array_equal(q.cpu().numpy(), want)
    assert np.array_equal(ref.as64(scale), want_scale, equal_nan=True)
    assert scale[0] == 0 and torch.isnan(scale[3:6]).all()
    weight, weight_scale = _weight(40, 33, 1)
    y = sd.int8_linear(x, weight, weight_scale, out_dtype=torch.float32)
    assert torch.isnan(y[3:6]).all() and (y[0] == 0).all() and torch.isfinite(y[[0, 1, 6]]).all()


def test_quantized_rows_of_strided_and_unaligned_inputs():
    base = _rows(12, 200, 3)
    for x in (base[:, 1:131], base[::2], base.t(), base[3:4, 5:], base.view(3, 4, 200)[:, 1:3], base[:1].expand(5, 200)):
        q, scale = sd.quantize_rows(x)
        want, want_scale = ref.quantize(ref.as64(x))
        assert np.array_equal(q.cpu().numpy(), want) and np.array_equal(ref.as64(scale), want_scale)
    q, scale = sd.quantize_rows(base[0])
    assert q.shape == (200,) and scale.shape == ()
    q, scale = sd.quantize_rows(base[:0])
    assert q.shape == (0, 200) and scale.shape == (0,)


# few rows (one launch, quantised in it or before it), tiles of every width, ragged in every direction, sums of one entry
SHAPES = ((1, 1, 1), (1, 64, 8), (1, 1024, 5632), (2, 100, 33), (3, 4100, 65), (8, 1024, 2368), (9, 1500, 77), (16, 2816, 1024),
          (17, 2816, 300), (32, 5000, 48), (32, 16384, 17), (33, 64, 64), (77, 1531, 301), (128, 128, 256), (129, 384, 255), (300, 1040, 1000),
          (1000, 72, 4096), (513, 2000, 4744), (2, 131072, 24), (40, 131072, 9))


@pytest.mark.parametrize("rows,width,columns", SHAPES)
def test_projection(rows, width, columns):
    x = _rows(rows, width, rows)
    weight, weight_scale = _weight(columns, width, columns)
    q, scale = ref.quantize(ref.as64(x))
    y = sd.int8_linear(x, weight, weight_scale)
    assert y.dtype == torch.bfloat16 and y.shape == (rows, columns)
    _check(y, q, scale, weight, weight_scale)
    bias = torch.randn(columns, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    y = sd.int8_linear(x, weight, weight_scale, bias, out_dtype=torch.float32)
    _check(y, q, scale, weight, weight_scale, bias)
    # in two steps: the same kernels on the same integers, or other kernels with the same exact sums
    again = sd.int8_matmul(*sd.quantize_rows(x), weight, weight_scale, bias, out_dtype=torch.float32)
    assert torch.equal(y, again)


@pytest.mark.parametrize("rows,width,columns", ((1, 1024, 5632), (1, 3, 2), (5, 333, 34), (16, 1024, 512), (31, 2000, 1130), (64, 1024, 5632),
                                                (130, 777, 1002), (1024, 512, 9000), (2048, 256, 5632)))
@pytest.mark.parametrize("out", (torch.bfloat16, torch.float32))
def test_gated_projection(rows, width, columns, out):
    x = _rows(rows, width, rows)
    weight, weight_scale = _weight(columns, width, columns)
    bias = torch.randn(columns, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(torch.bfloat16)
    q, scale = ref.quantize(ref.as64(x))
    for b in (None, bias):
        y = sd.int8_linear(x, weight, weight_scale, b, swiglu=True, out_dtype=out)
        assert y.shape == (rows, columns // 2) and y.dtype == out
        _check(y, q, scale, weight, weight_scale, b, swiglu=True)


def test_gated_projection_of_large_gates():
    """silu saturates to its argument and to zero: no overflow of the exponential reaches the result."""
    q = torch.tensor([[127], [-127], [1]], dtype=torch.int8, device="cuda")
    weight = torch.ones(32, 1, dtype=torch.int8, device="cuda")
    for top in (0.7, 2.0, 80.0):
        scale = torch.full((3,), top, device="cuda")
        ones = torch.ones(32, device="cuda")
        y = sd.int8_matmul(q, scale, weight, ones, swiglu=True, out_dtype=torch.float32)
        _check(y, ref.as64(q), ref.as64(scale), weight, ones, swiglu=True)
        assert torch.isfinite(y).all()


@pytest.mark.parametrize("rows", (2, 200))
def test_extreme_integers_sum_exactly(rows):
    """The longest sums of the largest products: 127 * 127 * 131072 < 2^31, and -128 as a caller may hold it."""
    width = 131072
    q = torch.full((rows, width), 127, dtype=torch.int8, device="cuda")
    weight = torch.full((16, width), -127, dtype=torch.int8, device="cuda")
    weight[1] = 127
    one = torch.ones(rows, device="cuda")
    y = sd.int8_matmul(q, one, weight, torch.ones(16, device="cuda"), out_dtype=torch.float32)
    assert (y[:, 1] == float(127 * 127 * width)).all() and (y[:, 0] == -float(127 * 127 * width)).all()
    short = torch.full((rows, 100), -128, dtype=torch.int8, device="cuda")
    y = sd.int8_matmul(short, one, torch.full((3, 100), -128, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"),
                       out_dtype=torch.float32)
    assert (y == 128.0 * 128 * 100).all()


@pytest.mark.parametrize("rows", (3, 50))
def test_layouts_that_are_not_the_quantizers_own(rows):
    """Odd strides, odd starts, transposed and expanded operands, storage that ends with the last entry, leading axes."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    store = torch.randint(-127, 128, (rows + 40, 107), generator=gen, device="cuda").to(torch.int8)
    scale, weight_scale = torch.rand(rows, generator=gen, device="cuda"), torch.rand(24, generator=gen, device="cuda")
    for width in (96, 101, 107):
        q, weight = store[:rows, :width], store[rows:rows + 24, 107 - width:]
        y = sd.int8_matmul(q, scale, weight, weight_scale, out_dtype=torch.float32)
        _check(y, ref.as64(q), ref.as64(scale), weight, weight_scale)
    q, weight = store[:rows, :rows], store[:rows, :24].t()
    y = sd.int8_matmul(q, scale, weight, weight_scale, out_dtype=torch.float32)
    _check(y, ref.as64(q), ref.as64(scale), weight, weight_scale)
    tight = torch.randint(-127, 128, (24, 96), generator=gen, device="cuda").to(torch.int8)
    x = _rows(rows * 2, 96, 4).view(2, rows, 96).transpose(0, 1)
    y = sd.int8_linear(x, tight, weight_scale[:1].expand(24))
    assert y.shape == (rows, 2, 24)
    q, scale = ref.quantize(ref.as64(x).reshape(-1, 96))
    _check(y, q, scale, tight, weight_scale[:1].expand(24))
    assert sd.int8_linear(x[:0], tight, weight_scale).shape == (0, 2, 24)
    assert sd.int8_linear(x[0, 0], tight, weight_scale).shape == (24,)


@pytest.mark.parametrize("rows", (4, 300))
def test_bytes_behind_a_row_do_not_count(rows):
    """The padding of int8 rows may hold anything."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, weight = (torch.randint(-127, 128, (n, 112), generator=gen, device="cuda").to(torch.int8)[:, :99] for n in (rows, 40))
    scale, weight_scale = torch.rand(rows, device="cuda", generator=gen), torch.rand(40, device="cuda", generator=gen)
    y = sd.int8_matmul(q, scale, weight, weight_scale, out_dtype=torch.float32)
    _check(y, ref.as64(q), ref.as64(scale), weight, weight_scale)


@pytest.mark.parametrize("rows", (1, 12, 400))
def test_streams_and_graphs(rows):
    """Another stream than the default, and a captured call replayed on new inputs."""
    width, columns = 1024, 1536
    weight, weight_scale = _weight(columns, width, 3)
    x = _rows(rows, width, 1)
    want = sd.int8_linear(x, weight, weight_scale, swiglu=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sd.int8_linear(x, weight, weight_scale, swiglu=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    static = x.clone()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(sd.int8_linear(static, weight, weight_scale, swiglu=True))
    for seed in (1, 2, 3):
        static.copy_(_rows(rows, width, seed))
        fresh = sd.int8_linear(static, weight, weight_scale, swiglu=True)
        for graph in graphs:
            graph.replay()
        for out in outs:
            assert torch.equal(out, fresh)


def test_rows_do_not_depend_on_their_batch():
    weight, weight_scale = _weight(2816, 1024, 3)
    x = _rows(700, 1024, 1)
    whole = sd.int8_linear(x, weight, weight_scale, out_dtype=torch.float32)
    for lo, hi in ((0, 1), (5, 13), (100, 132), (300, 700)):
        assert torch.equal(sd.int8_linear(x[lo:hi], weight, weight_scale, out_dtype=torch.float32), whole[lo:hi])


def test_gradients_are_refused():
    weight, weight_scale = _weight(32, 64, 1)
    x = _rows(4, 64, 1).requires_grad_()
    with pytest.raises(RuntimeError, match="no reverse pass"):
        sd.int8_linear(x, weight, weight_scale)
    with torch.no_grad():
        sd.int8_linear(x, weight, weight_scale)
    sd.int8_linear(x.detach(), weight, weight_scale)


def test_refusals():
    weight, weight_scale = _weight(32, 64, 1)
    x = _rows(4, 64, 1)
    q, scale = sd.quantize_rows(x)
    with pytest.raises(ValueError, match="as long as"):
        sd.int8_linear(x[:, :60], weight, weight_scale)
    with pytest.raises(TypeError, match="BF16 or FP32"):
        sd.int8_linear(x.half(), weight, weight_scale)
    with pytest.raises(TypeError, match="int8 CUDA"):
        sd.int8_linear(x, weight.float(), weight_scale)
    with pytest.raises(TypeError, match="int8 CUDA"):
        sd.int8_matmul(x, scale, weight, weight_scale)
    with pytest.raises(ValueError, match="gate rows"):
        sd.int8_linear(x, weight[:31], weight_scale[:31], swiglu=True)
    with pytest.raises(ValueError, match="weight_scale must be"):
        sd.int8_linear(x, weight, weight_scale[:31])
    with pytest.raises(ValueError, match="scale must have"):
        sd.int8_matmul(q, scale[:3], weight, weight_scale)
    with pytest.raises(TypeError, match="out_dtype"):
        sd.int8_linear(x, weight, weight_scale, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="device of the rows"):
        sd.int8_linear(x, weight, weight_scale.cpu())
    with pytest.raises(ValueError, match="131072"):
        sd.quantize_rows(torch.zeros(1, 131073, device="cuda"))
    with pytest.raises(ValueError, match="bias must be"):
        sd.int8_linear(x, weight, weight_scale, weight_scale[:5])


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("largest", (2.0e36, 2.6e36, 2.69e36, 1e38, 3.0e38, 3.38e38))
def test_rows_of_very_large_finite_entries(largest, dtype):
    """Up to the end of FP32's range, halves and entries off a half in one group of eight."""
    gen = torch.Generator(device="cuda").manual_seed(int(largest / 1e35))
    shares = torch.tensor([1, .5, .9, .8953, -.3, .56, .77, .11], device="cuda")
    steps = torch.arange(1, 17, device="cuda") / 16
    x = torch.cat((shares, steps, -steps, 2 * torch.rand(512 - 40, generator=gen, device="cuda") - 1)) * largest
    x = torch.stack((x, x.roll(3), -x, x.flip(0))).to(dtype)
    assert torch.isfinite(x).all()
    want, want_scale = ref.quantize(ref.as64(x))
    q, scale = sd.quantize_rows(x)
    assert np.array_equal(q.cpu().numpy(), want) and np.array_equal(ref.as64(scale), want_scale)
    odd = sd.quantize_rows(x[:, 1:])[0]   # rows that start anywhere
    assert np.array_equal(odd.cpu().numpy(), ref.quantize(ref.as64(x[:, 1:]))[0])
    # one row quantised inside the product, four in front of it, many in tiles: the unit matrix shows the integers
    unit = torch.eye(512, dtype=torch.int8, device="cuda")
    ones = torch.ones(512, device="cuda")
    for rows in (x[:1], x, x.repeat(10, 1)):
        y = ref.as64(sd.int8_linear(rows, unit, ones, out_dtype=torch.float32))
        whole, unit_of = ref.quantize(ref.as64(rows))
        assert (np.abs(y - whole * unit_of[:, None]) <= 2.0 ** -24 * np.abs(whole) * unit_of[:, None]).all()


def test_forward_mode_tangents_are_refused():
    weight, weight_scale = _weight(32, 64, 1)
    x = _rows(4, 64, 1)
    q, scale = sd.quantize_rows(x)
    bias = torch.zeros(32, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = {name: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
                for name, t in (("x", x), ("scale", scale), ("weight_scale", weight_scale), ("bias", bias))}
        for call in (lambda: sd.int8_linear(dual["x"], weight, weight_scale), lambda: sd.int8_linear(x, weight, dual["weight_scale"]),
                     lambda: sd.int8_linear(x, weight, weight_scale, dual["bias"]), lambda: sd.int8_matmul(q, dual["scale"], weight, weight_scale),
                     lambda: sd.int8_gated_mlp(dual["x"], weight, weight_scale, None, weight[:, :16], weight_scale, None)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            sd.int8_linear(dual["x"], weight, weight_scale)
        sd.int8_linear(x, weight, weight_scale)


@pytest.mark.parametrize("rows,width,columns", ((1, 1024, 520), (3, 33, 40), (16, 300, 128), (40, 1000, 96), (130, 77, 301)))
def test_projection_of_fp32_rows(rows, width, columns):
    x = _rows(rows, width, rows, torch.float32)
    weight, weight_scale = _weight(columns, width, columns)
    for given in (x, torch.cat((x, x), dim=1)[:, 1:width + 1], x.t().contiguous().t()):
        q, scale = ref.quantize(ref.as64(given))
        for out in (torch.bfloat16, torch.float32):
            _check(sd.int8_linear(given, weight, weight_scale, out_dtype=out), q, scale, weight, weight_scale)
            if columns % 2 == 0:
                _check(sd.int8_linear(given, weight, weight_scale, swiglu=True, out_dtype=out), q, scale, weight, weight_scale, swiglu=True)

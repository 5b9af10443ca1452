"""Host-side behaviour of the serving operators (no GPU): what they refuse, through Python and through the C ABI."""
import ctypes

import pytest
import torch

import solvedelta_b200 as sd
from solvedelta_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    _lib.build()
    return _lib.load()


def test_struct_sizes_match_header():
    assert ctypes.sizeof(_lib.QuantizeRowsArgs) == 16 + 5 * 8
    assert ctypes.sizeof(_lib.Int8LinearArgs) == 8 + 6 * 4 + 11 * 8 + 8
    assert ctypes.sizeof(_lib.SampleTokensArgs) == 16 + 3 * 8 + 4 * 8 + 3 * 8 + 8 + 2 * 8


def test_entries_refuse_cpu_tensors():
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    q, scale, weight, weight_scale = torch.zeros(2, 32, dtype=torch.int8), torch.ones(2), torch.zeros(8, 32, dtype=torch.int8), torch.ones(8)
    with pytest.raises(TypeError, match="CUDA"):
        sd.quantize_rows(x)
    with pytest.raises(TypeError, match="CUDA"):
        sd.int8_linear(x, weight, weight_scale)
    with pytest.raises(TypeError, match="CUDA"):
        sd.int8_matmul(q, scale, weight, weight_scale)
    with pytest.raises(TypeError, match="CUDA"):
        sd.sample_tokens(x, torch.zeros(2))


def test_argument_errors_are_status_codes(lib):
    """Nothing of this reaches a device: the addresses are never read."""
    at = 4096   # aligned, not null
    assert lib.sd_quantize_rows(None, None) == -1
    assert lib.sd_int8_linear(None, None) == -1
    assert lib.sd_sample_tokens(None, None) == -1
    assert lib.sd_int8_linear_scratch_bytes(None) == 0

    def rows(**change):
        a = _lib.QuantizeRowsArgs(rows=3, K=100, x_type=_lib.BF16, x=at, x_stride=100, q=at, q_stride=112, scale=at)
        for name, value in change.items():
            setattr(a, name, value)
        return lib.sd_quantize_rows(ctypes.byref(a), None)

    assert [rows(q_stride=96), rows(q_stride=104), rows(q=at + 8), rows(x=None), rows(rows=0), rows(x_type=_lib.I8)] == [-1] * 6
    assert rows(K=131073, q_stride=131088) == -2

    def linear(**change):
        a = _lib.Int8LinearArgs(rows=64, N=8, K=100, x_type=_lib.I8, y_type=_lib.F32, x=at, x_stride=112, x_scale=at, weight=at,
                                weight_stride=112, weight_scale=at, y=at, y_stride=8)
        for name, value in change.items():
            setattr(a, name, value)
        return lib.sd_int8_linear(ctypes.byref(a), None)

    assert [linear(weight_stride=96), linear(weight=at + 4), linear(x_stride=100), linear(x=at + 1), linear(x_scale=None),
            linear(y_type=_lib.I8), linear(x_type=7), linear(N=7, swiglu=1), linear(K=0), linear(bias=at, bias_type=_lib.I8)] == [-1] * 10
    assert linear(K=131073, weight_stride=131088, x_stride=131088) == -2
    assert linear(N=0x7fffff01) == -2 and linear(rows=0x7fffff01) == -2
    assert linear(x_type=_lib.BF16, x_stride=100) == -3   # no room for the quantised rows

    def scratch(count, width, x_type):
        return lib.sd_int8_linear_scratch_bytes(ctypes.byref(_lib.Int8LinearArgs(rows=count, N=8, K=width, x_type=x_type, x=at, x_stride=width)))

    assert scratch(100, 100, _lib.BF16) >= 100 * 112 + 400 and scratch(100, 100, _lib.I8) == 0

    def sample(**change):
        a = _lib.SampleTokensArgs(rows=3, V=100, logits_type=_lib.F32, logits=at, stride=100, uniform=at, tokens=at)
        for name, value in change.items():
            setattr(a, name, value)
        return lib.sd_sample_tokens(ctypes.byref(a), None)

    assert [sample(logits=None), sample(V=0), sample(uniform=None), sample(logits_type=_lib.I8), sample(logits=at + 2)] == [-1] * 5
    assert sample(V=262145) == -2


def test_projections_that_do_more_than_their_product_are_refused():
    class Scaled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    hooked = torch.nn.Linear(16, 16)
    handle = hooked.register_forward_hook(lambda module, args, out: 2 * out)
    parametrised = torch.nn.utils.parametrizations.weight_norm(torch.nn.Linear(16, 16))
    replaced = torch.nn.Linear(16, 16)
    replaced.forward = lambda x: x
    for module in (Scaled(16, 16), hooked, parametrised, replaced):
        with pytest.raises(TypeError, match="plain nn.Linear"):
            sd.Int8Linear.from_linear(module)
    handle.remove()
    with pytest.raises(TypeError, match="CUDA"):   # plain again: what is refused now is the device
        sd.Int8Linear.from_linear(hooked)


def test_chunked_loss_refuses_whole_numbers():
    with pytest.raises(TypeError, match="weight must be"):
        sd.fixed_dense_linear_cross_entropy(torch.zeros(3, 16), torch.zeros(3, dtype=torch.long), torch.zeros(8, 16, dtype=torch.int8), total=3)

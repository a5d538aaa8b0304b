"""Refusals of the layers on features: they come before anything is launched, so
they need no device."""
import ctypes

import pytest
import torch

import ash
from ash import common


@pytest.fixture(scope="module")
def backend():
    if not isinstance(ash.core.backend, common._Backend):
        pytest.fail("libash_hip.so is not loaded")


X, W, B = torch.zeros(4, 6), torch.zeros(5, 6), torch.zeros(5)
Q = ash.QuantizedRows(torch.zeros(4, 6).to(torch.float8_e4m3fn), torch.ones(4))
QW = ash.QuantizedRows(torch.zeros(5, 6).to(torch.float8_e4m3fn), torch.ones(5))


@pytest.mark.parametrize("call,message", [
    (lambda: ash.linear(X, W), "HIP device"),
    (lambda: ash.linear(X, torch.zeros(5, 7)), "weight must be"),
    (lambda: ash.linear(X, torch.zeros(6)), "weight must be"),
    (lambda: ash.linear(torch.zeros(()), W), "weight must be"),
    (lambda: ash.linear(torch.zeros(4, 0), torch.zeros(5, 0)), "at least one feature"),
    (lambda: ash.linear(X.double(), W.double()), "float32, bfloat16 or float16"),
    (lambda: ash.linear(X.long(), W.long()), "float32, bfloat16 or float16"),
    (lambda: ash.linear(X, W.half()), "weight must be Float"),
    (lambda: ash.linear(X, W, activation="tanh"), "unknown activation"),
    (lambda: ash.linear(X, W, out_dtype=torch.float16), "type of the input"),
    (lambda: ash.linear(Q, W), "8-bit weight"),
    (lambda: ash.linear(X, QW), "8-bit weight"),
    (lambda: ash.linear(Q, QW), "HIP device"),
    (lambda: ash.linear(ash.QuantizedRows(X, Q.scales), QW), "float8_e4m3fn"),
    (lambda: ash.linear(ash.QuantizedRows(Q.data, torch.ones(5)), QW), "one float32 scale a row"),
    (lambda: ash.linear(ash.QuantizedRows(Q.data, torch.ones(4).double()), QW), "one float32 scale a row"),
    (lambda: ash.linear(Q, QW, out_dtype=torch.float64), "float32, bfloat16 or float16"),
    (lambda: ash.rms_norm(X), "HIP device"),
    (lambda: ash.rms_norm(X.double()), "float32, bfloat16 or float16"),
    (lambda: ash.rms_norm(torch.zeros(())), "rows of 1 to 16384"),
    (lambda: ash.rms_norm(torch.zeros(2, 0)), "rows of 1 to 16384"),
    (lambda: ash.rms_norm(torch.zeros(2, 16385)), "rows of 1 to 16384"),
    (lambda: ash.rms_norm(X, eps=-1.0), "eps"),
    (lambda: ash.QuantizedRows.of(X), "HIP device"),
    (lambda: ash.QuantizedRows.of(X.long()), "float32, bfloat16 or float16"),
])
def test_refusals(backend, call, message):
    with pytest.raises(RuntimeError, match=message):
        call()


def test_function_transforms_and_subclasses_are_refused(backend):
    class Sub(torch.Tensor):
        pass

    with pytest.raises(RuntimeError, match="plain tensors"):
        ash.linear(X.as_subclass(Sub), W)
    with pytest.raises(RuntimeError, match="plain tensors"):
        torch.func.vmap(lambda x: ash.rms_norm(x))(X)


def test_decoder_declares_itself():
    d = ash.FeatureDecoder(7, 3, width=20, blocks=2, activation="sine", scale=30.0)
    assert "width=20" in repr(d)
    assert sum(p.numel() for p in d.parameters()) == (7 * 20 + 20) + 4 * (20 * 20 + 20) + (20 * 3 + 3) + 3 * 20
    other = ash.FeatureDecoder(7, 3, width=20, blocks=2)
    other.load_state_dict(d.state_dict())
    assert all(torch.equal(p, q) for p, q in zip(d.parameters(), other.parameters()))
    with pytest.raises(ValueError, match="activation"):
        ash.FeatureDecoder(7, 3, activation="tanh")


def linear_args(lib, **changes):
    a = common._LinearArgs(input=4096, weight=4096, rows=2, in_features=3, out_features=4, input_stride=3,
                           activation_scale=1.0)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(rows=-1), "rows"), (dict(in_features=0), "features"), (dict(out_features=65537), "features"),
    (dict(rows=2**31), "rows"), (dict(dtype=1), "operands"), (dict(dtype=9), "operands"),
    (dict(out_dtype=2), "type of the output"), (dict(activation=6), "activation"), (dict(activation=-1), "activation"),
    (dict(activation_scale=0.0), "scale"), (dict(activation_scale=float("nan")), "scale"),
    (dict(activation_scale=float("inf")), "scale"), (dict(input=None), "null"), (dict(weight=None), "null"),
    (dict(input_stride=-1), "strides"), (dict(residual_stride=-1), "strides"),
    (dict(dtype=4, out_dtype=0), "null"), (dict(dtype=4, out_dtype=4), "type of the output"),
])
def test_the_c_abi_refuses(changes, message):
    lib = common.load_library()
    a = linear_args(lib, **changes)
    assert lib.ash_linear_forward(ctypes.byref(a), 4096, None, None) == 1
    assert message in lib.ash_last_error().decode()


def test_the_c_abi_refuses_missing_buffers():
    lib = common.load_library()
    a = linear_args(lib)
    assert lib.ash_linear_forward(None, 4096, None, None) == 1
    assert lib.ash_linear_forward(ctypes.byref(a), None, None, None) == 1
    assert lib.ash_linear_backward_input(ctypes.byref(a), None, None, None, 4096, None) == 1
    assert lib.ash_linear_backward_weight(ctypes.byref(a), 4096, None, None, None, None, 0, 0, 4096, None, 4096, 8, None) == 1
    assert "scratch" in lib.ash_last_error().decode()
    assert lib.ash_linear_backward_weight(ctypes.byref(a), 4096, None, None, None, None, 0, 1, 4096, None, 4096, 1 << 30, None) == 1
    assert lib.ash_linear_second(ctypes.byref(a), None, None, 0, None, 0, 4096, None, None) == 1
    assert lib.ash_linear_backward_weight_scratch_bytes(0, 3, 4, 0, 1) == 0
    a8 = linear_args(lib, dtype=4, input_scales=4096, weight_scales=4096)
    assert lib.ash_linear_forward(ctypes.byref(a8), 4096, 4096, None) == 1
    assert "no gradients" in lib.ash_last_error().decode()
    assert lib.ash_linear_second(ctypes.byref(a8), 4096, None, 0, None, 0, 4096, None, None) == 1
    for changes in (dict(rows=-1), dict(cols=0), dict(cols=16385), dict(dtype=1), dict(input=None), dict(output=None),
                    dict(input_stride=-1)):
        n = common._NormArgs(input=4096, output=4096, grad=4096, rows=2, cols=3, input_stride=3, normalise=1)
        for name, value in changes.items():
            setattr(n, name, value)
        assert lib.ash_norm_forward(ctypes.byref(n), None) == 1, changes
    n = common._NormArgs(input=4096, grad=4096, weight_out=4096, rows=2, cols=3, input_stride=3, normalise=1)
    assert lib.ash_norm_backward(ctypes.byref(n), None) == 1
    assert "scratch" in lib.ash_last_error().decode()
    assert lib.ash_norm_forward(None, None) == 1


def test_the_c_abi_refuses_what_the_narrow_and_the_scaled_gradients_do_not_take():
    lib = common.load_library()
    a = linear_args(lib)
    both = lambda a, grad=4096, gx=4096, gw=4096, scratch=4096, size=1 << 30, second=(None, None, None), stride=0: \
        lib.ash_linear_backward_both(ctypes.byref(a), grad, None, *second, stride, gx, gw, None, scratch, size, None)
    assert lib.ash_linear_backward_both_scratch_bytes(2, 3, 4, 0, 1) >= (3 * 4 + 4) * 4
    for sizes in ((0, 3, 4, 0, 1), (2, 65, 4, 0, 1), (2, 3, 65, 0, 1), (2, 3, 4, 4, 1), (2, 3, 4, 0, 0), (-1, 3, 4, 0, 1)):
        assert lib.ash_linear_backward_both_scratch_bytes(*sizes) == 0
    for bad in (dict(grad=None), dict(gx=None), dict(gw=None), dict(scratch=None), dict(size=8),
                dict(second=(4096, None, None)), dict(second=(4096, None, 4096), stride=-1)):
        assert both(a, **bad) == 1, bad
    for changes in (dict(in_features=65), dict(out_features=65), dict(rows=0), dict(dtype=4, out_dtype=0), dict(rows=-1)):
        assert both(linear_args(lib, **changes)) == 1, changes
    # what the output tells of the slope: of float32, of two activations
    for dtype, activation in ((0, 2), (0, 0), (0, 5), (2, 1), (3, 4)):
        assert not lib.ash_linear_slope_by_output(dtype, activation)
        bent = linear_args(lib, dtype=dtype, out_dtype=dtype, activation=activation, slope_is_output=1)
        assert lib.ash_linear_backward_input(ctypes.byref(bent), 4096, 4096, None, 4096, None) == 1
        assert "slope" in lib.ash_last_error().decode()
    assert lib.ash_linear_slope_by_output(0, 1) and lib.ash_linear_slope_by_output(0, 4)
    assert not lib.ash_linear_wants_scaled_gradient(1 << 20, 1024, 1024, 0)
    told = linear_args(lib, activation=1, slope_is_output=1)
    assert lib.ash_linear_scale_gradient(ctypes.byref(told), 4096, 4096, 4096, None) == 1
    for missing in range(3):
        buffers = [None if i == missing else 4096 for i in range(3)]
        assert lib.ash_linear_scale_gradient(ctypes.byref(a), *buffers, None) == 1
    assert lib.ash_linear_scale_gradient(None, 4096, 4096, 4096, None) == 1


def test_the_c_abi_refuses_strides_of_the_second_order():
    lib = common.load_library()
    a = linear_args(lib)
    assert lib.ash_linear_second(ctypes.byref(a), 4096, 4096, -1, None, 0, 4096, None, None) == 1
    assert lib.ash_linear_second(ctypes.byref(a), 4096, 4096, 3, 4096, -1, 4096, None, None) == 1
    assert lib.ash_linear_second(ctypes.byref(a), 4096, 4096, 3, None, 0, None, None, None) == 1
    assert lib.ash_linear_second(ctypes.byref(linear_args(lib, input_stride=-1)), 4096, 4096, 3, None, 0, 4096, None, None) == 1
    for call in (lib.ash_norm_backward, lib.ash_norm_second):
        n = common._NormArgs(input=4096, output=4096, rows=2, cols=3, input_stride=3, normalise=1)
        assert call(ctypes.byref(n), None) == 1   # no grad
        assert call(None, None) == 1

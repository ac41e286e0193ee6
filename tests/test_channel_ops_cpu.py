"""Host-side checks of the layer norm and MXFP4 operators: what is refused before anything is launched."""
import ctypes

import pytest
import torch

import deltacnn_b200 as dc
from deltacnn_b200 import _lib
from deltacnn_b200._lib import lib


def test_no_cpu_path():
    x = torch.randn(4, 64)
    for call in (lambda: dc.layer_norm(x), lambda: dc.mx4_quantize(x), lambda: dc.mx4_quantize_both(x), lambda: dc.mx4_linear(x, torch.randn(8, 64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    q = dc.MX4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), (4, 64))
    for call in (lambda: q.dequantize(), lambda: dc.mx4_matmul(q, q), lambda: dc.mx4_linear(x, q)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("data,scales,shape", [
    ((4, 31), (1, 1, 32, 4, 4), (4, 64)), ((4, 32), (1, 2, 32, 4, 4), (4, 64)), ((4, 32), (1, 1, 32, 4, 4), (4, 65)), ((4, 32), (1, 1, 32, 4, 4), (5, 64)),
    ((4, 0), (1, 0, 32, 4, 4), (4, 0)), ((129, 32), (1, 1, 32, 4, 4), (129, 64))])
def test_mx4_tensor_shapes_are_checked(data, scales, shape):
    with pytest.raises(RuntimeError, match="MX4Tensor"):
        dc.MX4Tensor(torch.zeros(data, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), shape)


def test_mx4_tensor_types_and_layout_are_checked():
    data, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)
    dc.MX4Tensor(data, scales, (4, 64))
    for d, s in ((data.int(), scales), (data, scales.float()), (torch.zeros(32, 4, dtype=torch.uint8).t(), scales)):
        with pytest.raises(RuntimeError, match="MX4Tensor"):
            dc.MX4Tensor(d, s, (4, 64))


def test_c_entry_points_refuse_bad_arguments():
    buf = (ctypes.c_uint8 * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256                      # never dereferenced: every call is refused first
    null, shape, dtype, align, space = 1, 4, 5, 3, 7
    f32, f16, bf16 = _lib.DC_F32, _lib.DC_F16, _lib.DC_BF16
    assert lib.dc_layer_norm(None, p, p, p, None, None, 1, 8, f32, f32, 1e-5, None) == null
    assert lib.dc_layer_norm(p, p, p, p, p, None, 1, 8, f32, f32, 1e-5, None) == null
    assert lib.dc_layer_norm(p, p, p, p, None, None, 1, 0, f32, f32, 1e-5, None) == shape
    assert lib.dc_layer_norm(p, p, p, p, None, None, 1, (1 << 30) + 1, f32, f32, 1e-5, None) == shape
    assert lib.dc_layer_norm(p, p, p, p, None, None, -1, 8, f32, f32, 1e-5, None) == shape
    assert lib.dc_layer_norm(p, p, p, p, None, None, 1, 8, 3, f32, 1e-5, None) == dtype
    assert lib.dc_layer_norm(p, p, p, p, None, None, 1, 8, f32, f16, 1e-5, None) == dtype
    assert lib.dc_layer_norm(p, p, p, p, None, None, 1, 8, f16, bf16, 1e-5, None) == dtype
    assert lib.dc_layer_norm(p, p, p, p, None, None, 0, 8, f32, f32, 1e-5, None) == 0
    assert lib.dc_layer_norm_backward(p, p, p, p, p, p, p, p, 1, 8, f32, f32, None, 0, None) == null
    assert lib.dc_layer_norm_backward(p, p, p, p, p, p, p, p, 1, 8, f32, f32, p, 8, None) == space
    assert lib.dc_layer_norm_backward(p, p, p, None, p, p, p, p, 1, 8, f32, f32, p, 1 << 20, None) == null
    assert lib.dc_layer_norm_backward(p, p, p, p, p, p, p, p, 1, 8, f32, f32, 20, 1 << 20, None) == align
    assert lib.dc_layer_norm_backward(p, p, p, p, p, p, None, None, 1, 9001, f32, f32, None, 0, None) == null
    assert lib.dc_layer_norm_backward(p, p, p, p, p, p, None, None, 1, 9001, f32, f32, p, 7, None) == space
    assert lib.dc_layer_norm_backward_workspace_bytes(0, 8, f32) == 0
    assert lib.dc_layer_norm_delta(p, None, p, p, p, p, p, p, 1, 8, f32, f32, 0.0, 1e-5, None) == null
    assert lib.dc_layer_norm_delta(p, p, p, p, p, p, p, p, 1, 8, bf16, bf16, 0.0, 1e-5, None) == dtype
    assert lib.dc_layer_norm_delta(p, p, p, p, p, p, p, p, 0, 8, f32, f32, 0.0, 1e-5, None) == 0
    assert lib.dc_mx4_quantize(p, p, None, None, None, None, 1, 32, f32, f32, None, 0, None) == null
    assert lib.dc_mx4_quantize(p, None, None, None, None, None, 1, 32, f32, f32, None, 0, None) == null
    assert lib.dc_mx4_quantize(p, p, p, None, None, None, 1, 0, f32, f32, None, 0, None) == shape
    assert lib.dc_mx4_quantize(p, p, p, None, None, None, 1, 32, 7, f32, None, 0, None) == dtype
    assert lib.dc_mx4_quantize(p, p + 8, p, None, None, None, 1, 32, f32, f32, None, 0, None) == align
    assert lib.dc_mx4_quantize(p, p, p, None, None, p, 1, 32, f32, f32, p, 4, None) == space
    assert lib.dc_mx4_dequantize(p, p, None, 1, 32, f32, None) == null
    assert lib.dc_mx4_dequantize(p, p, p, 1, 32, 9, None) == dtype
    assert lib.dc_mx4_matmul(p, p, p, p, None, p, 1, 1, 0, 0, f32, None) == shape
    assert lib.dc_mx4_matmul(p, p, p, p, None, p, 1, 1, 32, 0, 4, None) == dtype
    assert lib.dc_mx4_matmul(p, p, p, p, None, None, 1, 1, 32, 0, f32, None) == null
    assert lib.dc_mx4_matmul(p + 4, p, p, p, None, p, 1, 1, 32, 0, f32, None) == align
    assert lib.dc_mx4_matmul(None, None, None, None, None, None, 0, 5, 32, 0, f32, None) == 0
    assert lib.dc_mx4_linear(p, p, p, None, p, 1, 1, 0, f32, f32, None, 0, None) == shape
    assert lib.dc_mx4_linear(p, p, p, None, p, 1, 1, 32, 5, f32, None, 0, None) == dtype
    assert lib.dc_mx4_linear(p, p, None, None, p, 1, 1, 32, f32, f32, None, 0, None) == null
    assert lib.dc_mx4_linear(p, p + 8, p, None, p, 1, 1, 32, f32, f32, None, 0, None) == align
    assert lib.dc_mx4_linear(p, p, p, None, p, 500, 500, 32, f32, f32, p, 64, None) == space
    assert lib.dc_mx4_linear(p, p, p, None, p, 500, 500, 32, f32, f32, None, 0, None) == null
    assert lib.dc_mx4_linear_workspace_bytes(1, 500, 64) == 0 and lib.dc_mx4_linear_workspace_bytes(500, 500, 64) == 500 * 32 + 4 * 512
    train = lib.dc_mx4_linear_train
    assert train(p, p, None, p, p, p, 4, 8, 0, f32, f32, f32, p, 1 << 20, None) == shape
    assert train(p, p, None, p, p, p, 0, 8, 32, f32, f32, f32, p, 1 << 20, None) == shape
    assert train(p, p, None, p, p, p, 4, 8, 32, f32, 3, f32, p, 1 << 20, None) == dtype
    assert train(p, None, None, p, p, p, 4, 8, 32, f32, f32, f32, p, 1 << 20, None) == null
    assert train(p, p, None, p, p + 8, p, 4, 8, 32, f32, f32, f32, p, 1 << 20, None) == align
    assert train(p, p, None, p, p, p, 4, 8, 32, f32, f32, f32, p, 64, None) == space
    back = lib.dc_mx4_linear_backward
    assert back(p, None, None, None, None, None, 4, 8, 32, f32, f32, f32, p, 1 << 20, None) == 0
    assert back(p, None, p, p, p, None, 4, 8, 32, f32, f32, f32, p, 1 << 20, None) == null
    assert back(p, p, None, p, p, None, 4, 8, 32, f32, f32, f32, p, 1 << 20, None) == null
    assert back(p, p, p, p, p, p, 4, 8, 32, f32, f32, 3, p, 1 << 20, None) == dtype
    assert back(p, p, p, p, p, p, 4, 8, 32, f32, f32, f32, p, 64, None) == space
    assert lib.dc_mx4_linear_train_workspace_bytes(4, 8, 32) == 4 * 16 + 512 + 8 * 16 + 512
    assert lib.dc_mx4_data_bytes(3, 33) == 3 * 32 and lib.dc_mx4_scale_bytes(129, 129) == 2 * 2 * 512


def test_modules_refuse_what_they_cannot_take():
    with pytest.raises(RuntimeError, match="DCLayerNorm"):
        dc.DCLayerNorm((4, 4))
    with pytest.raises(RuntimeError, match="DCMX4Linear"):
        dc.DCMX4Linear(8, 8)((torch.zeros(1, 8, 1, 1), None))

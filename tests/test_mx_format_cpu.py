"""The plain statement of the microscaled format that the GPU tests compare with, checked against torch's own 8-bit type and
against what the format's definition says of single values."""
import numpy as np
import pytest
import torch

import mx_util


def test_e4m3_values_are_those_of_torch():
    codes = torch.arange(127, dtype=torch.uint8)
    np.testing.assert_array_equal(mx_util.E4M3, codes.view(torch.float8_e4m3fn).to(torch.float64).numpy())


def test_e4m3_rounding_is_that_of_torch():
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(1)) * 50
    codes, scales = mx_util.quantize(x.double().numpy(), 8)
    unit = torch.from_numpy(np.ldexp(1.0, scales - 127)).repeat_interleave(32, dim=1).float()
    want = (x / unit).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).long().numpy()
    np.testing.assert_array_equal(codes, want)


@pytest.mark.parametrize("value, code", [(0.25, 0), (0.26, 1), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5.0, 6),
                                         (5.1, 7), (7.9, 7), (-0.75, 10), (-5.1, 15)])
def test_e2m1_ties_and_saturation(value, code):
    row = np.zeros((1, 32))
    row[0, :2] = 4.0, value                      # the block's largest magnitude is in [4, 8): a scale of one
    codes, scales = mx_util.quantize(row, 4)
    assert scales[0, 0] == 127 and codes[0, 1] == code


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows, k", [(1, 1), (3, 129), (130, 260)])
def test_packing_goes_back(bits, rows, k):
    from tinyinfer_b200.kernels import MxRows
    x = np.random.RandomState(rows).randn(rows, k)
    codes, scales = mx_util.quantize(x, bits)
    held, tiles = mx_util.pack(codes, scales, bits)
    assert held.shape == (rows, mx_util.padded(k) * bits // 8) and tiles.shape == (-(-rows // 128), mx_util.padded(k) // 128, 512)
    again = mx_util.unpack(MxRows(held, tiles, bits, k))
    np.testing.assert_array_equal(again[0], codes)
    np.testing.assert_array_equal(again[1], scales)
    off = np.abs(mx_util.numbers(codes, scales, bits)[:, :k] - x)
    assert (off <= mx_util.rounding(x, bits)).all()


def test_the_binding_is_a_module_of_its_own():
    from tinyinfer_b200.kernels.build import LIBRARIES, TORCH_MODULES
    assert set(TORCH_MODULES) <= set(LIBRARIES)

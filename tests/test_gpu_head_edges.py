"""Calls of the operators around the head at which their formulas are easily missed: FP32 values between two codes."""
import numpy as np
import pytest
import torch

import head_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture
def K(cuda):
    from strixite_b200 import kernels
    return kernels


# ---- codes ---------------------------------------------------------------------------------------------------------------------------

def between(dev, T, blocks, seed):
    """Rows of FP32 values whose blocks of 128 have 7 j as their largest and else t j / 64, t halfway between two codes: 448 v / (7 j) is t, and v takes all of FP32's bits.
    -> the rows, and the even one of each value's two codes."""
    g = np.random.default_rng(seed)
    j = g.integers(1 << 16, (1 << 24) // 32, (T, blocks, 1)).astype(np.float64)
    t = (2 * g.integers(8, 16, (T, blocks, 128)) + 1) * 2.0 ** g.integers(-8, 4, (T, blocks, 128)) * g.choice([-1.0, 1.0], (T, blocks, 128))
    t[:, :, 77] = 448
    v = t * j / 64
    assert np.array_equal(v, v.astype(np.float32))
    step = 2.0 ** (np.floor(np.log2(np.abs(t))) - 3)  # four significant bits; numpy rounds halves to even
    return torch.from_numpy(v.reshape(T, -1).astype(np.float32)).to(dev), (np.round(t / step) * step).reshape(T, -1)


@pytest.mark.parametrize("norm,y", [(True, False), (False, False), (True, True)])
@pytest.mark.parametrize("T,blocks", [(33, 2), (65, 5), (2400, 16)])
def test_codes_of_fp32_values_between_two_numbers(K, cuda, norm, y, T, blocks):
    """What is rounded to a code is the nearest FP32 of 448 v / most, so a tie stays one, whatever bits v and the row's factor have."""
    x, want = between(cuda, T, blocks, T)
    codes, scales = torch.zeros(x.shape, dtype=torch.uint8, device=cuda).view(K.F8), torch.zeros((T, blocks), device=cuda)
    K.add_norm(x, torch.zeros_like(x) if y else None, weight=torch.full((x.shape[1],), 0.25, device=cuda) if norm else None, codes=codes, scales=scales, norm=norm)
    assert np.array_equal(P.f64(codes), want)


def test_codes_of_weights_between_two_numbers(K, cuda):
    j = 300001
    t = np.random.default_rng(8).choice(np.arange(17, 32, 2), (128, 128)) / 16
    w = t * j / 64
    w[5, 9] = 7 * j
    want = np.round(t * 8) / 8
    want[5, 9] = 448
    assert np.array_equal(P.f64(K.quantize_f8(torch.from_numpy(w.astype(np.float32)).to(cuda)).q), want)

"""Calls of the operators around the head at which their formulas are easily missed: FP32 values between two codes, logits at FP32's ends."""
import numpy as np
import pytest
import torch

import head_plain as P
from test_gpu_head import batch, check, gen

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


# ---- verification --------------------------------------------------------------------------------------------------------------------

def far_apart(dev, V, f32, draft, seed):
    """Rows whose logits lie further apart than FP32 reaches, at temperatures at which both ends count."""
    s = batch(dev, [1, 3, 1, 2, 4], V, seed=seed, f32=f32, draft=draft)
    g = gen(seed + 1, dev)
    for t in [s["logits"]] + ([s["draft"]] if draft else []):
        t[:] = -3e38
        t[:, V // 2:] = torch.where(torch.rand((t.shape[0], V - V // 2), generator=g, device=dev) < 0.3, 3e38, -3e38).to(t.dtype)
        t[:, -1] = 3e38
    s["ids"][:] = torch.randint(0, V, (11,), generator=g, device=dev)
    s["t"][:] = torch.tensor([1e38, 3.4e38, 2e38, 8e36, 9e37], device=dev)
    return s


@pytest.mark.parametrize("V", [2, 5, 1000, 3000, 20003])
@pytest.mark.parametrize("f32,draft", [(True, None), (False, None), (True, torch.float32), (False, torch.bfloat16), (True, torch.bfloat16)])
def test_verify_logits_further_apart_than_fp32_reaches(K, cuda, V, f32, draft):
    s = far_apart(cuda, V, f32, draft, V)
    check(K, cuda, s)
    s["u"][:] = 1 - 2.0 ** -24
    check(K, cuda, s)


@pytest.mark.parametrize("f32", [True, False])
def test_verify_draws_from_chunks_of_far_tokens_alone(K, cuda, f32):
    """The first chunks hold only tokens 6e38 below the largest; each of them has 1 / 403 of its chance."""
    s = far_apart(cuda, 20003, f32, None, 3)
    s["t"][:], s["u_pick"][:], s["u"][:] = 1e38, 0.0, 1 - 2.0 ** -24
    s["ids"][:] = 20002
    s["logits"][:, 10000:] = -3e38
    s["logits"][:, 20002] = 3e38
    ids, n, _ = check(K, cuda, s)
    assert torch.all(n == 1) and torch.all(ids[[0, 1, 4, 5, 7]] == 0)

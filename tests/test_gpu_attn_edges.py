"""GPU tests of the attention operators at their edges: what is not finite, values of very different sizes, caps of any size, log-sums in every row, far pages,
long chunks.  The definition in 64 bits and the bounds are attn_plain.py's; what differs from them is derived beside the test."""
import numpy as np
import pytest
import torch

import attn_plain as plain
from test_gpu_attn import Batch, K

pytestmark = pytest.mark.gpu

UNTOUCHED = 12345.0


def run_and_compare(b, scale=None, softcap=0.0, window=0, rows=None):
    """The batch's output and log-sum against the definition: NaN and infinities where it has them and nowhere else, every row of both written.
    rows: those that are compared (all)."""
    b.out.fill_(UNTOUCHED), b.lse.fill_(UNTOUCHED)
    b.run(scale=scale, softcap=softcap, window=window)
    torch.cuda.synchronize()
    assert (b.guard == 0xA5).all() and int(b.err[0]) == 0
    with np.errstate(all="ignore"):
        want, lse, tol, lse_tol = plain.attend(b.q, b.cache, b.pages, b.q_start, b.kv_len, b.cache.D ** -0.5 if scale is None else scale, softcap, window)
        got, got_lse = plain.f64(b.out).reshape(want.shape), plain.f64(b.lse)
        for a, w, t in ((got, want, tol), (got_lse, lse, lse_tol)):
            a, w, t = (x if rows is None else x[rows] for x in (a, w, t))
            assert not (a == UNTOUCHED).any()
            assert np.array_equal(np.isfinite(a), np.isfinite(w)), np.argwhere(np.isfinite(a) != np.isfinite(w))[:5]
            assert np.array_equal(np.isneginf(got_lse), np.isneginf(lse))
            ok = np.isfinite(w)
            far = (np.abs(a - w) - t)[ok]
            assert far.size == 0 or far.max() <= 0, (far.max(), np.argwhere(ok)[far.argmax()])
    return got, want


# ---- quantized values ----------------------------------------------------------------------------------------------------------------

QUANT = [(64, 8, 32), (64, 4, 32), (128, 8, 32), (128, 8, 64), (128, 4, 32), (128, 4, 64), (256, 8, 128), (256, 4, 32)]


@pytest.mark.parametrize("word,bad", [(0, float("nan")), (0, float("inf")), (1, float("nan")), (1, float("inf")), (1, -float("inf"))])
@pytest.mark.parametrize("D,bits,G", QUANT)
def test_a_value_group_that_is_none_is_so_alone(cuda, D, bits, G, word, bad):
    """A V group's scale or min is NaN or infinite, of a key that every row sees and of one that only the last draft does: its own columns are so, no others.
    Tiles of 8 and 16 rows; lengths with tiles that every row sees all of and without."""
    for group in (2, 5):
        b = Batch(cuda, D, bits, G, 2, group, [70, 700, 300], [3, 3, 1], seed=D + bits)
        for s, j in ((0, 10), (1, 333), (1, 699), (2, 5)):
            b.cache.v_sm[int(b.pages[s, j // 16]), :, j % 16, 1, word] = bad
        got, want = run_and_compare(b)
        assert np.isfinite(want[:, :, :G]).all() and not np.isfinite(want[3:6, :, G:2 * G]).all()

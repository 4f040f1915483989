"""CPU tests of calls around the head that are refused before any launch, beside those of test_head_refusals.py."""
import pytest


@pytest.mark.parametrize("kw,said", [
    (dict(scale=1 << 24), "scale [0x1000000] overlaps w"), (dict(scale=(1 << 24) + 256 * 256 * 4 - 4), "scale [0x103fffc] overlaps w"), (dict(scale=2 << 24), "scale [0x2000000] overlaps q"),
    (dict(err=(1 << 24) + 64), "err [0x1000040] overlaps w"), (dict(err=(2 << 24) + 256 * 256 - 4), "q [0x2000000] overlaps err"), (dict(scale=3 << 24, err=(3 << 24) + 12), "scale [0x3000000] overlaps err"),
])
def test_quantize_into_its_own_inputs(lib, kw, said):
    a = dict(w=1 << 24, act=0, N=256, K=256, q=2 << 24, scale=3 << 24, err=4 << 24)
    a.update(kw)
    assert lib.sxb_quantize_f8(*a.values(), None) == 1 and said in lib.sxb_last_error().decode()


def test_rows_that_are_no_matrix():
    """Tensors of one and of three dimensions: the package's error."""
    import torch
    from strixite_b200 import kernels as K
    for shape in ((64,), (2, 3, 64), ()):
        x = torch.zeros(shape, dtype=torch.bfloat16)
        with pytest.raises(K.Error, match="add_norm: x is"):
            K.add_norm(x, out=x)
        with pytest.raises(K.Error, match="linear_f8: x is"):
            K.linear_f8(x.to(K.F8), x, None, x)
        with pytest.raises(K.Error, match="verify_drafts: logits is"):
            K.verify_drafts(x, x, x, x, x, x, x, x, x)

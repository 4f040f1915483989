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

"""CPU tests of what the entry points around the head refuse before any launch."""
import ctypes as C

import pytest
import torch


def call(fn, lib, layout, a, kw):
    assert set(kw) <= set(a)
    a.update(kw)
    return fn(layout.pack(*a.values()), None), lib.sxb_last_error().decode()


def norm(lib, **kw):
    from strixite_b200 import kernels as K
    a = dict(x=1 << 24, y=2 << 24, weight=3 << 24, total=4 << 24, out=5 << 24, codes=6 << 24, scales=7 << 24, T=4, d=256, x_ld=256, y_ld=256, total_ld=256, out_ld=256, codes_ld=256,
             scales_ld=2, eps=1e-6, act=1, y_act=0, normed=1)
    return call(lib.sxb_add_norm, lib, K._NORM_ARGS, a, kw)


def view(**kw):
    from strixite_b200 import _lib
    c = dict(q=1 << 24, scale=2 << 24, N=300, K=400)
    c.update(kw)
    return _lib.SxbF8View(*c.values())


def linear(lib, v=None, **kw):
    from strixite_b200 import kernels as K
    v = v or view()
    a = dict(x=3 << 24, xs=4 << 24, w=C.addressof(v), y=5 << 24, M=7, x_ld=400, xs_ld=4, y_ld=300, out_act=1)
    return call(lib.sxb_linear_f8, lib, K._LINEAR_F8_ARGS, a, kw)


def verify(lib, **kw):
    from strixite_b200 import kernels as K
    a = dict(logits=1 << 24, draft=0, ld=1000, draft_ld=1000, T=6, V=1000, B=2, ids=2 << 24, q_start=3 << 24, u=4 << 24, u_pick=5 << 24, temperature=0, next_ids=6 << 24, n_new=7 << 24,
             logp=8 << 24, ws=9 << 24, ws_bytes=1 << 30, err=10 << 24, act=0, draft_act=0)
    return call(lib.sxb_verify_drafts, lib, K._VERIFY_ARGS, a, kw)


def test_argument_blocks_match_the_header(tmp_path):
    """The packed forms against the C compiler's layout of the header's structs: every offset."""
    import pathlib
    import subprocess
    from strixite_b200 import kernels as K
    root = pathlib.Path(__file__).resolve().parent.parent
    fields = {
        "SxbAddNormArgs": (K._NORM_ARGS, "x y weight total out codes scales T d x_ld y_ld total_ld out_ld codes_ld scales_ld eps act y_act normed"),
        "SxbLinearF8Args": (K._LINEAR_F8_ARGS, "x x_scale w y M x_ld xs_ld y_ld out_act"),
        "SxbVerifyDraftsArgs": (K._VERIFY_ARGS, "logits draft_logits ld draft_ld T V B ids q_start u u_pick temperature next_ids n_new logp ws ws_bytes err act draft_act"),
    }
    src = tmp_path / "t.c"
    src.write_text('#include "strix_b200.h"\n#include <stddef.h>\n#include <stdio.h>\nint main(void) {\n' + "".join(
        f'printf("%zu\\n", offsetof({s}, {f}));\n' for s, (_, names) in fields.items() for f in names.split()) + "return 0; }\n")
    subprocess.run(["gcc", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "t")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    import struct
    for layout, names in fields.values():
        codes = layout.format.lstrip("@")
        assert len(codes) == len(names.split())
        want += [struct.calcsize("@" + codes[:i + 1]) - struct.calcsize("@" + codes[i]) for i in range(len(codes))]
    assert got == want


def test_null_argument_blocks(lib):
    for fn in (lib.sxb_add_norm, lib.sxb_linear_f8, lib.sxb_verify_drafts):
        assert fn(None, None) == 1 and "null argument block" in lib.sxb_last_error().decode()


@pytest.mark.parametrize("kw,message", [
    (dict(x=0), "null pointer"), (dict(act=2), "unsupported dtypes"), (dict(y_act=3), "unsupported dtypes"), (dict(T=0), "T = 0"), (dict(T=(1 << 24) + 1), "T = "), (dict(d=0), "d = 0"),
    (dict(d=250), "d = 250"), (dict(d=32784), "d = 32784"), (dict(total=0, out=0, codes=0, scales=0), "no output"), (dict(y=0), "total without y"), (dict(codes=0), "come together"),
    (dict(scales=0), "come together"), (dict(normed=0), "weight without the norm"), (dict(eps=0.0), "eps"), (dict(eps=7e-31), "eps"), (dict(eps=float("nan")), "eps"), (dict(weight=(3 << 24) + 4), "weight must be 16"),
    (dict(x_ld=255), "row stride 255 of x"), (dict(y_ld=0), "of y"), (dict(total_ld=-1), "of total"), (dict(scales_ld=1), "of scales"), (dict(x_ld=260), "rows of x must be"),
    (dict(codes_ld=264), "rows of codes must be"), (dict(out=(5 << 24) + 8), "rows of out must be"), (dict(scales=(7 << 24) + 2), "rows of scales must be"),
    (dict(total=1 << 24, total_ld=512), "total [0x1000000] overlaps x"), (dict(total=(1 << 24) + 512), "overlaps x"), (dict(out=1 << 24), "out [0x1000000] overlaps x"),
    (dict(codes=(5 << 24) + 1024), "codes [0x5000400] overlaps out"), (dict(scales=3 << 24), "scales overlaps the weight"), (dict(total=2 << 24), "overlaps y"),
])
def test_norm_refusals(lib, kw, message):
    rc, said = norm(lib, **kw)
    assert rc == 1 and message in said, said


@pytest.mark.parametrize("v,kw,message", [
    (dict(), dict(w=0), "null weight"), (dict(q=0), dict(), "null pointer"), (dict(scale=0), dict(), "null pointer"), (dict(), dict(x=0), "null pointer"), (dict(), dict(xs=0), "null pointer"),
    (dict(), dict(y=0), "null pointer"), (dict(), dict(M=0), "M (rows of x) = 0"), (dict(), dict(M=(1 << 20) + 1), "M (rows of x)"), (dict(N=0), dict(), "N = 0"), (dict(K=392), dict(), "K = 392"),
    (dict(K=0), dict(), "K = 0"), (dict(N=(1 << 24) + 1), dict(), "N = "), (dict(), dict(out_act=2), "output dtype 2"), (dict(), dict(x_ld=399), "row strides 399"), (dict(), dict(x_ld=408), "16-byte aligned"),
    (dict(), dict(xs_ld=3), "row strides"), (dict(), dict(y_ld=299), "row strides"), (dict(q=(1 << 24) + 8), dict(), "16-byte aligned"), (dict(), dict(x=(3 << 24) + 8), "16-byte aligned"),
    (dict(), dict(y=(5 << 24) + 1), "aligned to their types"), (dict(), dict(y=3 << 24), "overlaps"), (dict(), dict(y=(1 << 24) + 256), "overlaps"), (dict(), dict(y=2 << 24), "overlaps"),
    (dict(), dict(y=(4 << 24) - 2), "overlaps"),
])
def test_linear_refusals(lib, v, kw, message):
    rc, said = linear(lib, view(**v), **kw)
    assert rc == 1 and message in said, said


@pytest.mark.parametrize("kw,message", [
    (dict(T=0), "T = 0"), (dict(V=0), "V = 0"), (dict(B=0), "B = 0"), (dict(V=(1 << 20) + 1, ld=1 << 21), "V = "), (dict(logits=0), "null pointer"), (dict(ids=0), "null pointer"),
    (dict(q_start=0), "null pointer"), (dict(u=0), "null pointer"), (dict(u_pick=0), "null pointer"), (dict(next_ids=0), "null pointer"), (dict(n_new=0), "null pointer"), (dict(ws=0), "null pointer"),
    (dict(err=0), "null pointer"), (dict(act=2), "unsupported dtypes"), (dict(draft=11 << 24, draft_act=2), "unsupported dtypes"), (dict(ld=999), "row strides"),
    (dict(draft=11 << 24, draft_ld=999), "row strides"), (dict(logits=(1 << 24) + 2), "aligned to their type"), (dict(draft=(11 << 24) + 1, draft_act=1), "aligned to their type"),
    (dict(ws_bytes=100), "workspace of 100 bytes"), (dict(ws=(9 << 24) + 8), "16-byte aligned"), (dict(next_ids=2 << 24), "next_ids [0x2000000] overlaps ids"), (dict(n_new=5 << 24), "overlaps u_pick"),
    (dict(logp=6 << 24), "logp [0x6000000] overlaps next_ids"), (dict(ws=1 << 24), "overlaps logits"), (dict(temperature=7 << 24), "n_new [0x7000000] overlaps temperature"),
    (dict(temperature=(8 << 24) + 16), "overlaps temperature"), (dict(err=6 << 24), "overlaps err"), (dict(B=8193), "B = 8193"),
])
def test_verify_refusals(lib, kw, message):
    rc, said = verify(lib, **kw)
    assert rc == 1 and message in said, said


def test_workspace_sizes(lib):
    from strixite_b200 import kernels as K
    assert K.verify_drafts_workspace_bytes(1, 1, 1) > 0
    assert K.verify_drafts_workspace_bytes(16, 2, 131072) <= K.verify_drafts_workspace_bytes(17, 2, 131072)
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, (1 << 20) + 1)):
        with pytest.raises(K.Error, match="verify_drafts_workspace_bytes"):
            K.verify_drafts_workspace_bytes(*bad)


def test_quantize_refusals(lib):
    def q(w=1 << 24, act=0, N=256, K_=256, codes=2 << 24, scale=3 << 24, err=4 << 24):
        return lib.sxb_quantize_f8(w, act, N, K_, codes, scale, err, None), lib.sxb_last_error().decode()
    for kw, message in ((dict(w=0), "null pointer"), (dict(err=0), "null pointer"), (dict(act=2), "unsupported dtype"), (dict(N=0), "N = 0"), (dict(K_=24), "K = 24"), (dict(w=(1 << 24) + 4), "16-byte"),
                        (dict(codes=(1 << 24) + 16), "overlaps")):
        rc, said = q(**kw)
        assert rc == 1 and message in said, said


def test_report_errors(lib):
    from strixite_b200 import kernels as K
    K.report_verify_error([0, 0, 0], "step")
    for code, words in ((1, "not finite"), (2, "drafter"), (3, "out of range at row 7"), (4, "random number"), (5, "temperature"), (6, "at sequence 7")):
        with pytest.raises(K.Error, match=words):
            K.report_verify_error([1, 7, code], "step")


def test_python_refuses_before_the_library():
    """Tensors of other types and shapes are refused, on the CPU too."""
    from strixite_b200 import kernels as K
    with pytest.raises(K.Error, match="F8View"):
        K.F8View(torch.zeros((4, 16)), torch.zeros((1, 1)))
    codes = torch.zeros((4, 16), dtype=torch.uint8).view(K.F8)
    with pytest.raises(K.Error, match="expected contiguous"):
        K.F8View(codes, torch.zeros((2, 1)))
    with pytest.raises(K.Error, match="CUDA device"):
        K.F8View(codes, torch.zeros((1, 1)))
    with pytest.raises(K.Error, match="quantize_f8"):
        K.quantize_f8(torch.zeros((4, 16), dtype=torch.float16))
    for err in (torch.zeros(2, dtype=torch.int32), torch.zeros(4), torch.zeros(8, dtype=torch.int32)[::2], torch.zeros(4, dtype=torch.int32, device="meta")):
        with pytest.raises(K.Error, match="quantize_f8: err"):
            K.quantize_f8(torch.zeros((4, 16)), err=err)


def test_quantize_on_another_device_than_the_current(monkeypatch):
    """Its launch would be the current device's: a stand-in for a weight on a second one."""
    from strixite_b200 import kernels as K

    class There:
        dtype, shape, is_cuda, device = torch.float32, (4, 16), True, torch.device("cuda", 1)
        dim, is_contiguous, get_device = (lambda self: 2), (lambda self: True), (lambda self: 1)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(K.Error, match="lives on device 1, the current device is 0"):
        K.quantize_f8(There())

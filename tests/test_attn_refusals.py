"""CPU tests of what the attention entry points refuse before any launch."""
import ctypes as C

import pytest


def cache(**kw):
    from strixite_b200 import _lib
    c = dict(k=1 << 20, v=2 << 20, k_sm=3 << 20, v_sm=4 << 20, n_pages=10, n_kv=2, page=16, D=128, G=64, page_stride=32, head_stride=16, row_stride=1, bits=8)
    c.update(kw)
    return _lib.SxbKvCache(*[c[f[0]] for f in _lib.SxbKvCache._fields_])


BAD_CACHES = [
    (dict(bits=5), "5 bits unsupported"), (dict(D=96), "heads of 96"), (dict(k=0), "null pointer"), (dict(v=(2 << 20) + 8), "16-byte aligned"),
    (dict(G=48), "group size 48"), (dict(D=64, G=128), "group size 128"), (dict(k_sm=0), "null pointer"), (dict(v_sm=(4 << 20) + 4), "16-byte aligned"),
    (dict(n_pages=0), "n_pages = 0"), (dict(n_kv=0), "n_kv = 0"), (dict(page=24), "pages of 24"), (dict(page=4), "pages of 4"), (dict(page=8192), "pages of 8192"),
    (dict(page_stride=0), "strides of 0"), (dict(row_stride=-1), "strides of"), (dict(head_stride=1 << 40), "strides of"), (dict(row_stride=(1 << 22) + 1), "strides of"),
    (dict(page_stride=1 << 31, n_pages=10), "more than 2^36 bytes"), (dict(n_pages=(1 << 31) - 1, page_stride=(1 << 32) - 1), "more than 2^36 bytes"),
]


def call(fn, lib, layout, a, kw):
    assert set(kw) <= set(a)
    a.update(kw)
    return fn(layout.pack(*a.values()), None), lib.sxb_last_error().decode()


def write(lib, c=None, **kw):
    from strixite_b200 import kernels as K
    c = c or cache()
    a = dict(qkv=5 << 20, ld=8 * 128, T=4, n_q=4, q_norm=6 << 20, k_norm=6 << 20, inv=7 << 20, rot=128, seq=8 << 20, pos=8 << 20, pages=9 << 20, pages_ld=5, n_cols=5,
             n_seq=2, cache=C.addressof(c), q_out=10 << 20, q_ld=512, err=11 << 20, eps=1e-6, act=1, inter=0)
    return call(lib.sxb_attn_qkv_write, lib, K._WRITE_ARGS, a, kw)


def attend(lib, c=None, **kw):
    from strixite_b200 import kernels as K
    c = c or cache()
    a = dict(q=5 << 20, q_ld=512, T=4, n_q=4, cache=C.addressof(c), pages=9 << 20, pages_ld=5, n_cols=5, q_start=8 << 20, kv_len=8 << 20, B=2, max_q=2, out=10 << 20,
             out_ld=512, lse=0, ws=12 << 20, ws_bytes=1 << 30, err=11 << 20, window=0, scale=0.1, cap=0.0)
    return call(lib.sxb_attn_decode, lib, K._DECODE_ARGS, a, kw)


def read(lib, c=None, **kw):
    from strixite_b200 import kernels as K
    c = c or cache()
    a = dict(cache=C.addressof(c), seq=8 << 20, pos=8 << 20, pages=9 << 20, pages_ld=5, n_cols=5, n_seq=2, T=4, k=5 << 20, v=10 << 20, err=11 << 20, act=1)
    return call(lib.sxb_kv_read, lib, K._READ_ARGS, a, kw)


def test_null_argument_blocks(lib):
    for fn in (lib.sxb_attn_qkv_write, lib.sxb_attn_decode, lib.sxb_kv_read):
        assert fn(None, None) == 1 and "null argument block" in lib.sxb_last_error().decode()


@pytest.mark.parametrize("entry", [write, attend, read])
@pytest.mark.parametrize("kw,message", BAD_CACHES)
def test_bad_caches(lib, entry, kw, message):
    rc, said = entry(lib, cache(**kw))
    assert rc == 1 and message in said, said


@pytest.mark.parametrize("entry", [write, attend, read])
def test_null_cache_and_tables(lib, entry):
    for kw, message in ((dict(cache=0), "null cache"), (dict(pages=0), "null pointer"), (dict(err=0), "null pointer"), (dict(T=0), "T = 0"), (dict(n_cols=0), "0 columns"),
                        (dict(pages_ld=4), "stride of 4"), (dict(n_cols=1 << 27, pages_ld=1 << 27), "positions end below")):
        rc, said = entry(lib, **kw)
        assert rc == 1 and message in said, (kw, said)


@pytest.mark.parametrize("kw,message", [
    (dict(qkv=0), "null pointer"), (dict(q_out=0), "null pointer"), (dict(seq=0), "null pointer"), (dict(act=2), "activation dtype 2"), (dict(n_q=0), "n_q = 0"),
    (dict(ld=1023), "row strides"), (dict(ld=1028), "16-byte aligned"), (dict(q_ld=516), "16-byte aligned"), (dict(q_out=(10 << 20) + 8), "16-byte aligned"),
    (dict(q_out=(5 << 20) + 512), "overlaps"), (dict(inv=0), "without inv_freq"), (dict(rot=24), "rot = 24"), (dict(rot=144), "rot = 144"), (dict(rot=-16), "rot = -16"),
    (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(n_seq=0), "n_seq = 0"), (dict(T=(1 << 20) + 1), "T = "),
])
def test_write_refusals(lib, kw, message):
    rc, said = write(lib, **kw)
    assert rc == 1 and message in said, said


@pytest.mark.parametrize("kw,message", [
    (dict(q=0), "null pointer"), (dict(ws=0), "null pointer"), (dict(q_start=0), "null pointer"), (dict(n_q=3), "n_q = 3"), (dict(n_q=1), "n_q = 1"), (dict(B=0), "B = 0"),
    (dict(max_q=0), "max_q = 0"), (dict(q_ld=511), "row strides"), (dict(out_ld=516), "row strides"), (dict(q=(5 << 20) + 2), "16-byte aligned"),
    (dict(ws=(12 << 20) + 4), "16-byte aligned"), (dict(out=(5 << 20) + 64), "overlaps"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=0.0), "scale"), (dict(scale=-0.1), "scale"),
    (dict(cap=-1.0), "softcap"), (dict(cap=1e-9), "softcap"), (dict(cap=float("nan")), "softcap"), (dict(window=-1), "window = -1"), (dict(window=1 << 31), "window"), (dict(ws_bytes=16), "workspace of 16 bytes, needs"),
])
def test_attend_refusals(lib, kw, message):
    if "ws_bytes" in kw:
        pytest.importorskip("torch")
    rc, said = attend(lib, **kw)
    assert rc == 1 and message in said, said


@pytest.mark.parametrize("kw,message", [(dict(k=0), "null pointer"), (dict(act=3), "output dtype 3"), (dict(v=(10 << 20) + 2), "16-byte aligned"), (dict(v=5 << 20), "overlaps")])
def test_read_refusals(lib, kw, message):
    rc, said = read(lib, **kw)
    assert rc == 1 and message in said, said


def test_workspace_refusals(lib):
    for bad in ((0, 1, 128, 16, 1), (3, 2, 128, 16, 1), (4, 2, 96, 16, 1), (4, 2, 128, 6, 1), (4, 2, 128, 8, 0), (2048, 2, 128, 8, 1)):
        assert lib.sxb_attn_decode_workspace_bytes(*bad) == 0
        assert "attn_decode_workspace_bytes" in lib.sxb_last_error().decode()


def test_argument_blocks_match_the_header(tmp_path):
    """The packed layouts of kernels.py against the C compiler's sizes and offsets."""
    import pathlib
    import re
    import struct
    import subprocess
    from strixite_b200 import kernels as K
    root = pathlib.Path(__file__).resolve().parent.parent
    text = (root / "include" / "strix_b200.h").read_text()
    body, want = "", {}
    for name, layout in (("SxbAttnQkvWriteArgs", K._WRITE_ARGS), ("SxbKvReadArgs", K._READ_ARGS), ("SxbAttnDecodeArgs", K._DECODE_ARGS)):
        decl = re.sub(r"/\*.*?\*/", "", text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")], flags=re.S).split("{")[1]
        fields = [f.replace("*", " ").split()[-1] for line in decl.split(";") for f in line.split(",") if f.strip()]
        assert len(fields) == len(layout.format) - 1
        for i, f in enumerate(fields):
            body += f'    printf("{name}.{f} %zu\\n", offsetof({name}, {f}));\n'
            want[f"{name}.{f}"] = struct.calcsize(layout.format[:i + 2]) - struct.calcsize("@" + layout.format[i + 1])
        body += f'    printf("{name} %zu\\n", sizeof({name}));\n'
        want[name] = (layout.size + 7) // 8 * 8
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "strix_b200.h"\nint main(void) {\n' + body + "    return 0;\n}\n")
    subprocess.run(["gcc", "-std=c99", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    assert {line.split()[0]: int(line.split()[1]) for line in out.splitlines()} == want


def test_cache_struct_matches_the_header(tmp_path):
    import pathlib
    import subprocess
    from strixite_b200 import _lib
    root = pathlib.Path(__file__).resolve().parent.parent
    names = [f[0] for f in _lib.SxbKvCache._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "strix_b200.h"\nint main(void) {\n    printf("sizeof %zu\\n", sizeof(SxbKvCache));\n'
                   + "".join(f'    printf("{n} %zu\\n", offsetof(SxbKvCache, {n}));\n' for n in names) + "    return 0;\n}\n")
    subprocess.run(["gcc", "-std=c99", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(out["sizeof"]) == C.sizeof(_lib.SxbKvCache)
    for n in names:
        assert int(out[n]) == getattr(_lib.SxbKvCache, n).offset, n


def test_python_refuses_what_lives_nowhere_or_fits_nothing(lib):
    import torch
    from strixite_b200 import kernels as K
    z = torch.zeros
    with pytest.raises(K.Error, match="must live on a CUDA device"):
        K.KvCache(z(2, 1, 16, 64, dtype=torch.bfloat16), z(2, 1, 16, 64, dtype=torch.bfloat16), 16)
    with pytest.raises(K.Error, match="7 bits"):
        K.KvCache(z(2, 1, 16, 64), z(2, 1, 16, 64), 7)
    with pytest.raises(K.Error, match="expected the same"):
        K.KvCache(z(2, 1, 16, 64), z(2, 1, 16, 32), 16)


def test_report_attn_error(lib):
    from strixite_b200 import kernels as K
    K.report_attn_error([0, 0, 0], "step")
    with pytest.raises(K.Error, match=r"step: page, position, length or row range out of range at token or sequence 7 \(-1\)"):
        K.report_attn_error([1, 7, 0xFFFFFFFF], "step")


def test_layer_refuses_rows_that_do_not_fit(lib, monkeypatch):
    """What the projections would read or write beyond its end - x, y or buffers of another width, a view, another type - is refused before a launch."""
    import types
    import torch
    from strixite_b200 import kernels as K
    from strixite_b200.attention import AttnLayer, AttnWeights
    for name in ("linear_qw", "linear_qw_wmma", "attn_qkv_write", "attn_decode"):
        monkeypatch.setattr(K, name, lambda *a, **kw: pytest.fail("launched"))
    cache = types.SimpleNamespace(D=64, n_kv=2, device=torch.device("cpu"))
    def view(n, k):
        return K.QDeviceView(None, None, None, n, k, 64, 8)
    def buffers(n_qkv=512, n_q=256, rows=10):
        return types.SimpleNamespace(max_tokens=rows, max_q=4, qkv=torch.zeros(rows, n_qkv), q=torch.zeros(rows, n_q), o=torch.zeros(rows, n_q))
    weights = AttnWeights(view(512, 96), view(96, 256))
    for bad in (buffers(n_qkv=384), buffers(n_q=128)):
        with pytest.raises(K.Error, match="AttnLayer: buffers of"):
            AttnLayer(weights, 4, cache, bad)
    layer, batch = AttnLayer(weights, 4, cache, buffers()), types.SimpleNamespace(max_q=1)
    bf = torch.bfloat16
    x, y = torch.zeros(3, 96, dtype=bf), torch.zeros(3, 96, dtype=bf)
    for bad_x, bad_y in ((torch.zeros(3, 64, dtype=bf), y), (torch.zeros(3, 96, 1, dtype=bf), y), (torch.zeros(3, 192, dtype=bf)[:, :96], y), (x, y[:2]), (x, y[:, :64]),
                         (x, torch.zeros(96, 3, dtype=bf).t()), (x, y.double()), (x, y.to("meta"))):
        with pytest.raises(K.Error, match="AttnLayer: x .* expected contiguous rows of 96 and of 96"):
            layer.forward(bad_x, batch, bad_y)
    with pytest.raises(K.Error, match="the buffers hold 10"):
        layer.forward(torch.zeros(11, 96, dtype=bf), batch, torch.zeros(11, 96, dtype=bf))

"""The operators around the head against their formulas in 64 bits (head_plain.py has the bounds): norm into 8-bit codes, products of 8-bit floating point, verification."""
import numpy as np
import pytest
import torch

import head_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture
def K(cuda):
    from strixite_b200 import kernels
    return kernels


def gen(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def codes_like(K, shape, dev, fill=0):
    return torch.full(shape, fill, dtype=torch.uint8, device=dev).view(K.F8)


# ---- norm ----------------------------------------------------------------------------------------------------------------------------

def run_norm(K, dev, T, d, x32=False, y=torch.bfloat16, weight=True, norm=True, seed=0, size=1.0, eps=1e-6, in_place=None, wide=0):
    g = gen(seed, dev)
    kept = torch.float32 if x32 else torch.bfloat16

    def rows(n, dtype, fill=None):
        t = torch.full((T, n + wide), 7, dtype=torch.float32, device=dev).to(dtype)[:, :n]
        if fill is not None:
            t.copy_(fill)
        return t
    x = rows(d, kept, torch.randn((T, d), generator=g, device=dev) * size)
    yt = None if y is None else rows(d, y, torch.randn((T, d), generator=g, device=dev) * size)
    w = 1 + 0.3 * torch.randn(d, generator=g, device=dev) if weight else None
    nb = -(-d // 128)
    total = None if yt is None else {"x": x, "y": yt}.get(in_place, rows(d, kept))
    out = rows(d, torch.bfloat16)
    codes, scales = codes_like(K, (T, d + wide), dev, 0x55), torch.full((T, nb + (3 if wide else 0)), 5.0, device=dev)
    s = x.float() if yt is None else (x.float() + yt.float()).to(kept).float()
    K.add_norm(x, yt, weight=w, eps=eps, total=total, out=out, codes=codes[:, :d], scales=scales[:, :nb], norm=norm)
    torch.cuda.synchronize()
    if total is not None:
        assert torch.equal(total.float(), s)
    n = P.f64(s) if not norm else P.norm(P.f64(s), w, eps)
    off = P.NORM if norm else 0.0
    assert np.all(np.abs(P.f64(out) - n) <= (P.BF16 + off) * np.abs(n) + 1e-38)
    P.check_codes(codes[:, :d], scales[:, :nb], n, off)
    if wide:  # what lies between the rows stays
        assert torch.all(codes.view(torch.uint8)[:, d:] == 0x55) and torch.all(scales[:, nb:] == 5.0)
    return x, codes, scales


@pytest.mark.parametrize("T,d", [(1, 16), (2, 64), (3, 128), (5, 144), (1, 4096), (37, 2560), (9, 8192), (3, 8208), (2, 16400), (2, 32768), (400, 1040), (700, 4096)])
@pytest.mark.parametrize("x32,y", [(False, torch.bfloat16), (False, torch.float32), (False, None), (True, torch.float32), (True, torch.bfloat16), (True, None)])
def test_norm(K, cuda, T, d, x32, y):
    run_norm(K, cuda, T, d, x32, y, seed=T + d)


@pytest.mark.parametrize("kw", [dict(weight=False), dict(norm=False, weight=False), dict(wide=48), dict(wide=48, x32=True, y=torch.float32), dict(in_place="x"), dict(in_place="y"),
                                dict(in_place="x", x32=True, y=torch.float32), dict(size=1e33, norm=False, weight=False, x32=True, y=torch.float32), dict(size=1e-18), dict(size=1e15), dict(eps=1.0), dict(size=1e-30, norm=False, weight=False)])
@pytest.mark.parametrize("T,d", [(3, 400), (33, 4096), (600, 2560)])
def test_norm_forms(K, cuda, T, d, kw):
    run_norm(K, cuda, T, d, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(y=None), dict(wide=16), dict(in_place="x"), dict(in_place="y"), dict(x32=True), dict(x32=True, y=torch.float32), dict(norm=False, weight=False)])
@pytest.mark.parametrize("T,d", [(2368, 2048), (2500, 2064), (3001, 8192), (20011, 256), (20011, 16)])
def test_norm_of_many_rows(K, cuda, T, d, kw):
    """CTAs that go on from row to row, and rows of a warp each, the last CTA's not all there."""
    run_norm(K, cuda, T, d, seed=d, **kw)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("most", [64, 56, 96, 127])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_between_two_numbers_go_to_the_even_one(K, cuda, norm, most, dtype):
    """Whole numbers, a block's largest one known: 448 x / most is a number that FP64 holds or is far from a tie, and the row's factor must not move it."""
    x = torch.randint(-most, most + 1, (64, 512), generator=gen(most, cuda), device=cuda).to(dtype)
    x[:, ::128] = most
    codes, scales = codes_like(K, (64, 512), cuda), torch.zeros((64, 4), device=cuda)
    K.add_norm(x, codes=codes, scales=scales, norm=norm)
    v = P.f64(x) * 448 / most
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6))) - 3)
    assert np.array_equal(P.f64(codes), np.round(v / step) * step)  # numpy rounds halves to even


def test_norm_one_output_at_a_time(K, cuda):
    g = gen(3, cuda)
    x, y = (torch.randn((5, 272), generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    total, out, codes, scales = torch.zeros_like(x), torch.zeros_like(x), codes_like(K, (5, 272), cuda), torch.zeros((5, 3), device=cuda)
    K.add_norm(x, y, total=total, out=out, codes=codes, scales=scales)
    one = [torch.zeros_like(x), torch.zeros_like(x), codes_like(K, (5, 272), cuda), torch.zeros((5, 3), device=cuda)]
    K.add_norm(x, y, total=one[0])
    K.add_norm(x, y, out=one[1])
    K.add_norm(x, y, codes=one[2], scales=one[3])
    for a, b in zip((total, out, codes.view(torch.uint8), scales), (one[0], one[1], one[2].view(torch.uint8), one[3])):
        assert torch.equal(a, b)


def test_norm_of_zeros_and_of_what_is_not_finite(K, cuda):
    x = torch.randn((6, 300 // 16 * 16), generator=gen(5, cuda), device=cuda)
    x[0] = 0
    x[1, 130] = float("nan")
    x[2, 7] = float("inf")
    x[3] = 1e30  # squares beyond FP32: zeros
    x[4] = 1e-30
    codes, scales, out = codes_like(K, x.shape, cuda), torch.zeros((6, 3), device=cuda), torch.zeros(x.shape, dtype=torch.bfloat16, device=cuda)
    K.add_norm(x, codes=codes, scales=scales, out=out)
    v = codes.float() * scales.repeat_interleave(128, 1)[:, :x.shape[1]]
    assert torch.all(v[0] == 0) and torch.all(scales[0] == P.LEAST)
    assert torch.all(v[1].isnan()) and torch.all(out[1].float().isnan())
    assert torch.all(v[2, :128].isnan()) and torch.all(v[2, 128:] == 0)
    assert torch.all(v[3] == 0) and torch.all(v[4].abs() < 1e-26) and torch.all(v[5].isfinite())
    # without the norm only the block is lost
    K.add_norm(x, codes=codes, scales=scales, norm=False)
    v = codes.float() * scales.repeat_interleave(128, 1)[:, :x.shape[1]]
    assert torch.all(v[1, :128].isfinite()) and torch.all(v[1, 128:256].isnan()) and torch.all(v[1, 256:].isfinite())
    assert torch.all((v[3] / 1e30 - 1).abs() < 0.07)


@pytest.mark.parametrize("N,K_", [(1, 16), (128, 128), (129, 144), (300, 1040), (1000, 4096)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize(K, cuda, N, K_, dtype):
    w = (torch.randn((N, K_), generator=gen(N, cuda), device=cuda) * 0.02).to(dtype)
    v = K.quantize_f8(w)
    nb = -(-K_ // 128)
    most = torch.zeros((-(-N // 128) * 128, nb * 128), device=cuda)
    most[:N, :K_] = w.float().abs()
    want = P.f64(most.view(-1, 128, nb, 128).amax((1, 3))) / P.TOP
    assert np.all(np.abs(P.f64(v.scale) - want) <= 2 * P.U * want)
    x = P.f64(w) / P.spread(np.repeat(P.f64(v.scale), 128, 0)[:N], K_)
    assert np.all(np.abs(P.f64(v.q) - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10) * 1.001 + 4 * P.U * np.abs(x))


def test_quantize_reports_what_is_not_finite(K, cuda):
    w = torch.ones((200, 256), device=cuda)
    w[150, 17] = float("inf")
    with pytest.raises(K.Error, match=r"non-finite weight at \[150, 17\]"):
        K.quantize_f8(w)
    err = torch.zeros(4, dtype=torch.int32, device=cuda)
    v = K.quantize_f8(w, err=err)
    assert err[:3].tolist() == [1, 150, 17]
    assert v.scale[1, 0].isnan() and torch.all(v.scale.flatten()[[0, 1, 3]] == 1 / 448)


# ---- product -------------------------------------------------------------------------------------------------------------------------

def operands(K, dev, M, N, K_, seed):
    """Codes of every size, scales that differ by block."""
    g = gen(seed, dev)
    nb, rb = -(-K_ // 128), -(-N // 128)
    x = torch.randint(0, 256, (M, K_), generator=g, device=dev, dtype=torch.uint8)
    w = torch.randint(0, 256, (N, K_), generator=g, device=dev, dtype=torch.uint8)
    for t in (x, w):
        t[(t & 0x7f) == 0x7f] = 0x01
    xs = torch.exp(torch.randn((M, nb), generator=g, device=dev)) * 0.01
    ws = torch.exp(torch.randn((rb, nb), generator=g, device=dev)) * 0.01
    return x.view(K.F8), xs, w.view(K.F8), ws


def check_linear(K, dev, M, N, K_, f32, seed=0, wide=0):
    x, xs, w, ws = operands(K, dev, M, N, K_, seed)
    if wide:
        x = torch.cat((x.view(torch.uint8), torch.full((M, 32), 0x7f, dtype=torch.uint8, device=dev)), 1).view(K.F8)[:, :K_]
        xs = torch.cat((xs, torch.full((M, 3), float("nan"), device=dev)), 1)[:, :xs.shape[1]]
    full = torch.full((M + 1, N + wide), 3.0, device=dev).to(torch.float32 if f32 else torch.bfloat16)
    y = full[:M, :N]
    K.linear_f8(x, xs, K.F8View(w, ws), y)
    torch.cuda.synchronize()
    want, size, nb = P.linear(x, xs, w, ws)
    off = np.abs(P.f64(y) - want)
    bound = P.linear_bound(want, size, nb, not f32)
    assert np.all(off <= bound), (float((off / np.maximum(bound, 1e-300)).max()), np.unravel_index((off / np.maximum(bound, 1e-300)).argmax(), off.shape))
    assert torch.all(full[M] == 3.0) and torch.all(full[:M, N:] == 3.0)
    K.check_dense_status("linear_f8")


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 48, 64, 65, 100, 127, 128, 129, 200, 256, 257, 300, 513])
@pytest.mark.parametrize("N,K_", [(1, 16), (8, 128), (100, 144), (129, 1040), (384, 512), (1000, 400), (2560, 4096)])
@pytest.mark.parametrize("f32", [True, False])
def test_linear(K, cuda, M, N, K_, f32):
    check_linear(K, cuda, M, N, K_, f32, seed=M + N)


@pytest.mark.parametrize("M", [1, 16, 40, 70, 200, 1000])
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("wide", [1, 8, 24])
def test_linear_strides(K, cuda, M, f32, wide):
    check_linear(K, cuda, M, 333, 656, f32, seed=M, wide=wide)


@pytest.mark.parametrize("M,N,K_", [(3, 20000, 256), (64, 4096, 16384), (5, 64, 131072), (130, 64, 65536), (2000, 2000, 128), (777, 1000, 1040), (150, 2560, 4096), (4000, 520, 272), (1100, 5000, 656), (2049, 4097, 400),
                                    (1024, 4096, 1024), (8200, 130, 144)])
def test_linear_long(K, cuda, M, N, K_):
    check_linear(K, cuda, M, N, K_, True, seed=M)


@pytest.mark.parametrize("M,N,K_,wide", [(2049, 4097, 400, 0), (2100, 4098, 144, 0), (1500, 4100, 272, 2), (2303, 4099, 128, 4), (2049, 4104, 272, 0), (600, 1003, 128, 0), (600, 1002, 1040, 0)])
@pytest.mark.parametrize("f32", [True, False])
def test_linear_rows_of_any_alignment(K, cuda, M, N, K_, wide, f32):
    """Pairs' tiles and single ones whose rows begin on 2, 4, 8 and 16 bytes."""
    check_linear(K, cuda, M, N, K_, f32, seed=N, wide=wide)


@pytest.mark.parametrize("M", [4, 40, 100, 300, 1500])
def test_linear_what_is_not_finite_stays_in_its_row_and_column(K, cuda, M):
    N, K_ = 300, 400
    x, xs, w, ws = operands(K, cuda, M, N, K_, 1)
    clean = torch.zeros((M, N), device=cuda)
    K.linear_f8(x, xs, K.F8View(w, ws), clean)
    x, w = x.clone(), w.clone()
    x.view(torch.uint8)[2, 390] = 0x7f
    w.view(torch.uint8)[201, 5] = 0xff
    xs = xs.clone()
    xs[M - 1, 3] = float("nan")
    y = torch.zeros((M, N), device=cuda)
    K.linear_f8(x, xs, K.F8View(w, ws), y)
    bad = torch.zeros((M, N), dtype=torch.bool, device=cuda)
    bad[2], bad[M - 1], bad[:, 201] = True, True, True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])


def test_linear_zero_scales_and_codes(K, cuda):
    for M in (5, 300):
        x, xs, w, ws = operands(K, cuda, M, 200, 512, 2)
        xs[:, 1] = 0
        ws[0, 2] = 0
        x.view(torch.uint8)[:, 384:] = 0x80  # -0
        y = torch.zeros((M, 200), device=cuda)
        K.linear_f8(x, xs, K.F8View(w, ws), y)
        want, size, nb = P.linear(x, xs, w, ws)
        assert np.all(np.abs(P.f64(y) - want) <= P.linear_bound(want, size, nb, False))


@pytest.mark.parametrize("M", [3, 50, 100, 700])
def test_linear_repeats_bit_for_bit(K, cuda, M):
    x, xs, w, ws = operands(K, cuda, M, 1100, 2064, 4)
    v = K.F8View(w, ws)
    first = torch.zeros((M, 1100), device=cuda)
    K.linear_f8(x, xs, v, first)
    for _ in range(5):
        y = torch.zeros_like(first)
        K.linear_f8(x, xs, v, y)
        assert torch.equal(y, first)


@pytest.mark.parametrize("M,N,K_,slot", [(2048, 4096, 1024, 0), (2048, 4096, 1024, 7), (2048, 4096, 1024, 10), (100, 300, 2048, 0), (100, 300, 2048, 1), (300, 40000, 1024, 2), (300, 40000, 1024, 9)])
def test_linear_gives_up_a_wait(K, cuda, lib, M, N, K_, slot):
    """The product with CTA 0 told to leave a stage out, in a pair's first and second tile, in a tile that a cluster shares and in one of its own.  The kernel returns, the status names
    the role, the next call has the bits of the call before."""
    x, xs, w, ws = operands(K, cuda, M, N, K_, slot)
    v, out = K.F8View(w, ws), [torch.full((M, N), float("nan"), device=cuda) for _ in range(3)]
    K.linear_f8(x, xs, v, out[0])
    K.check_dense_status("warm-up")
    try:
        K.set_wait_limit(2_000_000)
        assert lib.sxb_test_skip_ring_slot(slot) == 0
        K.linear_f8(x, xs, v, out[1])
        torch.cuda.synchronize()
    finally:
        lib.sxb_test_skip_ring_slot(-1)
        K.set_wait_limit(2_000_000_000)
    with pytest.raises(K.Error, match=r"skipped fill: a tcgen05 kernel gave up a wait at work item \d+ \((an MMA warp|the epilogue|the activation copy)"):
        K.check_dense_status("skipped fill")
    K.linear_f8(x, xs, v, out[2])
    K.check_dense_status("after")
    assert torch.equal(out[2], out[0]) and not bool(torch.isnan(out[2]).any())


# ---- verification ----------------------------------------------------------------------------------------------------------------------

def batch(dev, counts, V, seed, f32=True, draft=None, greedy=False, wide=0, close=0.5, peak=6.0):
    """draft: None, or the type of the drafter's logits."""
    g = gen(seed, dev)
    T, B = sum(counts), len(counts)
    def rand(*shape):
        return torch.rand(shape, generator=g, device=dev)
    logits = 2 * torch.randn((T, V + wide), generator=g, device=dev)
    likely = torch.randint(0, V, (T, 3), generator=g, device=dev)
    logits.scatter_add_(1, likely, peak * rand(T, 3))
    q = logits + close * torch.randn((T, V + wide), generator=g, device=dev)
    ids = torch.cat((torch.zeros(1, dtype=torch.int64, device=dev), q[:, :V].argmax(1)[:-1])).to(torch.int32)
    t = 0.5 + rand(B)
    if greedy:
        t[::2] = 0
    starts = torch.tensor([sum(counts[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev)
    kept = torch.float32 if f32 else torch.bfloat16
    return dict(logits=logits.to(kept)[:, :V], draft=None if draft is None else q.to(draft)[:, :V], ids=ids, q_start=starts, u=rand(T), u_pick=rand(B), t=t)


def results(dev, T, B):
    return (torch.full((T,), -7, dtype=torch.int32, device=dev), torch.full((B,), -7, dtype=torch.int32, device=dev), torch.full((T,), -7.0, device=dev))


def run_verify(K, dev, s, T=None, ws=None, temperature=True, logp=True):
    T, V = s["logits"].shape
    B = s["u_pick"].shape[0]
    ids, n, lp = results(dev, T, B)
    ws = torch.full((K.verify_drafts_workspace_bytes(T, B, V),), 0xff, dtype=torch.uint8, device=dev) if ws is None else ws
    err = torch.zeros(4, dtype=torch.int32, device=dev)
    K.verify_drafts(s["logits"], s["ids"], s["q_start"], s["u"], s["u_pick"], ids, n, ws, err, draft_logits=s["draft"], temperature=s["t"] if temperature else None,
                    logp=lp if logp else None)
    torch.cuda.synchronize()
    return ids, n, lp, err


def check(K, dev, s, **kw):
    ids, n, lp, err = run_verify(K, dev, s, **kw)
    assert err.tolist() == [0, 0, 0, 0]
    P.check_verified(s["logits"], s["ids"], s["q_start"], s["u"], s["u_pick"], s["draft"], s["t"] if kw.get("temperature", True) else None, ids, n, lp if kw.get("logp", True) else None)
    return ids, n, lp


@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 31, 255, 1000, 4095, 4096, 4097, 4103, 8191, 20000, 100003])
@pytest.mark.parametrize("draft", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("f32", [True, False])
def test_verify(K, cuda, V, draft, f32):
    check(K, cuda, batch(cuda, [1, 4, 2, 8, 1, 3], V, seed=V, f32=f32, draft=draft, greedy=V % 2 == 0))


@pytest.mark.parametrize("draft", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("wide", [1, 2, 3, 5, 8])
def test_verify_rows_that_begin_anywhere(K, cuda, draft, f32, wide):
    check(K, cuda, batch(cuda, [3, 5, 2, 6], 5000, seed=wide, f32=f32, draft=draft, wide=wide))


@pytest.mark.parametrize("draft", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("V", [163841, 327681, 600001, 1 << 20])
def test_verify_long_rows(K, cuda, V, draft, f32):
    """More chunks than a warp holds, more than a CTA has threads, the largest."""
    check(K, cuda, batch(cuda, [2, 1, 3], V, seed=V, f32=f32, draft=draft))


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_verify_many_sequences(K, cuda, draft):
    counts = [1 + (7 * b) % 5 for b in range(300)]
    ids, n, _ = check(K, cuda, batch(cuda, counts, 777, seed=1, draft=draft, greedy=True, peak=9.0))
    assert n.min() == 1 and n.max() == 5  # some of everything


@pytest.mark.parametrize("draft", [None, torch.bfloat16])
def test_verify_the_most_sequences(K, cuda, draft):
    ids, n, _ = check(K, cuda, batch(cuda, [1 + (b % 7 == 3) for b in range(8192)], 130, seed=16, draft=draft, greedy=True))
    assert n.min() == 1 and n.max() == 2


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_verify_long_runs_of_drafts(K, cuda, draft):
    """More rows of one sequence than a CTA has warps, kept to the end and refused far inside."""
    s = batch(cuda, [40, 9, 17], 500, seed=2, draft=draft, close=0.05, peak=40.0)
    s["u"][:] = 0.0
    s["ids"][1:] = s["logits"].argmax(1)[:-1].to(torch.int32)
    s["u"][60] = 0.999999  # may refuse in the last sequence
    s["ids"][61] = (s["ids"][61] + 1) % 500
    ids, n, _ = check(K, cuda, s)
    assert n[0] == 40 and n[1] == 9


def test_verify_defaults(K, cuda):
    s = batch(cuda, [2, 3], 300, seed=3)
    ids, n, lp = check(K, cuda, s, temperature=False)
    again, n2, untouched, _ = run_verify(K, cuda, s, temperature=False, logp=False)
    assert torch.equal(ids, again) and torch.equal(n, n2) and torch.all(untouched == -7.0)


@pytest.mark.parametrize("u", [0.0, 0.25, 1 - 2.0 ** -24])
@pytest.mark.parametrize("draft", [None, torch.float32])
def test_verify_masked_tokens(K, cuda, u, draft):
    """Rows with -inf, with the type's lowest value, with one token left."""
    s = batch(cuda, [3, 3, 3, 3], 6000, seed=4, draft=draft)
    low = torch.finfo(torch.float32).min
    for t in [s["logits"]] + ([s["draft"]] if draft else []):
        t[0:3, 100:5900] = -float("inf")
        t[3:6, ::2] = low
        t[6:9] = -float("inf")
        t[6:9, 5555] = 3.0
        t[9:12] = low
    s["t"][1] = 0.1
    s["ids"][1:3], s["ids"][4:6], s["ids"][7:9] = 50, 4001, 5555
    s["u_pick"][:], s["u"][:] = u, 0.5
    ids, n, _ = check(K, cuda, s)
    assert ids[6:9].tolist() == [5555] * 3 and n[2] == 3


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_verify_greedy_ties_go_to_the_lowest(K, cuda, draft):
    s = batch(cuda, [2, 1], 9000, seed=5, draft=draft)
    s["t"][:] = 0
    s["logits"][:] = -1.0
    s["logits"][0, [8000, 4095, 4096, 5000]] = 2.0
    s["logits"][1, [8999]] = 2.0
    s["logits"][2] = -float("inf")
    s["logits"][2, 1:] = -5.0
    s["ids"][1] = 4095
    s["u"][:] = float("nan")  # not read
    ids, n, _ = check(K, cuda, s)
    assert ids.tolist() == [4095, 8999, 1] and n.tolist() == [2, 1]


def test_verify_extreme_temperatures_and_logits(K, cuda):
    s = batch(cuda, [2, 2, 2, 2], 3000, seed=6)
    s["t"][:] = torch.tensor([2.0 ** -126, 1e30, 1e-3, 1.0], device=cuda)
    s["logits"][6:8] *= 1e37
    check(K, cuda, s)


@pytest.mark.parametrize("f32", [True, False])
def test_verify_same_distribution_keeps_everything(K, cuda, f32):
    s = batch(cuda, [4, 4], 2000, seed=7, f32=f32, draft=torch.float32 if f32 else torch.bfloat16)
    s["draft"] = s["logits"].clone()
    s["u"][:] = 1 - 2.0 ** -10
    ids, n, _ = check(K, cuda, s)
    assert n.tolist() == [4, 4] and torch.equal(ids[0:3], s["ids"][1:4])


def test_verify_drafted_token_without_a_chance(K, cuda):
    """Masked in the target, or in the drafter's own distribution; and nothing but the refused token."""
    s = batch(cuda, [2, 2, 2], 1000, seed=8, draft=torch.float32)
    s["logits"][0, s["ids"][1]] = -float("inf")
    s["draft"][2, s["ids"][3]] = -float("inf")
    s["u"][2] = 0.0
    ids, n, _ = check(K, cuda, s)
    assert n[0] == 1 and n[1] == 2
    s = batch(cuda, [2], 50, seed=9)
    s["logits"][0] = -float("inf")
    s["logits"][0, 7], s["logits"][0, 9] = 30.0, -200.0  # the rest has a weight below 2^-126
    s["ids"][1], s["u"][0] = 9, 0.5
    ids, n, _, _ = run_verify(K, cuda, s)
    assert ids.tolist() == [7, -1] and n.tolist() == [1]


def test_verify_empty_sequences_and_rows_of_none(K, cuda):
    s = batch(cuda, [2, 3, 4], 600, seed=10, greedy=True)
    s["q_start"] = torch.tensor([1, 1, 4, 4, 7], dtype=torch.int32, device=cuda)  # rows 0, 7 and 8 are nobody's
    s["u_pick"], s["t"] = torch.rand(4, device=cuda), torch.tensor([1.0, 0.7, 1.0, 0.0], device=cuda)
    s["logits"][0], s["logits"][8] = float("nan"), float("nan")
    ids, n, lp, err = run_verify(K, cuda, s)
    assert err.tolist() == [0, 0, 0, 0] and n[0] == 0 and n[2] == 0
    P.check_verified(s["logits"], s["ids"], s["q_start"], s["u"], s["u_pick"], None, s["t"], ids, n, lp)
    assert ids[[0, 7, 8]].tolist() == [-7] * 3 and lp[[0, 7, 8]].tolist() == [-7.0] * 3


@pytest.mark.parametrize("draft", [None, torch.float32])
@pytest.mark.parametrize("name", ["nan", "inf", "masked", "id", "negative id", "u", "u nan", "u_pick", "temperature", "temperature nan", "drafter"])
def test_verify_data_errors(K, cuda, name, draft):
    """The sequence is refused, the others are not."""
    if name == "drafter" and draft is None:
        pytest.skip("there is no drafter's distribution")
    s = batch(cuda, [3, 3, 3], 5000, seed=11, draft=draft)
    s["u"][:] = 0.0  # every draft with a chance is kept: all rows are read
    for i, value in ((4, 3), (5, 4999)):
        s["ids"][i] = value
    code, row = {"nan": 1, "inf": 1, "masked": 1, "id": 3, "negative id": 3, "u": 4, "u nan": 4, "u_pick": 4, "temperature": 5, "temperature nan": 5, "drafter": 2}[name], 4
    if name in ("nan", "inf"):
        s["logits"][4, 4200] = float(name)
    elif name == "masked":
        s["logits"][4] = -float("inf")
    elif name in ("id", "negative id"):
        s["ids"][5] = 5000 if name == "id" else -1
    elif name in ("u", "u nan"):
        s["u"][4] = 1.0 if name == "u" else float("nan")
    elif name == "u_pick":
        s["u_pick"][1], row = -0.5, 5
    elif name == "drafter":
        s["draft"][4, 4999] = float("nan")
    else:
        s["t"][1], row = (-1.0 if name == "temperature" else float("nan")), 3
    ids, n, lp, err = run_verify(K, cuda, s)
    assert err[:3].tolist() == [1, row, code]
    assert n[1] == 0 and ids[3:6].tolist() == [-1] * 3 and torch.all(lp[3:6].isnan())
    P.check_verified(s["logits"], s["ids"], s["q_start"], s["u"], s["u_pick"], s["draft"], s["t"], ids, n, lp, skip=(1,))
    with pytest.raises(K.Error):
        K.check_verify_error(err, "step")


def test_verify_errors_behind_the_decision_do_not_count(K, cuda):
    s = batch(cuda, [4], 2000, seed=12)
    s["u"][:] = 1 - 2.0 ** -24
    s["ids"][1] = 1999
    s["logits"][0, 1999] = -3.0
    s["logits"][2], s["ids"][3] = float("nan"), -5
    ids, n, lp, err = run_verify(K, cuda, s)
    assert err.tolist() == [0, 0, 0, 0] and n.tolist() == [1] and ids[1:].tolist() == [-1] * 3


@pytest.mark.parametrize("starts,bad", [([0, 3, 2, 5], (1, 2)), ([-1, 3, 5, 6], (0,)), ([0, 3, 5, 100], (2,)), ([0, 50, 3, 5], (0, 1, 2))])
def test_verify_bad_row_ranges(K, cuda, starts, bad):
    s = batch(cuda, [2, 2, 2], 800, seed=13)
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=cuda)
    ids, n, lp, err = run_verify(K, cuda, s)
    assert err[0] == 1 and int(err[1]) in bad and err[2] == 6
    assert all(n[b] == 0 for b in bad)
    P.check_verified(s["logits"], s["ids"], s["q_start"], s["u"], s["u_pick"], None, s["t"], ids, n, lp, skip=bad)


def test_verify_beyond_32_bits(K, cuda):
    """Rows 2^31 elements and more behind the first."""
    V, T = 1 << 20, 2100
    logits = torch.zeros((T, V), dtype=torch.bfloat16, device=cuda)
    g = gen(14, cuda)
    logits[T - 3:] = torch.randn((3, V), generator=g, device=cuda).to(torch.bfloat16) * 3
    s = dict(logits=logits, draft=None, ids=torch.full((T,), 77, dtype=torch.int32, device=cuda), q_start=torch.tensor([T - 3, T], dtype=torch.int32, device=cuda),
             u=torch.full((T,), 0.5, device=cuda), u_pick=torch.rand(1, generator=g, device=cuda), t=torch.ones(1, device=cuda))
    ids, n, lp, err = run_verify(K, cuda, s)
    tail = {k: (v[T - 3:] if k in ("logits", "ids", "u") else v) for k, v in s.items()}
    P.check_verified(tail["logits"], tail["ids"], torch.tensor([0, 3], dtype=torch.int32), tail["u"], s["u_pick"], None, s["t"], ids[T - 3:], n, lp[T - 3:])
    assert torch.all(ids[:T - 3] == -7)


# ---- together ------------------------------------------------------------------------------------------------------------------------------

def head(K, dev, d=512, V=3000, T=24, B=4, seed=0):
    from strixite_b200.head import HeadBuffers, HeadWeights, VerifyHead
    g = gen(seed, dev)
    w = K.quantize_f8(torch.randn((V, d), generator=g, device=dev) * 0.2)
    buf = HeadBuffers(T, B, d, V, dev)
    return VerifyHead(HeadWeights(w, 1 + 0.1 * torch.randn(d, generator=g, device=dev)), buf), buf


@pytest.mark.parametrize("counts", [[1], [8, 8], [3, 1, 5, 2], [6, 6, 6, 6]])
def test_head(K, cuda, counts):
    h, buf = head(K, cuda)
    g = gen(21, cuda)
    T, B, d = sum(counts), len(counts), 512
    x, y = (torch.randn((T, d), generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    starts = torch.tensor([sum(counts[:b]) for b in range(B + 1)], dtype=torch.int32, device=cuda)
    ids = torch.randint(0, 3000, (T,), generator=g, device=cuda, dtype=torch.int32)
    u, u_pick, t = torch.rand(T, generator=g, device=cuda) * 0.01, torch.rand(B, generator=g, device=cuda), torch.ones(B, device=cuda)
    for drafts in (False, True):
        q = torch.randn((T, 3000), generator=g, device=cuda) if drafts else None
        next_ids, n_new, logp = h.forward(x, y, ids, starts, u, u_pick, draft_logits=q, temperature=t)
        h.check_errors()
        s = (x.float() + y.float()).to(torch.bfloat16)
        assert torch.equal(buf.total[:T], s)
        n = P.norm(P.f64(s), h.w.norm, 1e-6)
        P.check_codes(buf.codes[:T], buf.scales[:T], n, P.NORM)
        want, size, nb = P.linear(buf.codes[:T], buf.scales[:T], h.w.out.q, h.w.out.scale)
        assert np.all(np.abs(P.f64(buf.logits[:T]) - want) <= P.linear_bound(want, size, nb, False))
        P.check_verified(buf.logits[:T], ids, starts, u, u_pick, q, t, next_ids, n_new, logp)


def test_head_captured_and_replayed(K, cuda):
    """A step as a graph follows the batch that it finds: other rows, ranges and random numbers."""
    h, buf = head(K, cuda)
    g = gen(22, cuda)
    T, B, d = 12, 3, 512
    x, y = (torch.zeros((T, d), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    starts, ids = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=cuda), torch.zeros(T, dtype=torch.int32, device=cuda)
    u, u_pick, t = torch.zeros(T, device=cuda), torch.zeros(B, device=cuda), torch.ones(B, device=cuda)
    h.forward(x, y, ids, starts, u, u_pick, temperature=t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = h.forward(x, y, ids, starts, u, u_pick, temperature=t)
    for counts in ([4, 4, 4], [1, 10, 1], [0, 3, 9]):
        x.copy_(torch.randn((T, d), generator=g, device=cuda))
        y.copy_(torch.randn((T, d), generator=g, device=cuda))
        starts.copy_(torch.tensor([sum(counts[:b]) for b in range(B + 1)], dtype=torch.int32))
        ids.copy_(torch.randint(0, 3000, (T,), generator=g, device=cuda))
        u.copy_(torch.rand(T, generator=g, device=cuda) * 0.01)
        u_pick.copy_(torch.rand(B, generator=g, device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        h.check_errors()
        P.check_verified(buf.logits[:T], ids, starts, u, u_pick, None, t, *out)
        eager = [v.clone() for v in out]
        h.forward(x, y, ids, starts, u, u_pick, temperature=t)
        assert all(torch.equal(a, b) for a, b in zip(eager, out))


def test_two_streams_at_once(K, cuda):
    """Calls with buffers of their own on two streams, many times."""
    heads = [head(K, cuda, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    g = gen(23, cuda)
    T, B = 16, 2
    x = torch.randn((T, 512), generator=g, device=cuda).to(torch.bfloat16)
    ids = torch.randint(0, 3000, (T,), generator=g, device=cuda, dtype=torch.int32)
    starts, u, u_pick = torch.tensor([0, 8, 16], dtype=torch.int32, device=cuda), torch.rand(T, generator=g, device=cuda), torch.rand(B, generator=g, device=cuda)
    alone = []
    for h, _ in heads:
        alone.append([v.clone() for v in h.forward(x, None, ids, starts, u, u_pick)])
    torch.cuda.synchronize()
    for _ in range(20):
        for (h, _), st in zip(heads, streams):
            with torch.cuda.stream(st):
                h.forward(x, None, ids, starts, u, u_pick)
    torch.cuda.synchronize()
    for (h, buf), want in zip(heads, alone):
        assert torch.equal(buf.next_ids[:T], want[0]) and torch.equal(buf.n_new[:B], want[1]) and torch.equal(buf.logp[:T], want[2])


def test_python_refusals(K, cuda):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(K.Error, match="out is torch.float32"):
        K.add_norm(x, out=torch.zeros((4, 64), device=cuda))
    with pytest.raises(K.Error, match="y is torch.bfloat16 on cpu"):
        K.add_norm(x, torch.zeros((4, 64), dtype=torch.bfloat16), total=x)
    with pytest.raises(K.Error, match="shapes do not fit"):
        K.add_norm(x, codes=codes_like(K, (4, 64), cuda), scales=torch.zeros((4, 2), device=cuda))
    with pytest.raises(K.Error, match="strides"):
        K.add_norm(x.t().contiguous().t(), out=torch.zeros_like(x))
    w = K.quantize_f8(torch.randn((32, 64), device=cuda))
    with pytest.raises(K.Error, match="shapes do not fit"):
        K.linear_f8(codes_like(K, (4, 48), cuda), torch.zeros((4, 1), device=cuda), w, torch.zeros((4, 32), device=cuda))
    with pytest.raises(K.Error, match="x is torch.uint8"):
        K.linear_f8(torch.zeros((4, 64), dtype=torch.uint8, device=cuda), torch.zeros((4, 1), device=cuda), w, torch.zeros((4, 32), device=cuda))
    s = batch(cuda, [2, 2], 100, seed=1)
    with pytest.raises(K.Error, match="ids is torch.int64"):
        run_verify(K, cuda, dict(s, ids=s["ids"].long()))
    with pytest.raises(K.Error, match="workspace of 16 bytes"):
        run_verify(K, cuda, s, ws=torch.zeros(16, dtype=torch.uint8, device=cuda))
    from strixite_b200.head import HeadBuffers, HeadWeights, VerifyHead
    with pytest.raises(K.Error, match="VerifyHead"):
        VerifyHead(HeadWeights(w), HeadBuffers(4, 2, 128, 32, cuda))
    h = VerifyHead(HeadWeights(w), HeadBuffers(4, 2, 64, 32, cuda))
    with pytest.raises(K.Error, match="VerifyHead"):
        h.forward(torch.zeros((5, 64), dtype=torch.bfloat16, device=cuda), None, s["ids"], s["q_start"], s["u"], s["u_pick"])

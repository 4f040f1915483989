"""Calls of the operators around the head at which their formulas are easily missed: FP32 values between two codes, logits at FP32's ends, differences of two distributions that
are zero or small, waits that run out, other streams, padded steps."""
import numpy as np
import pytest
import torch

import head_plain as P
from test_gpu_head import batch, check, gen, head, operands, run_verify

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


@pytest.mark.parametrize("T", [1, 3000])
def test_norm_beyond_fp32_counts_as_an_infinity(K, cuda, T):
    """s * weight still fits FP32, its product with the row's factor does not: the block is lost, the others are not."""
    x = torch.full((T, 4096), 1e-3, device=cuda)
    x[:, 130] = 1.0
    codes, scales = torch.zeros(x.shape, dtype=torch.uint8, device=cuda).view(K.F8), torch.zeros((T, 32), device=cuda)
    K.add_norm(x, weight=torch.full((4096,), 1e38, device=cuda), codes=codes, scales=scales)
    v = codes.float() * scales.repeat_interleave(128, 1)
    assert torch.all(scales[:, 1].isnan()) and torch.all(v[:, 128:256].isnan())
    rest = torch.cat((scales[:, :1], scales[:, 2:]), 1)
    n = 1e35 / np.sqrt((1 + 4095e-6) / 4096 + 1e-6)
    assert np.all(np.abs(P.f64(rest) / (n / 448) - 1) <= P.NORM + 4 * P.U)


# ---- product -------------------------------------------------------------------------------------------------------------------------

def gives_up(K, dev, lib, M, N, K_, slot, f32):
    """The product with CTA 0 told to leave stage `slot` out: the kernel returns, the status names the role, the next call has the bits of the call before."""
    x, xs, w, ws = operands(K, dev, M, N, K_, slot)
    v, out = K.F8View(w, ws), [torch.full((M, N), float("nan"), dtype=torch.float32 if f32 else torch.bfloat16, device=dev) for _ in range(3)]
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


@pytest.mark.parametrize("M,N,K_,slot", [(2049, 4099, 1024, 0), (2049, 4099, 1024, 10), (600, 1003, 1024, 3), (2048, 4096, 1024, 9), (600, 1000, 1024, 5)])
@pytest.mark.parametrize("f32", [True, False])
def test_linear_gives_up_a_wait_whatever_way_its_rows_leave(K, cuda, lib, M, N, K_, slot, f32):
    """Rows that turn in shared memory, leave from registers or by tensor copies."""
    gives_up(K, cuda, lib, M, N, K_, slot, f32)


@pytest.mark.parametrize("M,N,K_,slot", [(16, 300, 2048, 0), (32, 300, 2048, 0), (16, 40000, 1024, 2), (32, 40000, 1024, 9), (4, 70000, 1024, 5), (9, 130, 144, 0)])
@pytest.mark.parametrize("f32", [True, False])
def test_linear_of_few_rows_gives_up_a_wait(K, cuda, lib, M, N, K_, slot, f32):
    """Both widths, k shared by a cluster and not, the first tile of a CTA and a later one."""
    gives_up(K, cuda, lib, M, N, K_, slot, f32)


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


def laid_out(dev, rows, dtype, lead):
    """Rows [T, V] as they are in a wider buffer, each `lead` elements behind a multiple of sixteen bytes."""
    T, V = rows.shape
    wide = torch.zeros((T, (V + lead + 15) // 8 * 8), dtype=dtype, device=dev)
    wide[:, lead:lead + V] = rows
    return wide[:, lead:lead + V]


LAYOUTS = [(torch.float32, 0, torch.float32, 0), (torch.float32, 1, torch.float32, 1), (torch.float32, 1, torch.float32, 0), (torch.float32, 2, torch.float32, 3), (torch.bfloat16, 0, torch.bfloat16, 0),
           (torch.bfloat16, 5, torch.bfloat16, 5), (torch.bfloat16, 0, torch.bfloat16, 3), (torch.float32, 0, torch.bfloat16, 0), (torch.bfloat16, 1, torch.float32, 2)]


def drawn(K, dev, p, q, drafted, u, picks, t, layout):
    """Two rows a sequence, each the same p and q [V], the drafted token refused by u: the token drawn for each of picks."""
    (xt, xl, qt, ql), B, V = layout, len(picks), p.shape[0]
    s = dict(logits=laid_out(dev, p.expand(2 * B, V), xt, xl), draft=laid_out(dev, q.expand(2 * B, V), qt, ql), ids=torch.full((2 * B,), drafted, dtype=torch.int32, device=dev),
             q_start=torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device=dev), u=torch.full((2 * B,), u, device=dev), u_pick=torch.tensor(picks, dtype=torch.float32, device=dev),
             t=torch.full((B,), t, device=dev))
    assert torch.equal(s["logits"][0].float(), p) and torch.equal(s["draft"][0].float(), q)
    ids, n, lp, err = run_verify(K, dev, s)
    assert err.tolist() == [0, 0, 0, 0] and torch.all(n == 1) and torch.all(ids[1::2] == -1)
    return ids[::2].tolist(), lp[::2]


def centres(p):
    """The middles of the tokens' shares of [0, 1), of tokens that have some."""
    p = p / p.sum()
    return [(i, c - w / 2) for i, (w, c) in enumerate(zip(p, np.cumsum(p))) if w > 1e-3]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("V", [9, 1000, 9001])
def test_verify_equal_distributions_draw_from_the_target(K, cuda, layout, V):
    """The drafter's row is the target's, the drafted token masked in both: the difference is zero, whatever type and place the rows have, and the token comes from p."""
    g = gen(V, cuda)
    p = 2 * torch.randn(V, generator=g, device=cuda)
    p[torch.randperm(V, generator=g, device=cuda)[40:]] -= 30
    p = p.to(torch.bfloat16).float()
    m = V // 3
    p[m] = -float("inf")
    want = centres(P.softmax(P.f64(p), 0.75))
    said, lp = drawn(K, cuda, p, p, m, 0.0, [c for _, c in want], 0.75, layout)
    assert said == [i for i, _ in want]
    logs = np.log(P.softmax(P.f64(p), 0.75)[said])
    assert np.all(np.abs(P.f64(lp) - logs) <= P.P_OFF + 4 * P.U * np.abs(logs))


@pytest.mark.parametrize("layout", [l for l in LAYOUTS if l[0] == l[2] and l[1] == l[3]])
def test_verify_equal_probabilities_have_no_weight(K, cuda, layout):
    """Weights that are powers of two, so that both sums are exact and alike: all tokens but two have the same chance twice, and the one that has more of it now is drawn for every number."""
    V, a, b = 5000, 4321, 17
    p = -torch.randint(0, 12, (V,), generator=gen(1, cuda), device=cuda).float()
    p[a], p[b] = 0.0, -6.0
    q = p.clone()
    q[a], q[b] = -6.0, 0.0
    said, _ = drawn(K, cuda, p, q, b, 1 - 2.0 ** -24, [0.0, 2.0 ** -24, 0.25, 1 - 2.0 ** -24], float(np.float32(1.4426950408889634)), layout)
    assert said == [a] * 4


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("step", [2.0 ** -8, 2.0 ** -10])
def test_verify_draws_from_a_small_difference(K, cuda, layout, step):
    """Sixteen tokens of 1 / 16, of which the drafter takes `step` from four and gives it to four others: a quarter of the difference's sum 4 step each.  A draw is off by at most
    2^-17 / (4 step), an eighth of which the middles are from their borders."""
    V = 9001
    at = np.sort(np.random.default_rng(5).choice(V, 16, replace=False))
    pp, qq = np.full(16, 1 / 16), np.full(16, 1 / 16)
    more, less = [2, 5, 11, 15], [0, 4, 8, 13]
    qq[more] -= step
    qq[less] += step
    p, q = (torch.full((V,), -float("inf"), device=cuda) for _ in range(2))
    for t, of, kind in ((p, pp, layout[0]), (q, qq, layout[2])):
        t[torch.from_numpy(at).to(cuda)] = torch.from_numpy(np.log(of)).to(cuda).to(kind).float()
    rest = np.maximum(P.softmax(P.f64(p), 1.0) - P.softmax(P.f64(q), 1.0), 0)
    want = centres(rest)
    said, _ = drawn(K, cuda, p, q, int(at[0]), 1 - 2.0 ** -24, [c for _, c in want], 1.0, layout)
    assert said == [i for i, _ in want]


# ---- streams -------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("raw", [False, True])
def test_quantize_on_another_stream(K, cuda, raw):
    """The call's own error words are cleared, written and read on the stream that it was given, not on the current one, which is busy."""
    w = torch.ones((200, 256), device=cuda)
    w[150, 17] = float("inf")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)
    with pytest.raises(K.Error, match=r"non-finite weight at \[150, 17\]"):
        K.quantize_f8(w, stream=st.cuda_stream if raw else st)
    with pytest.raises(K.Error, match=r"non-finite weight at \[150, \d+\]"):
        K.quantize(w, 64, 8, stream=st.cuda_stream if raw else st)
    w[150, 17] = 1.0
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)
    v = K.quantize_f8(w, stream=st.cuda_stream if raw else st)
    st.synchronize()
    with torch.cuda.stream(st):
        assert torch.all(v.scale == 1 / 448) and torch.all(v.q.float() == 448)
    torch.cuda.synchronize()


def test_head_rows_of_no_sequence(K, cuda):
    """A padded step: rows of no sequence and of a refused range say so, instead of what an earlier step left there."""
    h, buf = head(K, cuda)
    g = gen(31, cuda)
    x = torch.randn((12, 512), generator=g, device=cuda).to(torch.bfloat16)
    ids = torch.randint(0, 3000, (12,), generator=g, device=cuda, dtype=torch.int32)
    u, u_pick = torch.rand(12, generator=g, device=cuda), torch.rand(3, generator=g, device=cuda)
    h.forward(x, None, ids, torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=cuda), u, u_pick)
    h.check_errors()
    next_ids, n_new, logp = h.forward(x, None, ids, torch.tensor([1, 3, 3, 7], dtype=torch.int32, device=cuda), u, u_pick)
    h.check_errors()
    assert n_new.tolist()[1] == 0
    for row in (0, 7, 8, 9, 10, 11):
        assert int(next_ids[row]) == -1 and bool(logp[row].isnan())
    P.check_verified(buf.logits[:12], ids, torch.tensor([1, 3, 3, 7]), u, u_pick, None, None, next_ids, n_new, logp)
    next_ids, n_new, logp = h.forward(x, None, ids, torch.tensor([0, 4, 2, 12], dtype=torch.int32, device=cuda), u, u_pick)
    assert n_new.tolist()[1:] == [0, 0] and torch.all(next_ids[4:] == -1) and torch.all(logp[4:].isnan())
    with pytest.raises(K.Error, match="at sequence"):
        h.check_errors()


def test_head_captured_with_a_drafter(K, cuda):
    """A step with the drafter's distributions as a graph, replayed with other batches, padding rows among them: the bits of the same step run at once."""
    h, buf = head(K, cuda)
    g = gen(32, cuda)
    T, B = 12, 3
    x, y = (torch.zeros((T, 512), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    q, ids, starts = torch.zeros((T, 3000), device=cuda), torch.zeros(T, dtype=torch.int32, device=cuda), torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=cuda)
    u, u_pick, t = torch.zeros(T, device=cuda), torch.zeros(B, device=cuda), torch.tensor([1.0, 0.6, 0.0], device=cuda)
    call = (x, y, ids, starts, u, u_pick, q, t)
    h.forward(*call)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = h.forward(*call)
    for at in ([0, 4, 8, 12], [1, 11, 11, 12], [0, 2, 5, 9], [3, 3, 3, 3]):
        x.copy_(torch.randn((T, 512), generator=g, device=cuda))
        y.copy_(torch.randn((T, 512), generator=g, device=cuda))
        q.copy_(4 * torch.randn((T, 3000), generator=g, device=cuda))
        starts.copy_(torch.tensor(at, dtype=torch.int32))
        ids.copy_(torch.randint(0, 3000, (T,), generator=g, device=cuda))
        u.copy_(torch.rand(T, generator=g, device=cuda))
        u_pick.copy_(torch.rand(B, generator=g, device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        h.check_errors()
        P.check_verified(buf.logits, ids, starts, u, u_pick, q, t, *out)
        nobody = [r for r in range(T) if not at[0] <= r < at[3]]
        assert torch.all(out[0][nobody] == -1) and torch.all(out[2][nobody].isnan())
        graphed = [v.view(torch.int32).clone() for v in out]
        h.forward(*call)
        assert all(torch.equal(a, b.view(torch.int32)) for a, b in zip(graphed, out))

"""GPU tests of the attention operators at their edges: what is not finite, values of very different sizes, caps of any size, log-sums in every row, far pages,
long chunks.  The definition in 64 bits and the bounds are attn_plain.py's; what differs from them is derived beside the test."""
import numpy as np
import pytest
import torch

import attn_plain as plain
from test_gpu_attn import Batch, K, Rows

pytestmark = pytest.mark.gpu

UNTOUCHED = 2.0 ** 120  # a BF16 number that no case comes to


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


@pytest.mark.parametrize("D,bits,G", QUANT)
@pytest.mark.parametrize("power", [-6, -9, -12, -20, -40, 9, 20, 40])
def test_value_groups_of_very_different_sizes(cuda, D, bits, G, power):
    """A head's last group is 2^power times as large as the others, and every seventh key's first group: each column is as exact as by itself."""
    for group, new in ((1, 1), (4, 3)):
        b = Batch(cuda, D, bits, G, 2, group, [900, 41], [new, new], seed=D + bits + power)
        b.cache.v_sm[..., -1, :] *= 2.0 ** power
        b.cache.v_sm[:, :, 3::7, 0, :] *= 2.0 ** power
        run_and_compare(b)


def against(cache, page, head, at, q, score, scale):
    """Makes the key at (page, head, at) one whose score with the query row q is `score`, by the library's quantizer."""
    x = q.float() * (score / (scale * float((q.float() ** 2).sum())))
    w = K().quantize(x.view(1, -1).contiguous(), cache.G, cache.bits)
    cache.k[page, head, at] = w.q.view(-1)
    cache.k_sm[page, head, at] = torch.stack((w.scale, w.minv), -1).view(torch.bfloat16).view(cache.k_sm.shape[-2:])


@pytest.mark.parametrize("D,bits,G", QUANT)
@pytest.mark.parametrize("power", [14, 24, 40])
def test_a_large_value_that_a_row_does_not_look_at(cuda, D, bits, G, power):
    """One key's values are 2^power times the others', and its weight in the first query head is far below 2^-power (in the second it has its way): the first
    head's output is the other keys'.  The key comes first, in the middle, last."""
    for at in (0, 200, 511):
        b = Batch(cuda, D, bits, G, 1, 2, [512], [1], seed=D + bits + power)
        page, row = int(b.pages[0, at // 16]), at % 16
        against(b.cache, page, 0, row, b.q[0, :D], -60.0, D ** -0.5)
        b.cache.v_sm[page, 0, row] *= 2.0 ** power
        got, want = run_and_compare(b)
        assert np.abs(want[0, 0]).max() < 10.0


@pytest.mark.parametrize("still", [False, True], ids=["scores", "alike"])
@pytest.mark.parametrize("D,bits,G", [(128, 4, 32), (128, 8, 64), (128, 16, 0), (256, 4, 64), (64, 4, 32)])
def test_many_thousand_keys_a_warp(cuda, D, bits, G, still):
    """So many long sequences that a warp sums up thousands of keys by itself: what the codes are too large by, and what an accumulator rounds off in every step,
    must not add up."""
    B, n_kv, page = 64, 2, 256
    keys = (3 << 30) // (B * n_kv * 2 * (D * bits // 8 + (0 if bits == 16 else 4 * D // G)))
    b = Batch(cuda, D, bits, G, n_kv, 1, [keys] * B, [1] * B, page=page, seed=bits)
    if still:
        b.q.zero_()
    b.out.fill_(UNTOUCHED), b.lse.fill_(UNTOUCHED)
    b.run()
    torch.cuda.synchronize()
    for s in (7,):
        want, lse, tol, lse_tol = plain.attend(b.q[s:s + 1], b.cache, b.pages[s:s + 1], b.q_start[:2], b.kv_len[s:s + 1], D ** -0.5)
        got = plain.f64(b.out[s]).reshape(want.shape)
        assert (np.abs(got - want) <= tol).all(), ((np.abs(got - want) / tol).max(), (np.abs(got - want) / (np.abs(want) + 1e-30)).max())
        assert (np.abs(plain.f64(b.lse[s:s + 1]) - lse) <= lse_tol).all()


# ---- the cap -------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cap", [1e-6, 1e-3, 0.7, 5.0, 50.0, 1e3, 1e6, 1e9, 9e29])
@pytest.mark.parametrize("D,bits,G,group,new", [(128, 16, 0, 4, 2), (128, 16, 0, 70, 2), (64, 8, 32, 4, 2), (256, 4, 64, 8, 2)], ids=["bf16", "rows140", "q8", "q4"])
def test_caps_of_any_size(cuda, D, bits, G, group, new, cap):
    """The capped score is as good as a score is in FP32, whatever the cap.

    cap * tanh(s / cap) is within 2^-19 of itself: below a quarter of the cap by four terms of the odd series (the fifth is 2^-21.5) with a handful of roundings;
    above by 1 - 2 r, r = 1 / (exp(2 s / cap) + 1), whose exponential is off by 2^-22, its sum by 2^-24, the reciprocal by 2^-23: at a quarter
    0.755 * (0.62 + 0.25 + 0.5) * 2^-22 of a tanh of 0.245, 2^-19.9, and less above."""
    b = Batch(cuda, D, bits, G, 1, group, [300, 40], [new, new], seed=9)
    scale = 0.3
    b.out.fill_(UNTOUCHED), b.lse.fill_(UNTOUCHED)
    b.run(scale=scale, softcap=cap)
    torch.cuda.synchronize()
    assert int(b.err[0]) == 0 and (b.guard == 0xA5).all()
    q, got, got_lse = plain.f64(b.q).reshape(b.T, group, D), plain.f64(b.out).reshape(b.T, group, D), plain.f64(b.lse)
    kept, t = plain.BF16 if bits == 16 else plain.F16, 0
    for s, (n, length) in enumerate(zip(b.new, b.lens)):
        j = np.arange(length)
        page = b.pages[s].cpu().numpy()[j // 16].astype(np.int64)
        k, k_scaled, k_least = plain.values(b.cache, "k", page, 0, j % 16)
        v, v_scaled, v_least = plain.values(b.cache, "v", page, 0, j % 16)
        for i in range(n):
            last = length - n + i + 1
            x = q[t].T
            raw = (k[:last] @ x) * scale
            off = (D / 16 + 4) * 2.0 ** -22 * ((k_scaled + k_least)[:last] @ np.abs(x)) * scale
            sc = cap * np.tanh(raw / cap)
            off = np.minimum(off, 2 * cap) + 2.0 ** -19 * np.abs(sc)
            top = sc.max(0)
            w = np.exp(sc - top)
            lse = top + np.log(w.sum(0))
            w = w / w.sum(0)
            want = w.T @ v[:last]
            of_weights = (2 * off.max(0) + 2.0 ** -20)[:, None]
            tol = plain.BF16 * np.abs(want) + (kept + of_weights) * (w.T @ v_scaled[:last]) + (of_weights + 2.0 ** -20) * (w.T @ v_least[:last]) + 1e-30
            assert (np.abs(got[t] - want) <= tol).all(), (cap, (np.abs(got[t] - want) / tol).max())
            assert (np.abs(got_lse[t] - lse) <= off.max(0) + 2.0 ** -20 + 2.0 ** -22 * np.abs(lse)).all(), cap
            t += 1


# ---- the write -----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 16), (128, 32), (128, 64), (256, 32)])
def test_write_leaves_what_it_does_not_turn_alone(cuda, D, rot, f32, interleaved):
    """Without a norm the elements behind the first rot go through as they are, infinities and NaN too, and none reaches its neighbour."""
    r = Rows(cuda, 5, 2, 3, 2, D, 16, 0, f32=f32, seed=D + rot, norm=False)
    x = r.qkv.view(5, 7, D)
    x[0, :, rot], x[1, :, rot + 3], x[2, :, D - 1], x[3, :, rot + 8] = float("inf"), -float("inf"), float("nan"), float("inf")
    K().attn_qkv_write(r.qkv, r.cache, r.seq, r.pos, r.pages, r.q_out, r.err, inv_freq=r.inv_freq(rot), interleaved=interleaved)
    k, v = r.read()
    torch.cuda.synchronize()
    assert int(r.err[0]) == 0
    bits = x.to(torch.bfloat16)
    q = r.q_out.view(5, 3, D)
    for got, put in ((q[..., rot:], bits[:, :3, rot:]), (k[..., rot:], bits[:, 3:5, rot:].float()), (v, bits[:, 5:].float())):
        assert torch.equal(torch.isnan(got), torch.isnan(put))
        assert torch.equal(got.nan_to_num(nan=0.0, posinf=1e9, neginf=-1e9), put.nan_to_num(nan=0.0, posinf=1e9, neginf=-1e9))
    assert torch.isfinite(q[..., :rot]).all() and torch.isfinite(k[..., :rot]).all()


# ---- every row's log-sum -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("group,new", [(4, 1), (8, 2), (3, 7), (8, 8), (8, 17)], ids=["rows4", "rows16", "rows21", "rows64", "rows136"])
@pytest.mark.parametrize("D,bits,G", [(64, 16, 0), (128, 16, 0), (256, 16, 0), (128, 8, 64), (256, 4, 32)])
def test_every_log_sum_is_written(cuda, D, bits, G, group, new):
    """Rows without a key, with one, in whole segments and in joined ones: an output and a log-sum each, none left as it was, none NaN."""
    b = Batch(cuda, D, bits, G, 2, group, [1, new, 65, 0, 6000, max(1, new - 2)], [1, new, new, 1, new, new], page=16, seed=D + bits + group)
    run_and_compare(b)


def test_log_sums_beside_rows_of_no_sequence(cuda):
    """Ranges that begin behind row 0 and leave rows out: their log-sums, and the others as they were."""
    for group in (2, 40):
        b = Batch(cuda, 128, 16, 0, 2, group, [40, 20, 333], [2, 1, 1], seed=8)
        q = torch.randn((9, b.n_q * 128), device=cuda).to(torch.bfloat16)
        out, lse = torch.full_like(q, UNTOUCHED), torch.full((9, b.n_q), UNTOUCHED, device=cuda)
        starts = torch.tensor([1, 3, 3, 4], dtype=torch.int32, device=cuda)  # rows 1-2, none, row 3
        K().attn_decode(q, b.cache, b.pages, starts, b.kv_len, 2, out, b.ws, b.err, lse=lse)
        torch.cuda.synchronize()
        want, want_lse, tol, lse_tol = plain.attend(q, b.cache, b.pages, starts, b.kv_len, 128 ** -0.5)
        assert (np.abs(plain.f64(out).reshape(want.shape)[1:4] - want[1:4]) <= tol[1:4]).all() and (np.abs(plain.f64(lse)[1:4] - want_lse[1:4]) <= lse_tol[1:4]).all()
        rest = [0, 4, 5, 6, 7, 8]
        assert (lse[rest] == UNTOUCHED).all() and (out[rest] == UNTOUCHED).all()


# ---- far pages, long chunks ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("page,token_major", [(64, False), (8, False), (64, True), (8, True)])
def test_many_rows_beyond_32_bits(cuda, page, token_major):
    """Tiles of 128 rows and of 32 on pages that lie more than 2^32 bytes behind a pool's start: by tensor copies, and row by row (pages of eight)."""
    D, n_kv = 128, 8
    n_pages = (9 << 30) // (n_kv * page * D * 2)
    shape = (n_pages, page, n_kv, D) if token_major else (n_pages, n_kv, page, D)
    k, v = (torch.empty(shape, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    if token_major:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    cache = K().KvCache(k, v, 16)
    n, g = 150, torch.Generator(device=cuda)
    g.manual_seed(page)
    used = -(-n // page)
    pages = torch.randperm(used, generator=g, device=cuda).add(n_pages - used).to(torch.int32).view(1, used)
    for t in (k, v):
        t[n_pages - used:] = torch.randn((used, n_kv, page, D), generator=g, device=cuda).to(torch.bfloat16)
    err = torch.zeros(4, dtype=torch.int32, device=cuda)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    for new in (17, 3, 1):  # of eight heads a key head: 136, 24 and 8 rows
        q = torch.randn((new, n_kv * 8 * D), generator=g, device=cuda).to(torch.bfloat16)
        out, lse = torch.empty_like(q), torch.empty((new, n_kv * 8), device=cuda)
        ws = torch.zeros(K().attn_decode_workspace_bytes(cache, n_kv * 8, new), dtype=torch.uint8, device=cuda)
        starts = torch.tensor([0, new], dtype=torch.int32, device=cuda)
        K().attn_decode(q, cache, pages, starts, lens, new, out, ws, err, lse=lse)
        want, want_lse, tol, lse_tol = plain.attend(q, cache, pages, starts, lens, D ** -0.5)
        assert (np.abs(plain.f64(out).reshape(want.shape) - want) <= tol).all() and (np.abs(plain.f64(lse) - want_lse) <= lse_tol).all()
    assert int(err[0]) == 0
    K().check_dense_status("far pages")


@pytest.mark.parametrize("kept,window", [(0, 0), (6144, 0), (1000, 1024)])
def test_a_chunk_of_2048_tokens(cuda, kept, window):
    """A prompt's first chunk, one far into a context, one behind a window: rows at the tiles' ends and among them against the definition."""
    new, group, D = 2048, 8, 128
    b = Batch(cuda, D, 16, 0, 2, group, [kept + new], [new], page=64, seed=kept)
    b.out.fill_(UNTOUCHED), b.lse.fill_(UNTOUCHED)
    b.run(window=window)
    torch.cuda.synchronize()
    K().check_dense_status("chunk")
    assert int(b.err[0]) == 0 and (b.guard == 0xA5).all() and not (b.out == UNTOUCHED).any() and not (b.lse == UNTOUCHED).any()
    assert torch.isfinite(b.out).all() and torch.isfinite(b.lse).all()
    # tiles are of sixteen tokens; the last sixteen rows a call: a sequence of its own that ends with the row
    for t in (0, 1, 15, 16, 17, 127, 128, 1000, 1023, 1024, 2031, 2032, 2047):
        lens = torch.tensor([kept + t + 1], dtype=torch.int32, device=cuda)
        want, lse, tol, lse_tol = plain.attend(b.q[t:t + 1], b.cache, b.pages, torch.tensor([0, 1]), lens, D ** -0.5, 0.0, window)
        assert (np.abs(plain.f64(b.out[t:t + 1]).reshape(want.shape) - want) <= tol).all(), t
        assert (np.abs(plain.f64(b.lse[t:t + 1]) - lse) <= lse_tol).all(), t


# ---- waits that run out ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("slot", [0, 1, 5, 9])
@pytest.mark.parametrize("lens,new,page", [([60000], 17, 64), ([300] * 64, 17, 64), ([3000] * 6, 17, 8)], ids=["long", "many", "rows"])
def test_many_rows_give_up_a_wait(cuda, lib, lens, new, page, slot):
    """Tiles of 128 rows with CTA 0 told to leave one fill of keys and values out: the first, one behind a full turn of the places, one in a later segment.  The kernel
    returns and frees what it holds, the status names the role, every output is the right one, NaN or untouched - nothing of the call before -, and the next
    calls on the context, over the same workspace, have the bits of the first."""
    b = Batch(cuda, 128, 16, 0, 8, 8, lens, [new] * len(lens), page=page, seed=2)
    b.run()
    torch.cuda.synchronize()
    K().check_dense_status("warm-up")
    want, q = (b.out.clone(), b.lse.clone()), b.q.clone()
    b.q.copy_(torch.randn(b.q.shape, device=cuda))  # other parts in the workspace
    b.run()
    b.q.copy_(q)
    b.out.fill_(UNTOUCHED), b.lse.fill_(UNTOUCHED)
    try:
        K().set_wait_limit(2_000_000)
        assert lib.sxb_test_skip_ring_slot(slot) == 0
        b.run()
        torch.cuda.synchronize()
    finally:
        lib.sxb_test_skip_ring_slot(-1)
        K().set_wait_limit(2_000_000_000)
    with pytest.raises(K().Error, match=r"skipped fill: the attention of many rows gave up a wait in CTA 0 \((a copy warp|the MMA warp|a softmax warp) waiting for .*\); its outputs are incomplete"):
        K().check_dense_status("skipped fill")
    for got, right in zip((b.out, b.lse), want):
        assert ((got == right) | torch.isnan(got) | (got == UNTOUCHED)).all() and not torch.equal(got, right)
    for _ in range(3):
        b.out.fill_(UNTOUCHED), b.lse.fill_(UNTOUCHED)
        b.run()
        torch.cuda.synchronize()
        K().check_dense_status("after")
        assert torch.equal(b.out, want[0]) and torch.equal(b.lse, want[1])
    assert (b.guard == 0xA5).all() and int(b.err[0]) == 0


# ---- the sublayer ---------------------------------------------------------------------------------------------------------------------

def small_layer(device, D, n_q, n_kv, d, bits, G, max_tokens, max_q, n_pages, page, seed):
    from strixite_b200.attention import AttnBuffers, AttnLayer, AttnWeights
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    def weight(n, k):
        return K().quantize(torch.randn((n, k), generator=g, device=device) * 0.05, 64, 8)
    inv = (1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().to(device)
    cache = K().KvCache.empty(n_pages, n_kv, page, D, bits, G, device)
    norms = [1 + 0.1 * torch.randn(D, generator=g, device=device) for _ in range(2)]
    layer = AttnLayer(AttnWeights(weight((n_q + 2 * n_kv) * D, d), weight(d, n_q * D), *norms, inv), n_q, cache, AttnBuffers(max_tokens, max_q, n_q, cache))
    return layer, g


def test_layer_shows_nothing_of_earlier_steps(cuda):
    """Padding rows and rows of a refused range after a step that had other conversations in the same buffers: zeros and NaN, the rest as without them."""
    from strixite_b200.attention import AttnBatch
    d = 256
    layer, g = small_layer(cuda, 64, 4, 2, d, 8, 32, 16, 16, 20, 16, 3)
    pages = torch.arange(20, dtype=torch.int32, device=cuda).view(4, 5)
    x = torch.randn((16, d), generator=g, device=cuda).to(torch.bfloat16)
    y = torch.empty_like(x)
    layer.forward(x, AttnBatch.of((0, 0, 0, 0), (9, 5, 1, 1), pages), y)
    layer.check_errors()
    x = torch.randn((8, d), generator=g, device=cuda).to(torch.bfloat16)
    want, got = torch.empty((3, d), dtype=torch.bfloat16, device=cuda), torch.empty((8, d), dtype=torch.bfloat16, device=cuda)
    plain_batch = AttnBatch.of((9, 5), (2, 1), pages[:2])
    layer.forward(x[:3].contiguous(), plain_batch, want)
    batch = AttnBatch.of((9, 5), (2, 1), pages[:2])
    batch.seq = torch.cat((batch.seq, torch.full((5,), -1, dtype=torch.int32, device=cuda)))
    batch.pos = torch.cat((batch.pos, torch.zeros(5, dtype=torch.int32, device=cuda)))
    layer.forward(x, batch, got)
    layer.check_errors()
    assert torch.equal(got[:3], want) and (got[3:] == 0).all()
    batch.q_start[2] = 99  # the second sequence's range is refused
    layer.forward(x, batch, got)
    assert torch.equal(got[:2], want[:2]) and torch.isnan(got[2]).all() and (got[3:] == 0).all()
    with pytest.raises(K().Error, match="rows of a refused range"):
        layer.check_errors()


def test_layer_of_chunks_on_tcgen05(cuda):
    """Heads of 128 over a BF16 cache: a prompt in chunks of many rows a key head, then a step of one token; the attention is the definition's."""
    from strixite_b200.attention import AttnBatch
    d, n_q, n_kv, D = 256, 8, 2, 128
    layer, g = small_layer(cuda, D, n_q, n_kv, d, 16, 0, 300, 200, 40, 16, 5)
    pages = torch.randperm(40, generator=g, device=cuda).to(torch.int32).view(2, 20)
    kept = [0, 0]
    for new in ((200, 33), (90, 1), (1, 40), (1, 1)):
        T = sum(new)
        x = torch.randn((T, d), generator=g, device=cuda).to(torch.bfloat16)
        batch = AttnBatch.of(kept, new, pages)
        kept = [k + n for k, n in zip(kept, new)]
        y = torch.empty((T, d), dtype=torch.float32, device=cuda)
        layer.forward(x, batch, y)
        layer.check_errors()
        o, q = layer.buf.o[:T], layer.buf.q[:T]
        want, _, tol, _ = plain.attend(q, layer.cache, pages, batch.q_start, batch.kv_len, D ** -0.5)
        assert (np.abs(plain.f64(o).reshape(want.shape) - want) <= tol).all()
        again = torch.empty_like(y)
        (K().linear_qw_wmma if T >= 64 else K().linear_qw)(o.clone(), layer.w.out, again, T, K().Act.BF16, K().Act.F32)
        assert torch.equal(y, again) and torch.isfinite(y).all()


# ---- calls side by side, captured chains ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits,G,group", [(16, 0, 8), (16, 0, 40), (8, 64, 8), (4, 32, 16)])
def test_two_calls_at_once(cuda, bits, G, group):
    """Two streams with a workspace each: the bits of one call after the other."""
    pair = [Batch(cuda, 128, bits, G, 2, group, [9000, 70, 3000], [1, 2, 1], page=32, seed=40 + i) for i in range(2)]
    want = []
    for b in pair:
        b.run()
        torch.cuda.synchronize()
        want.append((b.out.clone(), b.lse.clone()))
    streams = [torch.cuda.Stream() for _ in pair]
    for _ in range(20):
        for b in pair:
            b.out.fill_(UNTOUCHED), b.lse.fill_(UNTOUCHED)
        torch.cuda.synchronize()
        for b, s in zip(pair, streams):
            b.run(stream=s)
        torch.cuda.synchronize()
        for b, w in zip(pair, want):
            assert torch.equal(b.out, w[0]) and torch.equal(b.lse, w[1]) and (b.guard == 0xA5).all() and int(b.err[0]) == 0


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_a_captured_step_replayed_with_other_batches(cuda, bits, G):
    """The whole sublayer in a graph of eight rows and three sequences, replayed with other positions, lengths, ranges and padding: the bits of calls one by one."""
    from strixite_b200.attention import AttnBatch
    d, D = 256, 128
    layer, g = small_layer(cuda, D, 8, 2, d, bits, G, 64, 16, 60, 16, 7)
    def fresh():
        layer.cache.k.zero_(), layer.cache.v.zero_()
    pages = torch.randperm(60, generator=g, device=cuda).to(torch.int32).view(3, 20)
    steps = [((0, 0, 0), (3, 4, 1)), ((3, 4, 1), (1, 1, 1)), ((4, 5, 2), (0, 2, 4)), ((4, 7, 6), (2, 0, 1)), ((200, 150, 300), (1, 6, 1))]
    def batch_of(kept, new):
        b = AttnBatch.of(kept, new, pages)
        more = 8 - sum(new)
        b.seq = torch.cat((b.seq, torch.full((more,), -1, dtype=torch.int32, device=cuda)))
        b.pos = torch.cat((b.pos, torch.zeros(more, dtype=torch.int32, device=cuda)))
        b.max_q = 8
        return b
    xs = [torch.randn((8, d), generator=g, device=cuda).to(torch.bfloat16) for _ in steps]
    want = []
    fresh()
    for x, step in zip(xs, steps):
        y = torch.empty_like(x)
        layer.forward(x, batch_of(*step), y)
        want.append(y.clone())
    layer.check_errors()
    held, x, y = batch_of(*steps[0]), xs[0].clone(), torch.empty_like(xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(x, held, y)
    fresh()
    for x_now, step, w in zip(xs, steps, want):
        now = batch_of(*step)
        for name in ("seq", "pos", "q_start", "kv_len"):
            getattr(held, name).copy_(getattr(now, name))
        x.copy_(x_now)
        graph.replay()
        assert torch.equal(y, w) and (y[sum(step[1]):] == 0).all()
    layer.check_errors()

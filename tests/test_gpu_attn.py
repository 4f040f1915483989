"""GPU tests of the attention operators over a paged key-value cache against their definition in 64 bits (attn_plain.py)."""
import numpy as np
import pytest
import torch

import attn_plain as plain

pytestmark = pytest.mark.gpu


def K():
    from strixite_b200 import kernels
    return kernels


def filled(cache, seed):
    """N(0, 1) with a mean a channel in every row of the cache, quantized by the library's own quantizer where it is."""
    g = torch.Generator(device=cache.device)
    g.manual_seed(seed)
    for name in ("k", "v"):
        shape = (cache.n_pages, cache.n_kv, cache.page, cache.D)
        x = torch.randn(shape, generator=g, device=cache.device) + 0.5 * torch.randn(cache.D, generator=g, device=cache.device)
        if cache.bits == 16:
            getattr(cache, name).copy_(x)
        else:
            w = K().quantize(x.reshape(-1, cache.D).contiguous(), cache.G, cache.bits)
            getattr(cache, name).copy_(w.q.view(getattr(cache, name).shape))
            sm = torch.stack((w.scale, w.minv), -1).view(torch.bfloat16)
            getattr(cache, name + "_sm").copy_(sm.view(getattr(cache, name + "_sm").shape))
    return cache


def tables(lens, page, n_pages, seed, device):
    """Pages scattered over the pool; entries behind a sequence's end name no page."""
    rng = np.random.default_rng(seed)
    wide = max(1, max(-(-max(n, 0) // page) for n in lens)) + 1
    t = np.full((len(lens), wide), 0x7ffffff, dtype=np.int32)
    ids = rng.permutation(n_pages)
    at = 0
    for b, n in enumerate(lens):
        need = -(-max(n, 0) // page)
        t[b, :need] = ids[at:at + need]
        at += need
    assert at <= n_pages
    return torch.from_numpy(t).to(device)


GUARD = 24 << 20  # more than a workspace: nothing may be written behind it


class Batch:
    """A batch of sequences over a filled cache: new[b] new tokens of lens[b] keys."""

    def __init__(self, device, D, bits, G, n_kv, group, lens, new, page=16, seed=0, max_q=None, spare=3):
        self.lens, self.new = lens, new
        n_pages = sum(-(-max(n, 0) // page) for n in lens) + spare
        self.cache = filled(K().KvCache.empty(n_pages, n_kv, page, D, bits, G, device), seed)
        self.pages = tables(lens, page, n_pages, seed, device)
        self.T, self.n_q = sum(new), n_kv * group
        g = torch.Generator(device=device)
        g.manual_seed(seed + 1)
        self.q = (1.5 * torch.randn((self.T, self.n_q * D), generator=g, device=device)).to(torch.bfloat16)
        self.q_start = torch.tensor(np.concatenate(([0], np.cumsum(new))), dtype=torch.int32, device=device)
        self.kv_len = torch.tensor(lens, dtype=torch.int32, device=device)
        self.max_q = max(new) if max_q is None else max_q
        self.out = torch.full_like(self.q, float("nan"))
        self.lse = torch.full((self.T, self.n_q), float("nan"), device=device)
        self.err = torch.zeros(4, dtype=torch.int32, device=device)
        n = K().attn_decode_workspace_bytes(self.cache, self.n_q, self.max_q)
        self.ws_and_more = torch.zeros(n + GUARD, dtype=torch.uint8, device=device)
        self.ws, self.guard = self.ws_and_more[:n], self.ws_and_more[n:]
        self.guard.fill_(0xA5)

    def run(self, **kw):
        kw.setdefault("lse", self.lse)
        K().attn_decode(self.q, self.cache, self.pages, self.q_start, self.kv_len, self.max_q, self.out, self.ws, self.err, **kw)

    def check(self, scale=None, softcap=0.0, window=0):
        torch.cuda.synchronize()
        assert (self.guard == 0xA5).all(), "written behind the workspace"
        assert int(self.err[0]) == 0
        D = self.cache.D
        want, lse, tol, lse_tol = plain.attend(self.q, self.cache, self.pages, self.q_start, self.kv_len, D ** -0.5 if scale is None else scale, softcap, window)
        got = plain.f64(self.out).reshape(want.shape)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        far = np.nan_to_num(np.abs(got - want) - tol, nan=0.0)
        assert far.max() <= 0, (far.max(), np.unravel_index(far.argmax(), far.shape))
        got = plain.f64(self.lse)
        assert np.array_equal(np.isneginf(got), np.isneginf(lse))
        with np.errstate(invalid="ignore"):
            far = np.nan_to_num(np.abs(got - lse) - lse_tol, nan=0.0)
        assert far.max() <= 0, (far.max(), np.unravel_index(far.argmax(), far.shape))


# Every form of the kernel: sizes, codes, groups, and the rows of a tile by the query heads a key head.
FORMS = [(D, bits, G) for D in (64, 128, 256) for bits, groups in ((16, (0,)), (8, (32, 64, 128)), (4, (32, 64, 128))) for G in groups if G <= D]


@pytest.mark.parametrize("group,new", [(4, 1), (1, 1), (3, 7), (8, 8), (5, 13)], ids=["rows4", "rows1", "rows21", "rows64", "rows65"])
@pytest.mark.parametrize("D,bits,G", FORMS)
def test_attend_against_the_definition(cuda, D, bits, G, group, new):
    """Lengths around the tiles' ends, a row that sees one key, rows that see none, sequences of uneven counts of new tokens."""
    lens = [1, new, 63, 64, 65, 128, 129, 0, 700, max(1, new - 2)]
    news = [1, new, new, 1, max(1, new - 1), new, 1, 1, new, new]
    b = Batch(cuda, D, bits, G, 2, group, lens, news, page=16, seed=D + bits + G + group)
    b.run()
    b.check()


@pytest.mark.parametrize("page", [8, 32, 128, 1024])
@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_attend_pages(cuda, bits, G, page):
    b = Batch(cuda, 128, bits, G, 2, 4, [1300, 5, 257], [1, 2, 1], page=page, seed=page)
    b.run()
    b.check()


@pytest.mark.parametrize("window", [1, 5, 64, 100, 5000, (1 << 31) - 1])
@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_attend_window_and_cap(cuda, bits, G, window):
    b = Batch(cuda, 128, bits, G, 2, 4, [1000, 64, 3, 130, 2], [3, 2, 3, 1, 4], seed=window)
    b.run(window=window, softcap=20.0, scale=0.3)
    b.check(window=window, softcap=20.0, scale=0.3)


@pytest.mark.parametrize("B", [1, 127, 128, 129, 300])
def test_attend_many_sequences(cuda, B):
    """More sequences than a CTA has threads: the list's place is found by several rounds."""
    rng = np.random.default_rng(B)
    lens = [int(n) for n in rng.integers(0, 90, B)]
    b = Batch(cuda, 64, 16, 0, 1, 4, lens, [int(n) for n in rng.integers(0, 3, B - 1)] + [1], seed=B)
    b.run()
    b.check()


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_attend_long_cache_is_split_and_joined(cuda, bits, G):
    b = Batch(cuda, 128, bits, G, 1, 8, [30011, 17], [1, 1], page=64, seed=5)
    b.run()
    b.check()
    first = b.out.clone(), b.lse.clone()
    for _ in range(3):  # the join adds in the list's order, whoever comes last
        b.out.fill_(7.0), b.lse.fill_(7.0)
        b.run()
        assert torch.equal(b.out, first[0]) and torch.equal(b.lse, first[1])


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 32)])
def test_attend_more_new_tokens_than_told(cuda, bits, G):
    """max_q picks the kernel; a sequence with more rows takes several passes."""
    b = Batch(cuda, 64, bits, G, 2, 2, [90, 200, 300], [33, 1, 150], max_q=1, seed=3)
    b.run()
    b.check()


def test_attend_leaves_other_rows_and_columns(cuda):
    """Rows before, between and behind the sequences and what lies beside a strided output stay as they were."""
    b = Batch(cuda, 64, 16, 0, 2, 2, [40, 20, 33], [2, 1, 1], seed=8)
    T, wide = 9, b.n_q * 64
    q = torch.randn((T, wide + 64), device=cuda).to(torch.bfloat16)[:, :wide]
    out = torch.full((T, wide + 8), 3.0, device=cuda, dtype=torch.bfloat16)
    lse = torch.full((T, b.n_q), 3.0, device=cuda)
    starts = torch.tensor([1, 3, 3, 4], dtype=torch.int32, device=cuda)  # rows 1-2, none, row 3
    K().attn_decode(q, b.cache, b.pages, starts, b.kv_len, 2, out[:, :wide], b.ws, b.err, lse=lse)
    torch.cuda.synchronize()
    want, want_lse, tol, _ = plain.attend(q, b.cache, b.pages, starts, b.kv_len, 64 ** -0.5)
    got = plain.f64(out[:, :wide]).reshape(want.shape)
    assert (np.abs(got[1:4] - want[1:4]) <= tol[1:4]).all()
    for t in (0, 4, 5, 6, 7, 8):
        assert (out[t] == 3.0).all() and (lse[t] == 3.0).all()
    assert (out[:, wide:] == 3.0).all()


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_attend_other_strides(cuda, bits, G):
    """A pool kept token by token ([n_pages, page, n_kv, D]), keys and values in one tensor, gives the same bits as the plain one."""
    b = Batch(cuda, 128, bits, G, 2, 4, [500, 77], [2, 1], seed=9)
    b.run()
    c = b.cache
    def moved(k, v):
        both = torch.empty((c.n_pages, 2, c.page, c.n_kv, *k.shape[3:]), dtype=k.dtype, device=cuda)
        both[:, 0].copy_(k.transpose(1, 2))
        both[:, 1].copy_(v.transpose(1, 2))
        return both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    k, v = moved(c.k, c.v)
    sm = moved(c.k_sm, c.v_sm) if bits != 16 else (None, None)
    other = K().KvCache(k, v, bits, G, *sm)
    out = torch.empty_like(b.out)
    K().attn_decode(b.q, other, b.pages, b.q_start, b.kv_len, b.max_q, out, b.ws, b.err)
    assert torch.equal(out, b.out)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attend_what_is_not_finite_reaches_only_rows_that_see_it(cuda, bad):
    """A NaN or an infinity in the newest key and value (BF16), rows of three drafts: only the last row sees it; junk behind the sequences' ends."""
    for where in ("k", "v"):
        b = Batch(cuda, 128, 16, 0, 2, 4, [70, 300], [3, 3], seed=11)
        for s, n in enumerate(b.lens):
            getattr(b.cache, where)[int(b.pages[s, (n - 1) // 16]), :, (n - 1) % 16, 5] = bad
            for at in range(n % 16, 16):  # the last page's rest
                getattr(b.cache, where)[int(b.pages[s, (n - 1) // 16]), :, at] = float("nan")
        b.run()
        torch.cuda.synchronize()
        want, lse, tol, _ = plain.attend(b.q, b.cache, b.pages, b.q_start, b.kv_len, 128 ** -0.5)
        got = plain.f64(b.out).reshape(want.shape)
        rows = [0, 1, 3, 4]
        assert np.isfinite(got[rows]).all() and (np.abs(got[rows] - want[rows]) <= tol[rows]).all()
        if where == "v":  # the channel alone
            assert np.array_equal(np.isfinite(got[[2, 5]]), np.isfinite(want[[2, 5]])) and not np.isfinite(got[[2, 5], :, 5]).any()
        elif bad != bad:
            assert np.isnan(got[[2, 5]]).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_attend_scales_that_are_none_reach_only_rows_that_see_them(cuda, bits):
    for where in ("k_sm", "v_sm"):
        b = Batch(cuda, 128, bits, 32, 2, 4, [70, 300], [3, 3], seed=12)
        for s, n in enumerate(b.lens):
            getattr(b.cache, where)[int(b.pages[s, (n - 1) // 16]), :, (n - 1) % 16, 1] = float("nan")
            getattr(b.cache, where)[int(b.pages[s, (n - 1) // 16]), :, n % 16:] = float("nan")
        b.run()
        torch.cuda.synchronize()
        want, lse, tol, _ = plain.attend(b.q, b.cache, b.pages, b.q_start, b.kv_len, 128 ** -0.5)
        got = plain.f64(b.out).reshape(want.shape)
        rows = [0, 1, 3, 4]
        assert np.isfinite(got[rows]).all() and (np.abs(got[rows] - want[rows]) <= tol[rows]).all()
        assert np.array_equal(np.isnan(got[[2, 5]]), np.isnan(want[[2, 5]]))


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -20, 1.0, 2.0 ** 20, 2.0 ** 60])
@pytest.mark.parametrize("bits", [8, 4])
def test_attend_values_and_queries_of_any_size(cuda, bits, size):
    """F16 operands' range is no limit: values (hence scales) and queries far outside of it, later values larger than earlier ones and smaller."""
    for grows in (1.0, 2.0 ** 20, 2.0 ** -20):
        b = Batch(cuda, 128, bits, 64, 1, 4, [400], [1], seed=13)
        b.cache.v_sm.mul_(size)
        b.cache.v_sm[b.pages[0, 10:20].long()] *= grows
        b.q.mul_(1.0 / size)
        b.cache.k_sm.mul_(size)
        b.run()
        b.check()


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64)])
def test_attend_bad_pages_lengths_and_rows(cuda, bits, G):
    """What the host cannot see is refused by the kernel: NaN for the rows that it concerns, the rest right, the error words set."""
    b = Batch(cuda, 64, bits, G, 2, 2, [100, 90, 80, 60, 50], [1, 2, 1, 1, 1], seed=14)
    clean = b.pages.clone(), b.kv_len.clone(), b.q_start.clone()
    want, lse, tol, _ = plain.attend(b.q, b.cache, b.pages, b.q_start, b.kv_len, 64 ** -0.5)
    b.pages[0, 2] = b.cache.n_pages
    b.pages[1, 5] = -3                    # keys 80..89: both rows see them
    b.kv_len[2] = b.pages.shape[1] * 16 + 1
    b.kv_len[3] = -1
    b.run()
    torch.cuda.synchronize()
    got = plain.f64(b.out).reshape(want.shape)
    assert np.isnan(got[:5]).all() and torch.isnan(b.lse[:5]).all()
    assert (np.abs(got[5] - want[5]) <= tol[5]).all()
    assert int(b.err[0]) == 1
    with pytest.raises(K().Error, match="batch: page, position, length"):
        K().check_attn_error(b.err, "batch")
    b.err.zero_()
    b.pages, b.kv_len, b.q_start = clean[0], clean[1], clean[2].clone()
    b.q_start[2] = b.T + 5  # sequences 1 and 2 have no rows to speak of
    b.out.fill_(3.0)
    b.run()
    torch.cuda.synchronize()
    got = plain.f64(b.out).reshape(want.shape)
    assert (got[1:4] == 3.0).all() and int(b.err[0]) == 1
    for t in (0, 4, 5):
        assert (np.abs(got[t] - want[t]) <= tol[t]).all()


def test_attend_captured_and_replayed_with_other_lengths(cuda):
    """A graph follows the lengths, tables and rows that it finds; two graphs that share a workspace run one behind the other."""
    b = Batch(cuda, 128, 8, 64, 2, 4, [1000, 300], [1, 2], seed=15)
    b.run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            b.run()
    for lens in ([1000, 300], [17, 2], [640, 0], [1, 299]):
        b.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        for graph in graphs:
            b.out.fill_(float("nan"))
            graph.replay()
            b.check()


@pytest.mark.parametrize("D,bits,G", FORMS)
def test_attend_keeps_to_its_workspace(cuda, D, bits, G):
    """Every form with all of its CTAs at work on segments that are split, in a workspace of the size asked for and not a byte more."""
    for rows in (8, 16, 32, 64):
        b = Batch(cuda, D, bits, G, 8, rows, [6000], [1], page=64, seed=rows)
        b.run()
        torch.cuda.synchronize()
        assert (b.guard == 0xA5).all() and torch.isfinite(b.out).all() and int(b.err[0]) == 0


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_attend_calls_of_every_form_share_a_workspace(cuda, bits, G):
    """A workspace made for many rows serves calls of few, in any order: each finds its counters at zero."""
    ws = None
    for turn, new in enumerate((8, 1, 4, 2, 1, 8, 2, 4)):
        b = Batch(cuda, 128, bits, G, 1, 8, [5000, 900], [new, 1], page=64, seed=20 + turn)
        if ws is None:
            ws = b.ws
        b.ws = ws
        b.run()
        b.check()


def test_attend_on_another_stream(cuda):
    b = Batch(cuda, 128, 16, 0, 2, 4, [3000], [1], seed=16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b.run(stream=side)
    side.synchronize()
    b.check()


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_offsets_beyond_32_bits(cuda, bits, G):
    """Pages at the end of a pool whose codes, and whose rows' words, lie more than 2^32 bytes behind its start."""
    D, n_kv, page = 128, 8, 64
    n_pages = (9 << 30) // (n_kv * page * D * bits // 8)
    k = torch.empty((n_pages, n_kv, page, D // 2 if bits == 4 else D), dtype=torch.bfloat16 if bits == 16 else torch.uint8, device=cuda)
    v = torch.empty_like(k)
    sm = [torch.empty((n_pages, n_kv, page, D // G, 2), dtype=torch.bfloat16, device=cuda) for _ in range(2)] if bits != 16 else [None, None]
    cache = K().KvCache(k, v, bits, G, *sm)
    T = 150
    pages = torch.arange(n_pages - 3, n_pages, dtype=torch.int32, device=cuda).view(1, 3)
    seq, pos = torch.zeros(T, dtype=torch.int32, device=cuda), torch.arange(T, dtype=torch.int32, device=cuda)
    qkv = torch.randn((T, (8 + 2 * n_kv) * D), device=cuda).to(torch.bfloat16)
    q = torch.empty((T, 8 * D), dtype=torch.bfloat16, device=cuda)
    err = torch.zeros(4, dtype=torch.int32, device=cuda)
    K().attn_qkv_write(qkv, cache, seq, pos, pages, q, err)
    ko, vo = (torch.empty((T, n_kv, D), dtype=torch.float32, device=cuda) for _ in range(2))
    K().kv_read(cache, seq, pos, pages, ko, vo, err)
    x = qkv.float().view(T, 8 + 2 * n_kv, D)
    step = 0.0 if bits == 16 else 8.0 / (2 ** bits - 1)
    assert (ko - x[:, 8:16]).abs().max() <= step and (vo - x[:, 16:]).abs().max() <= step
    out, ws = torch.empty_like(q[:1]), torch.zeros(K().attn_decode_workspace_bytes(cache, 8, 1), dtype=torch.uint8, device=cuda)
    starts, lens = torch.tensor([0, 1], dtype=torch.int32, device=cuda), torch.tensor([T], dtype=torch.int32, device=cuda)
    K().attn_decode(q[:1], cache, pages, starts, lens, 1, out, ws, err)
    want, _, tol, _ = plain.attend(q[:1], cache, pages, starts, lens, D ** -0.5)
    assert (np.abs(plain.f64(out).reshape(want.shape) - want) <= tol).all() and int(err[0]) == 0


# ---- writing and reading -----------------------------------------------------------------------------------------------------------

class Rows:
    """T tokens of B sequences, their places scattered, and what is to be written there."""

    def __init__(self, device, T, B, n_q, n_kv, D, bits, G, page=16, f32=False, far=0, seed=0, norm=True):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.T, self.n_q, self.D = T, n_q, D
        counts = [T // B + (b < T % B) for b in range(B)]
        self.lens = [far + 3 * b + n for b, n in enumerate(counts)]
        n_pages = sum(-(-n // page) for n in self.lens) + 2
        self.cache = filled(K().KvCache.empty(n_pages, n_kv, page, D, bits, G, device), seed + 7)
        self.pages = tables(self.lens, page, n_pages, seed, device)
        order = np.random.default_rng(seed).permutation(T)
        seq = np.concatenate([np.full(n, b) for b, n in enumerate(counts)])[order]
        pos = np.concatenate([np.arange(n) + self.lens[b] - n for b, n in enumerate(counts)])[order]
        self.seq, self.pos = (torch.from_numpy(v.astype(np.int32)).to(device) for v in (seq, pos))
        x = torch.randn((T, (n_q + 2 * n_kv) * D), generator=g, device=device) * 1.7
        self.qkv = x if f32 else x.to(torch.bfloat16)
        self.q_norm, self.k_norm = ((1 + 0.2 * torch.randn(D, generator=g, device=device)) if norm else None for _ in range(2))
        self.q_out = torch.full((T, n_q * D), float("nan"), dtype=torch.bfloat16, device=device)
        self.err = torch.zeros(4, dtype=torch.int32, device=device)

    def inv_freq(self, rot):
        return (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().to(self.qkv.device) if rot else None

    def read(self, dtype=torch.float32):
        k, v = (torch.full((self.T, self.cache.n_kv, self.D), float("nan"), dtype=dtype, device=self.qkv.device) for _ in range(2))
        K().kv_read(self.cache, self.seq, self.pos, self.pages, k, v, self.err)
        return k, v


@pytest.mark.parametrize("T,B,n_q,n_kv,f32", [(1, 1, 8, 2, False), (37, 5, 3, 1, True), (300, 2, 4, 4, False), (1500, 3, 2, 1, True)])
@pytest.mark.parametrize("rot,interleaved", [("D", False), (32, True), (16, False), (0, False)])
@pytest.mark.parametrize("D,bits,G", [f for f in FORMS if f[2] in (0, 32, f[0])])
def test_write_and_read_against_the_definition(cuda, D, bits, G, rot, interleaved, T, B, n_q, n_kv, f32):
    r = Rows(cuda, T, B, n_q, n_kv, D, bits, G, f32=f32, seed=T + D + bits)
    rot = D if rot == "D" else rot
    before = [t.clone() for t in (r.cache.k, r.cache.v)]
    inv = r.inv_freq(rot)
    K().attn_qkv_write(r.qkv, r.cache, r.seq, r.pos, r.pages, r.q_out, r.err, q_norm=r.q_norm, k_norm=r.k_norm, eps=1e-5, inv_freq=inv, interleaved=interleaved)
    k, v = r.read()
    torch.cuda.synchronize()
    assert int(r.err[0]) == 0
    x = plain.f64(r.qkv).reshape(T, n_q + 2 * n_kv, D)
    pos = r.pos.cpu().numpy()
    q, q_size = plain.norm_rotate(x[:, :n_q], r.q_norm, 1e-5, pos, inv, interleaved)
    kk, k_size = plain.norm_rotate(x[:, n_q:n_q + n_kv], r.k_norm, 1e-5, pos, inv, interleaved)
    vv = x[:, n_q + n_kv:]
    # FP32: the norm's sum (D / 32 + 5 roundings, halved by the root), root, division, two products, the turn's two products and sum: under 2^-20
    assert (np.abs(plain.f64(r.q_out).reshape(q.shape) - q) <= plain.BF16 * np.abs(q) + 2.0 ** -20 * q_size).all()
    page, at = r.pages.cpu().numpy()[r.seq.cpu().numpy(), pos // 16], pos % 16
    if bits == 16:
        assert (np.abs(plain.f64(k) - kk) <= plain.BF16 * np.abs(kk) + 2.0 ** -20 * k_size).all()
        assert np.array_equal(plain.f64(v), plain.f64(r.qkv.view(T, -1, D)[:, n_q + n_kv:].to(torch.bfloat16)))
    else:
        # V is not touched before it is quantized: the library's quantizer gives the same codes, bit for bit
        w = K().quantize(r.qkv.float().view(T, -1, D)[:, n_q + n_kv:].reshape(-1, D).contiguous(), G, bits)
        codes = torch.stack([r.cache.v[int(p), :, int(a)] for p, a in zip(page, at)])
        assert torch.equal(codes.reshape(w.q.shape), w.q)
        sm = torch.stack([r.cache.v_sm[int(p), :, int(a)] for p, a in zip(page, at)]).view(torch.int16)
        assert torch.equal(sm[..., 0].reshape(w.scale.shape), w.scale) and torch.equal(sm[..., 1].reshape(w.minv.shape), w.minv)
        # what is read is code * scale + min, one rounding
        for which, got in (("k", k), ("v", v)):
            for h in range(n_kv):
                y, _, _ = plain.values(r.cache, which, page.astype(np.int64), h, at)
                assert (np.abs(plain.f64(got)[:, h] - y) <= 2.0 ** -23 * np.abs(y)).all()
        # K: half a step of the group's range, the scale's and the min's rounding to BF16 (at the far end the scale's counts `levels` times, and codes
        # beyond the last are cut off), and FP32 on the way
        groups = kk.reshape(T, n_kv, -1, G)
        lo, hi = groups.min(-1, keepdims=True), groups.max(-1, keepdims=True)
        tol = 0.51 * (hi - lo) / (2 ** bits - 1) + 2 * plain.BF16 * (np.abs(lo) + np.abs(hi - lo)) + 2.0 ** -19 * k_size.reshape(groups.shape)
        assert (np.abs(plain.f64(k).reshape(groups.shape) - groups) <= tol).all()
    # nothing but the tokens' rows
    for name, old in zip(("k", "v"), before):
        new = getattr(r.cache, name).clone()
        p, a = torch.from_numpy(page.astype(np.int64)).to(cuda), torch.from_numpy(at.astype(np.int64)).to(cuda)
        new[p, :, a] = old[p, :, a]
        assert torch.equal(new.view(torch.uint8), old.view(torch.uint8))


def test_write_far_positions(cuda):
    """The angle of a position near 2^31: FP32 would lose whole turns."""
    r = Rows(cuda, 1, 1, 4, 1, 128, 16, 0, page=4096, norm=False)
    r.pages = torch.zeros((1, (1 << 19) - 1), dtype=torch.int32, device=cuda)
    inv = r.inv_freq(128)
    for pos in (0, 1, 123457, 1 << 24, (1 << 31) - 4097):
        r.pos.fill_(pos)
        K().attn_qkv_write(r.qkv, r.cache, r.seq, r.pos, r.pages, r.q_out, r.err, inv_freq=inv)
        q, size = plain.norm_rotate(plain.f64(r.qkv).reshape(1, 6, 128)[:, :4], None, 0, np.array([pos]), inv, False)
        assert (np.abs(plain.f64(r.q_out).reshape(q.shape) - q) <= plain.BF16 * np.abs(q) + 2.0 ** -20 * size).all(), pos
    assert int(r.err[0]) == 0


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_write_and_read_padding_and_bad_places(cuda, bits, G):
    """Padding rows stay as they are everywhere; a bad place gives NaN, writes nothing to the cache and sets the error words."""
    r = Rows(cuda, 6, 2, 2, 1, 128, bits, G, seed=4)
    r.q_out.fill_(3.0)
    seq, pos = r.seq.clone(), r.pos.clone()
    r.seq[1] = -1
    K().attn_qkv_write(r.qkv, r.cache, r.seq, r.pos, r.pages, r.q_out, r.err)
    k, v = r.read()
    torch.cuda.synchronize()
    assert int(r.err[0]) == 0 and (r.q_out[1] == 3.0).all() and torch.isfinite(r.q_out[[0, 2, 3, 4, 5]]).all()
    assert torch.isnan(k[1]).all() and torch.isnan(v[1]).all() and torch.isfinite(k[[0, 2, 3, 4, 5]]).all()
    old = r.cache.k.clone(), r.cache.v.clone()
    for bad in ("seq", "pos", "negative", "page"):
        r.err.zero_()
        r.seq.fill_(-1), r.pos.copy_(pos)
        r.seq[2] = seq[2]
        pages = r.pages.clone()
        if bad == "seq":
            r.seq[2] = 2
        elif bad == "pos":
            r.pos[2] = r.pages.shape[1] * 16
        elif bad == "negative":
            r.pos[2] = -5
        else:
            pages[int(seq[2]), int(pos[2]) // 16] = r.cache.n_pages
        K().attn_qkv_write(r.qkv, r.cache, r.seq, r.pos, pages, r.q_out, r.err)
        ko, vo = torch.zeros_like(k), torch.zeros_like(v)
        assert int(r.err[0]) == 1 and int(r.err[1]) == 2
        with pytest.raises(K().Error, match="token or sequence 2"):
            K().check_attn_error(r.err, "write")
        r.err.zero_()
        K().kv_read(r.cache, r.seq, r.pos, pages, ko, vo, r.err)
        torch.cuda.synchronize()
        assert int(r.err[0]) == 1
        assert torch.isnan(r.q_out[2]).all() and torch.isnan(ko[2]).all() and torch.isnan(vo[2]).all()
        assert (ko[[0, 1, 3, 4, 5]] == 0).all()
        assert torch.equal(r.cache.k.view(torch.uint8), old[0].view(torch.uint8)) and torch.equal(r.cache.v.view(torch.uint8), old[1].view(torch.uint8))


@pytest.mark.parametrize("bits", [8, 4])
def test_written_groups_of_one_value_and_of_none(cuda, bits):
    """A constant group comes back as its BF16 rounding, one with a NaN or an infinity as NaN, its neighbours as ever."""
    r = Rows(cuda, 3, 1, 1, 1, 128, bits, 32, seed=6, norm=False)
    x = r.qkv.view(3, 3, 128)
    x[0, 1:, 32:64] = 1.0 / 3
    x[1, 1:, 40] = float("nan")
    x[2, 1:, 127] = -float("inf")
    K().attn_qkv_write(r.qkv, r.cache, r.seq, r.pos, r.pages, r.q_out, r.err)
    k, v = r.read()
    for y in (k, v):
        assert (y[0, 0, 32:64] == x[0, 1, 32].float()).all()
        assert torch.isnan(y[1, 0, 32:64]).all() and torch.isfinite(y[1, 0, :32]).all() and torch.isfinite(y[1, 0, 64:]).all()
        assert torch.isnan(y[2, 0, 96:]).all() and torch.isfinite(y[2, 0, :96]).all()


def test_write_strided_rows_and_bf16_read(cuda):
    r = Rows(cuda, 20, 2, 4, 2, 64, 8, 64, seed=2)
    wide = torch.randn((20, 8 * 64 + 16), device=cuda).to(torch.bfloat16)
    q_wide = torch.full((20, 4 * 64 + 24), 3.0, dtype=torch.bfloat16, device=cuda)
    inv = r.inv_freq(64)
    K().attn_qkv_write(wide[:, :512], r.cache, r.seq, r.pos, r.pages, q_wide[:, :256], r.err, inv_freq=inv)
    k, v = r.read(torch.bfloat16)
    k32, v32 = r.read()
    assert torch.equal(k, k32.to(torch.bfloat16)) and torch.equal(v, v32.to(torch.bfloat16))
    assert (q_wide[:, 256:] == 3.0).all()
    q, size = plain.norm_rotate(plain.f64(wide[:, :256]).reshape(20, 4, 64), None, 0, r.pos.cpu().numpy(), inv, False)
    assert (np.abs(plain.f64(q_wide[:, :256]).reshape(q.shape) - q) <= plain.BF16 * np.abs(q) + 2.0 ** -20 * size).all()


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_steps_of_write_and_attend_together(cuda, bits, G):
    """A prompt of three conversations written, then decode steps of one token and of drafts: each step writes its keys and attends over them."""
    D, n_q, n_kv, page, B = 128, 8, 2, 16, 3
    cache = K().KvCache.empty(40, n_kv, page, D, bits, G, cuda)
    pages = torch.randperm(39, device=cuda).to(torch.int32).view(3, 13)
    lens, err = [0] * B, torch.zeros(4, dtype=torch.int32, device=cuda)
    inv = (1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().to(cuda)
    ws = torch.zeros(K().attn_decode_workspace_bytes(cache, n_q, 64), dtype=torch.uint8, device=cuda)
    for step, new in enumerate([(60, 17, 1), (1, 1, 1), (3, 1, 4), (1, 0, 8)]):
        T = sum(new)
        seq = torch.tensor([b for b in range(B) for _ in range(new[b])], dtype=torch.int32, device=cuda)
        pos = torch.tensor([lens[b] + i for b in range(B) for i in range(new[b])], dtype=torch.int32, device=cuda)
        lens = [n + m for n, m in zip(lens, new)]
        qkv = torch.randn((T, (n_q + 2 * n_kv) * D), device=cuda).to(torch.bfloat16)
        q, out = torch.empty((T, n_q * D), dtype=torch.bfloat16, device=cuda), torch.empty((T, n_q * D), dtype=torch.bfloat16, device=cuda)
        starts = torch.tensor(np.concatenate(([0], np.cumsum(new))), dtype=torch.int32, device=cuda)
        kv_len = torch.tensor(lens, dtype=torch.int32, device=cuda)
        K().attn_qkv_write(qkv, cache, seq, pos, pages, q, err, inv_freq=inv, q_norm=torch.ones(D, device=cuda), k_norm=torch.ones(D, device=cuda))
        K().attn_decode(q, cache, pages, starts, kv_len, max(new), out, ws, err)
        torch.cuda.synchronize()
        want, _, tol, _ = plain.attend(q, cache, pages, starts, kv_len, D ** -0.5)
        assert (np.abs(plain.f64(out).reshape(want.shape) - want) <= tol).all(), step
        assert int(err[0]) == 0


@pytest.mark.parametrize("bits,G", [(16, 0), (8, 64), (4, 32)])
def test_layer_is_its_parts(cuda, bits, G):
    """Two layers over buffers of their own stack: a prompt by the tensor-core projections, then steps of one token and of drafts.  Every step's output is
    what the launchers give one by one, bit for bit, and the attention in it is the definition's."""
    from strixite_b200.attention import AttnBatch, AttnBuffers, AttnLayer, AttnWeights
    D, n_q, n_kv, page, d = 64, 4, 2, 16, 256
    g = torch.Generator(device=cuda)
    g.manual_seed(bits)
    def weight(n, k):
        return K().quantize(torch.randn((n, k), generator=g, device=cuda) * 0.05, 64, 8)
    inv = (1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().to(cuda)
    caches = [K().KvCache.empty(20, n_kv, page, D, bits, G, cuda) for _ in range(2)]
    buf = AttnBuffers(100, 80, n_q, caches[0])
    layers = [AttnLayer(AttnWeights(weight((n_q + 2 * n_kv) * D, d), weight(d, n_q * D), 1 + 0.1 * torch.randn(D, generator=g, device=cuda),
                                    1 + 0.1 * torch.randn(D, generator=g, device=cuda), inv), n_q, c, buf) for c in caches]
    pages = torch.randperm(20, generator=g, device=cuda)[:18].to(torch.int32).view(2, 9)
    kept = [0, 0]
    for new in ((80, 3), (1, 1), (1, 4), (0, 1)):
        x = torch.randn((sum(new), d), generator=g, device=cuda).to(torch.bfloat16)
        batch = AttnBatch.of(kept, new, pages)
        kept = [k + n for k, n in zip(kept, new)]
        for layer in layers:
            T, w = sum(new), layer.w
            y = torch.empty((T, d), dtype=torch.bfloat16, device=cuda)
            layer.forward(x, batch, y)
            layer.check_errors()
            o, q = buf.o[:T].clone(), buf.q[:T].clone()
            want, _, tol, _ = plain.attend(q, layer.cache, pages, batch.q_start, batch.kv_len, D ** -0.5)
            assert (np.abs(plain.f64(o).reshape(want.shape) - want) <= tol).all()
            linear = K().linear_qw_wmma if T >= 64 else K().linear_qw
            qkv, q2, o2, y2 = torch.empty_like(buf.qkv[:T]), torch.empty_like(q), torch.empty_like(o), torch.empty_like(y)
            linear(x, w.qkv, qkv, T, K().Act.BF16, K().Act.F32)
            K().attn_qkv_write(qkv, layer.cache, batch.seq, batch.pos, pages, q2, buf.err, q_norm=w.q_norm, k_norm=w.k_norm, inv_freq=inv)
            K().attn_decode(q2, layer.cache, pages, batch.q_start, batch.kv_len, batch.max_q, o2, buf.ws, buf.err)
            linear(o2, w.out, y2, T, K().Act.BF16, K().Act.BF16)
            assert torch.equal(q, q2) and torch.equal(o, o2) and torch.equal(y, y2)
            x = (x.float() + y.float()).to(torch.bfloat16)
    with pytest.raises(K().Error, match="the buffers hold 100"):
        layers[0].forward(torch.zeros((101, d), dtype=torch.bfloat16, device=cuda), batch, y)
    with pytest.raises(K().Error, match="do not fit 3 query"):
        AttnLayer(layers[0].w, 3, caches[0], buf)


def test_python_refusals_on_the_device(cuda):
    """Another type, another device, a vector that is not contiguous, shapes that do not fit: refused by name before anything is enqueued."""
    b = Batch(cuda, 64, 16, 0, 2, 2, [40, 20], [2, 1], seed=1)
    def attend(**kw):
        a = dict(q=b.q, cache=b.cache, pages=b.pages, q_start=b.q_start, kv_len=b.kv_len, max_q=2, out=b.out, ws=b.ws, err=b.err, lse=b.lse)
        a.update(kw)
        K().attn_decode(**a)
    for kw, said in ((dict(q=b.q.float()), "q is torch.float32"), (dict(kv_len=b.kv_len.long()), "kv_len is torch.int64"), (dict(pages=b.pages.cpu()), "pages is torch.int32 on cpu"),
                     (dict(q_start=b.q_start[:2]), "shapes do not fit"), (dict(out=b.out[:, :64]), "shapes do not fit"), (dict(lse=b.lse[:2]), "shapes do not fit"),
                     (dict(q=b.q.t().contiguous().t()), "last dimension contiguous"), (dict(err=b.err[:2]), "shapes do not fit"), (dict(ws=b.ws[:64]), "workspace of 64 bytes"),
                     (dict(q_start=torch.zeros(6, dtype=torch.int32, device=cuda)[::2]), "q_start is"), (dict(softcap=1e-9), "softcap"), (dict(max_q=0), "max_q = 0")):
        with pytest.raises(K().Error, match=said):
            attend(**kw)
    r = Rows(cuda, 4, 2, 2, 1, 64, 8, 32)
    with pytest.raises(K().Error, match="shapes do not fit"):
        K().attn_qkv_write(r.qkv, r.cache, r.seq[:3], r.pos, r.pages, r.q_out, r.err)
    with pytest.raises(K().Error, match="q_out is torch.float32"):
        K().attn_qkv_write(r.qkv, r.cache, r.seq, r.pos, r.pages, r.q_out.float(), r.err)
    with pytest.raises(K().Error, match="rot = 24"):
        K().attn_qkv_write(r.qkv, r.cache, r.seq, r.pos, r.pages, r.q_out, r.err, inv_freq=torch.ones(12, device=cuda))
    with pytest.raises(K().Error, match="v_out is torch.float32"):
        K().kv_read(r.cache, r.seq, r.pos, r.pages, torch.empty((4, 1, 64), dtype=torch.bfloat16, device=cuda), torch.empty((4, 1, 64), device=cuda), r.err)
    with pytest.raises(K().Error, match="k_sm is"):
        K().KvCache(r.cache.k, r.cache.v, 8, 32, r.cache.k_sm[..., :1, :], r.cache.v_sm)
    with pytest.raises(K().Error, match="not whole rows|not those of k"):
        K().KvCache(torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16, device=cuda), torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device=cuda).transpose(1, 2), 16)


def test_attend_queries_that_are_none_stay_in_their_rows(cuda):
    """A NaN or an infinity in one query: its row is NaN, the others as ever (all heads of a key head share a tile)."""
    for bits, G in ((16, 0), (8, 64), (4, 32)):
        for bad in (float("nan"), float("inf")):
            b = Batch(cuda, 128, bits, G, 2, 4, [300], [2], seed=17)
            b.q[0, 128 + 7] = bad  # head 1 of the first token
            b.run()
            torch.cuda.synchronize()
            got = plain.f64(b.out).reshape(2, 8, 128)
            assert np.isnan(got[0, 1]).all()
            b.q[0, 128 + 7] = 0.0
            want, _, tol, _ = plain.attend(b.q, b.cache, b.pages, b.q_start, b.kv_len, 128 ** -0.5)
            ok = np.ones((2, 8), bool)
            ok[0, 1] = False
            assert (np.abs(got[ok] - want[ok]) <= tol[ok]).all()


# ---- tiles of 128 rows: a BF16 cache of heads of 128 and more than 128 rows a key head, or more than 32 and a table with room for many keys ----

def with_room(b, keys=400_000):
    """The batch's tables with columns for so many keys: what a table has room for picks the form."""
    more = torch.full((len(b.lens), keys // b.cache.page), 0x7ffffff, dtype=torch.int32, device=b.pages.device)
    b.pages = torch.cat((b.pages, more), 1)
    return b


@pytest.mark.parametrize("group,new", [(3, 11), (8, 8), (5, 13), (8, 16), (43, 3), (3, 50), (5, 77)], ids=["rows33", "rows64", "rows65", "rows128", "rows129", "rows150", "rows385"])
def test_attend_many_rows_against_the_definition(cuda, group, new):
    """Lengths around the tiles' ends, rows that see none, uneven counts of new tokens, in tiles of 128 rows and tokens that two of them share."""
    lens = [1, new, 63, 127, 128, 129, 256, 0, 700, max(1, new - 2), 257]
    news = [1, new, new, 1, max(1, new - 1), new, 1, 1, new, new, 2]
    b = with_room(Batch(cuda, 128, 16, 0, 2, group, lens, news, seed=group + new))
    b.run()
    b.check()


@pytest.mark.parametrize("page", [8, 16, 64, 1024])
@pytest.mark.parametrize("window", [0, 1, 100, 1000])
def test_attend_many_rows_pages_window_and_cap(cuda, page, window):
    b = with_room(Batch(cuda, 128, 16, 0, 2, 7, [1300, 64, 3, 389], [21, 2, 7, 30], page=page, seed=page + window))
    b.run(window=window, softcap=20.0, scale=0.3)
    b.check(window=window, softcap=20.0, scale=0.3)


def test_attend_many_rows_long_cache_is_split_and_joined(cuda):
    b = Batch(cuda, 128, 16, 0, 1, 8, [20011, 17], [17, 3], page=64, seed=5)
    b.run()
    b.check()
    first = b.out.clone(), b.lse.clone()
    for _ in range(3):
        b.out.fill_(7.0), b.lse.fill_(7.0)
        b.run()
        assert torch.equal(b.out, first[0]) and torch.equal(b.lse, first[1])


def test_attend_many_rows_scores_that_rise(cuda):
    """Keys whose scores rise tile by tile by more than the weights' slack, and fall again: sums are scaled on the way, and by hand what the last tile needs."""
    b = Batch(cuda, 128, 16, 0, 1, 10, [1500], [14], seed=6)
    for p in range(b.pages.shape[1] - 1):
        b.cache.k[int(b.pages[0, p])] *= (1 + p / 8) if p < 60 else 0.1
    b.run()
    b.check()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attend_many_rows_what_is_not_finite_reaches_only_rows_that_see_it(cuda, bad):
    """As above: the newest key or value is none, 50 heads a key head; the sequences' first tile is their last, or not."""
    for where in ("k", "v"):
        b = Batch(cuda, 128, 16, 0, 1, 50, [70, 300], [3, 3], seed=11)
        for s, n in enumerate(b.lens):
            getattr(b.cache, where)[int(b.pages[s, (n - 1) // 16]), :, (n - 1) % 16, 5] = bad
            for at in range(n % 16, 16):
                getattr(b.cache, where)[int(b.pages[s, (n - 1) // 16]), :, at] = float("nan")
        b.run()
        torch.cuda.synchronize()
        want, lse, tol, _ = plain.attend(b.q, b.cache, b.pages, b.q_start, b.kv_len, 128 ** -0.5)
        got = plain.f64(b.out).reshape(want.shape)
        rows = [0, 1, 3, 4]
        assert np.isfinite(got[rows]).all() and (np.abs(got[rows] - want[rows]) <= tol[rows]).all()
        if where == "v":
            assert np.array_equal(np.isfinite(got[[2, 5]]), np.isfinite(want[[2, 5]])) and not np.isfinite(got[[2, 5], :, 5]).any()
        elif bad != bad:
            assert np.isnan(got[[2, 5]]).all()


def test_attend_many_rows_one_query_that_is_none(cuda):
    for bad in (float("nan"), float("inf")):
        b = Batch(cuda, 128, 16, 0, 1, 70, [300], [2], seed=17)
        b.q[0, 128 + 7] = bad
        b.run()
        torch.cuda.synchronize()
        got = plain.f64(b.out).reshape(2, 70, 128)
        assert np.isnan(got[0, 1]).all()
        b.q[0, 128 + 7] = 0.0
        want, _, tol, _ = plain.attend(b.q, b.cache, b.pages, b.q_start, b.kv_len, 128 ** -0.5)
        ok = np.ones((2, 70), bool)
        ok[0, 1] = False
        assert (np.abs(got[ok] - want[ok]) <= tol[ok]).all()


def test_attend_many_rows_bad_pages_lengths_and_rows(cuda):
    b = Batch(cuda, 128, 16, 0, 1, 66, [100, 90, 80, 60, 50], [1, 2, 1, 1, 1], seed=14)
    clean = b.pages.clone(), b.kv_len.clone(), b.q_start.clone()
    want, lse, tol, _ = plain.attend(b.q, b.cache, b.pages, b.q_start, b.kv_len, 128 ** -0.5)
    b.pages[0, 2] = b.cache.n_pages
    b.pages[1, 5] = -3
    b.kv_len[2] = b.pages.shape[1] * 16 + 1
    b.kv_len[3] = -1
    b.run()
    torch.cuda.synchronize()
    got = plain.f64(b.out).reshape(want.shape)
    assert np.isnan(got[:5]).all() and torch.isnan(b.lse[:5]).all()
    assert (np.abs(got[5] - want[5]) <= tol[5]).all() and int(b.err[0]) == 1
    b.err.zero_()
    b.pages, b.kv_len, b.q_start = clean[0], clean[1], clean[2].clone()
    b.q_start[2] = b.T + 5
    b.out.fill_(3.0)
    b.run()
    torch.cuda.synchronize()
    got = plain.f64(b.out).reshape(want.shape)
    assert (got[1:4] == 3.0).all() and int(b.err[0]) == 1
    for t in (0, 4, 5):
        assert (np.abs(got[t] - want[t]) <= tol[t]).all()
    assert (b.guard == 0xA5).all()


def test_attend_many_rows_strides_rows_and_captures(cuda):
    """A token-major pool, a strided output, rows of no sequence, another stream, a graph replayed with other lengths and counts."""
    b = Batch(cuda, 128, 16, 0, 2, 13, [500, 277, 40], [12, 11, 1], seed=9)
    b.run()
    b.check()
    c = b.cache
    both = torch.empty((c.n_pages, 2, c.page, 2, 128), dtype=torch.bfloat16, device=cuda)
    both[:, 0].copy_(c.k.transpose(1, 2)), both[:, 1].copy_(c.v.transpose(1, 2))
    other = K().KvCache(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), 16)
    out = torch.full((b.T + 2, b.n_q * 128 + 8), 3.0, dtype=torch.bfloat16, device=cuda)
    q = torch.cat((b.q[:1], b.q, b.q[:1]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    K().attn_decode(q, other, b.pages, b.q_start + 1, b.kv_len, b.max_q, out[:, :b.n_q * 128], b.ws, b.err, stream=side)
    side.synchronize()
    assert torch.equal(out[1:-1, :b.n_q * 128], b.out)
    assert (out[0] == 3.0).all() and (out[-1] == 3.0).all() and (out[:, b.n_q * 128:] == 3.0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run()
    for lens, starts in (([500, 277, 40], [0, 12, 23, 24]), ([12, 0, 33], [0, 1, 12, 24]), ([380, 129, 1], [0, 22, 24, 24])):
        b.kv_len.copy_(torch.tensor(lens, dtype=torch.int32)), b.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        b.out.fill_(float("nan")), b.lse.fill_(float("nan"))
        graph.replay()
        b.check()
    K().check_dense_status("attention")


def test_attend_many_rows_keeps_to_its_workspace_and_shares_it(cuda):
    """All CTAs at work on split segments of full tiles in a workspace of the size asked for, which calls of fewer rows use in between."""
    big = Batch(cuda, 128, 16, 0, 8, 64, [6000], [2], page=64, seed=3)
    for turn, (group, new) in enumerate(((8, 1), (8, 4), (64, 2), (8, 2), (40, 5))):
        b = Batch(cuda, 128, 16, 0, 8, group, [6000 if group > 8 else 900], [new], page=64, seed=30 + turn)
        b.ws, b.guard = big.ws, big.guard
        b.run()
        if group == 8:
            b.check()
        torch.cuda.synchronize()
        assert (big.guard == 0xA5).all() and torch.isfinite(b.out).all() and int(b.err[0]) == 0


def test_attend_one_row_out_of_many_is_the_same_by_either_form(cuda):
    """More rows than told of, in tiles of 128, whose join is laid out for those told of; and max_q beyond what there is."""
    b = with_room(Batch(cuda, 128, 16, 0, 1, 8, [9000, 300], [40, 1], max_q=5, seed=4))
    b.run()
    b.check()
    b = Batch(cuda, 128, 16, 0, 1, 8, [9000, 300], [1, 1], max_q=500, seed=4)
    b.run()
    b.check()


@pytest.mark.parametrize("new", [1, 3])
def test_attend_many_rows_nothing_unseen_counts(cuda, new):
    """NaN in every row that no query sees: behind the sequences' ends and before their windows, in the same pages as what is seen."""
    lens, window = [70, 129, 400], 40
    b = Batch(cuda, 128, 16, 0, 1, 160, lens, [new] * 3, seed=19)
    for s, n in enumerate(lens):
        for j in list(range(0, n - new + 1 - window)) + list(range(n, -(-n // 16) * 16)):
            for t in (b.cache.k, b.cache.v):
                t[int(b.pages[s, j // 16]), :, j % 16] = float("nan")
    b.run(window=window)
    b.check(window=window)

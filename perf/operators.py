"""The attention operators of a decode step over a paged key-value cache, as cases that can be timed.

Three operators:

  "write"   the projections' output [T, (n_q + 2 n_kv) D] -> queries and keys normed per head and rotated by their position, the
            queries as BF16, keys and values into the cache's pages: BF16, or 8- or 4-bit codes with a scale and a minimum a group
            (a quantized cache's rows come back through the read, as the values that they stand for);
  "attend"  the new tokens of every sequence attend over its pages: grouped heads, causal among the new tokens, optionally a
            window and a tanh cap on the scores; output and log-sum-exp;
  "read"    rows of the cache back as BF16.

Pages of one sequence lie scattered over the pool; sequences of a batch have lengths and counts of new tokens of their own.
"""
import math
import random
import zlib

import torch

own = False

EPS = 1e-6


def _write(name, T, B, n_q, n_kv, D, bits=16, G=0, page=16, rot=None, interleaved=False, norm=True, f32=False, far=False):
    return dict(name=name, kind="write", T=T, B=B, n_q=n_q, n_kv=n_kv, D=D, bits=bits, G=G, page=page, rot=D if rot is None else rot,
                interleaved=interleaved, norm=norm, f32=f32, far=far)


def _attend(name, B, q_lo, q_hi, len_lo, len_hi, n_q, n_kv, D, bits=16, G=0, page=16, window=0, cap=0.0):
    return dict(name=name, kind="attend", B=B, q_lo=q_lo, q_hi=q_hi, len_lo=len_lo, len_hi=len_hi, n_q=n_q, n_kv=n_kv, D=D, bits=bits, G=G,
                page=page, window=window, cap=cap)


def _read(name, T, B, n_kv, D, bits, G, page=16):
    return dict(name=name, kind="read", T=T, B=B, n_kv=n_kv, D=D, bits=bits, G=G, page=page)


def listed():
    return [
        # one conversation's decode step far into a long context: the launch and the call are all there is
        _write("write_decode_1", 1, 1, 32, 8, 128, far=True),
        # two conversations of one token and seven drafts, 8-bit cache, written and read back
        _write("write_q8_16", 16, 2, 32, 4, 128, bits=8, G=64, page=64),
        # a short prompt of an odd length, FP32 projections, wide heads, a quarter of them rotated in neighbouring pairs, 4-bit cache
        _write("write_q4_777", 777, 3, 16, 2, 256, bits=4, G=32, page=32, rot=64, interleaved=True, f32=True),
        # a prefill chunk into a BF16 cache
        _write("write_chunk_4096", 4096, 4, 32, 8, 128),
        # the first steps of one conversation: a few hundred keys
        _attend("attend_short_1", 1, 1, 1, 300, 300, 32, 8, 128),
        # two conversations of one token and seven drafts, deep in their contexts
        _attend("attend_drafts_16", 2, 8, 8, 30000, 33000, 32, 4, 128, page=64),
        # a ragged batch of eight conversations with one to eight rows each, 8-bit cache
        _attend("attend_ragged_q8", 8, 1, 8, 500, 9000, 32, 4, 128, bits=8, G=64, page=64),
        # a decode batch of 64 conversations of uneven lengths, 8-bit cache
        _attend("attend_batch_64_q8", 64, 1, 1, 100, 16000, 32, 8, 128, bits=8, G=64, page=32),
        # one conversation with a very long context, BF16 cache
        _attend("attend_long_1", 1, 1, 1, 200001, 200001, 32, 8, 128, page=16),
        # a batch with wide heads, capped scores and a sliding window, 4-bit cache
        _attend("attend_window_q4", 32, 1, 2, 2000, 20000, 16, 2, 256, bits=4, G=32, page=64, window=4096, cap=50.0),
        # a short conversation's rows read back
        _read("read_q4_501", 501, 1, 8, 64, 4, 32),
        # a long prompt's rows read back for a prompt cache
        _read("read_q8_33000", 33000, 2, 8, 128, 8, 64, page=64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "read"])
    D = rng.choice([64, 128, 128, 256])
    bits = rng.choice([16, 8, 4])
    G = 0 if bits == 16 else rng.choice([g for g in (32, 64, 128) if g <= D])
    n_kv = rng.choice([1, 2, 4, 8])
    page = rng.choice([8, 16, 32, 64, 128])
    n_q = n_kv * rng.choice([1, 2, 3, 4, 6, 8])
    if kind == "write":
        T = _log(rng, 1, 4096)
        return _write("", T, rng.randint(1, min(T, 64)), n_q, n_kv, D, bits, G, page, rng.choice([0, 32, D]), rng.random() < 0.3,
                      rng.random() < 0.7, rng.random() < 0.3, rng.random() < 0.3) | {"name": "drawn"}
    if kind == "read":
        return _read("drawn", _log(rng, 1, 33000), rng.randint(1, 8), n_kv, D, bits, G, page)
    B = _log(rng, 1, 64)
    most = int(2.6e8 * (16 / bits) / (2 * D * n_kv * B))  # as many bytes of cache as the longest listed cases
    hi = _log(rng, 16, max(32, min(200000, most)))
    q_hi = rng.choice([1, 1, 2, 4, 8])
    return _attend("drawn", B, 1, q_hi, max(1, int(hi * rng.choice([0.01, 0.5, 1.0]))), hi, n_q, n_kv, D, bits, G, page,
                   rng.choice([0, 0, 100, 4096]), rng.choice([0.0, 0.0, 50.0]))


# ---- what a case holds -------------------------------------------------------------------------------------------------------------

def _spread(case, salt, lo, hi, n):
    """n numbers of [lo, hi] by the case alone."""
    r = random.Random(zlib.crc32(repr((salt, sorted((k, v) for k, v in case.items() if k != "name"))).encode()))
    return [r.randint(lo, hi) for _ in range(n)]


def _split(case):
    """A write's or a read's tokens per sequence."""
    T, B = case["T"], case["B"]
    return [T // B + (b < T % B) for b in range(B)]


def _starts(case):
    """Position of a write's or a read's first token in each sequence."""
    return _spread(case, "start", 90000, 110000, case["B"]) if case.get("far") else _spread(case, "start", 0, 500, case["B"])


def _new(case):
    return _spread(case, "new", case["q_lo"], case["q_hi"], case["B"])


def _lens(case):
    return [max(n, m) for n, m in zip(_spread(case, "len", case["len_lo"], case["len_hi"], case["B"]), _new(case))]


def _row_bytes(case):
    """Bytes of one cache row (a token's key or value in one head)."""
    D, bits = case["D"], case["bits"]
    return D * bits // 8 + (0 if bits == 16 else 4 * (D // case["G"]))


def work(case):
    D, n_kv = case["D"], case["n_kv"]
    if case["kind"] == "write":
        T, n_q, es = case["T"], case["n_q"], 4 if case["f32"] else 2
        b = T * (n_q + 2 * n_kv) * D * es + T * n_q * D * 2 + 2 * T * n_kv * _row_bytes(case) + 8 * T
        if case["bits"] != 16:
            b += 2 * T * n_kv * (_row_bytes(case) + 2 * D)  # the read back
        return {"bytes": b, "flops": 10 * T * (n_q + 2 * n_kv) * D}
    if case["kind"] == "read":
        return {"bytes": 2 * case["T"] * n_kv * (_row_bytes(case) + 2 * D) + 8 * case["T"], "flops": 4 * case["T"] * n_kv * D}
    keys = pairs = 0
    for n, length in zip(_new(case), _lens(case)):
        w = case["window"] or length + n
        keys += length - max(0, length - n + 1 - w)
        pairs += sum(min(length - n + 1 + i, w) for i in range(n))
    rows = sum(_new(case)) * case["n_q"]
    return {"bytes": 2 * keys * n_kv * _row_bytes(case) + rows * (4 * D + 4) + 4 * (keys // case["page"] + 1), "flops": 4 * pairs * case["n_q"] * D}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------

def _pages(case, lens, g):
    """A pool a little larger than the sequences need, and their pages scattered over it."""
    P = case["page"]
    need = [-(-n // P) for n in lens]
    n_pages, wide = sum(need) + 7, max(need)
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), wide), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return n_pages, table


def _quantize(x, G, bits):
    """x [..., D] -> codes (4 bits: two a byte, the even element low) and [..., D / G, 2], a group's scale and minimum."""
    levels = float(2 ** bits - 1)
    v = x.reshape(*x.shape[:-1], -1, G)
    lo, hi = v.amin(-1), v.amax(-1)
    scale, least = ((hi - lo) / levels).to(torch.bfloat16), lo.to(torch.bfloat16)
    s = scale.float().unsqueeze(-1)
    q = torch.where(s > 0, torch.round((v - least.float().unsqueeze(-1)) / torch.where(s > 0, s, 1.0)), 0.0).clamp(0, levels).to(torch.uint8)
    q = q.reshape(x.shape)
    return (q[..., 0::2] | (q[..., 1::2] << 4)) if bits == 4 else q, torch.stack((scale, least), -1)


def _pool(case, n_pages, g, filled):
    """Keys and values [n_pages, n_kv, page, D] of the pool: N(0, 1), the values with a mean of their own a channel."""
    shape = (n_pages, case["n_kv"], case["page"], case["D"])
    pool = {}
    for name in ("k", "v"):
        mean = torch.randn((case["n_kv"], 1, case["D"]), generator=g, device="cuda") * 0.5
        parts = []
        step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
        for p in range(0, n_pages, step):
            n = min(step, n_pages - p)
            x = torch.randn((n, *shape[1:]), generator=g, device="cuda") + mean if filled else torch.zeros((n, *shape[1:]), device="cuda")
            parts.append((x.to(torch.bfloat16),) if case["bits"] == 16 else _quantize(x, case["G"], case["bits"]))
        for key, t in zip(("", "_sm"), zip(*parts)):
            pool[name + key] = torch.cat(t)
    return pool


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 11)
    st = dict(case)
    D, n_kv = case["D"], case["n_kv"]
    if case["kind"] in ("write", "read"):
        T, counts, starts = case["T"], _split(case), _starts(case)
        st["n_pages"], st["pages"] = _pages(case, [s + n for s, n in zip(starts, counts)], g)
        st["seq"] = torch.tensor([b for b, n in enumerate(counts) for _ in range(n)], dtype=torch.int32, device="cuda")
        st["pos"] = torch.tensor([s + i for s, n in zip(starts, counts) for i in range(n)], dtype=torch.int32, device="cuda")
        st.update(_pool(case, st["n_pages"], g, case["kind"] == "read"))
        st["k_out"] = torch.zeros((T, n_kv, D), dtype=torch.bfloat16, device="cuda")
        st["v_out"] = torch.zeros((T, n_kv, D), dtype=torch.bfloat16, device="cuda")
    if case["kind"] == "write":
        n_q = case["n_q"]
        x = torch.randn((T, (n_q + 2 * n_kv) * D), generator=g, device="cuda")
        st["qkv"] = x if case["f32"] else x.to(torch.bfloat16)
        st["q_norm"] = 1 + 0.2 * torch.randn(D, generator=g, device="cuda") if case["norm"] else None
        st["k_norm"] = 1 + 0.2 * torch.randn(D, generator=g, device="cuda") if case["norm"] else None
        rot = case["rot"]
        st["inv_freq"] = (1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)).float() if rot else None
        st["q_out"] = torch.zeros((T, n_q * D), dtype=torch.bfloat16, device="cuda")
    if case["kind"] == "attend":
        new, lens, n_q = _new(case), _lens(case), case["n_q"]
        st["n_pages"], st["pages"] = _pages(case, lens, g)
        st.update(_pool(case, st["n_pages"], g, True))
        st["q_start"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        st["kv_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["seq"] = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], dtype=torch.int64, device="cuda")
        st["max_q"] = max(new)
        st["q"] = (torch.randn((sum(new), n_q * D), generator=g, device="cuda") * 1.5).to(torch.bfloat16)
        st["out"] = torch.zeros_like(st["q"])
        st["lse"] = torch.zeros((sum(new), n_q), device="cuda")
        st["scale"] = D ** -0.5
    st["err"] = torch.zeros(4, dtype=torch.int32, device="cuda")
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------

def _norm_rotate(st, x, weight):
    """x [T, heads, D] FP32: norm of each head, rotation of its first `rot` elements."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    if st["inv_freq"] is None:
        return x
    angle = st["pos"].double()[:, None, None] * st["inv_freq"].double()
    c, s = angle.cos().float(), angle.sin().float()
    rot = st["rot"]
    turned, rest = x[..., :rot], x[..., rot:]
    if st["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, rest), -1)


def _values(st, name, page, at):
    """Rows of the cache as FP32: page and at broadcast to [...]; -> [..., n_kv, D]."""
    codes = st[name][page, :, at]
    if st["bits"] == 16:
        return codes.float()
    if st["bits"] == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    sm = st[name + "_sm"][page, :, at].float()
    x = codes.reshape(*codes.shape[:-1], -1, st["G"]).float()
    return (x * sm[..., :1] + sm[..., 1:]).flatten(-2)


def _plain_read(st):
    page, at = st["pages"][st["seq"].long(), st["pos"].long() // st["page"]].long(), st["pos"].long() % st["page"]
    return _values(st, "k", page, at).to(torch.bfloat16), _values(st, "v", page, at).to(torch.bfloat16)


def _store(st, name, page, at, x):
    if st["bits"] == 16:
        st[name][page, :, at] = x.to(torch.bfloat16)
        return
    st[name][page, :, at], st[name + "_sm"][page, :, at] = _quantize(x, st["G"], st["bits"])


def _plain_write(st):
    n_q, n_kv, D = st["n_q"], st["n_kv"], st["D"]
    x = st["qkv"].float().view(-1, n_q + 2 * n_kv, D)
    q = _norm_rotate(st, x[:, :n_q], st["q_norm"]).to(torch.bfloat16).flatten(1)
    k = _norm_rotate(st, x[:, n_q:n_q + n_kv], st["k_norm"])
    page, at = st["pages"][st["seq"].long(), st["pos"].long() // st["page"]].long(), st["pos"].long() % st["page"]
    _store(st, "k", page, at, k)
    _store(st, "v", page, at, x[:, n_q + n_kv:])
    return (q, st["k"], st["v"]) if st["bits"] == 16 else (q, *_plain_read(st))


def _plain_attend(st):
    n_q, n_kv, D, B = st["n_q"], st["n_kv"], st["D"], st["kv_len"].numel()
    group, T = n_q // n_kv, st["q"].shape[0]
    new = (st["q_start"][1:] - st["q_start"][:-1]).long()
    j = torch.arange(st["pages"].shape[1] * st["page"], device="cuda")
    page, at = st["pages"].long()[:, j // st["page"]], (j % st["page"]).expand(B, -1)
    seq = st["seq"]
    row = torch.arange(T, device="cuda") - st["q_start"].long()[seq]
    q = torch.zeros((B, st["max_q"], n_kv, group, D), device="cuda")
    q[seq, row] = st["q"].float().view(T, n_kv, group, D)
    q = q.permute(0, 2, 1, 3, 4).reshape(B, n_kv, st["max_q"] * group, D)
    s = torch.matmul(q, _values(st, "k", page, at).permute(0, 2, 3, 1)) * st["scale"]
    if st["cap"]:
        s = st["cap"] * torch.tanh(s / st["cap"])
    p = (st["kv_len"].long() - new)[:, None] + torch.arange(st["max_q"], device="cuda")
    seen = j <= p[..., None]
    if st["window"]:
        seen = seen & (j > p[..., None] - st["window"])
    seen = seen[:, None, :, None].expand(B, n_kv, st["max_q"], group, -1).flatten(2, 3)
    s = torch.where(seen, s, -math.inf)
    most = s.amax(-1, keepdim=True).clamp_min(-1e30)
    e = torch.exp(s - most)
    total = e.sum(-1, keepdim=True)
    v = torch.where((j < st["kv_len"][:, None])[..., None, None], _values(st, "v", page, at), 0.0)
    o = torch.matmul(e, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    lse = (most + torch.log(total)).view(B, n_kv, st["max_q"], group).permute(0, 2, 1, 3).flatten(2)
    o = o.view(B, n_kv, st["max_q"], group, D).permute(0, 2, 1, 3, 4).flatten(2)
    return o[seq, row].to(torch.bfloat16), lse[seq, row]


def run(st):
    if not own:
        if st["kind"] == "write":
            return _plain_write(st)
        return _plain_read(st) if st["kind"] == "read" else _plain_attend(st)
    from strixite_b200 import kernels as K
    if "cache" not in st:  # the handle and the workspace that a program keeps
        st["cache"] = K.KvCache(st["k"], st["v"], st["bits"], st["G"], st.get("k_sm"), st.get("v_sm"))
        if st["kind"] == "attend":
            st["ws"] = torch.zeros(K.attn_decode_workspace_bytes(st["cache"], st["n_q"], st["max_q"]), dtype=torch.uint8, device="cuda")
    if st["kind"] == "attend":
        K.attn_decode(st["q"], st["cache"], st["pages"], st["q_start"], st["kv_len"], st["max_q"], st["out"], st["ws"], st["err"],
                      scale=st["scale"], softcap=st["cap"], window=st["window"], lse=st["lse"])
        return st["out"], st["lse"]
    if st["kind"] == "write":
        K.attn_qkv_write(st["qkv"], st["cache"], st["seq"], st["pos"], st["pages"], st["q_out"], st["err"], q_norm=st["q_norm"],
                         k_norm=st["k_norm"], eps=EPS, inv_freq=st["inv_freq"], interleaved=st["interleaved"])
        if st["bits"] == 16:
            return st["q_out"], st["k"], st["v"]
    K.kv_read(st["cache"], st["seq"], st["pos"], st["pages"], st["k_out"], st["v_out"], st["err"])
    return (st["q_out"], st["k_out"], st["v_out"]) if st["kind"] == "write" else (st["k_out"], st["v_out"])


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------

def _wide(st, name, rows_page, rows_at):
    """Cache rows as FP64 [rows, n_kv, D]."""
    c = st[name][rows_page][torch.arange(len(rows_at)), :, rows_at]
    if st["bits"] == 16:
        return c.double()
    D, G = st["D"], st["G"]
    c = c.long()
    x = torch.empty((*c.shape[:2], D), dtype=torch.float64, device="cuda")
    if st["bits"] == 4:
        x[..., 0::2] = (c % 16).double()
        x[..., 1::2] = (c // 16).double()
    else:
        x.copy_(c)
    sm = st[name + "_sm"][rows_page][torch.arange(len(rows_at)), :, rows_at].double()
    return x * sm[..., 0].repeat_interleave(G, -1) + sm[..., 1].repeat_interleave(G, -1)


def _as_kept(x, G, bits):
    """What a quantized cache holds of x [rows, heads, D] FP64: the scale and the minimum are BF16 numbers, codes go to the nearest."""
    top = 2.0 ** bits - 1
    y = torch.empty_like(x)
    for g0 in range(0, x.shape[-1], G):
        part = x[..., g0:g0 + G]
        m = part.min(-1, keepdim=True).values.float().to(torch.bfloat16).double()
        s = ((part.max(-1, keepdim=True).values - part.min(-1, keepdim=True).values) / top).float().to(torch.bfloat16).double()
        code = torch.where(s > 0, ((part - m) / s.clamp_min(1e-300)).round().clamp(0, top), torch.zeros_like(part))
        y[..., g0:g0 + G] = code * s + m
    return y


def exact(case, seed):
    st = prepare(case, seed)
    n_kv, D, P = case["n_kv"], case["D"], case["page"]
    if case["kind"] in ("write", "read"):
        page = st["pages"].cpu()[st["seq"].cpu().long(), st["pos"].cpu().long() // P].long().to("cuda")
        at = st["pos"].long() % P
    if case["kind"] == "read":
        return _wide(st, "k", page, at), _wide(st, "v", page, at)
    if case["kind"] == "write":
        n_q, T, rot = case["n_q"], case["T"], case["rot"]
        x = st["qkv"].double().view(T, n_q + 2 * n_kv, D).clone()
        if case["norm"]:
            for lo, hi, w in ((0, n_q, st["q_norm"]), (n_q, n_q + n_kv, st["k_norm"])):
                x[:, lo:hi] = x[:, lo:hi] / (x[:, lo:hi].pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        if rot:
            z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(st["pos"].double(), st["inv_freq"].double()))
            i = torch.arange(rot // 2, device="cuda")
            first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
            y = torch.complex(x[:, :n_q + n_kv, first], x[:, :n_q + n_kv, second]) * z[:, None]
            x[:, :n_q + n_kv, first], x[:, :n_q + n_kv, second] = y.real, y.imag
        q, k, v = x[:, :n_q].reshape(T, -1), x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]
        if case["bits"] != 16:
            return q, _as_kept(k, case["G"], case["bits"]), _as_kept(v, case["G"], case["bits"])
        kept = [st["k"].double(), st["v"].double()]
        for c, new in zip(kept, (k, v)):
            c[page, :, at] = new
        return q, kept[0], kept[1]
    group, out, lse, t = case["n_q"] // n_kv, [], [], 0
    for b, (n, length) in enumerate(zip(_new(case), _lens(case))):
        keys = torch.arange(length, device="cuda")
        k, v = (_wide(st, c, st["pages"][b].long()[keys // P], keys % P) for c in ("k", "v"))
        for i in range(n):
            first = max(0, length - n + i + 1 - case["window"]) if case["window"] else 0
            last = length - n + i + 1
            q = st["q"][t].double().view(n_kv, group, D)
            s = torch.einsum("hgd,jhd->hgj", q, k[first:last]) * st["scale"]
            s = case["cap"] * torch.tanh(s / case["cap"]) if case["cap"] else s
            lse.append(torch.logsumexp(s, -1).reshape(-1))
            out.append(torch.einsum("hgj,jhd->hgd", torch.softmax(s, -1), v[first:last]).reshape(-1))
            t += 1
    return torch.stack(out), torch.stack(lse)

"""The operators around the head of a decode or draft-verify step, as cases that can be timed.

Three operators:

  "norm"    residual's addition and root-mean-square norm: x + y stored in x's type, its norm as 8-bit floating-point codes (e4m3) with a scale for
            each block of 128;
  "linear"  matrix product of such codes with 8-bit floating-point weights that have a scale for each block of 128 x 128;
  "verify"  drafted tokens of every sequence against the target's probabilities, from given random numbers: tokens kept, the next token drawn.

Rows of a step's sequences stand one after the other; sequences of a batch have counts of their own.
"""
import math
import random
import zlib

import torch

own = False

EPS = 1e-6
BLOCK = 128
TOP = 448.0  # the largest e4m3 number
LEAST = 2.0 ** -64  # of a scale


def _norm(name, T, d, y="bf16", f32=False, weight=True):
    return dict(name=name, kind="norm", T=T, d=d, y=y, f32=f32, weight=weight)


def _linear(name, M, N, K, f32=False):
    return dict(name=name, kind="linear", M=M, N=N, K=K, f32=f32)


def _verify(name, B, m_lo, m_hi, V, f32=True, drafted="token", greedy=0):
    """drafted: "token" (the drafter's pick only) or "logits" (its distribution too); greedy: every so manieth sequence has temperature 0 (0: none)."""
    return dict(name=name, kind="verify", B=B, m_lo=m_lo, m_hi=m_hi, V=V, f32=f32, drafted=drafted, greedy=greedy)


def listed():
    return [
        # one conversation's decode step: the launch and the call are all there is
        _norm("norm_decode_1", 1, 4096),
        # a short prompt of an odd length, the expert layer's output in FP32
        _norm("norm_777", 777, 2560, y="f32"),
        # a prefill chunk
        _norm("norm_chunk_16384", 16384, 4096),
        # one conversation's decode step: queries, keys and values of 32 and 8 heads, FP32 for the norm and rotation behind it
        _linear("linear_decode_1", 1, 6144, 4096, f32=True),
        # two conversations of one token and seven drafts: the head's logits
        _linear("linear_head_16", 16, 131072, 4096, f32=True),
        # a batch of decoding conversations: an output projection
        _linear("linear_batch_150", 150, 2560, 4096),
        # a short prompt, sizes that no tile divides
        _linear("linear_odd_777", 777, 1000, 1040),
        # a prefill chunk's gate and up projection
        _linear("linear_chunk_8192", 8192, 8192, 4096),
        # one conversation without drafts: the next token drawn
        _verify("verify_one", 1, 1, 1, 32768),
        # two conversations of one token and seven drafts, of which the drafter gives the tokens
        _verify("verify_drafts_16", 2, 8, 8, 131072),
        # a ragged batch with greedy conversations in it, an odd vocabulary in BF16
        _verify("verify_ragged_16", 16, 1, 5, 100003, f32=False, greedy=3),
        # a large batch whose drafter gives its distributions
        _verify("verify_batch_64", 64, 1, 8, 131072, f32=False, drafted="logits"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "verify", "verify"])
    if kind == "norm":
        T = _log(rng, 1, 16384)
        d = 16 * _log(rng, 4, max(4, min(1024, 16384 * 4096 // (16 * T))))
        f32 = rng.random() < 0.2
        return _norm("drawn", T if not f32 else -(-T // 2), d, rng.choice(["bf16", "f32", "none"]), f32, rng.random() < 0.9)
    if kind == "linear":
        M = _log(rng, 1, 8192)
        K = 16 * _log(rng, 8, 512)
        most = min(131072 * 4096 // K, 8192 * 8192 * 4096 // (M * K), 131072 * 16 // M + 8192)
        return _linear("drawn", M, _log(rng, 32, max(32, most)), K, rng.random() < 0.3)
    B = _log(rng, 1, 64)
    m_hi = rng.choice([1, 2, 4, 8])
    return _verify("drawn", B, rng.choice([1, m_hi]), m_hi, _log(rng, 1000, 131072), rng.random() < 0.5, rng.choice(["token", "logits"]), rng.choice([0, 0, 2, 4]))


# ---- what a case holds -------------------------------------------------------------------------------------------------------------

def _counts(case):
    """Rows of each sequence of a verification, by the case alone."""
    r = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    return [r.randint(case["m_lo"], case["m_hi"]) for _ in range(case["B"])]


def work(case):
    if case["kind"] == "norm":
        T, d = case["T"], case["d"]
        es = 4 if case["f32"] else 2
        row = d * (es + 1) + 4 * -(-d // BLOCK)
        if case["y"] != "none":
            row += d * (es + (4 if case["y"] == "f32" else 2))
        return {"bytes": T * row + 4 * d * case["weight"], "flops": 8 * T * d}
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // BLOCK)
        return {"bytes": M * K + N * K + 4 * kb * (M + -(-N // BLOCK)) + M * N * (4 if case["f32"] else 2), "flops": 2 * M * N * K}
    rows = sum(_counts(case))
    read = rows + (rows - case["B"] if case["drafted"] == "logits" else 0)
    return {"bytes": read * case["V"] * (4 if case["f32"] else 2) + 16 * rows, "flops": 4 * read * case["V"]}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------

def _codes(x, rows):
    """x [R, K] -> e4m3 codes and FP32 scales of blocks of `rows` rows (1 or 128) and 128 columns."""
    R, K = x.shape
    rb, kb = -(-R // rows), -(-K // BLOCK)
    padded = torch.zeros((rb * rows, kb * BLOCK), device=x.device)
    padded[:R, :K] = x
    v = padded.view(rb, rows, kb, BLOCK)
    scale = (v.abs().amax((1, 3)) / TOP).clamp_min(LEAST)
    codes = (v / scale[:, None, :, None]).clamp(-TOP, TOP).view(rb * rows, kb * BLOCK)[:R, :K]
    return codes.to(torch.float8_e4m3fn).contiguous(), scale


def _weights(N, K, g):
    """N(0, 0.02) with a size of its own for every output row, quantized; made in slices."""
    parts = []
    step = max(BLOCK, (1 << 26) // K // BLOCK * BLOCK)
    for n in range(0, N, step):
        rows = min(step, N - n)
        w = torch.randn((rows, K), generator=g, device="cuda") * 0.02
        parts.append(_codes(w * torch.exp(0.3 * torch.randn((rows, 1), generator=g, device="cuda")), BLOCK))
    return torch.cat([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn), torch.cat([p[1] for p in parts])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 23)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    st = dict(case)
    if case["kind"] == "norm":
        T, d = case["T"], case["d"]
        kept = torch.float32 if case["f32"] else torch.bfloat16
        # a residual stream: a size of its own for each row, a few channels far larger than the others
        size = torch.exp(0.5 * randn(T, 1)) * torch.where(torch.rand(d, generator=g, device="cuda") < 0.005, 30.0, 1.0)
        st["x"] = (randn(T, d) * size).to(kept)
        st["y"] = None if case["y"] == "none" else (0.5 * randn(T, d)).to(torch.float32 if case["y"] == "f32" else torch.bfloat16)
        st["w"] = 1 + 0.2 * randn(d) if case["weight"] else None
        st["total"] = None if case["y"] == "none" else torch.zeros((T, d), dtype=kept, device="cuda")
        st["codes"] = torch.zeros((T, d), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        st["scales"] = torch.zeros((T, -(-d // BLOCK)), device="cuda")
    elif case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        st["x"], st["xs"] = _codes(randn(M, K) * torch.exp(0.5 * randn(1, K)), 1)
        st["w"], st["ws"] = _weights(N, K, g)
        st["y"] = torch.zeros((M, N), dtype=torch.float32 if case["f32"] else torch.bfloat16, device="cuda")
    else:
        B, V, counts = case["B"], case["V"], _counts(case)
        T = sum(counts)
        kept = torch.float32 if case["f32"] else torch.bfloat16
        starts = [sum(counts[:b]) for b in range(B + 1)]
        st["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        st["seq"] = torch.tensor([b for b, m in enumerate(counts) for _ in range(m)], dtype=torch.int64, device="cuda")
        t = 0.6 + 0.6 * torch.rand(B, generator=g, device="cuda")
        if case["greedy"]:
            t[::case["greedy"]] = 0.0
        st["temperature"] = t
        # a row's logits: many unlikely tokens, a few likely ones; the drafter sees them through noise
        logits = 2.5 * randn(T, V)
        likely = torch.randint(0, V, (T, 4), generator=g, device="cuda")
        logits.scatter_add_(1, likely, 7 + 5 * torch.rand((T, 4), generator=g, device="cuda"))
        drafts = 0.9 * logits + 0.5 * randn(T, V)
        drafts.scatter_add_(1, likely[:, :1], 2 * randn(T, 1))
        st["logits"], drafts = logits.to(kept), drafts.to(kept)
        del logits
        # drafted tokens: drawn from the drafter's distribution, or its pick
        if case["drafted"] == "logits":
            noise = -torch.log(-torch.log(torch.rand((T, V), generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
            picked = (drafts.float() / torch.where(t > 0, t, 1e-3)[st["seq"]][:, None] + noise).argmax(1)
            st["draft_logits"] = drafts
        else:
            picked = drafts.float().argmax(1)
            st["draft_logits"] = None
        st["ids"] = torch.cat((torch.randint(0, V, (1,), generator=g, device="cuda"), picked[:-1])).to(torch.int32)
        st["u"] = torch.rand(T, generator=g, device="cuda")
        st["u_pick"] = torch.rand(B, generator=g, device="cuda")
        st["next_ids"] = torch.zeros(T, dtype=torch.int32, device="cuda")
        st["n_new"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        st["logp"] = torch.zeros(T, device="cuda")
        st["err"] = torch.zeros(4, dtype=torch.int32, device="cuda")
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------

def _plain_norm(st):
    x = st["x"].float()
    total = None
    if st["y"] is not None:
        total = (x + st["y"].float()).to(st["x"].dtype)
        x = total.float()
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    if st["w"] is not None:
        n = n * st["w"]
    codes, scales = _codes(n, 1)
    return (codes, scales) if total is None else (total, codes, scales)


def _plain_linear(st):
    M, N, K = st["M"], st["N"], st["K"]
    x = st["x"].float() * st["xs"].repeat_interleave(BLOCK, 1)[:, :K]
    w = st["w"].float() * st["ws"].repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    return torch.matmul(x, w.t()).to(st["y"].dtype)


def _softmax(logits, t):
    """Probabilities [R, V] and log-sums [R, 1] in 64 bits: words next to a border of the sum go by them."""
    z = logits.double() / t[:, None]
    most = z.amax(1, keepdim=True)
    e = torch.exp(z - most)
    total = e.sum(1, keepdim=True)
    return e / total, most + torch.log(total)


def _plain_verify(st):
    T, V, B, seq = st["ids"].shape[0], st["V"], st["B"], st["seq"]
    t = st["temperature"].double()
    greedy = (t == 0)[seq]
    t = torch.where(t > 0, t, 1.0)[seq]
    p, lse = _softmax(st["logits"], t)
    rows = torch.arange(T, device="cuda")
    last = rows + 1 == st["q_start"].long()[1:][seq]
    drafted = st["ids"].long().roll(-1)
    px = p.gather(1, drafted[:, None])[:, 0]
    best = torch.where(st["logits"] == st["logits"].amax(1, keepdim=True), torch.arange(V, device="cuda"), V).amin(1)
    q = None
    qx = torch.ones_like(px)
    if st["draft_logits"] is not None:
        q = _softmax(st["draft_logits"], t)[0]
        qx = q.gather(1, drafted[:, None])[:, 0]
    kept = torch.where(greedy, best == drafted, st["u"].double() * qx < px) & ~last
    # the first row of each sequence that keeps no draft
    at = torch.full((B,), T, device="cuda").scatter_reduce(0, seq, torch.where(kept, T, rows), "amin")
    w = p[at]
    refused = ~last[at]
    if q is None:
        less = w.scatter(1, drafted[at][:, None], 0.0)
    else:
        less = (w - q[at]).clamp_min(0.0)
    refused = refused & (less.sum(1) > 0)
    cum = torch.where(refused[:, None], less, w).cumsum(1)
    token = torch.searchsorted(cum, st["u_pick"].double()[:, None] * cum[:, -1:], right=True)[:, 0].clamp_max(V - 1)
    token = torch.where(greedy[at], best[at], token)
    n_new = at - st["q_start"].long()[:-1] + 1
    ids = torch.where(rows < at[seq], drafted, torch.where(rows == at[seq], token[seq], -1))
    z = st["logits"].gather(1, ids.clamp_min(0)[:, None]).double()[:, 0] / t
    logp = torch.where(ids >= 0, z - lse[:, 0], 0.0)
    return ids.to(torch.int32), n_new.to(torch.int32), logp.float()


def run(st):
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "verify": _plain_verify}[st["kind"]](st)
    from strixite_b200 import kernels as K
    if st["kind"] == "norm":
        K.add_norm(st["x"], y=st["y"], weight=st["w"], eps=EPS, total=st["total"], codes=st["codes"], scales=st["scales"])
        return (st["codes"], st["scales"]) if st["total"] is None else (st["total"], st["codes"], st["scales"])
    if st["kind"] == "linear":
        if "view" not in st:  # the handle that a program keeps
            st["view"] = K.F8View(st["w"], st["ws"])
        K.linear_f8(st["x"], st["xs"], st["view"], st["y"])
        return st["y"]
    if "work" not in st:  # the workspace that a program keeps
        st["work"] = torch.zeros(K.verify_drafts_workspace_bytes(st["ids"].shape[0], st["B"], st["V"]), dtype=torch.uint8, device="cuda")
    K.verify_drafts(st["logits"], st["ids"], st["q_start"], st["u"], st["u_pick"], st["next_ids"], st["n_new"], st["work"], st["err"],
                    draft_logits=st["draft_logits"], temperature=st["temperature"], logp=st["logp"])
    return st["next_ids"], st["n_new"], st["logp"]


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------

def _exact_norm(case, st):
    d = case["d"]
    x = st["x"].double()
    if st["y"] is not None:
        x = x + st["y"].double()
        kept = x
        x = x.to(st["x"].dtype).double()  # the norm is of what is stored
    n = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt()
    if st["w"] is not None:
        n = n * st["w"].double()
    codes, scales = torch.empty_like(n), []
    for lo in range(0, d, BLOCK):
        part = n[:, lo:lo + BLOCK]
        s = (part.abs().max(1, keepdim=True).values / TOP).clamp_min(LEAST)
        v = part / s
        # e4m3: four significant bits, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        codes[:, lo:lo + BLOCK] = torch.round(v / step) * step
        scales.append(s)
    scales = torch.cat(scales, 1)
    return (codes, scales) if st["y"] is None else (kept, codes, scales)


def _exact_linear(case, st):
    y = torch.zeros((case["M"], case["N"]), dtype=torch.float64, device="cuda")
    by_row = torch.arange(case["N"], device="cuda") // BLOCK
    for b in range(st["xs"].shape[1]):
        cols = slice(b * BLOCK, (b + 1) * BLOCK)
        y += (st["x"][:, cols].double() @ st["w"][:, cols].double().T) * st["xs"][:, b].double()[:, None] * st["ws"][by_row, b].double()
    return y


def _exact_verify(case, st):
    V, ids, new, logp, r = case["V"], [], [], [], 0
    fed, u, u_pick, ts = st["ids"].tolist(), st["u"].double().cpu(), st["u_pick"].double().cpu(), st["temperature"].double().cpu()
    for b, m in enumerate(_counts(case)):
        t = float(ts[b])
        logs = torch.log_softmax(st["logits"][r:r + m].double() / (t or 1.0), 1)
        draft = None if st["draft_logits"] is None else torch.log_softmax(st["draft_logits"][r:r + m].double() / (t or 1.0), 1)
        said = []
        for i in range(m):
            p = logs[i].exp()
            likely = int((st["logits"][r + i] == st["logits"][r + i].max()).nonzero()[0])
            if i + 1 < m:
                x = fed[r + i + 1]
                q = float(draft[i, x].exp()) if draft is not None else 1.0
                if (x == likely) if t == 0 else float(u[r + i]) * q < float(p[x]):
                    said.append(x)
                    continue
                if t:
                    rest = p.clone()
                    if draft is None:
                        rest[x] = 0
                    else:
                        rest = torch.clamp(rest - draft[i].exp(), min=0)
                    p = rest if float(rest.sum()) > 0 else p
            c = torch.cumsum(p, 0)
            said.append(likely if t == 0 else min(V - 1, int((c <= u_pick[b] * c[-1]).sum())))
            break
        logp += [float(logs[i, x]) for i, x in enumerate(said)] + [0.0] * (m - len(said))
        ids += said + [-1] * (m - len(said))
        new.append(len(said))
        r += m
    return (torch.tensor(ids, dtype=torch.int32, device="cuda"), torch.tensor(new, dtype=torch.int32, device="cuda"),
            torch.tensor(logp, dtype=torch.float64, device="cuda"))


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "verify": _exact_verify}[case["kind"]](case, st)

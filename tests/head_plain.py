"""The operators around the head in 64 bits, and how far the kernels' results may be from it.

The bounds count roundings.  u = 2^-24 is FP32's.  A sum of d squares by threads of up to 32 terms and trees of at most 10 levels is off by (32 + 10) u at most, half of it in the
root, with mean, root, reciprocal and two products a few more: 32 u of the norm.  A block's sum of products is that of four matrix instructions of 33 addends, each of which may
lose a last place of the largest: 4 * 33 * 2 u of the sum of sizes; the blocks' sums add an u each."""
import numpy as np
import torch

U = 2.0 ** -24
BF16 = 2.0 ** -8
NORM = 32 * U
BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -64


def f64(t):
    return t.detach().to("cpu").to(torch.float32 if t.dtype == torch.float8_e4m3fn else t.dtype).to(torch.float64).numpy()


def norm(s, weight, eps):
    """s [T, d] FP64 -> its norm."""
    n = s / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    return n if weight is None else n * f64(weight)


def block_max(n):
    T, d = n.shape
    pad = np.zeros((T, -(-d // BLOCK) * BLOCK))
    pad[:, :d] = np.abs(n)
    return pad.reshape(T, -1, BLOCK).max(-1)


def spread(scale, d):
    return np.repeat(scale, BLOCK, -1)[..., :d]


def check_codes(codes, scales, n, off):
    """Codes and scales of blocks of a row against n [T, d], known to `off` of its size."""
    want = np.maximum(block_max(n) / TOP, LEAST)
    scales, codes = f64(scales), f64(codes)
    assert np.all(np.abs(scales - want) <= (off + 2 * U) * want)
    v = n / spread(scales, n.shape[1])
    # half a step: 2^-4 of the number, half of 2^-9 below 2^-6; n's own error and the product's with the reciprocal before it
    assert np.all(np.abs(codes - v) <= np.maximum(2.0 ** -4 * np.abs(v), 2.0 ** -10) * 1.001 + (off + 4 * U) * np.abs(v))
    assert np.all(np.abs(codes) <= TOP)


def linear(x, xs, w, ws):
    """-> y [M, N] FP64 and the sum of the sizes of what it is made of, with the number of blocks."""
    x, w, xs, ws = f64(x), f64(w), f64(xs), f64(ws)
    a = x * spread(xs, x.shape[1])
    b = w * spread(np.repeat(ws, BLOCK, 0)[:w.shape[0]], w.shape[1])
    return a @ b.T, np.abs(a) @ np.abs(b).T, xs.shape[1]


def linear_bound(y, size, blocks, bf16):
    return (4 * 33 * 2 + 2 * blocks + 4) * U * size + (BF16 * np.abs(y) if bf16 else 0)


P_OFF = 2.0 ** -19    # of a probability: 2^-23 of an exponent of some ten, ex2's 2^-22, 2 x 28 roundings of sums


def softmax(z, t):
    z = z.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        e = np.exp((z - z.max()) / t)
    return e / e.sum()


def check_verified(logits, ids, q_start, u, u_pick, draft, temperature, next_ids, n_new, logp, skip=()):
    """The results sequence by sequence; where a random number stands within the bound of a border either side of it will do."""
    logits, draft = f64(logits), None if draft is None else f64(draft)
    ids, q_start, u, u_pick = (t.cpu().numpy() for t in (ids, q_start, u, u_pick))
    next_ids, n_new = next_ids.cpu().numpy(), n_new.cpu().numpy()
    logp = None if logp is None else f64(logp)
    for b in range(len(n_new)):
        if b in skip:
            continue
        lo, hi = int(q_start[b]), int(q_start[b + 1])
        t = 1.0 if temperature is None else float(temperature[b])
        if lo == hi:
            assert n_new[b] == 0
            continue
        kept = int(n_new[b]) - 1
        assert 0 <= kept < hi - lo, (b, kept)
        assert np.all(next_ids[lo + kept + 1:hi] == -1)
        if logp is not None:
            assert np.all(logp[lo + kept + 1:hi] == 0)
        for i in range(kept + 1):
            row, last = lo + i, lo + i + 1 == hi
            said = int(next_ids[row])
            p = softmax(logits[row], t or 1.0)
            best = int(np.flatnonzero(logits[row] == logits[row].max())[0])
            if logp is not None:
                want = (logits[row, said] - logits[row].max()) / (t or 1.0) - np.log(np.exp((logits[row] - logits[row].max()) / (t or 1.0)).sum())
                assert abs(logp[row] - want) <= P_OFF + 4 * U * abs(want), (b, i, logp[row], want)
            if t == 0:
                assert said == best, (b, i)
                if i < kept:
                    assert said == ids[row + 1]
                elif not last:
                    assert best != ids[row + 1]
                continue
            q = None
            if not last:
                x = int(ids[row + 1])
                q = np.eye(1, len(p), x)[0] if draft is None else softmax(draft[row], t)
                side = float(u[row]) * q[x] - p[x]
                room = 2 * P_OFF * (p[x] + q[x])
                if i < kept:
                    assert said == x and side <= room, (b, i, side)
                    continue
                assert side >= -room, (b, i, side)
                rest = np.maximum(p - q, 0)
                if rest.sum() > 4 * P_OFF:
                    p = rest
                elif draft is not None:
                    continue  # a difference that is all rounding: any token of it will do
            cum = np.cumsum(p)
            target, room = float(u_pick[b]) * cum[-1], 4 * P_OFF
            assert p[said] > 0 and cum[said] >= target - room and cum[said] - p[said] <= target + room, (b, i, said, cum[said], target)

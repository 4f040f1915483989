"""The attention operators in 64 bits, sequence by sequence, and how far the kernels' results may be from it.

The bounds count roundings: a result's own to its type (eps / 2 of its size), a weight's to BF16 (BF16 cache) or F16 (quantized), which carries to the
output times the weighted sum of the values' sizes, and a score's error in FP32, which a weight takes times itself."""
import numpy as np
import torch

BF16, F16 = 2.0 ** -8, 2.0 ** -11


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def values(cache, which, page, head, at):
    """Rows [n, D] of a KvCache as FP64, and the same with codes * scale and |min| apart ([n, D] each; a BF16 cache's has no min)."""
    page, at = torch.as_tensor(page, device=cache.device), torch.as_tensor(at, device=cache.device)
    codes = getattr(cache, which)[page, head, at]
    if cache.bits == 16:
        x = f64(codes)
        return x, np.abs(x), np.zeros_like(x)
    if cache.bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    sm = f64(getattr(cache, which + "_sm")[page, head, at])
    scaled = f64(codes) * np.repeat(sm[..., 0], cache.G, -1)
    least = np.repeat(sm[..., 1], cache.G, -1)
    return scaled + least, np.abs(scaled), np.abs(least)


def attend(q, cache, pages, q_start, kv_len, scale, softcap=0.0, window=0):
    """-> out, lse, and the bounds of both, [T, n_q, D] and [T, n_q]; rows of no sequence stay NaN."""
    q, D = f64(q), cache.D
    T, n_q = q.shape[0], q.shape[1] // D
    group = n_q // cache.n_kv
    pages, q_start, kv_len = pages.cpu().numpy(), q_start.cpu().numpy(), kv_len.cpu().numpy()
    out, lse = np.full((T, n_q, D), np.nan), np.full((T, n_q), np.nan)
    out_tol, lse_tol = np.zeros_like(out), np.zeros_like(lse)
    for b, length in enumerate(kv_len):
        n = q_start[b + 1] - q_start[b]
        j = np.arange(max(int(length), 0))
        for h in range(cache.n_kv):
            page, at = pages[b][j // cache.page].astype(np.int64), j % cache.page
            k, k_scaled, k_least = values(cache, "k", page, h, at)
            v, v_scaled, v_least = values(cache, "v", page, h, at)
            for i in range(n):
                p = length - n + i
                first, last = max(0, p - window + 1) if window else 0, max(0, p + 1)
                for hq in range(h * group, (h + 1) * group):
                    t = q_start[b] + i
                    x = q[t].reshape(n_q, D)[hq]
                    if last <= first:
                        out[t, hq], lse[t, hq] = 0.0, -np.inf
                        continue
                    with np.errstate(all="ignore"):
                        s = (k[first:last] @ x) * scale
                        # D / 16 tensor-core steps, each off by 2^-22 of what it has summed up, and the scale's and the logarithm's base's roundings
                        off = (D / 16 + 4) * 2.0 ** -22 * ((k_scaled + k_least)[first:last] @ np.abs(x)) * abs(scale)
                        if softcap:
                            s = softcap * np.tanh(s / softcap)
                            off = off + softcap * 2.0 ** -21
                        off = off + 2.0 ** -22 * np.abs(s)
                        top = s.max()
                        w = np.exp(s - top)
                        lse[t, hq] = top + np.log(w.sum())
                        w = w / w.sum()
                        out[t, hq] = w @ v[first:last]
                        of_weights = 2 * off.max() + 2.0 ** -20
                        kept = BF16 if cache.bits == 16 else F16
                        out_tol[t, hq] = BF16 * np.abs(out[t, hq]) + (kept + of_weights) * (w @ v_scaled[first:last]) + (of_weights + 2.0 ** -20) * (w @ v_least[first:last]) + 1e-30
                        lse_tol[t, hq] = off.max() + 2.0 ** -20 + 2.0 ** -22 * abs(lse[t, hq])
    return out, lse, out_tol, lse_tol


def norm_rotate(x, weight, eps, pos, inv_freq, interleaved):
    """x [T, heads, D] FP64 -> normed and rotated, and the size that FP32 arithmetic's error is relative to."""
    x = x.copy()
    D = x.shape[-1]
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * f64(weight)
    size = np.abs(x)
    if inv_freq is not None:
        angle = pos[:, None].astype(np.float64) * f64(inv_freq)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        half = inv_freq.numel()
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        xa, xb = x[..., a].copy(), x[..., b].copy()
        x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
        size[..., a] = size[..., b] = np.abs(xa) + np.abs(xb)
    return x, size

"""The attention sublayer of a decode or draft-verify step over a paged, quantized cache, composed from the library's launchers.

    quantized qkv projection  ->  norm, rotation, write into the cache  ->  attention of the new tokens over their pages
                              ->  quantized output projection

`AttnLayer` does for this sublayer what `layer.MoeLayer` does for the MoE one: it owns the order of the calls and the choice of their forms, the buffers
are shared by every layer of a stack.  Everything is enqueued on the current CUDA stream; nothing synchronizes except `check_errors`.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import kernels as K
from .kernels import Act, KvCache, QDeviceView


@dataclass
class AttnWeights:
    """qkv [(n_q + 2 n_kv) D, d] (the query heads' rows, the key heads', the value heads'), out [d, n_q D]; norm weights [D] FP32 (the factor itself) or
    None, inv_freq [rot / 2] FP32 or None."""

    qkv: QDeviceView
    out: QDeviceView
    q_norm: Optional[torch.Tensor] = None
    k_norm: Optional[torch.Tensor] = None
    inv_freq: Optional[torch.Tensor] = None
    interleaved: bool = False


@dataclass
class AttnBatch:
    """A step's rows: row t is position pos[t] of sequence seq[t] (seq[t] < 0: a padding row); sequence b has the rows q_start[b] .. q_start[b + 1] - 1 and kv_len[b] keys, its new
    tokens' included, on the pages of table row b.  All int32 on the device."""

    seq: torch.Tensor
    pos: torch.Tensor
    pages: torch.Tensor
    q_start: torch.Tensor
    kv_len: torch.Tensor
    max_q: int

    @classmethod
    def of(cls, kept: Sequence[int], new: Sequence[int], pages: torch.Tensor) -> "AttnBatch":
        """The batch in which sequence b, kept[b] tokens of which are in the cache, gets new[b] more."""
        def put(v):
            return torch.tensor(v, dtype=torch.int32, device=pages.device)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        return cls(put([b for b, n in enumerate(new) for _ in range(n)]), put([k + i for k, n in zip(kept, new) for i in range(n)]), pages, put(starts),
                   put([k + n for k, n in zip(kept, new)]), max(new))


class AttnBuffers:
    """Work buffers for steps of up to max_tokens rows with up to max_q of one sequence; shared by every layer of a stack."""

    def __init__(self, max_tokens: int, max_q: int, n_q: int, cache: KvCache):
        dev, D = cache.device, cache.D
        self.max_tokens, self.max_q = max_tokens, max_q
        self.qkv = torch.empty((max_tokens, (n_q + 2 * cache.n_kv) * D), dtype=torch.float32, device=dev)
        self.q = torch.empty((max_tokens, n_q * D), dtype=torch.bfloat16, device=dev)
        self.o = torch.empty((max_tokens, n_q * D), dtype=torch.bfloat16, device=dev)
        self.ws = torch.zeros(K.attn_decode_workspace_bytes(cache, n_q, max_q), dtype=torch.uint8, device=dev)
        self.err = torch.zeros(4, dtype=torch.int32, device=dev)
        self.nothing, self.none = (torch.tensor(v, dtype=torch.bfloat16, device=dev) for v in (0.0, float("nan")))


class AttnLayer:
    """One attention sublayer; its cache is its own, its buffers are the stack's."""

    wmma_min_tokens = 64  # from here on the projections' tensor-core form

    def __init__(self, weights: AttnWeights, n_q: int, cache: KvCache, buffers: AttnBuffers, eps: float = 1e-6, scale: Optional[float] = None,
                 softcap: float = 0.0, window: int = 0):
        D = cache.D
        if weights.qkv.N != (n_q + 2 * cache.n_kv) * D or weights.out.K != n_q * D:
            raise K.Error(1, f"AttnLayer: qkv of {weights.qkv.N} rows and out of {weights.out.K} columns do not fit {n_q} query and {cache.n_kv} key heads of {D}")
        if buffers.qkv.shape[1] != weights.qkv.N or buffers.q.shape[1] != weights.out.K or buffers.qkv.device != cache.device:
            raise K.Error(1, f"AttnLayer: buffers of {buffers.qkv.shape[1]} and {buffers.q.shape[1]} columns on {buffers.qkv.device}, the layer has {weights.qkv.N} and "
                             f"{weights.out.K} on {cache.device}")
        self.w, self.n_q, self.cache, self.buf = weights, n_q, cache, buffers
        self.eps, self.scale, self.softcap, self.window = eps, scale, softcap, window

    def _project(self, x: torch.Tensor, w: QDeviceView, y: torch.Tensor, T: int):
        out_act = Act.F32 if y.dtype == torch.float32 else Act.BF16
        (K.linear_qw_wmma if T >= self.wmma_min_tokens else K.linear_qw)(x, w, y, T, Act.BF16, out_act)

    def forward(self, x: torch.Tensor, batch: AttnBatch, y: torch.Tensor):
        """x [T, d] BF16 -> y [T, d] (BF16 or FP32); the batch's keys and values are in the cache afterwards.  A padding row (seq < 0, behind the last
        sequence's rows) becomes zeros, a row that no accepted range of q_start holds NaN."""
        T, b, w = x.shape[0], self.buf, self.w
        if T > b.max_tokens or batch.max_q > b.max_q or x.dtype != torch.bfloat16:
            raise K.Error(1, f"AttnLayer: {T} rows of {x.dtype} with up to {batch.max_q} of a sequence, the buffers hold {b.max_tokens} of BF16 with {b.max_q}")
        if (x.shape != (T, w.qkv.K) or y.shape != (T, w.out.N) or y.dtype not in (torch.bfloat16, torch.float32) or not (x.is_contiguous() and y.is_contiguous())
                or x.device != self.cache.device or y.device != self.cache.device):
            raise K.Error(1, f"AttnLayer: x {tuple(x.shape)} on {x.device} and y {tuple(y.shape)} of {y.dtype} on {y.device}, expected contiguous rows of {w.qkv.K} and of "
                             f"{w.out.N}, y BF16 or FP32, on {self.cache.device}")
        qkv, q, o = b.qkv[:T], b.q[:T], b.o[:T]
        self._project(x, w.qkv, qkv, T)  # FP32: the norm, the rotation and the cache's codes are made of unrounded sums
        K.attn_qkv_write(qkv, self.cache, batch.seq, batch.pos, batch.pages, q, b.err, q_norm=w.q_norm, k_norm=w.k_norm, eps=self.eps, inv_freq=w.inv_freq,
                         interleaved=w.interleaved)
        # the attention writes the rows of sequences; the buffer's others are an earlier layer's or step's
        torch.where((batch.seq < 0).unsqueeze(1).expand_as(o), b.nothing, b.none, out=o)
        K.attn_decode(q, self.cache, batch.pages, batch.q_start, batch.kv_len, batch.max_q, o, b.ws, b.err, scale=self.scale, softcap=self.softcap,
                      window=self.window)
        self._project(o, w.out, y, T)
        return y

    def check_errors(self, what: str = "attention layer"):
        """Blocking: the error words of write and attention, the tensor-core projections' status."""
        K.check_attn_error(self.buf.err, what)
        K.check_dense_status(what)

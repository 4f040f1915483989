"""The end of a decode or draft-verify step, composed from the library's launchers.

    last sublayer's output added to the residual stream, norm, 8-bit codes  ->  head's product over 8-bit floating-point weights
                              ->  drafted tokens verified against the logits, next token drawn

`VerifyHead` does for it what `attention.AttnLayer` does for the attention sublayer: it owns the order of the calls, the buffers are the caller's to share.
Everything is enqueued on the current CUDA stream; nothing synchronizes except `check_errors`.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import kernels as K
from .kernels import F8View


@dataclass
class HeadWeights:
    """out [V, d]; norm [d] FP32 (the factor itself) or None."""

    out: F8View
    norm: Optional[torch.Tensor] = None


class HeadBuffers:
    """Work buffers and results for steps of up to max_tokens rows of up to max_seqs sequences."""

    def __init__(self, max_tokens: int, max_seqs: int, d: int, V: int, device="cuda"):
        def empty(*shape, dtype):
            return torch.empty(shape, dtype=dtype, device=device)
        self.max_tokens, self.max_seqs, self.d, self.V = max_tokens, max_seqs, d, V
        self.total = empty(max_tokens, d, dtype=torch.bfloat16)
        self.codes = empty(max_tokens, d, dtype=torch.uint8).view(K.F8)
        self.scales = empty(max_tokens, -(-d // 128), dtype=torch.float32)
        self.logits = empty(max_tokens, V, dtype=torch.float32)
        self.ws = empty(K.verify_drafts_workspace_bytes(max_tokens, max_seqs, V), dtype=torch.uint8)
        self.said = empty(2, max_tokens, dtype=torch.int32)
        self.next_ids, self.logp = self.said[0], self.said[1].view(torch.float32)
        self.n_new = empty(max_seqs, dtype=torch.int32)
        self.err = torch.zeros(4, dtype=torch.int32, device=device)
        self.device = self.total.device


class VerifyHead:
    def __init__(self, weights: HeadWeights, buffers: HeadBuffers, eps: float = 1e-6):
        if weights.out.K != buffers.d or weights.out.N != buffers.V or weights.out.device != buffers.device:
            raise K.Error(1, f"VerifyHead: a weight of {weights.out.N} x {weights.out.K} on {weights.out.device}, the buffers are for {buffers.V} x {buffers.d} on {buffers.device}")
        self.w, self.buf, self.eps = weights, buffers, eps

    def forward(self, x: torch.Tensor, y: Optional[torch.Tensor], ids: torch.Tensor, q_start: torch.Tensor, u: torch.Tensor, u_pick: torch.Tensor,
                draft_logits: Optional[torch.Tensor] = None, temperature: Optional[torch.Tensor] = None):
        """x [T, d] BF16 the residual stream, y [T, d] the last sublayer's output or None; rows q_start[b] .. q_start[b + 1] - 1 are sequence b's, ids [T] the tokens fed there.
        -> next_ids [T], n_new [B], logp [T] of kernels.verify_drafts, views of the buffers; the logits stay in them too.  Rows of no sequence (padding), or of a refused range, have -1 and NaN."""
        T, b, B = x.shape[0], self.buf, u_pick.shape[0]
        if T > b.max_tokens or B > b.max_seqs or x.dtype != torch.bfloat16:
            raise K.Error(1, f"VerifyHead: {T} rows of {x.dtype} of {B} sequences, the buffers hold {b.max_tokens} of BF16 of {b.max_seqs}")
        codes, scales, logits = b.codes[:T], b.scales[:T], b.logits[:T]
        next_ids, n_new, logp = b.next_ids[:T], b.n_new[:B], b.logp[:T]
        # the verification writes the rows of sequences; the others would be an earlier step's.  As FP32 these bits are a NaN.  (3 us of a step of 98, 4096 x 131072, one row.)
        b.said.fill_(-1)
        K.add_norm(x, y, weight=self.w.norm, eps=self.eps, total=None if y is None else b.total[:T], codes=codes, scales=scales)
        K.linear_f8(codes, scales, self.w.out, logits)
        K.verify_drafts(logits, ids, q_start, u, u_pick, next_ids, n_new, b.ws, b.err, draft_logits=draft_logits, temperature=temperature, logp=logp)
        return next_ids, n_new, logp

    def check_errors(self, what: str = "head"):
        """Blocking: the error words of the verification, the product's status."""
        K.check_verify_error(self.buf.err, what)
        K.check_dense_status(what)

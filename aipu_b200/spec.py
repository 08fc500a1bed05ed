"""Speculative batched verify over the MoE decode stack (M = K + 1 token rows in one pass).

The reference's speculative system (src/glm_q4k_spec_system.v:30-61) verifies K draft tokens in one
pass of the model over the batch {cur_tok, d_1, .., d_K}: the pass yields the greedy tokens
m_1 .. m_{K+1} (row j's argmax), the drafts are accepted while d_j == m_j, the longest accepted
prefix p commits m_1 .. m_{p+1}, and the next pass starts from m_{p+1}. Because a row is accepted only
when its input is the token greedy decoding would have fed there, the committed stream equals greedy
decoding for any draft quality; the drafts only set how many tokens commit per weight stream.

This module runs that pass over the part of the model this library computes: token rows (an embedding
table lookup), the MoE branch of every layer in turn (one GPU: ops.moe_layer on the bit-exact decode
path; several GPUs: an ep.DecodeStream), then the LM head under the reference's bf16 dot contract
(ops.bf16_dot_gemv) and the argmax. The attention, norms and residuals between blocks -- and with them
the KV-cache write-back of the accepted rows and the AIPUDevice.step backend that drives a full model
(host/aipu_device.py:222-316) -- are outside this library's path; ``stack`` can be any callable that
maps [rows, H] bf16 hidden states to the next ones, so a caller that owns those parts plugs them in.
Every row is computed independently and bit-exactly, so a row's result does not depend on how many
rows share the pass (M = K + 1 rows give the same bits as K + 1 single-row passes).

A Request carries what one request asks of its tokens: its adapter on the LM head (ops.lora_add), and
penalties, biases and a mask on the logits before the argmax (ops.greedy_tokens). Row j of a pass is
then judged by the request's context with the drafts before it, so the committed stream equals greedy
decoding under the same controls (the adapter's bits are those of a single row in passes of up to 256).
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Callable, Dict, List, Optional, Sequence

import torch

from . import ops


def longest_accepted_prefix(drafts: Sequence[int], truth: Sequence[int]) -> int:
    """p = number of leading drafts equal to the verified tokens: d_j == m_j for j = 1..p
    (src/glm_q4k_spec_system.v:41-45). truth holds m_1 .. m_{K+1}."""
    p = 0
    while p < len(drafts) and p < len(truth) and int(drafts[p]) == int(truth[p]):
        p += 1
    return p


@dataclass
class SpecStats:
    """Bookkeeping over passes: passes run, drafts offered, drafts accepted, tokens committed."""
    passes: int = 0
    drafted: int = 0
    accepted: int = 0
    committed: int = 0
    accepted_per_pass: List[int] = field(default_factory=list)

    @property
    def acceptance_rate(self) -> float:
        return self.accepted / self.drafted if self.drafted else 0.0

    @property
    def tokens_per_pass(self) -> float:
        return self.committed / self.passes if self.passes else 0.0


def _allows(words: torch.Tensor, token: int) -> bool:
    """Whether packed mask words allow a token."""
    return 0 <= token < 32 * words.numel() and bool(int(words[token // 32]) >> (token % 32) & 1)


@dataclass
class Request:
    """One request: its context (the last token is the next pass's input), of which the first n_prompt tokens were
    given and the rest generated, and the controls of its tokens. mask(context) gives the packed mask words (int32
    [ceil(V / 32)], ops.pack_mask) of the token that follows a context, or None for no mask. It is asked about the context
    and about the context with drafts that its own masks allow, and its words are read on the host where drafts follow.
    adapter: its row in the verifier's head adapters, negative for none."""

    context: List[int]
    n_prompt: int = 0
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: Dict[int, float] = field(default_factory=dict)
    mask: Optional[Callable[[Sequence[int]], Optional[torch.Tensor]]] = None
    adapter: int = -1

    def controls(self, drafts: Sequence[int], device) -> ops.LogitControls:
        """Controls of the rows {context, context + d_1, ..}: one shared run of tokens, each row's context ends at its
        own input token."""
        if self.n_prompt < 0:
            raise ValueError("n_prompt must not be negative")
        M, n = len(drafts) + 1, len(self.context)
        tokens = list(self.context) + [int(d) for d in drafts]
        spans = [[0, min(self.n_prompt, n), n + j] for j in range(M)]
        c = ops.LogitControls(
            tokens=torch.tensor(tokens, dtype=torch.int32, device=device),
            spans=torch.tensor(spans, dtype=torch.int64, device=device),
            penalties=torch.tensor([[self.repetition, self.presence, self.frequency]] * M, dtype=torch.float32, device=device))
        if self.bias:
            b = len(self.bias)
            c.bias_begin = torch.arange(M + 1, device=device) * b
            c.bias_ids = torch.tensor(list(self.bias.keys()) * M, dtype=torch.int32, device=device)
            c.bias_vals = torch.tensor(list(self.bias.values()) * M, dtype=torch.float32, device=device)
        if self.mask is not None:
            rows, live = [-1] * M, []
            for j in range(M):
                words = self.mask(tokens[:n + j])
                if words is None:
                    continue
                rows[j] = len(live)
                live.append(words)
                if j < M - 1 and not _allows(words, tokens[n + j]):
                    break  # that draft is not accepted, so the rows behind it count for nothing
            if live:
                c.mask = torch.stack([w.to(device) for w in live]).contiguous()
                c.mask_rows = torch.tensor(rows, dtype=torch.int32, device=device)
        return c


class SpecVerifier:
    """Verify passes of K drafts over the MoE decode stack.

    emb: bf16 [V, H] token rows; lm_head: bf16 [V, H] (rows of the output projection);
    stack: list of ops.MoeLayerWeights (applied in turn on one GPU) or a callable [M, H] -> [M, H];
    head_adapters: low-rank adapters of the LM head (a [L, R, H], b [L, V, R]) that requests name.
    """

    def __init__(self, emb: torch.Tensor, lm_head: torch.Tensor, stack, ctx: Optional[ops.Context] = None,
                 head_adapters: Optional[ops.LoraAdapters] = None):
        if emb.dtype != torch.bfloat16 or lm_head.dtype != torch.bfloat16 or emb.dim() != 2 or lm_head.dim() != 2:
            raise ValueError("emb and lm_head must be bf16 [V, H]")
        if emb.shape[1] != lm_head.shape[1]:
            raise ValueError("emb and lm_head must have the same hidden size")
        self.emb = emb
        self.lm_head = lm_head
        self.ctx = ctx
        self.head_adapters = head_adapters
        if callable(stack):
            self._stack: Callable[[torch.Tensor], torch.Tensor] = stack
        else:
            layers = list(stack)

            def run(x):
                for W in layers:
                    x = ops.moe_layer(W, x, ctx=self.ctx)
                return x

            self._stack = run
        self.stats = SpecStats()

    def greedy_tokens(self, rows: Sequence[int], request: Optional[Request] = None) -> List[int]:
        """m_j = argmax of the LM head over the stack's output for token row j (lowest index on ties); for a request, of
        its adapted logits under its controls (-1 where its mask leaves nothing), whose context ends with the first row."""
        rows = list(rows)
        if request is not None:
            if not request.context or not rows or request.context[-1] != rows[0]:
                raise ValueError("a request's context must end with cur_tok")
            if request.adapter >= 0 and (self.head_adapters is None or request.adapter >= self.head_adapters.a.shape[0]):
                raise ValueError("the request names an adapter that the verifier does not have")
        if not all(0 <= t < self.emb.shape[0] for t in rows):
            raise ValueError("a token is outside the embedding")
        idx = torch.as_tensor(rows, dtype=torch.long, device=self.emb.device)
        h = self._stack(self.emb.index_select(0, idx).contiguous())
        logits = ops.bf16_dot_gemv(self.lm_head, h, ctx=self.ctx)
        if request is None:
            return [int(v) for v in logits.float().argmax(dim=1).cpu().tolist()]
        if request.adapter >= 0:
            ids = torch.full((len(rows),), request.adapter, dtype=torch.int32, device=h.device)
            logits = ops.lora_add(self.head_adapters, ids, h, logits, out=logits, ctx=self.ctx)
        return ops.greedy_tokens(logits, request.controls(rows[1:], h.device), ctx=self.ctx).cpu().tolist()

    def verify(self, cur_tok: int, drafts: Sequence[int], request: Optional[Request] = None):
        """One pass over {cur_tok, d_1..d_K}: returns (committed tokens m_1..m_{p+1}, p). A request's context must end
        with cur_tok; the committed tokens are added to it. Where its mask leaves no token, the committed ones end."""
        rows = [cur_tok] + list(drafts)
        truth = self.greedy_tokens(rows) if request is None else self.greedy_tokens(rows, request)
        p = longest_accepted_prefix(drafts, truth)
        committed = truth[:p + 1]
        if request is not None:
            if committed[-1] < 0:
                committed.pop()
            request.context.extend(committed)
        s = self.stats
        s.passes += 1
        s.drafted += len(drafts)
        s.accepted += p
        s.committed += len(committed)
        s.accepted_per_pass.append(p)
        return committed, p

    def generate(self, cur_tok: int, n_tokens: int, draft_fn: Callable[[int, int], Sequence[int]], k: int,
                 request: Optional[Request] = None):
        """Commit n_tokens tokens after cur_tok with K-draft verify passes; draft_fn(tok, k) proposes
        the next k tokens after tok. With a request, fewer where its mask leaves none."""
        out: List[int] = []
        tok = cur_tok
        while len(out) < n_tokens:
            committed, _ = self.verify(tok, list(draft_fn(tok, k))[:k], request)
            if not committed:
                break
            out.extend(committed)
            tok = committed[-1]
        if request is not None and len(out) > n_tokens:  # committed by the last pass, but not asked for
            del request.context[n_tokens - len(out):]
        return out[:n_tokens]

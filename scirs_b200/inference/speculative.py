"""Speculative decoding by rejection sampling (Leviathan et al., 2023).

A cheap draft model proposes `draft_steps` tokens; the target model scores
them in one pass; each draft token x is kept with probability
min(1, p_target(x) / p_draft(x)) (optionally floored by
`acceptance_threshold`), and at the first rejection a correction token is
drawn from the residual max(0, p_target - p_draft) renormalised. When all
are kept, a bonus token is drawn from the last target distribution. With a
zero floor the output distribution equals the target model's.

Distributions are torch tensors (any device); sampling uses a Marsaglia
xorshift64 generator so runs are reproducible from a seed.

:func:`verify_drafts` does the same for a batch in one launch, from
probabilities on the device and given random numbers
(scirs_b200/csrc/draft_verify.cu).

Reference parity: scirs2-neural/src/inference/speculative/types.rs:23-143
(SpeculativeConfig, SpeculativeResult) and rejection_sampling.rs:46-667
(Xorshift64, TokenDist, SpeculativeDecoder::rejection_sampling_step / decode).
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import NamedTuple

import torch

from .. import _ext
from ..ops import kernels as K


@dataclass
class SpeculativeConfig:
    draft_steps: int = 4
    temperature: float = 1.0
    top_p: float = 0.9
    max_tokens: int = 256
    acceptance_threshold: float = 0.0


@dataclass
class SpeculativeResult:
    accepted_tokens: list = field(default_factory=list)
    n_draft_tokens: int = 0
    n_accepted_tokens: int = 0
    n_steps: int = 0

    @property
    def acceptance_rate(self) -> float:
        return self.n_accepted_tokens / self.n_draft_tokens if self.n_draft_tokens else 0.0


class Xorshift64:
    """Marsaglia's 64-bit xorshift generator (shifts 13, 7, 17)."""

    MASK = (1 << 64) - 1

    def __init__(self, seed: int):
        self.state = (seed & self.MASK) or 0x9E3779B97F4A7C15

    def next_u64(self) -> int:
        x = self.state
        x ^= (x << 13) & self.MASK
        x ^= x >> 7
        x ^= (x << 17) & self.MASK
        self.state = x
        return x

    def next_f64(self) -> float:
        return (self.next_u64() >> 11) / float(1 << 53)


def _probs(logits: torch.Tensor, temperature: float) -> torch.Tensor:
    t = max(float(temperature), 1e-6)
    return torch.softmax(logits.double() / t, dim=-1)


def _top_p(p: torch.Tensor, top_p: float) -> torch.Tensor:
    if top_p >= 1.0:
        return p
    srt, idx = torch.sort(p, descending=True)
    keep = torch.cumsum(srt, 0) - srt < top_p  # smallest prefix reaching top_p
    keep[0] = True
    out = torch.zeros_like(p)
    out[idx[keep]] = srt[keep]
    return out / out.sum()


def _sample(p: torch.Tensor, u: float) -> int:
    c = torch.cumsum(p, 0)
    i = int(torch.searchsorted(c, torch.tensor([u * float(c[-1])], dtype=c.dtype, device=c.device)))
    return min(i, p.numel() - 1)


class TokenDist:
    def __init__(self, logits):
        self.logits = torch.as_tensor(logits, dtype=torch.float64)

    def softmax(self) -> torch.Tensor:
        return _probs(self.logits, 1.0)

    def sample(self, temperature: float, rng: Xorshift64) -> int:
        return _sample(_probs(self.logits, temperature), rng.next_f64())

    def sample_top_p(self, temperature: float, top_p: float, rng: Xorshift64) -> int:
        return _sample(_top_p(_probs(self.logits, temperature), top_p), rng.next_f64())

    def prob(self, token: int, temperature: float) -> float:
        p = _probs(self.logits, temperature)
        return float(p[token]) if 0 <= token < p.numel() else 0.0


class DraftVerification(NamedTuple):
    accepted: torch.Tensor  # int32 [B]: how many drafted tokens are kept
    tokens: torch.Tensor  # int64 [B, n + 1]: those, then the token that is drawn, then -1


def verify_drafts(target_probs: torch.Tensor, draft_probs: torch.Tensor | None, draft_tokens: torch.Tensor,
                  uniforms: torch.Tensor, draft_lens: torch.Tensor | None = None,
                  acceptance_threshold: float = 0.0) -> DraftVerification:
    """Keep or replace the drafted tokens of a batch.

    target_probs [B, n + 1, V] holds the target's probabilities at each drafted token's place and at
    the one behind the last, draft_probs [B, n, V] the draft's (None: the draft is certain of its
    tokens, as a greedy or n-gram draft is); fp32, bf16 or fp16 with contiguous rows, both of one type.
    draft_tokens int64 [B, n]; uniforms fp32 [B, n + 1] in [0, 1); draft_lens int32 [B] says how many
    drafts a sequence has (default: n).

    Draft x_i is kept while u_i q_i(x_i) < p_i(x_i), or u_i < acceptance_threshold (a draft of
    probability 0: while p_i(x_i) > 0; one outside the vocabulary: never). At the first place that is
    not kept one token is drawn from max(p - q, 0), or from p where that is zero everywhere, and from
    the last p where all are kept: the first token whose cumulative weight exceeds u_n times the
    total. The weights need not sum to 1; negative, infinite and NaN ones count as zero, and -1 is
    returned in the token's place where nothing is left. Products and sums are formed in 64 bits.
    V and n are below 2^30."""
    t, d = target_probs, draft_probs
    if t.dim() != 3 or t.shape[1] < 1 or t.shape[2] < 1:
        raise ValueError("target probabilities must be [B, n + 1, V]")
    B, n, V = t.shape[0], t.shape[1] - 1, t.shape[2]
    if V >= 1 << 30 or n >= 1 << 30:
        raise ValueError("fewer than 2^30 tokens and drafts")
    if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError("probabilities must be fp32, bf16 or fp16")
    if d is not None and (d.shape != (B, n, V) or d.dtype != t.dtype or d.device != t.device):
        raise ValueError(f"draft probabilities must be [{B}, {n}, {V}], typed and placed as the target's")
    if draft_tokens.shape != (B, n) or draft_tokens.dtype != torch.int64:
        raise ValueError(f"draft tokens must be int64 [{B}, {n}]")
    if uniforms.shape != (B, n + 1) or uniforms.dtype != torch.float32:
        raise ValueError(f"uniforms must be fp32 [{B}, {n + 1}]")
    if draft_lens is not None and (draft_lens.shape != (B,) or draft_lens.dtype != torch.int32):
        raise ValueError(f"draft lengths must be int32 [{B}]")
    if t.is_cuda:
        t = t if V == 1 or t.stride(2) == 1 else t.contiguous()
        if d is not None and V > 1 and d.stride(2) != 1:
            d = d.contiguous()
        out = _ext.kernels().draft_verify(t, d, draft_tokens.contiguous(), uniforms.contiguous(),
                                          None if draft_lens is None else draft_lens.contiguous(),
                                          float(acceptance_threshold))
        K._count(1 if B else 0)
        return DraftVerification(*out)
    accepted, tokens = torch.zeros(B, dtype=torch.int32), torch.full((B, n + 1), -1, dtype=torch.int64)
    for b in range(B):
        m, kept, q = n if draft_lens is None else min(max(int(draft_lens[b]), 0), n), 0, None
        while kept < m:
            x, u = int(draft_tokens[b, kept]), float(uniforms[b, kept])
            q = torch.zeros(V, dtype=torch.float64)
            if d is not None:
                q = d[b, kept].double()
            elif 0 <= x < V:
                q[x] = 1.0
            if not 0 <= x < V:
                break
            px, qx = float(t[b, kept, x]), float(q[x])
            if not (px > 0.0 if qx <= 0.0 else u < 1.0 and (u * qx < px or u < acceptance_threshold)):
                break
            tokens[b, kept] = x
            kept += 1
        accepted[b] = kept
        p = t[b, kept].double()
        for w in ([p - q, p] if kept < m else [p]):
            w = torch.where((w > 0) & torch.isfinite(w), w, torch.zeros_like(w))
            if float(w.sum()) > 0.0:
                c = torch.cumsum(w, 0)
                past = torch.nonzero((c > float(uniforms[b, n]) * c[-1]) & (w > 0))
                tokens[b, kept] = int(past[0] if len(past) else torch.nonzero(w > 0)[-1])
                break
    return DraftVerification(accepted, tokens)


class SpeculativeDecoder:
    @staticmethod
    def accept_or_reject(q: float, p: float, threshold: float, rng: Xorshift64) -> bool:
        if q <= 0.0:
            return p > 0.0
        ratio = max(min(1.0, p / q), threshold)
        return rng.next_f64() < ratio

    @staticmethod
    def rejection_sampling_step(draft_logits, target_logits, draft_tokens, config: SpeculativeConfig,
                                rng: Xorshift64 | None = None):
        """Returns (accepted prefix, correction-or-bonus token)."""
        n = min(len(draft_tokens), len(draft_logits), len(target_logits))
        if n == 0:
            return [], 0
        if rng is None:
            rng = Xorshift64(int(draft_tokens[0]) * 0x9E3779B97F4A7C15 + len(draft_logits[0]))
        out = []
        for i in range(n):
            x = int(draft_tokens[i])
            qd = _top_p(_probs(torch.as_tensor(draft_logits[i]), config.temperature), config.top_p)
            pt = _top_p(_probs(torch.as_tensor(target_logits[i]), config.temperature), config.top_p)
            if SpeculativeDecoder.accept_or_reject(float(qd[x]), float(pt[x]), config.acceptance_threshold, rng):
                out.append(x)
                continue
            resid = torch.clamp(pt - qd, min=0.0)
            if float(resid.sum()) <= 0.0:
                resid = pt
            return out, _sample(resid / resid.sum(), rng.next_f64())
        last = _top_p(_probs(torch.as_tensor(target_logits[n - 1]), config.temperature), config.top_p)
        return out, _sample(last, rng.next_f64())

    @staticmethod
    def decode(context, draft_fn, target_fn, config: SpeculativeConfig, seed: int = 1) -> SpeculativeResult:
        """draft_fn(ctx) -> [(token, logits)] (up to draft_steps);
        target_fn(ctx, draft_tokens) -> [logits] (one per draft position)."""
        rng = Xorshift64(seed)
        ctx = list(context)
        res = SpeculativeResult()
        while len(res.accepted_tokens) < config.max_tokens:
            drafts = draft_fn(ctx)[: config.draft_steps]
            if not drafts:
                break
            toks = [int(t) for t, _ in drafts]
            tl = target_fn(ctx, toks)
            acc, extra = SpeculativeDecoder.rejection_sampling_step([lg for _, lg in drafts], tl, toks, config, rng)
            res.n_steps += 1
            res.n_draft_tokens += len(toks)
            res.n_accepted_tokens += len(acc)
            new = acc + [extra]
            room = config.max_tokens - len(res.accepted_tokens)
            new = new[:room]
            res.accepted_tokens += new
            ctx += new
        return res

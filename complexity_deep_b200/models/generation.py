"""Autoregressive generation shared by the model classes: sampling rules and the decode loop."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from .. import ops


def sample_next(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 50, top_p: float = 0.9,
                do_sample: bool = True) -> torch.Tensor:
    """Next token [B, 1] from the logits [B, V] of the last position; same filtering rules as the
    reference (complexity_deep/models/modeling.py:256-296): temperature, then top-k, then nucleus
    top-p that always keeps the best token."""
    scores = logits.float() / temperature
    if top_k > 0:
        kth = torch.topk(scores, min(top_k, scores.shape[-1])).values[..., -1:]
        scores = scores.masked_fill(scores < kth, float("-inf"))
    if top_p < 1.0:
        ordered, order = torch.sort(scores, descending=True)
        mass = torch.cumsum(F.softmax(ordered, dim=-1), dim=-1)
        drop = mass > top_p
        drop = torch.cat([torch.zeros_like(drop[..., :1]), drop[..., :-1]], dim=-1)
        scores = scores.masked_fill(drop.scatter(1, order, drop), float("-inf"))
    if do_sample:
        return torch.multinomial(F.softmax(scores, dim=-1), num_samples=1)
    return scores.argmax(dim=-1, keepdim=True)


class GenerationMixin:
    """``generate`` for a model whose forward takes ``past_key_values`` / ``use_cache`` and returns
    the logits together with the cache of all tokens seen so far."""

    @torch.no_grad()
    def generate(
        self,
        input_ids: torch.Tensor,
        max_new_tokens: int = 100,
        temperature: float = 1.0,
        top_k: int = 50,
        top_p: float = 0.9,
        do_sample: bool = True,
        eos_token_id: Optional[int] = None,
        min_p: float = 0.0,
        uniforms: Optional[torch.Tensor] = None,
    ) -> torch.Tensor:
        """Autoregressive sampling with a cache; stops when every sequence of the batch has just
        produced the end token (the config's, unless given here; none if neither has one).
        `uniforms` (fp32 [max_new_tokens, B], in [0, 1)): tokens are drawn from these numbers by
        ``ops.sample_tokens`` instead of torch's generator; min_p asks for that too and draws
        its own numbers unless they are given."""
        if min_p > 0.0 and uniforms is None:
            uniforms = torch.rand(max_new_tokens, input_ids.shape[0], device=input_ids.device)
        eos = getattr(self.config, "eos_token_id", None) if eos_token_id is None else eos_token_id
        cache = None
        for i in range(max_new_tokens):
            step_ids = input_ids if cache is None else input_ids[:, -1:]
            out = self.forward(step_ids, past_key_values=cache, use_cache=True)
            cache = out.past_key_values
            if uniforms is None:
                nxt = sample_next(out.logits[:, -1, :], temperature, top_k, top_p, do_sample)
            else:
                nxt = ops.sample_tokens(out.logits[:, -1, :], uniforms[i], temperature if do_sample else 0.0, top_k, top_p,
                                        min_p)[0][:, None]
            input_ids = torch.cat([input_ids, nxt], dim=-1)
            if eos is not None and bool((nxt == eos).all()):
                break
        return input_ids

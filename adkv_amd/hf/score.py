"""Log probabilities of texts under a model (what the reference's evaluation asks for, tools/lm_eval_adkv.py), for both of its Llama flavours."""
from __future__ import annotations

import torch

from ..kernel.gemv import TokenLogprobs, token_logprobs
from .packed import packs


class Scores:
    """``score`` for a causal language model with ``model``, ``lm_head`` and ``config``."""

    @torch.no_grad()
    def score(self, sequences, *, top: int = 0, rows: int = 4096, prefill_full_precision: bool | None = None) -> list[TokenLogprobs]:
        """Of every sequence (token ids ``[n]``, ``n >= 1``, of any lengths) the log probability of each of its tokens but the first, given those in
        front of it: ``n - 1`` of them, with the distributions' entropy and their ``top`` likeliest tokens.  ``rows`` of logits are made at a time.

        Prompts are attended with as they are, unless the evaluation flavour is given ``prefill_full_precision=False`` (its default is
        the model's: config.prefill_full_precision, else true): then every token looks at what the cache has kept of those in front of it, and scores show what the
        quantisation costs.  Texts are one batch padded behind them, where nothing looks at it; where ``config.adkv_prompt`` has its own attention run
        and no cache is read they are packed into one row axis without padding."""
        evaluates = getattr(self, "scores_with_cache", False)
        if prefill_full_precision is None:
            prefill_full_precision = not evaluates or getattr(self.config, "prefill_full_precision", True)
        if not (prefill_full_precision or evaluates):
            raise ValueError("only the evaluation flavour's prompts look at quantised tokens")
        dev = self.lm_head.weight.device
        ids = [torch.as_tensor(s, dtype=torch.int64, device=dev).reshape(-1) for s in sequences]
        if not ids:
            return []
        lengths = [s.shape[0] for s in ids]
        if min(lengths) < 1:
            raise ValueError("a sequence needs one token at least")
        if prefill_full_precision and packs(self.model, {}):
            ends = torch.tensor([0, *lengths], device="cpu").cumsum(0)
            at = torch.cat([torch.arange(n) for n in lengths]).to(dev)[None]
            total = int(ends[-1])
            hidden = self.model(input_ids=torch.cat(ids)[None], position_ids=at, cu_seq_lens_q=ends.to(dev, torch.int32), use_cache=False).last_hidden_state[0]
            keep = torch.ones(total, dtype=torch.bool)
            keep[ends[1:] - 1] = False
            hidden = hidden[keep.to(dev)]
        else:
            batch = torch.nn.utils.rnn.pad_sequence(ids, batch_first=True)
            extra = {} if prefill_full_precision else {"prefill_full_precision": False}
            hidden = self.model(input_ids=batch, use_cache=not prefill_full_precision, **extra).last_hidden_state
            hidden = torch.cat([h[:n - 1] for h, n in zip(hidden, lengths)])
        given = torch.cat([s[1:] for s in ids])
        parts = [token_logprobs(self.lm_head(h), t, top=top) for h, t in zip(hidden.split(rows), given.split(rows))]
        whole = [None if p[0] is None else torch.cat(p) for p in zip(*parts)]
        each = zip(*([None] * len(ids) if w is None else w.split([n - 1 for n in lengths]) for w in whole))
        return [TokenLogprobs(*e) for e in each]

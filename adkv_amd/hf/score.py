"""Log probabilities of texts under a model (what the reference's evaluation asks for, tools/lm_eval_adkv.py), for both of its Llama flavours."""
from __future__ import annotations

import torch

from ..kernel.gemv import TokenLogprobs, token_logprobs
from .packed import packs


class Scores:
    """``score`` for a causal language model with ``model``, ``lm_head`` and ``config``."""

    @torch.no_grad()
    def score(self, sequences, *, top: int = 0, rows: int = 4096, tokens: int = 16384, prefill_full_precision: bool | None = None) -> list[TokenLogprobs]:
        """Of every sequence (token ids ``[n]``, ``n >= 1``, of any lengths) the log probability of each of its tokens but the first, given those in
        front of it: ``n - 1`` of them, with the distributions' entropy and their ``top`` likeliest tokens.  The model is run with up to ``tokens`` at a time, padding
        among them (with one sequence, if that is longer), the longest sequences first; ``rows`` of logits are made at a time.

        Prompts are attended with as they are, unless the evaluation flavour is given ``prefill_full_precision=False`` (its default is
        the model's: config.prefill_full_precision, else true): then every token looks at what the cache has kept of those in front of it, and scores show what the
        quantisation costs.  Texts are batches padded behind them, where nothing looks at it; where ``config.adkv_prompt`` has its own attention run
        and no cache is read they are packed into one row axis without padding."""
        evaluates = getattr(self, "scores_with_cache", False)
        if prefill_full_precision is None:
            prefill_full_precision = not evaluates or getattr(self.config, "prefill_full_precision", True)
        if not (prefill_full_precision or evaluates):
            raise ValueError("only the evaluation flavour's prompts look at quantised tokens")
        dev = self.lm_head.weight.device
        ids = [torch.as_tensor(s, dtype=torch.int64, device=dev).reshape(-1) for s in sequences]
        if any(s.shape[0] < 1 for s in ids):
            raise ValueError("a sequence needs one token at least")
        packed = prefill_full_precision and packs(self.model, {})
        found = [None] * len(ids)
        for group in _groups([s.shape[0] for s in ids], tokens, packed):
            of = [ids[i] for i in group]
            hidden = self._packed_rows(of) if packed else self._padded_rows(of, prefill_full_precision)
            given = torch.cat([s[1:] for s in of])
            parts = [token_logprobs(self.lm_head(h), t, top=top) for h, t in zip(hidden.split(rows), given.split(rows))]
            whole = [None if p[0] is None else torch.cat(p) for p in zip(*parts)]
            each = zip(*([None] * len(of) if w is None else w.split([s.shape[0] - 1 for s in of]) for w in whole))
            for i, e in zip(group, each):
                found[i] = TokenLogprobs(*e)
        return found

    def _packed_rows(self, ids) -> torch.Tensor:
        """What the model makes of every sequence's tokens but the last, ``[rows, C]``, all of them in one row axis."""
        lengths = [s.shape[0] for s in ids]
        ends = torch.tensor([0, *lengths], device="cpu").cumsum(0)
        at = torch.cat([torch.arange(n) for n in lengths])[None]
        keep = torch.ones(int(ends[-1]), dtype=torch.bool)
        keep[ends[1:] - 1] = False
        dev = ids[0].device
        hidden = self.model(input_ids=torch.cat(ids)[None], position_ids=at.to(dev), cu_seq_lens_q=ends.to(dev, torch.int32), use_cache=False).last_hidden_state[0]
        return hidden[keep.to(dev)]

    def _padded_rows(self, ids, prefill_full_precision: bool) -> torch.Tensor:
        """The same from a padded batch."""
        extra = {} if prefill_full_precision else {"prefill_full_precision": False}
        batch = torch.nn.utils.rnn.pad_sequence(ids, batch_first=True)
        hidden = self.model(input_ids=batch, use_cache=not prefill_full_precision, **extra).last_hidden_state
        return torch.cat([h[:s.shape[0] - 1] for h, s in zip(hidden, ids)])


def _groups(lengths, tokens: int, packed: bool):
    """Which sequences are run together, the longest first."""
    group, used = [], 0
    for i in sorted(range(len(lengths)), key=lambda i: -lengths[i]):
        size = lengths[i] if packed or not group else lengths[group[0]]
        if group and used + size > tokens:
            yield group
            group, used, size = [], 0, lengths[i]
        group.append(i)
        used += size
    if group:
        yield group

"""Where config.adkv_prompt has the framework's own attention run over prompts, and sequences that share a row axis without a mask between them."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


def takes_prompts(attn, dtype, device, kwargs) -> bool:
    """Whether ``prompt_ctx`` attends for ``attn`` itself, with rows of this type on this device and where no derivative is wanted; without
    config.adkv_prompt, on the host, for other types and head sizes, where dropout or the weights are wanted, where later tokens are looked at
    or scores have a bias of their own, transformers' attention does."""
    return bool(getattr(attn.config, "adkv_prompt", False) and device.type == "cuda" and dtype in (torch.float16, torch.bfloat16)
                and attn.head_dim % 8 == 0 and attn.head_dim <= 256 and not (attn.training and attn.attention_dropout > 0)
                and not kwargs.get("output_attentions") and not getattr(attn.config, "output_attentions", False)
                and attn.is_causal and getattr(attn.config, "is_causal", True) and kwargs.get("is_causal") in (None, True) and kwargs.get("position_bias") is None)


def refuse_cache(attn, cached: bool, kwargs) -> None:
    """Ahead of anything that is written to a cache: it keeps sequences of one length, each a row of its batch."""
    if cached and kwargs.get("cu_seq_lens_q") is not None and getattr(attn.config, "adkv_prompt", False):
        raise ValueError("packed sequences have no cache: pass use_cache=False")


def derivatives_wanted(*tensors) -> bool:
    """Of what is computed from them: backward, forward, or a transform's."""
    backward, dual = torch.is_grad_enabled(), getattr(forward_ad, "_current_level", 0) >= 0      # without a level no tensor has a tangent
    for t in tensors:
        if isinstance(t, torch.Tensor) and ((backward and t.requires_grad) or torch._C._functorch.is_functorch_wrapped_tensor(t)
                                            or (dual and forward_ad.unpack_dual(t).tangent is not None)):
            return True
    return False


def packs(model, kwargs) -> bool:
    """Whether ``model`` keeps sequences that share a row axis apart by ``prompt_attention``, without a mask."""
    attn = model.layers[0].self_attn
    w = attn.q_proj.weight
    return not torch.is_grad_enabled() and takes_prompts(attn, w.dtype, w.device, kwargs) and not torch.is_autocast_enabled(w.device.type)


def says_nothing(mask) -> bool:
    """The mask of ``packed_mask``: of four axes, which transformers hands on as it is, and without an entry."""
    return isinstance(mask, torch.Tensor) and mask.dim() == 4 and mask.numel() == 0


def packed_mask(model, tokens: torch.Tensor, attention_mask, kwargs):
    """The mask for a model's ``tokens [1, T, ..]`` where config.adkv_prompt has each of the sequences that ``cu_seq_lens_q`` bounds look at itself only: one
    that says nothing where ``prompt_attention`` sees to that, else what transformers' own attention needs for it, ``[1, 1, T, T]``."""
    bounds = kwargs.get("cu_seq_lens_q")
    if bounds is None or not getattr(model.config, "adkv_prompt", False) or (attention_mask is not None and getattr(attention_mask, "ndim", 4) != 2):
        return attention_mask
    if attention_mask is not None:
        raise ValueError("packed sequences have no padding: pass no attention_mask")
    if tokens.shape[0] != 1:
        raise ValueError("packed sequences share one row axis: a batch of one")
    how = model.config._attn_implementation
    if packs(model, kwargs):
        return torch.empty(1, 1, 0, 0, dtype=torch.bool, device=tokens.device)
    if how not in ("sdpa", "eager") or not getattr(model.config, "is_causal", True):
        return None                    # transformers' others know the bounds, or make masks from the positions
    at = torch.arange(tokens.shape[1], device=tokens.device)
    of = torch.searchsorted(bounds.to(at), at, right=True)
    see = ((of[:, None] == of) & (at[:, None] >= at))[None, None]
    dtype = model.embed_tokens.weight.dtype
    return see if how == "sdpa" else torch.zeros(see.shape, dtype=dtype, device=see.device).masked_fill_(~see, torch.finfo(dtype).min)

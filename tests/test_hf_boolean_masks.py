"""Masks as the attention module gets them from a model with attn_implementation="sdpa", which is the default: boolean, true where a token
is looked at.  A decode step takes them like the additive ones of eager attention."""
import math

import pytest
import torch

from adkv_amd import synth
from adkv_amd.hf import cache as M
from adkv_amd.hf.cache import KVCacheLayer_ADKV
from adkv_amd.kernel import gemv

D = 128


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_a_step_hands_an_additive_mask_on(monkeypatch, dtype):
    """Without kernels: what decode_step is given."""
    got = {}

    def step(q, kc, vc, kn, vn, kp, vp, T, scaling, mask, **kw):
        got["mask"] = mask
        return torch.zeros(q.shape[0], q.shape[1], D, dtype=q.dtype), None
    monkeypatch.setattr(M, "decode_step", step)
    monkeypatch.setattr(M, "decode_step_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(M, "_workspace", lambda *a: None)
    c = KVCacheLayer_ADKV()
    c.reserve(2, 2, D, 40, "cpu")
    c.commit(9)
    par = [t.reshape(-1) for t in synth.make_params(2, D).astuple()] * 2
    rows = [torch.zeros(2, 2, 1, D, dtype=dtype) for _ in range(3)]
    seen = torch.ones(2, 1, 1, 10, dtype=torch.bool)
    seen[0, :, :, :4] = False
    c.decode(*rows, *par, attention_mask=seen)
    m = got["mask"]
    assert m.is_floating_point() and m.shape == seen.shape
    assert bool((m[seen] == 0).all()) and bool((m[~seen] <= -6e4).all()) and bool(torch.isfinite(m).all())
    c.decode(*rows, *par, attention_mask=None)
    assert got["mask"] is None


@pytest.mark.gpu
@pytest.mark.parametrize("G,dtype,T", [(1, torch.float16, 70), (4, torch.bfloat16, 300), (1, torch.float32, 33)])
def test_a_step_with_a_boolean_mask(gpu, G, dtype, T):
    H, B = 2, 3
    kg, vg = ([t.reshape(-1) for t in synth.make_params(H, D, seed=s).to(gpu).astuple()] for s in (3, 4))
    k, v = (synth.make_k(B, H, T + 1, D, seed=s, dtype=torch.float16).to(dtype).to(gpu) for s in (1, 2))
    q = torch.randn(B, H * G, 1, D, generator=torch.Generator().manual_seed(5)).to(dtype).to(gpu)
    seen = torch.ones(B, 1, 1, T + 1, dtype=torch.bool)
    seen[1, :, :, :T // 2] = False
    seen[2, :, :, 3] = False
    like = dtype if dtype != torch.float32 else torch.float32
    additive = torch.zeros(seen.shape, dtype=like).masked_fill(~seen, torch.finfo(like).min)
    outs = []
    for mask in (seen, additive):
        c = KVCacheLayer_ADKV()
        c.prefill(k[:, :, :T], v[:, :, :T], *kg, *vg)
        outs.append(c.decode(q, k[:, :, T:], v[:, :, T:], *kg, *vg, attention_mask=mask.to(gpu), scaling=D ** -0.5))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert bool((outs[0][1][1, :, :T // 2] == 0).all()) and bool((outs[0][1][2, :, 3] == 0).all())     # the weights of hidden tokens


@pytest.mark.gpu
@pytest.mark.parametrize("at_once", [False, True])
def test_a_padded_batch_with_either_attention(gpu, at_once):
    """The same model with eager attention and with sdpa, a padded batch: a prompt, a follow-up, steps.  The tolerance is the follow-up
    test's; hidden tokens that were looked at would be off by far more.  One layer: a padded token's row looks at nothing, which eager attention
    makes a mean and sdpa zero, and in a second layer the codes' stream would run through what came of it."""
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from adkv_amd.hf.llama_adkv import ADKVConfig, LlamaForCausalLM_ADKV
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(1, 128, (2, 40), generator=g).to(gpu)
    seen = torch.ones(2, 40, dtype=torch.long, device=gpu)
    seen[0, :9] = 0
    pos = (seen.cumsum(-1) - 1).clamp_(0)
    results = []
    for attention in ("eager", "sdpa"):
        cfg = LlamaConfig(vocab_size=128, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2,
                          head_dim=D, max_position_embeddings=512, attn_implementation=attention, adkv_extend=at_once)
        torch.manual_seed(0)
        model = LlamaForCausalLM_ADKV(cfg).to(gpu).to(torch.float16).eval()
        full = lambda v: torch.full((2 * D,), v)
        mk = lambda: ADKVConfig(zp_init=full(0.0), scale_init=full(0.05), alpha=full(0.95), beta=full(0.05), quant_target=full(3.5))
        model.load_adkv_config([(mk(), mk())])
        with torch.no_grad():
            out = model(ids[:, :20], attention_mask=seen[:, :20], position_ids=pos[:, :20], use_cache=True)
            logits = [out.logits]
            for a, b in ((20, 28), (28, 29), (29, 30), (30, 40)):
                logits.append(model(ids[:, a:b], attention_mask=seen[:, :b], position_ids=pos[:, a:b], past_key_values=out.past_key_values,
                                    use_cache=True).logits)
        results.append(torch.cat(logits, 1).float()[seen.bool()])
    assert torch.allclose(*results, atol=2e-2, rtol=2e-2)


def test_a_boolean_mask_is_refused_where_masks_are_added():
    from test_extend import _cpu_args
    with pytest.raises(RuntimeError, match="additive"):
        gemv.extend(**{**_cpu_args(), "mask": torch.ones(2, 1, 2, 18, dtype=torch.bool)})

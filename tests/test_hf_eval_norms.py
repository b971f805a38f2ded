"""config.adkv_qk_norm in the evaluation model: the norms of the model that is evaluated."""
import pytest
import torch

pytest.importorskip("transformers")

D = 128


def _models(device="cpu", dtype=torch.float32, norm=True, kv_heads=2):
    from transformers import LlamaConfig
    from adkv_amd.hf import llama_adkv, llama_adkv_eval
    cfg = LlamaConfig(vocab_size=128, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=kv_heads, head_dim=D, max_position_embeddings=256, attn_implementation="eager", adkv_qk_norm=norm)
    torch.manual_seed(0)
    model = llama_adkv.LlamaForCausalLM_ADKV(cfg)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith(("q_norm.weight", "k_norm.weight")):
                p.add_(0.3 * torch.randn(p.shape, generator=torch.Generator().manual_seed(1)))
    other = llama_adkv_eval.LlamaForCausalLM_ADKV(cfg)
    missing = other.load_state_dict(model.state_dict(), strict=True)
    assert not missing.missing_keys and not missing.unexpected_keys
    full = lambda v: torch.full((kv_heads * D,), v)
    mk = lambda: llama_adkv.ADKVConfig(zp_init=full(0.0), scale_init=full(0.05), alpha=full(0.95), beta=full(0.05), quant_target=full(3.5))
    for m in (model, other):
        m.load_adkv_config([(mk(), mk()) for _ in range(2)])
    return [m.to(device).to(dtype).eval() for m in (model, other)]


@pytest.mark.parametrize("norm", [True, False])
def test_the_same_logits_without_a_cache(norm):
    """Nothing is quantised where nothing is cached: the two models are one."""
    model, other = _models(norm=norm)
    ids = torch.randint(1, 128, (2, 9), generator=torch.Generator().manual_seed(3))
    with torch.no_grad():
        a, b = (m(ids, use_cache=False).logits for m in (model, other))
    assert torch.equal(a, b)
    assert hasattr(other.model.layers[0].self_attn, "q_norm") == norm


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_the_same_first_logits_on_the_device(gpu, dtype):
    """The prompt's own rows are attended with unquantised in both; the norms round once in either."""
    model, other = _models(gpu, dtype)
    ids = torch.randint(1, 128, (2, 40), generator=torch.Generator().manual_seed(3)).to(gpu)
    with torch.no_grad():
        a, b = (m(ids, use_cache=True).logits.float() for m in (model, other))
    assert torch.equal(a, b)
    with torch.no_grad():
        step = other(ids[:, :1], past_key_values=other(ids, use_cache=True).past_key_values, use_cache=True).logits
    assert bool(torch.isfinite(step).all())

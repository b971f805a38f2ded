"""What the head norms cost a model that has none."""
import pytest
import torch

pytest.importorskip("transformers")


@pytest.mark.parametrize("flavour", ["llama_adkv", "llama_adkv_eval"])
def test_absent_norms_are_not_looked_for_by_exception(monkeypatch, flavour):
    """A module's attribute that is not there is found out by an exception, a microsecond per layer and token."""
    import importlib

    from transformers import LlamaConfig
    M = importlib.import_module(f"adkv_amd.hf.{flavour}")
    cfg = LlamaConfig(vocab_size=64, hidden_size=256, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2,
                      head_dim=128, attn_implementation="eager")
    model = M.LlamaForCausalLM_ADKV(cfg).eval()
    asked, real = [], M.LlamaAttention_ADKV.__getattr__

    def watch(self, name):
        asked.append(name)
        return real(self, name)
    monkeypatch.setattr(M.LlamaAttention_ADKV, "__getattr__", watch, raising=False)
    with torch.no_grad():
        model(torch.arange(1, 5)[None], use_cache=False)
    assert "q_proj" in asked and "q_norm" not in asked

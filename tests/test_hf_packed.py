"""Sequences that share a row axis (cu_seq_lens_q, score()) under config.adkv_prompt, where the framework's attention runs and where transformers' does: each of
them is what it is by itself."""
import pytest
import torch

pytest.importorskip("transformers")

from test_hf_prompt import both, ids_of, make, config, near  # noqa: E402

from adkv_amd.hf import llama_adkv, llama_adkv_eval  # noqa: E402
from adkv_amd.hf.packed import packed_mask, says_nothing, takes_prompts  # noqa: E402

ENDS = [0, 5, 6, 17]
FLAVOURS = {"deployment": llama_adkv, "evaluation": llama_adkv_eval}


def packed(device):
    at = torch.cat([torch.arange(b - a) for a, b in zip(ENDS, ENDS[1:])])[None]
    return dict(position_ids=at.to(device), cu_seq_lens_q=torch.tensor(ENDS, dtype=torch.int32, device=device), use_cache=False)


@pytest.mark.parametrize("positions", [True, False])
@pytest.mark.parametrize("implementation", ["sdpa", "eager"])
@pytest.mark.parametrize("flavour", FLAVOURS)
def test_packed_sequences_on_the_host(flavour, implementation, positions):
    """Transformers' attention runs, in 64 bits: off by some hundred roundings of 2^-53 of numbers of size one."""
    m = make(FLAVOURS[flavour].LlamaForCausalLM_ADKV, config(adkv_prompt=True, attn_implementation=implementation), torch.float64, "cpu")
    ids, how = ids_of(1, ENDS[-1]), packed("cpu")
    if not positions:
        del how["position_ids"]      # rotations are relative
    with torch.no_grad():
        got = m(ids, **how).logits[0]
        for a, b in zip(ENDS, ENDS[1:]):
            # rotary angles are of 32 bits, 2^-24 of 17 radians, and the eager attention's softmax is
            off = 1e-12 if positions and implementation == "sdpa" else 17 * 2.0 ** -18
            assert (got[a:b] - m(ids[:, a:b], use_cache=False).logits[0]).abs().max() <= off


def test_refused_with_packed_sequences():
    m = make(llama_adkv.LlamaForCausalLM_ADKV, config(adkv_prompt=True), torch.float32, "cpu")
    with pytest.raises(ValueError, match="no padding"):
        m(ids_of(1, ENDS[-1]), attention_mask=torch.ones(1, ENDS[-1], dtype=torch.int64), **packed("cpu"))
    with pytest.raises(ValueError, match="batch of one"):
        m(ids_of(2, ENDS[-1]), **packed("cpu"))
    theirs = object()                  # a mask that is no tensor goes on
    assert packed_mask(m.model, ids_of(1, 17), theirs, packed("cpu")) is theirs
    # a mask that says nothing has nothing to say where the kernel does not run
    assert says_nothing(torch.empty(1, 1, 0, 0, dtype=torch.bool)) and not says_nothing(torch.ones(1, 1, 1, 17)) and not says_nothing(None)
    with pytest.raises(ValueError, match="apart"):
        m(ids_of(1, ENDS[-1]), attention_mask=torch.empty(1, 1, 0, 0, dtype=torch.bool), **packed("cpu"))


@pytest.mark.parametrize("flavour", FLAVOURS)
def test_a_cache_is_refused_before_it_is_written(flavour, monkeypatch):
    """A new one, and one that holds a prompt already (one more token, and several)."""
    module = FLAVOURS[flavour]
    m = make(module.LlamaForCausalLM_ADKV, config(adkv_prompt=True), torch.float32, "cpu")
    for name in ("update", "prefill", "decode", "extend"):
        monkeypatch.setattr(module.KVCacheLayer_ADKV, name, lambda *a, **k: pytest.fail("written"), raising=False)
    for length, n in ((0, ENDS[-1]), (30, ENDS[-1]), (30, 1)):
        cache = module.KVCache_ADKV(2)
        for layer in cache:
            layer._quant_len = layer._recent_len = length
        with torch.no_grad(), pytest.raises(ValueError, match="no cache"):
            m(ids_of(1, n), past_key_values=cache, use_cache=True, cu_seq_lens_q=torch.tensor([0, n], dtype=torch.int32))


def test_what_the_kernel_takes():
    at = lambda **how: make(llama_adkv.LlamaForCausalLM_ADKV, config(adkv_prompt=True, **how), torch.float32, "cpu").model.layers[0].self_attn
    dev, attn = torch.device("cuda"), at()
    assert takes_prompts(attn, torch.float16, dev, {}) and takes_prompts(attn, torch.bfloat16, dev, {})
    assert not takes_prompts(attn, torch.float32, dev, {}) and not takes_prompts(attn, torch.float16, torch.device("cpu"), {})
    assert not takes_prompts(attn, torch.float16, dev, dict(output_attentions=True)) and not takes_prompts(at(head_dim=36), torch.float16, dev, {})
    assert not takes_prompts(at(head_dim=264), torch.float16, dev, {}) and not takes_prompts(at(output_attentions=True, attn_implementation="eager"), torch.float16, dev, {})
    assert takes_prompts(attn, torch.float16, dev, dict(is_causal=True, position_bias=None)) and not takes_prompts(attn, torch.float16, dev, dict(is_causal=False))
    assert not takes_prompts(attn, torch.float16, dev, dict(position_bias=torch.zeros(1))) and not takes_prompts(at(is_causal=False), torch.float16, dev, {})
    attn.is_causal = False
    assert not takes_prompts(attn, torch.float16, dev, {})
    attn = at(attention_dropout=0.1)
    assert takes_prompts(attn, torch.float16, dev, {}) and not takes_prompts(attn.train(), torch.float16, dev, {})


@pytest.mark.gpu
@pytest.mark.parametrize("flavour", FLAVOURS)
@pytest.mark.parametrize("why", ["type", "head size", "weights", "dropout"])
def test_scores_by_transformers_attention(gpu, flavour, why):
    """(Dropout of 1e-9 drops nothing.)"""
    how = {"type": {}, "head size": dict(head_dim=36), "weights": dict(output_attentions=True, attn_implementation="eager"),
           "dropout": dict(attention_dropout=1e-9, attn_implementation="eager")}[why]
    if flavour == "evaluation" and why == "head size":
        how = dict(head_dim=264)
    mine, other, host = both(flavour, torch.float32 if why == "type" else torch.float16, gpu, **how)
    if why == "dropout":
        mine.train(), other.train()
    texts = [ids_of(1, n, n)[0] for n in (40, 1, 7, 33)]
    got, ref = mine.score(texts), other.score(texts)
    for text, g, r in zip(texts, got, ref):
        if len(text) > 1:
            with torch.no_grad():
                log = torch.log_softmax(host(text[None], use_cache=False).logits[0, :-1], -1)
            kind = torch.float32 if why == "type" else torch.float16
            near(g.logprobs.to(kind), r.logprobs.to(kind), log.gather(1, text[1:, None])[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("flavour", FLAVOURS)
@pytest.mark.parametrize("why", ["", "type", "gradient", "autocast", "mask"])
def test_packed_sequences(gpu, flavour, why, monkeypatch):
    mine, other, host = both(flavour, torch.float32 if why in ("type", "autocast") else torch.float16, gpu)
    ids, how = ids_of(1, ENDS[-1]), packed(gpu)
    calls = []
    real = llama_adkv.prompt_attention
    monkeypatch.setattr(llama_adkv, "prompt_attention", lambda *a, **k: calls.append(k) or real(*a, **k))
    if why == "mask":           # which goes on: the first two are one sequence then
        of = torch.tensor([0] * ENDS[2] + [1] * (ENDS[3] - ENDS[2]))
        how["attention_mask"] = ((of[:, None] == of) & torch.ones(17, 17).tril().bool())[None, None].to(gpu)
    with torch.set_grad_enabled(why == "gradient"), torch.autocast("cuda", torch.float16, enabled=why == "autocast"):
        got = mine(ids.to(gpu), **how).logits[0].detach()
        ends = [0, ENDS[2], ENDS[3]] if why == "mask" else ENDS
        if why == "mask":
            how["position_ids"][:, :ENDS[2]] = torch.arange(ENDS[2])
            got = mine(ids.to(gpu), **how).logits[0]
        ref = torch.cat([other(ids[:, a:b].to(gpu), use_cache=False).logits[0] for a, b in zip(ends, ends[1:])]).detach()
    assert len(calls) == (2 if why == "" else 0) and all("bounds" in k for k in calls)
    with torch.no_grad():
        exact = torch.cat([host(ids[:, a:b], use_cache=False).logits[0] for a, b in zip(ends, ends[1:])])
    if why == "autocast":
        got, ref = got.half(), ref.half()
    near(got, ref, exact)


def test_groups_of_sequences():
    from adkv_amd.hf.score import _groups
    lengths = [3, 9, 1, 30, 9, 2, 1]
    assert list(_groups(lengths, 20, True)) == [[3], [1, 4], [0, 5, 2, 6]] and list(_groups(lengths, 20, False)) == [[3], [1, 4], [0, 5, 2, 6]]
    assert list(_groups(lengths, 10, False)) == [[3], [1], [4], [0, 5, 2], [6]] and list(_groups(lengths, 10, True)) == [[3], [1], [4], [0, 5, 2, 6]]
    assert list(_groups([5] * 4, 10, True)) == [[0, 1], [2, 3]] and list(_groups([], 10, True)) == [] and list(_groups([4, 4], 1, False)) == [[0], [1]]


@pytest.mark.gpu
@pytest.mark.parametrize("flavour,how", [("deployment", {}), ("deployment", dict(adkv_prompt=True)), ("evaluation", {}), ("evaluation", dict(prefill_full_precision=False))], ids=str)
def test_scores_a_few_texts_at_a_time(gpu, flavour, how, monkeypatch):
    """No run of the model has more tokens than were asked for, and all of them are scored: as by themselves, but for the roundings of products over other rows
    (and for what these change in codes)."""
    m = make(FLAVOURS[flavour].LlamaForCausalLM_ADKV, config(**how), torch.float16, gpu)
    texts = [ids_of(1, n, n)[0] for n in (40, 1, 7, 133, 2, 41, 39)]
    shapes, real = [], m.model.forward
    monkeypatch.setattr(m.model, "forward", lambda *a, **k: shapes.append(k["input_ids"].shape) or real(*a, **k))
    got = m.score(texts, top=2, tokens=90)
    assert [tuple(s) for s in shapes] == ([(1, 133), (1, 81), (1, 49)] if "adkv_prompt" in how else [(1, 133), (2, 41), (2, 39), (2, 2)])
    for t, g in zip(texts, got):
        alone = m.score([t], top=2)[0]
        assert g.logprobs.shape == (len(t) - 1,) and g.top_tokens.shape == (len(t) - 1, 2)
        if len(t) > 1 and how.get("prefill_full_precision", True):
            assert (g.logprobs - alone.logprobs).abs().max() <= 2.0 ** -6 and (g.entropy - alone.entropy).abs().max() <= 2.0 ** -6


def test_scores_of_quantised_prompts_are_the_evaluation_models():
    m = make(llama_adkv.LlamaForCausalLM_ADKV, config(), torch.float32, "cpu")
    with pytest.raises(ValueError, match="evaluation"):
        m.score([[1, 2]], prefill_full_precision=False)


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", [True, False])
def test_scores_show_what_quantisation_costs(gpu, prompt):
    """What the model itself gives for the same batch; other parameters of the quantiser give other scores, and none where prompts are attended with as they are."""
    mine = make(llama_adkv_eval.LlamaForCausalLM_ADKV, config(adkv_prompt=prompt), torch.float32, gpu)
    texts = [ids_of(1, n, n)[0] for n in (40, 1, 7, 33)]
    batch = torch.nn.utils.rnn.pad_sequence(texts, batch_first=True).to(gpu)
    found = {}
    for target in (3.5, 0.5):
        for layer in mine.model.layers:
            for side in ("key", "value"):
                getattr(layer.self_attn, f"{side}_quant_target").fill_(target)
        for full in (True, False, None):
            found[target, full] = torch.cat([s.logprobs for s in mine.score(texts, prefill_full_precision=full)])
        with torch.no_grad():
            logits = mine(batch, use_cache=True, prefill_full_precision=False).logits
        want = torch.cat([torch.log_softmax(x[:len(t) - 1].double(), -1).gather(1, t[1:, None].to(gpu))[:, 0] for x, t in zip(logits, texts)])
        # one logit per token from a product of other rows: 256 roundings of 2^-24 of numbers of size one
        assert (found[target, False] - want).abs().max() <= 2.0 ** -14
        assert torch.equal(found[target, True], found[target, None])
        mine.config.prefill_full_precision = False
        assert torch.equal(found[target, False], torch.cat([s.logprobs for s in mine.score(texts)]))
        del mine.config.prefill_full_precision
    assert torch.equal(found[3.5, True], found[0.5, True])
    assert (found[3.5, False] - found[0.5, False]).abs().max() > 2.0 ** -10 and (found[3.5, False] - found[3.5, True]).abs().max() > 2.0 ** -10


# ------------------------------------------------------------------------------------------------ where transformers' attention runs without packed sequences
def rows_of(gpu, T=9, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return tuple(torch.randn(1, h, T, 128, generator=g, device=gpu).half() for h in (4, 2, 2))


@pytest.mark.gpu
def test_derivatives_are_transformers(gpu, monkeypatch):
    """A tangent of the activations, a transform around the call, a mask that is learned; the evaluation model's tangents are those without the flag."""
    mine, other, _ = both("evaluation", torch.float16, gpu, attn_implementation="eager")
    monkeypatch.setattr(llama_adkv, "prompt_attention", lambda *a, **k: pytest.fail("not for this call"))
    attn = mine.model.layers[0].self_attn
    q, k, v = rows_of(gpu)
    with torch.no_grad(), torch.autograd.forward_ad.dual_level():
        for i in range(3):
            t = [q, k, v]
            t[i] = torch.autograd.forward_ad.make_dual(t[i], torch.ones_like(t[i]))
            assert llama_adkv.prompt_ctx(attn, *t, None, {}) is None
    with torch.no_grad():
        none = []
        torch.func.vmap(lambda x: none.append(llama_adkv.prompt_ctx(attn, x, k, v, None, {})) or x)(q[None])
        torch.func.jvp(lambda x: none.append(llama_adkv.prompt_ctx(attn, q, k, x, None, {})) or x, (v,), (v,))
        assert none == [None, None]
    assert llama_adkv.prompt_ctx(attn, q, k, v, torch.zeros(1, 1, 9, 9, device=gpu, requires_grad=True), {}) is None
    found = []
    for m in (mine, other):
        with torch.no_grad(), torch.autograd.forward_ad.dual_level():
            x = m.model.embed_tokens(ids_of(1, 9).to(gpu))
            out = m(inputs_embeds=torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), use_cache=False).logits
            found += list(torch.autograd.forward_ad.unpack_dual(out))
    assert found[1] is not None and torch.equal(found[0], found[2]) and torch.equal(found[1], found[3])


@pytest.mark.gpu
def test_masks_of_other_kinds_are_transformers(gpu, monkeypatch):
    """flex_attention's, and those that are not of four axes or too short."""
    from torch.nn.attention.flex_attention import create_block_mask
    attn = make(llama_adkv.LlamaForCausalLM_ADKV, config(adkv_prompt=True), torch.float16, gpu).model.layers[0].self_attn
    monkeypatch.setattr(llama_adkv, "prompt_attention", lambda *a, **k: pytest.fail("not for this call"))
    rows = rows_of(gpu)
    with torch.no_grad():
        for mask in (create_block_mask(lambda b, h, i, j: i >= j, 1, 1, 9, 9, device=gpu), torch.ones(1, 9, dtype=torch.bool, device=gpu), torch.ones(1, 1, 9, 8, dtype=torch.bool, device=gpu)):
            for how in ({}, dict(cu_seq_lens_q=torch.tensor([0, 4, 9], dtype=torch.int32, device=gpu))):
                assert llama_adkv.prompt_ctx(attn, *rows, mask, how) is None

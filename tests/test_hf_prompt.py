"""The operators around a prompt as the models use them: config.adkv_prompt, score(), beam search and what else moves a cache's sequences.

A model's logits are compared with the same model's in 64 bits on the host: with the framework's attention they are no further from them than
twice what transformers' attention in the same type is (both round scores and weights where the type has them), plus two of the type's steps."""
import pytest
import torch

pytest.importorskip("transformers")

from adkv_amd.hf import cache as cache_module  # noqa: E402
from adkv_amd.hf.cache import KVCache_ADKV, KVCacheLayer_ADKV  # noqa: E402
from adkv_amd.kernel import gemv  # noqa: E402

D = 128


def config(**how):
    from transformers import LlamaConfig
    return LlamaConfig(**{**dict(vocab_size=200, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=D,
                                 max_position_embeddings=1024, attn_implementation="sdpa", bos_token_id=0, eos_token_id=None, pad_token_id=0), **how})


def make(cls, cfg, dtype, device):
    torch.manual_seed(0)
    model = cls(cfg)
    full = lambda v: torch.full((cfg.num_key_value_heads * cfg.head_dim,), v)
    from adkv_amd.hf.llama_adkv import ADKVConfig
    mk = lambda: ADKVConfig(zp_init=full(0.0), scale_init=full(0.25), alpha=full(0.95), beta=full(0.02), quant_target=full(3.5))
    model.load_adkv_config([(mk(), mk()) for _ in range(cfg.num_hidden_layers)])
    return model.to(device).to(dtype).eval()


def both(flavour, dtype, device, **how):
    """(with the framework's attention, with transformers', in 64 bits on the host), the same weights."""
    from adkv_amd.hf import llama_adkv, llama_adkv_eval
    cls = {"deployment": llama_adkv, "evaluation": llama_adkv_eval}[flavour].LlamaForCausalLM_ADKV
    models = [make(cls, config(adkv_prompt=True, **how), dtype, device), make(cls, config(**how), dtype, device)]
    host = make(cls, config(**{**how, "attn_implementation": "eager"}), dtype, "cpu").double()
    return (*models, host)


def near(got, other, exact):
    step = 2 * torch.finfo(got.dtype).eps * exact.abs().max()
    err = lambda x: (x.cpu().double() - exact).abs().max()
    assert err(got) <= 2 * err(other) + step, (float(err(got)), float(err(other)))


def ids_of(B, T, seed=3):
    return torch.randint(1, 200, (B, T), generator=torch.Generator().manual_seed(seed))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("implementation", ["sdpa", "eager"])
@pytest.mark.parametrize("flavour", ["deployment", "evaluation"])
def test_prompts(gpu, flavour, implementation, dtype, monkeypatch):
    mine, other, host = both(flavour, dtype, gpu, attn_implementation=implementation)
    ids = ids_of(3, 70)
    pad = torch.ones(3, 70, dtype=torch.int64)
    pad[1, :30] = pad[2, :69] = 0
    calls = []
    from adkv_amd.hf import llama_adkv
    real = llama_adkv.prompt_attention
    monkeypatch.setattr(llama_adkv, "prompt_attention", lambda *a, **k: calls.append(1) or real(*a, **k))
    with torch.no_grad():
        exact = host(ids, use_cache=False).logits
        near(mine(ids.to(gpu), use_cache=flavour == "deployment").logits, other(ids.to(gpu), use_cache=False).logits, exact)
        assert len(calls) == 2
        # by themselves: positions are relative, and transformers' eager softmax is one of 32 bits, where a mask's lowest value of 64 is minus infinity
        exact = torch.cat([host(i[None, m.bool()], use_cache=False).logits[0] for i, m in zip(ids, pad)])
        got, ref = (m(ids.to(gpu), attention_mask=pad.to(gpu), use_cache=False).logits[pad.bool().to(gpu)] for m in (mine, other))
        near(got, ref, exact)
        assert len(calls) == 4


@pytest.mark.gpu
def test_steps_of_the_evaluation_model(gpu):
    """One token over the kept values, and several."""
    mine, other, _ = both("evaluation", torch.float16, gpu)
    ids = ids_of(2, 90).to(gpu)
    with torch.no_grad():
        outs = []
        for m in (mine, other):
            r = m(ids[:, :60], use_cache=True)
            a = m(ids[:, 60:61], past_key_values=r.past_key_values, use_cache=True).logits
            outs.append((a, m(ids[:, 61:], past_key_values=r.past_key_values, use_cache=True).logits))
    # two ways of rounding the same attention, through two layers and the head: a few steps of the type each
    for x, y in zip(*outs):
        assert (x - y).abs().max() <= 2.0 ** -6 * y.abs().max()


@pytest.mark.gpu
def test_where_transformers_attention_runs(gpu, monkeypatch):
    from adkv_amd.hf import llama_adkv
    monkeypatch.setattr(llama_adkv, "prompt_attention", lambda *a, **k: pytest.fail("not for this call"))
    mine, _, _ = both("deployment", torch.float16, gpu)
    ids = ids_of(1, 9).to(gpu)
    mine(ids, use_cache=False).logits.float().sum().backward()                    # a gradient
    with torch.no_grad():
        mine.float()(ids, use_cache=False)                                        # another type


@pytest.mark.gpu
def test_packed_sequences_have_no_cache(gpu):
    mine, _, _ = both("deployment", torch.float16, gpu)
    with torch.no_grad(), pytest.raises(ValueError, match="no cache"):
        mine(ids_of(1, 9).to(gpu), cu_seq_lens_q=torch.tensor([0, 4, 9], dtype=torch.int32, device=gpu), use_cache=True)


@pytest.mark.gpu
@pytest.mark.parametrize("flavour", ["deployment", "evaluation"])
def test_scores(gpu, flavour):
    """Texts of different lengths: a run of the model, its attention packed or padded, and the scores; rows of logits in several pieces."""
    mine, other, host = both(flavour, torch.float16, gpu)
    texts = [ids_of(1, n, n)[0] for n in (40, 1, 7, 133, 2)]
    got, ref = mine.score(texts, top=3, rows=50), other.score(texts, top=3)
    assert [g.logprobs.shape[0] for g in got] == [39, 0, 6, 132, 1] and got[3].top_tokens.shape == (132, 3)
    for text, g, r in zip(texts, got, ref):
        if len(text) < 2:
            continue
        with torch.no_grad():
            log = torch.log_softmax(host(text[None], use_cache=False).logits[0, :-1], -1)
        near(g.logprobs.half(), r.logprobs.half(), log.gather(1, text[1:, None])[:, 0])
        near(g.entropy.half(), r.entropy.half(), -(log.exp() * log).sum(-1))
        near(g.top_logprobs.half(), r.top_logprobs.half(), log.topk(3)[0])
    assert mine.score([]) == []
    with pytest.raises(ValueError, match="one token"):
        mine.score([[]])
    assert mine.score([[5, 6]])[0].top_tokens is None


# ------------------------------------------------------------------------------------------------ sequences that take each other's place
def filled(B, layers=2, T=300, bits=4, H=2, device="cpu", seed=0):
    """As after a prefill, with anything in it (no kernel runs)."""
    c = KVCache_ADKV(layers, bits)
    g = torch.Generator(device=device).manual_seed(seed)
    for layer in c:
        layer._init_buffers(B, H, D, torch.device(device))
        layer._cap_buffers(T)
        layer._quant_len = T
        for t, n in layer._tensors():
            t[:, :, :n] = torch.randint(0, 200, t[:, :, :n].shape, generator=g, device=device).to(t.dtype)
    return c


def as_indexing(tensors, index, *, used=None, into=None):
    for i, t in enumerate(tensors):
        new = t[index, :, :used[i]].clone()
        to = t if into is None else into[i]
        if into is not None:
            to.zero_()
        to[:len(index), :, :used[i]] = new


def same(cache, other, rows, index):
    """Whether `cache` holds rows `index` of `other`."""
    assert all(layer._B == rows for layer in cache)
    for a, b in zip(cache, other):
        for (x, n), (y, _) in zip(a._tensors(), b._tensors()):
            assert x.shape[0] == rows and x.is_contiguous() and torch.equal(x[:, :, :n], y[index.to(y.device), :, :n])


@pytest.mark.parametrize("bits", [4, 2])
def test_moving_sequences_on_the_host(monkeypatch, bits):
    """Which tensors go where, and what is known of them afterwards; the copies themselves are as_indexing here."""
    monkeypatch.setattr(cache_module, "take_sequences", as_indexing)
    c, was = filled(4, bits=bits), filled(4, bits=bits)
    index = torch.tensor([2, 2, 0, 3])
    c.reorder_cache(index)
    same(c, was, 4, index)
    c = filled(4, bits=bits)
    c.batch_select_indices(torch.tensor([3, 1]))
    same(c, was, 2, torch.tensor([3, 1]))
    assert c.get_seq_length() == 300 and c[0].key_states.shape[0] == 2 and c[0]._span == slice(0, 2) and c[0]._state_valid
    c.batch_repeat_interleave(3)
    same(c, was, 6, torch.tensor([3, 3, 3, 1, 1, 1]))
    assert not c[0].key_states[:, :, c[0]._n_super(300):].any() and c[0]._cap_len == was[0]._cap_len
    c.batch_select_indices(torch.tensor([True, False, False, False, True, False]))
    same(c, was, 2, torch.tensor([3, 1]))
    c.batch_select_indices(torch.tensor([1, 1, 0]))
    same(c, was, 3, torch.tensor([1, 1, 3]))
    empty = KVCache_ADKV(2)
    empty.reorder_cache(index)
    empty.batch_repeat_interleave(2)
    empty.batch_select_indices(torch.tensor([0]))


def test_what_is_known_of_the_states(monkeypatch):
    monkeypatch.setattr(cache_module, "take_sequences", as_indexing)
    c = filled(4)
    view = c.batch_view(1, 3)
    view[0]._state_valid = False                                    # a slice was stepped
    assert not c[0]._state_valid and bytes(c[0]._valid) == b"\1\0\0\1" and c[1]._state_valid
    c.reorder_cache(torch.tensor([3, 3, 2, 0]))
    assert bytes(c[0]._valid) == b"\1\1\0\1" and bytes(c[1]._valid) == b"\1" * 4
    c.batch_select_indices(torch.tensor([0, 3]))
    assert c[0]._state_valid
    c = filled(4)
    view = c.batch_view(1, 3)
    view.reorder_cache(torch.tensor([1, 0]))                        # within the slice, where the parent has it too
    same(c, filled(4), 4, torch.tensor([0, 2, 1, 3]))
    for change in (lambda: view.batch_select_indices(torch.tensor([0])), lambda: view.batch_repeat_interleave(2)):
        with pytest.raises(ValueError, match="batch view"):
            change()
    same(c, filled(4), 4, torch.tensor([0, 2, 1, 3]))


def test_views_of_what_moved(monkeypatch):
    """A slice that is stepped after its parent's sequences took each other's place is known to be; one of a batch that is another one by now is refused."""
    monkeypatch.setattr(cache_module, "take_sequences", as_indexing)
    for change in (lambda c: c.reorder_cache(torch.tensor([3, 2, 1, 0])), lambda c: c.batch_select_indices(torch.tensor([1, 0, 3, 2])), lambda c: c.batch_repeat_interleave(1)):
        c = filled(4)
        view = c.batch_view(1, 3)
        change(c)
        assert view[0].key_states.data_ptr() == c[0].key_states[1:].data_ptr()
        view[0]._state_valid = False                                # stepped
        assert not c[0]._state_valid and bytes(c[0]._valid) == b"\1\0\0\1" and c[1]._state_valid
        view.batch_view(1, 2)[1]._state_valid = False
        assert bytes(c[1]._valid) == b"\1\1\0\1"
    x = torch.zeros(2, 2, 1, D)
    for change in (lambda c: c.batch_select_indices(torch.tensor([0, 1])), lambda c: c.batch_repeat_interleave(2), lambda c: c.batch_select_indices(torch.arange(4).repeat(2))):
        c = filled(4)
        view, part = c.batch_view(1, 3), c.batch_view(0, 3).batch_view(1, 2)
        change(c)
        assert c[0]._state_valid and c.batch_view(0, 2)[0]._state_valid
        for v in (view, part):
            for use in (lambda: v[0].prefill(x, x, *[None] * 10), lambda: v[0].decode(x, x, x, *[None] * 10), lambda: v[0].extend(x, x, x, *[None] * 10), lambda: v.batch_view(0, 1),
                        lambda: v.commit(300), lambda: v.reorder_cache(torch.arange(v[0]._B)), lambda: v[0].state_dict()):
                with pytest.raises(RuntimeError, match="other sequences"):
                    use()
    c = filled(1)
    view = c.batch_view(0, 1)
    c.batch_repeat_interleave(2)
    with pytest.raises(RuntimeError, match="other sequences"):
        view.share(2)


def test_moving_sequences_of_the_evaluation_cache(monkeypatch):
    """In place, states and all; a layer whose first prompt was refused has buffers and nothing in them."""
    from adkv_amd.hf import llama_adkv_eval as module
    monkeypatch.setattr(module, "take_sequences", as_indexing)
    c = module.KVCache_ADKV(3)
    g = torch.Generator().manual_seed(0)
    for layer in c[:2]:
        layer._init_buffers(3, 8, torch.device("cpu"), torch.float32)
    with pytest.raises(Exception):
        c[1].update(torch.zeros(3, 2, 8), torch.zeros(3, 2, 8), *[None] * 10)
    for t in (c[0]._key_buf, c[0]._value_buf):
        t[:, :5] = torch.randn(3, 5, 8, generator=g)
    c[0].key_dc, c[0].key_scale, c[0].value_dc, c[0].value_scale = (torch.randn(3, 8, generator=g) for _ in range(4))
    c[0]._recent_len = 5
    of = lambda: [t.clone() for t in (c[0].key_states, c[0].value_states, c[0].key_dc, c[0].key_scale, c[0].value_dc, c[0].value_scale)]
    was, index = of(), torch.tensor([2, 0, 0])
    c.reorder_cache(index)
    assert all(torch.equal(a, b[index]) for a, b in zip(of(), was))
    with pytest.raises(ValueError, match="every sequence"):
        c.reorder_cache(torch.tensor([0, 1]))


def test_slices_that_are_further_than_their_batch(monkeypatch):
    """What a slice has been prefilled or stepped with does not move before the batch knows of it: the states would move without the codes."""
    monkeypatch.setattr(cache_module, "take_sequences", as_indexing)
    monkeypatch.setattr(cache_module, "append_kv_pair", lambda *a, **k: None)
    x = torch.zeros(2, 2, 7, D)
    moves = (lambda c: c.reorder_cache(torch.tensor([3, 2, 1, 0])), lambda c: c.batch_select_indices(torch.tensor([0, 3])), lambda c: c.batch_repeat_interleave(2))
    for move in moves:
        c, was = filled(4), filled(4)
        c.batch_view(0, 2)[0].prefill(x, x, *[None] * 10)
        with pytest.raises(ValueError, match="commit"):
            move(c)
        same(c, was, 4, torch.arange(4))
        c.batch_view(2, 4)[0].prefill(x, x, *[None] * 10)
        c.commit(307)
        move(c)
        c.batch_view(0, 2).reorder_cache(torch.tensor([1, 0]))
    c = filled(4)
    for layer in c.batch_view(1, 3):
        layer.prefill(x, x, *[None] * 10)
    c.batch_view(0, 1).reorder_cache(torch.tensor([0]))             # another slice
    with pytest.raises(ValueError, match="commit"):
        c.batch_view(0, 2).reorder_cache(torch.tensor([1, 0]))


def test_refused_moves(monkeypatch):
    monkeypatch.setattr(cache_module, "take_sequences", as_indexing)
    c = filled(3)
    for call, error, message in [(lambda: c.reorder_cache(torch.tensor([0, 1])), ValueError, "every sequence"), (lambda: c.reorder_cache(torch.tensor([[0, 1, 2]])), ValueError, "every sequence"),
                                 (lambda: c.reorder_cache(torch.tensor([0, 1, 3])), IndexError, "3 sequences"), (lambda: c.batch_select_indices(torch.tensor([-1])), IndexError, "3 sequences"),
                                 (lambda: c.batch_select_indices(torch.tensor([], dtype=torch.int64)), ValueError, "one sequence"),
                                 (lambda: c.batch_select_indices(torch.tensor([True, False])), ValueError, "each"), (lambda: c.batch_repeat_interleave(0), ValueError, "at least")]:
        with pytest.raises(error, match=message):
            call()
    same(c, filled(3), 3, torch.arange(3))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 2])
def test_moving_sequences(gpu, bits):
    c = filled(5, bits=bits, device=gpu)
    was = filled(5, bits=bits, device=gpu)
    for index in (torch.tensor([4, 4, 0, 1, 3]), torch.tensor([4, 4, 0, 1, 3], device=gpu)):
        c = filled(5, bits=bits, device=gpu)
        c.reorder_cache(index)
        same(c, was, 5, index)
    c.batch_select_indices(torch.tensor([2, 3], device=gpu))
    same(c, was, 2, torch.tensor([0, 1]))
    c.batch_repeat_interleave(2)
    same(c, was, 4, torch.tensor([0, 0, 1, 1]))
    assert not c[0].key_states[:, :, c[0]._n_super(300):].any()


@pytest.mark.gpu
@pytest.mark.parametrize("prefixed", [False, True])
def test_sequences_go_on_as_they_would_have(gpu, prefixed):
    """A prefilled batch, moved about, then stepped: outputs and codes are those of a batch that was in that order from the start."""
    g = torch.Generator(device=gpu).manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device=gpu).half()
    H, T = 2, 300
    par = [torch.zeros(H * D), torch.full((H * D,), 0.25), torch.full((H * D,), 0.95), torch.full((H * D,), 0.02), torch.full((H * D,), 3.5)] * 2
    par = [p.half().to(gpu) for p in par]
    first = KVCacheLayer_ADKV()
    first.prefill(rand(1, H, 40, D), rand(1, H, 40, D), *par)

    def begun(rows, k, v):
        layer = first.share(rows, T + 8) if prefixed else KVCacheLayer_ADKV()
        layer.prefill(k, v, *par)
        c = KVCache_ADKV(0)
        list.append(c, layer)
        return c
    k, v = rand(3, H, T, D), rand(3, H, T, D)
    index = torch.tensor([2, 0, 2, 1])
    a = begun(3, k, v)
    a.batch_select_indices(index.to(gpu))
    b = begun(4, k[index.to(gpu)], v[index.to(gpu)])
    for _ in range(3):
        q, kn, vn = rand(4, H, 1, D), rand(4, H, 1, D), rand(4, H, 1, D)
        x, y = (c[0].decode(q, kn, vn, *par, scaling=0.1)[0] for c in (a, b))
        assert torch.equal(x, y)
    same(a, b, 4, torch.arange(4))


@pytest.mark.gpu
@pytest.mark.parametrize("flavour", ["deployment", "evaluation"])
def test_beam_search(gpu, flavour, monkeypatch):
    """generate() with beams, prompt attention and all: the tokens are those found with indexing in the place of the kernel."""
    mine, _, _ = both(flavour, torch.float16, gpu)
    ids = ids_of(2, 21).to(gpu)
    find = lambda: mine.generate(ids, num_beams=4, max_new_tokens=12, do_sample=False, num_return_sequences=2)
    moved = []
    module = cache_module if flavour == "deployment" else __import__("adkv_amd.hf.llama_adkv_eval", fromlist=["x"])
    real = module.take_sequences
    monkeypatch.setattr(module, "take_sequences", lambda t, i, **k: moved.append(i.tolist()) or real(t, i, **k))
    got = find()
    assert len(moved) >= 11 and any(i != list(range(8)) for i in moved)
    monkeypatch.setattr(module, "take_sequences", as_indexing)
    assert torch.equal(got, find())


@pytest.mark.gpu
def test_a_prompt_its_scores_and_its_answers(gpu):
    """All of it in one run: prompts attended with and quantised, the first tokens' candidates, a cache that is forked for them, a step of each."""
    mine, _, _ = both("deployment", torch.float16, gpu)
    ids = ids_of(2, 33).to(gpu)
    with torch.no_grad():
        r = mine(ids, use_cache=True)
        first = gemv.token_logprobs(r.logits[:, -1], torch.full((2,), -1, device=gpu), top=3)
        assert torch.equal(first.logprobs, torch.zeros(2, device=gpu))
        cache = r.past_key_values
        cache.batch_repeat_interleave(3)
        step = mine(first.top_tokens.reshape(6, 1), past_key_values=cache, use_cache=True).logits
        alone = []
        for i in range(6):
            c = mine(ids[i // 3:i // 3 + 1], use_cache=True).past_key_values
            alone.append(mine(first.top_tokens.reshape(6, 1)[i:i + 1], past_key_values=c, use_cache=True).logits)
    assert (step - torch.cat(alone)).abs().max() <= 2.0 ** -6 * step.abs().max()

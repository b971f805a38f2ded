"""A prefilled sequence shared by a batch, several new tokens at once, and norms of the heads, as the cache and the attention module
use them (KVCacheLayer_ADKV.share / extend, config.adkv_extend, config.adkv_qk_norm)."""
import numpy as np
import pytest
import torch

from adkv_amd import synth
from adkv_amd.hf.cache import KVCache_ADKV, KVCacheLayer_ADKV

D = 128


def _np16(t):
    return t.detach().cpu().contiguous().view(torch.int16).numpy().view(np.float16)


def _flat(p):
    return [t.reshape(-1) for t in p.astuple()]


def _layer(P=24, H=2, bits=4, device="cpu", B=1):
    """As after a prefill, with nothing in it (no kernel runs)."""
    c = KVCacheLayer_ADKV(bits)
    c._init_buffers(B, H, D, torch.device(device))
    c._cap_buffers(P)
    c._quant_len = P
    return c


def test_sharing_on_the_host():
    one = _layer()
    one._key_state[0, 1, 5, 0] = 3.0
    v = one.share(4, 100)
    assert v.get_seq_length() == 24 and v._quant_len == 0 and v._cap_len == 128 and v._B == 4
    assert v.key_states.shape == (4, 2, 16, 32, 4, 4) and not v.key_states.any()
    assert v.get_mask_sizes(torch.arange(3)) == (27, 0)
    assert v._prefix[0] is one._key_buf
    own = v._own((1, 2, 3, 4, 5), 0)
    assert own[0][1, 5] == 3.0 and own[2:] == (3, 4, 5)
    one._key_state.zero_()                                   # the first goes on by itself
    assert own[0][1, 5] == 3.0
    assert v.nbytes() == sum(t.numel() * t.element_size() for t in (v._key_buf, v._value_buf, v._key_ckpt, v._value_ckpt,
                                                                    one._key_buf, one._value_buf, one._key_ckpt, one._value_ckpt))
    view = v.batch_view(1, 3)
    assert view.get_seq_length() == 24 and view._prefix is v._prefix
    v.commit(34)
    assert v._quant_len == 10 and v.get_seq_length() == 34
    with pytest.raises(ValueError, match="fewer tokens"):
        v.commit(23)
    with pytest.raises(ValueError, match="more tokens"):
        v.commit(24 + 129)
    with pytest.raises(ValueError, match="room by share"):
        v.reserve(4, 2, D, 100, "cpu")
    whole = KVCache_ADKV(0)
    list.extend(whole, (one, _layer()))
    both = whole.share(2)
    assert len(both) == 2 and both.get_seq_length(1) == 24 and isinstance(both, KVCache_ADKV)


def test_sharing_refusals():
    with pytest.raises(ValueError, match="one prefilled sequence"):
        KVCacheLayer_ADKV().share(2)
    with pytest.raises(ValueError, match="one prefilled sequence"):
        _layer(P=0).share(2)
    with pytest.raises(ValueError, match="one prefilled sequence"):
        _layer(B=2).share(2)
    with pytest.raises(ValueError, match="one prefilled sequence"):
        _layer().share(1).share(2)
    with pytest.raises(ValueError, match="at least one"):
        _layer().share(0)
    wide = KVCacheLayer_ADKV()
    wide._init_buffers(1, 2, 256, torch.device("cpu"))
    wide._quant_len = 8
    with pytest.raises(ValueError, match="head_dim 128"):
        wide.share(2)
    stepped = _layer()
    stepped._state_valid = False
    with pytest.raises(NotImplementedError, match="before it is decoded"):
        stepped.share(2)


def test_extend_refusals():
    kp = _flat(synth.make_params(2, D))
    z = lambda *n: torch.zeros(*n)
    c = _layer()
    with pytest.raises(ValueError, match="as many keys"):
        c.extend(z(1, 2, 3, D), z(1, 2, 2, D), z(1, 2, 2, D), *kp, *kp)
    with pytest.raises(ValueError, match="head_dim 128"):
        c.extend(z(1, 2, 3, 256), z(1, 2, 3, 256), z(1, 2, 3, 256), *kp, *kp)
    with pytest.raises(ValueError, match="different \\(B, H, C\\)"):
        c.extend(z(2, 2, 3, D), z(2, 2, 3, D), z(2, 2, 3, D), *kp, *kp)
    with pytest.raises(RuntimeError, match="HIP device"):
        c.extend(z(1, 2, 3, D), z(1, 2, 3, D), z(1, 2, 3, D), *kp, *kp)
    shared = c.share(3)
    with pytest.raises(ValueError, match="exactly one"):
        shared.decode(z(3, 2, 2, D), z(3, 2, 2, D), z(3, 2, 2, D), *kp, *kp)
    assert c._quant_len == 24 and shared._quant_len == 0


def _words(c, first, n):
    return [b[:, :, first:first + n].cpu() for b in (c._key_buf, c._value_buf)]


@pytest.mark.gpu
@pytest.mark.parametrize("bits,G,dtype", [(4, 1, torch.float16), (2, 4, torch.bfloat16), (4, 8, torch.bfloat16)])
def test_shared_equals_copies(gpu, oracle, tmp_path, bits, G, dtype):
    """Questions and steps behind a shared prompt against the same on a cache of whole sequences: the same codes, and outputs that differ
    by what two runs of the operator may: weights and results each rounded once on either side."""
    H, B, P = 2, 3, 16 * 19
    kg, vg = (_flat(synth.make_params(H, D, bits=bits, seed=s).to(gpu)) for s in (3, 4))
    g = torch.Generator().manual_seed(6)
    lens = (37, 1, 1, 5, 250, 1)
    total = sum(lens)
    rows = []
    for make, seed, kw in ((synth.make_k, 1, {"t0": P}), (synth.make_v, 2, {})):
        pre = make(1, H, P, D, seed=seed, dtype=torch.float16)
        new = make(B, H, total, D, seed=seed + 5, dtype=torch.float16, **kw)
        rows.append((pre.to(dtype).to(gpu), new.to(dtype).to(gpu)))
    (kp, kn), (vp, vn) = rows
    one = KVCacheLayer_ADKV(bits)
    one.prefill(kp, vp, *kg, *vg)
    shared = one.share(B)
    whole = KVCacheLayer_ADKV(bits)
    whole.prefill(kp.expand(B, H, P, D), vp.expand(B, H, P, D), *kg, *vg)
    tps, at = 32 // bits, 0
    for n in lens:
        q = torch.randn(B, H * G, n, D, generator=g).to(dtype).to(gpu)
        k, v = kn[:, :, at:at + n], vn[:, :, at:at + n]
        want = whole.extend(q, k, v, *kg, *vg, scaling=D ** -0.5)
        if n == 1:
            got, weights = shared.decode(q, k, v, *kg, *vg, scaling=D ** -0.5)
            assert weights is None
            got = got[:, None]
        else:
            got = shared.extend(q, k, v, *kg, *vg, scaling=D ** -0.5)
        at += n
        assert shared.get_seq_length() == whole.get_seq_length() == P + at
        used = -(-at // tps)
        for a, b in zip(_words(shared, 0, used), _words(whole, P // tps, used)):
            assert torch.equal(a, b)
        with oracle.code_bits(bits):
            values = oracle.replay_f16(whole._value_buf.cpu().numpy(), *[_np16(t).reshape(H, D) for t in vg], P + at)[0]
        top = float(np.abs(values.astype(np.float32)).max())
        # either side: weights 2^-11 and, small ones, 2^-25 a token, fp32 2^-14, the result half a step
        bound = 2 * top * (2.0 ** -11 + 2.0 ** -14 + (P + at) * 2.0 ** -25 + torch.finfo(dtype).eps / 2)
        assert (got.float() - want.float()).abs().max().item() <= bound
        if at == 39:      # saved and restored with its prefix in between
            cache = KVCache_ADKV(0)
            list.extend(cache, [shared])
            cache.save(tmp_path / "cache.pt")
            shared = KVCache_ADKV.load(tmp_path / "cache.pt", gpu)[0]
            assert shared.get_seq_length() == P + at
            for a, b in zip(_words(shared, 0, used), _words(whole, P // tps, used)):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_prefill_behind_a_prefix(gpu):
    """Rows quantised without attention, in slices of the batch, continue the prompt's stream."""
    H, B, P, T = 2, 4, 64, 53
    kg, vg = (_flat(synth.make_params(H, D, seed=s).to(gpu)) for s in (3, 4))
    kp, vp = (synth.make_k(1, H, P, D, seed=s, dtype=torch.float16).to(gpu) for s in (1, 2))
    kn, vn = (synth.make_k(B, H, T, D, seed=s, t0=P, dtype=torch.float16).to(gpu) for s in (5, 6))
    one = KVCacheLayer_ADKV()
    one.prefill(kp, vp, *kg, *vg)
    shared = one.share(B)
    for b in (0, 2):
        shared.batch_view(b, b + 2).prefill(kn[b:b + 2], vn[b:b + 2], *kg, *vg)
    shared.commit(P + T)
    whole = KVCacheLayer_ADKV()
    whole.prefill(torch.cat([kp.expand(B, H, P, D), kn], 2), torch.cat([vp.expand(B, H, P, D), vn], 2), *kg, *vg)
    for a, b in zip(_words(shared, 0, 7), _words(whole, P // 8, 7)):
        assert torch.equal(a, b)
    # and in two parts
    again = one.share(B)
    again.prefill(kn[:, :, :20], vn[:, :, :20], *kg, *vg)
    again.prefill(kn[:, :, 20:], vn[:, :, 20:], *kg, *vg)
    for a, b in zip(_words(again, 0, 7), _words(shared, 0, 7)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_boolean_masks(gpu):
    H, B, n, T = 2, 3, 4, 20
    kg, vg = (_flat(synth.make_params(H, D, seed=s).to(gpu)) for s in (3, 4))
    k, v = (synth.make_k(B, H, T + n, D, seed=s, dtype=torch.float16).to(gpu) for s in (1, 2))
    q = torch.randn(B, H, n, D, generator=torch.Generator().manual_seed(5)).half().to(gpu)
    seen = torch.ones(B, 1, n, T + n, dtype=torch.bool)
    seen[1, :, :, :7] = False
    outs = []
    for mask in (seen, torch.zeros(seen.shape, dtype=torch.float16).masked_fill(~seen, torch.finfo(torch.float16).min)):
        c = KVCacheLayer_ADKV()
        c.prefill(k[:, :, :T], v[:, :, :T], *kg, *vg)
        outs.append(c.extend(q, k[:, :, T:], v[:, :, T:], *kg, *vg, attention_mask=mask.to(gpu), scaling=D ** -0.5))
    assert torch.equal(*outs)


def _model(gpu, heads=4, kv_heads=2, dtype=torch.float16, **kw):
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from adkv_amd.hf.llama_adkv import ADKVConfig, LlamaForCausalLM_ADKV
    cfg = LlamaConfig(vocab_size=128, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=heads,
                      num_key_value_heads=kv_heads, head_dim=D, max_position_embeddings=512, attn_implementation="eager", **kw)
    torch.manual_seed(0)
    model = LlamaForCausalLM_ADKV(cfg).to(gpu).to(dtype).eval()
    n = kv_heads * D
    full = lambda v: torch.full((n,), v)
    mk = lambda: ADKVConfig(zp_init=full(0.0), scale_init=full(0.05), alpha=full(0.95), beta=full(0.05), quant_target=full(3.5))
    model.load_adkv_config([(mk(), mk()) for _ in range(2)])
    if kw.get("adkv_qk_norm"):
        with torch.no_grad():
            for layer in model.model.layers:
                for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                    norm.weight.add_(0.1 * torch.randn(D, generator=torch.Generator().manual_seed(1)).to(norm.weight))
    return model


@pytest.mark.gpu
def test_model_answers_behind_a_shared_prompt(gpu):
    """A document prefilled once, three questions of different lengths about it in one padded call, then steps: the logits are those of
    whole sequences (the projections run over other shapes, hence the tolerance of the follow-up test)."""
    model = _model(gpu, adkv_qk_norm=True, adkv_extend=True)
    g = torch.Generator().manual_seed(5)
    B, P, n, steps = 3, 72, 9, 4
    prompt = torch.randint(0, 128, (1, P), generator=g).to(gpu)
    more = torch.randint(0, 128, (B, n + steps), generator=g).to(gpu)
    seen = torch.ones(B, P + n + steps, dtype=torch.long, device=gpu)
    seen[1, P:P + 4] = 0                                     # left-padded behind the prompt
    pos = seen.cumsum(-1) - 1
    with torch.no_grad():
        one = model(prompt, use_cache=True).past_key_values
        shared = one.share(B, n + steps)
        whole = model(prompt.expand(B, P), use_cache=True).past_key_values
        for at, k in ((0, n), *((n + i, 1) for i in range(steps))):
            ids, end = more[:, at:at + k], P + at + k
            kw = dict(attention_mask=seen[:, :end], position_ids=pos[:, end - k:end], use_cache=True)
            got = model(ids, past_key_values=shared, **kw).logits.float()
            want = model(ids, past_key_values=whole, **kw).logits.float()
            real = seen[:, end - k:end].bool()
            assert shared.get_seq_length() == whole.get_seq_length() == end
            assert torch.allclose(got[real], want[real], atol=2e-2, rtol=2e-2)
        assert one.get_seq_length() == P


@pytest.mark.gpu
def test_model_follow_up_at_once(gpu):
    """config.adkv_extend: a follow-up turn in one call leaves the codes that the steps leave, and their logits."""
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, 128, (2, 12), generator=g).to(gpu)
    more = torch.randint(0, 128, (2, 30), generator=g).to(gpu)
    results = []
    for at_once in (True, False):
        model = _model(gpu, adkv_extend=at_once)
        with torch.no_grad():
            cache = model(prompt, use_cache=True).past_key_values
            logits = model(more, past_key_values=cache, use_cache=True).logits.float()
        results.append((cache, logits))
    (a, got), (b, want) = results
    assert a.get_seq_length() == b.get_seq_length() == 42
    assert torch.equal(a[0]._key_buf, b[0]._key_buf) and torch.equal(a[0]._value_buf, b[0]._value_buf)
    assert torch.allclose(got, want, atol=2e-2, rtol=2e-2)


@pytest.mark.gpu
def test_model_trains_its_head_norms(gpu, monkeypatch):
    """Gradients of every parameter with the fused norms against those with the module's own norms and rotation, both in fp32."""
    from adkv_amd.hf import llama_adkv as M
    model = _model(gpu, dtype=torch.float32, adkv_qk_norm=True).train()
    ids = torch.randint(1, 128, (2, 33), generator=torch.Generator().manual_seed(2)).to(gpu)
    calls = []

    def gradients(f):
        monkeypatch.setattr(M, "rope_norm_qk", f)
        model.zero_grad(set_to_none=True)
        model(ids, use_cache=False, labels=ids).loss.backward()
        return {n: p.grad.clone() for n, p in model.named_parameters()}

    real = M.rope_norm_qk

    def fused(*a):
        calls.append(1)
        return real(*a)

    def plain(q, k, cos, sin, wq, wk, eps):
        norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
        return M.apply_rotary_pos_emb(norm(q, wq), norm(k, wk), cos, sin)
    got, want = gradients(fused), gradients(plain)
    assert len(calls) == 2
    for n in want:
        assert (got[n] - want[n]).abs().max() <= 1e-4 * want[n].abs().max(), n
    assert all(f"model.layers.{i}.self_attn.{n}_norm.weight" in got for i in range(2) for n in "qk")


def test_norms_without_a_device():
    """On the CPU the module's own norms and rotation run, and gradients reach their weights."""
    model = _model("cpu", dtype=torch.float32, adkv_qk_norm=True).train()
    ids = torch.randint(1, 128, (1, 6), generator=torch.Generator().manual_seed(2))
    model(ids, use_cache=False, labels=ids).loss.backward()
    for layer in model.model.layers:
        assert layer.self_attn.q_norm.weight.grad.abs().sum() > 0 and layer.self_attn.k_norm.weight.grad.abs().sum() > 0
    assert not hasattr(_model("cpu").model.layers[0].self_attn, "q_norm")


@pytest.mark.gpu
def test_extend_in_other_types(gpu):
    """Rows of fp32 are rounded to fp16 in front of the kernels, as in decode; the result comes back in the query's type."""
    H, B, n, T = 2, 2, 5, 33
    kg, vg = (_flat(synth.make_params(H, D, seed=s).to(gpu)) for s in (3, 4))
    k, v = (synth.make_k(B, H, T + n, D, seed=s, dtype=torch.float16).to(gpu) for s in (1, 2))
    q = torch.randn(B, H, n, D, generator=torch.Generator().manual_seed(5)).half().to(gpu)
    outs = []
    for to in (torch.float16, torch.float32):
        c = KVCacheLayer_ADKV()
        c.prefill(k[:, :, :T], v[:, :, :T], *kg, *vg)
        outs.append(c.extend(q.to(to), k[:, :, T:].to(to), v[:, :, T:].to(to), *kg, *vg, scaling=D ** -0.5))
        assert outs[-1].dtype == to and outs[-1].shape == (B, n, H, D)
    assert torch.equal(outs[0].float(), outs[1])

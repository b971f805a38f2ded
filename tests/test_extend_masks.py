"""gemv.extend with masks that do not hide the later tokens themselves (causality does), beside tokens at a type's lowest value."""
import pytest
import torch

from adkv_amd import synth
from adkv_amd.hf.cache import KVCacheLayer_ADKV
from test_extend import D, Case

SIZES = [  # B, H, G, P, T, n, padded own tokens
    (2, 2, 1, 0, 46, 5, 32),       # one matrix instruction's rows: every other 16 tokens go to waves with maxima of their own
    (2, 1, 2, 130, 46, 5, 32), (1, 1, 1, 0, 16, 16, 16), (2, 2, 4, 0, 40, 4, 44),
    (2, 1, 1, 130, 0, 100, 64),    # tiles of 64 tokens, the prefix apart: rows that see none of their own
    (1, 2, 4, 70, 130, 20, 128), (2, 1, 2, 90, 0, 200, 64), (1, 2, 1, 0, 3, 300, 190),
    (40, 8, 1, 0, 0, 100, 64), (40, 8, 1, 70, 0, 100, 64),          # pieces of more than one tile
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_padding_for_all_new_tokens_alike(gpu, oracle, size, dtype):
    B, H, G, P, T, n, pad = size
    c = Case(oracle, gpu, B, H, G, P, T, n, dtype=torch.bfloat16 if dtype == torch.bfloat16 else torch.float16, seed=41)
    for low in (torch.finfo(dtype).min, torch.finfo(dtype).min / 2):
        mask = torch.zeros(B, 1, 1, P + T + n, dtype=dtype)
        mask[0, :, :, P:P + pad] = low
        mask = mask.to(gpu)
        c.check(c.run(D ** -0.5, mask), D ** -0.5, mask)
    every = torch.zeros(B, 1, 1, P + T + n, dtype=dtype)
    every[:, :, :, :P + pad] = torch.finfo(dtype).min              # the prefix too
    every = every.to(gpu)
    c.check(c.run(D ** -0.5, every), D ** -0.5, every)


@pytest.mark.gpu
@pytest.mark.parametrize("P,T,n,pad", [(0, 46, 5, 32), (72, 0, 100, 64), (0, 46, 150, 32)])
def test_boolean_masks_in_bfloat16(gpu, oracle, P, T, n, pad):
    """Through the cache, behind a shared prompt and without one: what the attention module hands over."""
    B, H, G = 2, 2, 1
    c = Case(oracle, gpu, B, H, G, P, T, n, dtype=torch.bfloat16, S=256, seed=43)
    seen = torch.ones(B, 1, 1, P + T + n, dtype=torch.bool)
    seen[0, :, :, P:P + pad] = False
    mask = torch.zeros(seen.shape, dtype=torch.bfloat16).masked_fill_(~seen, torch.finfo(torch.bfloat16).min).to(gpu)
    kp, vp = ([t.reshape(-1) for t in synth.make_params(H, D, seed=43 + i).to(gpu).astuple()] for i in (1, 2))
    layer = KVCacheLayer_ADKV()
    if P:
        one = KVCacheLayer_ADKV()
        rows = [synth.make_k(1, H, P, D, seed=43, dtype=torch.float16), synth.make_v(1, H, P, D, seed=44, dtype=torch.float16)]
        one.prefill(*[r.to(gpu) for r in rows], *kp, *vp)
        layer = one.share(B, T + n)
    if T:
        old = [synth.make_k(B, H, T + n, D, seed=45, t0=P, dtype=torch.float16), synth.make_v(B, H, T + n, D, seed=46, dtype=torch.float16)]
        layer.prefill(*[t[:, :, :T].bfloat16().to(gpu) for t in old], *kp, *vp)
    out = layer.extend(c.q, *c.new, *kp, *vp, attention_mask=seen.to(gpu), scaling=D ** -0.5)
    want = c.run(D ** -0.5, mask)
    c.check(want, D ** -0.5, mask)
    c.check(out, D ** -0.5, mask)

"""gemv.extend with very many new tokens at once: some of them against the same tokens by themselves."""
import pytest
import torch

from adkv_amd import synth
from adkv_amd.kernel import gemv

D = 128


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,G,P,T,n", [(1, 1, 1, 0, 0, 65539), (4, 1, 2, 100, 9, 32768), (1, 2, 1, 0, 70, 70000)])
def test_tokens_of_a_long_call(gpu, B, H, G, P, T, n):
    """A token that is handed over again, with the tokens in front of it in the cache, gets the same code and the same output but for
    roundings: on either side weights (2^-11, small ones 2^-25 a token), sums (2^-14) and the result (2^-11), of values up to `top`."""
    gen = torch.Generator(device=gpu).manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen, device=gpu, dtype=torch.float16)
    params = [p.to(gpu).astuple() for p in (synth.make_params(H, D, seed=s) for s in (1, 2))]
    pre, own = None, params
    if P:
        pc, pst = [synth.alloc_cache(1, H, P, D, gpu) for _ in range(2)], [torch.zeros(1, H, D, 2, dtype=torch.float16, device=gpu) for _ in range(2)]
        gemv.append_kv_pair(*pc, rand(1, H, P, D), rand(1, H, P, D), *params, 0, *pst)
        pre = gemv.SharedPrefix(*pc, P, *params)
        own = [(st[0, :, :, 0].contiguous(), st[0, :, :, 1].contiguous(), *p[2:]) for st, p in zip(pst, params)]
    cache = [synth.alloc_cache(B, H, T + n, D, gpu) for _ in range(2)]
    ckpt = [torch.zeros(B, H, (T + n) // 256 + 1, D, 2, dtype=torch.float16, device=gpu) for _ in range(2)]
    if T:
        state = [torch.zeros(B, H, D, 2, dtype=torch.float16, device=gpu) for _ in range(2)]
        gemv.append_kv_pair(*cache, rand(B, H, T, D), rand(B, H, T, D), *own, 0, *state, k_ckpt=ckpt[0], v_ckpt=ckpt[1], ckpt_interval=256)
    q, new = rand(B, H * G, n, D), [rand(B, H, n, D) for _ in range(2)]

    def run(at, count):
        cut = lambda t: t[:, :, at:at + count]
        return gemv.extend(cut(q), *cache, *map(cut, new), *own, T + at, D ** -0.5, prefix=pre, k_ckpt=ckpt[0], v_ckpt=ckpt[1], ckpt_interval=256)
    whole = run(0, n)
    kept = [t.clone() for t in cache + ckpt]
    assert bool(torch.isfinite(whole).all())
    top = 16.0        # values follow rows of up to 6, and twice that where the scale has not settled
    for at in (0, 1, 255, n // 2 + 1, n - 300, n - 1):
        one = run(at, 1)
        far = (one[:, 0].float() - whole[:, at].float()).abs().max().item()
        assert far <= 2 * top * (2.0 ** -11 + 2.0 ** -14 + (P + T + at) * 2.0 ** -25 + 2.0 ** -11), at
    assert all(torch.equal(a, b) for a, b in zip(cache, kept[:2]))

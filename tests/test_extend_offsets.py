"""Rows of gemv.extend that are packed but start at an odd element: read by way of a copy, like any others that are not at words."""
import pytest
import torch

from test_extend import D, Case


def _odd(t):
    """The same values, contiguous, two bytes behind a word."""
    flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    v = flat[1:].view(t.shape)
    assert v.is_contiguous() and v.data_ptr() % 4 == 2
    return v


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 2, 1, 40, 30, 1), (3, 2, 2, 90, 30, 6), (1, 2, 4, 0, 70, 40)])
def test_packed_rows_at_odd_elements(gpu, oracle, size):
    c = Case(oracle, gpu, *size, seed=29)
    fresh = [t.clone() for t in c.cache + c.ckpt]
    c.q = c.q.contiguous()
    want = c.run(D ** -0.5).clone()
    q, new = c.q, [t.contiguous() for t in c.new]
    for which in ("q", "k", "v", "all"):
        c.q = _odd(q) if which in ("q", "all") else q
        c.new = [_odd(t) if which in (side, "all") else t for side, t in zip("kv", new)]
        for t, f in zip(c.cache + c.ckpt, fresh):
            t.copy_(f)
        assert torch.equal(c.run(D ** -0.5), want), which
    c.check(want, D ** -0.5)


@pytest.mark.gpu
def test_appended_rows_at_odd_elements(gpu):
    """The same for rows that are quantised without attention."""
    from adkv_amd import synth
    from adkv_amd.kernel import gemv
    B, H, T = 2, 2, 21
    params = [synth.make_params(H, D, seed=s).to(gpu).astuple() for s in (1, 2)]
    k, v = (synth.make_k(B, H, T, D, seed=s, dtype=torch.float16).to(gpu) for s in (3, 4))
    results = []
    for rows in ((k, v), (_odd(k), v), (k, _odd(v))):
        cache = [synth.alloc_cache(B, H, T, D, gpu) for _ in range(2)]
        state = [torch.zeros(B, H, D, 2, dtype=torch.float16, device=gpu) for _ in range(2)]
        gemv.append_kv_pair(*cache, *rows, *params, 0, *state)
        results.append(cache + [s.view(torch.int16) for s in state])
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(results[0], r))

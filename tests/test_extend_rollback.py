"""Drafted tokens that were not accepted: gemv.extend from an earlier token on, over slots and recorded states that hold what was rejected."""
import pytest
import torch

from test_extend import D, Case


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("T", [0, 3, 59, 64, 126])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_rejected_tokens_leave_nothing(gpu, oracle, bits, T, n):
    c = Case(oracle, gpu, 2, 2, 2, 40, T, n, bits=bits, seed=51, room=90)
    gen = torch.Generator(device=gpu).manual_seed(1)
    junk = [torch.randn(2, 2, 77, D, generator=gen, device=gpu, dtype=torch.float16) * 3 for _ in range(2)]
    q, new, keep, N = c.q, c.new, c.n, 77
    c.q, c.new = torch.randn(2, 4, N, D, generator=gen, device=gpu, dtype=torch.float16), junk
    c.run(D ** -0.5)
    assert any(bool((a != b).any()) for a, b in zip((t.cpu() for t in c.cache), map(torch.from_numpy, c.want_cache)))
    c.q, c.new = q, new
    out = c.run(D ** -0.5)
    per = 32 // bits
    full, rest = (T + n) // per, (T + n) % per
    for t, w in zip(c.cache, c.want_cache):      # what is behind the new tokens is nobody's: words that end with them, and the fields of the last
        a, b = (x.view(torch.int32).reshape(2, 2, -1, D) for x in (t.cpu(), torch.from_numpy(w)))
        assert torch.equal(a[:, :, :full], b[:, :, :full])
        if rest:
            low = (1 << bits * rest) - 1
            assert torch.equal(a[:, :, full] & low, b[:, :, full] & low)
        t.view(torch.int32).view(2, 2, -1, D).copy_(b.to(gpu))
    c.check(out, D ** -0.5)
    # and goes on from there as if nothing had been rejected: the states that were recorded are the new tokens'
    d = Case(oracle, gpu, 2, 2, 2, 40, T, n, bits=bits, seed=51, room=90)
    d.run(D ** -0.5)
    used = (T + n) // c.S if n > 1 else (T + n - 1) // c.S
    for a, b in zip(c.ckpt, d.ckpt):
        assert torch.equal(a[:, :, :used].view(torch.int16), b[:, :, :used].view(torch.int16))

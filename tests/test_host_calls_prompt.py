"""The host calls of the operators around a prompt: what they take gives what the Python functions give, and what they do not take goes there."""
import types

import pytest
import torch

from adkv_amd import _lib
from adkv_amd.kernel import gemv

NAMES = ("prompt_attention", "token_logprobs", "take_sequences")


def test_other_arguments_are_left_to_python():
    h = _lib.host()
    x = torch.zeros(1, 1, 1, 128, dtype=torch.float16)
    for name, n in zip(NAMES, (6, 3, 4)):
        f = getattr(h, name)
        assert f() is None and f(*[None] * n) is None and f(*[x] * n) is None and f(*[1 << 70] * n) is None and f(*[[x]] * n) is None
    assert h.prompt_attention(x, x, x, 1.0, None, None) is None                # not on a device
    assert h.token_logprobs(x[0, 0], torch.zeros(1, dtype=torch.int64), 0) is None
    assert h.take_sequences([x], torch.zeros(1, dtype=torch.int64), [1], None) is None
    assert h.take_sequences([], None, [], []) is None and h.take_sequences([None], x, [None], [None]) is None


@pytest.mark.gpu
def test_both_ways_are_one(gpu, monkeypatch):
    g = torch.Generator(device=gpu).manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device=gpu)
    q, k, v = rand(2, 9, 4, 64).half().transpose(1, 2), rand(2, 33, 2, 64).half().transpose(1, 2), rand(2, 33, 2, 64).half().transpose(1, 2)
    wide = rand(2, 3000, 1, 64).half().transpose(1, 2)
    mask = rand(2, 1, 9, 33) > 0
    x, t = rand(3, 5, 301), torch.randint(0, 301, (3, 5), generator=g, device=gpu)
    cache = torch.randint(0, 255, (5, 2, 7, 32, 4, 4), generator=g, device=gpu, dtype=torch.uint8)
    index = torch.tensor([1, 0, 4], device=gpu)
    bounds = torch.tensor([0, 5, 33], dtype=torch.int32, device=gpu)

    def all_of_them():
        found = [gemv.prompt_attention(q, k, v, 0.125), gemv.prompt_attention(q, k, v, 0.125, mask), gemv.prompt_attention(q, k, v, 0.125, mask.float()),
                 gemv.prompt_attention(wide[:, :, -1:], wide, wide, 0.125), gemv.prompt_attention(k[:1], k[:1], v[:1], 0.125, bounds=bounds)]
        for top in (0, 4):
            found += [r for r in gemv.token_logprobs(x[:, 1:], t[:, 1:].contiguous(), top=top) if r is not None]
            found += [r for r in gemv.token_logprobs(x[0, 0], t[0, 0], top=top) if r is not None]
        one, new = cache.clone(), torch.empty(3, 2, 9, 32, 4, 4, dtype=torch.uint8, device=gpu)
        gemv.take_sequences([one], index, used=[6])
        gemv.take_sequences([cache], index, used=[6], into=[new])
        return [*found, one, new]
    calls = []
    h = _lib.host()
    counted = {n: (lambda *a, f=getattr(h, n): [calls.append(r is not None) or r for r in [f(*a)]][0]) for n in NAMES}
    monkeypatch.setattr(_lib, "_host", types.SimpleNamespace(**counted))
    fast = all_of_them()
    assert len(calls) == 11 and all(calls)
    monkeypatch.setattr(_lib, "_host", types.SimpleNamespace(**{n: (lambda *a: None) for n in NAMES}))
    assert all(torch.equal(a, b) for a, b in zip(fast, all_of_them()))


class _Sub(torch.Tensor):
    pass


@pytest.mark.gpu
def test_what_is_left_to_python_on_the_device(gpu):
    h = _lib.host()
    x = torch.randn(1, 2, 8, 64, device=gpu).half()
    take = lambda *t, mask=None, bounds=None, scaling=1.0: h.prompt_attention(*t, scaling, mask, bounds) is None
    assert not take(x, x, x)
    assert take(x, x, x, scaling=1) and take(x.float(), x.float(), x.float()) and take(x, x, x.bfloat16()) and take(x.clone().requires_grad_(), x, x)
    assert take(x.as_subclass(_Sub), x, x) and take(x[:, :, :0], x, x) and take(x, x[:, :, :4], x[:, :, :4]) and take(x[..., ::2], x[..., ::2], x[..., ::2])
    assert take(x, x, x, mask=torch.zeros(1, 1, 8, 8, device=gpu).double()) and take(x, x, x, bounds=torch.tensor([0, 8], device=gpu))
    with torch.no_grad():
        assert not take(x.clone().requires_grad_(), x, x)
    y, t = torch.randn(4, 50, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    assert h.token_logprobs(y, t, 3) is not None
    for args in ((y.double(), t, 3), (y, t.int(), 3), (y, t[:3], 3), (y, t, 51), (y, t, -1), (y.t(), t, 0), (y.clone().requires_grad_(), t, 0), (y[:0], t[:0], 0)):
        assert h.token_logprobs(*args) is None
    c, i = torch.zeros(4, 2, 3, 16, dtype=torch.uint8, device=gpu), torch.tensor([1, 0], device=gpu)
    assert h.take_sequences([c], i, None, None) == 0
    for args in (([c], i.int(), None, None), ([c], i, [4], None), ([c], i, [-1], None), ([c[:, :, :, :4]], i, None, None), ([c.transpose(0, 1)], i, None, None), ([c, c[:3]], i, None, None),
                 ([c], i.repeat(3), None, None), ([c], i, None, [c[:2]]), ([c], i, None, [c.clone()]), ([c], i[:0], None, None), ((c,), i, None, None)):
        assert h.take_sequences(*args) is None

"""rope_norm_qk under what else torch does with saved tensors: recomputed in a checkpointed region, and hooks that raise."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from adkv_amd.kernel import gemv


def _inputs(gpu, B=2, Hq=4, H=2, T=9, D=64):
    gen = torch.Generator(device=gpu).manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen, device=gpu)
    return [rand(B, Hq, T, D), rand(B, H, T, D), rand(1, T, D), rand(1, T, D), rand(D), rand(D)], (rand(B, Hq, T, D), rand(B, H, T, D))


def _leaves(t):
    return [x.clone().requires_grad_(i not in (2, 3)) for i, x in enumerate(t)]


@pytest.mark.gpu
@pytest.mark.parametrize("behind", [False, True])
def test_in_a_checkpointed_region(gpu, behind):
    """The recomputation ends with the last tensor that is saved, by an exception out of the saving."""
    t, grads = _inputs(gpu)

    def f(*x):
        q, k = gemv.rope_norm_qk(*x, 1e-6)
        return (torch.sin(q), torch.exp(k)) if behind else (q, k)
    results = []
    for call in (f, lambda *x: checkpoint(f, *x, use_reentrant=False), lambda *x: checkpoint(f, *x, use_reentrant=True)):
        x = _leaves(t)
        out = call(*x)
        torch.autograd.backward(out, grads)
        results.append([*out, *(x[i].grad for i in (0, 1, 4, 5))])
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], r))


@pytest.mark.gpu
def test_hooks_of_saved_tensors(gpu):
    t, grads = _inputs(gpu)
    seen = []

    def pack(x):
        seen.append(x.shape)
        return x.cpu()
    x = _leaves(t)
    out = gemv.rope_norm_qk(*x, 1e-6)
    torch.autograd.backward(out, grads)
    y = _leaves(t)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda c: c.to(gpu)):
        again = gemv.rope_norm_qk(*y, 1e-6)
    torch.autograd.backward(again, grads)
    assert len(seen) == 6 and all(torch.equal(a.grad, b.grad) for a, b in zip((x[i] for i in (0, 1, 4, 5)), (y[i] for i in (0, 1, 4, 5))))

    def refuse(x):
        raise KeyError("not this one")
    with torch.autograd.graph.saved_tensors_hooks(refuse, lambda c: c):
        with pytest.raises(KeyError, match="not this one"):
            gemv.rope_norm_qk(*_leaves(t), 1e-6)
    calls = []

    def once(x):      # an error is the call's, not a reason to try another way
        calls.append(1)
        raise KeyError("again")
    with torch.autograd.graph.saved_tensors_hooks(once, lambda c: c):
        with pytest.raises(KeyError):
            gemv.rope_norm_qk(*_leaves(t), 1e-6)
    assert len(calls) == 1

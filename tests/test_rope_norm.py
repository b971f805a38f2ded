"""RMS norms of the heads of queries and keys with the rotary embedding (``gemv.rope_norm_qk``), against the formula in 64 bits.

Rounding: a result is off by half a step of its type, and by what fp32 does before it.  With u = 2^-24: a row's sum of squares has terms rounded at most
30 times in a lane and its exchanges, halved by the root, which itself is off by 2u; norm, weight and rotation are five more operations: 24u of
|a cos| + |b sin|.  The way back rounds each of the two sums 40 times and does some 20 operations more: 64u of the terms' sizes.  A weight's gradient
is a sum whose terms pass at most 160 additions outside of a lane's own, which are no more than a quarter of the rows.
"""
import pytest
import torch

from adkv_amd import _lib
from adkv_amd.kernel import gemv

U = 2.0 ** -24
EPS = 1e-6
TYPES = (torch.float16, torch.bfloat16, torch.float32)


def make(B, Hq, H, T, D, R, dtype, seed=0, dev="cuda", shared_table=False, rows="heads last"):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *n: torch.randn(*n, generator=gen)
    s = {}
    for name, heads in (("q", Hq), ("k", H)):
        if rows == "heads last":      # a projection's [B, T, heads, D], seen with the head axis first
            x = (rand(B, T, heads, D) * torch.exp(rand(heads, 1))).to(dtype).to(dev).transpose(1, 2)
        else:
            x = (rand(B, heads, T, D) * torch.exp(rand(heads, 1, 1))).to(dtype).to(dev)
        s[name] = x
        s["w" + name] = (1 + 0.1 * rand(D)).to(dtype).to(dev)
        s["g" + name] = rand(B, heads, T, D).to(dtype).to(dev)
    angle = rand(1 if shared_table else B, T, R // 2) * 3
    angle = torch.cat([angle, angle], -1)
    s["cos"], s["sin"] = angle.cos().to(dtype).to(dev), angle.sin().to(dtype).to(dev)
    return s


def call(s, **kw):
    return gemv.rope_norm_qk(s["q"], s["k"], s["cos"], s["sin"], s["wq"], s["wk"], kw.get("eps", EPS))


def formula(x, w, cos, sin, eps=EPS):
    """The result in 64 bits and the sum of its terms' sizes."""
    x, w, c, s = x.double(), w.double(), cos.double()[:, None], sin.double()[:, None]
    R = c.shape[-1]
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    a, b, rest = y[..., :R // 2], y[..., R // 2:R], y[..., R:]
    other = torch.cat([-b, a], -1) * s
    own = torch.cat([a, b], -1) * c
    return torch.cat([own + other, rest], -1), torch.cat([own.abs() + other.abs(), rest.abs()], -1)


def gradients(x, w, cos, sin, g, eps=EPS):
    """dx and dw in 64 bits, each with what the roundings before the last may be relative to."""
    x, w = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    z, _ = formula(x, w, cos, sin, eps)
    dx, dw = torch.autograd.grad(z, (x, w), g.double())
    x, w, c, s, g = x.detach(), w.detach(), cos.double()[:, None], sin.double()[:, None], g.double()
    R = c.shape[-1]
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    turned = g[..., :R].abs() * c.abs() + (g[..., :R].abs() * s.abs()).roll(R // 2, -1)
    dy = torch.cat([turned, g[..., R:].abs()], -1)
    n = (x * r).abs()
    return dx, r * (dy * w.abs() + n * (dy * w.abs() * n).mean(-1, keepdim=True)), dw, (dy * n).sum((0, 1, 2))


def close(got, want, size, steps):
    info = torch.finfo(got.dtype)
    bound = want.abs() * info.eps / 2 + steps * U * size + info.tiny * info.eps
    assert torch.isfinite(got).all()
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1, worst


def check(s, eps=EPS):
    s = dict(s)
    for n in ("q", "k", "wq", "wk"):
        s[n] = s[n].detach().requires_grad_()
    z = call(s, eps=eps)
    got = torch.autograd.grad(z, (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
    for i, n in enumerate("qk"):
        x, w = s[n].detach(), s["w" + n].detach()
        assert z[i].shape == x.shape and z[i].is_contiguous()
        close(z[i].detach(), *formula(x, w, s["cos"], s["sin"], eps), 24)
        dx, dx_size, dw, dw_size = gradients(x, w, s["cos"], s["sin"], s["g" + n], eps)
        close(got[i], dx, dx_size, 64)
        close(got[2 + i], dw, dw_size, 160 + x.shape[0] * x.shape[1] * x.shape[2] / 4)
    return z, got


SIZES = [  # B, Hq, H, T, D, R
    (1, 1, 1, 1, 8, 8),
    (1, 2, 1, 3, 16, 8),
    (2, 4, 4, 5, 32, 16),
    (3, 5, 5, 33, 64, 32),
    (2, 8, 1, 17, 80, 80),
    (2, 3, 1, 19, 80, 40),
    (1, 9, 3, 31, 96, 48),
    (5, 32, 8, 1, 128, 128),
    (2, 6, 2, 129, 128, 64),
    (1, 4, 2, 70, 256, 256),
    (1, 3, 2, 9, 512, 256),
    (1, 2, 2, 6, 504, 496),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, dtype):
    check(make(*size, dtype, seed=sum(size)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_rows(dtype):
    """More items than workgroups: each takes several, four heads to a lane."""
    check(make(2, 7, 3, 1500, 128, 128, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32), ids=str)
@pytest.mark.parametrize("kind", ("slices", "heads first", "aligned to 4", "odd", "reversed heads", "one for all heads", "one table", "tables apart"))
def test_layouts(kind, dtype):
    s = make(2, 4, 2, 37, 64, 64, dtype, shared_table=kind == "one table", rows="heads first" if kind == "heads first" else "heads last")
    if kind == "slices":            # q and k of one projection
        both = torch.cat([s["q"].transpose(1, 2), s["k"].transpose(1, 2)], 2).contiguous()
        s["q"], s["k"] = both[:, :, :4].transpose(1, 2), both[:, :, 4:].transpose(1, 2)
    elif kind in ("aligned to 4", "odd"):
        for n in ("q", "k", "gq", "cos", "wk"):
            t, by = s[n].contiguous(), 4 if kind == "aligned to 4" else 3
            room = torch.empty(t.numel() + by, dtype=dtype, device="cuda")
            room[by:] = t.view(-1)
            s[n] = room[by:].view(t.shape)
    elif kind == "reversed heads":  # every second row of the gradient, too
        s["q"] = s["q"].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
        s["gq"] = s["gq"].repeat_interleave(2, 2)[:, :, ::2]
    elif kind == "one for all heads":
        s["q"] = s["q"][:, :1].expand(2, 4, 37, 64)
        s["gk"] = s["gk"][:, :, :1, :1].expand(2, 2, 37, 64)
    elif kind == "tables apart":
        s["sin"] = s["sin"].transpose(0, 1).contiguous().transpose(0, 1)
    check(s)


@pytest.mark.gpu
def test_gradients_are_laid_out_as_their_inputs():
    s = make(2, 4, 2, 5, 64, 64, torch.bfloat16)
    _, got = check(s)
    assert got[0].stride() == s["q"].stride() and got[1].stride() == s["k"].stride()


@pytest.mark.gpu
@pytest.mark.parametrize("eps", (0.0, 1e-6, 1.0))
def test_eps(eps):
    check(make(2, 2, 1, 11, 32, 32, torch.float32), eps)


@pytest.mark.gpu
def test_zero_rows():
    s = make(2, 2, 1, 4, 64, 64, torch.float16)
    s["q"][0, 1, 2] = 0
    z, got = check(s)
    assert (z[0][0, 1, 2] == 0).all()


@pytest.mark.gpu
def test_a_bad_row_is_alone():
    s = make(2, 3, 1, 6, 64, 64, torch.bfloat16)
    good, good_grad = check(s)
    for bad in (float("nan"), float("inf")):
        t = dict(s, q=s["q"].clone())
        t["q"][1, 1, 3, 5] = bad
        t["q"].requires_grad_()
        z = call(t)
        dq, = torch.autograd.grad(z[0], t["q"], s["gq"])
        for got, want in ((z[0], good[0]), (dq, good_grad[0])):
            same = got == want
            same[1, 1, 3] = True
            assert same.all() and got[1, 1, 3].isnan().any()


@pytest.mark.gpu
def test_only_what_is_wanted():
    s = make(2, 4, 2, 9, 64, 64, torch.bfloat16)
    _, whole = check(s)
    names = ("q", "k", "wq", "wk")
    for wanted in ((0,), (1,), (2,), (3,), (0, 3), (1, 2)):
        t = dict(s)
        for i in wanted:
            t[names[i]] = s[names[i]].detach().requires_grad_()
        z = call(t)
        got = torch.autograd.grad(z, [t[names[i]] for i in wanted], (s["gq"], s["gk"]))
        for g, i in zip(got, wanted):
            assert torch.equal(g, whole[i])
    # of one result only
    t = {n: v.detach().requires_grad_() if n in names else v for n, v in s.items()}
    got = torch.autograd.grad(call(t)[1], [t[n] for n in names], s["gk"], allow_unused=True)
    assert got[0] is None and got[2] is None and torch.equal(got[1], whole[1]) and torch.equal(got[3], whole[3])
    with torch.no_grad():
        assert not call(t)[0].requires_grad


@pytest.mark.gpu
def test_the_same_every_time():
    s = make(2, 8, 2, 700, 128, 128, torch.float32)
    first = check(s)
    again = check(s)
    assert all(torch.equal(a, b) for x, y in zip(first, again) for a, b in zip(x, y))


@pytest.mark.gpu
def test_one_weight_for_both():
    s = make(2, 4, 2, 9, 64, 64, torch.float32)
    w = s["wq"].detach().requires_grad_()
    z = gemv.rope_norm_qk(s["q"], s["k"], s["cos"], s["sin"], w, w, EPS)
    got, = torch.autograd.grad(z, w, (s["gq"], s["gk"]))
    parts = [gradients(s[n], s["wq"], s["cos"], s["sin"], s["g" + n])[2:] for n in "qk"]
    close(got, parts[0][0] + parts[1][0], parts[0][1] + parts[1][1], 161 + 2 * 4 * 9 / 4)


@pytest.mark.gpu
def test_differences():
    """The gradient along a direction d against (f(x + hd) - f(x - hd)) / 2h of the sum f of z * g, with every row of d as long as x's: the
    third derivative of a row's norm is at most 15 |z| then (1.1 of it within h), the rotation and the weights lengthen nothing by more
    than the largest weight, and each z is off by 24u of its terms.  The gradient's own rounding is 64u of its terms."""
    s = make(2, 3, 2, 7, 64, 32, torch.float32, seed=4)
    h = 1e-2
    for n, other in (("q", "k"), ("k", "q")):
        x, w, g = s[n].contiguous(), s["w" + n], s["g" + n].double()
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).cuda()
        d = d * x.norm(dim=-1, keepdim=True) / d.norm(dim=-1, keepdim=True)
        f = lambda x: (call(dict(s, **{n: x}))["qk".index(n)].double() * g).sum()
        lo, hi = (x - h * d), (x + h * d)
        step = (hi.double() - lo.double()) / (2 * h)       # what was really stepped
        got = (f(hi) - f(lo)) / (2 * h)
        t = dict(s, **{n: x.clone().requires_grad_()})
        dx, = torch.autograd.grad(call(t)["qk".index(n)], t[n], s["g" + n])
        want = (dx.double() * step).sum()
        _, size = formula(x, w, s["cos"], s["sin"])
        _, dx_size, _, _ = gradients(x, w, s["cos"], s["sin"], s["g" + n])
        third = 15 * 1.1 * (g.norm(dim=-1) * w.double().abs().max() * 64 ** 0.5).sum()
        bound = (g.abs() * size).sum() * 25 * U / h + h * h / 6 * third + (dx_size * step.abs()).sum() * 65 * U
        assert (got - want).abs() <= bound
        assert want.abs() > 4 * bound        # the bound says something


@pytest.mark.gpu
def test_captured_with_its_gradients():
    s = make(2, 4, 2, 65, 128, 128, torch.bfloat16)
    names = ("q", "k", "wq", "wk")
    leaves = {n: s[n].detach().clone().requires_grad_() for n in names}

    def step():
        z = call(dict(s, **leaves))
        return [*(t.detach() for t in z), *torch.autograd.grad(z, [leaves[n] for n in names], (s["gq"], s["gk"]))]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2, 3):
        new = make(2, 4, 2, 65, 128, 128, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for n in names:
                leaves[n].copy_(new[n])
            for n in ("gq", "gk", "cos", "sin"):
                s[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        held_now = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(held_now, step()))


@pytest.mark.gpu
def test_on_another_stream():
    s = make(2, 4, 2, 33, 64, 64, torch.float16)
    want, want_grad = check(s)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got, got_grad = check(s)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*want, *want_grad), (*got, *got_grad)))


@pytest.mark.gpu
@pytest.mark.parametrize("B,T", ((0, 3), (2, 0)))
def test_nothing(B, T):
    s = make(B, 2, 1, T, 32, 32, torch.float32)
    for n in ("q", "k", "wq", "wk"):
        s[n] = s[n].detach().requires_grad_()
    z = call(s)
    assert z[0].shape == (B, 2, T, 32) and z[1].shape == (B, 1, T, 32)
    got = torch.autograd.grad(z, (s["q"], s["wq"]), (s["gq"], s["gk"]))
    assert got[0].shape == s["q"].shape and (got[1] == 0).all()


def broken(**kw):
    s = make(2, 4, 2, 3, 32, 16, torch.float16, dev="cpu")
    for n, f in kw.items():
        s[n] = f(s[n])
    return s


@pytest.mark.parametrize("s,message", [
    (broken(q=lambda t: t[0]), "q, k must be"),
    (broken(k=lambda t: t[:1]), "disagree in shape"),
    (broken(k=lambda t: t[:, :, :2]), "disagree in shape"),
    (broken(q=lambda t: t.double()), "float16, bfloat16 or float32"),
    (broken(cos=lambda t: t.float()), "share one dtype"),
    (broken(wk=lambda t: t.float()), "share one dtype"),
    (broken(sin=lambda t: t[:, :2]), "cos, sin must be"),
    (broken(cos=lambda t: t[:, :2], sin=lambda t: t[:, :2]), "cos, sin must be"),
    (broken(cos=lambda t: t[..., :12], sin=lambda t: t[..., :12]), "multiple of 8 channels"),
    (broken(cos=lambda t: t.repeat(1, 1, 4), sin=lambda t: t.repeat(1, 1, 4)), "multiple of 8 channels"),
    (broken(q=lambda t: t[..., :20], k=lambda t: t[..., :20]), "head dim must be"),
    (broken(q=lambda t: t.repeat(1, 1, 1, 20), k=lambda t: t.repeat(1, 1, 1, 20)), "head dim must be"),
    (broken(wq=lambda t: t[:16]), "the weights must be"),
    (broken(k=lambda t: t[:, :0]), "must have heads"),
    (broken(cos=lambda t: t.clone().requires_grad_()), "have no gradient"),
    (broken(), "HIP device"),
], ids=lambda x: x if isinstance(x, str) else "")
def test_refusals(s, message):
    with pytest.raises(RuntimeError, match=message):
        call(s)


def test_c_refusals():
    """No refused call reaches the device: the pointers are only looked at."""
    C, lib = _lib.C, _lib.lib()
    p = 4096
    three = (C.c_int64 * 3)(64, 32, 32)

    def there(D=32, R=16, dtype=1, q=p, strides=three, B=1, T=1, out=p):
        return lib.adkv_rope_norm_qk(q, p, p, p, p, p, out, p, B, 1, 1, T, D, R, 1e-6, strides, three, three, dtype, None)

    def back(D=32, grad=p, dq=p, dwq=None, workspace=None, size=0, strides=three):
        return lib.adkv_rope_norm_qk_backward(grad, None, p, p, p, p, p, p, dq, None, dwq, None, 1, 1, 1, 1, D, 16, 1e-6, strides, None,
                                              three, None, three, None, three, 1, workspace, size, None)
    assert there(q=None) == -1 and there(out=None) == -1
    assert there(D=36) == -2 and there(D=520) == -2 and there(R=12) == -2 and there(R=40) == -2 and there(D=0) == -2
    assert there(B=0) == -3 and there(T=0) == -3 and there(B=1 << 20, T=1 << 11) == -3
    assert there(dtype=3) == -6
    assert there(q=p + 2) == -5 and there(strides=(C.c_int64 * 3)(64, 33, 32)) == -5
    assert back(grad=None) == -1 and back(strides=None) == -1 and back(D=36) == -2
    assert back(grad=p + 2) == -5
    assert back(dq=None) == 0
    assert lib.adkv_rope_norm_qk_backward_workspace_bytes(0) == -2 and lib.adkv_rope_norm_qk_backward_workspace_bytes(513) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_host_call_equals_the_python_function(monkeypatch, dtype):
    import types
    real = _lib.host()
    for size, kw in (((2, 4, 2, 37, 128, 64), {}), ((1, 3, 1, 5, 80, 80), {"rows": "heads first"}), ((3, 2, 2, 1, 64, 64), {"shared_table": True})):
        s = make(*size, dtype, **kw)
        got = real.rope_norm_qk(s["q"], s["k"], s["cos"], s["sin"], s["wq"], s["wk"], EPS)
        monkeypatch.setattr(_lib, "host", lambda: types.SimpleNamespace(rope_norm_qk=lambda *a: None))
        want = call(s)
        monkeypatch.undo()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # with gradients
        leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")]
        grads = []
        for taken in (True, False):
            if not taken:
                monkeypatch.setattr(_lib, "host", lambda: types.SimpleNamespace(rope_norm_qk=lambda *a: None))
            z = gemv.rope_norm_qk(leaves[0], leaves[1], s["cos"], s["sin"], leaves[2], leaves[3], EPS)
            assert ("_RopeNorm" in type(z[0].grad_fn).__name__) == (not taken)
            grads.append(torch.autograd.grad(z, leaves, (s["gq"], s["gk"].transpose(0, 2).contiguous().transpose(0, 2))))
            monkeypatch.undo()
        assert all(torch.equal(a, b) and a.stride() == b.stride() for a, b in zip(*grads))


@pytest.mark.gpu
@pytest.mark.parametrize("taken", (True, False))
def test_differentiated_once_only(monkeypatch, taken):
    import types
    if not taken:
        monkeypatch.setattr(_lib, "host", lambda: types.SimpleNamespace(rope_norm_qk=lambda *a: None))
    s = make(2, 3, 1, 6, 64, 64, torch.float32)
    s["q"] = s["q"].detach().requires_grad_()
    z = call(s)
    first, = torch.autograd.grad(z[0], s["q"], s["gq"].requires_grad_(), create_graph=True)
    plain, = torch.autograd.grad(call(s)[0], s["q"], s["gq"])
    assert torch.equal(first, plain)
    with pytest.raises(RuntimeError, match="once"):
        first.sum().backward()


@pytest.mark.gpu
def test_a_changed_input_is_noticed():
    s = make(2, 3, 1, 6, 64, 64, torch.float32)
    s["wq"].requires_grad_()
    z = call(s)
    s["q"] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(z[0], s["wq"], s["gq"])


@pytest.mark.gpu
def test_gradients_of_sums():
    """Gradients that are one number expanded to a result's shape, and ones of the other result that nobody asked for."""
    s = make(2, 4, 2, 9, 64, 64, torch.float32)
    s["q"], s["wq"] = s["q"].detach().requires_grad_(), s["wq"].detach().requires_grad_()
    call(s)[0].sum().backward()
    dx, size, dw, dw_size = gradients(s["q"], s["wq"], s["cos"], s["sin"], torch.ones_like(s["gq"]))
    close(s["q"].grad, dx, size, 64)
    close(s["wq"].grad, dw, dw_size, 160 + 2 * 4 * 9 / 4)


@pytest.mark.gpu
def test_forward_derivatives_are_refused():
    from torch.autograd import forward_ad
    s = make(1, 2, 1, 3, 32, 32, torch.float32)
    with forward_ad.dual_level():
        dual = dict(s, q=forward_ad.make_dual(s["q"], torch.ones_like(s["q"])))
        with pytest.raises(RuntimeError, match="forward derivatives"):
            call(dual)

"""gemv.token_logprobs against its formula in 64 bits: vocabularies around the steps of a workgroup, rows between two vectors, ties, rows that overrun the
list of candidates, infinities and what is no number, strides, graphs.

Tolerances: a lane adds at most n / 256 + 8 numbers one after the other and lanes and waves 10 more, each number being off by 2^-22 and by its exponent
times 2^-24: eps in all, relative, of the sum S beside the largest.  The entropy's second sum comes from numbers relative to a reference that is at
least the largest of the first 2048 logits (less one).  Beside that, a probability below 2^-126, fp32's smallest normal number, may be lost as a whole:
up to 2^18 of them, times a logit's distance of up to 2^11 in the entropy, make 2^-97."""
import math

import pytest
import torch

from adkv_amd.kernel import gemv

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def plain(logits, tokens, top):
    x = logits.detach().cpu().double().reshape(-1, logits.shape[-1])
    t = tokens.cpu().reshape(-1)
    M = x.amax(-1, keepdim=True)
    d = x - M
    e = torch.exp(d)
    at = torch.zeros_like(e, dtype=torch.bool).scatter_(1, x.argmax(-1, keepdim=True), True)
    S = e.masked_fill(at, 0.0).sum(-1, keepdim=True)
    T = torch.where(e > 0, e * d, 0.0).masked_fill(at, 0.0).sum(-1, keepdim=True)
    log1 = torch.log1p(S)
    bad = torch.isnan(x).any(-1) | (M[:, 0] == math.inf) | (M[:, 0] == -math.inf)
    log = (d - log1).masked_fill(bad[:, None], math.nan)
    ent = (log1 - T / (1 + S))[:, 0].masked_fill(bad, math.nan)
    n = x.shape[1]
    eps = (n / 256 + 18) * 2.0 ** -24 + 2.0 ** -22 + 200 * 2.0 ** -24 * 1.5
    share = (S / (1 + S)).nan_to_num(0.0)
    near = (M - x[:, :2048].amax(-1, keepdim=True)).nan_to_num(0.0, 0.0, 0.0) + 1
    off_log = eps * share + 2.0 ** -24 * log.nan_to_num(0.0, 0.0, 0.0).abs()
    off_ent = (2 * eps * (share + (T / (1 + S)).abs().nan_to_num(0.0) + near * share))[:, 0] + 2.0 ** -24 * ent.nan_to_num(0.0).abs()
    given = t.clamp(0, n - 1)[:, None]
    p = torch.where(t < 0, 0.0, torch.where(t < n, log.gather(1, given)[:, 0], math.nan))
    order = torch.sort(x + 0.0, dim=-1, descending=True, stable=True)[1][:, :top]
    return p, off_log.gather(1, given)[:, 0], ent, off_ent, log.gather(1, order), off_log.gather(1, order), order


def near(got, want, off):
    got, want = got.cpu().double().reshape(want.shape), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    kind = torch.isfinite(want)
    assert torch.equal(got[~kind & ~torch.isnan(want)], want[~kind & ~torch.isnan(want)])
    d = (got - want)[kind].abs() - 1.05 * off[kind] - 2.0 ** -97
    assert d.numel() == 0 or d.max() <= 0, f"off by {float((got - want)[kind].abs().max()):.3e}, {float(d.max()):.3e} more than may be"


def check(logits, tokens, top):
    got = gemv.token_logprobs(logits, tokens, top=top)
    p, off_p, ent, off_ent, tp, off_tp, order = plain(logits, tokens, top)
    assert got.logprobs.shape == got.entropy.shape == tokens.shape and got.logprobs.dtype == torch.float32
    near(got.logprobs, p, off_p)
    near(got.entropy, ent, off_ent)
    if top:
        assert got.top_tokens.shape == (*tokens.shape, top) and got.top_tokens.dtype == torch.int64
        assert torch.equal(got.top_tokens.cpu().reshape(order.shape), order)
        near(got.top_logprobs, tp, off_tp)
    else:
        assert got.top_tokens is None and got.top_logprobs is None
    return got


def logits_of(N, V, dtype, dev, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, V, generator=g) * spread
    x.scatter_add_(1, torch.randint(0, V, (N, 3), generator=g), torch.full((N, 3), 9.0))
    return x.to(dtype).to(dev), torch.randint(0, V, (N,), generator=g).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (2, 8, 3), (5, 9, 9), (4, 33, 32), (2, 255, 32), (3, 256, 1), (3, 257, 20), (2, 1000, 32), (3, 2047, 5), (2, 4097, 8),
                                     (2, 16385, 20), (3, 32000, 8), (2, 50001, 32), (1, 131073, 20), (1300, 100, 4), (1200, 5000, 32), (1030, 9001, 0)])
def test_sizes(gpu, N, V, top, dtype):
    check(*logits_of(N, V, dtype, gpu), top)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [2, 1100])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
def test_rows_of_all_kinds(gpu, dtype, N):
    """Equal logits, ascending and descending ones (the list of candidates is overrun), one that is certain, a few infinities, zeros of both signs, lowest values."""
    V = 20000
    low = torch.finfo(dtype).min
    base, tokens = logits_of(16, V, torch.float32, "cpu", 1)
    rows = [base[0] * 0, torch.arange(V) * 1e-3, torch.arange(V).flip(0) * 1e-3, base[1], base[2], base[3], base[4].masked_fill(base[4] < 2, -math.inf), base[5] * 0 - 0.0,
            base[6].masked_fill(torch.arange(V) != 17, low), torch.full((V,), low), base[7].masked_fill(torch.arange(V) % 3 > 0, low), base[8] * 100, base[9] - 3e4, base[10] * 1e-6,
            torch.where(torch.arange(V) == V - 1, 0.0, -math.inf), base[11] + torch.arange(V) * 2e-3]
    rows[3][100] = 60.0
    rows[4][V - 1] = 25.0
    rows[5][:3] = rows[5].max()
    rows[7][::2] = 0.0
    x = torch.stack(rows).to(dtype)
    tokens[3], tokens[4], tokens[8], tokens[14] = 100, V - 1, 17, V - 1
    many = -(-N // 16) if N > 16 else 1
    x, tokens = x.repeat(many, 1).to(gpu), tokens.repeat(many).to(gpu)
    check(x, tokens, 20)
    check(x, tokens, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
def test_infinities_and_what_is_no_number(gpu, dtype):
    V = 3001
    x, tokens = logits_of(8, V, dtype, gpu, 2)
    x[0] = -math.inf
    x[1, 5] = math.nan
    x[2, V - 1] = math.inf
    x[3, 7], x[3, 9] = math.nan, math.inf
    x[4, :V - 1] = -math.inf
    x[5, 0] = math.nan
    x[6, ::2] = -math.inf
    for top in (0, 5):
        got = check(x, tokens, top)
        assert torch.isnan(got.logprobs[:4]).all() and torch.isfinite(got.entropy[[4, 6, 7]]).all()
    assert got.entropy[4] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["front", "behind", "every other", "all", "all but one"])
@pytest.mark.parametrize("value", [-1e4, -5e5, -1e6, -1e9, -1e10, -1e12, -1e20, -1e30, -8e37, -2e38, 4e5, 6e5, 1e6, 1e12, 1e38])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_logits_far_from_the_others(gpu, dtype, value, where):
    """Hidden tokens, in front of the others too; rows of nothing else; large ones.  They are next to others or far beyond what e^x tells from nothing."""
    for N, V, top in ((3, 100, 3), (3, 32000, 0), (2, 32000, 20), (1100, 3001, 0)):
        x, tokens = logits_of(N, V, dtype, gpu, 4)
        at = torch.arange(V, device=gpu)
        x[:, {"front": at < V * 2 // 3, "behind": at > V // 3, "every other": at % 2 == 0, "all": at >= 0, "all but one": at != V // 2}[where]] = value
        tokens[0] = V // 2
        got = check(x, tokens, top)
        assert torch.isfinite(got.logprobs).all()
        # beside check(), which allows for references far from the largest: those that are hidden are none, so that they are within 2^60 of it
        ent, (log, S, T) = got.entropy.cpu().double(), sums_of(x)
        eps, share = (V / 256 + 18) * 2.0 ** -24 + 2.0 ** -22 + 300 * 2.0 ** -24, S / (1 + S)
        want = log - T / (1 + S)
        assert ((ent - want).abs() <= 2 * eps * (62 * share + (T / (1 + S)).abs()) + 2.0 ** -24 * want.abs() + 2.0 ** -97).all()


def sums_of(x):
    """log(1 + S), S and T of the formula, without the first of the largest."""
    x = x.cpu().double()
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d).scatter_(1, x.argmax(-1, keepdim=True), 0.0)
    return torch.log1p(e.sum(-1)), e.sum(-1), torch.where(e > 0, e * d, 0.0).sum(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [400, 1600])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
def test_unlikely_tokens_beside_less_likely_ones(gpu, dtype, N):
    """What a lane begins with is e^-36 of others that it sees, which are e^-64 of the row's largest: they are all that the largest's log probability is made of."""
    for V, top in ((45, 0), (45, 3), (40001, 0)):
        g = torch.Generator().manual_seed(V)
        x = torch.full((N, V), -100.0)
        x[torch.rand(N, V, generator=g) < 0.3] = -64.0
        tokens = torch.randint(0, V, (N,), generator=g)
        x[torch.arange(N), tokens] = 0.0
        got = check(x.to(dtype).to(gpu), tokens.to(gpu), top)
        want = -(x == -64).sum(-1) * math.exp(-64) - (x == -100).sum(-1) * math.exp(-100)
        assert ((got.logprobs.cpu().double() - want).abs() <= 2e-5 * want.abs()).all()


@pytest.mark.gpu
def test_nearly_certain_tokens_keep_their_digits_far_from_zero(gpu):
    """Logits around a million, in steps of 2^-4."""
    x = torch.full((8, 5000), 1e6 - 20.0, device=gpu)
    x[:, 77] = 1e6 - 4 + torch.arange(8, device=gpu) * 2.0
    got = check(x, torch.full((8,), 77, device=gpu), 2)
    want = -torch.log1p(4999 * torch.exp(-20 - (x[:, 77].double() - 1e6)))
    assert ((got.logprobs.double() - want).abs() <= 1e-5 * want.abs()).all()


@pytest.mark.gpu
def test_nearly_certain_tokens_keep_their_digits(gpu):
    x = torch.full((40, 5000), -20.0, device=gpu)
    x[:, 77] = torch.linspace(-10, 60, 40, device=gpu)
    tokens = torch.full((40,), 77, device=gpu)
    got = check(x, tokens, 2)
    want = -torch.log1p(4999 * torch.exp(-20 - x[:, 77].double()))
    assert ((got.logprobs.double() - want).abs() <= 1e-5 * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
def test_layouts(gpu, dtype):
    """All but the last position of a batch, every other row, rows that begin between two vectors, columns that are not contiguous, a vector of logits."""
    x, tokens = logits_of(24, 999, dtype, gpu, 3)
    x, tokens = x.view(4, 6, 999), tokens.view(4, 6)
    check(x[:, :-1], tokens[:, 1:], 3)
    check(x.transpose(0, 1), tokens.t(), 3)
    check(x[::2, ::3], tokens[::2, ::3], 3)
    check(x[:, :, 1:], tokens - 1, 3)
    check(x[:, :, :700], tokens, 3)
    check(x.transpose(1, 2).contiguous().transpose(1, 2), tokens, 3)
    check(x[0, 0], tokens[0, 0], 3)
    check(x.view(2, 2, 6, 999), tokens.view(2, 2, 6), 3)
    check(x[:1].expand(5, 6, 999), tokens[:1].expand(5, 6), 3)
    check(x, tokens.to(torch.int32), 3)
    for shift in range(1, 16 // x.element_size()):
        flat = torch.empty(24 * 999 + shift, dtype=dtype, device=gpu)[shift:]
        check(flat.view(x.shape).copy_(x), tokens, 3)


@pytest.mark.gpu
def test_tokens_that_are_none(gpu):
    x, _ = logits_of(4, 100, torch.float32, gpu, 4)
    got = check(x, torch.tensor([-1, -100, 100, 99], device=gpu), 0)
    assert got.logprobs[:2].tolist() == [0.0, 0.0] and torch.isnan(got.logprobs[2])


@pytest.mark.gpu
def test_nothing_to_do(gpu):
    got = gemv.token_logprobs(torch.zeros(0, 5, device=gpu), torch.zeros(0, dtype=torch.int64, device=gpu), top=2)
    assert got.logprobs.shape == (0,) and got.top_tokens.shape == (0, 2)


@pytest.mark.gpu
def test_a_graph_and_another_stream(gpu):
    made = [logits_of(9, 7001, torch.bfloat16, gpu, s) for s in range(3)]
    want = [gemv.token_logprobs(*m, top=9) for m in made]
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gemv.token_logprobs(*made[0], top=9)
    side.synchronize()
    assert same(got, want[0])
    x, t = (v.clone() for v in made[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gemv.token_logprobs(x, t, top=9)
    for i in (1, 2, 0, 1):
        x.copy_(made[i][0])
        t.copy_(made[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want[i])
        assert same(gemv.token_logprobs(*made[i], top=9), want[i])


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu):
    x = torch.zeros(3, 2 ** 30 + 64, dtype=torch.float16, device=gpu)[:, 40:1040]       # rows 2 GiB apart
    g = torch.Generator(device=gpu).manual_seed(5)
    x.copy_(torch.randn(3, 1000, generator=g, device=gpu))
    check(x, torch.tensor([5, 6, 7], device=gpu), 4)


def test_refusals():
    x, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    for args, top, message in [((x, t[:2]), 0, "shape"), ((x.double(), t), 0, "float16"), ((x, t.float()), 0, "whole numbers"), ((x, t > 0), 0, "whole numbers"), ((x[:, :0], t), 0, "one column"),
                               ((x, t), 11, "top"), ((x, t), -1, "top"), ((torch.zeros(3, 100), t), 33, "top"), ((x.clone().requires_grad_(), t), 0, "no gradient"), ((x, t), 0, "device")]:
        with pytest.raises(RuntimeError, match=message):
            gemv.token_logprobs(*args, top=top)


def test_the_library_refuses_what_it_cannot_take():
    from adkv_amd import _lib
    L = _lib.lib()
    good = dict(x=4096, s0=0, s1=100, tokens=4096, n0=1, n1=4, V=100, dtype=0, top=5, p=4096, e=4096, tp=4096, tt=4096, stream=None)
    for change, code in [(dict(x=None), -1), (dict(tokens=None), -1), (dict(p=None), -1), (dict(tp=None), -1), (dict(n0=0), -3), (dict(n1=-1), -3), (dict(V=0), -3), (dict(top=33), -3),
                         (dict(top=5, V=4), -3), (dict(s1=-1), -3), (dict(V=2 ** 31 - 1), -3), (dict(n0=2 ** 15, n1=2 ** 15), -3), (dict(dtype=3), -6), (dict(x=4098), -5), (dict(tokens=4100), -5),
                         (dict(tt=4100), -5), (dict(x=4097, dtype=1), -5)]:
        assert L.adkv_token_logprobs(*{**good, **change}.values()) == code, change

"""gemv.prompt_attention against its formula in 64 bits: sizes around tiles and waves, the kernel's forms, packed sequences, masks, strides,
numbers that are none in hidden places, streams and graphs.

Tolerances: with u half a step of the type, a weight is off by u from its rounding and by the error of its score, which is a sum of D products in
fp32 (at most D + 8 roundings of the sum of the magnitudes), both in the numerator and in the sum that divides; the output is rounded once more.  fp16 weights
below the normal range are off by up to 2^-25 each, relative to a largest one of at least 2^7."""
import math

import pytest
import torch

from adkv_amd.kernel import gemv

F16, BF16 = torch.float16, torch.bfloat16


def shown(Tq, Tk, mask, b, hq):
    """(which keys a head's rows look at, what is added to their scores), [Tq, Tk]."""
    see = torch.arange(Tk)[None, :] <= torch.arange(Tk - Tq, Tk)[:, None]
    add = torch.zeros(Tq, Tk, dtype=torch.float64)
    if mask is not None:
        m = mask[min(b, mask.shape[0] - 1), min(hq, mask.shape[1] - 1)].cpu().expand(Tq, Tk)
        if m.dtype == torch.bool:
            see = see & m
        else:
            see, add = see & (m != -math.inf), m.double()
    return see, add


def plain(q, k, v, scaling, mask=None, bounds=None):
    """(out [B, Tq, Hq, D], how far off it may be) in 64 bits; hidden keys and values are not touched."""
    q, k, v = (t.detach().cpu() for t in (q, k, v))
    B, Hq, Tq, D = q.shape
    H, Tk = k.shape[1:3]
    u = torch.finfo(q.dtype).eps / 2
    out, off = torch.zeros(B, Tq, Hq, D, dtype=torch.float64), torch.zeros(B, Tq, Hq, D, dtype=torch.float64)
    spans = [(0, Tq, 0, Tk)] if bounds is None else [(x, y, x, y) for x, y in zip(bounds.tolist(), bounds.tolist()[1:])]
    for b in range(B):
        for hq in range(Hq):
            for q0, q1, k0, k1 in spans:
                if q1 == q0:
                    continue
                see, add = shown(q1 - q0, k1 - k0, mask, b, hq)
                x, kd, vd = q[b, hq, q0:q1].double(), k[b, hq // (Hq // H), k0:k1].double(), v[b, hq // (Hq // H), k0:k1].double()
                any_of = see.any(0)                     # what nobody looks at
                kd, vd = kd.masked_fill(~any_of[:, None], 0.0), vd.masked_fill(~any_of[:, None], 0.0)
                s = (x @ kd.t() * scaling + add).masked_fill(~see, -math.inf)
                top = s.amax(-1, keepdim=True)
                w = torch.exp(s - top.nan_to_num(neginf=0.0, nan=0.0)).masked_fill(~see, 0.0)
                total = w.sum(-1, keepdim=True)
                fine = torch.where(torch.isfinite(vd), vd, torch.zeros_like(vd))
                o = w @ fine / total
                for t in torch.nonzero(~torch.isfinite(vd).all(-1)).flatten().tolist():       # one that is looked at makes the row's channel what it is
                    rows = see[:, t]
                    o[rows] = o[rows] + w[rows, t:t + 1] / total[rows] * vd[t] - w[rows, t:t + 1] / total[rows] * fine[t]
                o = torch.where(see.any(-1, keepdim=True), o, torch.zeros_like(o))
                size = (x.abs() @ kd.abs().t() * abs(scaling) + add.abs().clamp(max=1e5)).masked_fill(~see, 0.0).nan_to_num(0.0, 0.0, 0.0)
                err = u + (D + 8) * 2.0 ** -24 * size + 2.0 ** -22
                spread = w * err
                e = (spread @ fine.abs() + spread.sum(-1, keepdim=True) * o.abs()) / total + u * o.abs()
                e = e + (see.sum(-1, keepdim=True) * 2.0 ** -32 * fine.abs().max() if q.dtype == F16 else 0.0) + torch.finfo(q.dtype).smallest_normal * 2.0 ** -8
                out[b, q0:q1, hq], off[b, q0:q1, hq] = o, 1.05 * e.nan_to_num(0.0)
    return out, off


def check(got, want, off):
    got = got.cpu().double()
    assert got.shape == want.shape
    kind = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "not a number elsewhere than in the formula"
    assert torch.equal(got[~kind & ~torch.isnan(want)], want[~kind & ~torch.isnan(want)])
    d = (got - want)[kind].abs() - off[kind]
    assert d.numel() == 0 or d.max() <= 0, f"off by {float((got - want)[kind].abs().max()):.3e}, {float(d.max()):.3e} more than may be"


def rows(B, heads, T, D, dtype, dev, seed=0, amount=1.0):
    """A projection [B, T, heads, D] seen with the head axis first."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, T, heads, D, generator=g) * amount).to(dtype).to(dev).transpose(1, 2)


def qkv(B, H, g, Tq, Tk, D, dtype, dev, seed=0):
    return rows(B, H * g, Tq, D, dtype, dev, seed, 1.5), rows(B, H, Tk, D, dtype, dev, seed + 1, 1.5), rows(B, H, Tk, D, dtype, dev, seed + 2)


SIZES = [  # B, H, g, Tq, Tk, D
    (1, 1, 1, 1, 1, 128), (1, 1, 1, 2, 2, 64), (2, 1, 1, 31, 31, 128), (1, 2, 1, 32, 32, 128), (1, 1, 3, 33, 33, 128), (1, 2, 2, 63, 64, 128),
    (1, 1, 1, 65, 65, 256), (1, 2, 5, 13, 129, 80), (3, 1, 8, 1, 300, 128), (1, 1, 1, 160, 160, 96), (1, 1, 4, 40, 1000, 64), (2, 1, 7, 5, 257, 136),
    (1, 1, 1, 1, 5000, 128), (1, 1, 1, 3, 4100, 256), (1, 1, 2, 70, 70, 8), (1, 1, 1, 129, 500, 248),
]
MANY = [(8, 32, 1, 130, 130, 128), (9, 32, 1, 31, 64, 64), (4, 16, 4, 65, 65, 128), (2, 20, 7, 129, 200, 72), (33, 8, 1, 127, 127, 256), (65, 4, 3, 50, 63, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("size", SIZES + MANY, ids=str)
def test_sizes(gpu, size, dtype):
    B, H, g, Tq, Tk, D = size
    q, k, v = qkv(*size, dtype, gpu)
    check(gemv.prompt_attention(q, k, v, D ** -0.5), *plain(q, k, v, D ** -0.5))


# For as many rows as keep the device busy with 128 at a time, with 64 and with 32
FORMS = [(40, 8, 1, 130, 131, 64), (20, 16, 1, 70, 200, 80), (20, 16, 1, 129, 129, 128), (64, 9, 1, 40, 65, 256),
         (2, 8, 1, 1100, 1100, 64), (1, 8, 1, 1101, 1101, 96), (1, 8, 4, 300, 2000, 128),
         (2, 4, 2, 300, 301, 64), (1, 3, 2, 200, 900, 88), (1, 4, 1, 515, 515, 128), (1, 2, 4, 100, 400, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "bool", "bool_heads", "bias", "fp16", "bf16", "fp64", "inf"])
@pytest.mark.parametrize("size", FORMS, ids=str)
def test_forms(gpu, size, kind):
    B, H, g, Tq, Tk, D = size
    dtype = BF16 if kind == "bf16" else F16
    q, k, v = qkv(*size, dtype, gpu)
    m = None if kind == "none" else masks(kind, B, H * g, Tq, Tk, gpu)
    got = gemv.prompt_attention(q, k, v, D ** -0.5, m)
    picks = sorted({0, B // 2, B - 1})          # sequences; the formula takes its time
    of = lambda t: t if t is None or t.shape[0] == 1 else t[picks]
    check(got[picks], *plain(of(q) if B > 1 else q, of(k), of(v), D ** -0.5, of(m)))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "bool", "inf"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("size", [(40, 8, 1, 100, 131, 64), (20, 16, 1, 129, 129, 96), (2, 8, 1, 1100, 1100, 64), (1, 8, 1, 1101, 1101, 128), (1, 4, 1, 200, 515, 128)], ids=str)
def test_forms_with_numbers_that_are_none_behind_a_row(gpu, size, bad, kind):
    B, H, g, Tq, Tk, D = size
    q, k, v = qkv(*size, F16, gpu)
    at = Tk - 20
    m = None if kind == "none" else masks(kind, B, H * g, Tq, Tk, gpu)
    v[:, :, at, 5] = bad
    k[:, :, at + 1:] = math.nan
    got = gemv.prompt_attention(q, k, v, D ** -0.5, m)
    n = Tq - 19          # rows that do not look at what is no key
    pick = slice(B - 1, B)
    m = m if m is None else m[pick, :, :n, :at + 1]
    check(got[pick, :n], *plain(q[pick, :, :n], k[pick, :, :at + 1], v[pick, :, :at + 1], D ** -0.5, m))


@pytest.mark.gpu
@pytest.mark.parametrize("H,g,D,ends", [(8, 1, 128, [0, 700, 701, 1100]), (16, 1, 64, [3, 500, 700, 1090]), (3, 2, 96, [0, 100, 333, 350])], ids=str)
def test_forms_of_packed_sequences(gpu, H, g, D, ends):
    T = ends[-1] + 3
    q, k, v = qkv(1, H, g, T, T, D, F16, gpu)
    bounds = torch.tensor(ends, dtype=torch.int32)
    got = gemv.prompt_attention(q, k, v, D ** -0.5, bounds=bounds.to(gpu))
    check(got, *plain(q, k, v, D ** -0.5, bounds=bounds))
    assert not got[:, ends[-1]:].any() and not got[:, :ends[0]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [-0.3, 0.0, 2.0])
def test_scalings(gpu, scaling):
    q, k, v = qkv(1, 2, 2, 70, 90, 64, F16, gpu)
    check(gemv.prompt_attention(q, k, v, scaling), *plain(q, k, v, scaling))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_scores_that_grow_along_the_row_and_large_ones(gpu, dtype):
    """The reference of the weights is replaced again and again, and by a lot."""
    q, k, v = qkv(1, 1, 1, 200, 200, 64, dtype, gpu)
    ramp = torch.linspace(0.1, 40.0, 200, device=gpu).to(dtype)[:, None]
    k = (q.abs().mean() * 0 + ramp * torch.ones(1, 1, 1, 64, dtype=dtype, device=gpu)).to(dtype) + k * 0.1
    q = q.abs()
    check(gemv.prompt_attention(q, k, v, 0.5), *plain(q, k, v, 0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "bool_keys", "some"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("size", [(20, 16, 1, 129, 129, 128), (2, 8, 1, 1101, 1101, 96), (1, 4, 2, 300, 301, 64), (1, 2, 1, 260, 300, 256), (1, 1, 4, 3, 1500, 128)], ids=str)
def test_scores_of_ten_digits(gpu, size, dtype, kind):
    """A step of such a score in 32 bits is more than e^x has room for.  Scores are at least 2^-8 of themselves apart, 250 and more, and off by 2^-16, so that a row's output is
    the value of its largest one, which the products of 11 bits leave as it is."""
    B, H, g, Tq, Tk, D = size
    r = torch.Generator().manual_seed(7)
    order = torch.randperm(Tk, generator=r)
    k = (0x4780 - Tk + order).to(torch.int16).view(BF16).to(dtype).to(gpu)[None, None, :, None].expand(B, H, Tk, D)       # bfloat16's numbers up to 65280
    v = rows(B, H, Tk, D, dtype, gpu, 2)
    at = order.cummax(0)[1][Tk - Tq:].to(gpu)
    m = {"none": None, "bool_keys": torch.ones(B, 1, 1, Tk, dtype=torch.bool, device=gpu), "some": torch.zeros(1, 1, Tq, Tk, dtype=dtype, device=gpu)}[kind]
    if kind == "some":
        m[..., ::2] = -1.0
    for amount in (1e3, 3e4):
        q = (torch.rand(B, H * g, Tq, 1, generator=r) + 1).mul(amount).to(dtype).to(gpu).expand(B, H * g, Tq, D)
        got = gemv.prompt_attention(q, k, v, 1.0, m)
        assert torch.equal(got, v[:, :, at].repeat_interleave(g, 1).transpose(1, 2)), amount


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("H,g,ends", [(1, 1, [0, 1]), (2, 3, [0, 5, 5, 70, 133]), (1, 1, [0, 0, 0, 64]), (2, 1, [3, 40, 40, 99]), (1, 4, [0]),
                                      (16, 1, [0, 300, 301, 303, 700]), (8, 4, [0, 31, 63, 64, 65, 400, 500, 500]), (1, 1, [0, *range(1, 150)]), (40, 1, [*range(0, 9000, 60)])],
                         ids=str)
def test_packed_sequences(gpu, H, g, ends, dtype):
    if len(ends) > 100 and dtype == BF16:
        ends = ends[:80]
    T = ends[-1] + 7
    q, k, v = qkv(1, H, g, T, T, 64, dtype, gpu)
    bounds = torch.tensor(ends, dtype=torch.int32)
    got = gemv.prompt_attention(q, k, v, 0.125, bounds=bounds.to(gpu))
    check(got, *plain(q, k, v, 0.125, bounds=bounds))
    assert not got[:, ends[-1]:].any() and not got[:, :ends[0]].any()
    assert torch.equal(got, gemv.prompt_attention(q, k, v, 0.125, bounds=bounds.long()))      # from the host


@pytest.mark.gpu
def test_a_packed_sequence_is_what_it_is_by_itself(gpu):
    q, k, v = qkv(1, 8, 4, 600, 600, 128, BF16, gpu)
    ends = [0, 129, 130, 600]
    got = gemv.prompt_attention(q, k, v, 0.1, bounds=torch.tensor(ends, dtype=torch.int32, device=gpu))
    for x, y in zip(ends, ends[1:]):
        check(got[:, x:y], *plain(q[:, :, x:y], k[:, :, x:y], v[:, :, x:y], 0.1))


@pytest.mark.gpu
def test_what_lies_outside_a_packed_sequence_does_not_matter(gpu):
    q, k, v = qkv(1, 2, 2, 200, 200, 64, F16, gpu)
    bounds = torch.tensor([0, 77, 150], dtype=torch.int32, device=gpu)
    want = gemv.prompt_attention(q, k, v, 0.125, bounds=bounds)
    k, v = k.clone(), v.clone()
    for t in (k, v):
        t[:, :, 150:] = math.nan
    assert torch.equal(want, gemv.prompt_attention(q, k, v, 0.125, bounds=bounds))
    for t in (k, v):
        t[:, :, 77:150] = math.inf
    assert torch.equal(want[:, :77], gemv.prompt_attention(q, k, v, 0.125, bounds=bounds)[:, :77])


@pytest.mark.gpu
def test_bounds_that_are_none_touch_nothing_else(gpu):
    """Values outside the rows, descending ones: the rows' results mean nothing, and nothing else is read or written."""
    q, k, v = qkv(1, 2, 1, 100, 100, 64, F16, gpu)
    for e in ([-5, 1 << 30], [50, 20, 90], [100, 0], [2 ** 31 - 1, -2 ** 31]):
        out = gemv.prompt_attention(q, k, v, 0.125, bounds=torch.tensor(e, dtype=torch.int32, device=gpu))
        torch.cuda.synchronize()
        assert out.shape == (1, 100, 2, 64)


def masks(kind, B, Hq, Tq, Tk, dev):
    g = torch.Generator().manual_seed(5)
    late = torch.arange(Tk)[None, :] > torch.arange(Tk - Tq, Tk)[:, None]
    pad = torch.arange(Tk)[None, :] < torch.randint(0, Tk, (B, 1), generator=g)
    hide = pad[:, None, None, :] | late
    if kind == "bool":
        return (~hide).to(dev)
    if kind == "bool_heads":
        return (torch.rand(B, Hq, Tq, Tk, generator=g) < 0.3).to(dev)
    if kind == "bool_keys":
        return (~pad[:, None, None, :]).to(dev)
    if kind == "bias":
        return torch.randn(1, Hq, Tq, Tk, generator=g).to(dev)
    dtype, value = {"fp16": (F16, None), "bf16": (BF16, None), "fp32": (torch.float32, None), "fp64": (torch.float64, -math.inf), "inf": (F16, -math.inf)}[kind]
    m = torch.zeros(B, 1, Tq, Tk, dtype=dtype).masked_fill_(hide, torch.finfo(dtype).min if value is None else value)
    if kind == "bf16":        # rows that begin between two words
        wide = torch.zeros(B, 1, Tq, Tk + 3, dtype=dtype)
        wide[..., 1:Tk + 1] = m
        return wide.to(dev)[..., 1:Tk + 1]
    return m.to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bool", "bool_heads", "bool_keys", "bias", "fp16", "bf16", "fp32", "fp64", "inf"])
@pytest.mark.parametrize("size", [(2, 2, 2, 70, 70, 64), (3, 1, 3, 33, 101, 128), (2, 1, 1, 1, 515, 64), (5, 32, 2, 65, 65, 64), (2, 2, 1, 40, 77, 256)], ids=str)
def test_masks(gpu, size, kind):
    """Left-padded batches (rows in front of the first token look at nothing, or at everything alike where the mask is additive), heads of their own."""
    B, H, g, Tq, Tk, D = size
    dtype = BF16 if kind == "bf16" else F16
    q, k, v = qkv(*size, dtype, gpu)
    m = masks(kind, B, H * g, Tq, Tk, gpu)
    check(gemv.prompt_attention(q, k, v, D ** -0.5, m), *plain(q, k, v, D ** -0.5, m))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("size", [(1, 2, 1, 100, 100, 64), (10, 32, 1, 100, 100, 64), (1, 1, 4, 9, 333, 128), (1, 1, 2, 50, 70, 256)], ids=str)
def test_later_tokens_leave_nothing_behind(gpu, size, bad, dtype):
    """Whatever a token's key and value hold, rows in front of it do not know; rows behind it are what the formula makes of it."""
    B, H, g, Tq, Tk, D = size
    q, k, v = qkv(*size, dtype, gpu)
    at = Tk - max(Tq // 2, 2)
    v[:, :, at, 3] = bad
    got = gemv.prompt_attention(q, k, v, D ** -0.5)
    check(got[:1], *plain(q[:1], k[:1], v[:1], D ** -0.5))
    k[:, :, at + 1:] = bad
    first = Tq - (Tk - at)          # queries in front of the bad value
    check(gemv.prompt_attention(q, k, v, D ** -0.5)[:1, :first], *plain(q[:1, :, :first], k[:1, :, :at], v[:1, :, :at], D ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bool", "inf"])
def test_masked_tokens_leave_nothing_behind(gpu, kind):
    q, k, v = qkv(3, 2, 2, 60, 60, 64, F16, gpu)
    m = masks(kind, 3, 4, 60, 60, gpu)
    want = gemv.prompt_attention(q, k, v, 0.125, m)
    hidden = ~m[:, 0, -1] if kind == "bool" else m[:, 0, -1] == -math.inf
    assert hidden.any()
    for bad in (math.nan, math.inf):
        kb, vb = (t.masked_fill(hidden[:, None, :, None], bad) for t in (k, v))
        got = gemv.prompt_attention(q, kb, vb, 0.125, m)
        check(got, *plain(q, kb, vb, 0.125, m))
        off = plain(q, k, v, 0.125, m)[1]
        assert ((got - want).cpu().double().abs() <= 2 * off).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,value", [(d, x) for d in (F16, BF16, torch.float32) for x in (-10000.0, -1e9, 3.0, -6.5, "lowest", -math.inf) if d != F16 or x != -1e9],
                         ids=lambda x: str(x).replace("torch.", ""))
@pytest.mark.parametrize("size", [(20, 16, 1, 129, 300, 128), (2, 8, 1, 1100, 1100, 64), (2, 4, 2, 100, 401, 64)], ids=str)
def test_the_same_added_to_many_keys(gpu, size, dtype, value):
    """Whole tiles of it, at the edge of one and from one head to the next; every row looks at a key that it is not added to."""
    B, H, g, Tq, Tk, D = size
    q, k, v = qkv(*size, F16 if dtype == torch.float32 else dtype, gpu)
    m = torch.zeros(B, 1, 1, Tk, dtype=dtype, device=gpu).expand(B, 1, Tq, Tk).contiguous()
    value = torch.finfo(dtype).min if value == "lowest" else value
    m[0, :, :, 64:192] = value
    m[B - 1, :, :, 50:290] = value
    m[B - 1, :, Tq // 2:, 130] = 1.0
    got = gemv.prompt_attention(q, k, v, D ** -0.5, m)
    pick = [0, B - 1]
    check(got[pick], *plain(q[pick], k[pick], v[pick], D ** -0.5, m[pick]))


@pytest.mark.gpu
@pytest.mark.parametrize("value", [-1e29, -1e30, -1e32, -2e38, -2.2e38, -3e38])
@pytest.mark.parametrize("dtype", [torch.float32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(20, 16, 1, 300, 300, 128), (2, 8, 1, 1101, 1101, 96), (1, 4, 2, 300, 301, 64), (1, 2, 1, 260, 300, 256)], ids=str)
def test_large_values_that_stand_for_hidden_keys(gpu, size, dtype, value):
    """In front of every text, over whole tiles and the beginning of one: rows that look at nothing else look at all of it alike, whatever tile a key is in.

    The scores are less than half a step of such a value, so that these rows' weights are equal: the output is a mean, of sums with a rounding of 2^-24 for each key,
    divided and rounded once more.  Other rows see nothing of it."""
    B, H, g, Tq, Tk, D = size
    q, k, v = qkv(*size, F16, gpu)
    n = 100
    m = torch.zeros(B, 1, Tq, Tk, dtype=dtype, device=gpu)
    m[..., :n] = value
    got = gemv.prompt_attention(q, k, v, D ** -0.5, m).cpu().double()
    first = n - (Tk - Tq)
    of = v[0].cpu().double().repeat_interleave(g, 0)[:, :n]
    seen = torch.arange(1, n + 1)[:, None]
    mean, size_of = of.cumsum(1) / seen, of.abs().cumsum(1) / seen
    want, off = (t[:, n - first:].transpose(0, 1) for t in (mean, 2.0 ** -11 * mean.abs() + (seen + 4) * 2.0 ** -24 * size_of + 2.0 ** -25))
    d = (got[0, :first] - want).abs() - off
    assert d.max() <= 0, f"{float((got[0, :first] - want).abs().max()):.3e}, {float(d.max()):.3e} more than may be"
    want, off = plain(q[:1], k[:1], v[:1], D ** -0.5, m[:1].masked_fill(m[:1] != 0, -math.inf))
    check(got[:1, first:], want[:, first:], off[:, first:])


@pytest.mark.gpu
def test_lowest_values_of_64_bits(gpu):
    """They are the lowest of 32 bits to the kernel, not minus infinity: rows of nothing else look at all tokens up to their own alike."""
    q, k, v = qkv(2, 2, 1, 50, 50, 64, F16, gpu)
    m = torch.zeros(2, 1, 50, 50, dtype=torch.float64, device=gpu)
    m[0, :, :, :20] = torch.finfo(torch.float64).min
    m[1, :, 30:, 10] = -math.inf
    low = m.clamp(min=torch.finfo(torch.float32).min).float().masked_fill_(m == -math.inf, -math.inf)
    got = gemv.prompt_attention(q, k, v, 0.125, m)
    assert torch.equal(got, gemv.prompt_attention(q, k, v, 0.125, low))
    check(got, *plain(q, k, v, 0.125, low))


@pytest.mark.gpu
def test_layouts(gpu):
    """Heads first, a slice of a fused projection, one key head for all sequences, rows that begin between two pieces of 16 bytes."""
    base = qkv(2, 2, 2, 40, 40, 64, F16, gpu)
    want = gemv.prompt_attention(*base, 0.125)
    assert torch.equal(want, gemv.prompt_attention(*(t.contiguous() for t in base), 0.125))
    fused = torch.cat([t.transpose(1, 2).reshape(2, 40, -1) for t in base], -1)
    q, k, v = (t.view(2, 40, -1, 64).transpose(1, 2) for t in fused.split([256, 128, 128], -1))
    assert torch.equal(want, gemv.prompt_attention(q, k, v, 0.125))
    shifted = []
    for t in base:
        flat = torch.empty(t.numel() + 5, dtype=t.dtype, device=gpu)[5:]
        shifted.append(flat.view(t.shape).copy_(t))
    assert shifted[0].is_contiguous() and shifted[0].data_ptr() % 16
    assert torch.equal(want, gemv.prompt_attention(*shifted, 0.125))
    back = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in base]      # channels are not contiguous
    assert torch.equal(want, gemv.prompt_attention(*back, 0.125))
    q, k, v = base
    one = (k[:1].expand(2, 2, 40, 64), v[:1].expand(2, 2, 40, 64))
    assert torch.equal(gemv.prompt_attention(q, *one, 0.125), gemv.prompt_attention(q, *(t.contiguous() for t in one), 0.125))
    m = torch.rand(2, 1, 40, 40, device=gpu) < 0.6
    assert torch.equal(gemv.prompt_attention(q, k, v, 0.125, m), gemv.prompt_attention(q, k, v, 0.125, m.transpose(2, 3).contiguous().transpose(2, 3)))


@pytest.mark.gpu
def test_nothing_to_do(gpu):
    q, k, v = qkv(2, 2, 1, 0, 5, 64, F16, gpu)
    assert gemv.prompt_attention(q, k, v, 1.0).shape == (2, 0, 2, 64)
    q, k, v = qkv(0, 2, 1, 5, 5, 64, F16, gpu)
    assert gemv.prompt_attention(q, k, v, 1.0).shape == (0, 5, 2, 64)


@pytest.mark.gpu
def test_two_streams_and_a_graph(gpu):
    """Pieces have a workspace: calls on two streams at once, and a captured call replayed between eager ones."""
    made = [qkv(1, 2, 1, 3, 5000, 128, F16, gpu, seed=s) for s in range(2)]
    want = [gemv.prompt_attention(*m, 0.1) for m in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for m, st in zip(made, streams):
            with torch.cuda.stream(st):
                got.append(gemv.prompt_attention(*m, 0.1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    fixed = [t.clone() for t in made[0]]
    bounds = torch.tensor([0, 100, 333], dtype=torch.int32, device=gpu)
    packed = qkv(1, 2, 2, 400, 400, 64, BF16, gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gemv.prompt_attention(*fixed, 0.1)
        other = gemv.prompt_attention(*packed, 0.125, bounds=bounds)
    for i, ends in enumerate([[0, 100, 333], [0, 333, 400], [10, 20, 30]]):
        for t, m in zip(fixed, made[i % 2]):
            t.copy_(m)
        bounds.copy_(torch.tensor(ends, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i % 2])
        assert torch.equal(other, gemv.prompt_attention(*packed, 0.125, bounds=bounds))


@pytest.mark.gpu
def test_long_rows(gpu):
    """Offsets beyond 32 bits: two heads of a long axis, strided as in a wide projection."""
    T, wide = 70000, 16384
    base = torch.zeros(T, wide * 2, dtype=F16, device=gpu)          # 4.6 GB
    g = torch.Generator(device=gpu).manual_seed(3)
    base[:, :64] = torch.randn(T, 64, generator=g, device=gpu).half()
    base[:, -64:] = torch.randn(T, 64, generator=g, device=gpu).half()
    k = v = base.as_strided((1, 2, T, 64), (0, 2 * wide - 64, 2 * wide, 1))
    q = torch.randn(1, 2, 3, 64, generator=g, device=gpu).half()
    check(gemv.prompt_attention(q, k, v, 0.125), *plain(q, k, v, 0.125))


def test_refusals():
    mk = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype)
    q, k = mk(1, 4, 8, 64), mk(1, 2, 8, 64)
    for bad, message in [
        ((mk(4, 8, 64), k, k), "q must be"), ((q, k, mk(1, 2, 7, 64)), "disagree"), ((q, mk(2, 2, 8, 64), mk(2, 2, 8, 64)), "disagree"),
        ((q.float(), k.float(), k.float()), "float16 or bfloat16"), ((q, k.bfloat16(), k), "one dtype"),
        ((mk(1, 4, 8, 60), mk(1, 2, 8, 60), mk(1, 2, 8, 60)), "multiple of 8"), ((mk(1, 4, 8, 264), mk(1, 2, 8, 264), mk(1, 2, 8, 264)), "up to 256"),
        ((mk(1, 3, 8, 64), k, k), "multiple of that"), ((mk(1, 4, 9, 64), k, k), "last of the tokens"),
        ((q.clone().requires_grad_(), k, k), "no gradient"), ((q, k, k), "device"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            gemv.prompt_attention(*bad, 1.0)
    for mask, message in [(mk(1, 1, 8, 7), "broadcast"), (mk(1, 3, 8, 8), "broadcast"), (mk(8, 8), "broadcast"), (torch.zeros(1, 1, 8, 8, dtype=torch.int32), "boolean or additive"),
                          (mk(1, 1, 8, 8).requires_grad_(), "no gradient")]:
        with pytest.raises(RuntimeError, match=message):
            gemv.prompt_attention(q, k, k, 1.0, mask)
    for bounds, message in [(torch.tensor([[0, 8]]), "whole numbers"), (torch.tensor([0.0, 8.0]), "whole numbers"), (torch.tensor([0, 9]), "ascend"), (torch.tensor([-1, 8]), "ascend"),
                            (torch.tensor([0, 5, 3]), "ascend"), (torch.tensor([], dtype=torch.int64), "whole numbers")]:
        with pytest.raises(RuntimeError, match=message):
            gemv.prompt_attention(q, k, k, 1.0, bounds=bounds)
    for args in [(mk(2, 4, 8, 64), mk(2, 2, 8, 64), mk(2, 2, 8, 64), 1.0, None), (mk(1, 4, 7, 64), k, k, 1.0, None), (q, k, k, 1.0, mk(1, 1, 8, 8))]:
        with pytest.raises(RuntimeError, match="packed"):
            gemv.prompt_attention(*args, bounds=torch.tensor([0, 7]))
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="device"):
            gemv.prompt_attention(q.clone().requires_grad_(), k, k, 1.0)


def test_the_library_refuses_what_it_cannot_take():
    import ctypes as C

    from adkv_amd import _lib
    L = _lib.lib()
    st = lambda *x: (C.c_int64 * 3)(*x)
    good = dict(q=4096, qs=st(512, 512, 64), k=4096, ks=st(512, 512, 64), v=4096, vs=st(512, 512, 64), mask=None, ms=None, scaling=1.0, bounds=None, n=0, out=4096,
                B=1, Hq=1, H=1, Tq=8, Tk=8, D=64, dtype=1, ws=None, size=0, stream=None)
    for change, code in [(dict(q=None), -1), (dict(out=None), -1), (dict(mask=4096), -1), (dict(n=1), -1), (dict(B=0), -3), (dict(Tq=9), -3), (dict(Hq=3, H=2), -3), (dict(n=-1), -3),
                         (dict(n=1, bounds=4096, B=2), -3), (dict(n=1, bounds=4096, Tq=4), -3), (dict(D=0), -2), (dict(D=60), -2), (dict(D=264), -2), (dict(dtype=0), -6),
                         (dict(dtype=3), -6), (dict(dtype=1 | 4 << 8), -6), (dict(n=1, bounds=4096, mask=4096, ms=st(0, 0, 8)), -6), (dict(q=4104), -5), (dict(ks=st(512, 512, 68)), -5),
                         (dict(ks=st(512, 512, -64)), -3), (dict(vs=st(512, 512, 1 << 23)), -3), (dict(mask=4097, ms=st(0, 0, 8), dtype=1 | 1 << 8), -5),
                         (dict(Hq=40000, Tq=8), -3), (dict(Tk=2 ** 31 - 1), -3)]:
        a = {**good, **change}
        assert L.adkv_prompt_attention(*a.values()) == code, change
    assert L.adkv_prompt_attention_workspace_bytes(1, 3, 2, 8, 8, 64, 0) == -3
    assert L.adkv_prompt_attention_workspace_bytes(1, 4, 2, 8, 8, 63, 0) == -2


def test_sizes_that_no_memory_has():
    from adkv_amd import _lib
    L, m = _lib.lib(), 2 ** 31 - 1
    for B, Hq, H, Tq, n_seq in [(m, m, m, 4, 0), (m, m, m, 1, 0), (1, m, 1, m, 0), (1, m, m, 4, m), (m, 1, 1, m, 0), (1 << 24, 1, 1, 1, 0), (1, 46341, 1, 1, 0)]:
        assert L.adkv_prompt_attention_workspace_bytes(B, Hq, H, Tq, min(Tq, 2 ** 30), 64, n_seq) == -3

"""Attention of several new tokens over codes, with a prefix that the batch shares (gemv.extend), against the oracle's codes
and values and 64-bit attention over them."""
import math

import numpy as np
import pytest
import torch

from adkv_amd import _lib, synth
from adkv_amd.kernel import gemv

D = 128


def _np16(t):
    return t.detach().cpu().contiguous().view(torch.int16).numpy().view(np.float16)


class Case:
    """Streams of P shared and T own tokens in caches as the framework writes them, n new ones, and what should come of them."""

    def __init__(self, oracle, dev, B, H, G, P, T, n, bits=4, dtype=torch.float16, S=64, seed=0, room=5):
        self.__dict__.update(B=B, H=H, G=G, P=P, T=T, n=n, bits=bits, dtype=dtype, S=S, dev=dev)
        kp, vp = (synth.make_params(H, D, bits=bits, seed=seed + i) for i in (1, 2))
        x = [synth.make_k(1, H, P, D, seed=seed, dtype=torch.float16), synth.make_v(1, H, P, D, seed=seed + 1, dtype=torch.float16)]
        y = [synth.make_k(B, H, T + n, D, seed=seed + 2, t0=P, dtype=torch.float16), synth.make_v(B, H, T + n, D, seed=seed + 3, dtype=torch.float16)]
        if dtype == torch.bfloat16:
            y = [t.bfloat16().half() for t in y]           # the new rows are given as bfloat16
        self.q = synth.make_q(B, H * G * n, D, seed=seed + 4).view(B, n, H * G, D).to(dtype).to(dev).transpose(1, 2)
        self.new = [t[:, :, T:].to(dtype).to(dev) for t in y]
        params = [p.to(dev).astuple() for p in (kp, vp)]
        tps = 32 // bits

        def stream(rows, params, tokens, cap):
            X = rows.shape[0]
            cache = synth.alloc_cache(X, H, cap, D, dev, bits=bits)
            state = torch.zeros(X, H, D, 2, dtype=torch.float16, device=dev)
            ck = torch.zeros(X, H, cap // S + 1, D, 2, dtype=torch.float16, device=dev) if S else None
            if tokens:
                gemv.append_kv(cache, rows.to(dev), *params, 0, state, ckpt=ck, ckpt_interval=S, bits=bits)
            else:
                state[..., 0], state[..., 1] = params[0], params[1]
            return cache, ck, state
        pre = [stream(x[i], params[i], P, max(P, 1)) for i in range(2)]
        self.prefix = None
        self.params = params
        if P:
            self.prefix = gemv.SharedPrefix(pre[0][0], pre[1][0], P, *params, pre[0][1], pre[1][1])
            self.params = [(pre[i][2][0, :, :, 0].contiguous(), pre[i][2][0, :, :, 1].contiguous(), *params[i][2:]) for i in range(2)]
        own = [stream(y[i][:, :, :T].contiguous(), self.params[i], T, T + n + room) for i in range(2)]
        self.cache, self.ckpt = [o[0] for o in own], [o[1] for o in own]

        # the whole streams by the oracle: codes of all tokens, values of all tokens
        self.want_cache, self.values = [], []
        with oracle.code_bits(bits):
            for i in range(2):
                pn = [_np16(t) for t in params[i]]
                c0 = oracle.alloc_cache(1, H, max(P, 1), D)
                shared = np.zeros((1, H, 0, D), np.float16)
                if P:
                    oracle.encode_kv_f16(c0, _np16(x[i]), *pn)
                    shared = oracle.replay_f16(c0, *pn, P)[0]
                po = [_np16(t) for t in self.params[i]]
                c1 = oracle.alloc_cache(B, H, T + n + room, D)
                oracle.encode_kv_f16(c1, _np16(y[i]), *po)
                own = oracle.replay_f16(c1, *po, T + n)[0]
                self.want_cache.append(c1)
                self.values.append(np.concatenate([np.broadcast_to(shared, (B, *shared.shape[1:])), own], 2).astype(np.float64))

    def run(self, scaling, mask=None, **kw):
        return gemv.extend(self.q, *self.cache, *self.new, *self.params, self.T, scaling, mask, prefix=self.prefix,
                           k_ckpt=self.ckpt[0], v_ckpt=self.ckpt[1], ckpt_interval=self.S, bits=self.bits, **kw)

    def want(self, scaling, mask=None):
        """The outputs in 64 bits, sums of |weight * value| that errors are measured in, and the size of each row's largest score."""
        B, H, G, n, P, T = self.B, self.H, self.G, self.n, self.P, self.T
        q = self.q.float().cpu().numpy().astype(np.float64).reshape(B, H, G * n, D)
        k, v = self.values
        x = np.matmul(q, k.transpose(0, 1, 3, 2)).reshape(B, H, G, n, P + T + n) * scaling
        if mask is not None:
            m = mask.float().cpu().numpy().astype(np.float64)
            m = m[:, :, None] if m.ndim == 3 else m
            x = x + np.broadcast_to(m, (B, H * G, n, P + T + n)).reshape(B, H, G, n, -1)
        hidden = np.arange(P + T + n)[None] > P + T + np.arange(n)[:, None]
        x = np.where(hidden, -np.inf, x)
        top = x.max(-1, keepdims=True)
        with np.errstate(invalid="ignore"):
            e = np.exp(x - top)
        w = (e / e.sum(-1, keepdims=True)).reshape(B, H, G * n, -1)
        place = lambda o: o.reshape(B, H, G, n, D).transpose(0, 3, 1, 2, 4).reshape(B, n, H * G, D)
        top = np.where(np.abs(top) < 2.0 ** 30, np.abs(top), 0.0)      # beyond, 53 bits lose the score beside the mask as 24 do
        return place(np.matmul(w, v)), place(np.matmul(w, np.abs(v))), place(np.broadcast_to(top, (B, H, G, n, D)))

    def check(self, out, scaling, mask=None):
        want, size, top = self.want(scaling, mask)
        got = out.float().cpu().numpy().astype(np.float64)
        assert out.dtype == self.dtype and got.shape == want.shape
        assert np.array_equal(np.isnan(got), np.isnan(want))
        # a weight is off by half a step of fp16 (2^-11 of it, 2^-25 of the largest where it is small), scores and sums by what
        # fp32 leaves (128 products of up to some hundred: 2^-15), the result by half a step of its type.  A score beside a large
        # mask is rounded with it, half a step of fp32 (2^-24 of the sum) for itself and for the largest, by which weights are off.
        small = (self.P + self.T + self.n) * 2.0 ** -25 * max(np.abs(self.values[1]).max(), 1.0)
        far = np.abs(got - want) - (size * (2.0 ** -11 + 2.0 ** -14 + top * 2.0 ** -23) + small + np.abs(want) * torch.finfo(self.dtype).eps / 2 + 2.0 ** -24)
        worst = np.nanmax(np.where(np.isnan(want), -1.0, far))
        assert worst <= 0, worst
        for c, w in zip(self.cache, self.want_cache):
            assert np.array_equal(c.cpu().numpy(), w)


f16, bf16 = torch.float16, torch.bfloat16
SIZES = [  # B, H, G, P, T, n, bits, type, interval
    (1, 1, 1, 0, 0, 1, 4, f16, 64), (1, 2, 1, 1, 0, 1, 4, f16, 64), (2, 2, 1, 64, 0, 1, 4, bf16, 64), (2, 1, 4, 65, 3, 1, 2, f16, 64),
    (3, 2, 2, 200, 64, 1, 4, f16, 64), (17, 2, 1, 300, 63, 1, 4, f16, 64), (5, 1, 8, 77, 128, 1, 2, bf16, 64), (70, 1, 2, 130, 9, 1, 4, f16, 64),
    (2, 2, 1, 0, 130, 2, 4, f16, 64), (2, 1, 4, 0, 127, 5, 4, bf16, 64), (1, 2, 8, 129, 191, 3, 2, f16, 64), (2, 2, 2, 100, 0, 70, 4, f16, 64),
    (1, 1, 1, 0, 0, 200, 4, f16, 64), (3, 1, 1, 500, 61, 67, 4, bf16, 64), (2, 1, 4, 40, 255, 129, 2, f16, 256), (1, 1, 2, 700, 300, 33, 4, f16, 0),
    (2, 1, 8, 513, 512, 16, 4, f16, 256), (2, 3, 1, 64, 192, 64, 4, f16, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(str(v).replace("torch.", "") for v in s))
def test_outputs_and_codes(gpu, oracle, size):
    c = Case(oracle, gpu, *size, seed=sum(size[:6]))
    out = c.run(D ** -0.5)
    c.check(out, D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [(3, 2, 2, 150, 70, 1), (2, 1, 4, 97, 33, 40), (2, 2, 1, 0, 20, 9)])
def test_masks(gpu, oracle, dtype, size):
    B, H, G, P, T, n = size
    c = Case(oracle, gpu, *size, dtype=torch.bfloat16 if dtype == torch.bfloat16 else torch.float16, seed=5)
    g = torch.Generator().manual_seed(3)
    mask = (torch.randn(B, H * G, n, P + T + n, generator=g) * 2).to(dtype)
    low = torch.finfo(dtype).min
    mask[0, :, :, :P // 2] = low
    mask[-1, :, :, P // 3:P + T // 2] = -math.inf
    mask[0, 0, 0, :] = low                               # a whole row: what is left is equal weights, or nearly
    mask = mask.to(gpu)
    c.check(c.run(D ** -0.5, mask), D ** -0.5, mask)
    nothing = mask.clone()
    nothing[1, 0, n - 1, :] = -math.inf                  # nothing is left of this row, and of no other
    out = c.run(D ** -0.5, nothing)
    assert bool(out[1, n - 1, 0].isnan().all())
    c.check(out, D ** -0.5, nothing)
    for m in (mask[:, :1], mask[:1], mask[:, :, :1], mask[:1, :1, :1], mask[:, :, 0], mask.double(),
              mask.transpose(1, 3).contiguous().transpose(1, 3)):      # broadcast, three axes, another type, other strides
        c.check(c.run(D ** -0.5, m), D ** -0.5, m)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [0.0, -0.3, 1.5])
def test_scalings(gpu, oracle, scaling):
    c = Case(oracle, gpu, 2, 2, 2, 100, 60, 7, seed=9)
    c.check(c.run(scaling), scaling)


@pytest.mark.gpu
def test_rows_are_read_where_they_lie(gpu, oracle):
    """Head-first views, rows of a wider projection, odd strides and offsets: the same bits as packed rows."""
    c = Case(oracle, gpu, 3, 2, 2, 90, 30, 6, seed=11)
    c.q = c.q.contiguous()
    want = c.run(D ** -0.5).clone()

    def wide(t, extra, at):                              # [B, h, n, D] inside [B, n, h * D + extra]
        B, h, n, _ = t.shape
        w = torch.zeros(B, n, h * D + extra, dtype=t.dtype, device=t.device)
        w[:, :, at:at + h * D] = t.transpose(1, 2).reshape(B, n, h * D)
        return w[:, :, at:at + h * D].view(B, n, h, D).transpose(1, 2)
    q, new = c.q, c.new
    for extra, at in ((0, 0), (6, 2), (7, 3), (8, 1)):
        c.q, c.new = wide(q, extra, at), [wide(t, extra, at) for t in new]
        assert torch.equal(c.run(D ** -0.5), want), (extra, at)
    c.q, c.new = q.transpose(2, 3).contiguous().transpose(2, 3), new      # channels apart
    assert torch.equal(c.run(D ** -0.5), want)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("T", [0, 63, 64, 130])
def test_as_many_decode_steps(gpu, oracle, bits, T):
    """The caches, checkpoints included, are those that single steps leave, and the outputs agree to what fp16 logits are off by."""
    c = Case(oracle, gpu, 2, 2, 2, 0, T, 70, bits=bits, seed=13)
    cache, ckpt = [t.clone() for t in c.cache], [t.clone() for t in c.ckpt]
    steps = []
    for i in range(c.n):
        one = lambda t: t[:, :, i:i + 1].contiguous()
        o, _ = gemv.decode_step(one(c.q), *cache, *map(one, c.new), *c.params, T + i, D ** -0.5, k_ckpt=ckpt[0], v_ckpt=ckpt[1],
                                ckpt_interval=c.S, bits=bits)
        steps.append(o)
    out = c.run(D ** -0.5)
    c.check(out, D ** -0.5)
    assert all(torch.equal(a, b) for a, b in zip(cache, c.cache))
    last = (T + c.n - 1) // c.S                          # a step records a checkpoint with the token behind it
    assert all(torch.equal(a[:, :, :last], b[:, :, :last]) for a, b in zip(ckpt, c.ckpt))
    assert float((torch.stack(steps, 1).float() - out.float()).abs().max()) < 2e-2
    # steps go on behind it, and it behind steps
    c2 = Case(oracle, gpu, 2, 2, 2, 0, T, 70, bits=bits, seed=13)
    for i in range(33):
        one = lambda t: t[:, :, i:i + 1].contiguous()
        gemv.decode_step(one(c2.q), *c2.cache, *map(one, c2.new), *c2.params, T + i, D ** -0.5, k_ckpt=c2.ckpt[0], v_ckpt=c2.ckpt[1],
                         ckpt_interval=c.S, bits=bits)
    rest = gemv.extend(c2.q[:, :, 33:], *c2.cache, *[t[:, :, 33:] for t in c2.new], *c2.params, T + 33, D ** -0.5, k_ckpt=c2.ckpt[0],
                       v_ckpt=c2.ckpt[1], ckpt_interval=c.S, bits=bits)
    assert all(torch.equal(a, b) for a, b in zip(c.cache + c.ckpt, c2.cache + c2.ckpt))
    assert float((rest.float() - out[:, 33:].float()).abs().max()) < 2e-3


@pytest.mark.gpu
def test_slots_behind_the_new_tokens_stay(gpu, oracle):
    c = Case(oracle, gpu, 2, 1, 1, 40, 13, 3, seed=17, room=20)
    for t in c.cache + c.ckpt:
        t.view(-1).view(torch.uint8)[:] = t.view(-1).view(torch.uint8)
    before = [t.clone() for t in c.cache]
    for t in c.cache:
        t[:, :, 3:] = 0x5A
    c.run(D ** -0.5)
    for t, b in zip(c.cache, before):
        assert bool((t[:, :, 3:] == 0x5A).all())
        w = t.view(torch.int32)[:, :, 1] >> 20           # tokens 13..15 of the second word are the new ones
        assert torch.equal(t[:, :, :1], b[:, :, :1]) and bool((w != 0).any())


@pytest.mark.gpu
def test_other_streams_and_graphs(gpu, oracle):
    """On a side stream, and captured: every replay, with eager work in between, writes what the eager call writes."""
    for size in ((3, 2, 2, 150, 70, 1), (2, 1, 4, 97, 64, 20)):
        c = Case(oracle, gpu, *size, seed=19)
        fresh = [t.clone() for t in c.cache + c.ckpt]
        want = c.run(D ** -0.5).clone()
        done = [t.clone() for t in c.cache + c.ckpt]
        ws = torch.empty(gemv.extend_workspace_bytes(c.B, c.H * c.G, c.H, c.T, c.n, c.ckpt[0].shape[2], c.S, c.P, c.prefix.k_ckpt.shape[2]),
                         dtype=torch.uint8, device=gpu)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(c.run(D ** -0.5, workspace=ws), want)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c.run(D ** -0.5, workspace=ws)
        for _ in range(3):
            for t, f in zip(c.cache + c.ckpt, fresh):
                t.copy_(f)
            out.zero_()
            ws.fill_(255)
            graph.replay()
            junk = (want.float() * 1.5).sum()
            torch.cuda.synchronize()
            assert torch.isfinite(junk) and torch.equal(out, want)
            assert all(torch.equal(a, b) for a, b in zip(c.cache + c.ckpt, done))


def _cpu_args(B=2, H=2, G=1, T=8, n=2, P=8, dtype=torch.float16):
    mk = lambda *s: torch.zeros(*s, dtype=dtype)
    par = lambda: tuple(torch.zeros(H, D, dtype=torch.float16) for _ in range(5))
    cache = lambda b: torch.zeros(b, H, 4, D // 4, 4, 4, dtype=torch.uint8)
    return dict(q=mk(B, H * G, n, D), k_cache=cache(B), v_cache=cache(B), k_new=mk(B, H, n, D), v_new=mk(B, H, n, D), k_params=par(),
                v_params=par(), T=T, scaling=1.0, prefix=gemv.SharedPrefix(cache(1), cache(1), P, par(), par()))


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(2, 2, 2, D)), "float16 or bfloat16"), (dict(k_new=torch.zeros(2, 2, 2, D)), "q's type"),
    (dict(k_new=torch.zeros(2, 2, 3, D, dtype=torch.float16)), "q must be"), (dict(q=torch.zeros(2, 6, 2, D, dtype=torch.float16)), "1, 2, 4 or 8"),
    (dict(k_cache=torch.zeros(2, 2, 4, 32, 4, 4)), "uint8"), (dict(T=-1), "non-negative"), (dict(T=31), "no room"), (dict(bits=3), "2 or 4"),
    (dict(bits=2, T=63), "no room"), (dict(mask=torch.zeros(2, 1, 2, 17)), "broadcast"), (dict(mask=torch.zeros(2, 3, 2, 18)), "broadcast"),
    (dict(k_ckpt=torch.zeros(2, 2, 1, D, 2, dtype=torch.float16)), "both checkpoint"), (dict(k_params=(torch.zeros(2, D),) * 5), "float16"),
    (dict(k_params=(torch.zeros(3, D, dtype=torch.float16),) * 5), "elements"), (dict(), "HIP device"),
], ids=lambda v: v if isinstance(v, str) else None)
def test_refusals(change, message):
    args = {**_cpu_args(), **change}
    with pytest.raises(RuntimeError, match=message):
        gemv.extend(**args)


@pytest.mark.parametrize("change, message", [
    (dict(tokens=33), "do not hold"), (dict(tokens=-1), "negative"), (dict(k_cache=torch.zeros(2, 2, 4, 32, 4, 4, dtype=torch.uint8)), "prefix's caches"),
    (dict(v_cache=torch.zeros(1, 2, 3, 32, 4, 4, dtype=torch.uint8)), "do not hold"), (dict(k_params=(torch.zeros(2, D),) * 5), "float16"),
    (dict(k_ckpt=torch.zeros(1, 2, 1, D, 2, dtype=torch.float16)), "both of the prefix's"),
])
def test_refusals_of_prefixes(change, message):
    args = _cpu_args()
    args["prefix"] = args["prefix"]._replace(**change)
    with pytest.raises(RuntimeError, match=message):
        gemv.extend(**args)


def test_other_head_dims_are_refused():
    mk = lambda: torch.zeros(1, 1, 1, 256, dtype=torch.float16)
    cache = torch.zeros(1, 1, 4, 64, 4, 4, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="DIM == 128"):
        gemv.extend(mk(), cache, cache.clone(), mk(), mk(), (), (), 0, 1.0)


def test_the_library_refuses_before_any_launch():
    """On the host: no pointer here is device memory."""
    import ctypes
    L = _lib.lib()
    one = ctypes.c_void_p(256)
    arr5 = (ctypes.c_void_p * 5)(*[256] * 5)
    st = (ctypes.c_int64 * 3)(256, 128, 128)
    need = L.adkv_extend_workspace_bytes(1, 1, 1, 8, 2, 0, 0, 0, 0, 0)
    assert need > 0 and L.adkv_extend_workspace_bytes(1, 3, 2, 8, 2, 0, 0, 0, 0, 0) == 0

    def call(q=one, params=arr5, mask=None, B=1, Hq=1, H=1, T=8, n=2, dim=128, cap=2, bits=4, act=1, ck=None, ncap=0, interval=0, prefix=None,
             ws=one, nbytes=need, strides=st):
        return L.adkv_extend(q, strides, one, one, one, one, None, None, params, params, mask, None, 1.0, one, B, Hq, H, T, n, dim, cap, bits, act,
                             ck, ck, ncap, interval, prefix, ws, nbytes, None)
    assert call(q=None) == call(params=None) == call(mask=one) == -1
    assert call(T=-1) == call(n=0) == call(B=0) == call(Hq=3, H=2) == call(T=1 << 24) == -3
    assert call(dim=256) == call(bits=3) == call(act=0) == call(Hq=3) == call(act=1 | 7 << 8) == -6
    assert call(cap=1) == -4 and call(q=ctypes.c_void_p(258)) == call(strides=(ctypes.c_int64 * 3)(255, 128, 128)) == -5
    assert call(nbytes=need - 1) == call(ws=None) == -7
    assert call(ck=one, ncap=1, interval=12) == call(ck=one, ncap=0, interval=8) == -3
    arr = ctypes.cast(arr5, ctypes.c_void_p)
    pre = lambda **k: ctypes.byref(_lib.Prefix(**{**dict(k_codes=256, v_codes=256, k_params=arr, v_params=arr, tokens=8, n_super=1), **k}))
    assert call(prefix=pre(k_codes=None)) == -1 and call(prefix=pre(tokens=9)) == -4 and call(prefix=pre(tokens=-1)) == -3
    assert call(prefix=pre(k_ckpt=256)) == -1 and call(prefix=pre(k_codes=260)) == -5


def test_host_calls_that_are_left_to_python():
    h = _lib.host()
    x = torch.zeros(1, 1, 1, 128, dtype=torch.float16)
    for f, n in ((h.extend, 15), (h.rope_norm_qk, 7)):
        assert f() is None and f(*[None] * n) is None and f(*[x] * n) is None and f(*[1 << 70] * n) is None


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(3, 2, 2, 150, 70, 1), (2, 1, 4, 97, 33, 40), (2, 2, 1, 0, 20, 9), (2, 2, 1, 30, 0, 3)])
@pytest.mark.parametrize("mask_type", [None, torch.bfloat16, torch.float32])
def test_host_calls_equal_the_python_function(gpu, oracle, monkeypatch, size, mask_type):
    """The same call through the host calls and without them: the same codes, checkpoints and outputs."""
    import types
    B, H, G, P, T, n = size
    results = []
    real = _lib.host()
    for taken in (True, False):
        c = Case(oracle, gpu, *size, dtype=torch.bfloat16, seed=11)
        mask = None
        if mask_type is not None:
            mask = torch.zeros(B, 1, n, P + T + n, dtype=mask_type)
            mask[0, :, :, :(P + T) // 2] = torch.finfo(mask_type).min
            mask = mask.to(gpu)
        calls = []

        def extend(*a):
            r = real.extend(*a) if taken else None
            calls.append(r is not None)
            return r
        monkeypatch.setattr(_lib, "host", lambda: types.SimpleNamespace(extend=extend))
        out = c.run(D ** -0.5, mask)
        monkeypatch.undo()
        assert calls == [taken]
        results.append([out.view(torch.int16), *c.cache, *[t.view(torch.int16) for t in c.ckpt]])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [(2, 2, 1, 400, 70, 130), (24, 1, 2, 500, 3, 1), (3, 1, 8, 0, 300, 21), (2, 2, 2, 333, 200, 10)])
def test_masks_that_are_zero_in_places(gpu, oracle, dtype, size):
    """Stretches of tokens without anything added, with a little added, and hidden, so that every way from one to the next is taken:
    also where all that was seen so far was hidden."""
    B, H, G, P, T, n = size
    c = Case(oracle, gpu, *size, dtype=torch.bfloat16 if dtype == torch.bfloat16 else torch.float16, seed=8)
    N, low = P + T + n, torch.finfo(dtype).min
    g = torch.Generator().manual_seed(4)
    for first in (low, -math.inf, 0.0, 2000.0):
        mask = torch.zeros(B, 1, n, N, dtype=dtype)
        mask[:, :, :, :N // 3] = first
        mask[0, :, :, N // 2:N // 2 + 70] = torch.randn(n, 70, generator=g).to(dtype)[:, :mask.shape[3] - N // 2]
        mask[-1, :, n // 2:, N // 2:N - 40] = low
        mask = mask.to(gpu)
        c.check(c.run(D ** -0.5, mask), D ** -0.5, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("G,n,P", [(4, 5, 0), (8, 16, 70)])
def test_own_tiles_in_several_batches(gpu, G, n, P):
    """More own tokens than there is room for tiles of at a time (1 GiB, two million tokens of a head): sequences of the first and the last batch
    against the same sequences by themselves.  Codes are equal; of the outputs either side rounds weights (2^-11, small ones 2^-25 a token), sums (2^-14)
    and the result (2^-11), of values up to `top`."""
    B, H, T = 66, 16, 2041
    gen = torch.Generator(device=gpu).manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=gen, device=gpu, dtype=torch.float16)
    params = [p.to(gpu).astuple() for p in (synth.make_params(H, D, seed=s) for s in (1, 2))]
    pre, own_params = None, params
    if P:
        pc, pst = [synth.alloc_cache(1, H, P, D, gpu) for _ in range(2)], [torch.zeros(1, H, D, 2, dtype=torch.float16, device=gpu) for _ in range(2)]
        gemv.append_kv_pair(*pc, rand(1, H, P, D), rand(1, H, P, D), *params, 0, *pst)
        pre = gemv.SharedPrefix(*pc, P, *params)
        own_params = [(st[0, :, :, 0].contiguous(), st[0, :, :, 1].contiguous(), *p[2:]) for st, p in zip(pst, params)]
    cache = [synth.alloc_cache(B, H, T + n, D, gpu) for _ in range(2)]
    ckpt = [torch.zeros(B, H, (T + n) // 256 + 1, D, 2, dtype=torch.float16, device=gpu) for _ in range(2)]
    state = [torch.zeros(B, H, D, 2, dtype=torch.float16, device=gpu) for _ in range(2)]
    gemv.append_kv_pair(*cache, rand(B, H, T, D), rand(B, H, T, D), *own_params, 0, *state, k_ckpt=ckpt[0], v_ckpt=ckpt[1], ckpt_interval=256)
    q, new = rand(B, H * G, n, D), [rand(B, H, n, D) for _ in range(2)]
    parts = [slice(0, 3), slice(B - 3, B)]
    few = [[t[p].clone() for t in (q, *cache, *new, *ckpt)] for p in parts]

    def run(q, kc, vc, kn, vn, kk, vk):
        return gemv.extend(q, kc, vc, kn, vn, *own_params, T, D ** -0.5, prefix=pre, k_ckpt=kk, v_ckpt=vk, ckpt_interval=256)
    whole = run(q, *cache, *new, *ckpt)
    assert torch.isfinite(whole).all()
    for p, f in zip(parts, few):
        got = run(*f)
        assert torch.equal(f[1], cache[0][p]) and torch.equal(f[2], cache[1][p])
        assert torch.equal(f[5].view(torch.int16), ckpt[0][p].view(torch.int16)) and torch.equal(f[6].view(torch.int16), ckpt[1][p].view(torch.int16))
        top = 16.0        # values follow rows of up to 6, and twice that where the scale has not settled
        assert (got.float() - whole[p].float()).abs().max().item() <= 2 * top * (2.0 ** -11 + 2.0 ** -14 + (P + T + n) * 2.0 ** -25 + 2.0 ** -11)

"""The workspace that gemv.extend allocates where the host call is not taken."""
import types

import pytest
import torch

from adkv_amd import _lib
from adkv_amd.kernel import gemv
from test_extend import D, Case


@pytest.mark.parametrize("own,shared", [(False, False), (False, True), (True, False), (True, True)])
def test_workspace_is_what_the_library_asks_for(monkeypatch, own, shared):
    """Checkpoints of either source or of both: the pieces, and with them the bytes, go by each source's own."""
    B, H, P, T, n, S = 2, 8, 8192, 0, 1, 256
    got = {}
    real = _lib.lib()

    def extend(*a):
        got["bytes"] = a[-2]
        return 0
    monkeypatch.setattr(_lib, "host", lambda: types.SimpleNamespace(extend=lambda *a: None))
    monkeypatch.setattr(_lib, "lib", lambda: types.SimpleNamespace(adkv_extend=extend, adkv_extend_workspace_bytes=real.adkv_extend_workspace_bytes))
    monkeypatch.setattr(gemv, "_need_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "device_guard", lambda d: _lib._NO_GUARD)
    monkeypatch.setattr(_lib, "current_stream_ptr", lambda d: None)
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)
    cache = lambda b, t: torch.zeros(b, H, -(-t // 8), D // 4, 4, 4, dtype=torch.uint8)
    par = tuple(half(H, D) for _ in range(5))
    ck = lambda b, t: half(b, H, t // S + 1, D, 2)
    kw = dict(k_ckpt=ck(B, T + n), v_ckpt=ck(B, T + n)) if own else {}
    pre = gemv.SharedPrefix(cache(1, P), cache(1, P), P, par, par, *((ck(1, P), ck(1, P)) if shared else ()))
    gemv.extend(half(B, H, n, D), cache(B, 64), cache(B, 64), half(B, H, n, D), half(B, H, n, D), par, par, T, 1.0, prefix=pre, ckpt_interval=S, **kw)
    need = real.adkv_extend_workspace_bytes(B, H, H, T, n, 1 if own else 0, S if own else 0, P, P // S + 1 if shared else 0, S if shared else 0)
    assert got["bytes"] >= need > 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3])
def test_checkpoints_of_the_prefix_only(gpu, oracle, n):
    c = Case(oracle, gpu, 2, 2, 1, 2000, 30, n, seed=23)
    out = gemv.extend(c.q.contiguous(), *c.cache, *c.new, *c.params, c.T, D ** -0.5, torch.zeros(2, 2, c.P + c.T + n, device=gpu, dtype=torch.float64),
                      prefix=c.prefix, ckpt_interval=c.S)     # a mask that has to be converted: not by the host call
    c.check(out, D ** -0.5)

"""Drop-in for the reference's ``adkv.kernel.gemv`` (src/adkv/kernel/gemv.py:16-132).

Same three functions, same argument order, same tensor layouts and the same error messages as the
reference's C++ bindings (src/adkv/kernel/gemv.cu:368-414, 883-939, 1233-1288); the work is done
by hand-written gfx950 kernels behind ``libadkv_hip.so``.  Differences, all on the safe side:

* launches go to PyTorch's *current* stream (the reference uses legacy stream 0);
* an unsupported head dim raises in ``forward_qk`` / ``forward_ov`` too (the reference's launcher
  silently skips the launch and returns uninitialised memory, gemv.cu:875-878, 1226-1229);
* logits and outputs are accumulated in fp32 and rounded once to fp16 (the reference accumulates in
  fp16); codes written to the cache and the filter state are bit-identical.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .. import _lib

_TILE = 4
_DIMS = (128, 256, 512)
_GROUPS = (1, 2, 4, 8)   # query heads per KV head


def _chk(cond: bool, msg: str) -> None:
    # TORCH_CHECK surfaces as RuntimeError in Python
    if not cond:
        raise RuntimeError(msg)


def _need_device(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    if dev.type == "cuda":
        for t in tensors:
            if t.device != dev:
                break
        else:
            return dev
    for t in tensors:
        _chk(t.is_cuda, "ADKV kernels need every tensor on a HIP device; there is no CPU path")
        _chk(t.device == dev, "ADKV kernels need all tensors on the same device")
    return dev


def _params(tensors, names, nh, dim):
    want = nh * dim
    res = []
    for t in tensors:
        if t.dtype != torch.float16 or t.numel() != want:
            break
        res.append(t if t.is_contiguous() else t.contiguous())
    else:
        return res
    for t, n in zip(tensors, names):      # same order of complaints as the reference's checks
        _chk(t.dtype == torch.float16, f"{n} must be float16")
    for t, n in zip(tensors, names):
        _chk(t.numel() == want, f"{n} must have nh*DIM = {want} elements")
    raise AssertionError("unreachable")


@functools.lru_cache(maxsize=4096)
def _row_pitch(n: int) -> int:
    """The library's row pitch for rows of ``n`` elements (a pure function of ``n``)."""
    return int(_lib.lib().adkv_row_pitch(n))


def _pitch(n: int) -> int:
    """Row pitch for a ``[rows, n]`` logits / weights matrix.  Long rows are padded to the library's
    recommended pitch (an odd multiple of 128 elements) so that rows of different heads do not all
    start in one memory channel; short rows stay packed."""
    return _row_pitch(n) if n >= 1024 else n


def _rows_view(t: torch.Tensor):
    """``(tensor, pitch)`` for a ``[B, nh, n]`` matrix whose rows are ``pitch`` elements apart: the
    tensor itself when it is packed or a padded view this module produced, else a packed copy."""
    B, nh, n = t.shape
    if t.is_contiguous():
        return t, n
    if t.stride(2) == 1 and t.stride(1) >= n and t.stride(0) == nh * t.stride(1):
        return t, t.stride(1)
    return t.contiguous(), n


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _ckpt_args(ckpt: torch.Tensor | None, ckpt_interval: int, B: int, nh: int, DIM: int, bits: int = 4):
    """Validates a checkpoint tensor ``[B, nh, n_ckpt_cap, DIM, 2]`` fp16 -> (ptr, cap, interval)."""
    if ckpt is None:
        return None, 0, 0
    _chk(ckpt.dtype == torch.float16 and ckpt.is_contiguous() and ckpt.dim() == 5
         and ckpt.shape[0] == B and ckpt.shape[1] == nh and ckpt.shape[3] == DIM and ckpt.shape[4] == 2
         and ckpt.shape[2] >= 1,
         "ckpt must be contiguous fp16 [B, nh, n_ckpt_cap, DIM, 2]")
    tps = 32 // bits
    _chk(ckpt_interval > 0 and ckpt_interval % tps == 0,
         f"ckpt_interval must be a positive multiple of {tps}")
    return ckpt.data_ptr(), ckpt.shape[2], int(ckpt_interval)


def forward_qk(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    k_new: torch.Tensor,
    k_zp: torch.Tensor,
    k_sc: torch.Tensor,
    k_alpha: torch.Tensor,
    k_beta: torch.Tensor,
    k_t: torch.Tensor,
    T: int,
    scale_min: float,
    scale_max: float,
    *,
    state_out: torch.Tensor | None = None,
    ckpt: torch.Tensor | None = None,
    ckpt_interval: int = 0,
    bits: int = 4,
) -> torch.Tensor:
    """Decode-phase QK^T over the nibble-packed ADKV cache (reference gemv.py:16-55).

    ``o[b,h,t] = sum_c q[b,h,c] * k_deq[b,h,t,c]`` for the ``T`` cached tokens; then ``k_new`` is
    quantised with the filter state after token ``T-1`` and written at position ``T`` in place, and
    its own logit is returned as the last element.

    Args:
        q, k_new: ``[B, nh, 1, DIM]`` float16.
        k_cache:  ``[B, nh, n_super_cap, DIM/4, 4, 4]`` uint8, contiguous, appended in place.
        k_zp, k_sc, k_alpha, k_beta, k_t: ``[nh, DIM]`` float16 ADKV parameters.
        T: number of cached tokens.
        scale_min, scale_max: kept for API compatibility (unused by the fp16 recurrence).
        state_out: optional ``[B, nh, DIM, 2]`` float16, receives (zp, sc) after token ``T-1``
            (extension; not in the reference).
        ckpt, ckpt_interval: optional state checkpoints of this cache, ``[B, nh, n, DIM, 2]`` float16
            with entry ``j`` = state before token ``(j+1)*ckpt_interval`` (extension).  With them
            the time axis is replayed in independent segments; entry ``T/ckpt_interval - 1`` is
            written when token ``T`` opens a new interval.

    Returns ``[B, nh, T+1]`` float16 logits.
    """
    _chk(q.dtype == torch.float16, "q must be float16")
    _chk(k_new.dtype == torch.float16, "k_new must be float16")
    _chk(k_cache.dtype == torch.uint8, "k_cache must be uint8")
    _chk(k_cache.is_contiguous(), "k_cache must be contiguous (appended in place)")
    B, nq = q.shape[0], q.shape[1]
    nh = k_cache.shape[1]          # KV heads; nq is a multiple of it under grouped-query attention
    n_super_cap, n_cgroup = k_cache.shape[2], k_cache.shape[3]
    DIM = n_cgroup * _TILE
    zp, sc, al, be, tg = _params((k_zp, k_sc, k_alpha, k_beta, k_t),
                                 ("k_zp", "k_sc", "k_alpha", "k_beta", "k_t"), nh, DIM)
    _chk(DIM == q.shape[3], "q head dimension does not match k_cache")
    _chk(nq % nh == 0 and nq // nh in _GROUPS, "query heads must be 1, 2, 4 or 8 times the KV heads")
    _chk(nq == nh or DIM == 128, "grouped-query attention needs DIM == 128")
    _chk(T >= 0, "T must be non-negative")
    _chk(bits in (2, 4), "bits must be 2 or 4")
    _chk(bits == 4 or DIM == 128, "2-bit codes need DIM == 128")
    _chk(T // (32 // bits) < n_super_cap, f"k_cache has no free supergroup to append token {T}")
    _chk(DIM in _DIMS, "DIM must be 128, 256 or 512")
    dev = _need_device(q, k_cache, k_new, zp, sc, al, be, tg)

    q_flat = q.contiguous()
    k_new_flat = k_new.reshape(B * nh, DIM).contiguous()
    ld = _pitch(T + 1)
    o = torch.empty((B, nq, ld), dtype=torch.float16, device=dev)
    if state_out is not None:
        _chk(state_out.dtype == torch.float16 and state_out.is_contiguous()
             and state_out.numel() == B * nh * DIM * 2, "state_out must be contiguous fp16 [B,nh,DIM,2]")
    cp, ccap, civ = _ckpt_args(ckpt, ckpt_interval, B, nh, DIM, bits)
    with _lib.device_guard(dev):
        rc = _lib.lib().adkv_forward_qk_gqa(
            q_flat.data_ptr(), k_cache.data_ptr(), k_new_flat.data_ptr(), o.data_ptr(),
            zp.data_ptr(), sc.data_ptr(), al.data_ptr(), be.data_ptr(), tg.data_ptr(),
            B, nq, nh, T, DIM, n_super_cap, bits, ld, _ptr(state_out), cp, ccap, civ,
            _lib.current_stream_ptr(dev))
    _lib.check(rc, "forward_qk")
    return o[:, :, :T + 1]


def forward_ov(
    attn: torch.Tensor,
    v_cache: torch.Tensor,
    v_new: torch.Tensor,
    v_zp: torch.Tensor,
    v_sc: torch.Tensor,
    v_alpha: torch.Tensor,
    v_beta: torch.Tensor,
    v_t: torch.Tensor,
    scale_min: float,
    scale_max: float,
    *,
    state_out: torch.Tensor | None = None,
    ckpt: torch.Tensor | None = None,
    ckpt_interval: int = 0,
    bits: int = 4,
) -> torch.Tensor:
    """Decode-phase OV over the nibble-packed ADKV cache (reference gemv.py:58-97).

    ``o[b,h,c] = sum_t attn[b,h,t] * v_deq[b,h,t,c]`` over the ``T = attn.shape[2]-1`` cached
    tokens plus ``attn[T] * v_deq_new``; ``v_new`` is quantised with the state after token ``T-1``
    and written at position ``T`` in place.

    Returns ``[B, nh, DIM]`` float16.
    """
    _chk(attn.dtype == torch.float16, "attn must be float16")
    _chk(v_new.dtype == torch.float16, "v_new must be float16")
    _chk(v_cache.dtype == torch.uint8, "v_cache must be uint8")
    _chk(v_cache.is_contiguous(), "v_cache must be contiguous (appended in place)")
    B, nq = attn.shape[0], attn.shape[1]
    nh = v_cache.shape[1]
    _chk(attn.shape[2] >= 1, "attn must contain the cached weights plus the self weight")
    T = attn.shape[2] - 1
    n_super_cap, n_cgroup = v_cache.shape[2], v_cache.shape[3]
    DIM = n_cgroup * _TILE
    zp, sc, al, be, tg = _params((v_zp, v_sc, v_alpha, v_beta, v_t),
                                 ("v_zp", "v_sc", "v_alpha", "v_beta", "v_t"), nh, DIM)
    _chk(DIM == v_new.shape[-1], "v_new head dimension does not match v_cache")
    _chk(nq % nh == 0 and nq // nh in _GROUPS, "query heads must be 1, 2, 4 or 8 times the KV heads")
    _chk(nq == nh or DIM == 128, "grouped-query attention needs DIM == 128")
    _chk(T >= 0, "T must be non-negative")
    _chk(bits in (2, 4), "bits must be 2 or 4")
    _chk(bits == 4 or DIM == 128, "2-bit codes need DIM == 128")
    _chk(T // (32 // bits) < n_super_cap, f"v_cache has no free supergroup to append token {T}")
    _chk(DIM in _DIMS, "DIM must be 128, 256 or 512")
    dev = _need_device(attn, v_cache, v_new, zp, sc, al, be, tg)

    attn_flat, ld = _rows_view(attn)
    v_new_flat = v_new.reshape(B * nh, DIM).contiguous()
    o = torch.empty((B * nq, DIM), dtype=torch.float16, device=dev)
    if state_out is not None:
        _chk(state_out.dtype == torch.float16 and state_out.is_contiguous()
             and state_out.numel() == B * nh * DIM * 2, "state_out must be contiguous fp16 [B,nh,DIM,2]")
    cp, ccap, civ = _ckpt_args(ckpt, ckpt_interval, B, nh, DIM, bits)
    L = _lib.lib()
    ws, ws_bytes = None, 0
    if cp is not None:
        ws_bytes = L.adkv_forward_ov_gqa_workspace_bytes(B, nq, nh, T, DIM, ccap, civ)
        if ws_bytes:
            ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=dev)
    with _lib.device_guard(dev):
        rc = L.adkv_forward_ov_gqa(
            attn_flat.data_ptr(), v_cache.data_ptr(), v_new_flat.data_ptr(), o.data_ptr(),
            zp.data_ptr(), sc.data_ptr(), al.data_ptr(), be.data_ptr(), tg.data_ptr(),
            B, nq, nh, T, DIM, n_super_cap, bits, ld, _ptr(state_out), cp, ccap, civ,
            _ptr(ws), ws_bytes, _lib.current_stream_ptr(dev))
    _lib.check(rc, "forward_ov")
    return o.view(attn.shape[0], attn.shape[1], -1)


def encode_kv(
    kv_cache: torch.Tensor,
    kv_new: torch.Tensor,
    kv_zp: torch.Tensor,
    kv_sc: torch.Tensor,
    kv_alpha: torch.Tensor,
    kv_beta: torch.Tensor,
    kv_t: torch.Tensor,
    scale_min: float,
    scale_max: float,
    *,
    state_out: torch.Tensor | None = None,
    ckpt: torch.Tensor | None = None,
    ckpt_interval: int = 0,
) -> torch.Tensor:
    """Prefill: quantise tokens ``[0, T)`` into the uint4-tiled KV cache (reference gemv.py:100-132).

    Replays the ADKV filter from ``(kv_zp, kv_sc)``; token ``t`` goes to byte row ``t/2``, low
    nibble for even ``t`` and high nibble for odd ``t``.  Purely in place; returns ``kv_cache``.
    ``ckpt`` (extension): receives the state before every token ``(j+1)*ckpt_interval <= T``.
    """
    _chk(kv_new.dtype == torch.float16, "kv_new must be float16")
    _chk(kv_cache.dtype == torch.uint8, "kv_cache must be uint8")
    _chk(kv_cache.is_contiguous(), "kv_cache must be contiguous (written in place)")
    B, nh, T, DIM = kv_new.shape
    zp, sc, al, be, tg = _params((kv_zp, kv_sc, kv_alpha, kv_beta, kv_t),
                                 ("kv_zp", "kv_sc", "kv_alpha", "kv_beta", "kv_t"), nh, DIM)
    n_super_cap = kv_cache.shape[2]
    _chk(kv_cache.shape[3] * _TILE == DIM, "kv_cache channel groups do not match kv_new head dim")
    n_super = ((T + 1) // 2 + _TILE - 1) // _TILE
    _chk(n_super <= n_super_cap,
         f"kv_cache capacity too small: need {n_super} supergroups for {T} tokens, have {n_super_cap}")
    _chk(DIM in _DIMS, "DIM must be 128, 256 or 512")
    dev = _need_device(kv_cache, kv_new, zp, sc, al, be, tg)

    kv_new_flat = kv_new.contiguous()
    if state_out is not None:
        _chk(state_out.dtype == torch.float16 and state_out.is_contiguous()
             and state_out.numel() == B * nh * DIM * 2, "state_out must be contiguous fp16 [B,nh,DIM,2]")
    if B * nh * T == 0 and state_out is None:
        return kv_cache
    cp, ccap, civ = _ckpt_args(ckpt, ckpt_interval, B, nh, DIM)
    with _lib.device_guard(dev):
        rc = _lib.lib().adkv_encode_kv_ex(
            kv_cache.data_ptr(), kv_new_flat.data_ptr(),
            zp.data_ptr(), sc.data_ptr(), al.data_ptr(), be.data_ptr(), tg.data_ptr(),
            B, nh, T, DIM, n_super_cap, _ptr(state_out), cp, ccap, civ,
            _lib.current_stream_ptr(dev))
    _lib.check(rc, "encode_kv")
    return kv_cache


def append_kv(
    kv_cache: torch.Tensor,
    kv_new: torch.Tensor,
    kv_zp: torch.Tensor,
    kv_sc: torch.Tensor,
    kv_alpha: torch.Tensor,
    kv_beta: torch.Tensor,
    kv_t: torch.Tensor,
    T0: int,
    state: torch.Tensor,
    *,
    ckpt: torch.Tensor | None = None,
    ckpt_interval: int = 0,
    bits: int = 4,
) -> torch.Tensor:
    """Streaming append (extension; the reference can only append inside forward_qk/forward_ov,
    after an O(T) replay): quantise ``kv_new [B, nh, n, DIM]`` as tokens ``T0 .. T0+n-1``.

    ``state`` ``[B, nh, DIM, 2]`` float16 carries (zp, sc): the state after token ``T0-1`` on entry
    (ignored when ``T0 == 0``), the state after the last new token on return.  The cache ends up
    byte-identical to ``encode_kv`` over all ``T0+n`` tokens.  Returns ``kv_cache``.
    """
    _chk(kv_new.dtype == torch.float16, "kv_new must be float16")
    _chk(kv_cache.dtype == torch.uint8, "kv_cache must be uint8")
    _chk(kv_cache.is_contiguous(), "kv_cache must be contiguous (written in place)")
    B, nh, n, DIM = kv_new.shape
    zp, sc, al, be, tg = _params((kv_zp, kv_sc, kv_alpha, kv_beta, kv_t),
                                 ("kv_zp", "kv_sc", "kv_alpha", "kv_beta", "kv_t"), nh, DIM)
    n_super_cap = kv_cache.shape[2]
    _chk(kv_cache.shape[3] * _TILE == DIM, "kv_cache channel groups do not match kv_new head dim")
    _chk(T0 >= 0, "T0 must be non-negative")
    _chk(bits in (2, 4), "bits must be 2 or 4")
    tps = 32 // bits
    need = (T0 + n + tps - 1) // tps
    _chk(need <= n_super_cap,
         f"kv_cache capacity too small: need {need} supergroups for {T0 + n} tokens, have {n_super_cap}")
    _chk(DIM in _DIMS, "DIM must be 128, 256 or 512")
    _chk(state.dtype == torch.float16 and state.is_contiguous() and state.numel() == B * nh * DIM * 2,
         "state must be contiguous fp16 [B,nh,DIM,2]")
    dev = _need_device(kv_cache, kv_new, zp, sc, al, be, tg, state)
    cp, ccap, civ = _ckpt_args(ckpt, ckpt_interval, B, nh, DIM, bits)
    if n == 0:
        return kv_cache
    x = kv_new.contiguous()
    with _lib.device_guard(dev):
        rc = _lib.lib().adkv_append_kv(
            kv_cache.data_ptr(), x.data_ptr(),
            zp.data_ptr(), sc.data_ptr(), al.data_ptr(), be.data_ptr(), tg.data_ptr(),
            B, nh, T0, n, DIM, n_super_cap, bits, state.data_ptr(), cp, ccap, civ,
            _lib.current_stream_ptr(dev))
    _lib.check(rc, "append_kv")
    return kv_cache


_DT_F16, _DT_BF16 = 1, 2     # ADKV_DT_F16 / ADKV_DT_BF16 of include/adkv_hip.h
_MASK_DT = {torch.float16: _DT_F16, torch.bfloat16: _DT_BF16}     # masks read as they are; any other becomes fp32


def _row_strides(t: torch.Tensor):
    """``(tensor, strides)`` for new rows ``[B, nh, n, DIM]``: ``strides`` is None for a packed
    tensor, a ctypes array of the (batch, head, token) element strides when the library can read
    the rows where they lie (contiguous channels, even strides, 4-byte aligned), else the tensor
    is packed first."""
    if t.is_contiguous():
        # contiguous() would give back a packed tensor that starts between two words as it is
        return (t.clone(memory_format=torch.contiguous_format) if t.data_ptr() & 3 else t), None
    sb, sh, st, sc = t.stride()
    if sc == 1 and st >= t.shape[3] and not ((sb | sh | st) & 1) and not (t.data_ptr() & 3) \
            and min(sb, sh) >= 0:
        return t, (_lib.C.c_int64 * 3)(sb, sh, st)
    return t.contiguous(), None


def append_kv_pair(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    k_params,
    v_params,
    T0: int,
    k_state: torch.Tensor,
    v_state: torch.Tensor,
    *,
    k_ckpt: torch.Tensor | None = None,
    v_ckpt: torch.Tensor | None = None,
    ckpt_interval: int = 0,
    bits: int = 4,
    fresh: bool = False,
) -> None:
    """``append_kv`` for the K and V rows of the same tokens in one launch (the two calls of
    src/adkv/hf/llama_adkv.py:144-153 made together).  Results are byte-identical to two
    ``append_kv`` calls; at small batch the pair takes the time of one tensor because channels are
    the encoder's only parallel axis.  ``k_params`` / ``v_params``: the five ``[nh, DIM]`` fp16
    tensors ``(zp, sc, alpha, beta, quant_target)``.

    ``k_new`` / ``v_new`` ``[B, nh, n, DIM]`` may be float16 or bfloat16 (rounded to fp16 as they
    are read, like the reference's ``.to(torch.float16)``, llama_adkv.py:141-142) and need not be
    packed: a ``[B, n, nh, DIM]`` projection output viewed with the head axis first is read in
    place.

    ``fresh``: the caches, states and checkpoints are uninitialised memory (``torch.empty``) and the
    tokens are their first (``T0 == 0``); the launch also zeroes the slots and checkpoints past them.
    """
    k_params, v_params = tuple(k_params), tuple(v_params)      # read twice: they may be iterators
    rc = _lib.host().append(k_cache, v_cache, k_new, v_new, k_params, v_params, T0, k_state, v_state, k_ckpt,
                            v_ckpt, ckpt_interval, bits, fresh)
    if rc is not None:      # None: something to check, convert or complain about below
        _lib.check(rc, "append_kv_pair")
        return
    _chk(k_new.dtype == v_new.dtype and k_new.dtype in (torch.float16, torch.bfloat16),
         "kv_new must be float16 or bfloat16 (K and V alike)")
    _chk(k_cache.dtype == torch.uint8 and v_cache.dtype == torch.uint8, "kv_cache must be uint8")
    _chk(k_cache.is_contiguous() and v_cache.is_contiguous(),
         "kv_cache must be contiguous (written in place)")
    _chk(k_new.shape == v_new.shape and k_cache.shape == v_cache.shape,
         "K and V must have the same shapes")
    B, nh, n, DIM = k_new.shape
    kp = _params(k_params, ("k_zp", "k_sc", "k_alpha", "k_beta", "k_t"), nh, DIM)
    vp = _params(v_params, ("v_zp", "v_sc", "v_alpha", "v_beta", "v_t"), nh, DIM)
    n_super_cap = k_cache.shape[2]
    _chk(k_cache.shape[3] * _TILE == DIM, "kv_cache channel groups do not match kv_new head dim")
    _chk(T0 >= 0, "T0 must be non-negative")
    _chk(not fresh or (T0 == 0 and n > 0), "a fresh cache starts at token 0")
    _chk(bits in (2, 4), "bits must be 2 or 4")
    tps = 32 // bits
    need = (T0 + n + tps - 1) // tps
    _chk(need <= n_super_cap,
         f"kv_cache capacity too small: need {need} supergroups for {T0 + n} tokens, have {n_super_cap}")
    _chk(DIM in _DIMS, "DIM must be 128, 256 or 512")
    for st in (k_state, v_state):
        _chk(st.dtype == torch.float16 and st.is_contiguous() and st.numel() == B * nh * DIM * 2,
             "state must be contiguous fp16 [B,nh,DIM,2]")
    _chk((k_ckpt is None) == (v_ckpt is None), "give both checkpoint tensors or neither")
    dev = _need_device(k_cache, v_cache, k_new, v_new, *kp, *vp, k_state, v_state)
    kc, ccap, civ = _ckpt_args(k_ckpt, ckpt_interval, B, nh, DIM, bits)
    vc, vcap, _ = _ckpt_args(v_ckpt, ckpt_interval, B, nh, DIM, bits)
    _chk(ccap == vcap, "K and V checkpoint tensors must have the same capacity")
    if n == 0:
        return
    xk, ks = _row_strides(k_new)
    xv, vs = _row_strides(v_new)
    arr = _lib.C.c_void_p * 5
    with _lib.device_guard(dev):
        entry, at = (_lib.lib().adkv_prefill_kv_pair, ()) if fresh else (_lib.lib().adkv_append_kv_pair, (T0,))
        rc = entry(
            k_cache.data_ptr(), v_cache.data_ptr(), xk.data_ptr(), xv.data_ptr(),
            _DT_BF16 if k_new.dtype == torch.bfloat16 else _DT_F16, ks, vs,
            arr(*[t.data_ptr() for t in kp]), arr(*[t.data_ptr() for t in vp]),
            B, nh, *at, n, DIM, n_super_cap, bits, k_state.data_ptr(), v_state.data_ptr(),
            kc, vc, ccap, civ, _lib.current_stream_ptr(dev))
    _lib.check(rc, "append_kv_pair")


def rope_qk(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor
            ) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotary position embedding of ``q [B, Hq, T, D]`` and ``k [B, H, T, D]`` in one launch.

    Bit-identical to ``transformers``' ``apply_rotary_pos_emb(q, k, cos, sin)`` as the attention
    module calls it (src/adkv/hf/llama_adkv.py:336-337): ``x*cos + rotate_half(x)*sin`` with each
    of the three operations rounded to the tensors' type.  fp16 or bf16, all four tensors of one
    type; ``cos`` / ``sin``: ``[B, T, D]`` (or ``[1, T, D]``).  Any batch / head / token strides with
    contiguous channels are read in place; the results are contiguous.
    """
    r = _lib.host().rope_qk(q, k, cos, sin)      # None: something to check, convert or complain about below
    if r is not None:
        if isinstance(r, int):
            _lib.check(r, "rope_qk")
        return r
    _chk(q.dim() == 4 and k.dim() == 4 and cos.dim() == 3 and sin.dim() == 3,
         "q, k must be [B, H, T, D] and cos, sin [B, T, D]")
    B, Hq, T, D = q.shape
    H = k.shape[1]
    _chk(k.shape[0] == B and k.shape[2] == T and k.shape[3] == D, "q and k disagree in shape")
    _chk(q.dtype in (torch.float16, torch.bfloat16), "q must be float16 or bfloat16")
    _chk(k.dtype == q.dtype and cos.dtype == q.dtype and sin.dtype == q.dtype,
         "q, k, cos, sin must share one dtype")
    _chk(cos.shape == sin.shape and cos.shape[1] == T and cos.shape[2] == D and cos.shape[0] in (1, B),
         "cos, sin must be [B, T, D] or [1, T, D]")
    _chk(D % 4 == 0 and B * Hq * T * D > 0, "head dim must be a positive multiple of 4")
    dev = _need_device(q, k, cos, sin)

    def rows(t):        # channels contiguous, even strides, 4-byte aligned base: read in place
        ok = t.stride(-1) == 1 and all(st % 2 == 0 for st in t.stride()[:-1]) and t.data_ptr() % 4 == 0
        return t if ok else t.contiguous()
    q_, k_, c_, s_ = rows(q), rows(k), rows(cos), rows(sin)
    if s_.stride() != c_.stride():
        c_, s_ = c_.contiguous(), s_.contiguous()
    q_out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=dev)
    k_out = torch.empty((B, H, T, D), dtype=q.dtype, device=dev)
    with _lib.device_guard(dev):
        rc = _lib.lib().adkv_rope_qk(
            q_.data_ptr(), k_.data_ptr(), c_.data_ptr(), s_.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
            B, Hq, H, T, D, q_.stride(0), q_.stride(1), q_.stride(2), k_.stride(0), k_.stride(1), k_.stride(2),
            c_.stride(0) if c_.shape[0] == B and B > 1 else 0, c_.stride(1),
            1 if q.dtype == torch.bfloat16 else 0, _lib.current_stream_ptr(dev))
    _lib.check(rc, "rope_qk")
    return q_out, k_out


_NORM_DT = {torch.float32: 0, torch.float16: _DT_F16, torch.bfloat16: _DT_BF16}     # ADKV_DT_*


def _norm_rows(t: torch.Tensor):
    """``t`` if ``adkv_rope_norm_qk`` can read it in place, else a copy: rows contiguous, each at a multiple of 4 elements."""
    ok = t.stride(-1) == 1 and all(st % 4 == 0 for n, st in zip(t.shape[:-1], t.stride()) if n > 1) \
        and t.data_ptr() % (4 * t.element_size()) == 0
    # a copy in memory of its own: contiguous() gives back what is contiguous already, however aligned
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _norm_strides(t: torch.Tensor):
    # of an axis of one element any stride may be given
    return (_lib.C.c_int64 * (t.dim() - 1))(*[st if n > 1 else 0 for n, st in zip(t.shape[:-1], t.stride())])


def _norm_like(t: torch.Tensor):
    """Laid out as ``t`` where the kernels can write that."""
    to = torch.empty_like(t)
    return to if to.stride(-1) == 1 and all(st % 4 == 0 for st in to.stride()[:-1]) else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _rope_norm_forward(q, k, cos, sin, q_weight, k_weight, eps):
    B, Hq, T, D = q.shape
    H, dev = k.shape[1], q.device
    q_out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=dev)
    k_out = torch.empty((B, H, T, D), dtype=q.dtype, device=dev)
    if B * T:
        with _lib.device_guard(dev):
            rc = _lib.lib().adkv_rope_norm_qk(
                q.data_ptr(), k.data_ptr(), cos.data_ptr(), sin.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(),
                q_out.data_ptr(), k_out.data_ptr(), B, Hq, H, T, D, cos.shape[-1], eps, _norm_strides(q), _norm_strides(k),
                _norm_strides(cos), _NORM_DT[q.dtype], _lib.current_stream_ptr(dev))
        _lib.check(rc, "rope_norm_qk")
    return q_out, k_out


class _RopeNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*args[:6])
        ctx.eps = args[6]
        return _rope_norm_forward(*args)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        q, k, cos, sin, q_weight, k_weight = ctx.saved_tensors
        B, Hq, T, D = q.shape
        H, dev = k.shape[1], q.device
        want = ctx.needs_input_grad
        # a side whose result nobody used has no gradient
        made = []
        for i, (x, w) in enumerate(((q, q_weight), (k, k_weight))):
            used = grads[i] is not None
            made.append((_norm_like(x) if used and want[i] else None,
                         (torch.empty_like(w) if B * T else torch.zeros_like(w)) if used and want[4 + i] else None))
        (dq, dwq), (dk, dwk) = made
        if B * T and any(t is not None for t in (dq, dwq, dk, dwk)):
            gq, gk = (None if g is None else _norm_rows(g) for g in grads)
            need = _lib.lib().adkv_rope_norm_qk_backward_workspace_bytes
            at = lambda t: None if t is None else t.data_ptr()
            by = lambda t: None if t is None else _norm_strides(t)
            with _lib.device_guard(dev):
                size = 0
                if dwq is not None or dwk is not None:
                    size = need(D)
                    _lib.check(min(size, 0), "rope_norm_qk")
                workspace = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
                rc = _lib.lib().adkv_rope_norm_qk_backward(
                    at(gq), at(gk), q.data_ptr(), k.data_ptr(), cos.data_ptr(), sin.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(),
                    at(dq), at(dk), at(dwq), at(dwk), B, Hq, H, T, D, cos.shape[-1], ctx.eps, by(gq), by(gk), _norm_strides(q),
                    _norm_strides(k), by(dq), by(dk), _norm_strides(cos), _NORM_DT[q.dtype], at(workspace), size,
                    _lib.current_stream_ptr(dev))
            _lib.check(rc, "rope_norm_qk")
        return dq, dk, None, None, dwq, dwk, None


def rope_norm_qk(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, q_weight: torch.Tensor,
                 k_weight: torch.Tensor, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q [B, Hq, T, D]`` and ``k [B, H, T, D]`` with its weight, then the rotary position
    embedding, in one launch; differentiable.

    ``y = x / sqrt(mean(x*x) + eps) * weight`` of every row, and ``y*cos + rotate_half(y)*sin`` of its first ``R`` channels, the
    others as they are: :func:`rope_qk` for models that norm the heads first.  Computed in fp32 and rounded once.  fp16,
    bf16 or fp32, all six tensors of one type; ``cos`` / ``sin``: ``[B, T, R]`` or ``[1, T, R]``, the weights ``[D]``; ``D`` and ``R`` multiples
    of 8, ``R <= D <= 512``.  Any batch / head / token strides with contiguous channels are read in place; the results are contiguous.
    Gradients reach ``q``, ``k`` and the weights (the latter's summed in fp32, in the same order every time), not the tables; those
    of ``q`` and ``k`` are laid out as ``q`` and ``k`` are.
    """
    r = _lib.host().rope_norm_qk(q, k, cos, sin, q_weight, k_weight, eps)      # None: something to record, check or convert
    if r is not None:
        if isinstance(r, int):
            _lib.check(r, "rope_norm_qk")
        return r
    _chk(q.dim() == 4 and k.dim() == 4 and cos.dim() == 3 and sin.dim() == 3, "q, k must be [B, H, T, D] and cos, sin [B, T, R]")
    B, Hq, T, D = q.shape
    H, R = k.shape[1], cos.shape[-1]
    _chk(k.shape[0] == B and k.shape[2] == T and k.shape[3] == D, "q and k disagree in shape")
    _chk(q.dtype in _NORM_DT, "q must be float16, bfloat16 or float32")
    _chk(all(t.dtype == q.dtype for t in (k, cos, sin, q_weight, k_weight)), "q, k, cos, sin and the weights must share one dtype")
    _chk(cos.shape == sin.shape and cos.shape[1] == T and cos.shape[0] in (1, B), "cos, sin must be [B, T, R] or [1, T, R]")
    _chk(0 < D <= 512 and D % 8 == 0, "head dim must be a multiple of 8 up to 512")
    _chk(0 < R <= D and R % 8 == 0, "cos, sin must have a multiple of 8 channels, head dim at most")
    _chk(q_weight.shape == (D,) and k_weight.shape == (D,), "the weights must be [head dim]")
    _chk(Hq > 0 and H > 0, "q and k must have heads")
    _chk(not (torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad)), "cos and sin have no gradient")
    _chk(all(forward_ad.unpack_dual(t).tangent is None for t in (q, k, cos, sin, q_weight, k_weight)), "rope_norm_qk has no forward derivatives")
    _need_device(q, k, cos, sin, q_weight, k_weight)
    # copies where there have to be any are made here, where autograd sees them
    q, k, cos, sin, q_weight, k_weight = (_norm_rows(t) for t in (q, k, cos, sin, q_weight, k_weight))
    if sin.shape[0] * T and _norm_strides(sin)[:] != _norm_strides(cos)[:]:
        cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
    wanted = torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, q_weight, k_weight))
    return (_RopeNorm.apply if wanted else _rope_norm_forward)(q, k, cos, sin, q_weight, k_weight, float(eps))


_PROMPT_MASK_DT = {torch.float32: 0, torch.float16: _DT_F16, torch.bfloat16: _DT_BF16, torch.bool: 3}     # ADKV_DT_*


def _no_derivatives(name: str, *tensors: torch.Tensor) -> None:
    _chk(not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)), f"{name} has no gradient")
    _chk(all(forward_ad.unpack_dual(t).tangent is None for t in tensors), f"{name} has no forward derivatives")


def _prompt_rows(t: torch.Tensor):
    """``t`` if ``adkv_prompt_attention`` can read it in place, else a copy; and its strides."""
    ok = t.stride(3) == 1 and all(st % 8 == 0 for n, st in zip(t.shape[:3], t.stride()) if n > 1) \
        and t.data_ptr() % 16 == 0 and (t.shape[2] == 1 or t.stride(2) < 1 << 23)
    t = t if ok else t.clone(memory_format=torch.contiguous_format)
    return t, _stride3(t)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scaling: float, mask: torch.Tensor | None = None, *,
                     bounds: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over the dense rows of a prompt, as prefill and the evaluation model need it: ``q [B, Hq, Tq, D]`` are the last
    ``Tq`` of ``Tk`` tokens, ``k``, ``v`` ``[B, H, Tk, D]``; returns ``[B, Tq, Hq, D]`` in their type.

    ``out_i = sum_t softmax(scaling * q_i . k_t + mask_it) v_t`` over every token ``t`` up to query ``i``'s own; rows that look at nothing are
    zeros.  (The reference calls transformers' attention here, src/adkv/hf/llama_adkv.py:365-378; queries of a single token over many are
    its evaluation model's steps, src/adkv/hf/llama_adkv_eval.py:400-420.)

    Args:
        q, k, v: float16 or bfloat16, ``H`` dividing ``Hq``, ``D`` a multiple of 8 up to 256; any batch / head / token strides with
            contiguous channels are read in place where rows are 16-byte aligned, and copied first where not.
        mask: ``[B or 1, Hq or 1, Tq or 1, Tk]``, boolean (true where a token is looked at) or additive (any float type; minus infinity hides a
            token whatever its key and value hold, a row of nothing but the type's lowest value looks at all tokens up to its own alike).
        bounds: ``n`` sequences of different lengths share the row axis (``B == 1``, ``Tq == Tk``, no mask): int32 ``[n + 1]``, ascending, sequence
            ``i`` is rows ``bounds[i] .. bounds[i+1]-1`` and looks at itself only; rows of no sequence are zeros.  On the device the values are
            not checked (that would wait for it); what is read and written stays inside the tensors whatever they are.  On the
            host they are checked and copied.

    No gradient: refused where one is wanted.  Weights are rounded to the tensors' type; scores, sums and outputs are fp32.
    """
    r = _lib.host().prompt_attention(q, k, v, scaling, mask, bounds)      # None: something to check, convert or complain about below
    if r is not None:
        if isinstance(r, int):
            _lib.check(r, "prompt_attention")
        return r
    _chk(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q must be [B, Hq, Tq, D], k and v [B, H, Tk, D]")
    B, Hq, Tq, D = q.shape
    H, Tk = k.shape[1], k.shape[2]
    _chk(k.shape == (B, H, Tk, D) and v.shape == k.shape, "q, k and v disagree in shape")
    _chk(q.dtype in (torch.float16, torch.bfloat16), "q must be float16 or bfloat16")
    _chk(k.dtype == q.dtype and v.dtype == q.dtype, "q, k and v must share one dtype")
    _chk(0 < D <= 256 and D % 8 == 0, "head dim must be a multiple of 8 up to 256")
    _chk(H > 0 and Hq > 0 and Hq % H == 0, "the number of query heads must be a multiple of that of KV heads")
    _chk(Tq <= Tk, "the queries are the last of the tokens: there cannot be more of them")
    _no_derivatives("prompt_attention", q, k, v)
    n_seq = 0
    if bounds is not None:
        _chk(B == 1 and Tq == Tk and mask is None, "packed sequences need B == 1, as many queries as keys and no mask")
        _chk(bounds.dim() == 1 and bounds.numel() >= 1 and not bounds.is_floating_point(), "bounds must be [n + 1] whole numbers")
        n_seq = bounds.numel() - 1
        if not bounds.is_cuda:
            e = bounds.tolist()
            _chk(0 <= e[0] and e[-1] <= Tq and all(x <= y for x, y in zip(e, e[1:])), "bounds must ascend within the rows")
    if mask is not None:
        _chk(mask.dim() == 4 and mask.shape[3] == Tk and mask.shape[0] in (1, B) and mask.shape[1] in (1, Hq) and mask.shape[2] in (1, Tq),
             "mask must broadcast to [B, Hq, Tq, Tk]")
        _chk(mask.dtype == torch.bool or mask.is_floating_point(), "mask must be boolean or additive")
        _no_derivatives("prompt_attention", mask)
    dev = _need_device(q, k, v)
    out = torch.empty((B, Tq, Hq, D), dtype=q.dtype, device=dev)
    if out.numel() == 0:
        return out
    if bounds is not None:
        if n_seq == 0:
            return out.zero_()
        bounds = bounds.to(device=dev, dtype=torch.int32).contiguous()
    mst, mdt = None, 0
    if mask is not None:
        mdt = _PROMPT_MASK_DT.get(mask.dtype, 0)
        if mask.dtype == torch.float64:        # its lowest value is no minus infinity in fp32 either
            most = torch.finfo(torch.float32).max
            mask = torch.where(mask.isinf(), mask, mask.clamp(-most, most))
        mask = mask.to(device=dev, dtype=mask.dtype if mask.dtype in _PROMPT_MASK_DT else torch.float32)
        if mask.stride(3) != 1 and Tk > 1:
            mask = mask.contiguous()
        mst = _stride3(mask)
    (q, qs), (k, ks), (v, vs) = _prompt_rows(q), _prompt_rows(k), _prompt_rows(v)
    L = _lib.lib()
    with _lib.device_guard(dev):
        size = L.adkv_prompt_attention_workspace_bytes(B, Hq, H, Tq, Tk, D, n_seq)
        _lib.check(min(size, 0), "prompt_attention")
        workspace = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        rc = L.adkv_prompt_attention(q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, _ptr(mask), mst, float(scaling), _ptr(bounds),
                                     n_seq, out.data_ptr(), B, Hq, H, Tq, Tk, D,
                                     (_DT_BF16 if q.dtype == torch.bfloat16 else _DT_F16) | mdt << 8, _ptr(workspace), size,
                                     _lib.current_stream_ptr(dev))
    _lib.check(rc, "prompt_attention")
    return out


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns, shaped as the tokens are; ``top_*`` have one more axis (None without ``top``)."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor | None = None
    top_tokens: torch.Tensor | None = None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """Log probabilities of ``tokens [...]`` under ``softmax(logits [..., V])``, the rows' entropy (nats) and their ``top`` likeliest
    tokens, in one pass over the logits (what the reference's evaluation, tools/lm_eval_adkv.py, asks its model for).

    Logits: float16, bfloat16 or float32, read in place whatever the strides of up to two leading axes are.  Tokens: whole numbers; a negative one
    stands for none (its log probability is 0), one from ``V`` on gives NaN.  ``top``: 0 to 32; equal logits come lowest token first.
    Everything is computed in fp32 or more and returned in fp32 (``top_tokens`` int64), with the digits of probabilities near one kept.  Minus
    infinity is a probability of zero; a row with a NaN or plus infinity, or of nothing but minus infinity, gives NaN, and its
    likeliest tokens in order, NaN first.  No gradient: refused where one is wanted.
    """
    r = _lib.host().token_logprobs(logits, tokens, top)      # None: something to check, convert or complain about below
    if r is not None:
        if isinstance(r, int):
            _lib.check(r, "token_logprobs")
        return TokenLogprobs(*r)
    _chk(logits.dim() >= 1 and tokens.shape == logits.shape[:-1], "tokens must have the shape of logits without its last axis")
    V = logits.shape[-1]
    _chk(logits.dtype in _NORM_DT, "logits must be float16, bfloat16 or float32")
    _chk(not (tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool), "tokens must be whole numbers")
    _chk(V > 0, "logits must have at least one column")
    _chk(0 <= top <= 32 and top <= V, "top must be 0 to 32, and at most the vocabulary")
    _no_derivatives("token_logprobs", logits)
    dev = _need_device(logits, tokens)
    shape = tokens.shape
    made = lambda *s, dtype=torch.float32: torch.empty((*shape, *s), dtype=dtype, device=dev)
    out = TokenLogprobs(made(), made(), *((made(top), made(top, dtype=torch.int64)) if top else ()))
    if out.logprobs.numel() == 0:
        return out
    x = logits if logits.stride(-1) == 1 or V == 1 else logits.contiguous()
    x = x.reshape(1, -1, V) if x.dim() < 3 else x if x.dim() == 3 else x.reshape(1, -1, V)
    tokens = tokens.to(torch.int64).contiguous()
    with _lib.device_guard(dev):
        rc = _lib.lib().adkv_token_logprobs(
            x.data_ptr(), x.stride(0) if x.shape[0] > 1 else 0, x.stride(1) if x.shape[1] > 1 else 0, tokens.data_ptr(), x.shape[0], x.shape[1], V,
            _NORM_DT[x.dtype], top, *[_ptr(t) for t in out], _lib.current_stream_ptr(dev))
    _lib.check(rc, "token_logprobs")
    return out


def take_sequences(tensors, index: torch.Tensor, *, used=None, into=None) -> None:
    """Sequences of a cache copied over one another: row ``r`` of every tensor becomes what its row ``index[r]`` was (extension: the reference's
    cache cannot be reordered).  Beams that go on from another one, finished sequences that leave a batch (the first ``len(index)`` rows are then
    what is left), one prompt that several answers begin with.

    Args:
        tensors: any number of contiguous tensors ``[B, H, n, ...]`` of one device, a cache's codes, checkpoints and states, of one layer or of all:
            one or two launches for all of them.  They begin at multiples of 16 bytes, and a head's entries (``[n, ...]``), those that are used too, are
            such multiples.
        index: ``[R]`` whole numbers, ``R <= 1024``; the same one may come several times.  On the device they are not checked (that would wait for it): a
            row whose index is none of the rows stays as it is, or is zeros in ``into``.  On the host they are checked and copied.
        used: how many entries along the third axis hold anything, one number per tensor (all): what is behind them is neither read nor written.
        into: as many tensors ``[R, H, m, ...]``, ``m >= used``, to write instead, which share no memory with ``tensors``; what is behind the entries that are
            used becomes zero.  Without it ``R <= B``, rows may be one another's sources in any way, and no two tensors may share memory
            (refused).
    """
    tensors = list(tensors)
    used = None if used is None else list(used)
    into = None if into is None else list(into)
    rc = _lib.host().take_sequences(tensors, index, used, into)      # None: something to check, convert or complain about below
    if rc is not None:
        _lib.check(rc, "take_sequences")
        return
    _chk(index.dim() == 1 and not (index.is_floating_point() or index.is_complex() or index.dtype == torch.bool), "index must be [R] whole numbers")
    R = index.shape[0]
    _chk(R <= 1024, "at most 1024 sequences")
    used = [None] * len(tensors) if used is None else used
    _chk(len(used) == len(tensors), "used must have a number for every tensor")
    _chk(into is None or len(into) == len(tensors), "into must have a tensor for every tensor")
    if not tensors:
        return
    B = tensors[0].shape[0] if tensors[0].dim() else 0
    _chk(into is not None or R <= B, "in place there are at most as many sequences as before")
    rows = []
    for i, t in enumerate(tensors):
        _chk(t.dim() >= 3 and t.shape[0] == B and t.is_contiguous(), "tensors must be contiguous [B, H, n, ...]")
        entry = t.element_size() * math.prod(t.shape[3:])
        n = t.shape[2] if used[i] is None else int(used[i])
        _chk(0 <= n <= t.shape[2], "used must be between 0 and the third axis's length")
        _chk(t.shape[2] * entry % 16 == 0 and n * entry % 16 == 0 and t.data_ptr() % 16 == 0, "heads and what is used of them must be multiples of 16 bytes")
        _no_derivatives("take_sequences", t)
        if into is None:
            if t.numel():
                rows.append(_lib.Rows(t.data_ptr(), None, t.shape[1], t.shape[2] * entry, 0, n * entry))
        else:
            to = into[i]
            _chk(to.dtype == t.dtype and to.dim() == t.dim() and to.shape[0] == R and to.shape[1] == t.shape[1] and to.shape[2] >= n
                 and to.shape[3:] == t.shape[3:] and to.is_contiguous() and to.data_ptr() % 16 == 0 and to.shape[2] * entry % 16 == 0,
                 "into must be contiguous [R, H, m, ...] of the tensors' types, with room for what is used")
            _chk(to.numel() == 0 or t.numel() == 0 or to.data_ptr() + to.numel() * to.element_size() <= t.data_ptr()
                 or t.data_ptr() + t.numel() * t.element_size() <= to.data_ptr(), "into must not share memory with the tensors")
            _no_derivatives("take_sequences", to)
            if to.numel():       # nothing is read where nothing is used
                rows.append(_lib.Rows((t if t.numel() else to).data_ptr(), to.data_ptr(), t.shape[1], t.shape[2] * entry, to.shape[2] * entry, n * entry))
    if not index.is_cuda:
        _chk(all(0 <= r < B for r in index.tolist()), "index must be of the sequences")
    dev = _need_device(*tensors, *(into or ()))
    if B == 0:                   # no row is one of none
        for to in into or ():
            to.zero_()
    if R == 0 or B == 0 or not rows:
        return
    index = index.to(device=dev, dtype=torch.int64).contiguous()
    with _lib.device_guard(dev):
        rc = _lib.lib().adkv_take_sequences((_lib.Rows * len(rows))(*rows), len(rows), index.data_ptr(), R, B, _lib.current_stream_ptr(dev))
    _lib.check(rc, "take_sequences")


def softmax_scale_mask(logits: torch.Tensor, scaling: float,
                       mask: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(logits.float()*scaling + mask) -> fp16`` in one launch.

    Fuses the element-wise chain the reference runs in torch between the two GEMVs
    (src/adkv/hf/llama_adkv.py:266-271).  ``logits``: fp16 ``[B, nh, n]``; ``mask``: optional
    ``[B, 1, n]`` / ``[B, nh, n]`` / ``[B, 1, 1, n]`` additive mask (any float dtype).
    """
    _chk(logits.dtype == torch.float16, "logits must be float16")
    _chk(logits.dim() == 3, "logits must be [B, nh, n]")
    B, nh, n = logits.shape
    dev = _need_device(logits)
    lg, ld = _rows_view(logits)
    out = torch.empty((B, nh, ld), dtype=torch.float16, device=dev)[:, :, :n]
    rpm, mptr = 1, None
    mk = None
    if mask is not None:
        mk = mask[:, :, 0, :] if mask.dim() == 4 else mask
        _chk(mk.dim() == 3 and mk.shape[0] == B and mk.shape[2] == n and mk.shape[1] in (1, nh),
             "mask must broadcast to [B, nh, n]")
        rpm = nh if mk.shape[1] == 1 else 1
        mk = mk.to(device=dev, dtype=torch.float32).contiguous()
        mptr = mk.data_ptr()
    L = _lib.lib()
    wsb = L.adkv_softmax_workspace_bytes(B * nh, n)
    ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
    with _lib.device_guard(dev):
        rc = L.adkv_softmax_ex(lg.data_ptr(), out.data_ptr(), mptr, B * nh, n, ld, rpm, float(scaling),
                               _ptr(ws), wsb, _lib.current_stream_ptr(dev))
    _lib.check(rc, "softmax_scale_mask")
    return out


def decode_step(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    k_params,
    v_params,
    T: int,
    scaling: float,
    mask: torch.Tensor | None = None,
    *,
    k_ckpt: torch.Tensor | None = None,
    v_ckpt: torch.Tensor | None = None,
    ckpt_interval: int = 0,
    bits: int = 4,
    workspace: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """One decode-attention step of a layer through a single library call.

    The body of the reference's ``KVCacheLayer_ADKV.decode`` (src/adkv/hf/llama_adkv.py:245-276):
    ``forward_qk`` -> ``softmax(logits*scaling + mask)`` -> ``forward_ov``, with ``k_new`` / ``v_new``
    appended at slot ``T`` of both caches.  ``k_params`` / ``v_params`` are the five ``[nh, DIM]``
    fp16 tensors ``(zp, sc, alpha, beta, quant_target)``.  Returns ``(out [B,nh,DIM] fp16,
    weights [B,nh,T+1] fp16)``.  ``q``, ``k_new`` and ``v_new`` may all be bfloat16: the kernels
    round them to fp16 as they read them and return ``out`` in bfloat16, with the values of the
    reference's ``.to(torch.float16)`` / ``.to(q.dtype)`` around its kernels
    (llama_adkv.py:248-250, 274) but without those launches.  ``workspace`` (uint8, 256-byte aligned, sized by
    ``decode_step_workspace_bytes``) may be passed to avoid the per-call allocation.
    """
    f16, u8 = torch.float16, torch.uint8
    act = q.dtype            # float16 as in the reference, or bfloat16 (extension; see the docstring)
    if not (act in (f16, torch.bfloat16) and k_new.dtype == act and v_new.dtype == act
            and k_cache.dtype == u8 and v_cache.dtype == u8 and k_cache.is_contiguous()
            and v_cache.is_contiguous()):
        for t, n in ((q, "q"), (k_new, "k_new"), (v_new, "v_new")):
            _chk(t.dtype == (act if act == torch.bfloat16 else f16),
                 f"{n} must be float16" + (" (or bfloat16 like q)" if act == torch.bfloat16 else ""))
        for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            _chk(t.dtype == u8, f"{n} must be uint8")
            _chk(t.is_contiguous(), f"{n} must be contiguous (appended in place)")
    _chk(k_cache.shape == v_cache.shape, "k_cache and v_cache shapes differ")
    B, nq, nh = q.shape[0], q.shape[1], k_cache.shape[1]
    n_super_cap, DIM = k_cache.shape[2], k_cache.shape[3] * _TILE
    _chk(nq % nh == 0 and nq // nh in _GROUPS, "query heads must be 1, 2, 4 or 8 times the KV heads")
    _chk(nq == nh or DIM == 128, "grouped-query attention needs DIM == 128")
    kp = _params(k_params, ("k_zp", "k_sc", "k_alpha", "k_beta", "k_t"), nh, DIM)
    vp = _params(v_params, ("v_zp", "v_sc", "v_alpha", "v_beta", "v_t"), nh, DIM)
    _chk(DIM == q.shape[-1], "q head dimension does not match k_cache")
    _chk(T >= 0, "T must be non-negative")
    _chk(bits in (2, 4), "bits must be 2 or 4")
    _chk(bits == 4 or DIM == 128, "2-bit codes need DIM == 128")
    if not T // (32 // bits) < n_super_cap:
        raise RuntimeError(f"k_cache has no free supergroup to append token {T}")
    _chk(DIM in _DIMS, "DIM must be 128, 256 or 512")
    dev = _need_device(q, k_cache, v_cache, k_new, v_new, *kp, *vp)
    n = T + 1
    rpm, mptr, mk, mdt = 1, None, None, 0
    if mask is not None:
        mk = mask[:, :, 0, :] if mask.dim() == 4 else mask
        _chk(mk.dim() == 3 and mk.shape[0] == B and mk.shape[2] == n and mk.shape[1] in (1, nq),
             "mask must broadcast to [B, nh, n]")
        rpm = nq if mk.shape[1] == 1 else 1
        mdt = _MASK_DT.get(mk.dtype, 0)
        mk = mk.to(device=dev, dtype=mk.dtype if mdt else torch.float32).contiguous()
        mptr = mk.data_ptr()
    kcp, ccap, civ = _ckpt_args(k_ckpt, ckpt_interval, B, nh, DIM, bits)
    vcp, vcap, _ = _ckpt_args(v_ckpt, ckpt_interval, B, nh, DIM, bits)
    _chk((k_ckpt is None) == (v_ckpt is None) and ccap == vcap,
         "k_ckpt and v_ckpt must both be given, with the same capacity, or both omitted")
    L = _lib.lib()
    if workspace is None:
        need = L.adkv_decode_step_workspace_bytes(B, nq, nh, T, DIM, ccap, civ)
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    # a caller's workspace is sized against the launch by the library itself ("workspace too small")
    _chk(workspace.dtype == torch.uint8 and workspace.is_cuda, "workspace must be a uint8 device tensor")
    qf = q.contiguous()
    knf = k_new.reshape(B * nh, DIM).contiguous()
    vnf = v_new.reshape(B * nh, DIM).contiguous()
    out = torch.empty((B, nq, DIM), dtype=act, device=dev)
    wld = _row_pitch(n)
    weights = torch.empty((B, nq, wld), dtype=torch.float16, device=dev)
    arr = _lib.C.c_void_p * 5
    with _lib.device_guard(dev):
        rc = L.adkv_decode_step(
            qf.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), knf.data_ptr(), vnf.data_ptr(),
            arr(*[t.data_ptr() for t in kp]), arr(*[t.data_ptr() for t in vp]),
            mptr, rpm, float(scaling), out.data_ptr(), weights.data_ptr(), wld,
            B, nq, nh, T, DIM, n_super_cap, bits, (_DT_BF16 if act == torch.bfloat16 else _DT_F16) | mdt << 8,
            kcp, vcp, ccap, civ,
            workspace.data_ptr(), workspace.numel(), _lib.current_stream_ptr(dev))
    _lib.check(rc, "decode_step")
    return out, weights[:, :, :n]


def decode_step_workspace_bytes(B: int, nq: int, nh: int, T: int, DIM: int, n_ckpt_cap: int = 0,
                                 ckpt_interval: int = 0) -> int:
    """Bytes ``decode_step`` needs for ``nq`` query heads over ``nh`` KV heads."""
    return int(_lib.lib().adkv_decode_step_workspace_bytes(B, nq, nh, T, DIM, n_ckpt_cap,
                                                            ckpt_interval))


class SharedPrefix(NamedTuple):
    """Codes of tokens that every sequence of a batch begins with, held once (extension: ``extend``): caches and checkpoints of one
    sequence, ``[1, nh, ...]``, of which the first ``tokens`` tokens are meant, and the parameters that they were quantised with.
    The sequences' own streams go on from the state behind the last of them (``append_kv``'s ``state``, ``forward_qk``'s
    ``state_out``): their parameters are these with that state's zp and sc in place of the first two."""
    k_cache: torch.Tensor
    v_cache: torch.Tensor
    tokens: int
    k_params: tuple
    v_params: tuple
    k_ckpt: torch.Tensor | None = None
    v_ckpt: torch.Tensor | None = None


def _stride3(t: torch.Tensor):
    """Element strides of the first three of four axes, 0 along an axis of length one."""
    return (_lib.C.c_int64 * 3)(*[st if n > 1 else 0 for st, n in zip(t.stride()[:3], t.shape[:3])])


def extend(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    k_params,
    v_params,
    T: int,
    scaling: float,
    mask: torch.Tensor | None = None,
    *,
    prefix: SharedPrefix | None = None,
    k_ckpt: torch.Tensor | None = None,
    v_ckpt: torch.Tensor | None = None,
    ckpt_interval: int = 0,
    bits: int = 4,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """``n >= 1`` new tokens of every sequence at once: quantised into slots ``T .. T+n-1`` of both caches (codes as ``append_kv``
    writes them) and attended with, each over the prefix, the cached tokens and the new ones up to itself.

    The reference takes tokens one at a time (src/adkv/hf/llama_adkv.py:235-276); ``n`` calls of ``decode_step`` write the same
    codes and give the same outputs up to rounding (scores stay fp32 here; a new token's value is what every later call reads).

    Args:
        q: ``[B, Hq, n, 128]`` float16 or bfloat16, 1, 2, 4 or 8 query heads per KV head; any strides with contiguous channels.
        k_new, v_new: ``[B, nh, n, 128]`` of the same type, strided likewise.
        k_params, v_params: the five ``[nh, 128]`` fp16 tensors; with a prefix zp and sc are the state behind its last token.
        mask: additive, ``[B or 1, Hq or 1, n or 1, P+T+n]`` (or three axes, ``[B or 1, Hq or 1, P+T+n]``, for all n alike), columns in the
            order prefix, own tokens.  fp16, bfloat16 and fp32 are read in place.  Later tokens are hidden without it.
        prefix: tokens that the whole batch begins with; its checkpoints are every ``ckpt_interval`` tokens too.
        workspace: uint8, 256-byte aligned, ``extend_workspace_bytes`` long, to avoid the per-call allocation.

    Returns ``[B, n, Hq, 128]`` in ``q``'s type.  Rows that the mask leaves nothing of are NaN.
    """
    k_params, v_params = tuple(k_params), tuple(v_params)
    if workspace is None:
        r = _lib.host().extend(q, k_cache, v_cache, k_new, v_new, k_params, v_params, T, scaling, mask, prefix, k_ckpt, v_ckpt,
                               ckpt_interval, bits)
        if r is not None:      # None: something to check, convert or complain about below
            if isinstance(r, int):
                _lib.check(r, "extend")
            return r
    act = q.dtype
    _chk(act in (torch.float16, torch.bfloat16), "q must be float16 or bfloat16")
    _chk(k_new.dtype == act and v_new.dtype == act, "k_new and v_new must have q's type")
    _chk(q.dim() == 4 and k_new.dim() == 4 and k_new.shape == v_new.shape, "q must be [B, Hq, n, DIM], k_new and v_new [B, nh, n, DIM]")
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _chk(t.dtype == torch.uint8 and t.dim() == 6, f"{name} must be uint8 [B, nh, n_super_cap, DIM/4, 4, 4]")
        _chk(t.is_contiguous(), f"{name} must be contiguous (appended in place)")
    _chk(k_cache.shape == v_cache.shape, "k_cache and v_cache shapes differ")
    B, nq, n, DIM = q.shape
    nh, n_super_cap = k_cache.shape[1], k_cache.shape[2]
    _chk(k_new.shape == (B, nh, n, DIM) and k_cache.shape[0] == B and k_cache.shape[3:] == (DIM // _TILE, 4, 4),
         "q, k_new, v_new and the caches disagree in shape")
    _chk(DIM == 128, "extend needs DIM == 128")
    _chk(nh > 0 and nq % nh == 0 and nq // nh in _GROUPS, "query heads must be 1, 2, 4 or 8 times the KV heads")
    _chk(B > 0 and n > 0, "extend needs at least one sequence and one new token")
    _chk(T >= 0, "T must be non-negative")
    _chk(bits in (2, 4), "bits must be 2 or 4")
    tps = 32 // bits
    _chk(-(-(T + n) // tps) <= n_super_cap, f"k_cache has no room for {T + n} tokens")
    kp = _params(k_params, ("k_zp", "k_sc", "k_alpha", "k_beta", "k_t"), nh, DIM)
    vp = _params(v_params, ("v_zp", "v_sc", "v_alpha", "v_beta", "v_t"), nh, DIM)
    _chk((k_ckpt is None) == (v_ckpt is None), "give both checkpoint tensors or neither")
    kcp, ccap, civ = _ckpt_args(k_ckpt, ckpt_interval, B, nh, DIM, bits)
    vcp, vcap, _ = _ckpt_args(v_ckpt, ckpt_interval, B, nh, DIM, bits)
    _chk(ccap == vcap, "K and V checkpoint tensors must have the same capacity")
    tensors = [q, k_cache, v_cache, k_new, v_new, *kp, *vp] + ([k_ckpt, v_ckpt] if k_ckpt is not None else [])
    arr = _lib.C.c_void_p * 5
    P = pcap = piv = 0
    pre = None
    if prefix is not None:
        P = int(prefix.tokens)
        _chk(P >= 0, "a prefix cannot have a negative number of tokens")
        for t in (prefix.k_cache, prefix.v_cache):
            _chk(t.dtype == torch.uint8 and t.is_contiguous() and t.dim() == 6 and t.shape[:2] == (1, nh) and t.shape[3:] == (DIM // _TILE, 4, 4),
                 "a prefix's caches must be contiguous uint8 [1, nh, n_super, DIM/4, 4, 4]")
        _chk(prefix.k_cache.shape == prefix.v_cache.shape and -(-P // tps) <= prefix.k_cache.shape[2], "the prefix's caches do not hold its tokens")
        pkp = _params(tuple(prefix.k_params), ("k_zp", "k_sc", "k_alpha", "k_beta", "k_t"), nh, DIM)
        pvp = _params(tuple(prefix.v_params), ("v_zp", "v_sc", "v_alpha", "v_beta", "v_t"), nh, DIM)
        _chk((prefix.k_ckpt is None) == (prefix.v_ckpt is None), "give both of the prefix's checkpoint tensors or neither")
        pkc, pcap, piv = _ckpt_args(prefix.k_ckpt, ckpt_interval, 1, nh, DIM, bits)
        pvc, pvcap, _ = _ckpt_args(prefix.v_ckpt, ckpt_interval, 1, nh, DIM, bits)
        _chk(pcap == pvcap, "the prefix's checkpoint tensors must have the same capacity")
        tensors += [prefix.k_cache, prefix.v_cache, *pkp, *pvp] + ([prefix.k_ckpt, prefix.v_ckpt] if prefix.k_ckpt is not None else [])
        pk, pv = arr(*[t.data_ptr() for t in pkp]), arr(*[t.data_ptr() for t in pvp])
        if P > 0 and prefix.k_cache.shape[2] > 0:
            pre = _lib.Prefix(prefix.k_cache.data_ptr(), prefix.v_cache.data_ptr(), _lib.C.cast(pk, _lib.C.c_void_p),
                              _lib.C.cast(pv, _lib.C.c_void_p), pkc, pvc, P, prefix.k_cache.shape[2], pcap, piv)
    if mask is not None:
        _chk(mask.dtype != torch.bool, "mask must be additive, not boolean")
        mask = mask[:, :, None] if mask.dim() == 3 else mask
        _chk(mask.dim() == 4 and mask.shape[3] == P + T + n and mask.shape[0] in (1, B) and mask.shape[1] in (1, nq) and mask.shape[2] in (1, n),
             "mask must broadcast to [B, nh, n, P + T + n]")
    dev = _need_device(*tensors)
    mst, mdt = None, 0
    if mask is not None:
        mdt = _MASK_DT.get(mask.dtype, 0)
        mask = mask.to(device=dev, dtype=mask.dtype if mdt else torch.float32)
        if mask.stride(3) != 1 and mask.shape[3] > 1:
            mask = mask.contiguous()
        mst = _stride3(mask)
    if q.stride(3) != 1 or any(st % 2 for st, k in zip(q.stride()[:3], q.shape[:3]) if k > 1) or q.data_ptr() % 4:
        q = q.clone(memory_format=torch.contiguous_format)     # also where it is packed, but starts between two words
    xk, ks = _row_strides(k_new)
    xv, vs = _row_strides(v_new)
    if workspace is None:
        with _lib.device_guard(dev):       # the size depends on the device
            workspace = torch.empty(extend_workspace_bytes(B, nq, nh, T, n, ccap, ckpt_interval, P, pcap), dtype=torch.uint8, device=dev)
    _chk(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.device == dev, "workspace must be a uint8 tensor on the same device")
    out = torch.empty((B, n, nq, DIM), dtype=act, device=dev)
    with _lib.device_guard(dev):
        rc = _lib.lib().adkv_extend(
            q.data_ptr(), _stride3(q), k_cache.data_ptr(), v_cache.data_ptr(), xk.data_ptr(), xv.data_ptr(), ks, vs,
            arr(*[t.data_ptr() for t in kp]), arr(*[t.data_ptr() for t in vp]), _ptr(mask), mst, float(scaling), out.data_ptr(),
            B, nq, nh, T, n, DIM, n_super_cap, bits, (_DT_BF16 if act == torch.bfloat16 else _DT_F16) | mdt << 8,
            kcp, vcp, ccap, civ, None if pre is None else _lib.C.addressof(pre), workspace.data_ptr(), workspace.numel(),
            _lib.current_stream_ptr(dev))
    _lib.check(rc, "extend")
    return out


def extend_workspace_bytes(B: int, nq: int, nh: int, T: int, n: int, n_ckpt_cap: int = 0, ckpt_interval: int = 0, P: int = 0,
                           prefix_n_ckpt_cap: int = 0) -> int:
    """Bytes ``extend`` needs for ``n`` new tokens behind ``T`` cached ones and a prefix of ``P``; ``ckpt_interval`` is that of whichever has
    checkpoints (a capacity above 0), as in ``extend``."""
    return int(_lib.lib().adkv_extend_workspace_bytes(B, nq, nh, T, n, n_ckpt_cap, ckpt_interval, P, prefix_n_ckpt_cap,
                                                      ckpt_interval if prefix_n_ckpt_cap else 0))

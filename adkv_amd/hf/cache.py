"""Per-layer packed ADKV KV cache: the host-side owner of the code buffers.

Counterpart of the reference's ``KVCacheLayer_ADKV`` / ``KVCache_ADKV``
(src/adkv/hf/llama_adkv.py:44-288) with the same public names, method signatures, buffer layout
``[B, H, n_super, C // 4, 4, 4]`` uint8 and error behaviour, so code written against the
reference's cache object works unchanged.  What differs is underneath:

* the three kernels are the gfx950 ones (``adkv_amd.kernel.gemv``), launched on the current stream;
* the scale/mask/softmax chain between QK and OV is one fused launch instead of five torch ops;
* capacity grows geometrically (the reference reallocates and copies both caches every 64 tokens,
  llama_adkv.py:104-123);
* next to each code buffer lives a small checkpoint tensor holding the exact fp16 filter state
  every ``CKPT_INTERVAL`` tokens (4 bytes per channel per checkpoint, ~3 % of the codes at 256).
  The kernels keep it up to date and use it to replay the time axis in independent segments;
* the filter state after the last prompt token is carried, so a prompt may be prefilled in chunks
  (the reference refuses: llama_adkv.py:195-197);
* several new tokens may be attended with at once (``extend``), and a batch may go on from one prefilled sequence whose codes it
  shares (``share``); the reference has neither.
"""
from __future__ import annotations

import math

import torch

from .. import _lib
from ..kernel.gemv import SharedPrefix, append_kv_pair, decode_step, decode_step_workspace_bytes, extend

SCALE_MIN = math.exp(-4.0)  # kept for API parity; the fp16 recurrence never clamps
SCALE_MAX = math.exp(4.0)

INIT_SEQ_LEN = 64    # token slots of a fresh cache (reference llama_adkv.py:40)
CAP_LEN = 64         # capacity granularity in tokens (reference llama_adkv.py:41)
GROWTH = 1.5         # geometric growth factor once the initial capacity is exceeded
CKPT_INTERVAL = 256  # tokens between state checkpoints (multiple of 8); 0 disables them

_HEAD_DIMS = (128, 256, 512)

# Scratch for the fused decode call (logits + partial sums), one per (device, stream): every layer's
# step on a stream runs after the previous one, so they can share it.
_workspaces: dict[tuple, torch.Tensor] = {}


def _workspace(dev: torch.device, need: int) -> torch.Tensor:
    key = (dev.index, torch.cuda.current_stream(dev).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(max(need, 1) * 5 // 4, dtype=torch.uint8, device=dev)
        _workspaces[key] = ws
    return ws


def _additive(mask: torch.Tensor | None, query: torch.Tensor) -> torch.Tensor | None:
    """A boolean mask (sdpa's: true where a token is looked at) as what is added to scores: the lowest value of the query's type where it is false."""
    if mask is None or mask.dtype is not torch.bool:
        return mask
    dt = query.dtype if query.dtype in (torch.float16, torch.bfloat16) else torch.float32
    return torch.full(mask.shape, torch.finfo(dt).min, dtype=dt, device=mask.device).masked_fill_(mask, 0.0)


class KVCacheLayer_ADKV:
    """Quantised K/V store of one attention layer."""

    def __init__(self, bits: int = 4):
        if bits not in (2, 4):
            raise ValueError("ADKV code width must be 2 or 4 bits")
        # 4 = the reference's format; 2 = the same recurrence over codes in [-2, 1], 16 tokens per
        # supergroup (head_dim 128 only), an extension the reference does not have
        self._bits = bits
        self._key_buf: torch.Tensor | None = None
        self._value_buf: torch.Tensor | None = None
        self._key_ckpt: torch.Tensor | None = None
        self._value_ckpt: torch.Tensor | None = None
        # (zp, sc) after the last quantised token, [B, H, C, 2] fp16; lets a prompt arrive in chunks.
        # A decode step appends inside the attention kernels and leaves these stale.
        self._key_state: torch.Tensor | None = None
        self._value_state: torch.Tensor | None = None
        # whether a sequence's is that behind its last token, a byte per sequence, and the sequences that are this object's: a batch_view()
        # has its parent's bytes, which is how the parent knows that a slice was stepped
        self._valid, self._span = bytearray(), slice(0, 0)
        self._quant_len = 0
        self._cap_len = 0
        self._B = self._H = self._C = 0
        self._device = None
        self._ckpt_interval = CKPT_INTERVAL
        self._views: dict = {}    # id(parameter) -> (parameter, its [H, C] view)
        self._shares_storage = False   # a batch_view(): its buffers belong to another layer object
        # a share(): what every sequence begins with, (codes, codes, tokens, checkpoints, checkpoints, zp and sc behind it), K then V,
        # [1, H, ..]; everything above is then of the tokens behind it
        self._prefix: tuple | None = None

    @property
    def _state_valid(self) -> bool:
        return self._B > 0 and 0 not in self._valid[self._span]

    @_state_valid.setter
    def _state_valid(self, valid: bool) -> None:
        if self._valid:      # there are buffers
            self._valid[self._span] = b"\1" * self._B if valid else bytes(self._B)

    # ------------------------------------------------------------------ HF cache protocol
    def get_seq_length(self) -> int:
        return self._quant_len + self._prefix_len()

    def _prefix_len(self) -> int:
        return 0 if self._prefix is None else self._prefix[2]

    def get_mask_sizes(self, cache_position) -> tuple[int, int]:
        """(kv_length, kv_offset) for mask construction.  ``cache_position`` is the query's position
        tensor (transformers 5.3, the version the reference pins) or the query length as an int
        (later 5.x releases)."""
        q_len = cache_position if isinstance(cache_position, int) else cache_position.shape[0]
        return self.get_seq_length() + q_len, 0

    @property
    def key_states(self) -> torch.Tensor | None:
        """Packed uint8 K codes (None before the first token)."""
        return self._key_buf

    @property
    def value_states(self) -> torch.Tensor | None:
        """Packed uint8 V codes (None before the first token)."""
        return self._value_buf

    # ------------------------------------------------------------------ storage
    def _n_super(self, tokens: int) -> int:
        return -(-tokens // (32 // self._bits))

    def _n_ckpt(self, cap_tokens: int) -> int:
        return cap_tokens // self._ckpt_interval + 1 if self._ckpt_interval else 0

    def _new_buffers(self, cap_tokens: int, alloc=torch.zeros):
        ns = self._n_super(cap_tokens)
        shape = (self._B, self._H, ns, self._C // 4, 4, 4)
        mk = lambda: alloc(shape, dtype=torch.uint8, device=self._device)
        ck = (lambda: alloc((self._B, self._H, self._n_ckpt(ns * (32 // self._bits)), self._C, 2),
                            dtype=torch.float16, device=self._device)) \
            if self._ckpt_interval else (lambda: None)
        return ns * (32 // self._bits), mk(), mk(), ck(), ck()

    @staticmethod
    def _capacity(cap: int, T: int) -> int:
        """Token slots of a cache of ``cap`` slots once it has room for ``T`` tokens."""
        if T <= cap:
            return cap
        return -(-max(T, int(cap * GROWTH)) // CAP_LEN) * CAP_LEN

    def _set_geometry(self, B: int, H: int, C: int, device: torch.device):
        if C not in _HEAD_DIMS:
            raise ValueError(f"ADKV kernels support head_dim in (128, 256, 512), got {C}")
        if self._bits == 2 and C != 128:
            raise ValueError("2-bit ADKV codes need head_dim 128")
        self._B, self._H, self._C, self._device = B, H, C, device
        self._quant_len = 0

    def _init_buffers(self, B: int, H: int, C: int, device: torch.device, tokens: int = INIT_SEQ_LEN, alloc=torch.zeros):
        self._set_geometry(B, H, C, device)
        (self._cap_len, self._key_buf, self._value_buf,
         self._key_ckpt, self._value_ckpt) = self._new_buffers(tokens, alloc)
        mk = lambda: alloc((B, H, C, 2), dtype=torch.float16, device=device)
        self._key_state, self._value_state = mk(), mk()
        self._valid, self._span = bytearray(b"\1" * B), slice(0, B)

    def _cap_buffers(self, T: int):
        """Make room for ``T`` tokens.  New slots are zero, as the append kernels expect."""
        if T <= self._cap_len:
            return
        if self._shares_storage:
            raise RuntimeError("a batch view cannot grow: reserve() the parent cache for the whole context")
        cap, key, value, kck, vck = self._new_buffers(self._capacity(self._cap_len, T))
        old = self._key_buf.shape[2]
        key[:, :, :old].copy_(self._key_buf)
        value[:, :, :old].copy_(self._value_buf)
        if kck is not None:
            n = self._key_ckpt.shape[2]
            kck[:, :, :n].copy_(self._key_ckpt)
            vck[:, :, :n].copy_(self._value_ckpt)
        self._key_buf, self._value_buf, self._key_ckpt, self._value_ckpt = key, value, kck, vck
        self._cap_len = cap

    # ------------------------------------------------------------------ big batches, prompt in slices
    def reserve(self, B: int, H: int, C: int, tokens: int, device) -> None:
        """Allocate for a known batch and context up front: no growth copies later, and the
        prompt of a batch too big for one dense prefill can be quantised slice by slice
        through ``batch_view`` (the dense attention of a long prompt, not the cache, is what
        limits the batch of a single prefill call)."""
        if self._prefix is not None:
            raise ValueError("a shared cache is given its room by share()")
        self._init_buffers(B, H, C, torch.device(device))
        self._cap_buffers(tokens)

    def batch_view(self, b0: int, b1: int) -> "KVCacheLayer_ADKV":
        """A layer object over sequences ``b0 .. b1-1`` of this one, sharing its storage (the batch
        axis is the outermost, so the slices are contiguous).  Quantise a slice of the prompt
        through it, then ``commit`` the parent."""
        if self._key_buf is None or not 0 <= b0 < b1 <= self._B:
            raise ValueError("batch_view needs a reserved cache and a slice inside its batch")
        v = KVCacheLayer_ADKV(self._bits)
        v._B, v._H, v._C, v._device = b1 - b0, self._H, self._C, self._device
        v._ckpt_interval, v._cap_len, v._quant_len = self._ckpt_interval, self._cap_len, self._quant_len
        v._key_buf, v._value_buf = self._key_buf[b0:b1], self._value_buf[b0:b1]
        if self._key_ckpt is not None:
            v._key_ckpt, v._value_ckpt = self._key_ckpt[b0:b1], self._value_ckpt[b0:b1]
        v._key_state, v._value_state = self._key_state[b0:b1], self._value_state[b0:b1]
        v._valid, v._span = self._valid, slice(self._span.start + b0, self._span.start + b1)
        v._shares_storage = True
        v._prefix = self._prefix
        return v

    # ------------------------------------------------------------------ one prompt for a whole batch
    def share(self, B: int, tokens: int = INIT_SEQ_LEN) -> "KVCacheLayer_ADKV":
        """A layer object of ``B`` sequences that all begin with this one's tokens (a system prompt, a document, a prompt that several
        answers are sampled for), with room for ``tokens`` more each.  This one holds one sequence, prefilled; its codes are held and
        read once, not copied, and it may go on by itself.  Steps of the batch give no weights."""
        if self._key_buf is None or self._B != 1 or self._C != 128 or self._quant_len == 0 or self._prefix is not None:
            raise ValueError("only the cache of one prefilled sequence with head_dim 128 can be shared")
        if not self._state_valid:
            # decode steps append inside the attention kernels: the state behind the last token is not carried
            raise NotImplementedError("a cache is shared before it is decoded with")
        if B < 1:
            raise ValueError("share needs at least one sequence")
        v = KVCacheLayer_ADKV(self._bits)
        v._ckpt_interval = self._ckpt_interval
        ends = [tuple(st[0, :, :, i].contiguous() for i in range(2)) for st in (self._key_state, self._value_state)]
        v._prefix = (self._key_buf, self._value_buf, self._quant_len, self._key_ckpt, self._value_ckpt, *ends)
        v._init_buffers(B, self._H, self._C, self._device, v._capacity(INIT_SEQ_LEN, tokens))
        return v

    def commit(self, tokens: int) -> None:
        """Declare that every sequence now holds ``tokens`` quantised tokens (all slices prefilled).  The carried state goes along
        unless a slice was decoded or extended with."""
        tokens -= self._prefix_len()
        if tokens > self._cap_len:
            raise ValueError("more tokens than the cache holds")
        if tokens < 0:
            raise ValueError("fewer tokens than the shared prefix has")
        self._quant_len = tokens

    def _check_geometry(self, B: int, H: int, C: int, device: torch.device):
        if self._key_buf is None:
            self._init_buffers(B, H, C, device)
        elif (B, H, C) != (self._B, self._H, self._C):
            raise ValueError("cache was created for a different (B, H, C)")

    @staticmethod
    def _rows(x: torch.Tensor) -> torch.Tensor:
        # fp16 and bf16 rows go to the encoder as they are (it rounds bf16 to fp16 and follows the
        # strides of a [B, T, H, C] projection output itself); anything else is converted first
        return x if x.dtype in (torch.float16, torch.bfloat16) else x.to(torch.float16)

    def _view(self, p: torch.Tensor) -> torch.Tensor:
        # the module passes the same parameter buffers at every step: keep their [H, C] views
        hit = self._views.get(id(p))
        if hit is not None and hit[0] is p:
            return hit[1]
        v = p.view(self._H, self._C)
        if len(self._views) > 64:
            self._views.clear()
        self._views[id(p)] = (p, v)
        return v

    def _own(self, params: tuple, which: int) -> tuple:
        """The parameters of this cache's own streams: behind a prefix they begin with its last state."""
        return params if self._prefix is None else (*self._prefix[5 + which], *params[2:])

    # ------------------------------------------------------------------ quantise
    def _append_tokens(self, key_states, value_states,
                       key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target,
                       value_zp_init, value_scale_init, value_alpha, value_beta, value_quant_target,
                       fresh: bool = False):
        """Quantise ``[B, H, T, C]`` keys/values as tokens ``quant_len ..`` of the stream."""
        append_kv_pair(
            self._key_buf, self._value_buf,
            self._rows(key_states), self._rows(value_states),
            self._own((key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target), 0),
            self._own((value_zp_init, value_scale_init, value_alpha, value_beta, value_quant_target), 1),
            self._quant_len, self._key_state, self._value_state,
            k_ckpt=self._key_ckpt, v_ckpt=self._value_ckpt, ckpt_interval=self._ckpt_interval, bits=self._bits, fresh=fresh)
        self._quant_len += key_states.shape[2]
        self._state_valid = True

    def prefill(self, key_states, value_states,
                key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target,
                value_zp_init, value_scale_init, value_alpha, value_beta, value_quant_target):
        """Quantise the prompt into the cache.  No attention is computed here."""
        B, H, T, C = key_states.shape
        if value_states.shape != key_states.shape:
            raise ValueError("key/value shapes differ")
        if self._key_buf is None and T > 0:
            # a new cache is allocated for the prompt at once and left uninitialised: the launch that
            # quantises the prompt writes all of it
            try:
                self._init_buffers(B, H, C, key_states.device, self._capacity(INIT_SEQ_LEN, T), torch.empty)
                self._append_tokens(key_states, value_states,
                                    key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target,
                                    value_zp_init, value_scale_init, value_alpha, value_beta,
                                    value_quant_target, fresh=True)
            except BaseException:
                self._key_buf = self._value_buf = self._key_ckpt = self._value_ckpt = None
                self._key_state = self._value_state = None
                self._state_valid, self._cap_len = False, 0
                raise
            return
        self._check_geometry(B, H, C, key_states.device)
        if T == 0:
            return
        if self._quant_len != 0 and not self._state_valid:
            # The reference refuses every second prefill (llama_adkv.py:195-197).  Here a prompt may
            # arrive in chunks because the filter state is carried; only after single-token decode
            # steps, which append inside the attention kernels, is that state gone.
            raise NotImplementedError(
                "ADKV prefill encodes from token 0; chunked prefill is not supported by the kernel")
        self._cap_buffers(self._quant_len + T)
        self._append_tokens(key_states, value_states,
                            key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target,
                            value_zp_init, value_scale_init, value_alpha, value_beta,
                            value_quant_target)

    # ------------------------------------------------------------------ decode
    def decode(self, query_states, key_states, value_states,
               key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target,
               value_zp_init, value_scale_init, value_alpha, value_beta, value_quant_target,
               attention_mask: torch.Tensor | None = None,
               scaling: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
        """One causal decode step: attend over the cached tokens and the new one, append the new
        K/V codes, return ``(output [B,H,C] in the query's dtype, weights [B,H,ctx+1] fp16)``
        (weights ``None`` behind a shared prefix).  A mask is additive, or boolean (true where a token is looked at)."""
        ctx = self._quant_len
        if self._prefix is not None:
            if query_states.shape[2] != 1 or key_states.shape[2] != 1:
                raise ValueError("decode expects exactly one query/key/value token")
            out = self.extend(query_states, key_states, value_states,
                              key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target,
                              value_zp_init, value_scale_init, value_alpha, value_beta, value_quant_target,
                              attention_mask, scaling)
            return out[:, 0], None
        attention_mask = _additive(attention_mask, query_states)
        if self._key_buf is not None and ctx < self._cap_len:
            r = _lib.host().decode(
                query_states, key_states, value_states,
                (key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target,
                 value_zp_init, value_scale_init, value_alpha, value_beta, value_quant_target),
                self._key_buf, self._value_buf, self._key_ckpt, self._value_ckpt, self._ckpt_interval, self._bits, ctx,
                float(scaling), attention_mask, _workspaces)
            if r is not None:      # None: something to check, convert, allocate or complain about below
                if isinstance(r, int):
                    _lib.check(r, "decode_step")
                self._quant_len, self._state_valid = ctx + 1, False
                return r
        B, Hq, Tq, C = query_states.shape
        H, Tk = key_states.shape[1], key_states.shape[2]
        if Tq != 1 or Tk != 1:
            raise ValueError("decode expects exactly one query/key/value token")
        if Hq % H or Hq // H not in (1, 2, 4, 8) or (Hq != H and C != 128):
            # the reference only takes Hq == H (llama_adkv.py:235-238); grouped queries are an extension
            raise ValueError("ADKV decode supports 1, 2, 4 or 8 query heads per KV head "
                             "(more than one only with head_dim 128)")
        self._check_geometry(B, H, C, query_states.device)
        self._cap_buffers(ctx + 1)

        # fp16 and bf16 activations go in as they are; the kernels convert (see decode_step)
        same = query_states.dtype in (torch.float16, torch.bfloat16) \
            and key_states.dtype == query_states.dtype == value_states.dtype
        f16 = (lambda t: t.contiguous()) if same else (lambda t: t.to(torch.float16).contiguous())
        v = self._view
        S = self._ckpt_interval
        dev = query_states.device
        ncap = self._key_ckpt.shape[2] if S else 0
        ws = _workspace(dev, decode_step_workspace_bytes(B, Hq, H, ctx, C, ncap, S))
        out, weights = decode_step(
            f16(query_states), self._key_buf, self._value_buf, f16(key_states), f16(value_states),
            (v(key_zp_init), v(key_scale_init), v(key_alpha), v(key_beta), v(key_quant_target)),
            (v(value_zp_init), v(value_scale_init), v(value_alpha), v(value_beta),
             v(value_quant_target)),
            ctx, scaling, attention_mask,
            k_ckpt=self._key_ckpt, v_ckpt=self._value_ckpt, ckpt_interval=S, bits=self._bits,
            workspace=ws)
        self._quant_len = ctx + 1
        self._state_valid = False
        return (out if out.dtype == query_states.dtype else out.to(query_states.dtype)), weights

    # ------------------------------------------------------------------ several tokens
    def extends(self, config=None) -> bool:
        """Whether an attention module hands several new tokens over at once: behind a shared prefix always, else where
        ``config.adkv_extend`` asks for it (one decode step after the other rounds the weights differently)."""
        return self._prefix is not None or (self._C == 128 and bool(getattr(config, "adkv_extend", False)))

    def extend(self, query_states, key_states, value_states,
               key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target,
               value_zp_init, value_scale_init, value_alpha, value_beta, value_quant_target,
               attention_mask: torch.Tensor | None = None, scaling: float = 1.0) -> torch.Tensor:
        """``n`` new tokens at once (head_dim 128): append their codes and attend, each over everything up to itself: a follow-up turn,
        drafted tokens to be checked, the questions behind a shared prompt.  Queries ``[B, Hq, n, C]``, keys and values
        ``[B, H, n, C]``; returns ``[B, n, Hq, C]`` in the query's dtype.  ``n`` calls of ``decode`` append the same codes and
        give the same outputs up to rounding.  A mask is additive, or boolean (true where a token is looked at)."""
        B, _, n, C = query_states.shape
        H = key_states.shape[1]
        if key_states.shape != value_states.shape or key_states.shape[2] != n:
            raise ValueError("extend expects as many keys and values as queries")
        if C != 128:
            raise ValueError("extend needs head_dim 128")
        self._check_geometry(B, H, C, query_states.device)
        self._cap_buffers(self._quant_len + n)
        key = (key_zp_init, key_scale_init, key_alpha, key_beta, key_quant_target)
        value = (value_zp_init, value_scale_init, value_alpha, value_beta, value_quant_target)
        prefix = None
        if self._prefix is not None:
            kc, vc, tokens, kck, vck = self._prefix[:5]
            prefix = SharedPrefix(kc, vc, tokens, key, value, kck, vck)
        attention_mask = _additive(attention_mask, query_states)
        same = query_states.dtype in (torch.float16, torch.bfloat16) and key_states.dtype == query_states.dtype == value_states.dtype
        act = (lambda t: t) if same else (lambda t: t.to(torch.float16))
        out = extend(act(query_states), self._key_buf, self._value_buf, act(key_states), act(value_states),
                     self._own(key, 0), self._own(value, 1), self._quant_len, scaling, attention_mask, prefix=prefix,
                     k_ckpt=self._key_ckpt, v_ckpt=self._value_ckpt, ckpt_interval=self._ckpt_interval, bits=self._bits)
        self._quant_len += n
        self._state_valid = False
        return out if out.dtype == query_states.dtype else out.to(query_states.dtype)

    # ------------------------------------------------------------------ save / restore
    def state_dict(self) -> dict:
        """Everything needed to continue decoding elsewhere: the used part of the code buffers, the
        state checkpoints that go with them and, while it is still valid, the carried filter state.
        Plain tensors and ints, so ``torch.save`` / ``torch.load(weights_only=True)`` round-trip it."""
        if self._key_buf is None:
            return {"quant_len": 0}
        ns = self._n_super(self._quant_len)
        nck = self._quant_len // self._ckpt_interval if self._ckpt_interval else 0
        sd = {"quant_len": self._quant_len, "ckpt_interval": self._ckpt_interval, "bits": self._bits,
              "geometry": (self._B, self._H, self._C),
              "key_codes": self._key_buf[:, :, :ns].contiguous(),
              "value_codes": self._value_buf[:, :, :ns].contiguous()}
        if self._ckpt_interval:
            sd["key_ckpt"] = self._key_ckpt[:, :, :nck].contiguous()
            sd["value_ckpt"] = self._value_ckpt[:, :, :nck].contiguous()
        if self._state_valid:
            sd["key_state"], sd["value_state"] = self._key_state.clone(), self._value_state.clone()
        if self._prefix is not None:
            key, value, tokens, kck, vck, ks, vs = self._prefix
            ns, nck = self._n_super(tokens), tokens // self._ckpt_interval if self._ckpt_interval else 0
            sd["prefix_len"] = tokens
            sd["prefix_key_codes"], sd["prefix_value_codes"] = key[:, :, :ns].contiguous(), value[:, :, :ns].contiguous()
            if self._ckpt_interval:
                sd["prefix_key_ckpt"], sd["prefix_value_ckpt"] = kck[:, :, :nck].contiguous(), vck[:, :, :nck].contiguous()
            sd["prefix_key_state"], sd["prefix_value_state"] = torch.stack(ks), torch.stack(vs)
        return sd

    def load_state_dict(self, sd: dict, device=None) -> None:
        """Rebuild the layer from ``state_dict()`` output on ``device`` (default: where the saved
        tensors live).  Slots past the saved tokens are zero, as the append kernels expect."""
        if sd.get("quant_len", 0) == 0 and "key_codes" not in sd:
            self.__init__(self._bits)
            return
        self._bits = int(sd.get("bits", 4))
        B, H, C = sd["geometry"]
        dev = torch.device(device) if device is not None else sd["key_codes"].device
        T = int(sd["quant_len"])
        self._ckpt_interval = int(sd["ckpt_interval"])
        self._init_buffers(B, H, C, dev)
        self._cap_buffers(T)
        ns = self._n_super(T)
        if tuple(sd["key_codes"].shape) != (B, H, ns, C // 4, 4, 4):
            raise ValueError("saved code tensor does not match its geometry")
        self._key_buf[:, :, :ns].copy_(sd["key_codes"])
        self._value_buf[:, :, :ns].copy_(sd["value_codes"])
        if self._ckpt_interval:
            nck = T // self._ckpt_interval
            if sd["key_ckpt"].shape[2] != nck:
                raise ValueError("saved checkpoints do not cover the saved tokens")
            self._key_ckpt[:, :, :nck].copy_(sd["key_ckpt"])
            self._value_ckpt[:, :, :nck].copy_(sd["value_ckpt"])
        self._quant_len = T
        self._state_valid = "key_state" in sd
        if self._state_valid:
            self._key_state.copy_(sd["key_state"])
            self._value_state.copy_(sd["value_state"])
        self._prefix = None
        if "prefix_len" in sd:
            P = int(sd["prefix_len"])
            to = lambda name: sd[name].to(dev).contiguous() if name in sd else None
            if tuple(sd["prefix_key_codes"].shape) != (1, H, self._n_super(P), C // 4, 4, 4):
                raise ValueError("saved code tensor does not match its geometry")
            if self._ckpt_interval and sd["prefix_key_ckpt"].shape[2] != P // self._ckpt_interval:
                raise ValueError("saved checkpoints do not cover the saved tokens")
            # a prefix shorter than an interval has no checkpoint yet, and the kernels take tensors of one at least
            ck = [t if t is None or t.shape[2] else t.new_zeros(1, H, 1, C, 2) for t in (to("prefix_key_ckpt"), to("prefix_value_ckpt"))]
            self._prefix = (to("prefix_key_codes"), to("prefix_value_codes"), P, *ck,
                            tuple(to("prefix_key_state")), tuple(to("prefix_value_state")))

    # ------------------------------------------------------------------ accounting
    def nbytes(self) -> int:
        """Device bytes held by this layer (codes + checkpoints), those of a shared prefix among them."""
        ts = (self._key_buf, self._value_buf, self._key_ckpt, self._value_ckpt)
        if self._prefix is not None:
            ts += tuple(self._prefix[i] for i in (0, 1, 3, 4))
        return sum(t.numel() * t.element_size() for t in ts if t is not None)


class KVCache_ADKV(list):
    """One ``KVCacheLayer_ADKV`` per decoder layer (reference llama_adkv.py:279-288)."""

    def __init__(self, num_layers: int, bits: int = 4):
        super().__init__(KVCacheLayer_ADKV(bits) for _ in range(num_layers))

    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self[layer_idx].get_seq_length()

    def reserve(self, B: int, H: int, C: int, tokens: int, device) -> None:
        for layer in self:
            layer.reserve(B, H, C, tokens, device)

    def batch_view(self, b0: int, b1: int) -> "KVCache_ADKV":
        view = KVCache_ADKV(0)
        view.extend(layer.batch_view(b0, b1) for layer in self)
        return view

    def commit(self, tokens: int) -> None:
        for layer in self:
            layer.commit(tokens)

    def share(self, B: int, tokens: int = INIT_SEQ_LEN) -> "KVCache_ADKV":
        """A cache of ``B`` sequences that all begin with this one's tokens (see the layer's ``share``)."""
        shared = KVCache_ADKV(0)
        shared.extend(layer.share(B, tokens) for layer in self)
        return shared

    def get_mask_sizes(self, cache_position, layer_idx: int) -> tuple[int, int]:
        return self[layer_idx].get_mask_sizes(cache_position)

    # the rest is what newer transformers releases ask of a cache object during generate()
    def get_query_offset(self, layer_idx: int = 0) -> int:
        return self.get_seq_length(layer_idx)

    def get_max_length(self) -> int:
        return -1

    is_sliding = [False]
    is_compileable = False

    def save(self, path) -> None:
        """Write all layers to one file (tensors moved to the CPU)."""
        cpu = lambda v: v.cpu() if isinstance(v, torch.Tensor) else v
        torch.save([{k: cpu(v) for k, v in layer.state_dict().items()} for layer in self], path)

    @classmethod
    def load(cls, path, device) -> "KVCache_ADKV":
        layers = torch.load(path, map_location="cpu", weights_only=True)
        cache = cls(len(layers))
        for layer, sd in zip(cache, layers):
            layer.load_state_dict(sd, device)
        return cache


def adkv_cache_bytes(B: int, H: int, C: int, tokens: int, layers: int, bits: int = 4,
                     ckpt_interval: int = CKPT_INTERVAL) -> int:
    """Bytes of a full ADKV cache: K and V codes plus fp16 (zp, sc) checkpoints.  Same accounting
    as the reference's memory model (tools/memory_comparison_fig.py:46-56) with
    ``ckpt_num = tokens // ckpt_interval``; the ten parameter vectors per layer are added once."""
    codes = B * H * (-(-tokens // 8) * 8) * C * bits // 8
    ckpt = (B * H * (tokens // ckpt_interval) * C * 2 * 2) if ckpt_interval else 0
    params = 10 * H * C * 2
    return layers * (2 * (codes + ckpt) + params)


def fp16_cache_bytes(B: int, H: int, C: int, tokens: int, layers: int) -> int:
    return layers * 2 * B * H * tokens * C * 2

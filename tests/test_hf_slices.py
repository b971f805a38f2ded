"""Slices of a batch (batch_view) that were decoded or extended with: the parent knows that the state which it carries is theirs no more."""
import copy

import pytest
import torch

from adkv_amd import synth
from adkv_amd.hf import cache as M
from adkv_amd.hf.cache import KVCacheLayer_ADKV

D, H = 128, 2


@pytest.fixture
def no_kernels(monkeypatch):
    """The cache's calls without what they compute."""
    monkeypatch.setattr(M, "extend", lambda q, *a, **k: torch.zeros(q.shape[0], q.shape[2], q.shape[1], D))
    monkeypatch.setattr(M, "decode_step", lambda q, *a, **k: (torch.zeros(q.shape[0], q.shape[1], D), None))
    monkeypatch.setattr(M, "decode_step_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(M, "_workspace", lambda *a: None)
    monkeypatch.setattr(M, "append_kv_pair", lambda *a, **k: None)


def _rows(B, n):
    return [torch.zeros(B, H, n, D, dtype=torch.float16) for _ in range(3)]


PAR = [t.reshape(-1) for t in synth.make_params(H, D).astuple()] * 2


def _reserved(B=4, P=0):
    if not P:
        c = KVCacheLayer_ADKV()
        c.reserve(B, H, D, 100, "cpu")
        return c
    one = KVCacheLayer_ADKV()
    one.prefill(*_rows(1, P)[1:], *PAR)
    return one.share(B, 100)


@pytest.mark.parametrize("P", [0, 24])
@pytest.mark.parametrize("n", [1, 5])
def test_the_parent_carries_no_state_behind_an_extended_slice(no_kernels, P, n):
    c = _reserved(P=P)
    for b in (0, 2):
        v = c.batch_view(b, b + 2)
        v.prefill(*_rows(2, 9)[1:], *PAR)
    c.commit(P + 9)
    assert c._state_valid
    c.prefill(*_rows(4, 3)[1:], *PAR)                # a second part of the prompt goes on from it
    assert c.get_seq_length() == P + 12 and c._state_valid
    v = c.batch_view(2, 4)
    q, k, v_ = _rows(2, n)
    (v.extend if n > 1 else v.decode)(q, k, v_, *PAR)
    c.batch_view(0, 2).prefill(*_rows(2, n)[1:], *PAR)
    c.commit(P + 12 + n)
    assert not c._state_valid and not v._state_valid and c.batch_view(0, 2)._state_valid
    assert "key_state" not in c.state_dict()
    with pytest.raises(NotImplementedError):
        c.prefill(*_rows(4, 2)[1:], *PAR)
    with pytest.raises(NotImplementedError):
        v.prefill(*_rows(2, 2)[1:], *PAR)
    again = copy.deepcopy(c)
    assert not again._state_valid and again.batch_view(0, 2)._state_valid
    # quantised from the first token on the state is carried again
    c.commit(P)
    for b in (0, 2):
        c.batch_view(b, b + 2).prefill(*_rows(2, 9)[1:], *PAR)
    c.commit(P + 9)
    assert c._state_valid and not again._state_valid


def test_a_sequence_is_not_shared_behind_an_extended_slice(no_kernels):
    c = _reserved(B=1)
    v = c.batch_view(0, 1)
    v.prefill(*_rows(1, 9)[1:], *PAR)
    v.extend(*_rows(1, 4), *PAR)
    c.commit(13)
    with pytest.raises(NotImplementedError, match="before it is decoded"):
        c.share(2)


@pytest.mark.gpu
def test_a_slice_that_was_stepped(gpu):
    """With the kernels: the slices that were not stepped go on, the batch as a whole does not."""
    par = [t.reshape(-1).to(gpu) for t in synth.make_params(H, D, seed=3).astuple()] * 2
    rows = lambda B, n, s: synth.make_k(B, H, n, D, seed=s, dtype=torch.float16).to(gpu)
    c = KVCacheLayer_ADKV()
    c.reserve(4, H, D, 100, gpu)
    k, v = rows(4, 20, 1), rows(4, 20, 2)
    for b in (0, 2):
        c.batch_view(b, b + 2).prefill(k[b:b + 2, :, :12], v[b:b + 2, :, :12], *par)
    c.commit(12)
    c.batch_view(2, 4).extend(rows(2, 8, 5), k[2:, :, 12:], v[2:, :, 12:], *par, scaling=0.1)
    c.batch_view(0, 2).prefill(k[:2, :, 12:], v[:2, :, 12:], *par)
    c.commit(20)
    whole = KVCacheLayer_ADKV()
    whole.prefill(k, v, *par)
    for a, b in ((c._key_buf, whole._key_buf), (c._value_buf, whole._value_buf)):
        assert torch.equal(a[:, :, :2], b[:, :, :2])
    with pytest.raises(NotImplementedError):
        c.prefill(rows(4, 3, 7), rows(4, 3, 8), *par)

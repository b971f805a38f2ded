"""Shared caches whose prefix has no state recorded yet (shorter than the interval), saved and restored."""
import pytest
import torch

from adkv_amd import synth
from adkv_amd.hf.cache import CKPT_INTERVAL, KVCache_ADKV, KVCacheLayer_ADKV
from adkv_amd.kernel import gemv

D = 128


def _saved(layer, path, device):
    cache = KVCache_ADKV(0)
    list.extend(cache, [layer])
    cache.save(path)
    return KVCache_ADKV.load(path, device)[0]


@pytest.mark.parametrize("P", [1, 100, CKPT_INTERVAL - 1, CKPT_INTERVAL, CKPT_INTERVAL + 9])
def test_restored_checkpoints_are_what_the_kernels_take(tmp_path, P):
    one = KVCacheLayer_ADKV()
    one._init_buffers(1, 2, D, torch.device("cpu"))
    one._cap_buffers(P)
    one._key_ckpt.fill_(3.0)
    one._quant_len = P
    layer = one.share(3)
    for _ in range(2):                     # saved, and what was restored saved again
        layer = _saved(layer, tmp_path / "c.pt", "cpu")
        key, value = layer._prefix[3:5]
        assert gemv._ckpt_args(key, CKPT_INTERVAL, 1, 2, D)[1] == gemv._ckpt_args(value, CKPT_INTERVAL, 1, 2, D)[1] >= 1
        n = P // CKPT_INTERVAL
        assert key.shape[2] >= n and bool((key[:, :, :n] == 3.0).all()) and layer.get_seq_length() == P
        assert layer.nbytes() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("P", [9, 100, CKPT_INTERVAL, 2 * CKPT_INTERVAL + 17])
def test_a_restored_cache_goes_on(gpu, tmp_path, P):
    """Steps and several tokens at once behind a restored prefix: codes and outputs of the cache that was saved."""
    H, B, lens = 2, 3, (1, 7, 1)
    kg, vg = ([t.reshape(-1) for t in synth.make_params(H, D, seed=s).to(gpu).astuple()] for s in (3, 4))
    kp, vp = (synth.make_k(1, H, P, D, seed=s, dtype=torch.float16).to(gpu) for s in (1, 2))
    kn, vn, q = (synth.make_k(B, H, sum(lens), D, seed=s, t0=P, dtype=torch.float16).to(gpu) for s in (5, 6, 7))
    one = KVCacheLayer_ADKV()
    one.prefill(kp, vp, *kg, *vg)
    kept = one.share(B)
    restored = _saved(one.share(B), tmp_path / "c.pt", gpu)
    at = 0
    for n in lens:
        cut = lambda t: t[:, :, at:at + n].contiguous()
        outs = [c.decode(cut(q), cut(kn), cut(vn), *kg, *vg, scaling=0.1)[0] if n == 1 else
                c.extend(cut(q), cut(kn), cut(vn), *kg, *vg, scaling=0.1) for c in (kept, restored)]
        assert torch.equal(*outs)
        at += n
    assert torch.equal(kept._key_buf[:, :, :2], restored._key_buf[:, :, :2]) and torch.equal(kept._value_buf[:, :, :2], restored._value_buf[:, :, :2])

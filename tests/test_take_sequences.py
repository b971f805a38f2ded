"""gemv.take_sequences against indexing: any map in place, into new buffers, partly filled segments, many rows, several launches, streams and graphs.
Bytes are copied: results are equal."""
import pytest
import torch

from adkv_amd.kernel import gemv


def tensors_of(B, H, spec, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    kinds = {"codes": ((32, 4, 4), torch.uint8), "ckpt": ((128, 2), torch.float16), "state": ((2,), torch.float16), "wide": ((64,), torch.float32)}
    made = []
    for kind, n in spec:
        shape, dtype = kinds[kind]
        size = (B, H, n, *shape)
        made.append(torch.randint(0, 256, size, generator=g, device=dev, dtype=torch.int32).to(dtype) if dtype != torch.float32 else torch.randn(size, generator=g, device=dev))
    return made


def wanted(tensors, index, used, into=None):
    index = index.cpu()
    out = []
    for i, t in enumerate(tensors):
        n, B = used[i], t.shape[0]
        if into is None:
            to = t.clone()
            for r, s in enumerate(index.tolist()):
                if 0 <= s < B:
                    to[r, :, :n] = t[s, :, :n]
        else:
            to = torch.zeros_like(into[i])
            for r, s in enumerate(index.tolist()):
                if 0 <= s < B:
                    to[r, :, :n] = t[s, :, :n]
        out.append(to)
    return out


def check(tensors, index, used=None, into=None):
    full = [t.shape[2] for t in tensors] if used is None else used
    want = wanted(tensors, index, full, into)
    gemv.take_sequences(tensors, index, used=used, into=into)
    for got, w in zip(tensors if into is None else into, want):
        assert torch.equal(got, w)


SPEC = [("codes", 13), ("ckpt", 3), ("state", 128), ("codes", 13), ("wide", 5)]
USED = [11, 2, 128, 0, 3]


@pytest.mark.gpu
@pytest.mark.parametrize("index", [[0], [0, 0], [1, 0], [2, 0, 1], [1, 2, 3, 0, 4], [4, 4, 4, 4, 4], [0, 1, 2, 3, 4], [3, 3, 1], [4, 3, 2, 1, 0], [0, -1, 9, 2, 1], []], ids=str)
def test_in_place(gpu, index):
    for used in (None, USED):
        check(tensors_of(max(5, len(index)), 3, SPEC, gpu), torch.tensor(index, dtype=torch.int64, device=gpu), used)


@pytest.mark.gpu
@pytest.mark.parametrize("B,R", [(1, 1), (1, 16), (4, 7), (7, 4), (33, 70), (3, 40)])
def test_into_new_buffers(gpu, B, R):
    g = torch.Generator().manual_seed(B * 100 + R)
    index = torch.randint(0, B, (R,), generator=g)
    t = tensors_of(B, 2, SPEC, gpu)
    for extra in (0, 4):
        for used in (None, USED):
            into = [torch.full((R, 2, x.shape[2] + extra, *x.shape[3:]), 7, dtype=x.dtype, device=gpu) for x in t]
            check(t, index.to(gpu), used, into)
    index = index.to(gpu)
    index[0] = -1
    check(t, index, USED, [torch.full((R, 2, x.shape[2], *x.shape[3:]), 7, dtype=x.dtype, device=gpu) for x in t])


@pytest.mark.gpu
@pytest.mark.parametrize("B", [16, 31, 32, 33, 64, 65, 200, 1000, 1024])
def test_many_rows(gpu, B):
    """All rows move: one of them, half of them, every one, in cycles and chains."""
    g = torch.Generator().manual_seed(B)
    maps = [torch.randperm(B, generator=g), torch.randint(0, B, (B,), generator=g), torch.arange(B).roll(1), torch.arange(B).flip(0), torch.zeros(B, dtype=torch.int64)]
    for index in maps:
        check(tensors_of(B, 2, [("codes", 3), ("state", 20)], gpu), index.to(gpu), [2, 16])


@pytest.mark.gpu
@pytest.mark.parametrize("moved", range(1, 41, 3))
def test_some_rows(gpu, moved):
    index = torch.arange(50)
    index[5:5 + moved] = torch.arange(5, 5 + moved).roll(2) if moved > 2 else 49
    check(tensors_of(50, 3, [("codes", 9), ("ckpt", 2)], gpu), index.to(gpu), [7, 1])


@pytest.mark.gpu
def test_all_layers_in_several_launches(gpu):
    layers = [t for i in range(70) for t in tensors_of(4, 2, [("codes", 6 + i % 3), ("ckpt", 2), ("state", 128)], gpu, i)]
    check(layers, torch.tensor([2, 1, 0, 2], device=gpu), [5, 1, 128] * 70)


@pytest.mark.gpu
def test_long_rows(gpu):
    """A row of 2.2 GB: offsets beyond 32 bits, more than one kilobyte column per wave."""
    t = torch.zeros(3, 4, 270000, 32, 4, 4, dtype=torch.uint8, device=gpu)
    t[1, 3, 269998] = 5
    t[1, 0, 0] = 6
    t[2, 3, 269999] = 9
    gemv.take_sequences([t], torch.tensor([1, 0, 1], device=gpu), used=[269999])
    assert (t[0, 3, 269998] == 5).all() and (t[2, 0, 0] == 6).all() and not t[1].any()
    assert (t[2, 3, 269999] == 9).all() and not t[0, 3, 269999].any()


@pytest.mark.gpu
def test_indices_from_the_host_and_of_other_types(gpu):
    for index in (torch.tensor([2, 0, 1]), torch.tensor([2, 0, 1], dtype=torch.int32, device=gpu), torch.tensor([2, 0, 1, 0], dtype=torch.uint8, device=gpu)[:3], torch.tensor([2, 9, 0, 9, 1, 9], device=gpu)[::2]):
        check(tensors_of(3, 2, SPEC, gpu), index, USED)


@pytest.mark.gpu
def test_a_graph(gpu):
    t = tensors_of(6, 2, SPEC, gpu)
    index = torch.arange(6, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gemv.take_sequences(t, index, used=USED)
    for new in ([1, 0, 2, 3, 5, 5], [0, 1, 2, 3, 4, 5], [5, 4, 3, 2, 1, 0]):
        index.copy_(torch.tensor(new))
        want = wanted(t, index, USED)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(t, want))


@pytest.mark.gpu
def test_nothing_to_do(gpu):
    gemv.take_sequences([], torch.tensor([0], device=gpu))
    check(tensors_of(2, 0, SPEC, gpu), torch.tensor([1, 0], device=gpu))
    check(tensors_of(2, 2, [("codes", 0)], gpu), torch.tensor([1, 0], device=gpu))
    check(tensors_of(2, 2, [("codes", 0)], gpu), torch.tensor([1, 0, 1], device=gpu), None, [torch.full((3, 2, 5, 32, 4, 4), 7, dtype=torch.uint8, device=gpu)])


@pytest.mark.gpu
def test_no_sequences(gpu):
    """No index is one of theirs: new buffers are zeros, as for every such row."""
    into = [torch.full((3, 2, n, 32, 4, 4), 7, dtype=torch.uint8, device=gpu) for n in (5, 6)]
    index = torch.tensor([0, -1, 2], device=gpu)
    gemv.take_sequences([torch.zeros(0, 2, 5, 32, 4, 4, dtype=torch.uint8, device=gpu)] * 2, index, used=[5, 0], into=into)
    assert not any(t.any() for t in into)
    with pytest.raises(RuntimeError, match="of the sequences"):
        gemv.take_sequences([torch.zeros(0, 2, 5, 16, dtype=torch.uint8, device=gpu)], index.cpu(), into=[torch.zeros(3, 2, 5, 16, dtype=torch.uint8, device=gpu)])


def test_refusals():
    t = torch.zeros(3, 2, 5, 32, 4, 4, dtype=torch.uint8)
    i = torch.tensor([0, 1])
    mk = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    for args, how, message in [(([t], i.float()), {}, "whole numbers"), (([t], i[None]), {}, "whole numbers"), (([t], torch.zeros(1025, dtype=torch.int64)), {}, "1024"), (([t], i), dict(used=[6]), "used"),
                               (([t], i), dict(used=[-1]), "used"), (([t], i), dict(used=[1, 2]), "used"), (([t], torch.zeros(4, dtype=torch.int64)), {}, "at most as many"),
                               (([t.transpose(0, 1)], i), {}, "contiguous"), (([t, mk(4, 2, 5, 16)], i), {}, "contiguous"), (([mk(3, 2, 5, 8)], i), {}, "16 bytes"),
                               (([t], i), dict(into=[mk(2, 2, 5, 32, 4, 4), t]), "into must have"), (([t], i), dict(into=[mk(3, 2, 5, 32, 4, 4)]), "into must be"),
                               (([t], i), dict(into=[mk(2, 2, 4, 32, 4, 4)]), "into must be"), (([t], i), dict(into=[mk(2, 2, 5, 32, 4, 4).to(torch.int8)]), "into must be"),
                               (([t], i), dict(into=[t[:2]]), "share memory"), (([t], torch.tensor([0, 3])), {}, "of the sequences"), (([t], torch.tensor([-1])), {}, "of the sequences"),
                               (([t], i), {}, "device"), (([torch.zeros(3, 2, 4, 4, requires_grad=True)], i), {}, "no gradient")]:
        with pytest.raises(RuntimeError, match=message):
            gemv.take_sequences(*args, **how)


def test_the_library_refuses_what_it_cannot_take():
    from adkv_amd import _lib
    L = _lib.lib()

    def call(n=1, index=4096, rows=2, batch=2, **change):
        d = {**dict(data=4096, into=None, segments=2, pitch=64, into_pitch=0, used=32), **change}
        return L.adkv_take_sequences((_lib.Rows * 1)(_lib.Rows(*d.values())), n, index, rows, batch, None)
    for change, code in [(dict(data=None), -1), (dict(index=None), -1), (dict(n=-1), -3), (dict(rows=-1), -3), (dict(rows=3), -3), (dict(rows=1025, into=8192, into_pitch=64), -3), (dict(batch=0), -3),
                         (dict(used=80), -3), (dict(used=-16), -3), (dict(into=8192, into_pitch=16), -3), (dict(pitch=2 ** 31), -3), (dict(data=4104), -5), (dict(used=24), -5), (dict(pitch=72), -5),
                         (dict(into=8200, into_pitch=64), -5)]:
        assert call(**change) == code, change
    both = (_lib.Rows * 2)(_lib.Rows(4096, None, 1, 64, 0, 64), _lib.Rows(4096, 8192, 1, 64, 64, 64))
    assert L.adkv_take_sequences(both, 2, 4096, 1, 1, None) == -6
    # what is written shares memory with another tensor: twice the same, one inside another, into what is read or written elsewhere
    for a, b in [((4096, None, 2, 64, 0, 64),) * 2, ((4096, None, 2, 64, 0, 64), (4096 + 192, None, 1, 32, 0, 16)),
                 ((4096, 8192, 1, 64, 64, 64), (16384, 4096 + 64, 1, 64, 64, 64)), ((4096, 8192, 1, 64, 64, 64), (16384, 8192, 1, 64, 64, 64)),
                 ((4096, 8192, 1, 64, 64, 64), (8192 + 64, 16384, 1, 64, 64, 64))]:
        for two in ((a, b), (b, a)):
            assert L.adkv_take_sequences((_lib.Rows * 2)(*(_lib.Rows(*t) for t in two)), 2, 4096, 2, 2, None) == -6
    assert L.adkv_take_sequences(None, 0, 4096, 1, 1, None) == 0 and L.adkv_take_sequences(both, 2, None, 0, 1, None) == -6


def test_sizes_that_no_memory_has():
    """Their products pass 64 bits: refused, not taken for nothing to do."""
    from adkv_amd import _lib
    L = _lib.lib()
    for batch, rows, segments, pitch, into_pitch, used in [(2, 2, 2 ** 60, 16, 0, 16), (2, 2, 2 ** 31, 64, 0, 32), (2 ** 31 - 1, 2, 2 ** 31 - 1, 2 ** 30, 0, 16), (1, 1024, 2 ** 31 - 1, 2 ** 30, 2 ** 30, 0)]:
        t = (_lib.Rows * 1)(_lib.Rows(4096, 8192 if into_pitch else None, segments, pitch, into_pitch, used))
        assert L.adkv_take_sequences(t, 1, 4096, rows, batch, None) == -3


@pytest.mark.gpu
def test_tensors_that_share_memory(gpu):
    """Refused where one of them is written; several of them may be copied from one."""
    t, = tensors_of(4, 2, [("codes", 6)], gpu)
    i = torch.tensor([1, 0], device=gpu)
    for pair in ([t, t], [t, t[:]]):
        with pytest.raises(RuntimeError):
            gemv.take_sequences(pair, i)
    into = torch.empty(2, 2, 6, 32, 4, 4, dtype=torch.uint8, device=gpu)
    with pytest.raises(RuntimeError):
        gemv.take_sequences([t, t], i, into=[into, into])
    check([t, t], i, None, [into, into.clone()])

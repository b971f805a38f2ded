"""gemv.extend where a context's pieces end inside a tile: checkpoint intervals that are no multiple of 32 tokens, few query rows.  What a
tile has behind its piece's end belongs to the next piece and counts there."""
import pytest
import torch

from test_extend import D, Case

f16, bf16 = torch.float16, torch.bfloat16
SIZES = [  # B, H, G, P, T, n, bits, type, interval
    (1, 1, 1, 0, 300, 1, 4, f16, 8), (2, 2, 4, 0, 1000, 1, 4, bf16, 48), (1, 1, 1, 900, 130, 1, 4, f16, 24), (3, 1, 4, 700, 77, 1, 2, f16, 48),
    (2, 2, 2, 0, 500, 5, 4, f16, 40), (1, 2, 8, 430, 333, 2, 2, bf16, 16), (1, 1, 16 // 4, 1200, 0, 1, 4, f16, 40), (2, 1, 1, 333, 100, 16, 4, f16, 56),
    (2, 1, 8, 300, 200, 20, 4, f16, 24), (1, 2, 1, 500, 90, 150, 2, f16, 48),       # many rows: pieces are whole tiles
]


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(str(v).replace("torch.", "") for v in s))
def test_intervals_that_are_no_multiple_of_a_tile(gpu, oracle, size, masked):
    B, H, G, P, T, n, _, dtype, _ = size
    c = Case(oracle, gpu, *size, seed=31)
    mask = None
    if masked:
        mask = torch.randn(B, 1, n, P + T + n, generator=torch.Generator().manual_seed(7)).mul_(2).to(dtype)
        mask[0, :, :, :(P + T) // 3] = torch.finfo(dtype).min
        mask = mask.to(gpu)
    c.check(c.run(D ** -0.5, mask), D ** -0.5, mask)

"""What does not turn is copied: infinities, NaN and negative zeros stay where they are, in either layout, whatever way the rows are taken."""
import pytest
import torch

from util_ops4 import TYPES

gpu = pytest.mark.gpu
BITS = {"f16": torch.int16, "bf16": torch.int16, "f32": torch.int32}


@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("half", [True, False], ids=["half", "interleaved"])
@pytest.mark.parametrize("aligned", [True, False], ids=["aligned", "shifted"])
@pytest.mark.parametrize("dim,rot", [(40, 34), (128, 126), (128, 2), (64, 12), (32, 22), (128, 64)])
def test_the_rest_of_a_head(built_lib, dtype, half, aligned, dim, rot):
    from kiln_b200 import ops
    rows, heads = 9, 3
    big = torch.randn(rows, heads * dim + 8, generator=torch.Generator().manual_seed(dim + rot)).to(TYPES[dtype]).cuda()
    x = big[:, :heads * dim] if aligned else big[:, 1:heads * dim + 1]
    head = x.unflatten(1, (heads, dim))                                    # a view
    head[:, :, rot:] = -0.0
    for c in range(rot, dim):
        head[c % rows, c % heads, c] = float("inf") * (-1) ** c
    head[rows - 1, 0, rot] = float("nan")
    head[0, 1, 0] = float("inf")                                           # spoils its own pair
    pos, freq = torch.arange(rows).int()[:, None].cuda() * 100, ops.rope_freqs(rot)
    out = torch.zeros_like(big)
    o = out[:, :heads * dim] if aligned else out[:, 1:heads * dim + 1]
    for inverse in (False, True):
        ops.rope([o], [x], [heads], dim, pos, freq, layout=ops.ROPE_HALF if half else ops.ROPE_INTERLEAVED, amplitude=1.5, inverse=inverse)
        got = o.unflatten(1, (heads, dim))
        nan = torch.isnan(head[:, :, rot:])
        assert torch.equal(torch.isnan(got[:, :, rot:]), nan) and int(nan.sum()) == 1
        assert torch.equal(got[:, :, rot:][~nan].view(BITS[dtype]), head[:, :, rot:][~nan].view(BITS[dtype]))
        bad = torch.zeros(rows, heads, rot, dtype=torch.bool)
        bad[0, 1, 0] = bad[0, 1, rot // 2 if half else 1] = True
        assert torch.isfinite(got[:, :, :rot].cpu()[~bad]).all()

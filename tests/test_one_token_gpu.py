"""The 4-bit product of a single token over the whole range of MX4 scales, against 64 bits and against the form for several rows."""
import numpy as np
import pytest
import torch

from util_ops4 import MX4, NV4, held

pytestmark = pytest.mark.gpu


def _blocks(seed, rows, blocks, exps, hit=0.5):
    """Normal numbers, blocks of 32 times 2^exps[block], with zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, blocks, 32, generator=g, dtype=torch.float64) * (torch.rand(rows, blocks, 32, generator=g) < hit)
    return (x * 2.0 ** torch.as_tensor(exps, dtype=torch.float64)[:, None]).view(rows, -1).float()


@pytest.mark.parametrize("exps_a,exps_w", [([100, 0], [100, 0]), ([-100, -40], [-40, -100]), ([110, -110, 3], [-110, 110, 3]), ([-75, 0], [-70, 3]), ([60] * 70, [59] * 70)])
def test_scales_far_from_one(built_lib, exps_a, exps_w):
    import kiln_b200 as kb
    from kiln_b200 import ops
    n, N = len(exps_a), 200
    x, w = _blocks(1, 1, n, exps_a), _blocks(2, N, n, exps_w)
    if exps_a[0] == 100:                                                   # a block whose products are all zero: 0, not infinity times 0
        x[:, :32:2], w[:, 1:32:2] = 0.0, 0.0
    A, W = ops.quant4(x.cuda(), MX4), ops.quant4(w.cuda(), MX4)
    A3 = ops.quant4(x.repeat(3, 1).cuda(), MX4)
    a, b = held(A), held(W)
    ref, big = a @ b.T, np.abs(a) @ np.abs(b).T
    one = ops.linear4(torch.empty(1, N, device="cuda"), A, W, ops.EPI_F32)
    three = ops.linear4(torch.empty(3, N, device="cuda"), A3, W, ops.EPI_F32)
    assert kb.check_status() == 0
    # a lane adds two halves a block, the shuffles five times: each rounds to 2^-24 of what is there, no more than the sum of magnitudes, or to 2^-150
    assert (np.abs(one.double().cpu().numpy() - ref) <= (2 * n + 6) * (2.0 ** -24 * big + 2.0 ** -150)).all()
    # a k step of 64 columns adds 65 numbers, each cut to 2^-23 of the largest
    assert (np.abs(three.double().cpu().numpy() - ref) <= (n // 2 + 1) * 66 * (2.0 ** -23 * big + 2.0 ** -149)).all()


def test_overflow_and_bad_blocks(built_lib):
    """A sum beyond fp32 is an infinity; a NaN in a block of any scale is a NaN."""
    from kiln_b200 import ops
    x, w = torch.zeros(1, 64), torch.zeros(8, 64)
    x[0, 0], w[:, 0], w[3, 0] = 2.0 ** 100, 2.0 ** 100, -2.0 ** 100
    w[5, 40] = float("nan")
    w[6, 0] = 2.0 ** -100
    w[7, 0] = 0.0
    y = ops.linear4(torch.empty(1, 8, device="cuda"), ops.quant4(x.cuda(), MX4), ops.quant4(w.cuda(), MX4), ops.EPI_F32).cpu()[0]
    inf = float("inf")
    assert y[[0, 1, 2, 4]].tolist() == [inf] * 4 and y[3] == -inf and torch.isnan(y[5]) and y[6] == 1.0 and y[7] == 0.0


@pytest.mark.parametrize("fmt", [MX4, NV4], ids=["mx4", "nv4"])
def test_gelu_as_in_a_batch(built_lib, fmt):
    """Where the sums are exact (few enough bits between the scales) a token's GELU has the same bits alone as among others."""
    from kiln_b200 import ops
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(9, 512, generator=g).half(), torch.randn(8192, 512, generator=g) / 16
    exp = -8 if fmt == NV4 else 0
    W = ops.quant4(w.cuda(), fmt, exp)
    A = ops.quant4(x.cuda(), fmt)
    rows = ops.linear4(torch.empty(9, 8192, device="cuda"), A, W, ops.EPI_F32)
    many = ops.linear4(ops.padded_empty(9, 8192, torch.float16, "cuda"), A, W, ops.EPI_GELU16)
    exact = torch.from_numpy(held(A) @ held(W).T).float()
    for i in range(9):
        one = ops.quant4(x[i:i + 1].cuda(), fmt)
        sums = ops.linear4(torch.empty(1, 8192, device="cuda"), one, W, ops.EPI_F32)
        assert torch.equal(sums, rows[i:i + 1]) and torch.equal(sums.cpu()[0], exact[i])
        assert torch.equal(ops.linear4(ops.padded_empty(1, 8192, torch.float16, "cuda"), one, W, ops.EPI_GELU16), many[i:i + 1])

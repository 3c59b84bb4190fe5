"""The gradient of a 4-bit product's input over the whole range of weights: every power of two of an NV4 matrix, and MX4 scales in and out of what fp16 holds."""
import numpy as np
import pytest
import torch

from util_ops4 import HALF_STEP, MX4, NV4, held

pytestmark = pytest.mark.gpu
RANGE = 2


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _sums(dy, w):
    """What fp32 sums of exact products may be off by: a k step of 16 adds 17 numbers, each cut to 2^-23 of the largest, no larger than the sum of magnitudes."""
    return (dy.shape[1] + 15) // 16 * 18 * 2.0 ** -23 * (np.abs(dy) @ np.abs(w))


@pytest.mark.parametrize("M,N,K", [(3, 64, 40), (200, 320, 264)])
@pytest.mark.parametrize("exp", [-64, -40, -20, -16, -9, 0, 4, 5, 6, 20, 40, 64])
def test_gradient_at_every_power_of_two(built_lib, exp, M, N, K):
    import kiln_b200 as kb
    from kiln_b200 import ops
    x = _randn(1, N, K)
    x[:, ::7] *= 100                                                       # scales up to 448 2^exp and codes of small elements next to them
    x[5] *= 2.0 ** -9                                                      # down to 2^-9 2^exp
    x[6] *= 100
    W = ops.quant4((x * 2.0 ** exp).cuda(), NV4, exp)
    w, dy = held(W), _randn(2, M, N).half()
    g = dy.double().numpy()
    ref, off = g @ w, _sums(g, w)
    d32 = ops.linear4_dx(torch.empty(M, K, device="cuda"), dy.cuda(), W).double().cpu().numpy()
    assert kb.check_status() == 0
    # (next to nothing of an fp32 subnormal: 2^-64 of anything here is not one)
    assert (np.abs(d32 - ref) <= off).all(), np.max(np.abs(d32 - ref) / off)
    d16 = ops.linear4_dx(torch.empty(M, K, dtype=torch.float16, device="cuda"), dy.cuda(), W).double().cpu().numpy()
    fits = np.abs(ref) + off < 65504
    assert (np.abs(d16 - ref) <= off + HALF_STEP["f16"] * (np.abs(ref) + off) + 2.0 ** -25)[fits].all()
    assert (np.abs(d16) >= 65504 * (1 - 2.0 ** -10))[~fits & (np.abs(ref) - off > 65520)].all()


@pytest.mark.parametrize("shift", [-21, -16, 0, 10])
def test_gradient_of_mx4_inside_the_range(built_lib, shift):
    """Blocks of scales from 2^-23 to 2^13 are exact, rows of zeros (scale 2^-127) among them."""
    import kiln_b200 as kb
    from kiln_b200 import ops
    x = _randn(3, 128, 96).clamp(-8, 8)
    x[:, ::32] = 2.0                                                       # every block's largest lies in [2, 8]: scales 2^-1 to 2^0, 2^1 at 8
    x[10], x[:, 32:64] = 0.0, 0.0
    W = ops.quant4((x * 2.0 ** shift).cuda(), MX4)
    w, dy = held(W), _randn(4, 50, 128).half()
    g = dy.double().numpy()
    got = ops.linear4_dx(torch.empty(50, 96, device="cuda"), dy.cuda(), W).double().cpu().numpy()
    assert kb.check_status() == 0
    assert (np.abs(got - g @ w) <= _sums(g, w)).all()


def test_gradient_of_mx4_outside_the_range_is_told(built_lib):
    import kiln_b200 as kb
    from kiln_b200 import ops
    kb.check_status()
    dy = _randn(4, 50, 128).half()
    g = dy.double().numpy()
    run = lambda W: ops.linear4_dx(torch.empty(50, 96, device="cuda"), dy.cuda(), W).double().cpu().numpy()
    x = _randn(5, 128, 96)
    x[3, 40:60] *= 2.0 ** -9                                               # not the block's largest: nothing out of range
    W = ops.quant4((x * 2.0 ** -24).cuda(), MX4)
    w = held(W)
    got = run(W)
    assert kb.check_status() == ops.STATUS_RANGE == RANGE and kb.check_status() == 0
    assert (np.abs(got - g @ w) <= _sums(g, np.abs(w) + 2.0 ** -25) + 2.0 ** -25 * np.abs(g).sum(1, keepdims=True)).all()
    y = x.clone()
    y[7, 33] = 2.0 ** 17                                                   # one block too large: infinities or NaN in its columns, no others
    got = run(ops.quant4(y.cuda(), MX4))
    assert kb.check_status() == RANGE
    assert not np.isfinite(got[:, 33]).any() and np.isfinite(got[:, :32]).all() and np.isfinite(got[:, 64:]).all()
    y[7, 33] = float("nan")                                                # a bad block shows as it does in products, and is no matter of range
    got = run(ops.quant4(y.cuda(), MX4))
    assert kb.check_status() == 0
    assert np.isnan(got[:, 32:64]).all() and np.isfinite(got[:, :32]).all() and np.isfinite(got[:, 64:]).all()

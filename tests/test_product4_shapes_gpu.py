"""The 4-bit product on every tile shape: CTA pairs in one and several rounds, single CTAs with a second tile and more, ragged in all three sizes, under all five
epilogues and both formats."""
import numpy as np
import pytest
import torch

from test_routes4 import EPI, pair  # noqa: F401  (pair: the rule that picks the tile, as a fixture)
from util_ops4 import BLOCK, HALF_STEP, MX4, NV4, held, round_e4m3
from util_routes import SMS

pytestmark = pytest.mark.gpu
SHAPES = [  # M, N, K, pairs, rounds of tiles
    (1000, 8100, 2000, True, 2),        # eight k steps
    (300, 9000, 2500, True, 1),         # ten; a last row tile of 44 rows: its second CTA has none
    (4097, 1000, 2600, True, 1),        # eleven; of one row
    (1793, 9001, 1800, True, 4),        # one row, 41 columns
    (2000, 8100, 300, False, 7),        # two k steps
    (700, 4101, 300, False, 2),
    (129, 9600, 64, False, 2)]          # one
FMTS = [pytest.param(MX4, id="mx4"), pytest.param(NV4, id="nv4")]


def _operands(fmt, M, N, K):
    from kiln_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x, w = torch.randn(M, K, generator=g, device="cuda"), torch.randn(N, K, generator=g, device="cuda") * 2.0 / K ** 0.5
    x[:, ::37] *= 9.0
    return ops.quant4(x, fmt), ops.quant4(w, fmt, -7 if fmt == NV4 else 0)


def _at(v, fmt, s):
    """v [rows, cols] to the nearest values of blocks with scales s [rows, blocks]."""
    s = np.repeat(s, BLOCK[fmt], 1)[:, :v.shape[1]]
    a = np.minimum(np.abs(v) / s, 6.0)
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    return np.copysign(np.round(a / step) * step * s, v)


def _scales(top, fmt):
    if fmt == NV4:
        return np.maximum(round_e4m3(top / 6.0), 2.0 ** -9)
    return np.where(top > 0, np.ldexp(1.0, np.maximum(np.frexp(top)[1] - 3, -127)), 2.0 ** -127)


def _check_gelu4(got, pre, fmt):
    """Every element lies between what GELU a little less and a little more would give. 5e-7: GELU's own error in fp32 (2.4e-7), twice. A block whose scale
    is not decided by so much may have either."""
    g, e = pre * torch.special.ndtr(torch.from_numpy(pre)).numpy(), 5e-7
    rows, n = g.shape
    wide = np.zeros((rows, -(-n // BLOCK[fmt]) * BLOCK[fmt]))
    wide[:, :n] = np.abs(g)
    top = wide.reshape(rows, -1, BLOCK[fmt]).max(2)
    lo, hi = _scales(np.maximum(top - e, 0.0), fmt), _scales(top + e, fmt)
    sure = np.repeat(lo == hi, BLOCK[fmt], 1)[:, :n]
    assert sure.mean() > 0.99
    assert ((_at(g - e, fmt, hi) <= got) & (got <= _at(g + e, fmt, hi)))[sure].all()
    # half a step of two scales, or 8 scales cut to 6
    most = np.repeat(hi, BLOCK[fmt], 1)[:, :n] * (2 if fmt == MX4 else 1) + e
    assert (np.abs(got - g) <= most)[~sure].all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K,pairs,rounds", SHAPES)
def test_product(built_lib, pair, fmt, M, N, K, pairs, rounds):  # noqa: F811
    import kiln_b200 as kb
    from kiln_b200 import ops
    assert all(bool(pair(M, N, (K + 255) // 256, e, SMS)) == pairs for e in EPI.values())
    tile, groups = (256, SMS // 2) if pairs else (128, SMS)
    assert -(-(-(-M // tile) * -(-N // tile)) // groups) == rounds
    A, W = _operands(fmt, M, N, K)
    a, w = torch.from_numpy(held(A)).cuda(), torch.from_numpy(held(W)).cuda()
    ref = a @ w.T
    # fp32 sums of exact products: a k step of 64 columns adds 65 numbers, each cut to 2^-23 of the largest of them, no larger than the sum of magnitudes
    off = (K + 63) // 64 * 66 * 2.0 ** -23 * (a.abs() @ w.abs().T)
    out = ops.padded_empty(M, N, torch.float32, "cuda").fill_(float("nan"))
    ops.linear4(out, A, W, ops.EPI_F32)
    assert kb.check_status() == 0
    assert ((out.double() - ref).abs() <= off).all()
    pre = out.double()                                                     # the same sums behind every epilogue
    out16 = ops.linear4(ops.padded_empty(M, N, torch.float16, "cuda").fill_(float("nan")), A, W, ops.EPI_F16)
    assert torch.equal(out16, out.half())
    g16 = ops.linear4(ops.padded_empty(M, N, torch.float16, "cuda").fill_(float("nan")), A, W, ops.EPI_GELU16).double()
    g = pre * torch.special.ndtr(pre)
    assert ((g16 - g).abs() <= 5e-7 + HALF_STEP["f16"] * (g.abs() + 5e-7) + 2.0 ** -25).all()
    gate = torch.randn(N, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    r0 = torch.randn(M, N, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    for gt in (None, gate):
        r = ops.padded_empty(M, N, torch.float32, "cuda").copy_(r0)
        ops.linear4(r, A, W, ops.EPI_RESID, gate=gt)
        part = pre if gt is None else gt.double() * pre
        want = r0.double() + part
        # the gated product and the sum round
        assert ((r.double() - want).abs() <= HALF_STEP["f32"] * (part.abs() + want.abs()) * 1.01).all()
    H = ops.quant4_empty(M, N, fmt, "cuda")
    ops.linear4(H, A, W, ops.EPI_GELU4)
    assert kb.check_status() == 0
    _check_gelu4(held(H), pre.cpu().numpy(), fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1000, 8100, 2000), (2000, 8100, 300)])
def test_repeats_and_what_lies_around(built_lib, fmt, M, N, K):
    """Twenty repeats are the same bits; what lies between and behind the rows of the output stays; scales and codes behind the operands' last rows may be anything."""
    from kiln_b200 import ops
    A, W = _operands(fmt, M, N, K)
    want = ops.linear4(ops.padded_empty(M, N, torch.float16, "cuda"), A, W, ops.EPI_F16)
    big = torch.full((M + 40, N + 60), 7.0, dtype=torch.float16, device="cuda")
    h4 = ops.linear4(ops.quant4_empty(M, N, fmt, "cuda"), A, W, ops.EPI_GELU4)
    for _ in range(20):
        assert torch.equal(ops.linear4(ops.padded_empty(M, N, torch.float16, "cuda"), A, W, ops.EPI_F16), want)
        h = ops.linear4(ops.quant4_empty(M, N, fmt, "cuda"), A, W, ops.EPI_GELU4)
        assert torch.equal(h.codes, h4.codes)
    ops.linear4(big[:M, :N], A, W, ops.EPI_F16)
    assert torch.equal(big[:M, :N], want) and (big[:, N:] == 7).all() and (big[M:] == 7).all()

    def in_garbage(q):
        rows = q.rows + 130
        codes = torch.full((rows, q.ld + 16), 0xFF, dtype=torch.uint8, device="cuda")
        codes[:q.rows, :q.ld] = q.codes
        scales = torch.full((ops.lib().kb_quant4_scale_bytes(rows, q.cols, fmt),), 0x7F if fmt == NV4 else 0xFF, dtype=torch.uint8, device="cuda")
        s = q.scales.view(-(-q.rows // 128), -1, 32, 4, 4)
        row = (torch.arange(s.shape[0])[:, None, None] * 128 + torch.arange(4)[None, None, :] * 32 + torch.arange(32)[None, :, None]).cuda()
        keep = (row < q.rows)[:, None, :, :, None].expand_as(s)
        part = scales[:q.scales.numel()].view_as(s)
        part.copy_(torch.where(keep, s, part))
        return ops.Quant4(codes, scales, q.rows, q.cols, fmt, q.exp)
    A2, W2 = in_garbage(A), in_garbage(W)
    assert torch.equal(ops.linear4(ops.padded_empty(M, N, torch.float16, "cuda"), A2, W2, ops.EPI_F16), want)
    h = ops.linear4(ops.quant4_empty(M, N, fmt, "cuda"), A2, W2, ops.EPI_GELU4)
    assert torch.equal(h.codes, h4.codes)
    assert torch.equal(ops.dequant4(torch.empty(M, N, device="cuda"), h), ops.dequant4(torch.empty(M, N, device="cuda"), h4))

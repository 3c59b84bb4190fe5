"""Dropout from a counter: the mask against Philox in 64-bit integers (exactly), values against 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

from util_ops4 import HALF_STEP, TYPES, dropout_words

gpu = pytest.mark.gpu


def _x(seed, rows, cols, dtype):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).to(TYPES[dtype])


def _rng(seed, offset):
    s = lambda v: v - 2 ** 64 if v >= 2 ** 63 else v
    return torch.tensor([s(seed), s(offset)], dtype=torch.int64)


def test_reference_words():
    """The known answers of Philox4x32 with ten rounds (Salmon et al., 2011): counters and keys of zeros and of ones."""
    w = dropout_words(1, 8, 0, 0)[0].astype(np.uint16).view("<u4")
    assert [int(v) for v in w] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def test_refusals(built_lib):
    from kiln_b200 import ops
    L = ops.lib()
    buf = (ctypes.c_char * 4096)()
    a = (ctypes.addressof(buf) + 255) & ~255
    r = lambda out=a, ldo=64, odt=0, x=a, ldx=64, idt=0, res=None, ldr=0, rows=2, cols=64, p=0.1, rng=a: L.kb_dropout(out, ldo, odt, x, ldx, idt, res, ldr, rows, cols, p, rng, None)
    assert [r(out=None), r(x=None), r(rng=None), r(rows=-1), r(cols=0), r(odt=3), r(idt=-1), r(p=1.0), r(p=-0.1), r(p=float("nan")), r(p=1 - 2.0 ** -18)] == [-1] * 11
    assert [r(ldo=63), r(ldx=63), r(res=a, ldr=63)] == [-3] * 3
    assert [r(out=a + 1), r(x=a + 1), r(res=a + 1, ldr=64), r(rng=a + 4), r(idt=2, x=a + 2)] == [-2] * 5
    with pytest.raises(ValueError):
        ops.dropout(torch.zeros(2, 8), torch.zeros(2, 9), _rng(1, 2), 0.1)
    with pytest.raises(ValueError):
        ops.dropout(torch.zeros(2, 8), torch.zeros(2, 8), torch.zeros(2), 0.1)


@gpu
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("rows,cols,p", [(1, 1, 0.5), (1, 7, 0.1), (3, 2048, 0.1), (65, 129, 0.3), (130, 68, 0.05), (200, 96, 0.0), (17, 300, 0.999)])
def test_values_and_mask(built_lib, xt, yt, rows, cols, p):
    from kiln_b200 import ops
    seed, offset = 0x9123456789abcdef, 0x8000000000000005 + rows
    rng = _rng(seed, offset).cuda()
    x, res = _x(rows, rows, cols, xt), _x(cols, rows, cols, yt)
    t = int(np.floor(65536 * p + 0.5))
    keep = dropout_words(rows, cols, seed, offset) >= t
    want = np.where(keep, x.double().numpy() * (65536 / (65536 - t)), 0)
    y = ops.dropout(torch.full((rows, cols), float("nan"), dtype=TYPES[yt], device="cuda"), x.cuda(), rng, p).double().cpu().numpy()
    assert (y[~keep] == 0).all()
    # the scale and the product round to fp32, then the output
    assert (np.abs(y - want) <= (2 * 2.0 ** -24 * 1.001 + HALF_STEP[yt] * 1.001) * np.abs(want) + (2.0 ** -25 if yt == "f16" else 0)).all()
    r = res.double().numpy()
    z = ops.dropout(torch.empty(rows, cols, dtype=TYPES[yt], device="cuda"), x.cuda(), rng, p, resid=res.cuda()).double().cpu().numpy()
    assert np.array_equal(z[~keep], r[~keep])
    s = want + r
    assert (np.abs(z - s) <= 2 * 2.0 ** -24 * 1.001 * np.abs(want) + (2.0 ** -24 + HALF_STEP[yt]) * 1.001 * (np.abs(s) + 2.0 ** -22 * np.abs(want)) + (2.0 ** -25 if yt == "f16" else 0)).all()


@gpu
def test_mask_does_not_depend_on_type_stride_or_alignment(built_lib):
    from kiln_b200 import ops
    rng = _rng(7, 9).cuda()
    want = ops.dropout(torch.empty(33, 100, device="cuda"), torch.ones(33, 100, device="cuda"), rng, 0.25) != 0
    for t in TYPES.values():
        for off, ld in [(0, 104), (8, 160), (1, 133)]:
            x = torch.ones(33, ld, dtype=t, device="cuda")[:, off:off + 100]
            big = torch.full((35, ld), 7.0, dtype=t, device="cuda")
            ops.dropout(big[:33, off:off + 100], x, rng, 0.25)
            assert torch.equal(big[:33, off:off + 100] != 0, want)
            big[:33, off:off + 100] = 7
            assert (big == 7).all()
    assert abs(want.float().mean().item() - 0.75) <= 5 * np.sqrt(0.25 * 0.75 / 3300)
    for other in (_rng(8, 9), _rng(7, 10), _rng(7 + 2 ** 40, 9), _rng(7, 9 + 2 ** 40)):
        again = ops.dropout(torch.empty(33, 100, device="cuda"), torch.ones(33, 100, device="cuda"), other.cuda(), 0.25) != 0
        # independent masks agree in 1 - 2 p (1 - p) = 0.625 of the places
        assert abs((again == want).float().mean().item() - 0.625) <= 6 * np.sqrt(0.625 * 0.375 / 3300)


@gpu
@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("bf16", "f32"), ("f32", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("rows,cols,off,ld", [(40001, 9, 0, 9), (20011, 100, 1, 103), (3000, 1001, 0, 1001), (700, 8190, 2, 8195), (3, 2049, 5, 2060), (31, 1, 0, 1)])
def test_rows_of_any_alignment_agree(built_lib, xt, yt, rows, cols, off, ld):
    """Rows that do not start on 16 bytes get what rows that do get, bit for bit, with a residual and in place too; nothing beside them is written."""
    from kiln_b200 import ops
    rng = _rng(cols, rows).cuda()
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, ld, generator=g, device="cuda").to(TYPES[xt])[:, off:off + cols]
    res = torch.randn(rows, ld, generator=g, device="cuda").to(TYPES[yt])
    wx, wr, want = (ops.padded_empty(rows, cols, t, "cuda") for t in (TYPES[xt], TYPES[yt], TYPES[yt]))
    wx.copy_(x)
    wr.copy_(res[:, off:off + cols])
    for with_res in (False, True):
        ops.dropout(want, wx, rng, 0.3, resid=wr if with_res else None)
        big = torch.full((rows, ld), 7.0, dtype=TYPES[yt], device="cuda")
        ops.dropout(big[:, off:off + cols], x, rng, 0.3, resid=res[:, off:off + cols] if with_res else None)
        assert torch.equal(big[:, off:off + cols], want)
        big[:, off:off + cols] = 7
        assert (big == 7).all()
    ops.dropout(res[:, off:off + cols], x, rng, 0.3, resid=res[:, off:off + cols])
    assert torch.equal(res[:, off:off + cols], want)
    if xt == yt:
        y = x.clone() if ld == cols else x
        ops.dropout(want, wx, rng, 0.3)
        assert torch.equal(ops.dropout(y, y, rng, 0.3), want)


@gpu
def test_in_place_nan_and_gradient(built_lib):
    """In place; a dropped infinity or NaN is a zero; the gradient is the same call."""
    from kiln_b200 import ops
    rng = _rng(3, 4).cuda()
    keep = torch.from_numpy(dropout_words(20, 72, 3, 4) >= int(np.floor(65536 * 0.4 + 0.5))).cuda()
    x = _x(1, 20, 72, "f32").cuda()
    x[~keep] = float("nan")
    x[0, ~keep[0]] = float("inf")
    y = ops.dropout(torch.empty_like(x), x, rng, 0.4)
    assert torch.isfinite(y).all()
    assert torch.equal(ops.dropout(x.clone(), x, rng, 0.4), y)
    z = x.clone()
    assert torch.equal(ops.dropout(z, z, rng, 0.4), y)
    r = _x(2, 20, 72, "f32").cuda()
    want = ops.dropout(torch.empty_like(x), x, rng, 0.4, resid=r)
    assert torch.equal(ops.dropout(r, x, rng, 0.4, resid=r), want)
    # <dy, y(a + e) - y(a)> = <dx, e>, exact up to the roundings of 1440 products
    a, e, dy = (_x(s, 20, 72, "f32").cuda() for s in (5, 6, 7))
    run = lambda v: ops.dropout(torch.empty_like(v), v, rng, 0.4).double()
    lhs, rhs = (dy.double() * (run(a + e) - run(a))).sum().item(), (run(dy) * e.double()).sum().item()
    assert abs(lhs - rhs) <= 20 * 72 * 6 * 2.0 ** -24 * 50


@gpu
def test_captured_with_new_offsets(built_lib):
    """The seed and offset are read at replay: every step of a captured trainer has a mask of its own."""
    from kiln_b200 import ops
    x, out, rng = torch.ones(16, 64, device="cuda"), torch.empty(16, 64, device="cuda"), _rng(11, 0).cuda()
    ops.dropout(out, x, rng, 0.5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.dropout(out, x, rng, 0.5)
        rng[1:] += 1
    for step in range(3):
        g.replay()
        assert np.array_equal(out.cpu().numpy() != 0, dropout_words(16, 64, 11, step) >= 32768)

"""Rotary positions against 64 bits: both layouts, part of a head, position axes, far positions, stretched contexts, the inverse as gradient."""
import ctypes

import numpy as np
import pytest
import torch

from util_ops4 import HALF_STEP, TYPES, rope64

gpu = pytest.mark.gpu


def _x(seed, rows, cols, dtype):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).to(TYPES[dtype])


def test_frequencies(built_lib):
    from kiln_b200 import ops
    i = np.arange(48)
    plain = 10000.0 ** (-2.0 * i / 96)
    close = lambda a, b: np.allclose(a, b, rtol=1e-14, atol=0)
    assert close(ops.rope_freqs(96), plain)
    assert close(ops.rope_freqs(96, scaling=ops.ROPE_LINEAR, factor=3.0), plain / 3)
    based = ops.rope_freqs(96, scaling=ops.ROPE_BASE, factor=3.0)
    assert close(based, (10000.0 * 3.0 ** (96 / 94)) ** (-2.0 * i / 96)) and based[0] == 1 and np.isclose(based[-1], plain[-1] / 3, rtol=1e-12)
    parts = ops.rope_freqs(96, scaling=ops.ROPE_PARTS, factor=4.0, trained_len=4096.0, slow_turns=1.0, fast_turns=32.0)
    turns = 4096 * plain / (2 * np.pi)
    assert close(parts[turns >= 32], plain[turns >= 32]) and close(parts[turns <= 1], plain[turns <= 1] / 4)
    mix = (turns > 1) & (turns < 32)
    r = (turns[mix] - 1) / 31
    assert mix.any() and close(parts[mix], plain[mix] * r + plain[mix] / 4 * (1 - r))
    assert ops.rope_freqs(2, scaling=ops.ROPE_BASE, factor=3.0)[0] == 1


def test_refusals(built_lib):
    from kiln_b200 import ops
    L = ops.lib()
    buf = (ctypes.c_char * 4096)()
    a = (ctypes.addressof(buf) + 255) & ~255
    f = (ctypes.c_double * 128)(*([0.5] * 128))
    import struct
    vp1, i1 = (lambda v: struct.pack('Q', v or 0)), (lambda v: struct.pack('i', v))

    def r(n=1, out=a, ldo=256, x=a, ldx=256, heads=2, dt=0, rows=4, dim=128, rot=128, layout=0, pos=a, prows=4, ldp=1, axes=1, freq=f, axis=None):
        return L.kb_rope(n, vp1(out), i1(ldo), vp1(x), i1(ldx), i1(heads), dt, rows, dim, rot, layout, pos, prows, ldp, axes, freq, axis, 1.0, 0, None)

    bad = (ctypes.c_double * 128)(*([0.5] * 127 + [float("inf")]))
    assert [r(n=0), r(n=5), r(out=None), r(x=None), r(dt=5), r(rows=-1), r(dim=0), r(rot=0), r(rot=63), r(layout=2), r(pos=None), r(prows=0), r(axes=0), r(freq=None),
            r(heads=0), r(freq=bad, dim=256, rot=256, ldx=512, ldo=512), r(axis=(ctypes.c_int * 128)(*([1] * 128)))] == [-1] * 17
    assert [r(dim=264, rot=8, ldx=528, ldo=528), r(rot=130), r(ldx=255), r(ldo=255), r(axes=2)] == [-3] * 5
    assert [r(x=a + 1), r(out=a + 1), r(pos=a + 2)] == [-2] * 3
    g = (ctypes.c_double * 4)()
    assert [L.kb_rope_freqs(g, n, b, s, k, t, 1.0, 32.0) for n, b, s, k, t in [(7, 1e4, 0, 1, 0), (0, 1e4, 0, 1, 0), (258, 1e4, 0, 1, 0), (8, 0.0, 0, 1, 0), (8, 1e4, 4, 1, 0),
                                                                              (8, 1e4, 1, 0.0, 0), (8, 1e4, 3, 2.0, 0.0)]] == [-1] * 7
    assert L.kb_rope_freqs(None, 8, 1e4, 0, 1, 0, 1, 32) == -1
    with pytest.raises(ValueError):
        ops.rope([torch.zeros(4, 128)], [torch.zeros(4, 128), torch.zeros(4, 128)], [1], 128, torch.zeros(4, 1, dtype=torch.int32), ops.rope_freqs(128))
    with pytest.raises(ValueError):
        ops.rope([torch.zeros(4, 128)], [torch.zeros(4, 128)], [1], 128, torch.zeros(4, 1), ops.rope_freqs(128))


def _bound(x, y, dtype, amplitude):
    """The angle is off by 2^-25 of a half turn, cos and sin by 2 units of fp32 and the amplitude's rounding; two products and a sum round; then the output does."""
    big = np.abs(x).max() * abs(amplitude)
    return big * (2 * np.pi * 2.0 ** -25 + 8 * 2.0 ** -23) + HALF_STEP[dtype] * (np.abs(y) + big * 2e-6) + 2.0 ** -25


CASES = [  # rows, pos_rows, heads, dim, rot, axes, start
    (1, 1, (1,), 8, 8, 1, 0), (1, 1, (16, 16), 128, 128, 1, 5), (300, 300, (16, 4), 128, 128, 3, 0), (37, 37, (3, 1), 64, 32, 1, 1000), (30, 10, (2,), 128, 96, 1, 0),
    (65, 13, (5, 2, 1), 80, 48, 2, 12), (9, 9, (2, 2), 72, 10, 1, 3), (7, 7, (3,), 6, 4, 1, 0), (11, 11, (1, 1, 1, 1), 256, 256, 1, 1 << 20), (33, 33, (2,), 96, 2, 1, 0),
    (50, 50, (4,), 128, 128, 1, (1 << 31) - 51), (50, 50, (4,), 128, 126, 1, -(1 << 31))]


@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("half", [True, False], ids=["half", "interleaved"])
@pytest.mark.parametrize("rows,pos_rows,heads,dim,rot,axes,start", CASES)
def test_rotation(built_lib, dtype, half, rows, pos_rows, heads, dim, rot, axes, start):
    from kiln_b200 import ops
    pos = (torch.arange(pos_rows)[:, None] * (1 + 2 * torch.arange(axes)) + start).clamp(-2 ** 31, 2 ** 31 - 1).int()
    freq = ops.rope_freqs(rot, scaling=ops.ROPE_PARTS, factor=4.0, trained_len=512.0)
    axis = (np.arange(rot // 2) * axes // (rot // 2)).astype(np.int32) if axes > 1 else None
    amp = 1.0 if rows % 2 else 1.25
    xs = [_x(10 * rows + k, rows, h * dim, dtype) for k, h in enumerate(heads)]
    p = pos.numpy()[np.arange(rows) % pos_rows].astype(np.int64)
    for inverse in (False, True):
        dev = [x.cuda() for x in xs]
        outs = ops.rope([torch.full_like(d, float("nan")) for d in dev], dev, list(heads), dim, pos.cuda(), freq, axis,
                        layout=ops.ROPE_HALF if half else ops.ROPE_INTERLEAVED, amplitude=amp, inverse=inverse)
        inplace = [d.clone() for d in dev]
        ops.rope(inplace, inplace, list(heads), dim, pos.cuda(), freq, axis, layout=ops.ROPE_HALF if half else ops.ROPE_INTERLEAVED, amplitude=amp, inverse=inverse)
        for x, o, i, h in zip(xs, outs, inplace, heads):
            x = x.double().numpy()
            y = rope64(x, h, dim, rot, p, freq, axis, half, amp, inverse)
            got = o.double().cpu().numpy()
            assert (np.abs(got - y) <= _bound(x, y, dtype, amp)).all(), np.abs(got - y).max()
            rest = np.arange(h * dim) % dim >= rot
            assert np.array_equal(got[:, rest], x[:, rest]) and torch.equal(o, i)


SHIFTED = [  # heads of whole pieces of eight whose halves begin inside one
    (21, 21, (16, 4), 128, 126, 1, 7), (5, 5, (33,), 256, 250, 2, 0), (40, 8, (1,), 8, 2, 1, 3), (19, 19, (1, 1), 32, 14, 1, 0), (6, 6, (40, 9, 2), 40, 36, 3, 0),
    (3, 3, (13, 5), 248, 8, 1, 100), (17, 17, (2, 1), 128, 34, 1, 0), (2, 2, (64, 64), 64, 62, 1, 0)]


@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,pos_rows,heads,dim,rot,axes,start", SHIFTED)
def test_shifted_halves(built_lib, dtype, rows, pos_rows, heads, dim, rot, axes, start):
    test_rotation(built_lib, dtype, True, rows, pos_rows, heads, dim, rot, axes, start)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("half", [True, False], ids=["half", "interleaved"])
@pytest.mark.parametrize("rows,rot", [(4739, 30), (2371, 32)])
def test_several_rows_of_a_thread_block(built_lib, dtype, half, rows, rot):
    test_rotation(built_lib, dtype, half, rows, 1000, (13, 7), 32, rot, 1, 11)


@gpu
def test_shifted_halves_keep_to_themselves(built_lib):
    """Infinities and NaN spoil their own pair only; what does not turn is copied bit for bit, a negative zero too."""
    from kiln_b200 import ops
    x = _x(4, 6, 2 * 40, "f16")
    x[:, 36:40], x[1, 3], x[2, 20], x[3, 77] = -0.0, float("inf"), float("nan"), float("inf")
    pos, freq = torch.arange(6).int()[:, None].cuda(), ops.rope_freqs(34)
    y = ops.rope([torch.empty_like(x).cuda()], [x.cuda()], [2], 40, pos, freq)[0].cpu()
    bad = torch.zeros(6, 80, dtype=torch.bool)
    bad[1, [3, 20]], bad[2, [3, 20]], bad[3, 77] = True, True, True
    assert torch.isfinite(y[~bad]).all() and not torch.isfinite(y[bad]).any()
    rest = torch.arange(80) % 40 >= 34
    assert torch.equal(y[:, rest].view(torch.int16), x[:, rest].view(torch.int16))


@gpu
@pytest.mark.parametrize("half", [True, False], ids=["half", "interleaved"])
def test_strides_and_alignment(built_lib, half):
    """Column slices of wider rows, aligned to 16 bytes and not; what lies around the output stays."""
    from kiln_b200 import ops
    pos, freq = torch.arange(20).int()[:, None].cuda(), ops.rope_freqs(64)
    lay = ops.ROPE_HALF if half else ops.ROPE_INTERLEAVED
    for off, ld in [(8, 160), (1, 160), (0, 133)]:
        big = _x(off, 20, ld, "f16").cuda()
        x = big[:, off:off + 128]
        want = ops.rope([torch.empty(20, 128, dtype=torch.float16, device="cuda")], [x.contiguous()], [2], 64, pos, freq, layout=lay)[0]
        o = torch.full((22, ld + 3), 7.0, dtype=torch.float16, device="cuda")
        ops.rope([o[:20, off:off + 128]], [x], [2], 64, pos, freq, layout=lay)
        assert torch.equal(o[:20, off:off + 128], want)
        o[:20, off:off + 128] = 7
        assert (o == 7).all()


@gpu
def test_inverse_is_the_gradient(built_lib):
    """<dout, rope(x + e) - rope(x)> = <rope_inverse(dout), e>, and the inverse undoes a rotation."""
    from kiln_b200 import ops
    pos, freq = (torch.arange(40).int()[:, None] * 977).cuda(), ops.rope_freqs(48)
    run = lambda x, inv: ops.rope([torch.empty_like(x)], [x], [3], 64, pos, freq, layout=ops.ROPE_INTERLEAVED, amplitude=1.5, inverse=inv)[0]
    x, e, d = (_x(s, 40, 192, "f32").cuda() for s in (1, 2, 3))
    lhs = (d.double() * (run(x + e, False).double() - run(x, False).double())).sum().item()
    rhs = (run(d, True).double() * e.double()).sum().item()
    # every element of either side is off by no more than _bound, and there are 40 * 192 of them
    assert abs(lhs - rhs) <= 3 * 40 * 192 * 16 * 8 * 2.0 ** -23
    back = run(run(x, False), True).double().cpu().numpy().reshape(40, 3, 64)
    want = x.double().cpu().numpy().reshape(40, 3, 64).copy()
    want[:, :, :48] *= 1.5 ** 2
    assert np.abs(back - want).max() <= 2 * _bound(want, want, "f32", 1.5).max()


@gpu
def test_agrees_with_the_tables(built_lib):
    """What kb_qk_prep rotates by fp32 tables, from positions: whole heads of 128, half layout."""
    from kiln_b200 import ops
    T, H = 100, 4
    freq = ops.rope_freqs(128)
    t = np.arange(T)[:, None] * freq
    cos, sin = torch.from_numpy(np.cos(t)).float().cuda(), torch.from_numpy(np.sin(t)).float().cuda()
    x = _x(1, 2 * T, H * 128, "f16").cuda()
    a = ops.qk_prep(torch.empty_like(x), x, 2 * T, H, T, rope_cos=cos, rope_sin=sin)
    b = ops.rope([torch.empty_like(x)], [x], [H], 128, torch.arange(T).int()[:, None].cuda(), freq)[0]
    big = x.abs().max().item()
    assert (a.double() - b.double()).abs().max().item() <= 2.0 ** -10 * 1.5 * big


@gpu
def test_captured(built_lib):
    """Positions are read at replay; the frequencies belong to the captured call."""
    from kiln_b200 import ops
    freq = ops.rope_freqs(128)
    x, pos, out = _x(1, 64, 256, "bf16").cuda(), torch.zeros(64, 1, dtype=torch.int32, device="cuda"), torch.empty(64, 256, dtype=torch.bfloat16, device="cuda")
    ops.rope([out], [x], [2], 128, pos, freq)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.rope([out], [x], [2], 128, pos, freq)
    for start in (0, 5000):
        pos.copy_(torch.arange(start, start + 64, dtype=torch.int32)[:, None])
        g.replay()
        assert torch.equal(out, ops.rope([torch.empty_like(out)], [x], [2], 128, pos, freq)[0])


@gpu
def test_no_rows(built_lib):
    from kiln_b200 import ops
    x = torch.empty(4, 128, device="cuda")[:0]
    base = torch.empty(1, 128, device="cuda")
    pos, f = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), ops.rope_freqs(128)
    import struct
    vp1, i1 = (lambda v: struct.pack('Q', v)), (lambda v: struct.pack('i', v))
    assert x.numel() == 0 and ops.lib().kb_rope(1, vp1(base.data_ptr()), i1(128), vp1(base.data_ptr()), i1(128), i1(1), 2, 0, 128, 128, 0, pos.data_ptr(), 1, 1, 1, f.ctypes.data,
                                                None, 1.0, 0, None) == 0

"""4-bit matrices: quantisation and its inverse against the definition (exactly), products and their gradients against 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

from util_ops4 import BLOCK, HALF_STEP, MX4, NV4, TYPES, buffers, gelu64, held, quantise, read4, round_e4m3

gpu = pytest.mark.gpu
FMTS = [pytest.param(MX4, id="mx4"), pytest.param(NV4, id="nv4")]


def _x(seed, rows, cols, dtype="f32", amp=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g) * amp).to(TYPES[dtype])


# ---------------------------------------------------------------- the definition itself, on the CPU
def test_reference_rounding():
    every = np.sort(np.concatenate([np.arange(8) * 2.0 ** -9, *[(8 + np.arange(8)) * 2.0 ** (e - 3) for e in range(-6, 9)]]))[:-1]   # without 480
    assert every[-1] == 448 and len(every) == 127
    assert np.array_equal(round_e4m3(every), every)
    mid = (every[1:] + every[:-1]) / 2
    even = np.where(np.arange(126) % 2 == 0, every[:-1], every[1:])
    assert np.array_equal(round_e4m3(mid), even)
    t = torch.tensor(np.abs(np.random.RandomState(0).randn(4000)) * np.exp2(np.random.RandomState(1).uniform(-8, 8, 4000)), dtype=torch.float32).clamp(max=448)
    assert np.array_equal(round_e4m3(t.double().numpy()), t.to(torch.float8_e4m3fn).double().numpy())


def test_sizes(built_lib):
    from kiln_b200 import ops
    L = ops.lib()
    assert [L.kb_quant4_row_bytes(c) for c in (1, 32, 33, 2048)] == [16, 16, 32, 1024]
    assert L.kb_quant4_row_bytes(0) == 0 and L.kb_quant4_row_bytes((1 << 24) + 1) == 0
    assert L.kb_quant4_scale_bytes(1, 1, MX4) == 512 and L.kb_quant4_scale_bytes(129, 129, MX4) == 2 * 2 * 512
    assert L.kb_quant4_scale_bytes(128, 65, NV4) == 2 * 512 and L.kb_quant4_scale_bytes(128, 64, 2) == 0
    assert L.kb_linear4_dx_workspace_bytes(64, 8) == 1024


def test_refusals(built_lib):
    """Every refusal comes before a device is asked for, so it can be tested without one."""
    from kiln_b200 import ops
    L = ops.lib()
    buf = (ctypes.c_char * 65536)()
    a = ctypes.c_void_p((ctypes.addressof(buf) + 255) & ~255)
    o = ctypes.c_void_p(a.value + 8)
    ARG, ALIGN, SHAPE, WS = -1, -2, -3, -4
    q = lambda codes=a, ld=32, sc=a, x=a, ldx=64, dt=0, r=4, c=64, fmt=0, exp=0: L.kb_quant4(codes, ld, sc, x, ldx, dt, r, c, fmt, exp, None)
    assert [q(codes=None), q(sc=None), q(x=None), q(r=-1), q(c=0), q(dt=3), q(fmt=2), q(fmt=-1), q(exp=1), q(fmt=1, exp=65)] == [ARG] * 10
    assert [q(codes=o), q(sc=o), q(ld=40), q(x=ctypes.c_void_p(a.value + 1))] == [ALIGN] * 4
    assert [q(ld=16), q(ldx=63), q(c=(1 << 24) + 1, ldx=1 << 25)] == [SHAPE] * 3
    d = lambda y=a, ldy=64, dt=0, codes=a, ld=32, sc=a, r=4, c=64, fmt=0, exp=0, t=0: L.kb_dequant4(y, ldy, dt, codes, ld, sc, r, c, fmt, exp, t, None)
    assert [d(y=None), d(dt=9), d(codes=None), d(fmt=1, exp=-65), d(c=-5)] == [ARG] * 5
    assert [d(ldy=63), d(t=1, ldy=3), d(ld=16)] == [SHAPE] * 3
    p = lambda C=a, ldc=64, Cs=None, A=a, lda=32, As=a, W=a, ldw=32, Ws=a, M=4, N=64, K=64, fmt=0, epi=1, gate=None: L.kb_linear4(
        C, ldc, Cs, A, lda, As, W, ldw, Ws, M, N, K, fmt, epi, 1.0, gate, None)
    assert [p(C=None), p(A=None), p(As=None), p(W=None), p(Ws=None), p(M=-1), p(N=0), p(K=0), p(fmt=3), p(epi=4), p(epi=6), p(gate=a), p(Cs=a), p(epi=5)] == [ARG] * 14
    assert [p(C=o), p(ldc=68), p(epi=0, ldc=66), p(A=o), p(lda=40), p(epi=5, Cs=o, ldc=32), p(epi=3, gate=ctypes.c_void_p(a.value + 2))] == [ALIGN] * 7
    assert [p(ldc=56), p(lda=16), p(ldw=16), p(epi=5, Cs=a, ldc=16)] == [SHAPE] * 4
    g = lambda dx=a, ldx=64, dt=0, dy=a, ldy=64, W=a, ldw=32, Ws=a, M=4, N=64, K=64, fmt=0, exp=0, ws=a, wb=1 << 20: L.kb_linear4_dx(
        dx, ldx, dt, dy, ldy, W, ldw, Ws, M, N, K, fmt, exp, ws, wb, None)
    assert [g(dx=None), g(dt=1), g(W=None), g(exp=2), g(N=0)] == [ARG] * 5
    assert [g(N=72, ldy=72), g(K=68, ldx=72, ldw=48), g(ldy=56), g(ldx=56), g(ldw=16)] == [SHAPE] * 5
    assert [g(ws=None), g(wb=8191)] == [WS] * 2
    assert g(ws=o) == ALIGN


def test_binding_refuses(built_lib):
    from kiln_b200 import ops
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8)
    with pytest.raises(ValueError):
        ops.Quant4(codes, scales, 5, 64, MX4)                      # rows
    with pytest.raises(ValueError):
        ops.Quant4(codes, scales, 4, 65, MX4)                      # columns
    with pytest.raises(ValueError):
        ops.Quant4(codes, scales[:100], 4, 64, MX4)                # scales
    with pytest.raises(ValueError):
        ops.Quant4(codes.float(), scales, 4, 64, MX4)
    A, W = ops.Quant4(codes, scales, 4, 64, MX4), ops.Quant4(codes, scales, 3, 64, NV4)
    with pytest.raises(ValueError):
        ops.linear4(torch.zeros(4, 3), A, W, ops.EPI_F32)          # formats


# ---------------------------------------------------------------- quantisation: exact
def _borders(fmt):
    """Blocks whose elements lie on and next to every border, at several scales."""
    rows = []
    for s in (1.0, 1.125, 1.75, 2.0 ** -6, 2.0 ** 3 * 1.375) if fmt == NV4 else (1.0, 2.0 ** -20, 2.0 ** 30):
        for top in (6.0, 5.9 if fmt == NV4 else 4.5):
            mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32) * np.float32(s)
            near = np.concatenate([mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(99) * np.float32(s)), -mids])
            for i in range(0, len(near), 15):
                part = near[i:i + 15]
                rows.append(np.concatenate([part, np.zeros(BLOCK[fmt] - 1 - len(part), np.float32), [np.float32(top * s)]]))
    return torch.from_numpy(np.stack(rows).astype(np.float32))


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2048), (3, 31), (5, 33), (129, 130), (200, 257), (77, 1024), (130, 68)])
def test_quantise(built_lib, fmt, dtype, rows, cols):
    from kiln_b200 import ops
    exp = -3 if fmt == NV4 and cols % 2 else 0
    x = _x(rows * 1000 + cols, rows, cols, dtype, 2.0 ** exp)
    code, s, val = quantise(x.double().numpy(), fmt, exp)
    q = ops.quant4(x.cuda(), fmt, exp)
    assert np.array_equal(held(q), val)
    c, sc = buffers(q)
    wide = np.zeros((rows, 2 * c.shape[1]), np.int64)
    wide[:, :cols] = code
    assert np.array_equal(c, wide[:, 0::2] | wide[:, 1::2] << 4)           # zeros behind the last column
    pieces, blocks = -(-s.shape[1] // 4), s.shape[1]
    r = np.arange(rows)
    for b in range(blocks, 4 * pieces):                                    # and behind the last block
        assert not sc[((r // 128) * pieces + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4].any()
    for name, t in TYPES.items():
        y = ops.dequant4(torch.empty(rows, cols, dtype=t, device="cuda"), q)
        yt = ops.dequant4(torch.empty(cols, rows, dtype=t, device="cuda"), q, transpose=True)
        assert np.array_equal(y.double().cpu().numpy(), val) and torch.equal(yt, y.t()), name


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_quantise_large(built_lib, fmt, dtype):
    """A matrix of more than 12 Mi elements, whose 16-bit form goes another way; sampled rows."""
    from kiln_b200 import ops
    rows, cols = 3001, 4265
    x = torch.randn(rows, cols, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(TYPES[dtype])
    q = ops.quant4(x, fmt)
    y = ops.dequant4(torch.empty(rows, cols, device="cuda"), q)
    pick = np.unique(np.r_[0:5, 126:131, 2990:3001, np.random.RandomState(0).randint(0, rows, 60)])
    want = quantise(x[torch.from_numpy(pick).cuda()].double().cpu().numpy(), fmt)[2]
    assert np.array_equal(y.double().cpu().numpy()[pick], want) and np.array_equal(held(q)[pick], want)


@gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_quantise_borders(built_lib, fmt):
    from kiln_b200 import ops
    x = _borders(fmt)
    assert np.array_equal(held(ops.quant4(x.cuda(), fmt)), quantise(x.double().numpy(), fmt)[2])
    if fmt == NV4:                                                         # scales on and next to a border between two E4M3 numbers
        every = np.arange(2, 126)
        mid = np.array([(8 + b % 8 + 0.5) * 2.0 ** (b // 8 - 10) if b >= 8 else (b + 0.5) * 2.0 ** -9 for b in every])
        tops = (6 * mid).astype(np.float32)
        assert np.array_equal(tops / 6, mid)
        tops = np.concatenate([tops, np.nextafter(tops, np.float32(0)), np.nextafter(tops, np.float32(1e9))])
        x = torch.zeros(len(tops), 16)
        x[:, 3] = torch.from_numpy(tops)
        x[:, 4] = x[:, 3] / 3
        assert np.array_equal(held(ops.quant4(x.cuda(), fmt)), quantise(x.double().numpy(), fmt)[2])


@gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_quantise_extremes(built_lib, fmt):
    """Zeros, the smallest and the largest numbers, infinities and NaN."""
    from kiln_b200 import ops
    x = _x(5, 8, 64)
    x[0] = 0
    x[1] = -0.0
    x[2] *= 2.0 ** -140
    x[3] *= 2.0 ** 125
    x[4, 5] = float("inf")
    x[5, 40] = float("-inf")
    x[6, 17] = float("nan")
    x[7] = torch.finfo(torch.float32).max
    q = ops.quant4(x.cuda(), fmt)
    got, want = held(q), quantise(x.double().numpy(), fmt)[2]
    assert np.array_equal(got, want, equal_nan=True)
    assert np.isnan(want).sum() == 3 * BLOCK[fmt]
    y = ops.dequant4(torch.empty(8, 64, device="cuda"), q)
    assert np.array_equal(np.isnan(y.cpu().numpy()), np.isnan(want))


@gpu
@pytest.mark.parametrize("exp", [-64, -40, -9, 64])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantise_beyond_the_largest_scale(built_lib, dtype, exp):
    """|x| 2^-exp beyond what 32 bits hold: the scale stays at 448, the codes at 6 with their sign, and smaller elements of the block keep theirs."""
    from kiln_b200 import ops
    big = torch.tensor([3e38, -3e38, 1e30, -1e30, 2.0 ** 64, -2.0 ** 63, 0.0, -0.0]).double()
    small = torch.tensor([2688.0, -1344.0, 448.0, 112.0, -560.0, 2.0 ** 13, -2.0 ** 13, 9000.0]).double() * 2.0 ** exp
    x = torch.cat([torch.cat([big, small]), torch.cat([small, -small]), torch.cat([small, big / 4])])[None].to(TYPES[dtype])
    assert torch.isfinite(x.double()).all()
    code, s, val = quantise(x.double().numpy(), NV4, exp)
    q = ops.quant4(x.cuda(), NV4, exp)
    assert np.array_equal(held(q), val)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantise_strides(built_lib, dtype):
    """Rows that start anywhere, codes in wider rows, the bytes between and behind left as they were."""
    from kiln_b200 import ops
    for off, ld in [(0, 200), (8, 208), (1, 203), (3, 200)]:
        big = _x(off + ld, 70, ld, dtype).cuda()
        x = big[:, off:off + 190]
        q = ops.Quant4(torch.full((70, 112), 0xEE, dtype=torch.uint8, device="cuda"), torch.full((1 * 3 * 512,), 0xEE, dtype=torch.uint8, device="cuda"), 70, 190, NV4)
        ops.quant4(x, NV4, out=q)
        assert np.array_equal(held(q), quantise(x.double().cpu().numpy(), NV4)[2])
        c, sc = buffers(q)
        assert (c[:, 96:] == 0xEE).all()
        r = np.arange(70, 128)
        assert (sc[(r % 32) * 16 + (r // 32 % 4) * 4] == 0xEE).all()
        y = torch.full((70, ld), 7.0, dtype=TYPES[dtype], device="cuda")
        ops.dequant4(y[:, off:off + 190], q)
        assert np.array_equal(y[:, off:off + 190].double().cpu().numpy(), held(q)) and (y[:, :off] == 7).all() and (y[:, off + 190:] == 7).all()


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols,off,ld", [(1700, 8191, 0, 8191), (300, 1030, 1, 1037), (5, 255, 3, 259), (129, 4097, 0, 4098)])
def test_rows_of_any_alignment_agree(built_lib, fmt, dtype, rows, cols, off, ld):
    """Rows that do not start on 16 bytes give what a copy that does gives, bit for bit, and so does decoding into such rows."""
    from kiln_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, ld, generator=g, device="cuda").to(TYPES[dtype])[:, off:off + cols]
    wide = ops.padded_empty(rows, cols, TYPES[dtype], "cuda")
    wide.copy_(x)
    a, b = ops.quant4(x, fmt), ops.quant4(wide, fmt)
    assert torch.equal(a.codes, b.codes)
    assert np.array_equal(held(a), held(b)) if rows * cols < 1 << 20 else torch.equal(ops.dequant4(torch.empty(rows, cols, device="cuda"), a), ops.dequant4(torch.empty(rows, cols, device="cuda"), b))
    ops.dequant4(wide, b)
    for t in (False, True):
        shape = (cols, rows) if t else (rows, cols)
        big = torch.full((shape[0], shape[1] + 5), 7.0, dtype=TYPES[dtype], device="cuda")
        ops.dequant4(big[:, 2:2 + shape[1]], b, t)
        assert torch.equal(big[:, 2:2 + shape[1]], wide.T if t else wide)
        assert (big[:, :2] == 7).all() and (big[:, 2 + shape[1]:] == 7).all()


# ---------------------------------------------------------------- products
def _sum_bounds(a, w, K):
    """What fp32 sums of exact products may be off by, per element: a k step of 64 columns adds 65 numbers, each cut to 2^-23 of the largest of them, which is no
    larger than the sum of magnitudes."""
    return (K + 63) // 64 * 66 * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T)


def _pair(ops, seed, M, N, K, fmt, dtype="f16"):
    x, w = _x(seed, M, K, dtype), _x(seed + 1, N, K, "f32", 0.05)
    return ops.quant4(x.cuda(), fmt), ops.quant4(w.cuda(), fmt, -8 if fmt == NV4 else 0)


SHAPES = [(1, 1, 1), (1, 8, 32), (1, 2048, 512), (2, 300, 1000), (7, 130, 96), (8, 96, 2048), (9, 520, 64), (77, 256, 1024), (128, 128, 256), (129, 129, 257), (300, 257, 300),
          (257, 512, 4096), (1000, 64, 160), (513, 577, 1100)]


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(built_lib, fmt, M, N, K):
    import kiln_b200 as kb
    from kiln_b200 import ops
    A, W = _pair(ops, M + N + K, M, N, K, fmt)
    a, w = held(A), held(W)
    ref, off = a @ w.T, _sum_bounds(a, w, K)
    out = ops.padded_empty(M, N, torch.float32, "cuda")
    ops.linear4(out, A, W, ops.EPI_F32, alpha=0.75)
    assert kb.check_status() == 0
    err = np.abs(out.double().cpu().numpy() - 0.75 * ref)
    assert (err <= 0.75 * off + 2.0 ** -24 * np.abs(ref)).all(), f"fp32: {np.max(err / (off + 1e-30)):.3g} of the bound"
    assert np.linalg.norm(err) <= 4 * (K // 64 + 1) * 2.0 ** -23 * np.linalg.norm(ref)
    out16 = ops.linear4(ops.padded_empty(M, N, torch.float16, "cuda"), A, W, ops.EPI_F16).double().cpu().numpy()
    assert (np.abs(out16 - ref) <= off + 2.0 ** -11 * (np.abs(ref) + off) + 2.0 ** -25).all()
    g16 = ops.linear4(ops.padded_empty(M, N, torch.float16, "cuda"), A, W, ops.EPI_GELU16).double().cpu().numpy()
    g = gelu64(ref)
    # the slope of GELU is at most 1.13, its own error in fp32 5e-7
    assert (np.abs(g16 - g) <= 1.13 * off + 5e-7 + 2.0 ** -11 * (np.abs(g) + 1.13 * off) + 2.0 ** -25).all()
    gate = _x(3, 1, N)[0].cuda()
    for gt in (None, gate):
        r0 = _x(4, M, N).cuda()
        r = ops.padded_empty(M, N, torch.float32, "cuda")
        r.copy_(r0)
        ops.linear4(r, A, W, ops.EPI_RESID, gate=gt)
        gv = np.ones(N) if gt is None else gt.double().cpu().numpy()
        want = r0.double().cpu().numpy() + gv * ref
        # three more roundings: the gated product, the sum
        assert (np.abs(r.double().cpu().numpy() - want) <= np.abs(gv) * off * 1.01 + 2.0 ** -23 * (np.abs(want) + np.abs(gv * ref))).all()


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 8, 64), (3, 40, 96), (9, 100, 300), (130, 129, 256), (300, 520, 512), (257, 1000, 288)])
def test_product_gelu_in_4_bits(built_lib, fmt, M, N, K):
    """The hidden activations of an MLP: the codes and scales of GELU, and the next product on them."""
    import kiln_b200 as kb
    from kiln_b200 import ops
    A, W = _pair(ops, M + N, M, N, K, fmt)
    W.exp += 3                                                             # into GELU's bend and beyond
    H = ops.Quant4(torch.full((M, -(-N // 32) * 16 + 16), 0xEE, dtype=torch.uint8, device="cuda"),
                   torch.full((ops.lib().kb_quant4_scale_bytes(M, N, fmt),), 0xEE, dtype=torch.uint8, device="cuda"), M, N, fmt)
    ops.linear4(H, A, W, ops.EPI_GELU4)
    assert kb.check_status() == 0
    h = gelu64(held(A) @ held(W).T)
    _, s, val = quantise(h, fmt)
    got = held(H)
    # With g the GELU that the kernel has (5e-7 off h at most), s' its block's scale and S = max |h|: |got - val| <= |got - g| + |g - h| + |h - val|.
    # mx4: a value is 2 scales off at most (8 s saturates to 6 s), s' <= max(2 s, (S + 5e-7) / 4) <= 2 s + 1.3e-7, together 6 s + 1e-6.
    # nv4: 1 scale (half a step of 2 s; 6.4 s saturates to 6 s), s' <= 1.125 s + 1e-7, together 2.125 s + 1e-6.
    # Only values next to a border, and what is below GELU's own error, may differ at all.
    sw = np.repeat(s, BLOCK[fmt], 1)[:, :N]
    assert (np.abs(got - val) <= (6 if fmt == MX4 else 2.125) * sw + 1e-6).all()
    assert np.mean(np.abs(got - val) > 1e-6) <= 2e-3 + 4.0 / val.size
    c, sc = buffers(H)
    assert (c[:, -(-N // 32) * 16:] == 0xEE).all()                          # nothing behind the last 32 columns
    wide = read4(c, sc, M, -(-N // 32) * 32, fmt) if -(-N // 32) * 32 // BLOCK[fmt] <= 4 * -(-s.shape[1] // 4) else None
    if wide is not None:
        assert (wide[:, N:] == 0).all()
    pieces, r = -(-s.shape[1] // 4), np.arange(M)
    for b in range(s.shape[1], 4 * pieces):
        assert not sc[((r // 128) * pieces + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4].any()
    W2 = ops.quant4(_x(9, 72, N, "f32", 0.05).cuda(), fmt)
    out = ops.linear4(ops.padded_empty(M, 72, torch.float32, "cuda"), H, W2, ops.EPI_F32).double().cpu().numpy()
    w2 = held(W2)
    assert (np.abs(out - got @ w2.T) <= _sum_bounds(got, w2, N) + 1e-30).all()


@gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_product_garbage_behind_the_last_rows(built_lib, fmt):
    """Scales of rows that do not exist may be NaN: no stored column or row may show it."""
    from kiln_b200 import ops
    M, N, K = 70, 100, 200
    def make(x):
        q = ops.Quant4(torch.full((x.shape[0], 112), 0xFF, dtype=torch.uint8, device="cuda"),
                       torch.full((ops.lib().kb_quant4_scale_bytes(x.shape[0], K, fmt),), 0x7F if fmt == NV4 else 0xFF, dtype=torch.uint8, device="cuda"), x.shape[0], K, fmt)
        return ops.quant4(x.cuda(), fmt, out=q)
    A, W = make(_x(1, M, K)), make(_x(2, N, K))
    a, w = held(A), held(W)
    out = ops.linear4(ops.padded_empty(M, N, torch.float32, "cuda"), A, W, ops.EPI_F32).double().cpu().numpy()
    assert (np.abs(out - a @ w.T) <= _sum_bounds(a, w, K)).all()
    H = ops.linear4(ops.quant4_empty(M, N, fmt, "cuda"), A, W, ops.EPI_GELU4)
    assert np.isfinite(held(H)).all()


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [1, 3, 70, 300])
def test_product_shows_bad_blocks(built_lib, fmt, M):
    """A NaN or an infinity in an operand reaches every output that its block is summed into, and no other."""
    from kiln_b200 import ops
    x, w = _x(1, M, 256), _x(2, 40, 256)
    x[M // 2, 77] = float("inf")
    w[11, 200] = float("nan")
    out = ops.linear4(ops.padded_empty(M, 40, torch.float32, "cuda"), ops.quant4(x.cuda(), fmt), ops.quant4(w.cuda(), fmt), ops.EPI_F32).cpu().numpy()
    want = np.zeros((M, 40), bool)
    want[M // 2] = True
    want[:, 11] = True
    assert np.array_equal(np.isnan(out), want)
    A, W = ops.quant4(x.cuda(), fmt), ops.quant4(w.cuda(), fmt)
    assert np.array_equal(np.isnan(ops.linear4(ops.padded_empty(M, 40, torch.float16, "cuda"), A, W, ops.EPI_GELU16).float().cpu().numpy()), want)
    H = held(ops.linear4(ops.quant4_empty(M, 40, fmt, "cuda"), A, W, ops.EPI_GELU4))
    blocks = np.arange(40) // BLOCK[fmt]
    want[:, blocks == blocks[11]] = True                                   # in 4 bits the whole block of a NaN
    assert np.array_equal(np.isnan(H), want)


@gpu
def test_product_outputs_in_wider_rows(built_lib):
    """Strided outputs: what lies between the rows and behind the last one stays."""
    from kiln_b200 import ops
    for M, N in [(1, 100), (5, 33), (70, 100), (200, 264)]:
        A, W = _pair(ops, 3, M, N, 192, NV4)
        for epi, t in [(ops.EPI_F32, torch.float32), (ops.EPI_F16, torch.float16)]:
            big = torch.full((M + 3, 320), 7.0, dtype=t, device="cuda")
            ops.linear4(big[:M, :N], A, W, epi)
            want = ops.linear4(ops.padded_empty(M, N, t, "cuda"), A, W, epi)
            assert torch.equal(big[:M, :N], want) and (big[:, N:] == 7).all() and (big[M:] == 7).all()


@gpu
def test_product_of_no_rows(built_lib):
    from kiln_b200 import ops
    A, W = ops.quant4_empty(0, 64, NV4, "cuda"), ops.quant4(_x(1, 16, 64).cuda(), NV4)
    some = W.scales_ptr                                                    # an address, as an empty tensor has none
    assert ops.lib().kb_linear4(some, 16, None, some, 32, some, W.codes_ptr, 32, W.scales_ptr, 0, 16, 64, NV4, 0, 1.0, None, None) == 0 and A.rows == 0
    assert ops.lib().kb_quant4(some, 32, some, some, 64, 0, 0, 64, NV4, 0, None) == 0
    assert ops.lib().kb_linear4_dx(some, 64, 0, some, 64, W.codes_ptr, 32, W.scales_ptr, 0, 64, 64, NV4, 0, None, 0, None) == 0


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 64, 8), (5, 64, 72), (130, 192, 264), (300, 512, 1024)])
def test_input_gradient(built_lib, fmt, M, N, K):
    import kiln_b200 as kb
    from kiln_b200 import ops
    W = ops.quant4(_x(1, N, K, "f32", 0.05).cuda(), fmt, -8 if fmt == NV4 else 0)
    dy = _x(2, M, N, "f16").cuda()
    w, g = held(W), dy.double().cpu().numpy()
    ref = g @ w
    off = (N + 15) // 16 * 18 * 2.0 ** -23 * (np.abs(g) @ np.abs(w))       # k steps of 16 columns in the fp16 product
    d32 = ops.linear4_dx(torch.empty(M, K, device="cuda"), dy, W).double().cpu().numpy()
    assert kb.check_status() == 0
    assert (np.abs(d32 - ref) <= off).all()
    d16 = ops.linear4_dx(torch.empty(M, K, dtype=torch.float16, device="cuda"), dy, W).double().cpu().numpy()
    assert (np.abs(d16 - ref) <= off + 2.0 ** -11 * (np.abs(ref) + off) + 2.0 ** -25).all()
    # against differences of the product itself: <dy, y(a + e) - y(a)> = <dx, e> for a step e that 4 bits hold
    a, e = quantise(_x(3, M, K).double().numpy(), fmt)[2], quantise(_x(4, M, K).double().numpy(), fmt)[2]
    lhs, rhs = (g * ((a + e) @ w.T - a @ w.T)).sum(), (d32 * e).sum()
    assert abs(lhs - rhs) <= (off * np.abs(e)).sum() + 1e-9 * (np.abs(g) * (np.abs(a) @ np.abs(w).T)).sum()


@gpu
def test_captured_and_on_another_stream(built_lib):
    """Quantisation, product and gradient in a graph, replayed on new inputs, next to a call on another stream."""
    from kiln_b200 import ops
    M, N, K = 200, 320, 256
    W = ops.quant4(_x(1, N, K, "f32", 0.1).cuda(), NV4, -5)
    x, dy = torch.empty(M, K, dtype=torch.float16, device="cuda"), torch.empty(M, N, dtype=torch.float16, device="cuda")
    A, out, dx = ops.quant4_empty(M, K, NV4, "cuda"), torch.empty(M, N, device="cuda"), torch.empty(M, K, device="cuda")
    ws = torch.empty(ops.lib().kb_linear4_dx_workspace_bytes(N, K), dtype=torch.uint8, device="cuda")

    def step():
        ops.quant4(x, NV4, out=A)
        ops.linear4(out, A, W, ops.EPI_F32)
        ops.linear4_dx(dx, dy, W, workspace=ws)

    x.copy_(_x(2, M, K, "f16"))
    dy.copy_(_x(3, M, N, "f16"))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (10, 11, 12):
        xs, dys = _x(seed, M, K, "f16"), _x(seed + 50, M, N, "f16")
        x.copy_(xs)
        dy.copy_(dys)
        graph.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = ops.linear4(torch.empty(M, N, device="cuda"), ops.quant4(xs.cuda(), NV4), W, ops.EPI_F32)
            odx = ops.linear4_dx(torch.empty(M, K, device="cuda"), dys.cuda(), W)
        torch.cuda.synchronize()
        assert torch.equal(out, other) and torch.equal(dx, odx)
        a = quantise(xs.double().numpy(), NV4)[2]
        assert (np.abs(out.double().cpu().numpy() - a @ held(W).T) <= _sum_bounds(a, held(W), K)).all()


@gpu
def test_binding_errors_on_the_gpu(built_lib):
    """What the library refuses becomes KilnError with its code, what the tensors do not fit a ValueError; a tensor elsewhere never reaches a kernel."""
    import kiln_b200 as kb
    from kiln_b200 import ops
    x = _x(1, 5, 64).cuda()
    with pytest.raises(kb.KilnError) as e:
        ops.quant4(x, MX4, exp=1)
    assert e.value.code == -1
    with pytest.raises(kb.KilnError) as e:
        ops.dropout(torch.empty_like(x), x, torch.zeros(2, dtype=torch.int64, device="cuda"), 1.0)
    assert e.value.code == -1
    A, W = ops.quant4(x, NV4), ops.quant4(_x(2, 24, 64).cuda(), NV4)
    for bad in (lambda: ops.quant4(x.cpu(), NV4), lambda: ops.quant4(x.double(), NV4), lambda: ops.quant4(x[:, ::2], NV4), lambda: ops.quant4(x, 7),
                lambda: ops.quant4(x, NV4, out=ops.quant4_empty(5, 65, NV4, "cuda")), lambda: ops.dequant4(torch.empty(5, 63, device="cuda"), A),
                lambda: ops.linear4(torch.empty(5, 24, device="cuda"), A, W, ops.EPI_F16), lambda: ops.linear4(torch.empty(5, 25, device="cuda"), A, W, ops.EPI_F32),
                lambda: ops.linear4(torch.empty(5, 24), A, W, ops.EPI_F32), lambda: ops.linear4(x, A, W, ops.EPI_GELU4),
                lambda: ops.linear4(ops.quant4_empty(5, 24, MX4, "cuda"), A, W, ops.EPI_GELU4),
                lambda: ops.linear4(torch.empty(5, 24, device="cuda"), A, W, ops.EPI_RESID, gate=torch.ones(23, device="cuda")),
                lambda: ops.linear4(torch.empty(5, 24, device="cuda"), A, x, ops.EPI_F32), lambda: ops.linear4_dx(torch.empty(5, 64, device="cuda"), x[:, :24], W)):
        with pytest.raises(ValueError):
            bad()
    assert kb.check_status() == 0


@gpu
def test_rows_of_any_stride(built_lib):
    """A single row whose stride says nothing, an empty matrix, one column."""
    from kiln_b200 import ops
    row = _x(3, 1, 96)[0].cuda()
    for x in (row.expand(1, 96), torch.as_strided(row, (1, 96), (5, 1))):
        q = ops.quant4(x, NV4)
        assert np.array_equal(held(q), quantise(row[None].double().cpu().numpy(), NV4)[2])
        W = ops.quant4(_x(4, 40, 96).cuda(), NV4)
        want = ops.linear4(torch.empty(1, 40, device="cuda"), q, W, ops.EPI_F32)
        assert torch.equal(ops.linear4(torch.as_strided(torch.empty(40, device="cuda"), (1, 40), (3, 1)), q, W, ops.EPI_F32), want)
    e = ops.quant4(torch.empty(0, 96, device="cuda"), NV4)
    assert ops.linear4(torch.empty(0, 40, device="cuda"), e, W, ops.EPI_F32).shape == (0, 40) and ops.dequant4(torch.empty(0, 96, device="cuda"), e).numel() == 0
    c = _x(5, 7, 1).cuda()
    assert np.array_equal(held(ops.quant4(c, MX4)), quantise(c.double().cpu().numpy(), MX4)[2])


@gpu
def test_two_threads_on_two_streams(built_lib):
    """Calls from two host threads, each on its own stream, at the same time."""
    import threading
    from kiln_b200 import ops
    W = ops.quant4(_x(1, 512, 256, "f32", 0.1).cuda(), NV4, -5)
    xs = [_x(2 + i, 300 + 100 * i, 256, "f16").cuda() for i in range(2)]
    want = [ops.linear4(torch.empty(len(x), 512, device="cuda"), ops.quant4(x, NV4), W, ops.EPI_F32) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(50):
                y = ops.linear4(torch.empty(len(xs[i]), 512, device="cuda"), ops.quant4(xs[i], NV4), W, ops.EPI_F32)
                s.synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad

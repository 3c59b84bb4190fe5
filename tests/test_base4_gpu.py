"""The 4-bit, rotary and dropout calls together, as a LoRA is trained and served on a 4-bit base: one attention block's projections with a LoRA behind dropout,
rotary positions, attention, and all gradients back to the block's input and the LoRA, against the same chain in 64 bits on the values that the 4-bit matrices
hold."""
import numpy as np
import pytest
import torch

from util_ops4 import MX4, NV4, dropout_words, gelu64, held, quantise, rope64

pytestmark = pytest.mark.gpu
H, DH = 2, 128
D = H * DH


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _n(t):
    return t.double().cpu().numpy()


def _attention64(q, k, v, dout):
    """softmax(q k^T / sqrt(128)) v per head and its gradients."""
    T = len(q)
    split = lambda x: x.reshape(T, H, DH).transpose(1, 0, 2)
    q, k, v, dout = split(q), split(k), split(v), split(dout)
    s = q @ k.transpose(0, 2, 1) / np.sqrt(DH)
    p = np.exp(s - s.max(2, keepdims=True))
    p /= p.sum(2, keepdims=True)
    o = p @ v
    dp = dout @ v.transpose(0, 2, 1)
    ds = p * (dp - (dp * p).sum(2, keepdims=True)) / np.sqrt(DH)
    join = lambda x: x.transpose(1, 0, 2).reshape(T, D)
    return join(o), join(ds @ k), join(ds.transpose(0, 2, 1) @ q), join(p.transpose(0, 2, 1) @ dout)


@pytest.mark.parametrize("fmt", [pytest.param(MX4, id="mx4"), pytest.param(NV4, id="nv4")])
@pytest.mark.parametrize("T", [70, 256])
def test_lora_step_on_a_4bit_base(built_lib, fmt, T):
    import kiln_b200 as kb
    from kiln_b200 import ops
    R, P = 16, 0.25
    exp = -8 if fmt == NV4 else 0
    x = _randn(1, T, D).half().cuda()
    W = [ops.quant4((_randn(2 + i, D, D) / np.sqrt(D)).cuda(), fmt, exp) for i in range(3)]
    A = (_randn(10, R, D) / np.sqrt(D)).half().cuda()                    # the LoRA on the q projection
    B = (_randn(11, D, R) / np.sqrt(R)).half().cuda()
    dout = _randn(12, T, D).half().cuda()
    rng = torch.tensor([77, 5], device="cuda")
    pos = torch.stack([torch.zeros(T), torch.arange(T) // 16, torch.arange(T) % 16], 1).int().cuda()
    freq = ops.rope_freqs(DH, scaling=ops.ROPE_BASE, factor=2.0)
    axis = (np.arange(DH // 2) * 3 // (DH // 2)).astype(np.int32)

    # forward: 4-bit projections, the LoRA behind dropout added into q, rotary positions, attention
    x4 = ops.quant4(x, fmt)
    q, k, v = (torch.empty(T, D, device="cuda") for _ in range(3))
    for out, w in zip((q, k, v), W):
        ops.linear4(out, x4, w, ops.EPI_F32)
    xd = ops.dropout(torch.empty_like(x), x, rng, P)
    t = torch.empty(T, R, dtype=torch.float16, device="cuda")
    ops.linear16(t, xd, A, ops.EPI_F16)
    pad = torch.zeros(T, 64, dtype=torch.float16, device="cuda")
    pad[:, :R] = t
    Bpad = torch.zeros(D, 64, dtype=torch.float16, device="cuda")
    Bpad[:, :R] = B
    ops.linear16(q, pad, Bpad, ops.EPI_RESID)
    ops.rope([q, k], [q, k], [H, H], DH, pos, freq, axis)
    ws = torch.empty(kb.workspace_bytes(T, T, H, torch.float32), dtype=torch.uint8, device="cuda")
    o = ops.attn_self(torch.empty(T, D, device="cuda"), q, k, v, 1, T, H, workspace=ws)
    # backward
    dq, dk, dv = (torch.empty(T, D, device="cuda") for _ in range(3))
    ops.attn_bwd(dq, dk, dv, q, k, v, dout.float(), 1, T, T, 0, H)
    ops.rope([dq, dk], [dq, dk], [H, H], DH, pos, freq, axis, inverse=True)
    d16 = [g.half() for g in (dq, dk, dv)]
    dx = torch.zeros(T, D, device="cuda")
    part = torch.empty(T, D, device="cuda")
    for g, w in zip(d16, W):
        dx += ops.linear4_dx(part, g, w)
    dt = ops.linear16(torch.empty(T, 64, dtype=torch.float16, device="cuda"), d16[0], Bpad.t().contiguous(), ops.EPI_F16)   # dq . B
    At = torch.zeros(D, 64, dtype=torch.float16, device="cuda")
    At[:, :R] = A.t()
    dxd = ops.linear16(torch.empty(T, D, device="cuda"), dt, At, ops.EPI_F32)
    ops.dropout(dx, dxd, rng, P, resid=dx)
    assert kb.check_status() == 0

    # the same in 64 bits
    xn, Wn, An, Bn, pn = _n(x), [held(w) for w in W], _n(A), _n(B), pos.cpu().numpy().astype(np.int64)
    xq = quantise(xn, fmt)[2]
    keep = dropout_words(T, D, 77, 5) >= 16384
    qn, kn, vn = (xq @ w.T for w in Wn)
    tn = (np.where(keep, xn / (1 - P), 0)) @ An.T
    qn = qn + tn @ Bn.T
    rot = lambda m, inv: rope64(m, H, DH, DH, pn, freq, axis, True, 1.0, inv)
    qr, kr = rot(qn, False), rot(kn, False)
    on, dqn, dkn, dvn = _attention64(qr, kr, vn, _n(dout))
    dqn, dkn = rot(dqn, True), rot(dkn, True)
    dxn = dqn @ Wn[0] + dkn @ Wn[1] + dvn @ Wn[2] + np.where(keep, dqn @ Bn @ An / (1 - P), 0)
    rel = lambda a, b: np.linalg.norm(a - b) / np.linalg.norm(b)
    # The chain rounds to fp16 (2^-11 each, relative): q, k, v, P and t on the way to o; besides them dout, P, dS and the gradients on the way back. Independent roundings
    # add as squares, and a softmax of scores up to s turns a relative error e of a score into s e: scores here reach about 12.
    scale = np.abs(qr.reshape(T, H, DH).transpose(1, 0, 2) @ kr.reshape(T, H, DH).transpose(1, 2, 0)).max() / np.sqrt(DH)
    step = 2.0 ** -11
    assert rel(_n(q), qr) <= 3 * step and rel(_n(k), kr) <= 2.0 ** -20
    assert rel(_n(o), on) <= (4 + scale) * step
    for got, want in ((dq, dqn), (dk, dkn), (dv, dvn)):
        assert rel(_n(got), want) <= (6 + 2 * scale) * step
    assert rel(_n(dx), dxn) <= (8 + 2 * scale) * step


@pytest.mark.parametrize("fmt", [pytest.param(MX4, id="mx4"), pytest.param(NV4, id="nv4")])
@pytest.mark.parametrize("T", [1, 33, 300])
def test_mlp_on_a_4bit_base(built_lib, fmt, T):
    """Quantise, up-projection with GELU in 4 bits, down-projection into a gated residual."""
    import kiln_b200 as kb
    from kiln_b200 import ops
    F = 4 * D
    x, r0, gate = _randn(1, T, D).half().cuda(), _randn(2, T, D).cuda(), _randn(3, D).cuda()
    up, down = (ops.quant4((_randn(4 + i, *s) / np.sqrt(s[1])).cuda(), fmt, -8 if fmt == NV4 else 0) for i, s in enumerate(((F, D), (D, F))))
    h4 = ops.linear4(ops.quant4_empty(T, F, fmt, "cuda"), ops.quant4(x, fmt), up, ops.EPI_GELU4)
    r = ops.linear4(r0.clone(), h4, down, ops.EPI_RESID, gate=gate)
    assert kb.check_status() == 0
    h = gelu64(quantise(_n(x), fmt)[2] @ held(up).T)
    hq, got = quantise(h, fmt)[2], held(h4)
    # few values lie so near a border that fp32 decides otherwise
    assert np.mean(hq != got) <= 2e-3
    want = _n(r0) + _n(gate) * (got @ held(down).T)
    off = (F + 63) // 64 * 66 * 2.0 ** -23 * (np.abs(got) @ np.abs(held(down)).T)         # sums as in the products' own test
    assert (np.abs(_n(r) - want) <= np.abs(_n(gate)) * off * 1.01 + 2.0 ** -23 * (np.abs(want) + np.abs(_n(gate) * (got @ held(down).T)))).all()


def test_one_stream_of_captured_steps(built_lib):
    """Serving and training calls side by side in one graph, replayed on new inputs, give what eager calls give."""
    from kiln_b200 import ops
    T = 96
    W = ops.quant4((_randn(1, D, D) / 16).cuda(), NV4, -8)
    x, dy, rng = torch.empty(T, D, dtype=torch.float16, device="cuda"), torch.empty(T, D, dtype=torch.float16, device="cuda"), torch.tensor([1, 0], device="cuda")
    pos, freq = torch.arange(T).int()[:, None].cuda(), ops.rope_freqs(DH)
    y, dx = torch.empty(T, D, device="cuda"), torch.empty(T, D, device="cuda")

    def step():
        xd = ops.dropout(torch.empty_like(x), x, rng, 0.1)
        ops.linear4(y, ops.quant4(xd, NV4), W, ops.EPI_F32)
        ops.rope([y], [y], [H], DH, pos, freq)
        ops.linear4_dx(dx, dy, W)
        ops.dropout(dx, dx, rng, 0.1)

    x.copy_(_randn(2, T, D))
    dy.copy_(_randn(3, T, D))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (5, 6):
        x.copy_(_randn(seed, T, D))
        dy.copy_(_randn(seed + 1, T, D))
        rng[1:] += 1
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone(), dx.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], y) and torch.equal(got[1], dx)

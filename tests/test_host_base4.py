"""The 4-bit, rotary and dropout functions of the C++ op-set shim through their C trampolines: what they compute is what the calls of kiln_b200.ops compute, to
the bit; what they refuse becomes an exception."""
import ctypes

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
P = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
VP, I, D, F, SZ = ctypes.c_void_p, ctypes.c_int, ctypes.c_double, ctypes.c_float, ctypes.c_size_t


@pytest.fixture(scope="module")
def shim(built_lib):
    from kiln_b200 import build
    S = ctypes.CDLL(build.build_host())
    S.kbh_set_context.argtypes = [VP, VP, SZ]
    S.kbh_base4.argtypes = [VP, I, VP, I, VP, VP, I, I, VP, VP, I, I, I, I, VP, ctypes.c_char_p, I]
    S.kbh_base4_workspace.argtypes, S.kbh_base4_workspace.restype = [I, I, I, I], SZ
    S.kbh_rope_positions.argtypes = [VP, VP, I, I, I, I, I, VP, I, VP, VP, F, I, ctypes.c_char_p, I]
    S.kbh_lora_dropout.argtypes = [VP, VP, I, I, D, VP, ctypes.c_char_p, I]
    return S


def _call(f, *args):
    err = ctypes.create_string_buffer(256)
    return f(*args, err, 256), err.value.decode()


def test_errors_become_exceptions(shim):
    """No workspace, weights that do not follow one another: refused before anything runs."""
    buf = (ctypes.c_char * 4096)()
    a = ctypes.addressof(buf)
    shim.kbh_set_context(None, None, 0)
    rc, msg = _call(shim.kbh_base4, a, 64, a, 4, a, a, 64, 64, None, None, 0, 1, 0, 1, None)
    assert rc == -1 and "workspace" in msg
    shim.kbh_set_context(None, a, 4096)
    rc, msg = _call(shim.kbh_base4, a, 64, a, 4000, a, a, 64, 64, None, None, 0, 1, 0, 1, None)
    assert rc == -1 and "workspace" in msg
    rc, msg = _call(shim.kbh_base4, a, 64, a, 400, a, a, 128, 64, a, a, 64, 1, 0, 4, None)
    assert rc == -1 and "workspace" in msg
    rc, msg = _call(shim.kbh_lora_dropout, a, a, 4, 64, 1.5, a)
    assert rc == -1 and "lora_dropout" in msg
    rc, msg = _call(shim.kbh_rope_positions, a, a, 4, 1, 64, 63, 0, a, 1, a, None, 1.0, 0)
    assert rc == -1 and "rope_positions" in msg
    shim.kbh_set_context(None, None, 0)
    assert shim.kbh_base4_workspace(1, 32, 0, 1) == 256 + 512 and shim.kbh_base4_workspace(129, 64, 128, 0) == (129 * 32 + 255) // 256 * 256 + 1024 + (129 * 64 + 255) // 256 * 256 + 1024


@gpu
@pytest.mark.parametrize("fmt", [0, 1], ids=["mx4", "nv4"])
@pytest.mark.parametrize("T", [1, 45, 300])
def test_base4_matches_the_calls(shim, fmt, T):
    import kiln_b200 as kb
    from kiln_b200 import ops
    g = torch.Generator().manual_seed(T)
    randn = lambda *s: torch.randn(*s, generator=g)
    K, N = 256, 320
    exp = -8 if fmt else 0
    x, dy, up32, down32 = randn(T, K).half().cuda(), randn(T, N).half().cuda(), (randn(N, K) / 16).cuda(), (randn(K, N) / 16).cuda()
    gate = randn(K).cuda()
    need = max(shim.kbh_base4_workspace(T, K, N, fmt), 2 * N * K)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    shim.kbh_set_context(torch.cuda.current_stream().cuda_stream, P(ws), ws.numel())
    packed = [ops.quant4_empty(*w.shape, fmt, "cuda", exp) for w in (up32, down32)]
    for q, w in zip(packed, (up32, down32)):
        assert _call(shim.kbh_base4, P(q.codes), 0, P(w), 0, None, None, *w.shape, P(q.scales), None, 0, fmt, exp, 6, None) == (0, "")
        same = ops.quant4(w, fmt, exp)
        assert torch.equal(q.codes, same.codes) and torch.equal(ops.dequant4(torch.empty_like(w), q), ops.dequant4(torch.empty_like(w), same))
    up, down = packed
    x4 = ops.quant4(x, fmt)
    for epi, t in ((0, torch.float32), (1, torch.float16), (2, torch.float16)):
        y = torch.empty(T, N, dtype=t, device="cuda")
        assert _call(shim.kbh_base4, P(y), N, P(x), T, P(up.codes), P(up.scales), N, K, None, None, 0, fmt, exp, epi, None) == (0, "")
        assert torch.equal(y, ops.linear4(torch.empty_like(y), x4, up, epi))
    r = randn(T, K).cuda()
    want = ops.linear4(r.clone(), ops.linear4(ops.quant4_empty(T, N, fmt, "cuda"), x4, up, ops.EPI_GELU4), down, ops.EPI_RESID, gate=gate)
    assert _call(shim.kbh_base4, P(r), K, P(x), T, P(up.codes), P(up.scales), N, K, P(down.codes), P(down.scales), K, fmt, exp, 4, P(gate)) == (0, "")
    assert torch.equal(r, want)
    dx = torch.empty(T, K, device="cuda")
    assert _call(shim.kbh_base4, P(dx), K, P(dy), T, P(up.codes), P(up.scales), N, K, None, None, 0, fmt, exp, 5, None) == (0, "")
    assert torch.equal(dx, ops.linear4_dx(torch.empty_like(dx), dy, up))
    assert kb.check_status() == 0


@gpu
def test_rope_and_dropout_match_the_calls(shim):
    from kiln_b200 import ops
    g = torch.Generator().manual_seed(3)
    shim.kbh_set_context(torch.cuda.current_stream().cuda_stream, None, 0)
    T, H, DH, R = 50, 3, 64, 48
    q, k = torch.randn(T, H * DH, generator=g).cuda(), torch.randn(T, H * DH, generator=g).cuda()
    pos = torch.randint(0, 5000, (T, 2), generator=g, dtype=torch.int32).cuda()
    freq, axis = ops.rope_freqs(R), (np.arange(R // 2) % 2).astype(np.int32)
    want = ops.rope([torch.empty_like(q), torch.empty_like(k)], [q, k], [H, H], DH, pos, freq, axis, layout=ops.ROPE_INTERLEAVED, amplitude=1.1, inverse=True)
    assert _call(shim.kbh_rope_positions, P(q), P(k), T, H, DH, R, 1, P(pos), 2, freq.ctypes.data, axis.ctypes.data, 1.1, 1) == (0, "")
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    x, rng = torch.randn(40, 96, generator=g).half().cuda(), torch.tensor([9, 1], device="cuda")
    y = torch.empty_like(x)
    assert _call(shim.kbh_lora_dropout, P(y), P(x), 40, 96, 0.2, P(rng)) == (0, "")
    assert torch.equal(y, ops.dropout(torch.empty_like(x), x, rng, 0.2))


def test_powers_of_two_that_no_weight_has(shim):
    """Refused before anything runs, by the product as by the gradient."""
    buf = (ctypes.c_char * 65536)()
    a = (ctypes.addressof(buf) + 255) & ~255
    shim.kbh_set_context(None, a, 32768)
    for fmt, exp in ((0, 1), (0, -1), (1, 65), (1, -65), (1, 1000)):
        for what in (1, 5):
            rc, msg = _call(shim.kbh_base4, a, 64, a, 4, a, a, 64, 64, None, None, 0, fmt, exp, what, None)
            assert rc == -1 and "linear4" in msg and ("power of two" in msg or what == 5)
    shim.kbh_set_context(None, None, 0)

"""The handle of a 4-bit matrix: where its buffers lie is asked for in every call, since their tensors can be given other memory."""
import pytest
import torch

from util_ops4 import MX4, NV4

gpu = pytest.mark.gpu


def _made(rows=4, cols=64, fmt=MX4):
    from kiln_b200 import ops
    codes, scales = torch.zeros(rows, (cols + 31) // 32 * 16, dtype=torch.uint8), torch.zeros(2048, dtype=torch.uint8)
    return codes, scales, ops.Quant4(codes, scales, rows, cols, fmt)


def test_addresses_follow_the_tensors(built_lib):
    codes, scales, q = _made()
    assert (q.codes_ptr, q.scales_ptr, q.ld, q.device) == (codes.data_ptr(), scales.data_ptr(), 32, -1)
    other = torch.zeros(6, 48, dtype=torch.uint8)
    codes.data = other
    assert q.codes_ptr == other.data_ptr() and q.ld == 48 and q.codes is codes
    more = torch.zeros(4096, dtype=torch.uint8)
    scales.data = more[512:]
    assert q.scales_ptr == more.data_ptr() + 512


def test_addresses_follow_the_views_of_a_made_matrix(built_lib):
    from kiln_b200 import ops
    q = ops.quant4_empty(4, 64, NV4, "cpu")
    assert q.scales_ptr == q.codes_ptr + 4 * 32 and q.ld == 32 and q.device == -1
    assert q.codes.data_ptr() == q.codes_ptr and q.scales.data_ptr() == q.scales_ptr
    other = torch.zeros(4, 64, dtype=torch.uint8)
    q.codes.data = other
    assert q.codes_ptr == other.data_ptr() and q.ld == 64 and q.scales.data_ptr() == q.scales_ptr


def test_buffers_that_no_longer_fit_are_refused(built_lib):
    from kiln_b200 import ops
    look = lambda q: (q.codes_ptr, q.scales_ptr)
    codes, scales, q = _made()
    for bad in (torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 64, dtype=torch.uint8)[:, ::2], torch.zeros(128, dtype=torch.uint8)):
        codes.data = bad
        with pytest.raises(ValueError):
            look(q)
    codes, scales, q = _made()
    codes.untyped_storage().resize_(0)
    with pytest.raises(ValueError):
        look(q)
    codes, scales, q = _made()
    scales.untyped_storage().resize_(511)
    with pytest.raises(ValueError):
        look(q)
    codes, scales, q = _made()
    scales.data = torch.zeros(2048, dtype=torch.uint8)[::2]
    with pytest.raises(ValueError):
        look(q)
    q = ops.quant4_empty(4, 64, NV4, "cpu")
    q.scales.untyped_storage().resize_(4 * 32 + 511)
    with pytest.raises(ValueError):
        look(q)
    with pytest.raises(ValueError):
        ops.linear4(torch.zeros(4, 4), q, q, ops.EPI_F32)
    with pytest.raises(ValueError):
        look(ops.Quant4.__new__(ops.Quant4))


def test_matrices_of_few_or_no_rows(built_lib):
    from kiln_b200 import ops
    one = ops.Quant4(torch.zeros(16, dtype=torch.uint8).expand(1, 16), torch.zeros(512, dtype=torch.uint8), 1, 20, MX4)
    assert one.ld == 16
    none = ops.quant4_empty(0, 64, NV4, "cpu")
    assert none.ld == 32 and none.codes.shape == (0, 32) and none.scales.numel() == 0
    assert ops.Quant4(none.codes, none.scales, 0, 64, NV4).rows == 0


@gpu
def test_a_weight_moved_off_the_gpu_and_back(built_lib):
    """A weight that leaves the GPU is refused until it is back, and is then read where it has come to lie."""
    from kiln_b200 import ops
    g = torch.Generator().manual_seed(1)
    x = ops.quant4(torch.randn(5, 256, generator=g).cuda(), NV4)
    made = ops.quant4(torch.randn(40, 256, generator=g).cuda(), NV4, -4)
    codes, scales = made.codes.clone(), made.scales.clone()
    W = ops.Quant4(codes, scales, 40, 256, NV4, -4)
    run = lambda: ops.linear4(torch.empty(5, 40, device="cuda"), x, W, ops.EPI_F32)
    want = ops.linear4(torch.empty(5, 40, device="cuda"), x, made, ops.EPI_F32)
    assert torch.equal(run(), want)
    codes.data, scales.data = codes.cpu(), scales.cpu()
    assert W.device == -1
    with pytest.raises(ValueError):
        run()
    held = torch.full((1 << 20,), 0x33, dtype=torch.uint8, device="cuda")      # takes the freed memory
    codes.data, scales.data = codes.cuda(), scales.cuda()
    assert W.device == 0 and torch.equal(run(), want) and W.codes_ptr == codes.data_ptr() and held.numel()
    y = ops.dequant4(torch.empty(40, 256, device="cuda"), W)
    assert torch.equal(y, ops.dequant4(torch.empty(40, 256, device="cuda"), made))


def test_powers_of_two(built_lib):
    """-64 to 64 wherever a handle is made or changed; a factor of a product that 32 bits do not hold is refused."""
    from kiln_b200 import ops
    codes, scales, q = _made(fmt=NV4)
    for good in (-64, 0, 64):
        assert ops.Quant4(codes, scales, 4, 64, NV4, good).exp == good == ops.quant4_empty(4, 64, NV4, "cpu", good).exp
        q.exp = good
        assert q.exp == good
    for bad in (-65, 65, 1000, -2 ** 31, 2 ** 40):
        for make in (lambda: ops.Quant4(codes, scales, 4, 64, NV4, bad), lambda: ops.quant4_empty(4, 64, NV4, "cpu", bad), lambda: setattr(q, "exp", bad)):
            with pytest.raises((ValueError, OverflowError)):
                make()
    with pytest.raises(TypeError):
        q.exp = 1.5
    with pytest.raises(ValueError):
        del q.exp
    assert q.exp == 64


@gpu
def test_factors_of_a_product(built_lib):
    from kiln_b200 import ops
    A, W = ops.quant4(torch.ones(3, 64).cuda(), NV4), ops.quant4(torch.ones(8, 64).cuda(), NV4)
    run = lambda alpha=1.0: ops.linear4(torch.empty(3, 8, device="cuda"), A, W, ops.EPI_F32, alpha=alpha)
    plain = run()
    for ea, ew, alpha in [(64, 64, 2.0 ** -10), (-64, -64, 1.0), (64, -64, 1.0), (-64, -63, 2.0 ** 127)]:
        A.exp, W.exp = ea, ew
        assert torch.equal(run(alpha).double(), (plain.double() * 2.0 ** (ea + ew) * alpha).float().double())
    for ea, ew, alpha in [(64, 64, 1.0), (64, 64, -4.0), (-64, -64, 1e-30), (0, 0, float("nan")), (0, 0, float("inf")), (0, 0, 1e300), (-64, -64, 1.0 / 3)]:
        A.exp, W.exp = ea, ew
        with pytest.raises(ValueError):
            run(alpha)
    A.exp = W.exp = 0
    assert torch.equal(run(0.0), torch.zeros_like(plain))


def test_copies_and_pickles(built_lib):
    """A copy shares the buffers, a deep copy and a pickled one have their own; a module with a 4-bit weight can be copied and saved."""
    import copy
    import io
    import pickle
    from kiln_b200 import ops
    made = ops.quant4_empty(5, 70, NV4, "cpu", -7)
    made.codes.copy_(torch.arange(5 * 48).view(5, 48) % 256)
    made.scales.copy_(torch.arange(1024) % 120)
    wide = torch.zeros(6, 100, dtype=torch.uint8)
    own = ops.Quant4(wide[:, :64], torch.zeros(600, dtype=torch.uint8), 5, 70, MX4)
    for q in (made, own, ops.quant4_empty(0, 70, MX4, "cpu")):
        same = copy.copy(q)
        assert same.codes.data_ptr() == q.codes.data_ptr() and same.scales.data_ptr() == q.scales.data_ptr()
        for other in (same, copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
            assert (other.rows, other.cols, other.fmt, other.exp) == (q.rows, q.cols, q.fmt, q.exp) and type(other) is ops.Quant4
            assert torch.equal(other.codes, q.codes) and torch.equal(other.scales, q.scales)
            assert other is same or q.rows == 0 or (other.codes_ptr != q.codes_ptr and other.scales_ptr != q.scales_ptr)
    layer = torch.nn.Module()
    layer.weight = made
    assert torch.equal(copy.deepcopy(layer).weight.codes, made.codes)
    f = io.BytesIO()
    torch.save(layer, f)
    f.seek(0)
    assert torch.equal(torch.load(f, weights_only=False).weight.scales, made.scales)

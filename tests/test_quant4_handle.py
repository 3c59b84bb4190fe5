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

"""Weight gradients of experts whose rows are summed in pieces: the workspace for the pieces' sums follows the rows,
not the number of experts, and every group gets its own pieces."""
import pytest
import torch


@pytest.mark.parametrize('rows,experts,inputs,outputs', [
    (131072, 1024, 1024, 1024), (131072, 4096, 1024, 1024), (131072, 64, 256, 512), (262144, 8, 512, 2048),
    (65536, 48, 64, 3), (1 << 20, 2, 64, 64), (300, 500, 40, 72), (5431, 5, 40, 72), (1 << 22, 32768, 128, 128),
    ((1 << 31) - 1, 3, 8, 8)])
def test_workspace_of_grouped_gradients(native, rows, experts, inputs, outputs):
    """Partial sums below twice what the operands hold, however many experts there are."""
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        partial = native.odie_linear_workspace(rows, experts, 1, inputs, outputs, dtype, 0, 1, 0)
        assert 0 <= partial <= 2 * size * rows * (inputs + outputs) + 256
    assert native.odie_linear_workspace(0, experts, 1, inputs, outputs, 1, 0, 1, 0) == 0


# counts around a piece of 256 rows: groups of one piece and of several next to each other, empty ones between
COUNTS = [('mixed', [257, 1, 513, 256, 0, 255, 770, 0, 0, 300, 511, 512, 258, 2]),
          ('all of two pieces', [257] * 40), ('one long among many', [3] * 100 + [5000] + [1] * 100),
          ('first and last', [1025] + [0] * 30 + [600])]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', (torch.float16, torch.float32), ids=str)
@pytest.mark.parametrize('name,counts', COUNTS, ids=[c[0] for c in COUNTS])
def test_pieces_of_every_group(name, counts, dtype):
    """Whole numbers: every sum is exact in fp32, and rounded once."""
    from odie_amd.linear import linear
    generator = torch.Generator(device='cuda').manual_seed(len(counts))
    n, inputs, outputs = sum(counts) + 5, 8, 16

    def values(*shape):
        return torch.randint(-2, 3, shape, generator=generator, device='cuda').to(dtype)
    x, w, b, dy = values(n, inputs), values(len(counts), outputs, inputs), values(len(counts), outputs), values(n, outputs)
    offsets = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device='cuda')
    print('pieces', name, dtype, n, flush=True)
    w.requires_grad_(True)
    b.requires_grad_(True)
    dw, db = torch.autograd.grad(linear(x, w, b, offsets=offsets), (w, b), dy)
    at = 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        assert torch.equal(dw[e], (dy[rows].double().t() @ x[rows].double()).to(dtype)), e
        assert torch.equal(db[e], dy[rows].double().sum(0).to(dtype)), e
        at += count

"""odie_amd.linear with 4-bit weights, and rows, against the formula in 64 bits on the values they stand for (bounds
derived in rows64: the products of 4-bit values are exact, and sums are fp32's)."""
import pytest
import torch

from microscale64 import values64
from odie_amd.linear import ACTIVATIONS, linear
from odie_amd.microscale import Microscaled, quantize
from rows64 import DTYPES, Layer64, check

pytestmark = pytest.mark.gpu

# few rows and their edges; ends of blocks, slabs and tiles; every tile; rows that reach LDS by each way
SHAPES = [(1, 1, 1), (1, 2048, 2048), (2, 31, 64), (3, 33, 65), (16, 1000, 24), (17, 128, 40), (32, 200, 300), (33, 64, 63),
          (63, 64, 63), (64, 128, 64), (65, 130, 129), (200, 257, 100), (129, 8, 300), (100, 3, 70), (7, 2049, 130),
          (1000, 520, 264), (300, 1056, 72)]
LARGE = [(32773, 24, 40), (4099, 40, 1000), (2500, 136, 2056), (66000, 264, 520), (66000, 265, 517), (8192, 992, 2048)]


def _values(generator, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=generator, device='cuda') * scale).to(dtype)


def _case(seed, n, inputs, outputs, dtype, lead=(), whole=False):
    generator = torch.Generator(device='cuda').manual_seed(seed)
    if whole:       # small whole numbers, which 4 bits hold too: every sum is exact, and relu's mask with it
        def values(*shape):
            value = torch.randint(-2, 3, shape, generator=generator, device='cuda').to(dtype)
            value[..., 0] = 4
            return value
        return values(n, inputs), values(*lead, outputs, inputs), values(*lead, outputs), values(n, outputs), values(n, outputs)
    return (_values(generator, dtype, n, inputs), _values(generator, dtype, *lead, outputs, inputs, scale=inputs ** -0.5),
            _values(generator, dtype, *lead, outputs, scale=0.5), _values(generator, dtype, n, outputs),
            _values(generator, dtype, n, outputs))


def _weight64(q):
    return values64(q.codes.view(-1, q.codes.shape[-1]), q.scales.view(-1, q.scales.shape[-1]), q.width).view(q.shape)


def _check_held(got, expected, error, what):
    """check, where a sum past the type's largest value, by more than half a step and what it may be off by, is an
    infinity: 65536 dy's bias gradient in fp16, whose largest is 65504."""
    most = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    past = expected.abs() - error > most
    assert torch.equal(got[past].double(), torch.copysign(torch.full_like(expected, float('inf')), expected)[past]), what
    check(torch.where(past, 0.0, got.double()), torch.where(past, 0.0, expected), error, what)


def _check_rows_of_t(x, q, b, r, dy, activation, what):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, b, r)]
    y = linear(leaves[0], q, leaves[1], activation=activation, residual=leaves[2])
    wanted = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, wanted, dy))
    dx, db, dr = [next(grads) if t is not None else None for t in leaves]
    # the weight's values as x's type holds them
    layer = Layer64(x, _weight64(q).to(x.dtype), b, r, dy, activation)
    check(y, layer.y, layer.y_error, what + ' y')
    check(dx, layer.dx, layer.dx_error, what + ' dx')
    if b is not None:
        _check_held(db, layer.db, layer.db_error, what + ' db')
    if r is not None:
        assert torch.equal(dr, dy)
    assert torch.equal(linear(x, q, b, activation=activation, residual=r), y), what


def _check_rows_of_4_bits(x, q, b, r, activation, what):
    xq = quantize(x)
    y = linear(xq, q, b, activation=activation, residual=r)
    assert y.dtype == x.dtype
    layer = Layer64(_Typed(_weight64(xq), x.dtype), _weight64(q), b, r, None, activation)
    check(y, layer.y, layer.y_error, what + ' y of 4-bit rows')


class _Typed:
    """64-bit values that Layer64 takes for a tensor of another type."""

    def __init__(self, value, dtype):
        self.value, self.dtype, self.shape, self.device = value, dtype, value.shape, value.device

    def detach(self):
        return self.value


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', SHAPES + LARGE, ids=str)
def test_layer_matches_formula(shape, dtype):
    n, inputs, outputs = shape
    activation = ACTIVATIONS[(n + inputs) % len(ACTIVATIONS)]
    print('linear of 4 bits', shape, dtype, activation, flush=True)
    x, w, b, r, dy = _case(n + outputs, n, inputs, outputs, dtype, whole=activation == 'relu')
    q = quantize(w)
    _check_rows_of_t(x, q, b, r, dy, activation, str(shape))
    _check_rows_of_4_bits(x, q, b, r, activation, str(shape))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('activation', ACTIVATIONS)
def test_every_activation_bias_and_residual(activation, dtype):
    for n in (5, 70):
        for bias, residual in ((False, False), (True, False), (False, True), (True, True)):
            x, w, b, r, dy = _case(5, n, 96, 50, dtype, whole=activation == 'relu')
            b, r = b if bias else None, r if residual else None
            _check_rows_of_t(x, quantize(w), b, r, dy, activation, activation)
            _check_rows_of_4_bits(x, quantize(w), b, r, activation, activation)


# few tiles, whose depth is cut into shares: shares that end inside slabs, uneven and empty ones, one and two a CU
SHARES = [(65, 264, 70), (100, 512, 64), (70, 520, 130), (66, 1032, 65), (65, 1288, 96), (100, 2048, 200), (129, 2312, 64),
          (100, 4104, 72), (300, 1024, 4096), (20, 520, 13200), (33, 4096, 8000), (64, 2304, 40)]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', SHARES, ids=str)
def test_shares_of_the_depth(shape, dtype):
    n, inputs, outputs = shape
    for activation in ('none', 'silu'):
        print('shares', shape, dtype, activation, flush=True)
        x, w, b, r, dy = _case(n + inputs, n, inputs, outputs, dtype)
        _check_rows_of_t(x, quantize(w), b, r, dy, activation, str(shape))
        _check_rows_of_4_bits(x, quantize(w), b, r, activation, str(shape))
    # every sum exact: each share takes its own part, once
    x, w, b, r, dy = _case(n + inputs, n, inputs, outputs, dtype, whole=True)
    _check_rows_of_t(x, quantize(w), b, r, dy, 'relu', str(shape))
    _check_rows_of_4_bits(x, quantize(w), b, r, 'relu', str(shape))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_shares_of_experts(dtype):
    """Groups that end inside tiles, an empty one, and rows of no expert."""
    counts, inputs, outputs = [70, 0, 200, 1], 2312, 100
    n = sum(counts) + 40
    x, w, b, r, _ = _case(11, n, inputs, outputs, dtype, lead=(len(counts),))
    x[n - 40:] = float('nan')
    q, offsets = quantize(w), _offsets(counts)
    y = linear(x, q, b, activation='gelu', residual=r, offsets=offsets)
    y4 = linear(quantize(x), q, b, activation='gelu', residual=r, offsets=offsets)
    wide, wide_x = _weight64(q), _weight64(quantize(x))
    at = 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        layer = Layer64(x[rows], wide[e].to(dtype), b[e], r[rows], None, 'gelu')
        check(y[rows], layer.y, layer.y_error, 'group %d' % e)
        layer = Layer64(_Typed(wide_x[rows], dtype), wide[e], b[e], r[rows], None, 'gelu')
        check(y4[rows], layer.y, layer.y_error, 'group %d, 4-bit rows' % e)
        at += count
    assert torch.equal(y[at:], r[at:]) and torch.equal(y4[at:], r[at:])


# gradients that are formed in one pass: each tile's and slab's edges, rows that fill no tile
ONE_PASS = [(65536, 1, 8), (65537, 64, 9), (65600, 65, 64), (65665, 128, 71), (65700, 129, 264), (66000, 256, 136),
            (70000, 33, 12), (65999, 250, 520)]


@pytest.mark.parametrize('dtype', (torch.float16, torch.bfloat16), ids=str)
@pytest.mark.parametrize('shape', ONE_PASS, ids=str)
def test_gradients_in_one_pass(shape, dtype):
    n, inputs, outputs = shape
    for activation in ACTIVATIONS[1:]:
        print('gradients of 4 bits', shape, dtype, activation, flush=True)
        x, w, b, r, dy = _case(inputs, n, inputs, outputs, dtype, whole=activation == 'relu')
        _check_rows_of_t(x, quantize(w), b, r, dy, activation, str(shape) + activation)
        # alone, and from rows of another stride and start
        q = quantize(w)
        leaf, shift = x.clone().requires_grad_(True), b.clone().requires_grad_(True)
        whole = torch.autograd.grad(linear(leaf, q, shift, activation=activation), (leaf, shift), dy)
        assert torch.equal(torch.autograd.grad(linear(leaf, q, b, activation=activation), leaf, dy)[0], whole[0])
        wide = torch.zeros(n, outputs + 13, dtype=dtype, device='cuda')
        wide[:, 5:5 + outputs] = dy
        got = torch.autograd.grad(linear(leaf, q, shift, activation=activation), (leaf, shift), wide[:, 5:5 + outputs])
        assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])


@pytest.mark.parametrize('dtype', (torch.float16, torch.bfloat16), ids=str)
@pytest.mark.parametrize('inputs', (48, 100, 200))
def test_experts_gradients_in_one_pass(inputs, dtype):
    """Groups that end inside tiles, empty ones, and rows of no expert, whose upstream and sums may be anything."""
    counts, rest, outputs = [30001, 1, 0, 20000, 127, 16384, 0], 77, 72
    n, experts = sum(counts) + rest, len(counts)
    x, w, b, r, dy = _case(inputs, n, inputs, outputs, dtype, lead=(experts,))
    x[sum(counts):], dy[sum(counts):] = float('nan'), float('inf')
    q, offsets = quantize(w), _offsets(counts)
    leaves = [t.detach().requires_grad_(True) for t in (x, b)]
    dx, db = torch.autograd.grad(linear(leaves[0], q, leaves[1], activation='gelu', offsets=offsets), leaves, dy)
    at = 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        layer = Layer64(x[rows], _weight64(q)[e].to(dtype), b[e], None, dy[rows], 'gelu')
        check(dx[rows], layer.dx, layer.dx_error, 'expert %d' % e)
        check(db[e], layer.db, layer.db_error, 'expert %d' % e)
        at += count
    assert not dx[at:].any()


def _offsets(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device='cuda')


GROUPS = [('one row each', [1] * 9, 0), ('empty ones', [0, 5, 0, 0, 64, 0], 0), ('tile edges', [64, 128, 63, 65, 1], 0),
          ('rows of no expert', [30, 0, 40], 77), ('all of no expert', [0, 0], 50), ('one of all', [0, 700, 0], 3),
          ('many', [(7 * e) % 5 for e in range(200)], 11), ('more experts than rows', [e % 97 == 0 for e in range(500)], 1),
          ('a long one', [300, 5000, 2, 0, 129], 0)]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('name,counts,rest', GROUPS, ids=[g[0] for g in GROUPS])
def test_experts_match_formula(name, counts, rest, dtype):
    counts = [int(c) for c in counts]
    n, inputs, outputs, experts = sum(counts) + rest, 40, 72, len(counts)
    print('experts of 4 bits', name, dtype, n, flush=True)
    x, w, b, r, dy = _case(len(name), n, inputs, outputs, dtype, lead=(experts,))
    held = sum(counts)
    x[held:] = float('nan')     # whatever lies in rows of no expert reaches nothing else
    q, offsets = quantize(w), _offsets(counts)
    leaves = [t.detach().requires_grad_(True) for t in (x, b, r)]
    y = linear(leaves[0], q, leaves[1], activation='silu', residual=leaves[2], offsets=offsets)
    dx, db, _ = torch.autograd.grad(y, leaves, dy)
    xq = quantize(x)
    y4 = linear(xq, q, b, activation='silu', residual=r, offsets=offsets)
    wide, wide_x = _weight64(q), _weight64(xq)
    at = 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        layer = Layer64(x[rows], wide[e].to(dtype), b[e], r[rows], dy[rows], 'silu')
        check(y[rows], layer.y, layer.y_error, name)
        check(dx[rows], layer.dx, layer.dx_error, name)
        check(db[e], layer.db, layer.db_error, name)
        layer = Layer64(_Typed(wide_x[rows], dtype), wide[e], b[e], r[rows], None, 'silu')
        check(y4[rows], layer.y, layer.y_error, name + ', 4-bit rows')
        at += count
    assert torch.equal(y[held:], r[held:]) and torch.equal(y4[held:], r[held:]) and not dx[held:].any()
    assert not linear(x, q, b, offsets=offsets)[held:].any() and not linear(xq, q, b, offsets=offsets)[held:].any()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('counts', ([5000] * 8, [3000, 9000, 0, 40, 1500]), ids=str)
def test_experts_in_large_tiles(counts, dtype):
    n, inputs, outputs = sum(counts) + 100, 192, 520
    x, w, b, r, _ = _case(7, n, inputs, outputs, dtype, lead=(len(counts),))
    q, offsets = quantize(w), _offsets(counts)
    y, y4 = linear(x, q, b, offsets=offsets), linear(quantize(x), q, b, offsets=offsets)
    wide, wide_x = _weight64(q), _weight64(quantize(x))
    at = 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        layer = Layer64(x[rows], wide[e].to(dtype), b[e], None, None, 'none')
        check(y[rows], layer.y, layer.y_error, str(counts))
        layer = Layer64(_Typed(wide_x[rows], dtype), wide[e], b[e], None, None, 'none')
        check(y4[rows], layer.y, layer.y_error, str(counts))
        at += count


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n', (1, 20, 100, 40000))
def test_rows_of_any_stride_and_start(n, dtype):
    generator = torch.Generator(device='cuda').manual_seed(n)
    wide = _values(generator, dtype, n, 333)
    q = quantize(_values(generator, dtype, 136, 150))
    residual = _values(generator, dtype, n, 300)
    for x in (wide[:, 5:155], wide[:, :150], wide[:, 160:310]):
        y = linear(x, q, residual=residual[:, 9:145])
        assert torch.equal(y, linear(x.contiguous(), q, residual=residual[:, 9:145].contiguous()))
    assert torch.equal(linear(quantize(wide[:, 5:155]), q), linear(quantize(wide[:, 5:155].contiguous()), q))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', ((3, 2047, 8192), (3, 2045, 8192), (3, 2046, 8192), (20, 1023, 8192), (40, 1027, 8192)), ids=str)
def test_few_rows_that_end_inside_16_bytes(shape, dtype):
    """Every lane's last loads move down in registers, with the CUs full of other waves."""
    n, inputs, outputs = shape
    x, w, b, _, _ = _case(inputs, n, inputs, outputs, dtype)
    q = quantize(w)
    for _ in range(3):
        layer = Layer64(x, _weight64(q).to(dtype), b, None, None, 'none')
        check(linear(x, q, b), layer.y, layer.y_error, str(shape))


def test_blocks_of_nan_and_infinite_rows():
    """A NaN block makes its output column NaN and no other; a NaN or infinite row its own outputs."""
    for n, outputs in ((3, 40), (50, 70), (3000, 300)):
        generator = torch.Generator(device='cuda').manual_seed(n)
        x, w = _values(generator, torch.bfloat16, n, 100), _values(generator, torch.bfloat16, outputs, 100)
        w[7, 40] = float('nan')
        x[1, 99] = float('inf')
        q = quantize(w)
        others = torch.arange(n, device='cuda') != 1
        columns = torch.arange(outputs, device='cuda') != 7
        for y in (linear(x, q), linear(quantize(x), q)):
            assert y[:, 7].isnan().all() and y[others][:, columns].isfinite().all() and not y[1].isfinite().any()
        assert linear(quantize(x), q)[1].isnan().all()


def test_wide_ranges_of_scales():
    """Blocks of very differing sizes, whose scales the products take in full (fp32 and bf16 hold them)."""
    generator = torch.Generator(device='cuda').manual_seed(8)
    for dtype in (torch.float32, torch.bfloat16):
        size = torch.exp2(torch.randint(-60, 60, (1, 8, 1), generator=generator, device='cuda').double()).expand(1, 8, 32).reshape(1, 256)
        for n in (9, 200):
            x = (_values(generator, torch.float32, n, 256) / size).to(dtype)
            w = (_values(generator, torch.float32, 80, 256) * size).to(dtype)
            q = quantize(w)
            _check_rows_of_4_bits(x, q, None, None, 'none', 'ranges')
            layer = Layer64(x, _weight64(q).to(dtype), None, None, None, 'none')
            check(linear(x, q), layer.y, layer.y_error, 'ranges')


def test_weights_that_fp16_does_not_hold_are_rounded_to_it():
    x = torch.ones(2, 32, device='cuda', dtype=torch.float16)
    q = quantize(torch.full((1, 32), 2.0 ** -25, device='cuda'))
    assert not linear(x, q).any()                                               # half the least subnormal: to even
    q = quantize(torch.full((1, 32), 2.0 ** 17, device='cuda'))
    assert linear(x, q).isinf().all()
    assert (linear(x.float(), q) == 2.0 ** 22).all()


def test_no_rows_and_refusals():
    x = torch.randn(4, 64, device='cuda')
    w = torch.randn(3, 6, 64, device='cuda')
    q, dense, x4 = quantize(w), quantize(w[0]), quantize(x)
    offsets = torch.tensor([0, 1, 2, 4], dtype=torch.int32, device='cuda')
    assert linear(x[:0], dense).shape == (0, 6) and linear(quantize(x[:0]), dense).shape == (0, 6)
    leaf = x[:0].clone().requires_grad_(True)
    assert torch.autograd.grad(linear(leaf, dense).sum(), leaf)[0].shape == (0, 64)
    for bad in (lambda: linear(x, q), lambda: linear(x, dense, offsets=offsets), lambda: linear(x[:, :60], dense),
                lambda: linear(x4, w[0]), lambda: linear(quantize(w), dense), lambda: linear(x, dense, torch.zeros(5, device='cuda')),
                lambda: linear(x.half(), dense, torch.zeros(6, device='cuda')), lambda: linear(x, dense, residual=x),
                lambda: linear(x4, dense, torch.zeros(6, device='cuda', requires_grad=True)),
                lambda: linear(x4, dense, residual=torch.zeros(4, 6, device='cuda', requires_grad=True)),
                lambda: linear(x4, dense, torch.zeros(6, device='cuda', dtype=torch.float16)),
                lambda: linear(x, quantize(w[:, :0])), lambda: linear(x, dense, activation='tanh')):
        with pytest.raises(ValueError):
            bad()


def test_gradient_against_differences():
    """A layer without activation is linear in x: differences of exact whole numbers are the gradient itself."""
    generator = torch.Generator(device='cuda').manual_seed(9)
    x = torch.randint(-4, 5, (3, 40), generator=generator, device='cuda').float()
    q = quantize(torch.randint(-3, 4, (20, 40), generator=generator, device='cuda').float())
    mix = torch.randint(-2, 3, (3, 20), generator=generator, device='cuda').float()
    leaf = x.clone().requires_grad_(True)
    gradient, = torch.autograd.grad((linear(leaf, q) * mix).sum(), leaf)
    for i in range(3):
        for k in range(40):
            up = x.clone()
            up[i, k] += 1
            assert float(((linear(up, q) - linear(x, q)) * mix).sum()) == float(gradient[i, k])


def test_what_a_backward_reads_must_not_change():
    x = torch.randn(4, 64, device='cuda', requires_grad=True)
    q = quantize(torch.randn(6, 64, device='cuda'))
    y = linear(x, q)
    q.codes.zero_()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    x4 = Microscaled(q.codes, q.scales, 64, torch.float32)
    assert not linear(x.detach(), x4).any()

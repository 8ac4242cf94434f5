"""odie_amd.linear against its formulas in 64 bits (bounds derived in rows64) and against differences."""
import pytest
import torch

from odie_amd.linear import ACTIVATIONS, linear
from rows64 import DTYPES, Layer64, check

pytestmark = pytest.mark.gpu

# one value; odd sizes below and above every tile edge; an empty batch; wide and narrow tiles in earnest
SHAPES = [(1, 1, 1), (2, 32, 64), (3, 33, 65), (63, 64, 63), (64, 128, 64), (65, 130, 129), (200, 257, 100),
          (129, 8, 300), (16, 1000, 24), (7, 2049, 130), (1000, 520, 264)]
LARGE = [(32773, 24, 40), (4099, 40, 1000), (2500, 136, 2056), (65436, 264, 520), (65436, 265, 517)]


def _normal(generator, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=generator, device='cuda') * scale).to(dtype)


def _inputs(seed, n, inputs, outputs, dtype, *, lead=(), whole=False):
    generator = torch.Generator(device='cuda').manual_seed(seed)
    if whole:   # small whole numbers: every sum is exact, and relu's mask with it

        def values(*shape):
            return torch.randint(-2, 3, shape, generator=generator, device='cuda').to(dtype)
        return (values(n, inputs), values(*lead, outputs, inputs), values(*lead, outputs), values(n, outputs),
                values(n, outputs))
    return (_normal(generator, dtype, n, inputs), _normal(generator, dtype, *lead, outputs, inputs, scale=inputs ** -0.5),
            _normal(generator, dtype, *lead, outputs, scale=0.5), _normal(generator, dtype, n, outputs),
            _normal(generator, dtype, n, outputs))


def _run(x, w, b, r, dy, activation, offsets=None):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = linear(leaves[0], leaves[1], leaves[2], activation=activation, residual=leaves[3], offsets=offsets)
    wanted = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, wanted, dy))
    return [y.detach()] + [next(grads) if t is not None else None for t in leaves]


def _check_layer(got, x, w, b, r, dy, activation, what):
    layer = Layer64(x, w, b, r, dy, activation)
    y, dx, dw, db, dr = got
    check(y, layer.y, layer.y_error, what + ' y')
    check(dx, layer.dx, layer.dx_error, what + ' dx')
    check(dw, layer.dw, layer.dw_error, what + ' dw')
    if b is not None:
        check(db, layer.db, layer.db_error, what + ' db')
    if r is not None:
        assert torch.equal(dr, dy)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', SHAPES + LARGE, ids=str)
def test_layer_matches_formula(shape, dtype):
    n, inputs, outputs = shape
    activation = ACTIVATIONS[(n + inputs) % len(ACTIVATIONS)]
    print('linear', shape, dtype, activation, flush=True)
    x, w, b, r, dy = _inputs(n + outputs, n, inputs, outputs, dtype, whole=activation == 'relu')
    _check_layer(_run(x, w, b, r, dy, activation), x, w, b, r, dy, activation, str(shape))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('activation', ACTIVATIONS)
def test_every_activation_bias_and_residual(activation, dtype):
    for bias, residual in ((False, False), (True, False), (False, True), (True, True)):
        x, w, b, r, dy = _inputs(5, 70, 96, 50, dtype, whole=activation == 'relu')
        b, r = b if bias else None, r if residual else None
        print('linear', activation, dtype, bias, residual, flush=True)
        _check_layer(_run(x, w, b, r, dy, activation), x, w, b, r, dy, activation, activation)


@pytest.mark.parametrize('activation', ACTIVATIONS)
def test_activations_at_their_ends(activation):
    """Large and infinite sums: the limits of the function and its slope, and no NaN where they are finite."""
    z = torch.tensor([-1e30, -200.0, -90.0, -30.0, 0.0, 30.0, 90.0, 200.0, 1e30], device='cuda').view(-1, 1)
    one = torch.ones(1, 1, device='cuda')
    y, dx = _run(z, one, None, None, torch.ones_like(z), activation)[:2]
    layer = Layer64(z, one, None, None, torch.ones_like(z), activation)
    check(y, layer.y, layer.y.abs() * 2.0 ** -18 + 2.0 ** -120, activation)
    check(dx, layer.dx, torch.full_like(layer.dx, 2.0 ** -18), activation + ' slope')
    nan = linear(torch.full((1, 1), float('nan'), device='cuda'), one, activation=activation)
    assert nan.isnan().all()


def _offsets(counts):
    ends = torch.tensor(counts).cumsum(0).tolist()
    return torch.tensor([0] + ends, dtype=torch.int32, device='cuda')


GROUPS = [('one row each', [1] * 9, 0), ('empty ones', [0, 5, 0, 0, 64, 0], 0), ('tile edges', [64, 128, 63, 65, 1], 0),
          ('rows of no expert', [30, 0, 40], 77), ('all of no expert', [0, 0], 50), ('one of all', [0, 700, 0], 3),
          ('many', [(7 * e) % 5 for e in range(200)], 11), ('more experts than rows', [e % 97 == 0 for e in range(500)], 1),
          ('a long one', [300, 5000, 2, 0, 129], 0)]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('name,counts,rest', GROUPS, ids=[g[0] for g in GROUPS])
def test_experts_match_formula(name, counts, rest, dtype):
    counts = [int(c) for c in counts]
    n, inputs, outputs, experts = sum(counts) + rest, 40, 72, len(counts)
    print('experts', name, dtype, n, flush=True)
    x, w, b, r, dy = _inputs(len(name), n, inputs, outputs, dtype, lead=(experts,))
    # whatever lies in rows of no expert reaches nothing else
    held = sum(counts)
    x[held:] = float('nan')
    got = _run(x, w, b, r, dy, 'silu', offsets=_offsets(counts))
    at = 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        part = [got[0][rows], got[1][rows], got[2][e], got[3][e], got[4][rows]]
        _check_layer(part, x[rows], w[e], b[e], r[rows], dy[rows], 'silu', '%s, expert %d' % (name, e))
        at += count
    assert torch.equal(got[0][held:], r[held:]) and not got[1][held:].any()
    bare = linear(x, w, b, offsets=_offsets(counts))
    assert not bare[held:].any()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_experts_with_wide_layers(dtype):
    """The wide tiles, long groups that are cut into pieces, and a rounding of the cut to tile edges."""
    counts = [1500, 0, 3000, 257]
    n, inputs, outputs = sum(counts), 264, 1160
    print('experts wide', dtype, flush=True)
    x, w, b, r, dy = _inputs(3, n, inputs, outputs, dtype, lead=(len(counts),))
    got = _run(x, w, b, None, dy, 'gelu', offsets=_offsets(counts))
    at = 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        part = [got[0][rows], got[1][rows], got[2][e], got[3][e], None]
        _check_layer(part, x[rows], w[e], b[e], None, dy[rows], 'gelu', 'expert %d' % e)
        at += count


def test_a_row_that_is_not_finite_stays_alone():
    x, w, b, r, dy = _inputs(1, 200, 72, 88, torch.float16)
    clean = _run(x, w, b, r, dy, 'none')
    x[50], dy[70] = float('inf'), float('nan')
    got = _run(x, w, b, r, dy, 'none')
    others = torch.ones(200, dtype=torch.bool, device='cuda')
    others[[50, 70]] = False
    assert torch.equal(got[0][others], clean[0][others]) and torch.equal(got[1][others], clean[1][others])
    assert not got[0][50].isfinite().any() and got[1][70].isnan().all()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_strides_and_alignment(dtype):
    """Slices that start at odd elements, rows further apart than they are wide, transposed and expanded tensors:
    the same bits as contiguous ones."""
    n, inputs, outputs = 100, 48, 40
    x, w, b, r, dy = _inputs(2, n, inputs, outputs, dtype)
    expected = _run(x, w, b, r, dy, 'gelu')

    def inside(t):
        wide = torch.full((t.shape[0], t.shape[1] + 11), float('nan'), dtype=dtype, device='cuda')
        wide[:, 3:3 + t.shape[1]] = t
        return wide[:, 3:3 + t.shape[1]]
    for change in (inside, lambda t: t.t().contiguous().t()):
        got = _run(change(x), change(w), b, change(r), change(dy), 'gelu')
        assert all(torch.equal(a, c) for a, c in zip(got, expected))
    got = _run(x, w, b, r, torch.ones(1, 1, dtype=dtype, device='cuda').expand(n, outputs), 'gelu')
    same = _run(x, w, b, r, torch.ones(n, outputs, dtype=dtype, device='cuda'), 'gelu')
    assert all(torch.equal(a, c) for a, c in zip(got[:4], same[:4]))
    flat = torch.empty(n * inputs + 1, dtype=dtype, device='cuda')[1:].view(n, inputs).copy_(x)
    assert torch.equal(_run(flat, w, b, r, dy, 'gelu')[2], expected[2])


def test_no_rows():
    x, w, b, r, dy = _inputs(4, 0, 24, 16, torch.float32)
    y, dx, dw, db, dr = _run(x, w, b, r, dy, 'relu')
    assert y.shape == (0, 16) and dx.shape == (0, 24) and not dw.any() and not db.any()
    x, w, b, r, dy = _inputs(4, 0, 24, 16, torch.float16, lead=(3,))
    y, dx, dw, db, dr = _run(x, w, b, r, dy, 'relu', offsets=torch.zeros(4, dtype=torch.int32, device='cuda'))
    assert dw.shape == (3, 16, 24) and not dw.any() and not db.any()


@pytest.mark.parametrize('activation', ('sigmoid', 'softplus', 'gelu', 'silu'))
def test_gradient_against_differences(activation):
    """The derivative of sum(dy y) along random directions, by central differences of the fp32 forward."""
    n, inputs, outputs, h = 20, 24, 16, 2.0 ** -6
    third = {'sigmoid': 0.125, 'softplus': 0.1, 'gelu': 0.8, 'silu': 0.32}[activation]   # of the activation, at most
    x, w, b, r, dy = _inputs(8, n, inputs, outputs, torch.float32)
    _, dx, dw, db, dr = _run(x, w, b, r, dy, activation)
    layer = Layer64(x, w, b, r, dy, activation)
    generator = torch.Generator(device='cuda').manual_seed(9)
    for index, (value, gradient) in enumerate(zip((x, w, b, r), (dx, dw, db, dr))):
        direction = torch.randn(value.shape, generator=generator, device='cuda').sign()
        ends = []
        for sign in (1, -1):
            moved = [x, w, b, r]
            moved[index] = value + sign * h * direction
            ends.append((linear(moved[0], moved[1], moved[2], activation=activation, residual=moved[3]), moved[index]))
        # the step that the fp32 addition really made
        step = (ends[0][1].double() - ends[1][1].double())
        measured = ((ends[0][0].double() - ends[1][0].double()) * dy.double()).sum()
        expected = (gradient.double() * step).sum()
        # rounding of the two forwards, and the third derivative's share of a central difference
        moves = (step.abs() / 2)
        dz = {0: lambda: moves @ w.double().abs().t(), 1: lambda: x.double().abs() @ moves.t(),
              2: lambda: moves.expand(n, outputs), 3: lambda: torch.zeros(n, outputs, dtype=torch.float64, device='cuda')}[index]()
        allowed = (dy.double().abs() * (3 * layer.y_error + third * dz ** 3 / 3)).sum() + 1e-5 * (gradient.double() * step).abs().sum()
        assert (measured - expected).abs() <= allowed, (activation, index, float(measured), float(expected), float(allowed))
        assert allowed < 0.25 * (gradient.double() * step).abs().sum(), 'the bound says something'


def test_the_same_bits_every_time_and_on_any_stream():
    counts = [900, 0, 2000, 33]
    x, w, b, r, dy = _inputs(6, sum(counts), 200, 136, torch.bfloat16, lead=(4,))
    first = _run(x, w, b, r, dy, 'gelu', offsets=_offsets(counts))
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            again = _run(x, w, b, r, dy, 'gelu', offsets=_offsets(counts))
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_gradients_of_some_tensors_alone():
    x, w, b, r, dy = _inputs(7, 90, 40, 56, torch.float16)
    everything = _run(x, w, b, r, dy, 'silu')[1:]
    for index in range(4):
        leaves = [t.detach().requires_grad_(i == index) for i, t in enumerate((x, w, b, r))]
        y = linear(leaves[0], leaves[1], leaves[2], activation='silu', residual=leaves[3])
        assert torch.equal(torch.autograd.grad(y, leaves[index], dy)[0], everything[index])


def test_forward_in_a_graph():
    """Captured once, replayed over changed inputs with eager work between."""
    x, w, b, r, _ = _inputs(11, 300, 64, 96, torch.float16, lead=(3,))
    offsets = _offsets([100, 0, 150])
    with torch.no_grad():
        linear(x, w, b, activation='relu', residual=r, offsets=offsets)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = linear(x, w, b, activation='relu', residual=r, offsets=offsets)
        for replay in range(3):
            x.copy_(torch.randn_like(x))
            offsets.copy_(_offsets([100 - 40 * replay, 20 * replay, 150]))
            expected = linear(x, w, b, activation='relu', residual=r, offsets=offsets)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, expected), replay


def test_refusals():
    x, w, b, r, _ = _inputs(1, 8, 16, 24, torch.float16)
    offsets = _offsets([4, 4])
    stacked = torch.stack((w, w))
    for bad in (lambda: linear(x.cpu(), w), lambda: linear(x.double(), w.double()), lambda: linear(x, w.float()),
                lambda: linear(x, w[:, :8]), lambda: linear(x[0], w), lambda: linear(x, w, b[:3]),
                lambda: linear(x, w, b.float()), lambda: linear(x, w, residual=r[:, :3]),
                lambda: linear(x, w, residual=r[:3]), lambda: linear(x, w, activation='tanh'),
                lambda: linear(x, w, offsets=offsets), lambda: linear(x, stacked),
                lambda: linear(x, stacked, b, offsets=offsets), lambda: linear(x, stacked, offsets=offsets.long()),
                lambda: linear(x, stacked, offsets=offsets[:2]), lambda: linear(x, stacked, offsets=offsets.cpu()),
                lambda: linear(x[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            bad()

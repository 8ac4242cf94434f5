"""odie_amd.mixture and odie_amd.embedding against their definitions: places and moved rows exact, sums within
bounds derived in rows64."""
import numpy as np
import pytest
import torch

from odie_amd import _lib
from odie_amd.embedding import embed
from odie_amd.linear import linear
from odie_amd.mixture import ExpertMixture, combine, dispatch, expert_order
from rows64 import DTYPES, check, rounding, sum_error

pytestmark = pytest.mark.gpu


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _normal(generator, dtype, *shape):
    return torch.randn(*shape, generator=generator, device='cuda').to(dtype)


def _experts(seed, n, choices, experts, kind='even'):
    generator = _generator(seed)
    if kind == 'even':
        e = torch.randint(0, experts, (n, choices), generator=generator, device='cuda')
    elif kind == 'one':
        e = torch.full((n, choices), experts - 1, device='cuda')
    elif kind == 'lost':
        e = torch.randint(-2, experts + 2, (n, choices), generator=generator, device='cuda')
    else:
        e = torch.full((n, choices), -1, device='cuda')
    return e


def _expected_order(expert, experts):
    flat = expert.cpu().numpy().reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < experts), flat, experts)
    source = np.argsort(key, kind='stable')
    slots = np.empty(flat.size, dtype=np.int64)
    slots[source] = np.arange(flat.size)
    slots[key == experts] = -1
    offsets = np.searchsorted(key[source], np.arange(experts + 1))
    return slots.reshape(expert.shape), source, offsets


# one entry; below, at and past the sizes where the sort changes its way (4096 keys; 2047 and more buckets)
ORDERS = [(1, 1, 1), (1, 2, 64), (3, 4, 5), (63, 1, 300), (1000, 4, 16), (4096, 1, 64), (4097, 1, 64), (2049, 2, 2047),
          (30011, 3, 2048), (50000, 2, 4096), (70000, 1, 1), (9000, 1, 3000000), (5, 1, 5000000)]


@pytest.mark.parametrize('kind', ('even', 'one', 'lost', 'none'))
@pytest.mark.parametrize('n,choices,experts', ORDERS)
def test_order(n, choices, experts, kind):
    expert = _experts(n, n, choices, experts, kind)
    slots, source, offsets = _expected_order(expert, experts)
    for dtype in (torch.int32, torch.int64):
        print('order', n, choices, experts, kind, dtype, flush=True)
        order = expert_order(expert.to(dtype), experts)
        assert np.array_equal(order.slots.cpu().numpy(), slots)
        assert np.array_equal(order.source.cpu().numpy(), source)
        assert np.array_equal(order.offsets.cpu().numpy(), offsets)


def test_order_of_long_keys_that_wrap():
    """int64 values whose low 32 bits name an expert are none."""
    expert = torch.tensor([[1], [(1 << 32) + 1], [-(1 << 32) + 2], [2]], device='cuda')
    order = expert_order(expert, 4)
    assert order.slots.flatten().tolist() == [0, -1, -1, 1] and order.offsets.tolist() == [0, 0, 1, 2, 2]


def test_order_of_nothing():
    order = expert_order(torch.empty(0, 2, dtype=torch.int32, device='cuda'), 7)
    assert order.offsets.tolist() == [0] * 8 and order.slots.shape == (0, 2)
    x = torch.empty(0, 5, device='cuda', requires_grad=True)
    y = combine(dispatch(x, order), order, torch.empty(0, 2, device='cuda'))
    assert y.shape == (0, 5) and torch.autograd.grad(y.sum(), x)[0].shape == (0, 5)


WIDTHS = (1, 7, 8, 32, 131, 256, 1000)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', WIDTHS)
@pytest.mark.parametrize('n,choices,experts,kind', [(1, 1, 3, 'even'), (1, 2, 64, 'lost'), (50, 3, 7, 'lost'),
                                                    (700, 4, 40, 'even'), (333, 2, 9, 'none'), (2100, 2, 5, 'lost')])
def test_exchange(n, choices, experts, kind, width, dtype):
    print('exchange', n, choices, experts, kind, width, dtype, flush=True)
    generator = _generator(n + width)
    expert = _experts(n, n, choices, experts, kind)
    order = expert_order(expert, experts)
    slots, source, offsets = (torch.from_numpy(a).cuda() for a in _expected_order(expert, experts))
    held = int(offsets[-1])
    x = _normal(generator, dtype, n, width).requires_grad_(True)
    sent = dispatch(x, order)
    assert torch.equal(sent[:held], x.detach()[source[:held] // choices]) and not sent[held:].any()

    rows = _normal(generator, dtype, n * choices, width)
    rows[held:] = float('nan')               # rows of no expert reach nothing
    rows.requires_grad_(True)
    weights = torch.randn(n, choices, generator=generator, device='cuda').requires_grad_(True)
    y = combine(rows, order, weights)
    valid = slots >= 0
    taken = torch.where(valid[..., None], rows.detach().double()[slots.clamp(min=0)], 0.0)
    taken = taken.nan_to_num(0.0)
    w = weights.detach().double()
    products = taken * w[..., None]
    check(y, products.sum(1), sum_error(choices, products.abs().sum(1)) + rounding(dtype, products.sum(1)), 'y')

    up = _normal(generator, dtype, n, width)
    drows, dweights = torch.autograd.grad(y, (rows, weights), up)
    expected = up.double()[source[:held] // choices] * w.flatten()[source[:held]][:, None]
    check(drows[:held], expected, rounding(dtype, expected) + 2.0 ** -23 * expected.abs(), 'drows')
    assert not drows[held:].any()
    dots = taken * up.double()[:, None]
    check(dweights, dots.sum(2), sum_error(width, dots.abs().sum(2)), 'dweights')

    sent_up = _normal(generator, dtype, n * choices, width)
    sent_up[held:] = float('nan')
    dx, = torch.autograd.grad(sent, x, sent_up)
    back = torch.where(valid[..., None], sent_up.double()[slots.clamp(min=0)], 0.0).nan_to_num(0.0)
    check(dx, back.sum(1), sum_error(choices, back.abs().sum(1)) + rounding(dtype, back.sum(1)), 'dx')


def test_exchange_without_weights_in_other_types_and_strides():
    generator = _generator(1)
    expert = _experts(1, 90, 2, 6, 'lost')
    order = expert_order(expert.t().contiguous().t(), 6)       # the order of entries, whatever their strides
    plain = expert_order(expert.int(), 6)
    assert torch.equal(order.slots, plain.slots)
    rows = _normal(generator, torch.float16, 180, 40)
    ones = torch.ones(90, 2, device='cuda')
    assert torch.equal(combine(rows, order), combine(rows, order, ones))
    half = torch.rand(90, 2, generator=generator, device='cuda').half().requires_grad_(True)
    y = combine(rows, order, half)
    assert torch.equal(y, combine(rows, order, half.detach().float()))
    assert torch.autograd.grad(y, half, torch.ones_like(y))[0].dtype == torch.float16
    wide = torch.full((180, 57), float('nan'), dtype=torch.float16, device='cuda')
    wide[:, 9:49] = rows
    assert torch.equal(combine(wide[:, 9:49], order, ones), combine(rows, order, ones))
    x = _normal(generator, torch.float16, 90, 40)
    wide[:90, 9:49] = x
    assert torch.equal(dispatch(wide[:90, 9:49], order), dispatch(x, order))
    x.requires_grad_(True)                                       # an expanded upstream
    dx, = torch.autograd.grad(dispatch(x, order).sum(), x)
    counts = (order.slots >= 0).sum(1, keepdim=True).half().expand(90, 40)
    assert torch.equal(dx, counts)
    bare = expert_order(expert[:, 0], 6)                         # one choice, a vector
    assert bare.slots.shape == (90, 1)


# --- lookups -----------------------------------------------------------------------------------------

LOOKUPS = [(1, 1, 1), (64, 1024, 32), (1000, 3, 33), (5000, 5000, 8), (70001, 300, 17), (40000, 100000, 24),
           (20000, 2, 260), (3000, 70, 1030)]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('kind', ('even', 'one', 'lost', 'none'))
@pytest.mark.parametrize('n,vocab,width', LOOKUPS)
def test_lookup_and_gradient(n, vocab, width, kind, dtype):
    print('lookup', n, vocab, width, kind, dtype, flush=True)
    generator = _generator(n + width)
    ids = _experts(n, n, 1, vocab, kind)[:, 0]
    table = _normal(generator, dtype, vocab, width).requires_grad_(True)
    up = _normal(generator, dtype, n, width)
    scale = 1.7
    scale32 = float(np.float32(scale))
    valid = (ids >= 0) & (ids < vocab)
    up[~valid] = float('nan')
    y = embed(table, ids, scale)
    expected = torch.where(valid[:, None], table.detach().double()[ids.clamp(0, vocab - 1)], 0.0) * scale32
    check(y, expected, rounding(dtype, expected) + 2.0 ** -24 * expected.abs(), 'y')
    assert torch.equal(embed(table.detach(), ids.int(), scale), y.detach())
    dtable, = torch.autograd.grad(y, table, up)
    rows = ids[valid]
    total = torch.zeros(vocab, width, dtype=torch.float64, device='cuda').index_add_(0, rows, up[valid].double())
    size = torch.zeros(vocab, width, dtype=torch.float64, device='cuda').index_add_(0, rows, up[valid].double().abs())
    count = torch.bincount(rows, minlength=vocab).double()[:, None]
    total, size = total * scale32, size * scale32
    check(dtable, total, 1.1 * (count + 3) * 2.0 ** -24 * size + rounding(dtype, total), 'dtable')
    again, = torch.autograd.grad(embed(table, ids, scale), table, up)
    assert torch.equal(again, dtable)


def test_lookup_shapes_and_strides():
    generator = _generator(3)
    table = _normal(generator, torch.float32, 20, 6).requires_grad_(True)
    ids = torch.randint(0, 20, (3, 4, 5), generator=generator, device='cuda')
    y = embed(table, ids)
    assert torch.equal(y, table.detach()[ids]) and y.shape == (3, 4, 5, 6)
    dtable, = torch.autograd.grad(y.sum(), table)              # an expanded upstream
    assert torch.equal(dtable, torch.bincount(ids.flatten(), minlength=20).float()[:, None].expand(20, 6))
    wide = torch.zeros(20, 9, device='cuda')
    wide[:, 1:7] = table.detach()
    assert torch.equal(embed(wide[:, 1:7], ids.transpose(0, 2)), table.detach()[ids.transpose(0, 2)])
    empty = embed(table, ids[:0])
    assert empty.shape == (0, 4, 5, 6) and not torch.autograd.grad(empty.sum(), table)[0].any()


def test_lookup_gradient_against_differences():
    """The lookup is linear in the table: a difference of any step is its derivative, up to the roundings."""
    generator = _generator(4)
    table = _normal(generator, torch.float32, 11, 5).requires_grad_(True)
    ids = torch.randint(0, 11, (40,), generator=generator, device='cuda')
    up = _normal(generator, torch.float32, 40, 5)
    dtable, = torch.autograd.grad(embed(table, ids, 0.5), table, up)
    step = _normal(generator, torch.float32, 11, 5)
    with torch.no_grad():
        moved = embed(table + step, ids, 0.5).double() - embed(table, ids, 0.5).double()
    measured, expected = (moved * up.double()).sum(), (dtable.double() * step.double()).sum()
    size = ((table.abs() + step.abs()).double()[ids] * up.double().abs()).sum()
    assert (measured - expected).abs() <= 50 * 2.0 ** -24 * size


def test_exchange_gradient_against_differences():
    """Combine is linear in its rows and in its weights, dispatch in its rows."""
    generator = _generator(5)
    order = expert_order(_experts(2, 60, 3, 8, 'lost'), 8)
    values = [_normal(generator, torch.float32, 60, 12), _normal(generator, torch.float32, 180, 12),
              torch.rand(60, 3, generator=generator, device='cuda')]
    held = int(order.offsets[-1])
    calls = [(0, lambda v: dispatch(v[0], order)), (1, lambda v: combine(v[1], order, v[2])),
             (2, lambda v: combine(v[1], order, v[2]))]
    for index, call in calls:
        leaves = [v.clone().requires_grad_(i == index) for i, v in enumerate(values)]
        y = call(leaves)
        up = _normal(generator, torch.float32, *y.shape)
        gradient, = torch.autograd.grad(y, leaves[index], up)
        step = _normal(generator, torch.float32, *values[index].shape)
        moved = [v + step if i == index else v for i, v in enumerate(values)]
        difference = ((call(moved).double() - call(values).double()) * up.double()).sum()
        expected = (gradient.double() * step.double()).sum()
        size = (up.double().abs() * (call([v.abs() for v in moved]) + call([v.abs() for v in values])).double()).sum()
        assert (difference - expected).abs() <= 30 * 2.0 ** -24 * size + 30 * 2.0 ** -24 * (gradient * step).abs().sum()
    assert held < 180


# --- together ----------------------------------------------------------------------------------------

def _mixture64(model, x, expert, weights, ids):
    p = {name: value.detach().double().requires_grad_(True) for name, value in model.named_parameters()}
    x = torch.cat((x.double(), p['table'][ids] * float(np.float32(model.scale))), 1)
    y = 0.0
    for j in range(expert.shape[1]):
        e = expert[:, j].clamp(0, model.experts - 1).long()
        valid = ((expert[:, j] >= 0) & (expert[:, j] < model.experts)).double()[:, None]
        h = torch.nn.functional.silu((p['weight1'][e] @ x[..., None])[..., 0] + p['bias1'][e])
        y = y + valid * weights[:, j:j + 1].double() * ((p['weight2'][e] @ h[..., None])[..., 0] + p['bias2'][e])
    return y, p


def test_mixture_together():
    """Codes, sort, both layers and the return with every gradient, in fp32 against 64 bits: sums of at most 61 terms
    through three products, within 2**-14 of the largest entry."""
    model = ExpertMixture(6, 24, 40, 3, activation='silu', codes=8, vocab=30, dtype=torch.float32)
    generator = _generator(6)
    x = _normal(generator, torch.float32, 500, 24)
    expert = _experts(3, 500, 2, 6, 'lost')
    weights = torch.rand(500, 2, generator=generator, device='cuda')
    ids = torch.randint(0, 30, (500,), generator=generator, device='cuda')
    y = model(x, expert, weights, ids)
    up = _normal(generator, torch.float32, 500, 3)
    names = [name for name, _ in model.named_parameters()]
    grads = dict(zip(names, torch.autograd.grad(y, list(model.parameters()), up)))
    y64, p = _mixture64(model, x, expert, weights, ids)
    largest = float(y64.detach().abs().max())
    grads64 = dict(zip(names, torch.autograd.grad(y64, [p[name] for name in names], up.double())))
    check(y, y64.detach(), torch.full_like(y64, 2.0 ** -14 * largest), 'y')
    for name in names:
        check(grads[name], grads64[name], torch.full_like(grads64[name], 2.0 ** -14 * float(grads64[name].abs().max())), name)


def test_mixture_in_a_graph():
    model = ExpertMixture(5, 16, 32, 3, activation='gelu')
    generator = _generator(7)
    x = _normal(generator, torch.float16, 64, 16)
    expert = _experts(4, 64, 2, 5, 'lost').int()
    weights = torch.rand(64, 2, generator=generator, device='cuda')
    with torch.no_grad():
        model(x, expert, weights)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model(x, expert, weights)
        for replay in range(3):
            x.copy_(torch.randn_like(x))
            expert.copy_(_experts(20 + replay, 64, 2, 5, 'lost'))
            expected = model(x, expert, weights)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, expected), replay


def test_on_another_stream():
    generator = _generator(8)
    x = _normal(generator, torch.float16, 3000, 48)
    expert = _experts(5, 3000, 2, 40, 'lost')
    order = expert_order(expert, 40)
    expected = combine(dispatch(x, order), order)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = expert_order(expert, 40)
        got = combine(dispatch(x, there), there)
    torch.cuda.synchronize()
    assert torch.equal(got, expected)


def test_refusals():
    x = torch.zeros(6, 4, device='cuda')
    order = expert_order(torch.zeros(6, 2, dtype=torch.int32, device='cuda'), 3)
    rows = torch.zeros(12, 4, device='cuda')
    table = torch.zeros(5, 4, device='cuda')
    ids = torch.zeros(3, dtype=torch.int64, device='cuda')
    for bad in (lambda: expert_order(torch.zeros(6, device='cuda'), 3), lambda: expert_order(ids.cpu(), 3),
                lambda: expert_order(ids, 0), lambda: expert_order(ids.view(3, 1, 1), 3),
                lambda: expert_order(torch.empty(3, 0, dtype=torch.int32, device='cuda'), 3),
                lambda: dispatch(x[:5], order), lambda: dispatch(x.cpu(), order), lambda: dispatch(x.double(), order),
                lambda: dispatch(x[:, :0], order), lambda: combine(rows[:7], order), lambda: combine(rows.int(), order),
                lambda: combine(rows, order, torch.ones(6, device='cuda')),
                lambda: combine(rows, order, torch.ones(6, 2, dtype=torch.int32, device='cuda')),
                lambda: combine(rows, order, torch.ones(6, 2)), lambda: embed(table, ids.float()),
                lambda: embed(table, ids.cpu()), lambda: embed(table.cpu(), ids), lambda: embed(table.double(), ids),
                lambda: embed(table[:0], ids), lambda: embed(table[0], ids),
                lambda: ExpertMixture(2, 4, 4, 3, activation='tanh'), lambda: ExpertMixture(2, 4, 4, 3, codes=2),
                lambda: ExpertMixture(2, 4, 4, 3)(x.half(), ids, ids=ids)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.NativeError):       # more buckets than 31 bits hold
        expert_order(ids, 1 << 31)

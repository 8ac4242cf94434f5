"""odie_amd.router against its formulas in 64 bits and against differences.

Bounds: a softmax's exponential of a difference d is off by at most 2^-22 (1 + |d|) relative (the difference's and the
argument's rounding, and the function's), an fp32 sum as rows64.sum_error has it; below 2^-120 a result may be 0."""
import math

import pytest
import torch

from odie_amd.router import balance, choose, distill
from rows64 import DTYPES, check, rounding

pytestmark = pytest.mark.gpu

FAINT = 2.0 ** -120
# one value, ends of 16-byte chunks, of a lane group's, of a wave's registers, and rows longer than those
WIDTHS = (1, 2, 3, 7, 8, 9, 31, 64, 65, 127, 128, 200, 513, 1000, 1024, 2049, 4096, 4097, 10007)


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _logits(generator, dtype, n, width, scale=2.0, blocked=0.0):
    value = (torch.randn(n, width, generator=generator, device='cuda') * scale).to(dtype)
    if blocked:
        value[torch.rand(n, width, generator=generator, device='cuda') < blocked] = -math.inf
    return value


def _softmax64(logits):
    """p (0 in rows of nothing), and what a computed p may be off by, relative: [N, 1] for the sum, [N, E] each."""
    x = logits.detach().double()
    top = x.amax(1, keepdim=True)
    d = torch.where(x > -math.inf, x - torch.where(top > -math.inf, top, 0.0), 0.0)
    power = torch.where(x > -math.inf, torch.exp(d), 0.0)
    total = power.sum(1, keepdim=True).clamp(min=1e-300)
    p = power / total
    each = 2.0 ** -22 * (1 + d.abs())
    sums = (p * each).sum(1, keepdim=True) + 1.1 * (x.shape[1] + 4) * 2.0 ** -24
    return p, each + sums, sums


def _chosen64(logits, choices):
    order = torch.sort(torch.where(logits.isnan(), math.inf, logits.double()), dim=1, descending=True, stable=True)
    value, at = order.values[:, :choices], order.indices[:, :choices]
    return torch.where(value > -math.inf, at, -1)


def _choose64(logits, choices, normalize, upstream):
    n, experts = logits.shape
    chosen = _chosen64(logits, choices)
    held, at = chosen >= 0, chosen.clamp(min=0)
    taken = torch.zeros(logits.shape, device=logits.device).scatter_add(1, at, held.float()) > 0
    base = torch.where(taken, logits, -math.inf) if normalize else logits
    p, off, _ = _softmax64(base)
    w = torch.where(held, p.gather(1, at), 0.0)
    w_off = w * off.gather(1, at) + FAINT
    g = upstream.double()
    t, size = (w * g).sum(1, keepdim=True), (w * g.abs()).sum(1, keepdim=True)
    t_off = (w_off * g.abs()).sum(1, keepdim=True) + 1.1 * (choices + 3) * 2.0 ** -24 * size
    d = -p * t
    d_off = p * t_off + p * off * size
    d = d.scatter_add(1, at, torch.where(held, w * g, 0.0))
    d_off = d_off.scatter_add(1, at, torch.where(held, w_off * g.abs() + 2.0 ** -22 * w * (g.abs() + size), 0.0))
    d_off = d_off + 2.0 ** -22 * (d.abs() + p * size) + 2 * FAINT
    return chosen, w, w_off, d, d_off * 1.01 + rounding(logits.dtype, d)


def _check_choose(logits, choices, normalize, seed, what):
    upstream = torch.randn(logits.shape[0], choices, generator=_generator(seed + 1), device='cuda')
    leaf = logits.detach().clone().requires_grad_(True)
    expert, weights = choose(leaf, choices, normalize=normalize)
    gradient, = torch.autograd.grad(weights, leaf, upstream)
    chosen, w, w_off, d, d_off = _choose64(logits, choices, normalize, upstream)
    assert expert.dtype == torch.int32 and weights.dtype == torch.float32 and gradient.dtype == logits.dtype
    assert torch.equal(expert.long(), chosen), what
    check(weights, w, w_off, what + ' weights')
    check(gradient, d, d_off, what + ' gradient')
    again = choose(logits.detach(), choices, normalize=normalize)
    assert torch.equal(again[0], expert) and torch.equal(again[1], weights), what


@pytest.mark.parametrize('normalize', (True, False))
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', WIDTHS)
def test_choose(width, dtype, normalize):
    for n, choices, blocked in ((1, 1, 0.0), (5, min(2, width), 0.3), (67, min(8, width), 0.0), (33, min(64, width), 0.5)):
        print('choose', n, width, choices, dtype, normalize, blocked, flush=True)
        logits = _logits(_generator(width + n), dtype, n, width, blocked=blocked)
        _check_choose(logits, choices, normalize, width, '%dx%d, %d of them' % (n, width, choices))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', (2051, 4099, 8192, 8193, 16384, 16391, 32768))
def test_choose_of_long_rows(width, dtype):
    """Rows of several waves, by the number of rows and choices; all choices of some lie in one lane's part."""
    for n, choices, normalize in ((1, 4, False), (1030, 1, True), (1030, 4, False), (1030, 5, True), (3, 64, False)):
        print('choose', n, width, choices, dtype, normalize, flush=True)
        logits = _logits(_generator(width + n), dtype, n, width, blocked=0.1)
        logits[n // 2, :16] = logits[n // 2].abs().amax().clamp(max=100) + torch.arange(16, device='cuda').to(dtype)
        logits[n // 3, -1] = 300.0
        _check_choose(logits, choices, normalize, width, '%dx%d, %d of them' % (n, width, choices))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', (15, 62, 131, 515, 2051))
def test_choose_of_many_rows_that_end_inside_16_bytes(width, dtype):
    for choices, normalize in ((2, False), (8, False), (8, True)):
        _check_choose(_logits(_generator(width), dtype, 20000, width), choices, normalize, width, '20000x%d' % width)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', (8, 64, 1000, 2100, 5000, 12000, 20000))
def test_choose_ties_and_masks(width, dtype):
    """Equal logits go by index, -0 and 0 are equal, and rows may have fewer allowed experts than choices, or none."""
    logits = torch.zeros(6, width, device='cuda', dtype=dtype)
    logits[1, ::2] = -0.0
    logits[2] = -math.inf
    logits[3] = -math.inf
    logits[3, width - 2] = 1.0
    logits[4] = torch.arange(width, device='cuda').flip(0) // 3
    logits[5, :-1] = -torch.finfo(dtype).max        # the lowest value is not a mask
    logits[5, -1] = -math.inf
    for normalize in (True, False):
        _check_choose(logits, 4, normalize, width, 'ties')
    expert, weights = choose(logits, 4)
    assert expert[0].tolist() == [0, 1, 2, 3] and expert[1].tolist() == [0, 1, 2, 3]
    assert expert[2].tolist() == [-1] * 4 and not weights[2].any()
    assert expert[3].tolist() == [width - 2, -1, -1, -1] and weights[3].tolist() == [1, 0, 0, 0]
    assert expert[5].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', (16, 300, 2100, 5000, 12000, 20000))
def test_choose_infinities_and_nan(width, dtype):
    """A NaN or +inf is the largest and makes its own row's weights NaN, and no other row's."""
    logits = _logits(_generator(3), dtype, 4, width)
    logits[1, 5], logits[2, 7], logits[2, 3] = math.nan, math.inf, -math.nan
    for normalize in (True, False):
        expert, weights = choose(logits, 3, normalize=normalize)
        assert torch.equal(expert[0::3].long(), _chosen64(logits[0::3], 3))
        assert expert[1, 0] == 5 and expert[2, :2].tolist() == [3, 7]
        assert weights[1:3].isnan().all() and not weights[0::3].isnan().any()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_rows_of_any_stride_and_start(dtype):
    """Rows inside wider ones, at odd elements; every second row; transposed; one row whose stride means nothing."""
    generator = _generator(4)
    wide = _logits(generator, dtype, 30, 150)
    for logits in (wide[:, 3:104], wide[::2, 1:66], wide.t(), wide[5:6, 7:90], wide[:, :1], wide[3:3]):
        expert, weights = choose(logits, 1)
        same = choose(logits.contiguous(), 1)
        assert torch.equal(expert, same[0]) and torch.equal(weights, same[1])
        chosen = expert
        for a, b in zip(balance(logits, chosen), balance(logits.contiguous(), chosen)):
            assert torch.equal(a, b)
        ids = torch.zeros(logits.shape[0], 1, dtype=torch.int64, device='cuda')
        teacher = torch.zeros(logits.shape[0], 1, device='cuda')
        assert torch.equal(distill(logits, ids, teacher), distill(logits.contiguous(), ids, teacher))
        leaf = logits.detach().requires_grad_(True)
        copy = logits.detach().clone().contiguous().requires_grad_(True)
        for call in (lambda x: choose(x, 1, normalize=False)[1].sum(), lambda x: balance(x, chosen)[0],
                     lambda x: distill(x, ids, teacher).sum()):
            got, = torch.autograd.grad(call(leaf), leaf)
            expected, = torch.autograd.grad(call(copy), copy)
            assert torch.equal(got, expected)


def _balance64(logits, expert, upstream):
    n, experts = logits.shape
    e = expert.long()
    valid = (e >= 0) & (e < experts)
    counts = torch.bincount(e[valid], minlength=experts).double()
    part = valid.any(1, keepdim=True)
    entries, rows = valid.sum().item(), part.sum().item()
    norm = experts / (entries * rows) if entries else 0.0
    p, off, _ = _softmax64(torch.where(part, logits, 0.0))
    p = torch.where(part, p, 0.0)
    t = (p * counts).sum(1, keepdim=True)
    t_off = (p * counts * (off + 2.0 ** -23)).sum(1, keepdim=True) + 1.1 * (2 * experts + 6) * 2.0 ** -24 * t
    loss, loss_off = norm * t.sum(), norm * t_off.sum() + 2.0 ** -22 * norm * t.sum()
    scale = upstream * norm
    d = scale * p * (counts - t)
    d_off = abs(scale) * (p * (off + 2.0 ** -21) * (counts - t).abs() + p * (t_off + 2.0 ** -23 * (counts + t))) + FAINT
    return loss, loss_off, counts, d, d_off * 1.01 + rounding(logits.dtype, d)


def _check_balance(logits, expert, what):
    leaf = logits.detach().clone().requires_grad_(True)
    loss, counts = balance(leaf, expert)
    scale = float(logits.shape[0])
    gradient, = torch.autograd.grad(loss, leaf, torch.tensor(scale, device='cuda'))
    expected, off, entries, d, d_off = _balance64(logits, expert, scale)
    assert loss.shape == () and loss.dtype == torch.float32 and counts.dtype == torch.int32
    assert torch.equal(counts.double(), entries), what
    check(loss, torch.as_tensor(expected, device='cuda', dtype=torch.float64), torch.as_tensor(off, device='cuda'), what)
    check(gradient, d, d_off, what + ' gradient')
    again = balance(logits.detach(), expert)
    assert torch.equal(again[0], loss) and torch.equal(again[1], counts), what


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', WIDTHS)
def test_balance(width, dtype):
    for n, choices in ((1, 1), (6, 3), (130, 2), (4099, 1), (9001, 3)):
        if n * width > 5_000_000:
            continue
        print('balance', n, width, choices, dtype, flush=True)
        generator = _generator(width + n)
        logits = _logits(generator, dtype, n, width)
        expert = torch.randint(-2, width + 2, (n, choices), generator=generator, device='cuda', dtype=torch.int32)
        _check_balance(logits, expert, '%dx%d' % (n, width))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_balance_of_padding_and_masks(dtype):
    """Rows of no entry take no part whatever they hold; a row that is masked whole has shares of 0; no rows, no entries."""
    logits = _logits(_generator(5), dtype, 9, 40, blocked=0.2)
    expert = torch.randint(0, 40, (9, 2), generator=_generator(6), device='cuda', dtype=torch.int32)
    expert[2:4] = -1
    expert[7] = torch.tensor([40, -5])
    _check_balance(logits, expert, 'padding')
    clean = balance(logits, expert)
    logits[2], logits[3, 1], logits[7] = math.nan, math.inf, -math.inf
    dirty = logits.clone().requires_grad_(True)
    loss, counts = balance(dirty, expert)
    assert torch.equal(loss, clean[0]) and torch.equal(counts, clean[1])
    gradient, = torch.autograd.grad(loss, dirty)
    assert not gradient[2:4].any() and not gradient[7].any() and not gradient.isnan().any()
    logits = logits[:2].clone()
    logits[1] = -math.inf
    _check_balance(logits, expert[:2], 'a masked row')
    for rows, chosen in ((logits[:0], expert[:0]), (logits, torch.full_like(expert[:2], -1))):
        leaf = rows.clone().requires_grad_(True)
        loss, counts = balance(leaf, chosen)
        assert loss == 0 and not counts.any()
        assert not torch.autograd.grad(loss, leaf)[0].any()


@pytest.mark.parametrize('dtype', (torch.float16, torch.float32), ids=str)
@pytest.mark.parametrize('n, width, choices', ((300, 40, 100), (5, 10, 1000), (400, 10000, 64), (130, 32768, 130), (700, 5000, 30), (1030, 8200, 2),
                                                 (50, 16384, 3), (40, 16392, 3)))
def test_balance_of_many_entries_a_row(n, width, choices, dtype):
    """More entries than lanes of a row; counts of many experts, from many entries; long rows with padding."""
    generator = _generator(n)
    logits = _logits(generator, dtype, n, width)
    expert = torch.randint(-width // 4, width, (n, choices), generator=generator, device='cuda', dtype=torch.int32)
    expert[1::3] = -1
    expert[0, :-1] = -1
    expert[0, -1] = width - 1       # the only entry of its row is the last
    _check_balance(logits, expert, '%dx%d, %d entries' % (n, width, choices))


def test_entries_of_any_layout():
    """Entries that do not lie on 16 bytes, or not together; a teacher of another type, in columns of a wider one."""
    generator = _generator(21)
    logits = _logits(generator, torch.float32, 9000, 50)
    wide = torch.randint(-1, 50, (9002, 6), generator=generator, device='cuda', dtype=torch.int32)
    for expert in (wide.flatten()[1:1 + 9000 * 3].view(9000, 3), wide[2:, 1:5], wide[1:9001, ::2], wide[:9000, :1].expand(9000, 4)):
        _check_balance(logits, expert, 'entries')
        teacher = _logits(generator, torch.bfloat16, expert.shape[1], 9000).t()
        ids, copy = expert.long(), (expert.long().contiguous(), teacher.contiguous())
        ids = ids.t().contiguous().t()
        leaf = logits.clone().requires_grad_(True)
        got = distill(leaf, ids, teacher)
        expected = distill(logits, *copy)
        assert torch.equal(got, expected) and torch.equal(distill(logits, expert, teacher), expected)
        twin = logits.clone().requires_grad_(True)
        assert torch.equal(torch.autograd.grad(got.sum(), leaf)[0], torch.autograd.grad(distill(twin, *copy).sum(), twin)[0])


def test_no_rows():
    for width in (1, 40, 9000):
        x = torch.zeros(0, width, device='cuda', dtype=torch.bfloat16, requires_grad=True)
        ids, teacher = torch.zeros(0, 2, device='cuda', dtype=torch.int64), torch.zeros(0, 2, device='cuda')
        for normalize in (True, False):
            expert, weights = choose(x, 1, normalize=normalize)
            assert expert.shape == weights.shape == (0, 1)
            assert torch.autograd.grad(weights.sum(), x)[0].shape == (0, width)
        loss = distill(x, ids, teacher)
        assert loss.shape == (0,) and torch.autograd.grad(loss.sum(), x)[0].shape == (0, width)
        loss, counts = balance(x, expert)
        assert loss == 0 and counts.shape == (width,) and not counts.any()


def test_inference_mode():
    x = torch.randn(5, 12, device='cuda')
    ids = torch.zeros(5, 1, device='cuda', dtype=torch.int64)
    expected = [*choose(x, 3), *balance(x, choose(x, 3)[0]), distill(x, ids, x[:, :1])]
    with torch.inference_mode():
        got = [*choose(x, 3), *balance(x, choose(x, 3)[0]), distill(x, ids, x[:, :1])]
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_even_load_has_a_loss_of_one():
    logits = torch.zeros(64, 16, device='cuda')
    expert = torch.arange(64, device='cuda', dtype=torch.int32).view(64, 1) % 16
    assert abs(float(balance(logits, expert)[0]) - 1) < 2.0 ** -20


def _distill64(logits, ids, teacher, temperature, upstream):
    n, classes = logits.shape
    valid = (ids >= 0) & (ids < classes) & (teacher > -math.inf)
    at = torch.where(valid, ids, 0).long()
    inverse = float(1.0 / torch.tensor(temperature))      # as fp32 holds it
    # scaling rounds a logit by 2^-24 of itself, which moves its exponential by as much
    moved = 2.0 ** -22 * torch.where(logits > -math.inf, logits.double().abs(), 0.0) * inverse
    q, q_off, q_sum = _softmax64(torch.where(valid, teacher.double() * inverse, -math.inf))
    q_moved = 2.0 ** -22 * torch.where(valid, teacher.double().abs(), 0.0) * inverse
    q_off = q_off + q_moved + (q * q_moved).sum(1, keepdim=True)
    p, off, p_sum = _softmax64(logits.double() * inverse)
    off = off + moved + (p * moved).sum(1, keepdim=True)
    x = logits.double() * inverse
    lse = torch.logsumexp(x, 1, keepdim=True)
    y = torch.where(valid, teacher.double() * inverse, -math.inf)
    log_q = y - torch.logsumexp(y, 1, keepdim=True)
    log_p = x.gather(1, at) - lse
    term = torch.where(valid, log_q - log_p, 0.0)
    loss = torch.where(q > 0, q * term, 0.0).sum(1)
    # each logarithm's parts are off by their rounding and their sums' relative error
    parts = torch.where(valid, y.abs() + x.gather(1, at).abs(), 0.0) + x.amax(1, keepdim=True).abs() + y.amax(1, keepdim=True).nan_to_num(neginf=0).abs()
    term_off = 2.0 ** -21 * (parts + lse.abs() + 20) + off.gather(1, at) + q_off
    loss_off = torch.where(q > 0, q * term_off + q * (q_off + 2.0 ** -20) * term.abs(), 0.0).sum(1) + FAINT
    g = (upstream.double() * inverse)[:, None] * valid.any(1, keepdim=True)
    share = torch.zeros_like(p).scatter_add(1, at, torch.where(valid, q, 0.0))
    share_off = torch.zeros_like(p).scatter_add(1, at, torch.where(valid, q * (q_off + 2.0 ** -20), 0.0))
    d = g * (p - share)
    d_off = g.abs() * (p * (off + 2.0 ** -21) + share_off) + 2.0 ** -22 * d.abs() + FAINT
    return loss, loss_off, d, d_off * 1.01 + rounding(logits.dtype, d)


def _check_distill(logits, ids, teacher, temperature, what):
    upstream = torch.randn(logits.shape[0], generator=_generator(9), device='cuda')
    leaf = logits.detach().clone().requires_grad_(True)
    loss = distill(leaf, ids, teacher, temperature=temperature)
    gradient, = torch.autograd.grad(loss, leaf, upstream)
    expected, off, d, d_off = _distill64(logits, ids, teacher, temperature, upstream)
    check(loss, expected, off, what)
    check(gradient, d, d_off, what + ' gradient')
    assert torch.equal(distill(logits.detach(), ids, teacher, temperature=temperature), loss), what


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', WIDTHS + (70001,))
def test_distill(width, dtype):
    # from 513 classes on: 1100 rows a workgroup a row, fewer several, 4100 rows a wave a row
    for n, top, temperature in ((1, 1, 1.0), (5, 3, 2.0), (70, 33, 0.7), (1100, 8, 1.0), (3, 300, 4.0), (4100, 70, 2.0)):
        if n * width > 12_000_000:
            continue
        print('distill', n, width, top, dtype, flush=True)
        generator = _generator(width + n)
        logits = _logits(generator, dtype, n, width)
        ids = torch.randint(-1, width + 1, (n, top), generator=generator, device='cuda', dtype=(torch.int32, torch.int64)[n % 2])
        teacher = (torch.randn(n, top, generator=generator, device='cuda') * 3).to(DTYPES[(n + top) % 3])
        _check_distill(logits, ids, teacher, temperature, '%dx%d, %d entries' % (n, width, top))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('width', (40, 600))
def test_distill_masks(width, dtype):
    """The same class several times; masked logits and teachers; rows without an entry; a class the student masks."""
    logits = _logits(_generator(10), dtype, 6, width, blocked=0.2)
    logits[:, :8] = 1.0
    ids = torch.tensor([[3, 3, 5, 3], [0, 1, 2, 3], [-1, width, -7, 2 ** 30], [7, -1, 7, 6], [4, 5, 6, 7], [0, 0, 0, 0]],
                       device='cuda')
    teacher = torch.randn(6, 4, generator=_generator(11), device='cuda').to(dtype)
    teacher[1, 2], teacher[2], teacher[3, 1] = -math.inf, math.nan, math.nan
    teacher[4] = torch.tensor([-math.inf] * 3 + [2.0])
    _check_distill(logits, ids, torch.where(teacher.isnan(), 0.0, teacher), 1.5, 'masks')
    # what lies in entries of no class is not read
    assert torch.equal(distill(logits, ids, teacher), distill(logits, ids, torch.where(teacher.isnan(), 0.0, teacher)))
    logits[2] = math.nan
    leaf = logits.clone().requires_grad_(True)
    loss = distill(leaf, ids, teacher)
    gradient, = torch.autograd.grad(loss.sum(), leaf)
    assert loss[2] == 0 and not gradient[2].any() and not gradient.isnan().any()
    masked = logits.clone()
    masked[1, 1], masked[5] = -math.inf, -math.inf
    leaf = masked.requires_grad_(True)
    loss = distill(leaf, ids, teacher)
    assert loss[1] == math.inf and loss[5] == math.inf and loss[0].isfinite()
    gradient, = torch.autograd.grad(loss[5], leaf)
    assert gradient[5, 0] == -1 and not gradient[5, 1:].any()
    poisoned = teacher.clone()
    poisoned[0, 1] = math.nan
    loss = distill(logits, ids, poisoned)
    assert loss[0].isnan() and not loss[1:].isnan().any()


def test_one_entry_is_the_cross_entropy():
    logits = torch.randn(50, 700, generator=_generator(12), device='cuda')
    label = torch.randint(0, 700, (50, 1), generator=_generator(13), device='cuda')
    loss = distill(logits, label, torch.zeros(50, 1, device='cuda'))
    expected = -torch.log_softmax(logits.double(), 1).gather(1, label)[:, 0]
    assert (loss.double() - expected).abs().max() < 2.0 ** -18


@pytest.mark.parametrize('operator', ('choose', 'choose all', 'balance', 'distill'))
def test_gradients_against_differences(operator):
    """Central differences in fp32 of step 2^-6: off by its square times a third derivative (at most 8 of the largest
    weight here), and by the value's rounding over the step."""
    generator = _generator(14)
    logits = torch.randn(3, 12, generator=generator, device='cuda')
    mix = torch.randn(3, 4, generator=generator, device='cuda')
    expert = torch.topk(logits, 4, dim=1).indices.int()
    teacher = torch.randn(3, 4, generator=generator, device='cuda')
    calls = {'choose': lambda x: (choose(x, 4)[1] * mix).sum(),
             'choose all': lambda x: (choose(x, 4, normalize=False)[1] * mix).sum(),
             'balance': lambda x: balance(x, expert)[0], 'distill': lambda x: (distill(x, expert, teacher) * mix[:, 0]).sum()}
    call = calls[operator]
    # no logit near another, so that a step changes no choice
    logits = torch.argsort(torch.argsort(logits, 1), 1).float() * 0.25
    expert = torch.topk(logits, 4, dim=1).indices.int()
    leaf = logits.clone().requires_grad_(True)
    gradient, = torch.autograd.grad(call(leaf), leaf)
    step = 2.0 ** -6
    bound = step ** 2 * 8 * float(mix.abs().max().clamp(min=1)) / 6 + 2.0 ** -20 / step * 16
    for i in range(3):
        for e in range(12):
            up, down = logits.clone(), logits.clone()
            up[i, e] += step
            down[i, e] -= step
            slope = (float(call(up)) - float(call(down))) / (2 * step)
            assert abs(slope - float(gradient[i, e])) <= bound, (operator, i, e, slope, float(gradient[i, e]))


def test_refusals():
    x = torch.zeros(4, 8, device='cuda')
    expert = torch.zeros(4, 2, dtype=torch.int32, device='cuda')
    ids, teacher = torch.zeros(4, 2, dtype=torch.int64, device='cuda'), torch.zeros(4, 2, device='cuda')
    for bad in (lambda: choose(x, 0), lambda: choose(x, 9), lambda: choose(x, 2.0), lambda: choose(x.cpu(), 2),
                lambda: choose(x.double(), 2), lambda: choose(x[0], 2), lambda: choose(x.tolist(), 2),
                lambda: choose(torch.zeros(2, 80, device='cuda'), 65),
                lambda: balance(x, expert.long()), lambda: balance(x, expert[:3]), lambda: balance(x, expert[:, 0]),
                lambda: balance(x, expert.cpu()), lambda: balance(x, [[0]] * 4), lambda: balance(x, expert[:, :0]),
                lambda: distill(x, ids[:3], teacher), lambda: distill(x, ids, teacher[:, :1]),
                lambda: distill(x, ids.float(), teacher), lambda: distill(x, ids, teacher.double()),
                lambda: distill(x, ids[:, :0], teacher[:, :0]), lambda: distill(x, ids, teacher, temperature=0.0),
                lambda: distill(x, ids, teacher, temperature=float('nan')), lambda: distill(x, ids, teacher, temperature='1'),
                lambda: distill(x, ids, teacher.clone().requires_grad_(True)), lambda: distill(x, ids, teacher.cpu())):
        with pytest.raises(ValueError):
            bad()
    from odie_amd._lib import NativeError
    with pytest.raises(NativeError, match='experts'):
        choose(torch.zeros(1, 40000, device='cuda'), 2)


def test_double_backward_and_forward_mode_are_refused():
    import torch.autograd.forward_ad as forward_ad
    x = torch.randn(4, 8, device='cuda')
    expert, ids = torch.zeros(4, 2, dtype=torch.int32, device='cuda'), torch.zeros(4, 2, dtype=torch.int64, device='cuda')
    teacher = torch.zeros(4, 2, device='cuda')
    for call in (lambda t: choose(t, 2)[1], lambda t: balance(t, expert)[0], lambda t: distill(t, ids, teacher)):
        leaf = x.clone().requires_grad_(True)
        gradient, = torch.autograd.grad(call(leaf).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            gradient.sum().backward()
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x, torch.ones_like(x)))


def test_what_a_backward_reads_must_not_change():
    x = torch.randn(4, 8, device='cuda', requires_grad=True)
    expert, weights = choose(x, 2)
    expert.zero_()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        weights.sum().backward()
    loss, counts = balance(x, choose(x.detach(), 2)[0])
    counts.zero_()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()

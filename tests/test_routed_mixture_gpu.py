"""The learned router, the experts' layers and their 4-bit form together, as a program trains and serves them."""
import math

import pytest
import torch

from microscale64 import values64
from odie_amd.linear import linear
from odie_amd.microscale import Microscaled, quantize
from odie_amd.mixture import ExpertMixture, RoutedMixture, combine, dispatch, expert_order
from odie_amd.router import balance, choose, distill

pytestmark = pytest.mark.gpu


def _weight64(mixture, layer):
    codes, scales = getattr(mixture, 'codes%d' % layer), getattr(mixture, 'scales%d' % layer)
    width = mixture.widths[layer - 1]
    return values64(codes.flatten(0, 1), scales.flatten(0, 1), width).view(*codes.shape[:2], width)


def _blend64(x, expert, weights, w1, b1, w2, b2):
    """sum_j weights_j (W2_e relu(W1_e x + b1_e) + b2_e) in the type of x, for expert >= 0."""
    y = 0
    for j in range(expert.shape[1]):
        e = expert[:, j].long()
        held, e = (e >= 0)[:, None], e.clamp(min=0)
        hidden = torch.relu((w1[e] * x[:, None, :]).sum(2) + b1[e])
        y = y + torch.where(held, ((w2[e] * hidden[:, None, :]).sum(2) + b2[e]) * weights[:, j:j + 1], 0.0)
    return y


def test_a_training_step_of_all_parameters():
    """fp32 against torch's own autograd in 64 bits: the blend, the balance loss and the distillation in one loss.  Every
    value is a few hundred fp32 operations on numbers up to about ten: 2^-13 is a hundred times their rounding."""
    torch.manual_seed(0)
    model = RoutedMixture(6, 2, 20, 24, 5, dtype=torch.float32, seed=3)
    with torch.no_grad():
        model.mixture.bias1.copy_(0.3 * torch.randn_like(model.mixture.bias1))
    x = torch.randn(97, 20, device='cuda', requires_grad=True)
    target = torch.randn(97, 5, device='cuda')
    teacher_ids = torch.randint(0, 6, (97, 3), device='cuda')
    teacher = torch.randn(97, 3, device='cuda')
    allowed = torch.rand(97, 6, device='cuda') < 0.8
    allowed[5] = False
    y, logits, expert = model(x, allowed=allowed)
    loss, counts = balance(logits, expert)
    clear = logits.masked_fill(~allowed, -30.0)      # a student without masked classes
    total = (y - target).square().mean() + 0.1 * loss + 0.05 * distill(clear, teacher_ids, teacher, temperature=2.0).mean()
    names = [name for name, _ in model.named_parameters()]
    grads = torch.autograd.grad(total, [x] + list(model.parameters()))

    p = {name: value.detach().double().requires_grad_(True) for name, value in model.named_parameters()}
    x64 = x.detach().double().requires_grad_(True)
    raw = x64 @ p['router'].t()
    masked = raw.masked_fill(~allowed, -math.inf)
    part = expert >= 0
    at = expert.long().clamp(min=0)
    chosen = torch.where(part, masked.gather(1, at), -1e300)
    weights = torch.where(part, torch.softmax(chosen, 1), 0.0)
    y64 = _blend64(x64, expert, weights, *(p['mixture.' + name] for name in ('weight1', 'bias1', 'weight2', 'bias2')))
    assert not y[5].any() and (expert[5] == -1).all()
    rows = part.any(1)
    share = torch.softmax(masked[rows], 1)
    entries = torch.bincount(expert[part].long(), minlength=6)
    assert torch.equal(counts.long(), entries)
    frequency = entries.double() / part.sum()
    loss64 = 6 * (frequency * share.mean(0)).sum()
    own = torch.log_softmax(raw.masked_fill(~allowed, -30.0) / 2, 1).gather(1, teacher_ids)
    q = torch.log_softmax(teacher.double() / 2, 1)
    total64 = (y64 - target.double()).square().mean() + 0.1 * loss64 + 0.05 * (q.exp() * (q - own)).sum(1).mean()
    grads64 = torch.autograd.grad(total64, [x64] + [p[name] for name in names])
    assert abs(float(total.detach()) - float(total64.detach())) < 2.0 ** -13
    for name, got, expected in zip(['x'] + names, grads, grads64):
        assert (got.double() - expected).abs().max() <= 2.0 ** -13 * max(1.0, float(expected.abs().max())), name


@pytest.mark.parametrize('rows', (False, True))
@pytest.mark.parametrize('n', (1, 5, 300))
def test_a_mixture_served_in_4_bits(n, rows):
    """fp16 layers against the decoders of the values that the codes stand for.  Each of the two layers rounds its sums to
    fp16 and takes fp16 (or 4-bit) rows: sums of up to 48 terms of magnitude about 1, 2^-11 each and as much for the
    rows that enter the next, so that 48 * 2^-10 * 2 = 0.1 is more than all of it.  4-bit rows in between make steps of
    a quarter: their second layer is checked from the framework's own hidden rows."""
    torch.manual_seed(n)
    mixture = ExpertMixture(5, 40, 48, 3, codes=8, vocab=11, seed=2)
    with torch.no_grad():
        mixture.bias1.copy_(0.3 * torch.randn_like(mixture.bias1))
    served = mixture.microscaled(rows=rows)
    x = torch.randn(n, 40, device='cuda', dtype=torch.float16)
    ids = torch.randint(0, 11, (n,), device='cuda')
    expert = torch.randint(-1, 5, (n, 2), device='cuda', dtype=torch.int32)
    weights = torch.rand(n, 2, device='cuda')
    y = served(x, expert, weights, ids)
    assert y.dtype == torch.float16 and y.shape == (n, 3)
    joined = torch.cat((x, mixture.table[ids] * mixture.scale), 1)
    order = expert_order(expert, 5)
    w1, w2 = _weight64(served, 1), _weight64(served, 2)
    if not rows:
        expected = _blend64(joined.double(), expert, weights.double(), w1, served.bias1.double(), w2, served.bias2.double())
        assert (y.double() - expected).abs().max() < 0.1
        leaf, scale = x.clone().requires_grad_(True), weights.clone().requires_grad_(True)
        got = torch.autograd.grad(served(leaf, expert, scale, ids).float().sum(), (leaf, scale))
        x64, s64 = x.double().requires_grad_(True), weights.double().requires_grad_(True)
        joined = torch.cat((x64, (mixture.table[ids] * mixture.scale).detach().double()), 1)
        expected = torch.autograd.grad(_blend64(joined, expert, s64, w1, served.bias1.double(), w2, served.bias2.double()).sum(),
                                       (x64, s64))
        for a, b in zip(got, expected):
            close = (a.double() - b).abs() < 0.1
            # relu's slope jumps where a hidden sum is within its rounding of 0
            assert close.float().mean() > 0.98
        return
    hidden = linear(quantize(dispatch(joined, order)), Microscaled(served.codes1, served.scales1, 48, torch.float16),
                    served.bias1, activation='relu', offsets=order.offsets)
    xq, hq = quantize(dispatch(joined, order)), quantize(hidden)
    held = int(order.offsets[-1])
    owner = torch.repeat_interleave(torch.arange(5, device='cuda'), (order.offsets[1:] - order.offsets[:-1]).long())
    sums = torch.relu((w1[owner] * xq.dequantize().double()[:held, None]).sum(2) + served.bias1.double()[owner])
    assert (hidden.double()[:held] - sums).abs().max() < 0.1 if held else True
    second = (w2[owner] * hq.dequantize().double()[:held, None]).sum(2) + served.bias2.double()[owner]
    full = torch.zeros(2 * n, 3, device='cuda', dtype=torch.float64)
    full[:held] = second
    slots = order.slots.long()
    expected = (torch.where(slots[..., None] >= 0, full[slots.clamp(min=0)], 0.0) * weights.double()[..., None]).sum(1)
    assert (y.double() - expected).abs().max() < 0.1
    with pytest.raises(ValueError):
        served(x.clone().requires_grad_(True), expert, weights, ids)


def test_saved_and_loaded():
    served = ExpertMixture(3, 16, 32, 4, seed=1).microscaled()
    other = ExpertMixture(3, 16, 32, 4, seed=9).microscaled()
    x = torch.randn(20, 16, device='cuda', dtype=torch.float16)
    expert = torch.randint(0, 3, (20, 1), device='cuda')
    assert not torch.equal(served(x, expert), other(x, expert))
    other.load_state_dict(served.state_dict())
    assert torch.equal(served(x, expert), other(x, expert))
    assert not list(served.parameters())


def _step(model, served, x, ids, teacher):
    """A student router trained against a teacher and its frozen 4-bit experts; what a replay has to reproduce."""
    leaf = x.detach().requires_grad_(True)
    logits = linear(leaf, model.router)
    expert, weights = choose(logits, 2)
    y = served(leaf, expert, weights)
    loss, counts = balance(logits, expert)
    total = y.float().square().mean() + 0.1 * loss + distill(logits, ids, teacher, temperature=2.0).mean()
    grads = torch.autograd.grad(total * 256, (leaf, model.router))
    rows = linear(quantize(x), Microscaled(served.codes1[0], served.scales1[0], served.widths[0], torch.float16))
    return [t.detach() for t in (y, total, counts, expert, weights, rows, *grads)]


def test_captured_and_replayed():
    """One training step of all of them in a graph, replayed on other inputs with eager work in between."""
    model = RoutedMixture(8, 2, 32, 64, 16, seed=5)
    served = model.mixture.microscaled()
    x = torch.randn(500, 32, device='cuda', dtype=torch.float16)
    ids = torch.randint(-1, 8, (500, 3), device='cuda')
    teacher = torch.randn(500, 3, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(model, served, x, ids, teacher)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = _step(model, served, x, ids, teacher)
    for replay in range(4):
        x.copy_(torch.randn(500, 32, device='cuda', dtype=torch.float16))
        ids.copy_(torch.randint(-1, 8, (500, 3), device='cuda'))
        teacher.copy_(torch.randn(500, 3, device='cuda'))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in outputs]
        eager = _step(model, served, x, ids, teacher)
        torch.cuda.synchronize()
        for index, (a, b) in enumerate(zip(kept, eager)):
            assert torch.equal(a, b), (replay, index)


def test_two_streams_at_once():
    """Calls on two streams share nothing: each gives what it gives alone."""
    def work(seed):
        generator = torch.Generator(device='cuda').manual_seed(seed)
        logits = torch.randn(3000, 700, generator=generator, device='cuda')
        expert, weights = choose(logits, 4, normalize=False)
        loss, counts = balance(logits, expert)
        d = distill(logits[:7], expert[:7].long(), weights[:7])
        q = quantize(logits)
        return [expert, weights, loss, counts, d, q.codes, q.scales, linear(q, quantize(logits[:100]))]

    alone = [work(seed) for seed in (1, 2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for seed, stream in zip((1, 2), streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(work(seed))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


def test_router_of_a_whole_batch_without_an_expert():
    model = RoutedMixture(4, 2, 16, 32, 3, seed=1)
    x = torch.randn(10, 16, device='cuda', dtype=torch.float16, requires_grad=True)
    y, logits, expert = model(x, allowed=torch.zeros(4, dtype=torch.bool, device='cuda'))
    assert not y.any() and (expert == -1).all() and float(balance(logits, expert)[0]) == 0
    gradient, = torch.autograd.grad(y.float().sum() + balance(logits, expert)[0], x)
    assert not gradient.any()


def test_combine_takes_what_choose_gives():
    """Masked choices (-1) have no slot and add nothing."""
    logits = torch.tensor([[1.0, -math.inf, -math.inf], [0.0, 2.0, 1.0]], device='cuda')
    expert, weights = choose(logits, 2)
    order = expert_order(expert, 3)
    rows = dispatch(torch.tensor([[1.0], [10.0]], device='cuda'), order)
    y = combine(rows, order, weights)
    assert torch.allclose(y, torch.tensor([[1.0], [10.0]], device='cuda'))


def test_no_rows():
    model = RoutedMixture(4, 2, 16, 32, 3, codes=4, vocab=5, seed=1)
    x = torch.zeros(0, 16, device='cuda', dtype=torch.float16, requires_grad=True)
    ids = torch.zeros(0, device='cuda', dtype=torch.int64)
    y, logits, expert = model(x, ids)
    assert y.shape == (0, 3) and logits.shape == (0, 4) and expert.shape == (0, 2)
    loss = y.float().sum() + balance(logits, expert)[0] + distill(logits, expert, logits.detach()[:, :2]).sum()
    grads = torch.autograd.grad(loss, [x] + list(model.parameters()))
    assert float(loss) == 0 and not any(g.any() for g in grads)
    for rows in (False, True):
        assert model.mixture.microscaled(rows=rows)(x.detach(), expert, None, ids).shape == (0, 3)


def _passes(x, q, bias, ids, teacher):
    """A layer whose gradients come in one pass, and a distillation of few rows, cut in pieces."""
    leaf, own = x.detach().requires_grad_(True), bias.detach().requires_grad_(True)
    y = linear(leaf, q, own, activation='silu')
    logits = y.view(-1, 64 * 4096)[:1]
    loss = distill(logits, ids, teacher)
    return [t.detach() for t in (y, loss, *torch.autograd.grad(y.float().square().sum() / 64 + loss.sum(), (leaf, own)))]


def test_two_graphs_at_once():
    """Two captured passes with workspaces, replayed on two streams together, each on inputs of its own."""
    generator = torch.Generator(device='cuda').manual_seed(3)
    made, graphs = [], []
    for seed in range(2):
        x = torch.empty(70000 // 4096 * 4096, 48, device='cuda', dtype=torch.float16)
        q = quantize(torch.randn(64, 48, generator=generator, device='cuda', dtype=torch.float16))
        bias = torch.randn(64, generator=generator, device='cuda', dtype=torch.float16)
        ids = torch.randint(0, 64 * 4096, (1, 9), generator=generator, device='cuda')
        teacher = torch.randn(1, 9, generator=generator, device='cuda')
        made.append((x, q, bias, ids, teacher))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for inputs in made:
        inputs[0].normal_(generator=generator)
        with torch.cuda.stream(side):
            _passes(*inputs)
    torch.cuda.synchronize()
    for inputs in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = _passes(*inputs)
        graphs.append((graph, outputs))
    streams = [torch.cuda.Stream() for _ in graphs]
    for replay in range(3):
        for inputs in made:
            inputs[0].normal_(generator=generator)
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for inputs, (_, outputs) in zip(made, graphs):
            kept = [t.clone() for t in outputs]
            for index, (a, b) in enumerate(zip(kept, _passes(*inputs))):
                assert torch.equal(a, b), (replay, index)

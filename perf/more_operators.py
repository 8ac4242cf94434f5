"""The measured calls of the learned router and of layers with 4-bit weights: plain forms in 32 bits, and the
framework's own.

A case is a dict of plain values whose "kind" names the operator:

  choose    odie_amd.router.choose: each row's largest logits, their experts and softmax weights, and the
            logits' gradient
  balance   odie_amd.router.balance: the balance loss and the entries of each expert, and the logits' gradient
  distill   odie_amd.router.distill: the divergence from a teacher's top logits, and the logits' gradient
  quantize  odie_amd.microscale.quantize and back: microscaled 4-bit floating point, blocks of 32 with a power of two
  product   odie_amd.linear.linear with 4-bit weights, dense or one matrix per expert; rows as they are, or
            quantised to 4 bits too ("rows4"); the gradients of rows, bias and residual

"train" is True for the forward with its gradients, False for the forward alone (serving).
Inputs come from the seed alone.  exact() restates each operator in 64 bits with its gradients written out.
"""
import math

import torch

own = False

DTYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
ACTIVATIONS = ('none', 'relu', 'sigmoid', 'softplus', 'gelu', 'silu')
BLOCK = 32      # values that share a scale


def listed():
    return [
        # one sample's two of 64 experts: the latency of a serving call
        dict(name='choose_1', kind='choose', n=1, experts=64, choices=2, dtype='bf16', normalize=True, blocked=0.0,
             empty=0.0, train=False),
        # a training batch over the 1024 tiles of a gigapixel image, weights among all of them
        dict(name='choose_train_65536', kind='choose', n=65536, experts=1024, choices=4, dtype='fp16', normalize=False,
             blocked=0.0, empty=0.0, train=True),
        # a small step's router in full precision
        dict(name='balance_train_4096', kind='balance', n=4096, experts=64, choices=2, dtype='fp32', empty=0.0, train=True),
        # a ragged batch padded with rows of no expert, over 1000 experts
        dict(name='balance_train_300007', kind='balance', n=300007, experts=1000, choices=4, dtype='bf16', empty=0.1,
             train=True),
        # a few samples scored against the teacher while a fit runs
        dict(name='distill_64', kind='distill', n=64, classes=1024, top=8, dtype='fp16', temperature=1.0, lost=0.0,
             train=False),
        # a training batch over as many classes as a code table has rows
        dict(name='distill_train_8192', kind='distill', n=8192, classes=65032, top=64, dtype='bf16', temperature=2.0,
             lost=0.05, train=True),
        # the rows of a small serving batch
        dict(name='quantize_16', kind='quantize', n=16, width=2048, dtype='bf16'),
        # a whole batch of wide rows
        dict(name='quantize_65536', kind='quantize', n=65536, width=4096, dtype='fp16'),
        # one row through one wide layer with the whole epilogue: serving
        dict(name='product_1', kind='product', n=1, experts=0, inputs=2048, outputs=2048, dtype='bf16',
             activation='silu', bias=True, residual=True, rows4=False, skew=0.0, lost=0.0, train=False),
        # sixteen rows over 64 experts' layers: serving
        dict(name='product_experts_16', kind='product', n=16, experts=64, inputs=512, outputs=1024, dtype='fp16',
             activation='relu', bias=True, residual=False, rows4=False, skew=0.5, lost=0.0, train=False),
        # a large batch through a wide layer, rows and weights both in 4 bits
        dict(name='product_16384_rows4', kind='product', n=16384, experts=0, inputs=4096, outputs=4096, dtype='bf16',
             activation='gelu', bias=True, residual=False, rows4=True, skew=0.0, lost=0.0, train=False),
        # the sorted rows of a training batch through 64 experts' layers that stay as they are
        dict(name='product_experts_train_131072', kind='product', n=131072, experts=64, inputs=256, outputs=512,
             dtype='fp16', activation='silu', bias=True, residual=False, rows4=False, skew=0.3, lost=0.0, train=True),
    ]


def _size(rng, least, most):
    """A whole number spread over the logarithm of [least, most]: as it falls but odd, a power of two, or a
    multiple of 40, a third of the time each."""
    value = math.exp(rng.uniform(math.log(least), math.log(most)))
    form = rng.choice(('odd', 'power', 'even'))
    value = {'odd': round(value) | 1, 'power': 1 << round(math.log2(value)), 'even': round(value / 40) * 40}[form]
    return min(most, max(least, value))


def draw(rng):
    kind = rng.choice(('choose', 'balance', 'distill', 'quantize', 'product'))
    dtype = rng.choice(tuple(DTYPES))
    train = rng.random() < 0.6
    if kind in ('choose', 'balance'):
        n, experts = _size(rng, 1, 1 << 20), _size(rng, 4, 4096)
        while n * experts > 1 << 26:
            n = _size(rng, 1, 1 << 20)
        common = dict(kind=kind, n=n, experts=experts, choices=min(experts, rng.choice((1, 2, 3, 4, 8))), dtype=dtype,
                      empty=rng.choice((0.0, 0.1)), train=train)
        if kind == 'balance':
            return common
        return dict(**common, normalize=rng.random() < 0.5, blocked=rng.choice((0.0, 0.3)))
    if kind == 'distill':
        n, classes = _size(rng, 1, 1 << 17), _size(rng, 16, 1 << 17)
        while n * classes > 1 << 28:
            n = _size(rng, 1, 1 << 17)
        return dict(kind=kind, n=n, classes=classes, top=min(classes, _size(rng, 1, 128)), dtype=dtype,
                    temperature=rng.choice((1.0, 2.0, 0.7)), lost=rng.choice((0.0, 0.1)), train=train)
    if kind == 'quantize':
        n, width = _size(rng, 1, 1 << 17), _size(rng, 32, 16384)
        while n * width > 1 << 27:
            n = _size(rng, 1, 1 << 17)
        return dict(kind=kind, n=n, width=width, dtype=dtype)
    experts = _size(rng, 4, 128) if rng.random() < 0.5 else 0
    most = 1024 if experts else 4096
    inputs, outputs = _size(rng, 32, most), _size(rng, 32, most)
    rows4 = rng.random() < 0.4
    train = train and not rows4             # rows of 4 bits have no gradient
    n = _size(rng, 1, 1 << 17)
    while n * inputs * outputs > (1 << 34 if dtype == 'fp32' and not rows4 else 1 << 37):
        n = _size(rng, 1, 1 << 17)
    # relu's gradient jumps at 0, where two right sums of other orders may stand on either side: its forward alone
    return dict(kind=kind, n=n, experts=experts, inputs=inputs, outputs=outputs, dtype=dtype,
                activation=rng.choice([a for a in ACTIVATIONS if a != 'relu' or not train]), bias=rng.random() < 0.7,
                residual=rng.random() < 0.5, rows4=rows4, skew=round(rng.uniform(0.0, 0.5), 2),
                lost=rng.choice((0.0, 0.1)), train=train)


def _popular(generator, count, buckets, skew):
    """Ids in [0, buckets) whose popularity falls as rank ** -skew, the ranks in a random order."""
    weight = torch.arange(1, buckets + 1, device='cuda', dtype=torch.float64).pow(-skew)
    edges = weight.cumsum(0)
    point = torch.rand(count, generator=generator, device='cuda', dtype=torch.float64) * edges[-1]
    rank = torch.searchsorted(edges, point).clamp_(max=buckets - 1)
    return torch.randperm(buckets, generator=generator, device='cuda')[rank]


def prepare(case, seed):
    generator = torch.Generator(device='cuda').manual_seed(seed)
    kind, n, dtype = case['kind'], case['n'], DTYPES[case['dtype']]
    train = case.get('train', False)

    def normal(*shape, scale=1.0, grad=False, type=dtype):
        value = torch.randn(*shape, generator=generator, device='cuda', dtype=torch.float32).mul_(scale).to(type)
        return value.requires_grad_(grad and train)

    def some(share, *shape):
        return torch.rand(*shape, generator=generator, device='cuda') < share

    state = dict(kind=kind, train=train)
    if kind in ('choose', 'balance'):
        experts, choices = case['experts'], case['choices']
        # a router under training: some experts are liked by most rows
        logits = normal(n, experts, scale=1.5, type=torch.float32)
        logits += normal(experts, scale=0.7, type=torch.float32)
        logits = logits.to(dtype)
        lost = some(case['empty'], n)
        if kind == 'choose':
            logits[some(case['blocked'], n, experts)] = -math.inf
            logits[lost] = -math.inf
            state.update(logits=logits.requires_grad_(train), choices=choices, normalize=case['normalize'])
            if train:
                state.update(upstream=normal(n, choices, type=torch.float32))
            return state
        expert = torch.topk(logits.float(), choices, dim=1).indices.to(torch.int32)
        expert[lost] = -1
        state.update(logits=logits.requires_grad_(train), expert=expert)
        if train:
            state.update(upstream=torch.tensor(float(n), device='cuda'))     # a loss scale: 16 bits hold the gradient
        return state
    if kind == 'distill':
        classes, top = case['classes'], case['top']
        # the teacher's classes spread over the range, one from each stretch of it; the student half agrees with them
        stretch = torch.rand(n, top, generator=generator, device='cuda')
        ids = ((torch.arange(top, device='cuda') + stretch) * (classes / top)).long().clamp_(max=classes - 1)
        teacher = normal(n, top, scale=2.0, type=torch.float32) + 6.0
        logits = normal(n, classes, scale=1.5)
        logits.scatter_(1, ids, (0.5 * teacher + normal(n, top, type=torch.float32)).to(dtype))
        ids[some(case['lost'], n, top)] = -1
        state.update(logits=logits.requires_grad_(train), ids=ids, teacher=teacher.to(dtype),
                     temperature=case['temperature'])
        if train:
            # a weight for each row, times a loss scale
            state.update(upstream=64.0 * torch.rand(n, generator=generator, device='cuda'))
        return state
    if kind == 'quantize':
        # rows and blocks of differing sizes, as activations have them
        width = case['width']
        size = torch.exp(normal(n, 1, type=torch.float32) + normal(1, width, type=torch.float32))
        state.update(x=(normal(n, width, type=torch.float32).mul_(size)).to(dtype))
        return state
    inputs, outputs, experts = case['inputs'], case['outputs'], case['experts']
    lead = (experts,) if experts else ()
    codes, scales = _plain_quantize(normal(max(experts, 1) * outputs, inputs, scale=inputs ** -0.5, type=torch.float32))
    state.update(activation=case['activation'], x=normal(n, inputs, grad=True), rows4=case['rows4'],
                 codes=codes.view(*lead, outputs, -1), scales=scales.view(*lead, outputs, -1), inputs=inputs,
                 bias=normal(*lead, outputs, scale=0.1, grad=True) if case['bias'] else None,
                 residual=normal(n, outputs, grad=True) if case['residual'] else None, offsets=None)
    if experts:
        expert = _popular(generator, n, experts, case['skew'])
        expert[some(case['lost'], n)] = experts
        counts = torch.bincount(expert, minlength=experts + 1)[:experts]
        state['offsets'] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
    if train:
        state.update(upstream=normal(n, outputs))
    return state


# --- the plain forms ---------------------------------------------------------------------------------

def _plain_choose(logits, choices):
    """expert [N, choices] by falling logits, the lowest index first among equal ones, -1 past those above -inf."""
    left = logits.float().clone()
    index = torch.arange(left.shape[1], device=left.device)
    chosen = []
    for _ in range(choices):
        best = left.amax(1, keepdim=True)
        at = torch.where(left == best, index, left.shape[1]).amin(1, keepdim=True)
        chosen.append(torch.where(best > -math.inf, at, -1))
        left.scatter_(1, at, -math.inf)
    return torch.cat(chosen, 1)


def _plain_softmax(values):
    """Rows' softmax; 0 in rows that hold nothing above -inf."""
    top = values.amax(1, keepdim=True)
    share = torch.exp(values - torch.where(top > -math.inf, top, 0.0))
    return share / share.sum(1, keepdim=True).clamp(min=1e-30)


def _run_plain_choose(state):
    logits = state['logits'].detach()
    expert = _plain_choose(logits, state['choices'])
    held, at = expert >= 0, expert.clamp(min=0)
    if state['normalize']:
        weights = _plain_softmax(torch.where(held, logits.float().gather(1, at), -math.inf))
    else:
        share = _plain_softmax(logits.float())
        weights = torch.where(held, share.gather(1, at), 0.0)
    got = {'expert': expert.int(), 'weights': weights}
    if state['train']:
        up = state['upstream']
        total = (weights * up).sum(1, keepdim=True)
        if state['normalize']:
            gradient = torch.zeros(logits.shape, dtype=torch.float32, device=logits.device)
            gradient.scatter_add_(1, at, weights * (up - total))
        else:
            gradient = (-total * share).scatter_add_(1, at, weights * up)
        got['logits'] = gradient.to(logits.dtype)
    return got


def _run_plain_balance(state):
    logits, expert = state['logits'].detach(), state['expert'].long()
    n, experts = logits.shape
    held = expert >= 0
    counts = torch.zeros(experts, dtype=torch.int64, device=logits.device)
    counts.index_add_(0, expert[held], torch.ones_like(expert[held]))
    part = held.any(1)
    share = _plain_softmax(logits.float())
    rows, entries = part.sum().double(), held.sum().double()
    # a row's mean count under its softmax, over the entries
    mean = (share * counts.float()).sum(1, keepdim=True)
    norm = torch.where(rows > 0, experts / (rows * entries).clamp(min=1), 0.0)
    got = {'loss': (torch.where(part, mean[:, 0], 0.0).double().sum() * norm).float(), 'counts': counts.int()}
    if state['train']:
        gradient = share * (counts.float() - mean) * (norm * state['upstream'].double()).float()
        got['logits'] = torch.where(part[:, None], gradient, 0.0).to(logits.dtype)
    return got


def _run_plain_distill(state):
    logits, ids, warmth = state['logits'].detach(), state['ids'], state['temperature']
    held = (ids >= 0) & (ids < logits.shape[1])
    at = ids.clamp(min=0)
    target = torch.where(held, state['teacher'].float() / warmth, -math.inf)
    target = target - target.amax(1, keepdim=True).clamp(min=-1e30)
    share = torch.where(held, torch.exp(target), 0.0)
    total = share.sum(1, keepdim=True).clamp(min=1e-30)
    log_target, share = target - torch.log(total), share / total
    scaled = logits.float() / warmth
    scaled = scaled - scaled.amax(1, keepdim=True)
    power = torch.exp(scaled)
    sums = power.sum(1, keepdim=True)
    log_own = scaled.gather(1, at) - torch.log(sums)
    got = {'loss': torch.where(held, share * (log_target - log_own), 0.0).sum(1)}
    if state['train']:
        up = torch.where(held.any(1), state['upstream'] / warmth, 0.0)[:, None]
        gradient = power.mul_(up / sums)
        got['logits'] = gradient.scatter_add_(1, at, -share * up).to(logits.dtype)
    return got


def _plain_quantize(x):
    """codes [N, 16 * blocks] (two values a byte, the first in the low half) and scales [N, blocks rounded up to 4]
    (a power of two's exponent + 127) of rows x."""
    n, width = x.shape
    blocks = (width + BLOCK - 1) // BLOCK
    rows = torch.zeros(n, blocks * BLOCK, dtype=torch.float32, device=x.device)
    rows[:, :width] = x
    rows = rows.view(n, blocks, BLOCK)
    exponent = torch.frexp(rows.abs().amax(2)).exponent - 3       # of the largest's leading bit, less that of 4
    exponent = torch.where((rows == 0).all(2), -127, exponent).clamp(-127, 127)
    size = torch.ldexp(rows.abs(), -exponent[..., None])
    # the middles between 0, 0.5, 1, 1.5, 2, 3, 4 and 6; one that falls on a middle goes to the even code
    code = torch.zeros(rows.shape, dtype=torch.uint8, device=x.device)
    for value, even in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += size >= value if even else size > value
    code += 8 * torch.signbit(rows).to(torch.uint8)
    codes = code.view(n, blocks * BLOCK // 2, 2)
    scales = torch.zeros(n, (blocks + 3) // 4 * 4, dtype=torch.uint8, device=x.device)
    scales[:, :blocks] = (exponent + 127).to(torch.uint8)
    return codes[..., 0] + 16 * codes[..., 1], scales


def _plain_values(codes, scales, width):
    """The fp32 values [.., width] that codes and scales stand for."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat((table, -table))
    code = torch.stack((codes & 15, codes >> 4), -1).view(*codes.shape[:-1], -1, BLOCK)
    blocks = code.shape[-2]
    exponent = scales[..., :blocks, None].int() - 127
    return torch.ldexp(table[code.int()], exponent).flatten(-2)[..., :width]


def _activate(z, activation):
    if activation == 'relu':
        return torch.where(z > 0, z, 0.0)
    if activation == 'sigmoid':
        return 1.0 / (1.0 + torch.exp(-z))
    if activation == 'softplus':
        return torch.where(z > 0, z, 0.0) + torch.log1p(torch.exp(-z.abs()))
    if activation == 'gelu':
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if activation == 'silu':
        return z / (1.0 + torch.exp(-z))
    return z


def _run_plain_product(state):
    """Every expert's rows padded to the longest's count, one batched product each way; one expert without offsets."""
    x, bias, residual, train = (state[name] for name in ('x', 'bias', 'residual', 'train'))
    dtype, n = x.dtype, x.shape[0]
    x = x.detach().float()
    if state['rows4']:
        x = _plain_values(*_plain_quantize(x), state['inputs'])
    weight = _plain_values(state['codes'], state['scales'], state['inputs'])
    if state['offsets'] is None:
        weight = weight[None]
        offsets = torch.tensor([0, n], device=x.device)
    else:
        offsets = state['offsets'].long()
    experts = weight.shape[0]
    row = torch.arange(n, device=x.device)
    expert = torch.searchsorted(offsets[1:], row, right=True)
    held = (expert < experts)[:, None]
    expert = expert.clamp(max=experts - 1)
    place = torch.where(held[:, 0], row - offsets[expert], 0)
    counts = offsets[1:] - offsets[:-1]
    at = torch.arange(max(1, int(counts.max())), device=x.device)
    inside = (at < counts[:, None])[..., None]
    filled = (offsets[:-1, None] + at).clamp(max=n - 1)
    z = torch.bmm(torch.where(inside, x[filled], 0.0), weight.transpose(1, 2))
    if bias is not None:
        z = z + bias.detach().float().view(experts, 1, -1)
    with torch.enable_grad():
        value = _activate(z.requires_grad_(train), state['activation'])
    y = torch.where(held, value.detach()[expert, place], 0.0)
    if residual is not None:
        y = y + residual.detach().float()
    got = {'y': y.to(dtype)}
    if not train:
        return got
    dz, = torch.autograd.grad(value, z, torch.where(inside, state['upstream'].float()[filled], 0.0))
    got['x'] = torch.where(held, torch.bmm(dz, weight)[expert, place], 0.0).to(dtype)
    if bias is not None:
        got['bias'] = dz.sum(1).view(bias.shape).to(dtype)
    if residual is not None:
        got['residual'] = state['upstream']
    return got


def _run_plain(state):
    with torch.no_grad():
        if state['kind'] == 'choose':
            return _run_plain_choose(state)
        if state['kind'] == 'balance':
            return _run_plain_balance(state)
        if state['kind'] == 'distill':
            return _run_plain_distill(state)
        if state['kind'] == 'quantize':
            x = state['x']
            return {'values': _plain_values(*_plain_quantize(x.float()), x.shape[1]).to(x.dtype)}
        return _run_plain_product(state)


# --- the framework's operators -----------------------------------------------------------------------

def _run_own(state):
    kind, train = state['kind'], state['train']
    if kind == 'choose':
        from odie_amd.router import choose
        expert, weights = choose(state['logits'], state['choices'], normalize=state['normalize'])
        got = {'expert': expert, 'weights': weights}
        value = weights
    elif kind == 'balance':
        from odie_amd.router import balance
        loss, counts = balance(state['logits'], state['expert'])
        got = {'loss': loss, 'counts': counts}
        value = loss
    elif kind == 'distill':
        from odie_amd.router import distill
        value = distill(state['logits'], state['ids'], state['teacher'], temperature=state['temperature'])
        got = {'loss': value}
    elif kind == 'quantize':
        from odie_amd.microscale import quantize
        return {'values': quantize(state['x']).dequantize()}
    else:
        from odie_amd.linear import linear
        from odie_amd.microscale import Microscaled, quantize
        weight = Microscaled(state['codes'], state['scales'], state['inputs'])
        value = linear(quantize(state['x']) if state['rows4'] else state['x'], weight, state['bias'],
                       activation=state['activation'], residual=state['residual'], offsets=state['offsets'])
        got = {'y': value}
    if train:
        names = [name for name in ('logits', 'x', 'bias', 'residual') if state.get(name) is not None]
        got.update(zip(names, torch.autograd.grad(value, [state[name] for name in names], state['upstream'])))
    return got


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --- what a pass cannot do without -------------------------------------------------------------------

def work(case):
    n, kind, train = case['n'], case['kind'], case.get('train', False)
    size = 4 if case['dtype'] == 'fp32' else 2
    if kind == 'choose':
        logits, entries = n * case['experts'] * size, n * case['choices']
        moved = logits + 8 * entries                                # logits; experts and weights
        if train:                                                   # upstream; gradient
            moved += 4 * entries + logits
        return {'bytes': moved, 'flops': (5 if train else 3) * n * case['experts']}
    if kind == 'balance':
        logits, entries = n * case['experts'] * size, n * case['choices']
        moved = logits + 4 * entries + 4 * case['experts']
        if train:
            moved += logits
        return {'bytes': moved, 'flops': (8 if train else 4) * n * case['experts']}
    if kind == 'distill':
        logits, entries = n * case['classes'] * size, n * case['top']
        moved = logits + (8 + size) * entries + 4 * n
        if train:
            moved += logits + 4 * n
        return {'bytes': moved, 'flops': (6 if train else 3) * n * case['classes']}
    if kind == 'quantize':
        rows, blocks = n * case['width'] * size, n * ((case['width'] + BLOCK - 1) // BLOCK)
        return {'bytes': 2 * rows + 2 * 17 * blocks, 'flops': 3 * n * case['width']}    # rows there and back
    inputs, outputs = case['inputs'], case['outputs']
    # of the experts' matrices only those that some row needs
    needed = min(case['experts'], n) if case['experts'] else 1
    moved = size * (n * inputs + n * outputs * (2 if case['residual'] else 1))
    moved += needed * outputs * 17 * ((inputs + BLOCK - 1) // BLOCK)
    moved += size * needed * outputs if case['bias'] else 0
    if train:
        moved += size * (n * outputs + n * inputs)
        moved += size * max(case['experts'], 1) * outputs if case['bias'] else 0
    return {'bytes': moved, 'flops': (4 if train else 2) * n * inputs * outputs}


# --- the definitions in 64 bits ----------------------------------------------------------------------

def _pieces(rows, width):
    """Slices of rows of about 2^25 values."""
    step = max(1, (1 << 25) // width)
    return [slice(a, min(rows, a + step)) for a in range(0, rows, step)]


def _exact_choose(case, state):
    logits = state['logits'].detach()
    got = {'expert': None, 'weights': torch.zeros(case['n'], case['choices'], dtype=torch.float64, device='cuda')}
    if case['train']:
        got['logits'] = torch.zeros(logits.shape, dtype=torch.float64, device='cuda')
    for rows in _pieces(*logits.shape):
        order = torch.sort(logits[rows].double(), dim=1, descending=True, stable=True)
        value, at = order.values[:, :case['choices']], order.indices[:, :case['choices']]
        held = value > -math.inf
        base = value if case['normalize'] else logits[rows].double()
        log_weight = value - torch.logsumexp(base, 1, keepdim=True)
        weight = torch.where(held, torch.exp(log_weight), 0.0)
        got['weights'][rows] = weight
        if case['train']:
            up = state['upstream'][rows].double()
            inner = (weight * up).sum(1, keepdim=True)
            if not case['normalize']:
                spread = torch.softmax(logits[rows].double(), 1)
                got['logits'][rows] = -inner * torch.where(held[:, :1], spread, 0.0)
                inner = 0.0
            got['logits'][rows].scatter_add_(1, at, weight * (up - inner))
    return got


def _exact_balance(case, state):
    logits, expert = state['logits'].detach(), state['expert'].cpu()
    n, experts = logits.shape
    valid = expert >= 0
    frequency = torch.bincount(expert[valid].long(), minlength=experts).double().cuda()
    part = valid.any(1).cuda()
    got = {'loss': None, 'counts': None}
    if not bool(part.any()):
        got['loss'] = torch.zeros((), dtype=torch.float64, device='cuda')
        if case['train']:
            got['logits'] = torch.zeros(logits.shape, dtype=torch.float64, device='cuda')
        return got
    frequency /= frequency.sum()
    importance, gradients = torch.zeros(experts, dtype=torch.float64, device='cuda'), []
    rows_taken = part.sum().double()
    for rows in _pieces(n, experts):
        spread = torch.softmax(logits[rows].double(), 1) * part[rows, None]
        importance += spread.sum(0)
        if case['train']:
            factor = state['upstream'].double() * experts / rows_taken
            gradients.append(factor * spread * (frequency - (spread @ frequency)[:, None]))
    got['loss'] = experts * (frequency * importance / rows_taken).sum()
    if case['train']:
        got['logits'] = torch.cat(gradients)
    return got


def _exact_distill(case, state):
    logits, ids = state['logits'].detach(), state['ids']
    n, classes = logits.shape
    warmth = case['temperature']
    losses, gradients = [], []
    for rows in _pieces(n, classes):
        valid = ids[rows] >= 0
        target = (state['teacher'][rows].double() / warmth).masked_fill(~valid, -math.inf)
        log_target = target - torch.logsumexp(target, 1, keepdim=True)
        log_own = torch.log_softmax(logits[rows].double() / warmth, 1)
        at = ids[rows].clamp(min=0)
        share = torch.where(valid, torch.exp(log_target), 0.0)
        losses.append(torch.where(valid, share * (log_target - log_own.gather(1, at)), 0.0).sum(1))
        if case['train']:
            up = (state['upstream'][rows].double() / warmth)[:, None]
            own_share = torch.exp(log_own) * valid.any(1, keepdim=True)
            gradients.append(own_share.scatter_add_(1, at, -share) * up)
    got = {'loss': torch.cat(losses)}
    if case['train']:
        got['logits'] = torch.cat(gradients)
    return got


def _exact_levels(x):
    """The 64-bit values [N, width] nearest to x among those that its blocks' scales allow."""
    n, width = x.shape
    got = torch.empty(n, width, dtype=torch.float64, device=x.device)
    magnitudes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    middles = (magnitudes[1:] + magnitudes[:-1]) / 2
    for start in range(0, width, BLOCK):
        part = x[:, start:start + BLOCK].double()
        largest = part.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.floor(torch.log2(largest.clamp(min=2.0 ** -160))) - 2).clamp(2.0 ** -127, 2.0 ** 127)
        size = part.abs() / scale
        below, above = torch.bucketize(size, middles), torch.bucketize(size, middles, right=True)
        code = torch.where(below % 2 == 0, below, above)        # they differ on a middle alone
        got[:, start:start + BLOCK] = torch.copysign(magnitudes[code] * scale, part)
    return got


def _exact_activation(z, activation):
    """The activation and its derivative."""
    if activation == 'none':
        return z, torch.ones_like(z)
    if activation == 'relu':
        return z.clamp(min=0), (z > 0).double()
    sigmoid = torch.special.expit(z)
    if activation == 'sigmoid':
        return sigmoid, sigmoid * torch.special.expit(-z)
    if activation == 'softplus':
        return torch.logaddexp(z, torch.zeros_like(z)), sigmoid
    if activation == 'silu':
        return z * sigmoid, sigmoid * (1 + z * torch.special.expit(-z))
    area = torch.special.ndtr(z)
    return z * area, area + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _exact_weight(codes, scales, width):
    """A matrix' 64-bit values: sign, then exponent and fraction of each half byte."""
    half = torch.empty(*codes.shape, 2, dtype=torch.int64, device=codes.device)
    half[..., 0], half[..., 1] = codes % 16, codes // 16
    half = half.view(codes.shape[0], -1)
    power, fraction = half % 8 // 2, (half % 2).double()
    size = torch.where(power == 0, 0.5 * fraction, (1 + 0.5 * fraction) * torch.exp2(power.double() - 1))
    scale = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)[:, :half.shape[1]]
    return (torch.where(half >= 8, -size, size) * scale)[:, :width]


def _exact_product(case, state):
    x, train = state['x'].detach(), case['train']
    x = _exact_levels(x) if case['rows4'] else x.double()
    experts, n, outputs = max(case['experts'], 1), case['n'], case['outputs']
    codes, scales = state['codes'].view(experts, outputs, -1), state['scales'].view(experts, outputs, -1)
    bias = state['bias'].detach().double().view(experts, outputs) if case['bias'] else None
    ends = state['offsets'].tolist() if case['experts'] else [0, n]
    got = {'y': state['residual'].detach().double() if case['residual'] else x.new_zeros(n, outputs)}
    if train:
        got['x'] = torch.zeros_like(x)
        if case['bias']:
            got['bias'] = x.new_zeros(experts, outputs)
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if a == b:
            continue
        weight = _exact_weight(codes[e], scales[e], case['inputs'])
        z = x[a:b] @ weight.t()
        if case['bias']:
            z += bias[e]
        value, slope = _exact_activation(z, case['activation'])
        got['y'][a:b] += value
        if train:
            slope *= state['upstream'][a:b].double()
            got['x'][a:b] = slope @ weight
            if case['bias']:
                got['bias'][e] = slope.sum(0)
    if train and case['bias'] and not case['experts']:
        got['bias'] = got['bias'][0]
    if train and case['residual']:
        got['residual'] = state['upstream']
    return got


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case['kind'] == 'choose':
            return _exact_choose(case, state)
        if case['kind'] == 'balance':
            return _exact_balance(case, state)
        if case['kind'] == 'distill':
            return _exact_distill(case, state)
        if case['kind'] == 'quantize':
            return {'values': _exact_levels(state['x'])}
        return _exact_product(case, state)

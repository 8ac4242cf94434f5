"""The measured calls of the expert-mixture operators: plain forms in 32 bits, and the framework's own.

A case is a dict of plain values whose "kind" names the operator:

  embed     odie_amd.embedding.embed: rows of a table by id, scaled, and the table's gradient
  exchange  odie_amd.mixture: rows sorted by expert, sent to their slots and brought back with weights;
            gradients of the sent rows, the returned rows and the weights
  linear    odie_amd.linear.linear: x W^T + b, an activation, a residual, and every gradient
  experts   the same with one weight matrix per expert over rows that lie sorted by expert

"train" is True for the forward with its gradients, False for the forward alone (serving).
Inputs come from the seed alone.  exact() restates each operator in 64 bits with its gradients written out.
"""
import math

import torch

own = False

DTYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
ACTIVATIONS = ('none', 'relu', 'sigmoid', 'softplus', 'gelu', 'silu')


def listed():
    return [
        # the codes of a handful of samples, as an interactive preview looks them up
        dict(name='embed_64', kind='embed', n=64, vocab=1024, width=32, dtype='fp16', skew=0.0, train=False),
        # one training batch of the native step's size: a code for each of the 16384 tiles of a gigapixel image
        dict(name='embed_train_65536', kind='embed', n=65536, vocab=16384, width=64, dtype='fp16', skew=0.0,
             train=True),
        # ids that pile up on few rows, a ragged count, full precision
        dict(name='embed_train_300007_skewed', kind='embed', n=300007, vocab=65032, width=97, dtype='fp32', skew=1.1,
             train=True),
        # a multi-expert step's batch of coordinates, each with the code of its tile
        dict(name='embed_train_4m', kind='embed', n=1 << 22, vocab=16384, width=32, dtype='bf16', skew=0.5,
             train=True),
        # one sample between two experts: the latency of the whole round trip
        dict(name='exchange_1', kind='exchange', n=1, choices=2, experts=64, width=64, dtype='fp16', skew=0.0,
             lost=0.0, train=False),
        # a training batch, each sample blended from two of 64 experts
        dict(name='exchange_train_65536', kind='exchange', n=65536, choices=2, experts=64, width=256, dtype='fp16',
             skew=0.5, lost=0.0, train=True),
        # a ragged batch blended from the four nearest of 1024 tiles, some of them without an expert
        dict(name='exchange_train_300007', kind='exchange', n=300007, choices=4, experts=1024, width=131,
             dtype='bf16', skew=0.8, lost=0.1, train=True),
        # one row through one wide layer with the whole epilogue: serving
        dict(name='linear_1', kind='linear', n=1, inputs=2048, outputs=2048, dtype='bf16', activation='silu',
             bias=True, residual=True, train=False),
        # odd sizes in full precision
        dict(name='linear_train_odd', kind='linear', n=4099, inputs=333, outputs=517, dtype='fp32',
             activation='softplus', bias=True, residual=False, train=True),
        # a large batch through a wide layer
        dict(name='linear_train_65536', kind='linear', n=65536, inputs=1024, outputs=4096, dtype='bf16',
             activation='gelu', bias=True, residual=True, train=True),
        # sixteen rows over 64 experts' layers: serving
        dict(name='experts_16', kind='experts', n=16, experts=64, inputs=512, outputs=1024, dtype='fp16',
             activation='relu', bias=True, residual=False, skew=0.5, lost=0.0, train=False),
        # the sorted rows of a training batch through 64 experts' layers
        dict(name='experts_train_131072', kind='experts', n=131072, experts=64, inputs=256, outputs=512, dtype='fp16',
             activation='silu', bias=True, residual=False, skew=0.3, lost=0.0, train=True),
    ]


def _size(rng, least, most):
    """A whole number spread over the logarithm of [least, most]: as it falls but odd, a power of two, or a
    multiple of 40, a third of the time each."""
    value = math.exp(rng.uniform(math.log(least), math.log(most)))
    form = rng.choice(('odd', 'power', 'even'))
    value = {'odd': round(value) | 1, 'power': 1 << round(math.log2(value)), 'even': round(value / 40) * 40}[form]
    return min(most, max(least, value))


def draw(rng):
    kind = rng.choice(('embed', 'exchange', 'linear', 'experts'))
    train = rng.random() < 0.7
    dtype = rng.choice(tuple(DTYPES))
    skew = round(rng.uniform(0.0, 1.1), 2)
    if kind == 'embed':
        n, width = _size(rng, 64, 1 << 22), _size(rng, 32, 256)
        while n * width > 1 << 27:
            n = _size(rng, 64, 1 << 22)
        return dict(kind=kind, n=n, vocab=_size(rng, 1024, 65536), width=width, dtype=dtype, skew=skew, train=train)
    if kind == 'exchange':
        n, choices, width = _size(rng, 1, 300007), rng.choice((1, 2, 3, 4)), _size(rng, 64, 512)
        while n * choices * width > 150_000_000:
            n = _size(rng, 1, 300007)
        return dict(kind=kind, n=n, choices=choices, experts=_size(rng, 16, 1024), width=width, dtype=dtype, skew=skew,
                    lost=rng.choice((0.0, 0.1)), train=train)
    inputs, outputs = _size(rng, 32, 4096), _size(rng, 32, 4096)
    # relu's gradient jumps at 0, where two right sums of other orders may stand on either side: its forward alone
    common = dict(dtype=dtype, activation=rng.choice([a for a in ACTIVATIONS if a != 'relu' or not train]),
                  bias=rng.random() < 0.7,
                  residual=rng.random() < 0.5)
    # full precision costs sixteen times as much a product
    most = (1 << 38) // (16 if dtype == 'fp32' else 1)
    n = _size(rng, 1, 1 << 16)
    if kind == 'linear':
        while n * inputs * outputs > most:
            n = _size(rng, 1, 1 << 16)
        return dict(kind=kind, n=n, inputs=inputs, outputs=outputs, train=train, **common)
    experts = _size(rng, 4, 128)
    inputs, outputs = min(inputs, 1024), min(outputs, 1024)
    n = _size(rng, 16, 1 << 17)
    while n * inputs * outputs > most:
        n = _size(rng, 16, 1 << 17)
    return dict(kind=kind, n=n, experts=experts, inputs=inputs, outputs=outputs, skew=min(skew, 0.5),
                lost=rng.choice((0.0, 0.1)), train=train, **common)


def _chosen(generator, count, buckets, skew):
    """Ids in [0, buckets) whose popularity falls as rank ** -skew, the ranks in a random order."""
    weight = torch.arange(1, buckets + 1, device='cuda', dtype=torch.float64).pow(-skew)
    edges = weight.cumsum(0)
    point = torch.rand(count, generator=generator, device='cuda', dtype=torch.float64) * edges[-1]
    rank = torch.searchsorted(edges, point).clamp_(max=buckets - 1)
    return torch.randperm(buckets, generator=generator, device='cuda')[rank]


def prepare(case, seed):
    generator = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    train = case['train']

    def normal(*shape, scale=1.0, grad=False):
        value = torch.randn(*shape, generator=generator, device='cuda', dtype=torch.float32).mul_(scale).to(dtype)
        return value.requires_grad_(grad and train)

    n, kind = case['n'], case['kind']
    state = dict(kind=kind, train=train)
    if kind == 'embed':
        width = case['width']
        state.update(table=normal(case['vocab'], width, scale=0.1, grad=True), scale=math.sqrt(width),
                     ids=_chosen(generator, n, case['vocab'], case['skew']))
        if train:
            state.update(upstream=normal(n, width))
        return state
    if kind == 'exchange':
        width, choices, experts = case['width'], case['choices'], case['experts']
        expert = _chosen(generator, n * choices, experts, case['skew']).to(torch.int32)
        expert[torch.rand(n * choices, generator=generator, device='cuda') < case['lost']] = -1
        weights = torch.rand(n, choices, generator=generator, device='cuda') + 0.1
        weights = weights / weights.sum(1, keepdim=True)
        state.update(expert=expert.view(n, choices), experts=experts, x=normal(n, width, grad=True),
                     rows=normal(n * choices, width, grad=True), weights=weights.requires_grad_(train))
        if train:
            state.update(upstream=normal(n, width), sent_upstream=normal(n * choices, width))
        return state
    inputs, outputs = case['inputs'], case['outputs']
    lead = (case['experts'],) if kind == 'experts' else ()
    state.update(activation=case['activation'], x=normal(n, inputs, grad=True),
                 weight=normal(*lead, outputs, inputs, scale=inputs ** -0.5, grad=True),
                 bias=normal(*lead, outputs, scale=0.1, grad=True) if case['bias'] else None,
                 residual=normal(n, outputs, grad=True) if case['residual'] else None, offsets=None)
    if kind == 'experts':
        expert = _chosen(generator, n, case['experts'], case['skew'])
        expert[torch.rand(n, generator=generator, device='cuda') < case['lost']] = case['experts']
        counts = torch.bincount(expert, minlength=case['experts'] + 1)[:case['experts']]
        state['offsets'] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
    if train:
        state.update(upstream=normal(n, outputs))
    return state


# --- the plain forms ---------------------------------------------------------------------------------

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


def _plain_embed(table, ids, scale):
    return (table.float()[ids] * scale).to(table.dtype)


def _plain_embed_gradient(table, ids, scale, upstream):
    total = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
    return total.index_add_(0, ids, upstream.float() * scale).to(table.dtype)


def _plain_order(expert, experts):
    """(slots, source, offsets) of the rows sorted by expert, ties by row and choice."""
    flat = expert.reshape(-1).long()
    held = (flat >= 0) & (flat < experts)
    key, source = torch.sort(torch.where(held, flat, experts), stable=True)
    slots = torch.empty_like(source)
    slots[source] = torch.arange(source.numel(), device=source.device)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=key.device))
    return torch.where(held, slots, -1).view(expert.shape), source, offsets, key < experts


def _plain_dispatch(x, source, held, choices):
    return torch.where(held[:, None], x.float()[source // choices], 0.0).to(x.dtype)


def _plain_combine(rows, slots, weights):
    taken = torch.where(slots[..., None] >= 0, rows.float()[slots.clamp(min=0)], 0.0)
    return (taken * weights[..., None]).sum(1).to(rows.dtype)


def _plain_combine_gradient(rows, slots, source, held, weights, upstream):
    choices = weights.shape[1]
    up = upstream.float()
    weight = torch.where(held, weights.reshape(-1)[source], 0.0)
    drows = up[source // choices] * weight[:, None]
    taken = torch.where(slots[..., None] >= 0, rows.float()[slots.clamp(min=0)], 0.0)
    return drows.to(rows.dtype), (taken * up[:, None]).sum(2)


def _plain_linear(x, weight, bias, activation, residual):
    z = x.float() @ weight.float().t()
    if bias is not None:
        z = z + bias.float()
    y = _activate(z, activation)
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def _plain_experts(state):
    """Every expert's rows padded to the longest's count: one batched product each way."""
    x, weight, bias, residual, train = (state[name] for name in ('x', 'weight', 'bias', 'residual', 'train'))
    offsets, experts = state['offsets'].long(), weight.shape[0]
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(offsets[1:], row, right=True)
    held = (expert < experts)[:, None]
    expert = expert.clamp(max=experts - 1)
    place = torch.where(held[:, 0], row - offsets[expert], 0)
    counts = offsets[1:] - offsets[:-1]
    at = torch.arange(max(1, int(counts.max())), device=x.device)
    inside = (at < counts[:, None])[..., None]
    filled = (offsets[:-1, None] + at).clamp(max=x.shape[0] - 1)
    xs = torch.where(inside, x.float()[filled], 0.0)
    z = torch.bmm(xs, weight.float().transpose(1, 2))
    if bias is not None:
        z = z + bias.float()[:, None]
    with torch.enable_grad():
        value = _activate(z.requires_grad_(train), state['activation'])
    y = torch.where(held, value.detach()[expert, place], 0.0)
    if residual is not None:
        y = y + residual.float()
    got = {'y': y.to(x.dtype)}
    if not train:
        return got
    upstream = torch.where(inside, state['upstream'].float()[filled], 0.0)
    dz, = torch.autograd.grad(value, z, upstream)
    got['x'] = torch.where(held, torch.bmm(dz, weight.float())[expert, place], 0.0).to(x.dtype)
    got['weight'] = torch.bmm(dz.transpose(1, 2).contiguous(), xs).to(x.dtype)
    if bias is not None:
        got['bias'] = dz.sum(1).to(x.dtype)
    if residual is not None:
        got['residual'] = state['upstream']
    return got


def _run_plain(state):
    if state['kind'] == 'linear':
        y = _plain_linear(state['x'], state['weight'], state['bias'], state['activation'], state['residual'])
        return _with_gradients(state, y)
    with torch.no_grad():
        return _plain_experts(state) if state['kind'] == 'experts' else _run_plain_moves(state)


def _run_plain_moves(state):
    train = state['train']
    if state['kind'] == 'embed':
        got = {'y': _plain_embed(state['table'], state['ids'], state['scale'])}
        if train:
            got['table'] = _plain_embed_gradient(state['table'], state['ids'], state['scale'], state['upstream'])
        return got
    choices = state['expert'].shape[1]
    slots, source, offsets, held = _plain_order(state['expert'], state['experts'])
    got = {'slots': slots.int(), 'offsets': offsets.int(),
           'sent': _plain_dispatch(state['x'], source, held, choices),
           'y': _plain_combine(state['rows'], slots, state['weights'])}
    if train:
        got['x'] = _plain_combine(state['sent_upstream'], slots, torch.ones_like(state['weights']))
        got['rows'], got['weights'] = _plain_combine_gradient(state['rows'], slots, source, held,
                                                              state['weights'], state['upstream'])
    return got


def _with_gradients(state, y):
    if not state['train']:
        return {'y': y}
    names = [name for name in ('x', 'weight', 'bias', 'residual') if state[name] is not None]
    grads = torch.autograd.grad(y, [state[name] for name in names], state['upstream'])
    return {'y': y, **dict(zip(names, grads))}


# --- the framework's operators -----------------------------------------------------------------------

def _run_own(state):
    kind, train = state['kind'], state['train']
    if kind == 'embed':
        from odie_amd.embedding import embed
        y = embed(state['table'], state['ids'], state['scale'])
        if not train:
            return {'y': y}
        return {'y': y, 'table': torch.autograd.grad(y, state['table'], state['upstream'])[0]}
    if kind == 'exchange':
        from odie_amd.mixture import combine, dispatch, expert_order
        order = expert_order(state['expert'], state['experts'])
        sent = dispatch(state['x'], order)
        y = combine(state['rows'], order, state['weights'])
        got = {'slots': order.slots, 'offsets': order.offsets, 'sent': sent, 'y': y}
        if train:
            got['x'], = torch.autograd.grad(sent, state['x'], state['sent_upstream'])
            got['rows'], got['weights'] = torch.autograd.grad(y, (state['rows'], state['weights']), state['upstream'])
        return got
    from odie_amd.linear import linear
    y = linear(state['x'], state['weight'], state['bias'], activation=state['activation'], residual=state['residual'],
               offsets=state['offsets'])
    return _with_gradients(state, y)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --- what a pass cannot do without -------------------------------------------------------------------

def work(case):
    n, train, size = case['n'], case['train'], 4 if case['dtype'] == 'fp32' else 2
    if case['kind'] == 'embed':
        rows, vocab = n * case['width'] * size, case['vocab'] * case['width'] * size
        moved = 8 * n + min(rows, vocab) + rows
        if train:
            moved += rows + vocab
        return {'bytes': moved, 'flops': (2 if train else 1) * n * case['width']}
    if case['kind'] == 'exchange':
        slots = n * case['choices']
        few, many = n * case['width'] * size, slots * case['width'] * size
        moved = 4 * slots + 4 * slots + 4 * (case['experts'] + 1)       # expert ids, slots, offsets
        moved += few + many                                             # send
        moved += many + 4 * slots + few                                 # return
        if train:
            moved += many + few                                         # gradient of the sent rows
            moved += few + many + 4 * slots                             # gradients of the returned rows and weights
        return {'bytes': moved, 'flops': slots * case['width'] * (7 if train else 2)}
    inputs, outputs, experts = case['inputs'], case['outputs'], case.get('experts', 1)
    # of the experts' matrices only those that some row needs
    needed = min(experts, n)
    moved = n * inputs + needed * outputs * inputs + n * outputs * (2 if case['residual'] else 1)
    moved += needed * outputs if case['bias'] else 0
    if train:
        moved += n * outputs + n * inputs + experts * outputs * inputs  # upstream; gradients
        moved += experts * outputs if case['bias'] else 0
    return {'bytes': moved * size, 'flops': (6 if train else 2) * n * inputs * outputs}


# --- the definitions in 64 bits ----------------------------------------------------------------------

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


def _exact_product(state, x, weight, bias, residual, upstream):
    z = x @ weight.transpose(0, 1)
    if bias is not None:
        z += bias
    y, slope = _exact_activation(z, state['activation'])
    if residual is not None:
        y = y + residual
    if upstream is None:
        return y, None, None, None
    slope *= upstream
    return y, slope @ weight, slope.transpose(0, 1) @ x, slope.sum(0)


def _doubles(state):
    return {name: value.detach().double() if torch.is_tensor(value) and value.is_floating_point() else value
            for name, value in state.items()}


def exact(case, seed):
    state = _doubles(prepare(case, seed))
    train = state['train']
    if case['kind'] == 'embed':
        got = {'y': torch.index_select(state['table'], 0, state['ids']) * state['scale']}
        if train:
            got['table'] = torch.zeros_like(state['table']).index_add_(0, state['ids'], state['upstream'],
                                                                       alpha=state['scale'])
        return got
    if case['kind'] == 'exchange':
        return _exact_exchange(case, state)
    if case['kind'] == 'linear':
        y, dx, dw, db = _exact_product(state, state['x'], state['weight'], state['bias'], state['residual'],
                                       state.get('upstream'))
        got = {'y': y}
        if train:
            got.update(x=dx, weight=dw)
    else:
        x, residual, up = state['x'], state['residual'], state.get('upstream')
        got = {'y': residual.clone() if residual is not None else x.new_zeros(case['n'], case['outputs'])}
        if train:
            got.update(x=torch.zeros_like(x), weight=torch.zeros_like(state['weight']))
            db = x.new_zeros(case['experts'], case['outputs'])
        ends = state['offsets'].tolist()
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            if a == b:
                continue
            y, dx, dw, db_e = _exact_product(state, x[a:b], state['weight'][e],
                                             state['bias'][e] if case['bias'] else None,
                                             residual[a:b] if residual is not None else None,
                                             up[a:b] if train else None)
            got['y'][a:b] = y
            if train:
                got['x'][a:b], got['weight'][e], db[e] = dx, dw, db_e
    if train and case['bias']:
        got['bias'] = db
    if train and case['residual']:
        got['residual'] = state['upstream']
    return got


def _exact_exchange(case, state):
    n, choices, experts, width = case['n'], case['choices'], case['experts'], case['width']
    expert = state['expert'].cpu().numpy().reshape(-1)
    bucket = expert.astype('int64')
    bucket[(bucket < 0) | (bucket >= experts)] = experts
    source = bucket.argsort(kind='stable')
    held = int((bucket < experts).sum())
    device = state['x'].device
    flat = torch.from_numpy(source[:held]).to(device)         # of every slot that an expert owns
    row, choice = flat // choices, flat % choices
    sent = state['x'].new_zeros(n * choices, width)
    sent[:held] = state['x'][row]
    weight = state['weights'][row, choice][:, None]
    y = state['x'].new_zeros(n, width).index_add_(0, row, state['rows'][:held] * weight)
    got = {'slots': None, 'offsets': None, 'sent': sent, 'y': y}
    if case['train']:
        got['x'] = state['x'].new_zeros(n, width).index_add_(0, row, state['sent_upstream'][:held])
        up = state['upstream'][row]
        got['rows'] = torch.zeros_like(state['rows'])
        got['rows'][:held] = up * weight
        got['weights'] = torch.zeros_like(state['weights'])
        got['weights'][row, choice] = (up * state['rows'][:held]).sum(1)
    return got

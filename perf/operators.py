"""Measured cases of the gated delta rule (whole sequences and single tokens) and of counter-based dropout.

The gated delta rule is the second sequence mixer of a hybrid DISM language model.  Per value head, with a state S [D,DV]:

    S_t = exp(g_t) S_{t-1} + k_t u_t^T,    u_t = beta_t (v_t - exp(g_t) S_{t-1}^T k_t),    o_t = scale S_t^T q_t

Dropout keeps element i of a tensor when its 16-bit random number is at least round(65536 p); the numbers come from
Philox4x32-10 (Salmon et al., SC 2011) with the seed as the key and (i // 8, site, offset) as the counter.
"""
import math

import numpy as np
import torch

own = False

CHUNK = 64


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    train = dict(op='delta_train', documents='')
    return [
        # training step of the mixer (forward and backward) on the benchmark model's layer: 16 sequences of 2048, 10 heads of 128
        dict(train, name='train_model', batch=16, n=2048, key_heads=10, heads=10, d=128, dv=128),
        # long sequences, 16 heads: the sequence length and heads of the benchmark shape
        dict(train, name='train_long', batch=2, n=8192, key_heads=16, heads=16, d=64, dv=64),
        # one packed row of documents of odd lengths (one of a single token), key heads shared by pairs of value heads
        dict(train, name='train_packed', batch=1, n=7019, key_heads=4, heads=8, d=64, dv=128,
             documents='1,700,63,2049,64,65,511,3000,566'),
        # a fine-tuning microbatch of one short sequence: latency of the chain of chunks
        dict(train, name='train_small', batch=1, n=500, key_heads=4, heads=4, d=128, dv=128),
        # prompt processing: one long prompt continued from a cached state, new state kept
        dict(op='delta_prefill', name='prefill_long', batch=1, n=16384, key_heads=8, heads=16, d=128, dv=128, documents=''),
        # a batch of ragged prompts in one pack, with states
        dict(op='delta_prefill', name='prefill_ragged', batch=1, n=4133, key_heads=8, heads=16, d=128, dv=128,
             documents='512,17,1024,130,255,1,2048,146'),
        # one decoded token of one sequence: the smallest call
        dict(op='delta_step', name='step_one', batch=1, slots=1, key_heads=10, heads=10, d=128, dv=128),
        # one decoded token of every sequence of a server's batch, states in a larger pool, some rows padding
        dict(op='delta_step', name='step_server', batch=96, slots=128, key_heads=8, heads=16, d=128, dv=128),
        # residual dropout of the benchmark model, forward and backward: batch 16 x 2048 x 1280
        dict(op='dropout', name='dropout_model', rows=16 * 2048, width=1280, p=0.1, residual=True, dtype='bfloat16'),
        # dropout of a tensor with an odd number of elements in 32 bits, no residual
        dict(op='dropout', name='dropout_odd', rows=997, width=1283, p=0.25, residual=False, dtype='float32'),
        # residual dropout of one short sequence: launch latency
        dict(op='dropout', name='dropout_small', rows=500, width=512, p=0.1, residual=True, dtype='float16'),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(['delta_train', 'delta_train', 'delta_prefill', 'delta_step', 'dropout'])
    if op == 'dropout':
        width = _log(rng, 33, 2560)
        return dict(op=op, rows=max(1, _log(rng, 30_000, 16 * 2048 * 1280) // width), width=width,
                    p=rng.choice([0.05, 0.1, 0.2, 0.5]), residual=rng.random() < .7,
                    dtype=rng.choice(['bfloat16', 'bfloat16', 'float16', 'float32']))
    d, dv = rng.choice([(32, 64), (64, 64), (64, 128), (128, 64), (128, 128), (128, 128)])
    key_heads = rng.choice([1, 2, 4, 5, 8, 10])
    heads = key_heads * rng.choice([1, 1, 1, 2])
    if op == 'delta_step':
        batch = _log(rng, 1, 128)
        return dict(op=op, batch=batch, slots=batch + rng.randrange(0, 33), key_heads=key_heads, heads=heads, d=d, dv=dv)
    packed = rng.random() < .4
    most = 327_680 if op == 'delta_train' else 262_144  # positions x heads of the largest listed cases
    n = _log(rng, 65, min(16_384, most // heads))
    batch = 1 if packed else max(1, min(_log(rng, 1, 16), most // (n * heads)))
    documents = ''
    if packed:
        cuts = sorted(rng.sample(range(1, n), min(n - 1, rng.randrange(1, 9))))
        documents = ','.join(str(b - a) for a, b in zip([0] + cuts, cuts + [n]))
    return dict(op=op, batch=batch, n=n, key_heads=key_heads, heads=heads, d=d, dv=dv, documents=documents)


def work(case):
    if case['op'] == 'dropout':  # forward and backward: x (and the residual) and dy in, y and dx out
        size = {'bfloat16': 2, 'float16': 2, 'float32': 4}[case['dtype']]
        count = case['rows'] * case['width']
        return dict(bytes=count * size * (4 + case['residual']), flops=4 * count)
    hk, h, d, dv = case['key_heads'], case['heads'], case['d'], case['dv']
    if case['op'] == 'delta_step':
        active = case['batch'] - len(_padding(case))
        return dict(bytes=active * h * d * dv * 8 + case['batch'] * (4 * hk * d + 4 * h * dv + 8 * h), flops=7 * active * h * d * dv)
    tokens = case['batch'] * case['n']
    sequences = len(case['documents'].split(',')) if case['documents'] else case['batch']
    if case['op'] == 'delta_prefill':
        return dict(bytes=tokens * (4 * hk * d + 4 * h * dv + 8 * h) + sequences * h * d * dv * 8, flops=6 * tokens * h * d * dv)
    # q, k, v, gates and the output's gradient in; the output and five gradients out
    return dict(bytes=tokens * (8 * hk * d + 8 * h * dv + 8 * h), flops=18 * tokens * h * d * dv)


# ---- inputs ------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device='cuda')


def _padding(case):
    """Rows of a decoding batch that hold no sequence: every seventh of a batch larger than the smallest."""
    return [] if case['slots'] == case['batch'] else list(range(6, case['batch'], 7))


def _gates(g, *shape):
    """Log decay and write strength as the layer makes them: -A softplus(x + bias) with A in [0, 16) and steps of
    1e-3 to 0.1 a head, and a sigmoid."""
    h = shape[-1]
    rate = torch.rand(h, generator=g, device='cuda') * 16
    step = torch.exp(torch.rand(h, generator=g, device='cuda') * (math.log(.1) - math.log(.001)) + math.log(.001))
    bias = step + torch.log(-torch.expm1(-step))
    decay = -rate * torch.nn.functional.softplus(_randn(g, *shape) + bias)
    return decay, torch.sigmoid(_randn(g, *shape))


def prepare(case, seed):
    g = _generator(seed)
    if case['op'] == 'dropout':
        dtype = getattr(torch, case['dtype'])
        make = lambda: _randn(g, case['rows'], case['width']).to(dtype)
        counter = torch.tensor([seed * 1_000_003 + 12345, seed % 1000], dtype=torch.int64, device='cuda')
        return dict(case=case, x=make(), residual=make() if case['residual'] else None, dy=make(), seed=counter, site=3)
    hk, h, d, dv = case['key_heads'], case['heads'], case['d'], case['dv']
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)
    if case['op'] == 'delta_step':
        b = case['batch']
        decay, beta = _gates(g, b, h)
        slots = torch.randperm(case['slots'], generator=g, device='cuda')[:b].to(torch.int32)
        slots[_padding(case)] = -1
        return dict(case=case, q=unit(_randn(g, b, hk, d)).bfloat16(), k=unit(_randn(g, b, hk, d)).bfloat16(),
                    v=_randn(g, b, h, dv).bfloat16(), g=decay, beta=beta, state=_randn(g, case['slots'], h, d, dv) * .1,
                    slots=slots if case['slots'] > b or b > 1 else None)
    b, n = case['batch'], case['n']
    decay, beta = _gates(g, b, n, h)
    state = dict(case=case, q=unit(_randn(g, b, n, hk, d)).bfloat16(), k=unit(_randn(g, b, n, hk, d)).bfloat16(),
                 v=_randn(g, b, n, h, dv).bfloat16(), lengths=None, cu_seqlens=None)
    if case['documents']:
        state['lengths'] = [int(x) for x in case['documents'].split(',')]
        state['cu_seqlens'] = torch.tensor([0] + state['lengths'], device='cuda').cumsum(0).to(torch.int32)
    if case['op'] == 'delta_train':
        state.update(g=decay.bfloat16(), beta=beta.bfloat16(), dout=_randn(g, b, n, h, dv).bfloat16())
        for name in ('q', 'k', 'v', 'g', 'beta'):
            state[name].requires_grad_()
    else:
        sequences = len(state['lengths']) if state['lengths'] else b
        state.update(g=decay, beta=beta, initial=_randn(g, sequences, h, d, dv) * .1)
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------
def _pad(x, lengths):
    """[1,T,...] packed -> [documents, longest, ...], zeros behind each document."""
    rows = torch.split(x[0], lengths)
    return torch.nn.utils.rnn.pad_sequence(rows, batch_first=True)


def _unpad(x, lengths):
    return torch.cat([x[i, :m] for i, m in enumerate(lengths)])[None]


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular a [..., C, C], C a power of two: blocks joined two by two."""
    c = a.size(-1)
    inverse = torch.ones(*a.shape[:-2], c, 1, 1, dtype=a.dtype, device=a.device)
    size = 1
    while size < c:
        pairs = c // (2 * size)
        blocks = a.reshape(*a.shape[:-2], pairs, 2, size, pairs, 2, size)
        below = torch.diagonal(blocks[..., :, 1, :, :, 0, :], dim1=-4, dim2=-2).movedim(-1, -3)
        inverse = inverse.reshape(*a.shape[:-2], pairs, 2, size, size)
        top, bottom = inverse[..., 0, :, :], inverse[..., 1, :, :]
        corner = -(bottom @ below @ top)
        inverse = torch.cat((torch.cat((top, torch.zeros_like(top)), -1), torch.cat((corner, bottom), -1)), -2)
        size *= 2
    return inverse[..., 0, :, :]


def _delta(q, k, v, g, beta, scale, s):
    """The rule over whole sequences in 32 bits, [B,N,H,*] operands, state s [B,H,D,DV]: chunks of 64 positions."""
    b, n, h, dv = v.shape
    groups = h // q.size(2)
    q, k = (x.repeat_interleave(groups, 2) for x in (q, k))
    fill = -n % CHUNK
    chunks = lambda x: torch.nn.functional.pad(x, (0, 0) * (x.dim() - 2) + (0, fill)).transpose(1, 2).reshape(b, h, -1, CHUNK, *x.shape[3:])
    q, k, v, g, beta = (chunks(x) for x in (q, k, v, g, beta))
    total = g.double().cumsum(-1)
    later = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=v.device).tril()
    between = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~later, -math.inf)).float()
    decay, tail = torch.exp(total).float(), torch.exp(total[..., -1:] - total).float()
    mixed = beta[..., None] * between * (k @ k.transpose(-1, -2))
    inverse = _unit_lower_inverse(mixed.tril(-1))
    read = inverse @ ((beta * decay)[..., None] * k)
    written = inverse @ (beta[..., None] * v)
    inside = between * (q @ k.transpose(-1, -2)) * scale
    outer = (scale * decay)[..., None] * q
    kept = tail[..., None] * k
    out = []
    for c in range(q.size(2)):
        u = written[:, :, c] - read[:, :, c] @ s
        out.append(outer[:, :, c] @ s + inside[:, :, c] @ u)
        s = decay[:, :, c, -1, None, None] * s + kept[:, :, c].transpose(-1, -2) @ u
    return torch.stack(out, 2).reshape(b, h, -1, dv)[:, :, :n].transpose(1, 2), s


def _plain_sequences(state):
    case, lengths = state['case'], state['lengths']
    h, d, dv = case['heads'], case['d'], case['dv']
    names = ('q', 'k', 'v', 'g', 'beta')
    training = case['op'] == 'delta_train'
    leaves = [state[x].detach().float().requires_grad_(training) for x in names]
    rows = [_pad(x, lengths) for x in leaves] if lengths else leaves
    start = rows[0].new_zeros(rows[0].size(0), h, d, dv) if training else state['initial']
    out, final = _delta(*rows, d ** -.5, start)
    if lengths:
        out = _unpad(out, lengths)
    if not training:
        return out.bfloat16(), final
    grads = torch.autograd.grad(out, leaves, state['dout'].float())
    return [out.detach().bfloat16()] + [x.bfloat16() for x in grads]


def _plain_step(state):
    case = state['case']
    groups = case['heads'] // case['key_heads']
    q, k = (state[x].float().repeat_interleave(groups, 1) for x in ('q', 'k'))
    v, g, beta = state['v'].float(), state['g'].float(), state['beta'].float()
    pool, slots = state['state'], state['slots']
    live = slots >= 0 if slots is not None else None
    if live is not None:
        q, k, v, g, beta = (x[live] for x in (q, k, v, g, beta))
    s = pool[slots[live].long()] if live is not None else pool
    s = torch.exp(g)[..., None, None] * s
    u = beta[..., None] * (v - (s * k[..., None]).sum(-2))
    s = s + k[..., None] * u[..., None, :]
    o = (s * q[..., None]).sum(-2) * case['d'] ** -.5
    if live is None:
        pool.copy_(s)
        return o.bfloat16(), pool
    pool[slots[live].long()] = s
    out = torch.zeros_like(state['v'])
    out[live] = o.bfloat16()
    return out, pool


def _numbers(count, seed, site, device):
    """16-bit random numbers of `count` elements: eight to a Philox4x32-10 block, in integer tensor operations."""
    low = 0xFFFFFFFF
    block = torch.arange((count + 7) // 8, device=device, dtype=torch.int64)
    c = [block & low, torch.full_like(block, site), (seed[1] & low).expand_as(block), ((seed[1] >> 32) & low).expand_as(block)]
    key = [seed[0] & low, (seed[0] >> 32) & low]

    def wide(m, x):  # high and low words of a 32 x 32 bit product
        a, b = m * (x & 0xFFFF), m * (x >> 16)
        mid = (a >> 16) + (b & 0xFFFF)
        return ((b >> 16) + (mid >> 16)) & low, ((mid << 16) | (a & 0xFFFF)) & low

    for _ in range(10):
        h0, l0 = wide(0xD2511F53, c[0])
        h1, l1 = wide(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    words = torch.stack([half for x in c for half in (x & 0xFFFF, x >> 16)], -1)
    return words.reshape(-1)[:count]


def _plain_dropout(state):
    x, p = state['x'], state['case']['p']
    threshold = round(65536 * p)
    keep = (_numbers(x.numel(), state['seed'], state['site'], x.device) >= threshold).reshape(x.shape)
    factor = keep.float() * (65536 / (65536 - threshold))
    y = x.float() * factor
    if state['residual'] is not None:
        y = y + state['residual'].float()
    return y.to(x.dtype), (state['dy'].float() * factor).to(x.dtype)


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    op = state['case']['op']
    if not own:
        return _plain_dropout(state) if op == 'dropout' else _plain_step(state) if op == 'delta_step' else _plain_sequences(state)
    import dism_b200
    dism_b200.install_dropin()
    import flash_dism
    if op == 'dropout':
        x = state['x'].requires_grad_()
        y = flash_dism.dropout_add(x, state['residual'], state['case']['p'], state['seed'], site=state['site'])
        return y.detach(), torch.autograd.grad(y, x, state['dy'])[0]
    if op == 'delta_step':
        out = flash_dism.gated_delta_step(state['q'], state['k'], state['v'], state['g'], state['beta'], state['state'],
                                          slots=state['slots'])
        return out, state['state']
    operands = [state[x] for x in ('q', 'k', 'v', 'g', 'beta')]
    if op == 'delta_prefill':
        return flash_dism.gated_delta_rule(*operands, initial_state=state['initial'], output_final_state=True,
                                           cu_seqlens=state['cu_seqlens'])
    out = flash_dism.gated_delta_rule(*operands, cu_seqlens=state['cu_seqlens'])
    return [out.detach(), *torch.autograd.grad(out, operands, state['dout'])]


# ---- 64 bits -----------------------------------------------------------------------------------------------------
def _advance(s, k, v, a, beta):
    """One token on every head: the new state and the written value."""
    s = a[..., None, None] * s
    u = beta[..., None] * (v - torch.einsum('bhij,bhi->bhj', s, k))
    return s + torch.einsum('bhi,bhj->bhij', k, u), u


def _exact_sequences(case, state):
    """Token by token; the gradients by the adjoint of each token's step, states recomputed from marks every 64 tokens."""
    lengths, scale = state['lengths'], case['d'] ** -.5
    groups = case['heads'] // case['key_heads']
    get = lambda name: (_pad(state[name].detach(), lengths) if lengths else state[name].detach()).double()
    q, k = (get(x).repeat_interleave(groups, 2) for x in ('q', 'k'))
    v, g, beta = get('v'), get('g'), get('beta')
    b, n, h, dv = v.shape
    a = torch.exp(g)
    training = case['op'] == 'delta_train'
    s = q.new_zeros(b, h, case['d'], dv) if training else state['initial'].double()
    marks, out = [], torch.empty_like(v)
    for t in range(n):
        if training and t % 64 == 0:
            marks.append(s)
        s, _ = _advance(s, k[:, t], v[:, t], a[:, t], beta[:, t])
        out[:, t] = scale * torch.einsum('bhij,bhi->bhj', s, q[:, t])
    cut = (lambda x: _unpad(x, lengths)) if lengths else (lambda x: x)
    if not training:
        return cut(out), s
    do = get('dout')
    dq, dk, dvv, dg, dbeta = (torch.zeros_like(x) for x in (q, k, v, g, beta))
    ds = torch.zeros_like(s)
    for m in reversed(range(len(marks))):
        states, s = [], marks[m]
        for t in range(64 * m, min(n, 64 * m + 64)):
            states.append(s)
            s, _ = _advance(s, k[:, t], v[:, t], a[:, t], beta[:, t])
        states.append(s)
        for t in reversed(range(64 * m, min(n, 64 * m + 64))):
            before, after = states[t - 64 * m], states[t - 64 * m + 1]
            dq[:, t] = scale * torch.einsum('bhij,bhj->bhi', after, do[:, t])
            ds = ds + scale * torch.einsum('bhi,bhj->bhij', q[:, t], do[:, t])
            decayed = a[:, t][..., None, None] * before
            rest = v[:, t] - torch.einsum('bhij,bhi->bhj', decayed, k[:, t])
            du = torch.einsum('bhij,bhi->bhj', ds, k[:, t])
            drest = beta[:, t][..., None] * du
            dbeta[:, t] = (du * rest).sum(-1)
            dvv[:, t] = drest
            dk[:, t] = torch.einsum('bhij,bhj->bhi', ds, beta[:, t][..., None] * rest) - torch.einsum('bhij,bhj->bhi', decayed, drest)
            ddecayed = ds - torch.einsum('bhi,bhj->bhij', k[:, t], drest)
            dg[:, t] = (ddecayed * decayed).sum((-1, -2))
            ds = a[:, t][..., None, None] * ddecayed
    shared = lambda x: x.reshape(b, n, -1, groups, case['d']).sum(3)
    return [cut(x) for x in (out, shared(dq), shared(dk), dvv, dg, dbeta)]


def _exact_step(case, state):
    groups = case['heads'] // case['key_heads']
    pool, out = state['state'].double(), torch.zeros_like(state['v'], dtype=torch.float64)
    for row in range(case['batch']):
        slot = row if state['slots'] is None else int(state['slots'][row])
        if slot < 0:
            continue
        q, k = (state[x][row].double().repeat_interleave(groups, 0) for x in ('q', 'k'))
        s = pool[slot] * torch.exp(state['g'][row].double())[:, None, None]
        u = state['beta'][row].double()[:, None] * (state['v'][row].double() - (k[:, None] @ s)[:, 0])
        pool[slot] = s + k[:, :, None] * u[:, None]
        out[row] = (q[:, None] @ pool[slot])[:, 0] * case['d'] ** -.5
    return out, pool


def _exact_dropout(case, state):
    seed, offset = (int(x) for x in state['seed'])
    shift, word = np.uint64(32), np.uint64(0xFFFFFFFF)
    blocks = np.arange((state['x'].numel() + 7) // 8, dtype=np.uint64)
    x0, x1 = blocks & word, np.full_like(blocks, state['site'])
    x2, x3 = np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, (offset >> 32) & 0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for turn in range(10):
        first, second = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        r0, r1 = np.uint64((k0 + turn * 0x9E3779B9) & 0xFFFFFFFF), np.uint64((k1 + turn * 0xBB67AE85) & 0xFFFFFFFF)
        x0, x1, x2, x3 = (second >> shift) ^ x1 ^ r0, second & word, (first >> shift) ^ x3 ^ r1, first & word
    pieces = np.stack([x0, x1, x2, x3], 1).astype(np.uint32).view(np.uint16).reshape(-1)[:state['x'].numel()]
    threshold = round(65536 * case['p'])
    keep = torch.from_numpy(pieces.astype(np.int64) >= threshold).to('cuda').reshape(state['x'].shape)
    factor = 65536 / (65536 - threshold)
    y = torch.where(keep, state['x'].double() * factor, 0.)
    if state['residual'] is not None:
        y = y + state['residual'].double()
    return y, torch.where(keep, state['dy'].double() * factor, 0.)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case['op'] == 'dropout':
            return _exact_dropout(case, state)
        return _exact_step(case, state) if case['op'] == 'delta_step' else _exact_sequences(case, state)

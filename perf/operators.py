"""Measured cases of the decode-step operators: the append into a paged KV cache with the position
rotation on the way, the attention of one new token over that cache, and the log-probabilities of
given tokens with entropy and top alternatives, forward and with their gradient.

``run`` computes each operator in plain torch operations in 32 bits (``own`` false) or makes the calls
a user makes (``own`` true); ``exact`` is the operator's definition in 64 bits.
"""
import math

import torch

own = False

DEV = 'cuda'
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
BYTES = {'bf16': 2, 'fp16': 2, 'fp32': 4}
THETA = 1000000.0
# (query heads, KV heads) of the verify workloads, then generic ones: no sharing, a single KV head
HEADS = [(16, 2), (28, 4), (40, 8), (8, 8), (12, 1)]


# ---- cases -----------------------------------------------------------------------------------

def _append(name, batch, rows, q_heads, kv_heads, dim, rot, page, past, dtype, ragged, placed, interleaved=False):
    case = {'op': 'append', 'batch': batch, 'rows': rows, 'q_heads': q_heads, 'kv_heads': kv_heads, 'dim': dim,
            'rot': rot, 'page': page, 'past': past, 'dtype': dtype, 'ragged': ragged, 'placed': placed,
            'interleaved': interleaved}
    return case if name is None else {'name': name, **case}


def _attend(name, batch, q_heads, kv_heads, dim, page, lo, hi, idle, dtype):
    case = {'op': 'attend', 'batch': batch, 'q_heads': q_heads, 'kv_heads': kv_heads, 'dim': dim, 'page': page,
            'lo': lo, 'hi': hi, 'idle': idle, 'dtype': dtype}
    return case if name is None else {'name': name, **case}


def _logprobs(name, rows, vocab, dtype, top, temperature, skipped, grad):
    case = {'op': 'grad' if grad else 'logprobs', 'rows': rows, 'vocab': vocab, 'dtype': dtype, 'top': top,
            'temperature': temperature, 'skipped': skipped}
    return case if name is None else {'name': name, **case}


def listed():
    return [
        # one decode step of eight sequences: latency
        _append('append_decode_8', 8, 1, 16, 2, 128, 128, 16, 900, 'bf16', False, False),
        # one decode step of a full serving batch
        _append('append_decode_256', 256, 1, 28, 4, 128, 128, 64, 1500, 'bf16', False, False),
        # the tree rows of a verify round: positions by tree depth, not by cache slot
        _append('append_tree_64x61', 64, 61, 16, 2, 128, 128, 16, 1000, 'bf16', False, True),
        # prompts of unequal length entering the cache, right-padded to the longest
        _append('append_prefill_8x4001', 8, 4001, 40, 8, 128, 128, 32, 0, 'fp16', True, False),
        # one short sequence: latency
        _attend('attend_1x200', 1, 16, 2, 128, 16, 200, 200, 0, 'bf16'),
        # the decode step of a rollout batch, two slots idle
        _attend('attend_64x2048', 64, 16, 2, 128, 16, 256, 2048, 2, 'bf16'),
        # a large batch of longer sequences
        _attend('attend_256x6144', 256, 28, 4, 128, 64, 512, 6144, 0, 'fp16'),
        # two very long contexts: the cache's length has to be split
        _attend('attend_2x130000', 2, 40, 8, 128, 128, 100001, 130000, 0, 'bf16'),
        # the next-token scores of four sequences, ten alternatives each (32-bit logits)
        _logprobs('logprobs_4', 4, 151644, 'fp32', 10, 1.0, 0, False),
        # every tree row of a verify round: greedy sample, log-probability, ten alternatives
        _logprobs('logprobs_tree_3904', 3904, 151680, 'bf16', 10, 1.0, 61, False),
        # a micro-batch of a small vocabulary in 32 bits, forward and gradient
        _logprobs('grad_200', 200, 32000, 'fp32', 0, 0.8, 3, True),
        # the policy's log-probabilities and entropy of a training batch, with their gradient; rows of
        # this vocabulary start at odd multiples of eight bytes
        _logprobs('grad_4096', 4096, 151644, 'bf16', 0, 1.0, 300, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['append', 'attend', 'logprobs', 'grad'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    hq, hkv = rng.choice(HEADS)
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    if op == 'append':
        batch = _log(rng, 1, 300)
        rows = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 16000 // batch))
        rot = rng.choice([dim, dim, dim // 2])
        return _append(None, batch, rows, hq, hkv, dim, rot, page, _log(rng, 1, 1200), dtype, rng.random() < 0.5,
                       rng.random() < 0.3, rng.random() < 0.3)
    if op == 'attend':
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, 130000)
        # K and V together stay within 1 GB
        hi = max(1, min(hi, int(1e9 / (batch * hkv * dim * 2 * BYTES[dtype]))))
        return _attend(None, batch, hq, hkv, dim, page, max(1, int(hi * rng.uniform(0.05, 1.0))), hi,
                       rng.choice([0, 0, 1, batch // 8]) if batch > 1 else 0, dtype)
    vocab = rng.choice([32000, 151644, 151680, _log(rng, 1000, 160000)])
    rows = _log(rng, 1, max(1, min(4096, int(6e8 / vocab))) if dtype != 'fp32' else max(1, int(3e8 / vocab)))
    top = rng.choice([0, 1, 5, 10, 20]) if op == 'logprobs' else 0
    return _logprobs(None, rows, vocab, dtype, top, rng.choice([1.0, 0.7, 1.3]), rng.choice([0, rows // 10]),
                     op == 'grad')


# ---- inputs ----------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _spread(lo, hi, n, gen):
    """n whole numbers spread evenly over [lo, hi] (the same ones for every seed), in the seed's order."""
    values = torch.linspace(float(lo), float(hi), n, device=DEV, dtype=torch.float64).round().long()
    return values[torch.randperm(n, generator=gen, device=DEV)]


def _rotation(positions, rot):
    """(cos, sin) tables (positions, rot / 2) float32 of angles held in 64 bits."""
    freq = THETA ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _pages(batch, positions, case, dtype, gen):
    """Pools of more pages than are used, and the pages of each sequence in no order."""
    per = max(1, -(-positions // case['page']))
    total = batch * per + 3
    shape = (total, case['kv_heads'], case['page'], case['dim'])
    k = torch.randn(shape, device=DEV, dtype=dtype, generator=gen)
    v = torch.randn(shape, device=DEV, dtype=dtype, generator=gen)
    table = torch.randperm(total, generator=gen, device=DEV)[:batch * per].view(batch, per).contiguous()
    return k, v, table


def prepare(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case['dtype']]
    state = {'case': dict(case)}
    if case['op'] == 'append':
        batch, rows, dim = case['batch'], case['rows'], case['dim']
        state['k_pages'], state['v_pages'], state['table'] = _pages(batch, case['past'] + rows, case, dtype, gen)
        # projection outputs (batch, rows, heads * dim), viewed by head
        for name, heads in (('q', case['q_heads']), ('k', case['kv_heads']), ('v', case['kv_heads'])):
            x = torch.randn(batch, rows, heads * dim, device=DEV, dtype=dtype, generator=gen)
            state[name] = x.view(batch, rows, heads, dim).transpose(1, 2)
        state['starts'] = _spread(case['past'] // 2, case['past'], batch, gen)
        state['counts'] = _spread(max(1, rows // 4), rows, batch, gen) if case['ragged'] else None
        if case['placed']:  # a tree row's position is its sequence's length plus its depth
            depth = torch.randint(0, min(rows, 7), (batch, rows), device=DEV, generator=gen)
            state['positions'] = state['starts'][:, None] + depth
        else:
            state['positions'] = None
        state['cos'], state['sin'] = _rotation(case['past'] + rows, case['rot'])
    elif case['op'] == 'attend':
        batch, dim = case['batch'], case['dim']
        state['k_pages'], state['v_pages'], state['table'] = _pages(batch, case['hi'], case, dtype, gen)
        lengths = _spread(case['lo'], case['hi'], batch, gen)
        if case['idle']:
            lengths[torch.argsort(lengths)[:case['idle']]] = 0
        state['lengths'] = lengths
        state['scale'] = dim ** -0.5
        q = torch.randn(batch, 1, case['q_heads'] * dim, device=DEV, dtype=dtype, generator=gen)
        state['q'] = q.view(batch, 1, case['q_heads'], dim).transpose(1, 2)
    else:
        rows, vocab = case['rows'], case['vocab']
        logits = torch.empty(rows, vocab, device=DEV, dtype=dtype).normal_(0.0, 2.5, generator=gen)
        # a few tokens are forbidden in every row
        logits[:, torch.randint(0, vocab, (16,), device=DEV, generator=gen)] = -math.inf
        # the given token is a likely one: its row's best of 64 at random
        some = torch.randint(0, vocab, (rows, 64), device=DEV, generator=gen)
        best = logits.gather(1, some).float().argmax(1, keepdim=True)
        tokens = some.gather(1, best)[:, 0].contiguous()
        if case['skipped']:
            tokens[torch.randperm(rows, device=DEV, generator=gen)[:case['skipped']]] = -1
        state['logits'], state['tokens'] = logits, tokens
        if case['op'] == 'grad':
            logits.requires_grad_(True)
            state['g_logprob'] = torch.randn(rows, device=DEV, generator=gen) / rows
            state['g_entropy'] = torch.randn(rows, device=DEV, generator=gen) * (0.1 / rows)
    return state


# ---- the operators in plain torch operations -------------------------------------------------

def _rotate(x, cos, sin, rot, interleaved):
    """x (batch, heads, rows, dim) in 32 bits; cos / sin (batch, 1, rows, rot / 2)."""
    part, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_append(state):
    case = state['case']
    rows, page, rot = case['rows'], case['page'], case['rot']
    at = torch.arange(rows, device=DEV)
    slots = state['starts'][:, None] + at
    positions = slots if state['positions'] is None else state['positions']
    live = torch.ones_like(slots, dtype=torch.bool) if state['counts'] is None else at < state['counts'][:, None]
    cos, sin = state['cos'][positions][:, None], state['sin'][positions][:, None]
    q = _rotate(state['q'].float(), cos, sin, rot, case['interleaved'])
    q = torch.where(live[:, None, :, None], q, torch.zeros_like(q)).to(state['q'].dtype)
    k = _rotate(state['k'].float(), cos, sin, rot, case['interleaved']).to(state['k'].dtype)
    b, t = live.nonzero(as_tuple=True)
    where = state['table'][b, slots[b, t] // page]
    state['k_pages'][where, :, slots[b, t] % page] = k.transpose(1, 2)[b, t]
    state['v_pages'][where, :, slots[b, t] % page] = state['v'].transpose(1, 2)[b, t]
    return [q, state['k_pages'], state['v_pages']]


def _plain_attend(state):
    case = state['case']
    batch, hkv, dim, page = case['batch'], case['kv_heads'], case['dim'], case['page']
    group = case['q_heads'] // hkv
    table, lengths = state['table'], state['lengths']
    keys = state['k_pages'][table].transpose(1, 2).reshape(batch, hkv, -1, dim).float()
    q = state['q'].reshape(batch, hkv, group, dim).float()
    s = torch.matmul(q, keys.transpose(2, 3)) * state['scale']
    del keys
    seen = torch.arange(table.shape[1] * page, device=DEV) < lengths[:, None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    values = state['v_pages'][table].transpose(1, 2).reshape(batch, hkv, -1, dim).float()
    o = torch.matmul(p, values) / torch.where(total == 0, torch.ones_like(total), total)
    return o.reshape(batch, 1, case['q_heads'], dim).to(state['q'].dtype)


def _plain_statistics(logits, tokens, temperature):
    """Scaled log-probabilities of every entry (32 bits), those of the tokens, and the entropy."""
    z = logits.float() * (1.0 / temperature)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    logp = z - top - torch.log(e.sum(-1, keepdim=True))
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    chosen = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    live = tokens >= 0
    return logp, torch.where(live, chosen, torch.zeros_like(chosen)), torch.where(live, entropy,
                                                                                  torch.zeros_like(entropy)), live


def _top_ids(logits, k):
    """The k largest entries of each row, equal ones by the lower index: unique 64-bit keys of (value, index)."""
    x = logits.float() + 0.0
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, (bits ^ 0x7fffffff), bits)
    key = order * (1 << 32) + (0xffffffff - torch.arange(x.shape[1], device=x.device))
    return key.topk(k, dim=1).indices


def _plain_logprobs(state):
    case = state['case']
    logp, chosen, entropy, live = _plain_statistics(state['logits'], state['tokens'], case['temperature'])
    out = [chosen, entropy]
    if case['top']:
        ids = _top_ids(state['logits'], case['top'])
        values = logp.gather(1, ids)
        out += [torch.where(live[:, None], values, torch.zeros_like(values)),
                torch.where(live[:, None], ids, torch.full_like(ids, -1))]
    return out


def _plain_grad(state):
    case = state['case']
    logits, tokens = state['logits'].detach(), state['tokens']
    logp, chosen, entropy, live = _plain_statistics(logits, tokens, case['temperature'])
    a = torch.where(live, state['g_logprob'], torch.zeros_like(state['g_logprob']))
    h = torch.where(live, state['g_entropy'], torch.zeros_like(state['g_entropy']))
    p = torch.exp(logp)
    g = -p * (a[:, None] + h[:, None] * (torch.where(p > 0, logp, torch.zeros_like(logp)) + entropy[:, None]))
    del p, logp
    g.scatter_add_(1, tokens.clamp(min=0)[:, None], a[:, None])
    return [chosen, entropy, (g * (1.0 / case['temperature'])).to(logits.dtype)]


# ---- the same calls as a user makes them -----------------------------------------------------

def _own_append(state):
    from analysis_spec_b200.paged_cache import paged_append
    q = paged_append(state['k'], state['v'], state['k_pages'], state['v_pages'], state['table'], state['starts'],
                     counts=state['counts'], query=state['q'], rotation=(state['cos'], state['sin']),
                     positions=state['positions'], interleaved=state['case']['interleaved'])
    return [q, state['k_pages'], state['v_pages']]


def _own_attend(state):
    from analysis_spec_b200.paged_cache import paged_attention
    return paged_attention(state['q'], state['k_pages'], state['v_pages'], state['table'], state['lengths'],
                           state['scale'])


def _own_logprobs(state):
    from analysis_spec_b200.token_logprobs import token_logprobs
    case = state['case']
    r = token_logprobs(state['logits'], state['tokens'], top=case['top'], temperature=case['temperature'])
    return [r.logprobs, r.entropy] + ([r.top_logprobs, r.top_ids] if case['top'] else [])


def _own_grad(state):
    from analysis_spec_b200.token_logprobs import token_logprobs
    case = state['case']
    r = token_logprobs(state['logits'], state['tokens'], temperature=case['temperature'])
    grad, = torch.autograd.grad((r.logprobs, r.entropy), state['logits'], (state['g_logprob'], state['g_entropy']))
    return [r.logprobs.detach(), r.entropy.detach(), grad]


def run(state):
    op = state['case']['op']
    if own:
        return {'append': _own_append, 'attend': _own_attend, 'logprobs': _own_logprobs, 'grad': _own_grad}[op](state)
    return {'append': _plain_append, 'attend': _plain_attend, 'logprobs': _plain_logprobs,
            'grad': _plain_grad}[op](state)


# ---- what one pass cannot do without ---------------------------------------------------------

def _spread_host(lo, hi, n):
    return [int(round(v)) for v in torch.linspace(float(lo), float(hi), n, dtype=torch.float64).tolist()]


def work(case):
    size = BYTES[case['dtype']]
    if case['op'] == 'append':
        batch, rows, dim = case['batch'], case['rows'], case['dim']
        live = sum(_spread_host(max(1, rows // 4), rows, batch)) if case['ragged'] else batch * rows
        heads = case['q_heads'] + 2 * case['kv_heads']
        turned = case['q_heads'] + case['kv_heads']
        # K, V and Q of the live tokens read and written, the padded queries written, a table row a token
        moved = live * heads * dim * size * 2 + (batch * rows - live) * case['q_heads'] * dim * size
        moved += live * (case['rot'] * 4 + (8 if case['placed'] else 0)) + batch * 16
        return {'bytes': moved, 'flops': live * turned * case['rot'] * 3}
    if case['op'] == 'attend':
        lengths = sorted(_spread_host(case['lo'], case['hi'], case['batch']))
        keys = sum(lengths[case['idle']:])
        moved = 2 * keys * case['kv_heads'] * case['dim'] * size
        moved += 2 * case['batch'] * case['q_heads'] * case['dim'] * size
        moved += 8 * case['batch'] + 8 * sum(-(-n // case['page']) for n in lengths[case['idle']:])
        return {'bytes': moved, 'flops': 4 * keys * case['q_heads'] * case['dim']}
    rows, vocab = case['rows'], case['vocab']
    live = rows - case['skipped']
    if case['op'] == 'logprobs':
        return {'bytes': live * vocab * size + rows * (16 + 12 * case['top']), 'flops': 6 * live * vocab}
    # forward reads the logits, the gradient reads them again and writes every row
    return {'bytes': 2 * live * vocab * size + rows * vocab * size + rows * 32, 'flops': 12 * live * vocab}


# ---- the definitions in 64 bits --------------------------------------------------------------

def _exact_append(state):
    case = state['case']
    page, half = case['page'], case['rot'] // 2
    outs = [torch.zeros(state['q'].shape, device=DEV, dtype=torch.float64),
            state['k_pages'].double(), state['v_pages'].double()]
    for b in range(case['batch']):
        n = case['rows'] if state['counts'] is None else int(state['counts'][b])
        slot = int(state['starts'][b]) + torch.arange(n, device=DEV)
        place = slot if state['positions'] is None else state['positions'][b, :n]
        c, s = state['cos'][place].double(), state['sin'][place].double()
        turned = []
        for x in (state['q'][b, :, :n].double(), state['k'][b, :, :n].double()):
            y = x.clone()
            i = torch.arange(half, device=DEV)
            first, second = (2 * i, 2 * i + 1) if case['interleaved'] else (i, i + half)
            y[..., first] = x[..., first] * c - x[..., second] * s
            y[..., second] = x[..., second] * c + x[..., first] * s
            turned.append(y)
        outs[0][b, :, :n] = turned[0]
        to = state['table'][b][slot // page]
        outs[1][to, :, slot % page] = turned[1].transpose(0, 1)
        outs[2][to, :, slot % page] = state['v'][b, :, :n].double().transpose(0, 1)
    return outs


def _exact_attend(state):
    case = state['case']
    hkv, dim = case['kv_heads'], case['dim']
    out = torch.zeros(case['batch'], 1, case['q_heads'], dim, device=DEV, dtype=torch.float64)
    for b in range(case['batch']):
        n = int(state['lengths'][b])
        if n == 0:
            continue
        pages = state['table'][b][:-(-n // case['page'])]
        k = state['k_pages'][pages].permute(1, 0, 2, 3).reshape(hkv, -1, dim)[:, :n].double()
        v = state['v_pages'][pages].permute(1, 0, 2, 3).reshape(hkv, -1, dim)[:, :n].double()
        q = state['q'][b, :, 0].double().view(hkv, -1, dim)
        w = torch.softmax(torch.einsum('hgd,hnd->hgn', q, k) * state['scale'], dim=-1)
        out[b, 0] = torch.einsum('hgn,hnd->hgd', w, v).reshape(-1, dim)
    return out


def _exact_scores(state):
    case = state['case']
    logits, tokens = state['logits'].detach(), state['tokens']
    grad = case['op'] == 'grad'
    rows, step = case['rows'], max(1, int(1e8) // case['vocab'])
    chosen = torch.zeros(rows, device=DEV, dtype=torch.float64)
    entropy = torch.zeros_like(chosen)
    k = case['top']
    values = torch.zeros(rows, k, device=DEV, dtype=torch.float64)
    ids = torch.full((rows, k), -1, device=DEV, dtype=torch.long)
    g = torch.zeros(logits.shape, device=DEV, dtype=torch.float64) if grad else None
    for lo in range(0, rows, step):
        part = torch.arange(lo, min(rows, lo + step), device=DEV)
        part = part[tokens[part] >= 0]
        if not part.numel():
            continue
        z = logits[part].double() / case['temperature']
        lp = torch.log_softmax(z, dim=-1)
        chosen[part] = lp.gather(1, tokens[part][:, None])[:, 0]
        p = lp.exp()
        entropy[part] = torch.special.entr(p).sum(-1)
        if k:
            order = torch.sort(logits[part].double(), dim=1, descending=True, stable=True).indices[:, :k]
            ids[part], values[part] = order, lp.gather(1, order)
        if grad:
            a, h = state['g_logprob'][part].double()[:, None], state['g_entropy'][part].double()[:, None]
            d = -a * p - h * p * (torch.where(p > 0, lp, 0.0) + entropy[part][:, None])
            d[torch.arange(len(part), device=DEV), tokens[part]] += a[:, 0]
            g[part] = d / case['temperature']
    if grad:
        return [chosen, entropy, g]
    return [chosen, entropy] + ([values, ids] if k else [])


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'append':
        return _exact_append(state)
    return _exact_attend(state) if case['op'] == 'attend' else _exact_scores(state)

"""The paged key-value cache's operators, as cases that can be timed: append,
attention of new tokens, eviction by accumulated attention weight.

With `own` false, `run` computes a case in elementary torch operations in 32
bits; with `own` true it calls the entry points of `include/qwen_gpu.h`. Both
take what `prepare` gives. A cache's pool is [pages, KV heads, slots of a page,
head size] (whatever its strides), sequence s holds its position j in slot
j % page of page table[s, j // page]. E4M3 rows carry an exponent byte each
for key and value: the row's values are e4m3 * 2^(byte - 127).
"""
import ctypes
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
TYPES = {'f16': (0, torch.float16, 2), 'bf16': (1, torch.bfloat16, 2), 'e4m3': (2, torch.uint8, 1)}
GOLDEN = (math.sqrt(5) - 1) / 2

_loaded = {}


def _package():
    if 'package' not in _loaded:
        directory = ROOT / 'fpga-qwen_amd'
        spec = importlib.util.spec_from_file_location('fpga_qwen_amd', directory / '__init__.py',
                                                      submodule_search_locations=[str(directory)])
        module = importlib.util.module_from_spec(spec)
        sys.modules['fpga_qwen_amd'] = module
        spec.loader.exec_module(module)
        _loaded['package'] = module
        _loaded['library'] = module.load_library()
    return _loaded['package']


# ---- the cases ----

def _case(op, **more):
    """16 query heads on 8 KV heads of 128, pages of 16, FP16: the model's layer."""
    case = {'op': op, 'type': 'f16', 'kv_heads': 8, 'group': 2, 'head_dim': 128, 'page': 16, 'layout': 'head',
            'sequences': 1, 'shortest': 0, 'longest': 1, 'rows': 1, 'ragged': False, 'track': False}
    case.update(more)
    return case


def listed():
    return [
        # One layer's keys and values of a batched decode step.
        _case('append', name='append-8x1', sequences=8, shortest=2048, longest=2048),
        # A prompt's 512-row chunk behind a reused prefix of another 512.
        _case('append', name='append-512-bf16', type='bf16', page=64, longest=1024, shortest=1024, rows=512),
        # Prompts of several users at once, into an 8-bit cache with weights tracked.
        _case('append', name='append-ragged-e4m3', type='e4m3', page=64, sequences=24, shortest=40, longest=2000,
              rows=2000, ragged=True, track=True),
        # Decoding of one user after a short chat.
        _case('attention', name='attention-1x300', longest=300),
        # Eight sequences at the batch benchmark's length.
        _case('attention', name='attention-8x2048', sequences=8, shortest=2048, longest=2048),
        # Verification of a drafted token at the end of the context.
        _case('attention', name='attention-1x4096-pair', longest=4096, rows=2, page=64),
        # A decode step whose weights feed the eviction below.
        _case('attention', name='attention-8x1025-tracked', sequences=8, shortest=1025, longest=1025, track=True),
        # A full server: many users, lengths of all kinds.
        _case('attention', name='attention-64-ragged-bf16', type='bf16', page=64, sequences=64, shortest=1,
              longest=4096, layout='slot'),
        # Long documents in an 8-bit cache, wide groups, up to four drafted rows.
        _case('attention', name='attention-16-long-e4m3', type='e4m3', page=128, sequences=16, shortest=1000,
              longest=16384, group=4, rows=4, ragged=True),
        # One token too many in every sequence: each step of a bounded cache.
        _case('evict', name='evict-8x1025', sequences=8, shortest=1025, longest=1025, keep=1024, sinks=4,
              recent=256),
        # A prompt cut to a quarter once it has been read.
        _case('evict', name='evict-1x4001', longest=4001, keep=1000, sinks=4, recent=200),
        # The same for many users and an 8-bit cache.
        _case('evict', name='evict-32-ragged-e4m3', type='e4m3', page=64, sequences=32, shortest=100, longest=8192,
              keep=2048, sinks=16, recent=512),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['append', 'attention', 'attention', 'attention', 'evict'])
    kv_heads, group = rng.choice([(8, 2), (8, 2), (8, 1), (2, 7), (4, 4), (1, 16), (8, 5), (16, 1), (3, 3)])
    case = _case(op, type=rng.choice(['f16', 'bf16', 'e4m3']), kv_heads=kv_heads, group=group,
                 head_dim=rng.choice([64, 128, 128, 128, 256]), page=rng.choice([1, 7, 16, 16, 24, 32, 64, 128, 256]),
                 layout=rng.choice(['head', 'head', 'slot']), sequences=_spread(rng, 1, 64))
    # Slots of all sequences together: the cost of a case stays below the largest listed one's.
    most = 100_000 * 1024 // (kv_heads * case['head_dim'])
    case['longest'] = _spread(rng, 1, max(2, min(16384, most // case['sequences'])))
    case['shortest'] = rng.choice([0, 1, case['longest'] // 2, case['longest']])
    if op == 'attention':
        case['rows'] = rng.choice([1, 1, 1, 2, 3, 8])
        case['ragged'] = rng.random() < 0.5
        case['track'] = rng.random() < 0.4
    elif op == 'append':
        case['rows'] = rng.choice([1, 2, max(1, case['longest'] // 2), max(1, case['longest'])])
        case['ragged'] = rng.random() < 0.5
        case['track'] = rng.random() < 0.5
    else:
        longest = case['longest'] = max(2, case['longest'])
        case['shortest'] = min(case['shortest'], longest)
        case['keep'] = rng.choice([longest - 1, max(1, longest // 2), _spread(rng, 1, longest)])
        case['sinks'] = rng.randint(0, min(16, case['keep'] // 2))
        case['recent'] = rng.randint(0, case['keep'] - case['sinks'])
    return case


def _lengths(case):
    """Cached positions of each sequence, its new rows among them."""
    low, high = case['shortest'], case['longest']
    return [high if i == 0 else low + int((i * GOLDEN % 1) * (high - low + 1)) for i in range(case['sequences'])]


def _rows(case):
    """New rows of each sequence: all have the most, or from none to the most where they are ragged."""
    lengths = _lengths(case)
    if not case['ragged']:
        return [case['rows']] * len(lengths)
    return [case['rows'] if i == 0 else min(int((i * GOLDEN * 3 % 1) * (case['rows'] + 1)), n)
            for i, n in enumerate(lengths)]


# ---- what the caller holds ----

def _pool(case, pages, generator, scale):
    """A pool of keys or values, normal with the scale given (quantised rows: e4m3 of about unit exponent)."""
    shape = (pages, case['kv_heads'], case['page'], case['head_dim'])
    if case['layout'] == 'slot':
        shape = (shape[0], shape[2], shape[1], shape[3])
    real = torch.randn(shape, device='cuda', generator=generator)
    if case['type'] == 'e4m3':
        pool = (real * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        pool = (real * scale).to(TYPES[case['type']][1])
    return pool.permute(0, 2, 1, 3) if case['layout'] == 'slot' else pool


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(int(seed))
    heads, dim, page = case['kv_heads'], case['head_dim'], case['page']
    lengths, rows = _lengths(case), _rows(case)
    width = max(1, -(-max(lengths) // page))
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + 3
    order = torch.randperm(pages, device='cuda', generator=g).to(torch.int32)
    table = torch.zeros(len(lengths), width, dtype=torch.int32)
    order = order.cpu()
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    state = {'case': case, 'table': table.cuda(), 'lengths': torch.tensor(lengths, dtype=torch.int32, device='cuda'),
             'keys': _pool(case, pages, g, 1.0), 'values': _pool(case, pages, g, 0.64), 'pages': pages, 'width': width,
             'offsets': None, 'total': sum(rows), 'longest': max(lengths), 'exponents': None}
    if case['type'] == 'e4m3':
        state['exponents'] = torch.randint(119, 122, (pages, heads, page, 2), device='cuda', generator=g,
                                           dtype=torch.uint8)
    if case['ragged']:
        state['offsets'] = torch.tensor([0] + rows, device='cuda').cumsum(0).to(torch.int32)
    # Rows of a QKV projection; queries leave a norm, some heads attend more sharply than others.
    q_size, kv_size = heads * case['group'] * dim, heads * dim
    qkv = torch.randn(max(1, sum(rows)), q_size + 2 * kv_size, device='cuda', generator=g)
    sharp = 0.5 + 2.5 * torch.rand(heads * case['group'], 1, device='cuda', generator=g)
    qkv[:, :q_size] = (qkv[:, :q_size].view(-1, heads * case['group'], dim) * sharp).view(-1, q_size)
    state['q'], state['k'], state['v'] = qkv.split([q_size, kv_size, kv_size], 1)
    state['scale'] = dim ** -0.5
    state['out'] = torch.zeros(qkv.shape[0], q_size, device='cuda')
    if case['track'] or case['op'] == 'evict':
        slots = width * page
        gap = 100  # positions evicted earlier, behind the sinks
        state['seen'] = state['lengths'] + gap
        state['weights'] = torch.exp(torch.randn(len(lengths), heads, slots, device='cuda', generator=g))
        place = torch.arange(slots, device='cuda', dtype=torch.int32)
        place = torch.where(place < case.get('sinks', 0), place, place + gap)
        state['positions'] = place.expand(len(lengths), heads, slots).contiguous()
    if case['op'] == 'evict':
        state['new_lengths'] = torch.zeros_like(state['lengths'])
        state['new_weights'] = torch.zeros_like(state['weights'])
        state['new_positions'] = torch.zeros_like(state['positions'])
    return state


# ---- the calls ----

def _plan(state):
    """The descriptions of cache and batch that a program keeps, and the workspace (zeroed once)."""
    package, case = _package(), state['case']
    library = _loaded['library']
    pointer = lambda name: state[name].data_ptr() if state.get(name) is not None else None  # noqa: E731
    page_stride, head_stride, slot_stride, _ = state['keys'].stride()
    cache = package.PagedCache(keys=pointer('keys'), values=pointer('values'), exponents=pointer('exponents'),
                               page_stride=page_stride, head_stride=head_stride, slot_stride=slot_stride,
                               pages=state['pages'], page_size=case['page'], kv_heads=case['kv_heads'],
                               head_dim=case['head_dim'], type=TYPES[case['type']][0])
    batch = package.PagedBatch(table=pointer('table'), lengths=pointer('lengths'), offsets=pointer('offsets'),
                               seen=pointer('seen'), weights=pointer('weights'), positions=pointer('positions'),
                               track_stride=state['weights'].shape[2] if 'weights' in state else 0,
                               sequences=case['sequences'], table_stride=state['width'],
                               max_length=max(1, state['longest']), rows=case['rows'], total_rows=state['total'])
    bytes_ = ctypes.c_size_t()
    query_heads = case['kv_heads'] * case['group']
    if case['op'] != 'append':  # which takes none
        if library.qwen_gpu_op_paged_workspace(ctypes.byref(cache), ctypes.byref(batch), query_heads,
                                               ctypes.byref(bytes_)):
            raise RuntimeError(library.qwen_gpu_last_error().decode())
    state['workspace'] = torch.zeros(bytes_.value, dtype=torch.uint8, device='cuda')
    state['plan'] = library, cache, batch, ctypes.byref(cache), ctypes.byref(batch), query_heads
    return state['plan']


def _own(state):
    library, _, _, cache, batch, query_heads = state.get('plan') or _plan(state)
    case, work = state['case'], state['workspace']
    stream = torch.cuda.current_stream().cuda_stream
    if case['op'] == 'append':
        k, v = state['k'], state['v']
        failed = library.qwen_gpu_op_paged_append(cache, batch, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                                  stream)
    elif case['op'] == 'attention':
        q, out = state['q'], state['out']
        failed = library.qwen_gpu_op_paged_attention(cache, batch, q.data_ptr(), q.stride(0), query_heads,
                                                     state['scale'], out.data_ptr(), out.stride(0), work.data_ptr(),
                                                     work.numel(), stream)
    else:
        failed = library.qwen_gpu_op_paged_evict(cache, batch, case['keep'], case['sinks'], case['recent'],
                                                 state['new_lengths'].data_ptr(), state['new_weights'].data_ptr(),
                                                 state['new_positions'].data_ptr(), work.data_ptr(), work.numel(),
                                                 stream)
    if failed:
        raise RuntimeError(library.qwen_gpu_last_error().decode())


# ---- the plain forms ----

def _power(exponents):
    """2^(byte - 127)."""
    return (exponents.int() << 23).view(torch.float32)


def _new_rows(state):
    """Sequence, rank among its rows, and slot of every new row."""
    case, lengths = state['case'], state['lengths'].long()
    row = torch.arange(state['total'], device='cuda')
    if state['offsets'] is None:
        sequence = row // case['rows']
        count = torch.full_like(lengths, case['rows'])
        rank = row % case['rows']
    else:
        offsets = state['offsets'].long()
        sequence = torch.searchsorted(offsets, row, right=True) - 1
        count = offsets[1:] - offsets[:-1]
        rank = row - offsets[sequence]
    return sequence, rank, lengths[sequence] - count[sequence] + rank


def _append(state):
    case = state['case']
    heads, dim, page = case['kv_heads'], case['head_dim'], case['page']
    sequence, _, slot = _new_rows(state)
    live = slot >= 0
    sequence, slot = sequence[live], slot[live]
    where = state['table'][sequence, slot // page].long()
    inside = slot % page
    for name, pool, side in (('k', state['keys'], 0), ('v', state['values'], 1)):
        rows = state[name][:live.numel()][live].reshape(-1, heads, dim)
        if case['type'] == 'e4m3':
            # The smallest power of two that brings the row's largest magnitude to 448 or below.
            mantissa, power = torch.frexp(rows.abs().amax(-1))
            power = torch.where(mantissa <= 0.875, power - 9, power - 8)
            byte = torch.where(mantissa == 0, -126, power.clamp(-126, 127)) + 127
            state['exponents'][where, :, inside, side] = byte.to(torch.uint8)
            rows = (rows * _power(254 - byte)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        pool[where, :, inside] = rows.to(pool.dtype)
    if case['track']:
        state['weights'][sequence, :, slot] = 0
        gone = (state['seen'] - state['lengths'])[sequence]
        state['positions'][sequence, :, slot] = (slot + gone).to(torch.int32)[:, None]


def _cached(state, name, side):
    """Keys or values of all sequences in 32 bits: [sequences, KV heads, longest, head size]."""
    case = state['case']
    place = torch.arange(state['longest'], device='cuda')
    where, inside = state['table'][:, place // case['page']].long(), place % case['page']
    rows = state[name][where, :, inside.expand_as(where)]
    if case['type'] == 'e4m3':
        power = _power(state['exponents'][where, :, inside.expand_as(where), side])
        rows = rows.view(torch.float8_e4m3fn).float() * power[..., None]
    return rows.float().permute(0, 2, 1, 3)


def _attention(state):
    case, lengths = state['case'], state['lengths'].long()
    heads, group, dim, n = case['kv_heads'], case['group'], case['head_dim'], case['rows']
    if not state['longest'] or not state['total']:
        state['out'][:state['total']] = 0
        return
    sequence, rank, slot = _new_rows(state)
    q = torch.zeros(case['sequences'], n, heads, group, dim, device='cuda')
    q[sequence, rank] = state['q'][:state['total']].reshape(-1, heads, group, dim)
    sees = torch.zeros(case['sequences'], n, dtype=torch.long, device='cuda')
    sees[sequence, rank] = slot + 1
    q = q.permute(0, 2, 3, 1, 4).reshape(case['sequences'], heads, group * n, dim)
    keys = _cached(state, 'keys', 0)
    scores = torch.matmul(q, keys.transpose(2, 3)) * state['scale']
    del keys
    scores = scores.view(case['sequences'], heads, group, n, -1)
    hidden = torch.arange(state['longest'], device='cuda') >= sees[:, None, None, :, None]
    scores = scores.masked_fill(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p.view(case['sequences'], heads, group * n, -1), _cached(state, 'values', 1))
    out = out.view(case['sequences'], heads, group, n, dim).permute(0, 3, 1, 2, 4)
    state['out'][:state['total']] = out[sequence, rank].reshape(state['total'], -1)
    if case['track']:
        state['weights'][:, :, :state['longest']] += p.sum((2, 3))


def _evict(state):
    case, lengths = state['case'], state['lengths'].long()
    page, keep, slots = case['page'], case['keep'], state['weights'].shape[2]
    place = torch.arange(slots, device='cuda')
    inside = place < lengths[:, None, None]
    positions = state['positions']
    fixed = (positions < case['sinks']) | (positions >= state['seen'][:, None, None] - case['recent'])
    value = torch.where(fixed, math.inf, state['weights'])
    value = torch.where(inside, value, -math.inf)
    order = torch.sort(value, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(inside.expand_as(value)).scatter(2, order[..., :keep], True) & inside
    # The i-th kept slot from `keep` on moves into the i-th hole before it.
    hole, source = ~kept & inside & (place < keep), kept & (place >= keep)
    sequence, head, to = torch.nonzero(hole & (lengths > keep)[:, None, None], as_tuple=True)
    start = torch.nonzero(source, as_tuple=True)[2]
    new_lengths = lengths.clamp(max=keep)
    stays = place < new_lengths[:, None, None]
    for new, old in ((state['new_weights'], state['weights']), (state['new_positions'], state['positions'])):
        rows = old.clone()
        rows[sequence, head, to] = old[sequence, head, start]
        new.copy_(torch.where(stays, rows, new))
    state['new_lengths'].copy_(new_lengths)
    from_page, to_page = (state['table'][sequence, at // page].long() for at in (start, to))
    for pool in (state['keys'], state['values'], state['exponents']):
        if pool is not None:
            pool[to_page, head, to % page] = pool[from_page, head, start % page]


def run(state):
    op = state['case']['op']
    if own:
        _own(state)
    elif op == 'append':
        _append(state)
    elif op == 'attention':
        _attention(state)
    else:
        _evict(state)
    return _outputs(state, op)


def _outputs(state, op):
    if op == 'attention':
        return (state['out'], state['weights']) if state['case']['track'] else state['out']
    pools = [state['keys'], state['values']]
    if state['exponents'] is not None:
        pools = [pool.view(torch.float8_e4m3fn) for pool in pools] + [state['exponents']]
    if op == 'evict':
        return pools + [state['new_lengths'], state['new_weights'], state['new_positions']]
    return pools + ([state['weights'], state['positions']] if state['case']['track'] else [])


# ---- what a pass cannot do without ----

def work(case):
    heads, dim, size = case['kv_heads'], case['head_dim'], TYPES[case['type']][2]
    lengths, rows = _lengths(case), _rows(case)
    row = 2 * dim * size + (2 if case['type'] == 'e4m3' else 0)  # a position's key and value of one head
    tables = 4 * sum(1 + -(-n // case['page']) for n in lengths)
    if case['op'] == 'append':
        written = sum(min(r, n) for r, n in zip(rows, lengths))
        return {'bytes': written * heads * (8 * dim + row + (8 if case['track'] else 0)) + tables, 'flops': 0}
    if case['op'] == 'attention':
        read = sum(n for r, n in zip(rows, lengths) if r)
        pairs = sum(max(0, n - r + i + 1) for r, n in zip(rows, lengths) for i in range(r))
        return {'bytes': read * heads * (row + (8 if case['track'] else 0)) + 8 * sum(rows) * heads * case['group'] * dim
                + tables, 'flops': 4 * pairs * heads * case['group'] * dim}
    total, keep, recent, sinks = tables, case['keep'], case['recent'], case['sinks']
    for n in lengths:
        total += heads * 8 * (n + min(n, keep))
        if n > keep:
            last = min(recent, n - keep)
            share = (keep - sinks - recent) / max(1, n - sinks - recent)
            total += heads * 2 * row * (last + share * (n - keep - last))
    return {'bytes': total, 'flops': 0}


# ---- the same results in 64 bits ----

def _exact_cache(state, case, s, h, n, name, side):
    place = torch.arange(n, device='cuda')
    where, inside = state['table'][s, place // case['page']].long(), place % case['page']
    rows = state[name][where, h, inside]
    if case['type'] != 'e4m3':
        return rows.double()
    return rows.view(torch.float8_e4m3fn).double() * \
        torch.pow(2.0, state['exponents'][where, h, inside, side].double() - 127)[:, None]


def _exact_attention(state, case):
    dim, group = case['head_dim'], case['group']
    out = torch.zeros(state['out'].shape, dtype=torch.float64, device='cuda')
    weights = state['weights'].double() if case['track'] else None
    first = 0
    for s, (n, count) in enumerate(zip(_lengths(case), _rows(case))):
        for h in range(case['kv_heads']):
            if not n or not count:
                continue
            keys, values = (_exact_cache(state, case, s, h, n, *x) for x in (('keys', 0), ('values', 1)))
            for g in range(group):
                column = (h * group + g) * dim
                q = state['q'][first:first + count, column:column + dim].double()
                scores = q @ keys.T.contiguous() * dim ** -0.5
                last = n - count + torch.arange(count, device='cuda')[:, None]
                unseen = torch.arange(n, device='cuda')[None] > last
                p = torch.nan_to_num(torch.softmax(scores.masked_fill(unseen, -math.inf), 1))
                out[first:first + count, column:column + dim] = p @ values
                if weights is not None:
                    weights[s, h, :n] += p.sum(0)
        first += count
    return (out, weights) if case['track'] else out


def _exact_append(state, case):
    dim, first = case['head_dim'], 0
    pools = [state['keys'].clone(), state['values'].clone()]
    exponents = state['exponents'].clone() if state['exponents'] is not None else None
    for s, (n, count) in enumerate(zip(_lengths(case), _rows(case))):
        skipped = max(0, count - n)
        place = torch.arange(n - count + skipped, n, device='cuda')
        where, inside = state['table'][s, place // case['page']].long(), place % case['page']
        for side, (name, pool) in enumerate(zip('kv', pools)):
            rows = state[name][first + skipped:first + count].double().reshape(place.numel(), case['kv_heads'], dim)
            if exponents is not None:
                power = torch.ceil(torch.log2(rows.abs().amax(-1) / 448)).clamp(-126, 127)
                exponents[where, :, inside, side] = (power + 127).to(torch.uint8)
                rows = (rows / torch.pow(2.0, power)[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
            pool[where, :, inside] = rows.to(pool.dtype)
        if case['track']:
            state['weights'][s, :, n - count + skipped:n] = 0
            state['positions'][s, :, n - count + skipped:n] = \
                place.to(torch.int32) + (state['seen'][s] - state['lengths'][s])
        first += count
    if exponents is not None:
        pools = [pool.view(torch.float8_e4m3fn) for pool in pools] + [exponents]
    return pools + ([state['weights'], state['positions']] if case['track'] else [])


def _exact_evict(state, case):
    keep, page = case['keep'], case['page']
    pools = [state['keys'].clone(), state['values'].clone()]
    if state['exponents'] is not None:
        pools.append(state['exponents'].clone())
    lengths = _lengths(case)
    new_weights, new_positions = (torch.zeros_like(state[x]) for x in ('weights', 'positions'))
    for s, n in enumerate(lengths):
        for h in range(case['kv_heads']):
            weights, positions = state['weights'][s, h, :n], state['positions'][s, h, :n]
            come = list(range(n))
            if n > keep:
                seen = int(state['seen'][s])
                listed_weights, listed_positions = weights.tolist(), positions.tolist()
                rank = sorted(range(n), key=lambda i: (-math.inf if listed_positions[i] < case['sinks'] or
                                                       listed_positions[i] >= seen - case['recent']
                                                       else -listed_weights[i], i))[:keep]
                chosen = set(rank)
                late = sorted(i for i in chosen if i >= keep)
                holes = [i for i in range(keep) if i not in chosen]
                come = come[:keep]
                for to, start in zip(holes, late):
                    come[to] = start
            come = torch.tensor(come, dtype=torch.long, device='cuda')
            new_weights[s, h, :come.numel()] = weights[come]
            new_positions[s, h, :come.numel()] = positions[come]
            to = torch.arange(come.numel(), device='cuda')
            for pool in pools:
                old = pool[state['table'][s, come // page].long(), h, come % page]
                pool[state['table'][s, to // page].long(), h, to % page] = old
    if state['exponents'] is not None:
        pools = [pool.view(torch.float8_e4m3fn) for pool in pools[:2]] + pools[2:]
    new_lengths = torch.tensor([min(n, keep) for n in lengths], dtype=torch.int32, device='cuda')
    return pools + [new_lengths, new_weights, new_positions]


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'attention':
        if sum(_lengths(case)) * case['kv_heads'] * case['group'] * max(1, case['rows']) > 60_000_000:
            return None
        return _exact_attention(state, case)
    return _exact_append(state, case) if case['op'] == 'append' else _exact_evict(state, case)

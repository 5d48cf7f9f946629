"""What a server's step needs around a paged key-value cache, as cases that can
be timed: pages reserved and rows mapped on the GPU, heads normed and rotated
by position, attention of a batch that shares a prefix, drafted tokens verified
against the target's probabilities.

With `own` false, `run` computes a case in elementary torch operations; with
`own` true it calls the entry points of `include/qwen_gpu.h`. Both take what
`prepare` gives. Pools are [pages, KV heads, slots of a page, head size]
(whatever their strides), sequence s holds its position j in slot j % page of
page table[s, j // page]. E4M3 rows carry an exponent byte each for key and
value: the row's values are e4m3 * 2^(byte - 127).
"""
import ctypes
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
CACHE_TYPES = {'f16': (0, torch.float16, 2), 'bf16': (1, torch.bfloat16, 2), 'e4m3': (2, torch.uint8, 1)}
TYPES = {'f32': (0, torch.float32, 4), 'f16': (1, torch.float16, 2), 'bf16': (2, torch.bfloat16, 2)}
GOLDEN = (math.sqrt(5) - 1) / 2

_loaded = {}


def _package():
    if 'package' not in _loaded:
        package = sys.modules.get('fpga_qwen_amd')
        if package is None:
            directory = ROOT / 'fpga-qwen_amd'
            spec = importlib.util.spec_from_file_location('fpga_qwen_amd', directory / '__init__.py',
                                                          submodule_search_locations=[str(directory)])
            package = importlib.util.module_from_spec(spec)
            sys.modules['fpga_qwen_amd'] = package
            spec.loader.exec_module(package)
        _loaded['package'] = package
        _loaded['library'] = package.load_library()
    return _loaded['package']


# ---- the cases ----

def _rotate(**more):
    """16 query and 8 key heads of 128, FP32, normed, whole heads turned by halves: the model's layer."""
    return {'op': 'rotate', 'type': 'f32', 'kv_heads': 8, 'group': 2, 'head_dim': 128, 'dims': 128,
            'interleaved': False, 'norm': True, 'scaled': False, 'base': 1e6, 'rows': 1, 'far': 4096,
            'padding': 0, **more}


def _reserve(**more):
    return {'op': 'reserve', 'sequences': 1, 'page': 16, 'longest': 1, 'rows': 1, 'mode': 'step', 'scarce': False, **more}


def _shared(**more):
    """16 query heads on 8 KV heads of 128, pages of 16, FP16: the model's layer."""
    return {'op': 'shared', 'type': 'f16', 'kv_heads': 8, 'group': 2, 'head_dim': 128, 'page': 16, 'layout': 'head',
            'groups': 1, 'sequences': 1, 'prefix': 1, 'shortest': 1, 'longest': 1, 'rows': 1, 'ragged': False, **more}


def _verify(**more):
    return {'op': 'verify', 'type': 'f32', 'vocabulary': 151936, 'sequences': 1, 'rows': 2, 'ragged': False,
            'draft': True, 'greedy': False, 'filtered': False, **more}


def listed():
    return [
        # A decode step of eight sequences.
        _rotate(name='rotate-8', rows=8),
        # A prompt's chunk.
        _rotate(name='rotate-512', rows=512, far=1024),
        # Chunks of many long documents: half of each head turned, positions scaled far beyond the trained ones.
        _rotate(name='rotate-8191-bf16', type='bf16', group=4, dims=64, interleaved=True, scaled=True, rows=8191,
                far=1 << 20, base=1e4),
        # A decode step's bookkeeping on a full server.
        _reserve(name='reserve-64-step', sequences=64, longest=4096),
        # Prompts of many users admitted beside others that decode, verify and end, with too few pages for all.
        _reserve(name='reserve-1000-mixed', sequences=1000, longest=4096, rows=1000, mode='mixed', scarce=True),
        # The batch benchmark's last step: 8 users behind one prefix.
        _shared(name='shared-8x512', sequences=8, prefix=512, shortest=1600, longest=1663),
        # A full server behind one long system prompt.
        _shared(name='shared-64x8192', sequences=64, prefix=8192, shortest=1, longest=500),
        # Four assistants with prompts of their own, drafted tokens verified.
        _shared(name='shared-4x24x4000-bf16', type='bf16', page=64, layout='slot', groups=4, sequences=96, prefix=4000,
                shortest=1, longest=1500, rows=5, ragged=True),
        # Questions about one very long document in an 8-bit cache.
        _shared(name='shared-32x65000-e4m3', type='e4m3', page=128, group=4, sequences=32, prefix=65000, shortest=10,
                longest=300),
        # One user's guessed token (from an n-gram: no probabilities of its own).
        _verify(name='verify-1x2', draft=False),
        # Eight users, four tokens of a small model each.
        _verify(name='verify-8x5', sequences=8, rows=5, greedy=True),
        # A full server, BF16 logits, drafts of 0 to 6 tokens, filtered by the largest logits.
        _verify(name='verify-64x7-bf16', type='bf16', sequences=64, rows=7, ragged=True, filtered=True),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['rotate', 'reserve', 'shared', 'shared', 'verify'])
    heads = [(8, 2), (8, 2), (8, 1), (2, 7), (4, 4), (1, 16), (8, 5), (16, 1), (3, 3)]
    if op == 'rotate':
        kv_heads, group = rng.choice(heads)
        dim = rng.choice([32, 64, 80, 96, 128, 128, 128, 192, 256])
        most = 8191 * 40 * 128 // ((kv_heads * (group + 1)) * dim)
        case = _rotate(type=rng.choice(['f32', 'f32', 'f16', 'bf16']), kv_heads=kv_heads, group=group, head_dim=dim,
                       dims=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                       norm=rng.random() < 0.7, scaled=rng.random() < 0.4, base=rng.choice([1e4, 5e5, 1e6]),
                       far=_spread(rng, 1, 1 << 23))
        # Twice the bytes in FP32 cost twice as much.
        case['rows'] = _spread(rng, 1, most // 2 if case['type'] == 'f32' else most)
        case['padding'] = rng.choice([0, 0, 4, 7])
        return case
    if op == 'reserve':
        case = _reserve(sequences=_spread(rng, 1, 4096), page=rng.choice([1, 7, 16, 16, 24, 64, 256]),
                        mode=rng.choice(['step', 'mixed', 'mixed', 'admit']), scarce=rng.random() < 0.4)
        case['longest'] = _spread(rng, 1, min(8192, (4_000_000 if case['page'] > 8 else 500_000) // case['sequences']))
        case['rows'] = 1 if case['mode'] == 'step' else _spread(rng, 1, max(1, min(case['longest'],
                                                                                    250_000 // case['sequences'])))
        return case
    if op == 'shared':
        kv_heads, group = rng.choice(heads)
        case = _shared(type=rng.choice(['f16', 'bf16', 'e4m3']), kv_heads=kv_heads, group=group,
                       head_dim=rng.choice([64, 128, 128, 128, 256]), page=rng.choice([1, 7, 16, 16, 24, 64, 128]),
                       layout=rng.choice(['head', 'head', 'slot']), groups=rng.choice([1, 1, 1, 2, 5]))
        case['sequences'] = _spread(rng, case['groups'], 64)
        # Slots of a group's prefix and of all rests together: the cost stays below the largest listed case's.
        most = 60_000 * 1024 // (kv_heads * case['head_dim'])
        case['prefix'] = _spread(rng, 1, min(32768, most // case['groups']))
        case['longest'] = _spread(rng, 1, max(2, min(4096, most // case['sequences'])))
        case['shortest'] = rng.choice([1, 1 + case['longest'] // 2, case['longest']])
        case['rows'] = min(rng.choice([1, 1, 1, 2, 4, 7]), case['longest'])
        case['ragged'] = rng.random() < 0.5
        return case
    case = _verify(type=rng.choice(['f32', 'f32', 'f16', 'bf16']), vocabulary=rng.choice(
        [151936, 151936, 32000, _spread(rng, 2, 260_000), _spread(rng, 2, 260_000)]), rows=rng.choice([1, 2, 2, 4, 5, 8]),
        ragged=rng.random() < 0.5, draft=rng.random() < 0.6, greedy=rng.random() < 0.4, filtered=rng.random() < 0.3)
    case['sequences'] = _spread(rng, 1, max(1, min(64, 30_000_000 // (case['vocabulary'] * case['rows']))))
    return case


def _lengths(case):
    """Cached positions of each sequence: those behind the prefix, the new rows among them (shared); those of the step
    before (reserve)."""
    low, high = case.get('shortest', 0), case['longest']
    return [high if i == 0 else low + int((i * GOLDEN % 1) * (high - low + 1)) for i in range(case['sequences'])]


def _rows(case):
    """New rows of each sequence: all have the most, or up to the most where they are ragged."""
    if not case['ragged']:
        return [case['rows']] * case['sequences']
    low = 1 if case['op'] == 'verify' else 0
    return [case['rows'] if i == 0 else low + int((i * GOLDEN * 3 % 1) * (case['rows'] + 1 - low))
            for i in range(case['sequences'])]


def _fitting(case):
    """Lengths behind the prefix and new rows that fit into them."""
    lengths = _lengths(case)
    return lengths, [min(n, r) for n, r in zip(lengths, _rows(case))]


def _groups(case):
    """First sequence of each group, and their number behind the last."""
    n, groups = case['sequences'], case['groups']
    return [g * n // groups for g in range(groups)] + [n]


def _changes(case):
    """Lengths, new rows (below zero: rows taken back) and pages held of each sequence."""
    lengths, changes, held = _lengths(case), [], []
    for i, n in enumerate(lengths):
        kind = int((i * GOLDEN * 5 % 1) * 10)
        if case['mode'] == 'step':
            change = 1
        elif case['mode'] == 'admit':
            n, change = 0, max(1, int((i * GOLDEN * 7 % 1) * (case['rows'] + 1)))
        elif kind < 3:  # a new prompt
            n, change = 0, max(1, int((i * GOLDEN * 7 % 1) * (case['rows'] + 1)))
        elif kind < 4:  # one that has ended
            change = -n
        elif kind < 6:  # refused drafts
            change = -min(n, 3)
        else:
            change = kind - 5
        lengths[i] = n
        changes.append(change)
        held.append(-(-n // case['page']))
    return lengths, changes, held


# ---- what the caller holds ----

def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _frequencies(case):
    """Radians a position of each turned pair; scaled: short wavelengths as they are, long ones sixteen times slower,
    between them a ramp by the turns within 4096 positions."""
    dims = case['dims']
    plain = [case['base'] ** (-2 * i / dims) for i in range(dims // 2)]
    if not case['scaled']:
        return plain, 1.0
    share = [min(1.0, max(0.0, (4096 * f / (2 * math.pi) - 1) / 31)) for f in plain]
    return [f * s + f / 16 * (1 - s) for f, s in zip(plain, share)], 0.1 * math.log(16) + 1


def _prepare_rotate(case, g):
    heads, dim, rows = case['kv_heads'], case['head_dim'], case['rows']
    q_heads, dtype = heads * case['group'], TYPES[case['type']][1]
    # Rows of a projection: queries, keys, values, and whatever the caller pads them with.
    width = (q_heads + 2 * heads) * dim + case['padding']
    qkv = torch.randn(rows, width, device='cuda', generator=g)
    qkv *= torch.exp(0.5 * torch.randn(1, width, device='cuda', generator=g))
    qkv = qkv.to(dtype)
    frequencies, magnitude = _frequencies(case)
    state = {'q': qkv[:, :q_heads * dim].view(rows, q_heads, dim),
             'k': qkv[:, q_heads * dim:(q_heads + heads) * dim].view(rows, heads, dim),
             'frequencies': torch.tensor(frequencies, dtype=torch.float64, device='cuda'), 'magnitude': magnitude,
             'epsilon': 1e-6,
             'positions': torch.randint(0, case['far'], (rows,), device='cuda', generator=g, dtype=torch.int32),
             'q_out': torch.zeros(rows, q_heads, dim, dtype=dtype, device='cuda'),
             'k_out': torch.zeros(rows, heads, dim, dtype=dtype, device='cuda'), 'q_norm': None, 'k_norm': None}
    if case['norm']:
        for name in ('q_norm', 'k_norm'):
            state[name] = 1 + 0.3 * torch.randn(dim, device='cuda', generator=g)
    return state


def _prepare_reserve(case, g):
    lengths, changes, held = _changes(case)
    page, n = case['page'], case['sequences']
    wanted = [max(0, -(-max(0, a + c) // page) - h) for a, c, h in zip(lengths, changes, held)]
    spare = sum(wanted) // 2 if case['scarce'] else sum(wanted) + 5
    pages = sum(held) + spare + 1
    width = max(max(h + w for h, w in zip(held, wanted)), 1) + 1
    order = torch.randperm(pages, device='cuda', generator=g).to(torch.int32).cpu()
    table, at = torch.full((n, width), -1, dtype=torch.int32), 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    free = torch.full((pages,), -1, dtype=torch.int32)
    free[:spare] = order[at:at + spare]
    room = max(1, sum(max(0, c) for c in changes))
    # Rows of the text that an earlier eviction took from some of the sequences.
    gone = torch.randint(0, 3, (n,), device='cuda', generator=g, dtype=torch.int32) * 100
    state = {'table': table.cuda(), 'free': free.cuda(), 'held': _ints(held), 'free_count': _ints([spare]),
             'lengths': _ints(lengths), 'changes': _ints(changes), 'pages': pages, 'width': width, 'room': room}
    state['seen'] = state['lengths'] + gone
    for name, count in (('new_lengths', n), ('new_seen', n), ('new_held', n), ('new_free_count', 1), ('offsets', n + 1),
                        ('row_sequence', room), ('row_position', room)):
        state[name] = torch.zeros(count, dtype=torch.int32, device='cuda')
    state['row_slot'] = torch.zeros(room, dtype=torch.int64, device='cuda')
    return state


def _pool(case, pages, generator, scale):
    """A pool of keys or values, normal with the scale given (quantised rows: e4m3 of about unit exponent)."""
    shape = (pages, case['kv_heads'], case['page'], case['head_dim'])
    if case['layout'] == 'slot':
        shape = (shape[0], shape[2], shape[1], shape[3])
    real = torch.randn(shape, device='cuda', generator=generator)
    if case['type'] == 'e4m3':
        pool = (real * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        pool = (real * scale).to(CACHE_TYPES[case['type']][1])
    return pool.permute(0, 2, 1, 3) if case['layout'] == 'slot' else pool


def _prepare_shared(case, g):
    heads, dim, page, prefix = case['kv_heads'], case['head_dim'], case['page'], case['prefix']
    rests, rows = _fitting(case)
    firsts = _groups(case)
    # A prefix' last page that it does not fill is every sequence's own copy.
    whole = prefix // page
    lengths = [prefix + n for n in rests]
    used = [-(-n // page) - whole for n in lengths]
    pages = sum(used) + whole * case['groups'] + 3
    width = max(-(-n // page) for n in lengths)
    order = torch.randperm(pages, device='cuda', generator=g).to(torch.int32).cpu()
    table, at = torch.zeros(case['sequences'], width, dtype=torch.int32), 0
    for first, last in zip(firsts, firsts[1:]):
        table[first:last, :whole] = order[at:at + whole]
        at += whole
    for s, n in enumerate(used):
        table[s, whole:whole + n] = order[at:at + n]
        at += n
    state = {'table': table.cuda(), 'lengths': _ints(lengths), 'keys': _pool(case, pages, g, 1.0),
             'values': _pool(case, pages, g, 0.64), 'pages': pages, 'width': width, 'total': sum(rows),
             'longest': max(lengths), 'exponents': None, 'offsets': None,
             'prefixes': _ints([prefix] * case['groups']), 'firsts': _ints(firsts), 'scale': dim ** -0.5}
    if case['type'] == 'e4m3':
        state['exponents'] = torch.randint(119, 122, (pages, heads, page, 2), device='cuda', generator=g,
                                           dtype=torch.uint8)
    if any(r != case['rows'] for r in rows):
        state['offsets'] = torch.tensor([0] + rows, device='cuda').cumsum(0).to(torch.int32)
    if prefix % page:  # the copies
        for first, last in zip(firsts, firsts[1:]):
            to, start = state['table'][first + 1:last, whole].long(), int(table[first, whole])
            for pool in (state['keys'], state['values'], state['exponents']):
                if pool is not None and to.numel():
                    pool[to, :, :prefix % page] = pool[start, :, :prefix % page].clone()
    # Rows of a QKV projection; queries leave a norm, some heads attend more sharply than others.
    q_size, kv_size = heads * case['group'] * dim, heads * dim
    qkv = torch.randn(max(1, sum(rows)), q_size + 2 * kv_size, device='cuda', generator=g)
    sharp = 0.5 + 2.5 * torch.rand(heads * case['group'], 1, device='cuda', generator=g)
    state['q'] = (qkv[:, :q_size].view(-1, heads * case['group'], dim) * sharp).view(-1, q_size)
    qkv[:, :q_size] = state['q']
    state['q'] = qkv[:, :q_size]
    state['out'] = torch.zeros(qkv.shape[0], q_size, device='cuda')
    return state


def _prepare_verify(case, g):
    n, vocabulary, rows = case['sequences'], case['vocabulary'], _rows(case)
    total, firsts = sum(rows), [0]
    for r in rows:
        firsts.append(firsts[-1] + r)
    sequence = torch.repeat_interleave(torch.arange(n, device='cuda'), torch.tensor(rows, device='cuda'))
    # Some tokens are common everywhere, the rest go by the row.
    logits = 2.5 * torch.randn(total, vocabulary, device='cuda', generator=g)
    logits += 2 * torch.randn(vocabulary, device='cuda', generator=g)
    temperature = 0.5 + torch.rand(n, device='cuda', generator=g)
    if case['greedy']:
        temperature[::2] = 0
    heat = torch.where(temperature > 0, temperature, 1.0)[sequence, None]
    guess = logits + torch.randn(total, vocabulary, device='cuda', generator=g)
    if case['filtered']:
        kept = min(vocabulary, 50)
        logits = torch.where(logits >= logits.topk(kept, -1).values[:, -1:], logits, -math.inf)
        guess = torch.where(guess >= guess.topk(kept, -1).values[:, -1:], guess, -math.inf)
    guess = torch.softmax(guess / heat, -1)
    noise = -torch.log(torch.rand(total, vocabulary, device='cuda', generator=g).clamp(1e-30))
    drawn = (guess / noise).argmax(-1)
    tokens = torch.randint(0, vocabulary, (total,), device='cuda', generator=g)
    if not case['draft']:  # an n-gram is right at times
        hit = torch.rand(total, device='cuda', generator=g) < 0.5
        drawn = torch.where(hit, logits.argmax(-1), tokens)
    tokens[1:] = drawn[:-1]  # row r's guess is row r + 1's token
    return {'logits': logits.to(TYPES[case['type']][1]), 'draft': guess.contiguous() if case['draft'] else None,
            'tokens': tokens.to(torch.int32), 'temperature': temperature, 'sequence': sequence,
            'offsets': _ints(firsts) if case['ragged'] else None, 'firsts': torch.tensor(firsts, device='cuda'),
            'accept': torch.rand(total, device='cuda', generator=g), 'sample': torch.rand(n, device='cuda', generator=g),
            'total': total, 'accepted': torch.zeros(n, dtype=torch.int32, device='cuda'),
            'next': torch.zeros(n, dtype=torch.int32, device='cuda'),
            'back': torch.zeros(n, dtype=torch.int32, device='cuda')}


def prepare(case, seed):
    make = {'rotate': _prepare_rotate, 'reserve': _prepare_reserve, 'shared': _prepare_shared, 'verify': _prepare_verify}
    state = make[case['op']](case, _generator(seed))
    state['case'] = case
    return state


# ---- the calls ----

def _pointer(state, name):
    return state[name].data_ptr() if state.get(name) is not None else None


def _check(failed):
    if failed:
        raise RuntimeError(_loaded['library'].qwen_gpu_last_error().decode())


def _workspace(call, *given):
    need = ctypes.c_size_t()
    _check(call(*given, ctypes.byref(need)))
    return torch.zeros(max(1, need.value), dtype=torch.uint8, device='cuda')


def _plan(state):
    """The descriptions that a program keeps, and the workspace."""
    package, case = _package(), state['case']
    library, at = _loaded['library'], lambda name: _pointer(state, name)
    if case['op'] == 'rotate':
        rotary = package.Rotary(frequencies=at('frequencies'), dims=case['dims'], layout=int(case['interleaved']),
                                head_dim=case['head_dim'], type=TYPES[case['type']][0], magnitude=state['magnitude'],
                                epsilon=state['epsilon'])
        sides = []
        for name in 'qk':
            rows, out = state[name], state[f'{name}_out']
            sides.append(package.RotaryHeads(rows=rows.data_ptr(), out=out.data_ptr(), norm=at(f'{name}_norm'),
                                             row_stride=rows.stride(0), head_stride=rows.stride(1),
                                             out_row_stride=out.stride(0), out_head_stride=out.stride(1),
                                             heads=rows.shape[1]))
        state['plan'] = [rotary] + sides
    elif case['op'] == 'reserve':
        pool = package.PagedPool(table=at('table'), free_pages=at('free'), held=at('held'), free_count=at('free_count'),
                                 shared=None, pages=state['pages'], page_size=case['page'],
                                 sequences=case['sequences'], table_stride=state['width'])
        growth = package.PagedGrowth(lengths=at('lengths'), seen=at('seen'), changes=at('changes'),
                                     new_lengths=at('new_lengths'), new_seen=at('new_seen'), new_held=at('new_held'),
                                     new_free_count=at('new_free_count'), offsets=at('offsets'),
                                     row_sequences=at('row_sequence'), row_positions=at('row_position'),
                                     row_slots=at('row_slot'), total_rows=state['room'])
        state['plan'] = [pool, growth]
    elif case['op'] == 'shared':
        page_stride, head_stride, slot_stride, _ = state['keys'].stride()
        cache = package.PagedCache(keys=at('keys'), values=at('values'), exponents=at('exponents'),
                                   page_stride=page_stride, head_stride=head_stride, slot_stride=slot_stride,
                                   pages=state['pages'], page_size=case['page'], kv_heads=case['kv_heads'],
                                   head_dim=case['head_dim'], type=CACHE_TYPES[case['type']][0])
        batch = package.PagedBatch(table=at('table'), lengths=at('lengths'), offsets=at('offsets'),
                                   sequences=case['sequences'], table_stride=state['width'],
                                   max_length=state['longest'], rows=case['rows'], total_rows=state['total'])
        prefix = package.PagedPrefix(lengths=at('prefixes'), offsets=at('firsts'), groups=case['groups'],
                                     max_length=case['prefix'], max_rest=case['longest'])
        state['plan'] = [cache, batch, prefix]
        heads = case['kv_heads'] * case['group']
        state['workspace'] = _workspace(library.qwen_gpu_op_paged_shared_workspace, *map(ctypes.byref, state['plan']), heads)
    else:
        draft = package.Draft(logits=at('logits'), draft=at('draft'), tokens=at('tokens'), offsets=at('offsets'),
                              temperature=at('temperature'), accept=at('accept'), sample=at('sample'),
                              logit_stride=state['logits'].stride(0),
                              draft_stride=state['draft'].stride(0) if case['draft'] else 0,
                              type=TYPES[case['type']][0], vocabulary=case['vocabulary'], sequences=case['sequences'],
                              rows=case['rows'], total_rows=state['total'])
        state['plan'] = [draft]
        state['workspace'] = _workspace(library.qwen_gpu_op_verify_workspace, ctypes.byref(draft))
    state['given'] = [ctypes.byref(x) for x in state['plan']]
    return library


def _own(state):
    library = _loaded['library'] if 'given' in state else _plan(state)
    case, given = state['case'], state['given']
    stream = torch.cuda.current_stream().cuda_stream
    if case['op'] == 'rotate':
        failed = library.qwen_gpu_op_rotate(*given, state['positions'].data_ptr(), case['rows'], stream)
    elif case['op'] == 'reserve':
        failed = library.qwen_gpu_op_paged_reserve(*given, stream)
    elif case['op'] == 'shared':
        q, out, work = state['q'], state['out'], state['workspace']
        failed = library.qwen_gpu_op_paged_attention_shared(*given, q.data_ptr(), q.stride(0),
                                                            case['kv_heads'] * case['group'], state['scale'],
                                                            out.data_ptr(), out.stride(0), work.data_ptr(), work.numel(),
                                                            stream)
    else:
        work = state['workspace']
        failed = library.qwen_gpu_op_verify_draft(*given, state['accepted'].data_ptr(), state['next'].data_ptr(),
                                                  state['back'].data_ptr(), work.data_ptr(), work.numel(), stream)
    _check(failed)


# ---- the plain forms ----

def _plain_rotate(state):
    case = state['case']
    # Angles of far positions do not fit 32 bits.
    angle = state['positions'].double()[:, None] * state['frequencies']
    turn = [(f(angle).float() * state['magnitude'])[:, None] for f in (torch.cos, torch.sin)]
    pairs = case['dims'] // 2
    for name in 'qk':
        x = state[name].float()
        if case['norm']:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + state['epsilon']) * state[f'{name}_norm']
        out = x.clone()
        one, two = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if case['interleaved'] else
                    (slice(0, pairs), slice(pairs, 2 * pairs)))
        out[..., one] = x[..., one] * turn[0] - x[..., two] * turn[1]
        out[..., two] = x[..., two] * turn[0] + x[..., one] * turn[1]
        state[f'{name}_out'].copy_(out)


def _plain_reserve(state):
    page, room, width, pages = state['case']['page'], state['room'], state['width'], state['pages']
    lengths, held = state['lengths'].long(), state['held'].long()
    most = width * page
    changes = torch.maximum(state['changes'].long(), -lengths)
    changes = torch.where(lengths + changes > most, 0, changes)
    needed = (lengths + changes + page - 1) // page
    surplus, need = (held - needed).clamp(min=0), (needed - held).clamp(min=0)
    table, free = state['table'], state['free']
    entry = torch.arange(width, device='cuda')
    # Pages given back, behind the free ones: by sequence, then by place in the table.
    given = (entry >= needed[:, None]) & (entry < held[:, None])
    back = table[given]
    count = state['free_count'].long()
    free[count + torch.arange(back.numel(), device='cuda')] = back
    count = count + surplus.sum()
    has_pages = (need == 0) | (need.cumsum(0) <= count)
    rows = torch.where(has_pages, changes.clamp(min=0), 0)
    upto = rows.cumsum(0)
    granted = has_pages & (upto <= room)
    rows = torch.where(granted, rows, 0)
    changes = torch.where(granted, changes, changes.clamp(max=0))
    taken = torch.where(granted, need, 0)
    # Pages taken from the end of the free ones, in the same order.
    wanted = (entry >= held[:, None]) & (entry < (held + taken)[:, None])
    rank = torch.arange(wanted.numel(), device='cuda')[:int(taken.sum())]
    table[wanted] = free[count - 1 - rank]
    new_lengths, new_seen = lengths + changes, state['seen'] + changes
    state['new_lengths'].copy_(new_lengths)
    state['new_seen'].copy_(new_seen)
    state['new_held'].copy_(held - surplus + taken)
    state['new_free_count'].copy_(count - taken.sum())
    state['offsets'][0] = 0
    state['offsets'][1:] = rows.cumsum(0)
    offsets = state['offsets'].long()
    row = torch.arange(room, device='cuda')
    live = row < offsets[-1]
    sequence = (torch.searchsorted(offsets, row, right=True) - 1).clamp(max=lengths.numel() - 1)
    behind = offsets[sequence + 1] - row
    slot = (new_lengths[sequence] - behind).clamp(min=0)
    where = table[sequence, (slot // page).clamp(max=width - 1)].long()
    state['row_sequence'].copy_(torch.where(live, sequence, -1))
    state['row_position'].copy_(torch.where(live, new_seen[sequence] - behind, -1))
    state['row_slot'].copy_(torch.where(live, where * page + slot % page, -1))


def _cached(state, sequence, first, last, name, side):
    """Keys or values of a sequence's positions first .. last - 1 in 32 bits: [KV heads, positions, head size]."""
    case = state['case']
    place = torch.arange(first, last, device='cuda')
    where, inside = state['table'][sequence, place // case['page']].long(), place % case['page']
    rows = state[name][where, :, inside]
    if case['type'] == 'e4m3':
        power = (state['exponents'][where, :, inside, side].int() << 23).view(torch.float32)
        rows = rows.view(torch.float8_e4m3fn).float() * power[..., None]
    return rows.float().transpose(0, 1)


def _plain_shared(state):
    case = state['case']
    heads, group, dim, prefix = case['kv_heads'], case['group'], case['head_dim'], case['prefix']
    rests, rows = _fitting(case)
    firsts, at = _groups(case), [0]
    for r in rows:
        at.append(at[-1] + r)
    for first, last in zip(firsts, firsts[1:]):
        count = at[last] - at[first]
        if not count:
            continue
        q = state['q'][at[first]:at[last]].view(count, heads, group, dim).permute(1, 2, 0, 3).contiguous() * state['scale']
        # The prefix for all of the group's rows at once.
        keys = _cached(state, first, 0, prefix, 'keys', 0)
        scores = torch.matmul(q.view(heads, group * count, dim), keys.transpose(1, 2).contiguous())
        top = scores.amax(-1)
        p = torch.exp(scores - top[..., None])
        total = p.sum(-1).view(heads, group, count)
        out = torch.matmul(p, _cached(state, first, 0, prefix, 'values', 1)).view(heads, group, count, dim)
        top = top.view(heads, group, count)
        del keys, scores, p
        for s in range(first, last):
            n, r = rests[s], rows[s]
            if not r:
                continue
            mine = slice(at[s] - at[first], at[s + 1] - at[first])
            keys = _cached(state, s, prefix, prefix + n, 'keys', 0)
            scores = torch.matmul(q[:, :, mine].reshape(heads, group * r, dim), keys.transpose(1, 2).contiguous())
            scores = scores.view(heads, group, r, n)
            hidden = torch.arange(n, device='cuda') > n - r + torch.arange(r, device='cuda')[:, None]
            scores = scores.masked_fill(hidden, -math.inf)
            high = torch.maximum(scores.amax(-1), top[:, :, mine])
            p, shrink = torch.exp(scores - high[..., None]), torch.exp(top[:, :, mine] - high)
            values = _cached(state, s, prefix, prefix + n, 'values', 1)
            rest = torch.matmul(p.view(heads, group * r, n), values).view(heads, group, r, dim)
            rest += out[:, :, mine] * shrink[..., None]
            rest /= (p.sum(-1) + total[:, :, mine] * shrink)[..., None]
            state['out'][at[s]:at[s + 1]] = rest.permute(2, 0, 1, 3).reshape(r, -1)


def _plain_verify(state):
    case = state['case']
    vocabulary, most, total = case['vocabulary'], case['rows'], state['total']
    sequence, firsts = state['sequence'], state['firsts']
    # Which token a number falls on is a matter of borders: 64 bits.
    x = state['logits'].double()
    top = x.amax(-1, keepdim=True)
    heat = state['temperature'][sequence].double()[:, None]
    place = torch.arange(vocabulary, device='cuda')
    best = torch.where(x == top, place, vocabulary).amin(-1, keepdim=True)
    weight = torch.where(heat > 0, torch.exp((x - top) / torch.where(heat > 0, heat, 1.0)), (place == best).double())
    del x
    p = weight / weight.sum(-1, keepdim=True)
    row = torch.arange(total, device='cuda')
    last = row == firsts[sequence + 1] - 1
    token = state['tokens'][(row + 1).clamp(max=total - 1)].long()[:, None]
    q = state['draft'].gather(1, token)[:, 0].double() if case['draft'] else 1.0
    fits = (state['accept'].double() * q < p.gather(1, token)[:, 0]) & ~last
    run = torch.zeros(case['sequences'], most + 1, dtype=torch.bool, device='cuda')
    run[sequence, row - firsts[sequence]] = fits
    accepted = run.long().cumprod(1).sum(1)
    drawn = firsts[:-1] + accepted
    refused = ~last[drawn]
    share = p[drawn]
    if case['draft']:
        other = state['draft'][drawn].double()
    else:
        other = (place == token[drawn]).double()
    rest = torch.where(refused[:, None], (share - other).clamp(min=0), share)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, share)
    upto = rest.cumsum(-1)
    chosen = (upto <= state['sample'].double()[:, None] * upto[:, -1:]).sum(-1)
    highest = torch.where(rest > 0, place, -1).amax(-1)
    state['accepted'].copy_(accepted)
    state['next'].copy_(torch.minimum(chosen, highest))
    state['back'].copy_(accepted - (firsts[1:] - firsts[:-1] - 1))


def run(state):
    op = state['case']['op']
    if own:
        _own(state)
    else:
        {'rotate': _plain_rotate, 'reserve': _plain_reserve, 'shared': _plain_shared, 'verify': _plain_verify}[op](state)
    return [state[name] for name in OUTPUTS[op]]


OUTPUTS = {'rotate': ['q_out', 'k_out'], 'shared': ['out'], 'verify': ['accepted', 'next', 'back'],
           'reserve': ['table', 'free', 'new_lengths', 'new_seen', 'new_held', 'new_free_count', 'offsets',
                       'row_sequence', 'row_position', 'row_slot']}


# ---- what a pass cannot do without ----

def work(case):
    if case['op'] == 'rotate':
        heads, size = case['kv_heads'] * (case['group'] + 1), TYPES[case['type']][2]
        norms = 8 * case['head_dim'] if case['norm'] else 0
        return {'bytes': case['rows'] * (2 * size * heads * case['head_dim'] + 4) + 4 * case['dims'] + norms,
                'flops': case['rows'] * heads * (3 * case['dims'] + (4 * case['head_dim'] if case['norm'] else 0))}
    if case['op'] == 'reserve':
        lengths, changes, held = _changes(case)
        pages = sum(abs(-(-max(0, n + c) // case['page']) - h) for n, c, h in zip(lengths, changes, held))
        rows = sum(max(0, c) for c in changes)
        # Where pages are scarce, half of them are there.
        share = 0.5 if case['scarce'] else 1
        return {'bytes': 32 * case['sequences'] + int(share * (8 * pages + 16 * rows)), 'flops': 0}
    if case['op'] == 'shared':
        heads, dim, size = case['kv_heads'], case['head_dim'], CACHE_TYPES[case['type']][2]
        rests, rows = _fitting(case)
        row = 2 * dim * size + (2 if case['type'] == 'e4m3' else 0)
        read = case['groups'] * case['prefix'] + sum(n for n, r in zip(rests, rows) if r)
        pairs = sum(case['prefix'] + n - r + i + 1 for n, r in zip(rests, rows) for i in range(r))
        return {'bytes': read * (heads * row + 4 // case['page']) + 8 * sum(rows) * heads * case['group'] * dim,
                'flops': 4 * pairs * heads * case['group'] * dim}
    total = sum(_rows(case))
    drafts = 4 * case['vocabulary'] * case['sequences'] if case['draft'] and case['rows'] > 1 else 0
    return {'bytes': total * case['vocabulary'] * TYPES[case['type']][2] + drafts, 'flops': 4 * total * case['vocabulary']}


# ---- the same results in 64 bits ----

def _exact_rotate(state, case):
    dim, dims = case['head_dim'], case['dims']
    turn = torch.polar(torch.full((case['rows'], dims // 2), float(state['magnitude']), dtype=torch.float64, device='cuda'),
                       torch.outer(state['positions'].double(), state['frequencies']))[:, None]
    results = []
    for name in 'qk':
        x = state[name].double()
        if case['norm']:
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / dim + state['epsilon']) * state[f'{name}_norm'].double()
        head = x[..., :dims]
        if case['interleaved']:
            turned = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
        else:
            turned = torch.complex(head[..., :dims // 2], head[..., dims // 2:]) * turn
            turned = torch.cat((turned.real, turned.imag), -1)
        results.append(torch.cat((turned, x[..., dims:]), -1))
    return results


def _exact_reserve(state, case):
    page, room, width = case['page'], state['room'], state['width']
    table, free = state['table'].cpu().tolist(), state['free'].cpu().tolist()
    lengths, seen, held, changes = (state[x].cpu().tolist() for x in ('lengths', 'seen', 'held', 'changes'))
    count = int(state['free_count'])
    wished, short, full = [], False, False
    for s, n in enumerate(lengths):
        change = max(changes[s], -n)
        wished.append(0 if n + change > width * page else change)
        pages = -(-(n + wished[s]) // page)
        while held[s] > pages:  # from the first one that is given back on
            back = table[s][pages:held[s]]
            free[count:count + len(back)] = back
            count += len(back)
            held[s] = pages
    before, offsets, maps = list(held), [0], [[], [], []]
    for s, n in enumerate(lengths):
        need = -(-(n + wished[s]) // page) - before[s]
        short = short or need > count
        change = wished[s]
        if need > 0 and short:
            change = min(0, change)
        if change > 0 and (full or offsets[-1] + change > room):
            full, change = True, 0
        if change > 0:
            for _ in range(max(0, need)):
                count -= 1
                table[s][held[s]] = free[count]
                held[s] += 1
        for i in range(max(0, change)):
            maps[0].append(s)
            maps[1].append(seen[s] + i)
            maps[2].append(table[s][(n + i) // page] * page + (n + i) % page)
        lengths[s] += change
        seen[s] += change
        offsets.append(offsets[-1] + max(0, change))
    maps = [m + [-1] * (room - len(m)) for m in maps]
    results = [table, free, lengths, seen, held, [count], offsets] + maps
    return [torch.tensor(r, dtype=torch.int32, device='cuda') for r in results[:-1]] + [torch.tensor(results[-1], device='cuda')]


def _exact_cache(state, case, s, h, n, name, side):
    place = torch.arange(n, device='cuda')
    where, inside = state['table'][s, place // case['page']].long(), place % case['page']
    rows = state[name][where, h, inside]
    if case['type'] != 'e4m3':
        return rows.double()
    return rows.view(torch.float8_e4m3fn).double() * \
        torch.pow(2.0, state['exponents'][where, h, inside, side].double() - 127)[:, None]


def _exact_shared(state, case):
    """Every sequence by itself, as if it shared nothing."""
    dim, group = case['head_dim'], case['group']
    rests, rows = _fitting(case)
    out, first = torch.zeros(state['out'].shape, dtype=torch.float64, device='cuda'), 0
    for s, (rest, count) in enumerate(zip(rests, rows)):
        n = case['prefix'] + rest
        for h in range(case['kv_heads']):
            if not count:
                continue
            keys, values = (_exact_cache(state, case, s, h, n, *x) for x in (('keys', 0), ('values', 1)))
            for g in range(group):
                column = (h * group + g) * dim
                q = state['q'][first:first + count, column:column + dim].double()
                scores = q @ keys.T.contiguous() * dim ** -0.5
                unseen = torch.arange(n, device='cuda')[None] > n - count + torch.arange(count, device='cuda')[:, None]
                out[first:first + count, column:column + dim] = \
                    torch.softmax(scores.masked_fill(unseen, -math.inf), 1) @ values
        first += count
    return [out]


def _exact_verify(state, case):
    results, first = [[], [], []], 0
    for s, count in enumerate(_rows(case)):
        heat = float(state['temperature'][s])

        def distribution(row):
            x = state['logits'][row].double()
            if heat > 0:
                return torch.softmax(x / heat, 0)
            only = torch.zeros_like(x)
            only[int(torch.nonzero(x == x.max())[0])] = 1
            return only

        def guessed(row):
            if case['draft']:
                return state['draft'][row].double()
            only = torch.zeros(case['vocabulary'], dtype=torch.float64, device='cuda')
            only[int(state['tokens'][row + 1])] = 1
            return only

        accepted, weights = 0, None
        while accepted < count - 1:
            row = first + accepted
            token, p, q = int(state['tokens'][row + 1]), distribution(row), guessed(row)
            if not float(state['accept'][row]) * float(q[token]) < float(p[token]):
                weights = torch.clamp(p - q, min=0)
                if not float(weights.sum()) > 0:
                    weights = p
                break
            accepted += 1
        if weights is None:
            weights = distribution(first + count - 1)
        possible = torch.nonzero(weights)[:, 0]
        upto = torch.cumsum(weights[possible], 0)
        found = int(torch.searchsorted(upto, float(state['sample'][s]) * upto[-1], right=True))
        results[0].append(accepted)
        results[1].append(int(possible[min(found, possible.numel() - 1)]))
        results[2].append(accepted - (count - 1))
        first += count
    return [_ints(r) for r in results]


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'shared':
        rests, rows = _fitting(case)
        if sum(case['prefix'] + n for n, r in zip(rests, rows) if r) * case['kv_heads'] * case['group'] * \
                (case['rows'] + 4) > 400_000_000:
            return None
        return _exact_shared(state, case)
    return {'rotate': _exact_rotate, 'reserve': _exact_reserve, 'verify': _exact_verify}[case['op']](state, case)

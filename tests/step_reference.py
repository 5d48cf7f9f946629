"""What a step needs around a paged cache, in plain NumPy and 64 bits: heads
normed and turned, pages and rows of a step, drafted tokens verified."""
from fractions import Fraction

import numpy as np

import paged_reference

U = 2.0 ** -24
TYPES = ('f32', 'f16', 'bf16')
HALF_STEP = {'f32': 0.0, 'f16': 2.0 ** -11, 'bf16': 2.0 ** -8}  # of the last rounding, relative
SMALLEST = {'f32': 2.0 ** -126, 'f16': 2.0 ** -25, 'bf16': 2.0 ** -126}  # half a step of the smallest numbers, at most


def encode(x, kind):
    """FP32 values as an array of the type's raw values."""
    return np.asarray(x, np.float32) if kind == 'f32' else paged_reference.to_bits(x, kind)


def decode(raw, kind):
    return raw.astype(np.float64) if kind == 'f32' else paged_reference.from_bits(raw, kind)


def rotate(x, positions, frequencies, interleaved, magnitude, norm, epsilon, kind='f32'):
    """x [rows, heads, head_dim] in 64 bits; returns (result, tolerance).

    Tolerance, to first order with u = 2^-24: a head's squares are summed in FP32
    by at most 16 in a lane and 6 steps over lanes (22 roundings of positive
    terms, halved by the root), with the mean, epsilon, root, quotient and two
    products 8 more: a normed channel is off by 19 u at most. Sine and cosine:
    the angle's rounding at an eighth of a turn or less 0.8 u, the functions 2
    units in the last place (4 u), the magnitude 1 u; the products and their sum
    2 u. So a turned channel is off by 27 u of magnitude * (|a| + |b|)."""
    x = np.asarray(x, np.float64)
    if norm is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + epsilon) * np.asarray(norm, np.float64)
    out, size = x.copy(), np.abs(x)
    half = len(frequencies)
    # 2^24 positions and more leave 64 bits' angles 2^-29 of a turn off.
    turns = np.asarray(positions, np.longdouble)[:, None] * np.asarray(frequencies, np.longdouble)
    angle = np.asarray(np.fmod(turns, 2 * np.longdouble('3.14159265358979323846264338327950288')), np.float64)[:, None]
    cos, sin = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    one, two = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else
                (slice(0, half), slice(half, 2 * half)))
    a, b = x[..., one], x[..., two]
    out[..., one], out[..., two] = a * cos - b * sin, b * cos + a * sin
    size[..., one] = size[..., two] = abs(magnitude) * (np.abs(a) + np.abs(b))
    return out, 27 * U * size + HALF_STEP[kind] * np.abs(out) * (1 + 27 * U) + SMALLEST[kind]


def reserve(table, held, free, lengths, changes, page_size, pages, room, seen=None, shared=None):
    """One sequence after the other; the same dictionary as the package's paged_reserve."""
    table, free = np.array(table, np.int64), [int(x) for x in free]
    n, width = table.shape
    most = min(width * page_size, 1 << 30)
    lengths = [min(max(int(x), 0), most) for x in lengths]
    held = [min(max(int(x), 0), width) for x in held]
    text = [int(x) for x in (lengths if seen is None else seen)]
    wished = []
    for s in range(n):
        change = max(int(changes[s]), -lengths[s])
        change = 0 if lengths[s] + change > most else change
        wished.append(change)
    before = list(held)
    for s in range(n):
        needed = -(-(lengths[s] + wished[s]) // page_size)
        fixed = 0 if shared is None else min(max(int(shared[s]), 0), held[s])
        for entry in range(max(needed, fixed), held[s]):
            if len(free) < pages:
                free.append(int(table[s, entry]))
        held[s] = min(held[s], max(needed, fixed))
    offsets, maps = [0], {'sequences': [], 'positions': [], 'slots': []}
    short = full = False
    wished_rows = 0  # of the sequences that have pages, whether there is room for them or not
    left = len(free)
    for s in range(n):
        change = wished[s]
        need = max(0, -(-(lengths[s] + change) // page_size) - before[s]) if change > 0 else 0
        short = short or need > left
        if change > 0 and need and short:
            change = 0
        elif change > 0:
            wished_rows += change
            full = full or wished_rows > room
            if full:
                change = 0
            else:
                left -= need
                for entry in range(before[s], before[s] + need):
                    table[s, entry] = free.pop()
                held[s] = max(held[s], before[s] + need) if need else held[s]
        for i in range(max(0, change)):
            j = lengths[s] + i
            page = int(table[s, j // page_size])
            maps['sequences'].append(s)
            maps['positions'].append(text[s] + i)
            maps['slots'].append(page * page_size + j % page_size if 0 <= page < pages else -1)
        lengths[s] += change
        text[s] += change
        offsets.append(offsets[-1] + max(0, change))
    for name, values in maps.items():
        maps[name] = np.asarray(values + [-1] * (room - len(values)), np.int64)
    return dict(table=table, held=np.asarray(held), free=np.asarray(free, np.int64), lengths=np.asarray(lengths),
                seen=np.asarray(text), offsets=np.asarray(offsets), **maps)


def probabilities(logits, temperature):
    """A row's, all 0 where no token is left."""
    x = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float64))
    top = x.max()
    if top == -np.inf:
        return np.zeros(x.size)
    if not temperature > 0:
        return (np.arange(x.size) == np.argmax(x)).astype(np.float64)
    if top == np.inf:
        p = (x == np.inf).astype(np.float64)
    else:
        with np.errstate(invalid='ignore'):
            p = np.where(x == -np.inf, 0.0, np.exp((x - top) / np.float64(temperature)))
    return p / p.sum()


def cumulated(weights):
    """Exact sums of few weights, so that a number on a border falls where the definition has it; those of many in 64 bits."""
    if weights.size > 64:
        return np.cumsum(weights)
    upto = [Fraction(0)]
    for w in weights:
        upto.append(upto[-1] + Fraction(float(w)))
    return upto[1:]


def verify(logits, tokens, accept, sample, draft=None, counts=None, temperature=None):
    """(accepted, next) of each sequence."""
    n = len(sample)
    counts = [len(logits) // n] * n if counts is None else counts
    accepted, following, first = [], [], 0
    for s, count in enumerate(counts):
        heat = 1.0 if temperature is None else temperature[s]
        done, weights = 0, np.zeros(1)
        for i in range(count):
            row = first + i
            p = probabilities(logits[row], heat)
            weights = p
            if i + 1 == count:
                break
            token = int(tokens[row + 1])
            inside = 0 <= token < p.size
            if draft is not None:
                q = np.fmax(np.asarray(draft[row], np.float64), 0)
                q = np.where(np.isnan(q), 0, q)
            else:
                q = (np.arange(p.size) == token).astype(np.float64)
            if inside and float(accept[row]) * q[token] < p[token]:
                done += 1
                continue
            weights = np.maximum(p - q, 0)
            weights = weights if weights.sum() > 0 else p
            break
        accepted.append(done)
        if not weights.sum() > 0:
            following.append(-1)
        else:
            upto = cumulated(weights)
            if np.isfinite(sample[s]):
                target = Fraction(float(sample[s])) * upto[-1] if weights.size <= 64 else float(sample[s]) * upto[-1]
                over = np.flatnonzero([w > 0 and u > target for u, w in zip(upto, weights)])
            else:
                over = np.zeros(0)
            following.append(int(over[0]) if over.size else int(np.flatnonzero(weights > 0)[-1]))
        first += count
    return np.asarray(accepted), np.asarray(following)

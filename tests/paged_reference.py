"""The paged cache's operators in plain NumPy and 64 bits, on the raw bytes that
the device holds: conversions of the three cache types, where rows lie, and
what append, attention and eviction make of them."""
import numpy as np

TYPES = {'f16': (0, np.uint16), 'bf16': (1, np.uint16), 'e4m3': (2, np.uint8)}


def _e4m3_values():
    code = np.arange(256)
    exponent, fraction = (code >> 3) & 15, (code & 7).astype(np.float64)
    value = np.where(exponent == 0, fraction / 8 * 2.0 ** -6, (1 + fraction / 8) * 2.0 ** (exponent - 7.0))
    value[(code & 127) == 127] = np.nan
    return np.where(code >= 128, -value, value)


E4M3 = _e4m3_values()
_FINITE = E4M3[:127]  # rising, 0 .. 448


def to_e4m3(x):
    """Nearest code, ties to even ones; what lies beyond 448 (464 and above) or is NaN gives NaN."""
    x = np.asarray(x, np.float64)
    size = np.abs(x)
    above = np.clip(np.searchsorted(_FINITE, size), 1, 126)
    low, high = _FINITE[above - 1], _FINITE[above]
    up = (size - low > high - size) | ((size - low == high - size) & (above % 2 == 0))
    code = np.where(size == 0, 0, np.where(up, above, above - 1))
    code = np.where(np.isnan(x) | (size >= 464), 127, code)
    return (code + 128 * np.signbit(x)).astype(np.uint8)


def to_bits(x, kind):
    """FP32 rounded to the raw 16 bits of a type, to nearest even."""
    x = np.asarray(x, np.float32)
    if kind == 'f16':
        with np.errstate(over='ignore'):
            return x.astype(np.float16).view(np.uint16)
    bits = x.view(np.uint32).astype(np.uint64)
    rounded = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), rounded)


def from_bits(raw, kind):
    if kind == 'f16':
        return raw.view(np.float16).astype(np.float64)
    if kind == 'bf16':
        return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return E4M3[raw]


def quantise(rows):
    """E4M3 codes and exponent bytes of FP32 rows (last axis)."""
    rows = np.asarray(rows, np.float32)
    size = np.where(np.isfinite(rows), np.abs(rows), 0).max(-1).astype(np.float64)
    with np.errstate(divide='ignore'):
        power = np.ceil(np.log2(size / 448))
    power = np.clip(power, -126, 127)
    return to_e4m3(rows.astype(np.float64) * 2.0 ** -power[..., None]), (power + 127).astype(np.uint8)


class Cache:
    """Host image of a cache: flat pools, strides in elements (page, head, slot)."""

    def __init__(self, kind, pages, page_size, kv_heads, head_dim, layout='head', pad=0, fill=None, rng=None):
        self.kind, self.pages, self.page_size = kind, pages, page_size
        self.kv_heads, self.head_dim = kv_heads, head_dim
        row = head_dim + pad
        if layout == 'head':
            self.strides = (kv_heads * page_size * row, page_size * row, row)
        elif layout == 'slot':
            self.strides = (kv_heads * page_size * row, row, kv_heads * row)
        else:  # one slab per head: [head][page][slot]
            self.strides = (page_size * row, pages * page_size * row, row)
        count = pages * page_size * kv_heads * row
        dtype = TYPES[kind][1]
        if fill is not None:
            self.keys, self.values = np.full(count, fill, dtype), np.full(count, fill, dtype)
        elif kind == 'e4m3':
            self.keys, self.values = (rng.integers(0, 126, count) + 128 * rng.integers(0, 2, count) for _ in range(2))
            self.keys, self.values = self.keys.astype(np.uint8), self.values.astype(np.uint8)
        else:
            self.keys = to_bits(rng.standard_normal(count), kind)
            self.values = to_bits(0.64 * rng.standard_normal(count), kind)
        self.exponents = None
        if kind == 'e4m3':  # rows of about unit size
            self.exponents = np.full((pages, kv_heads, page_size, 2), 119, np.uint8)
            if rng is not None and fill is None:
                self.exponents = rng.integers(118, 122, self.exponents.shape).astype(np.uint8)

    def copy(self):
        other = object.__new__(Cache)
        other.__dict__.update(self.__dict__)
        other.keys, other.values = self.keys.copy(), self.values.copy()
        other.exponents = None if self.exponents is None else self.exponents.copy()
        return other

    def where(self, page, head, slot):
        at = page * self.strides[0] + head * self.strides[1] + slot * self.strides[2]
        return slice(at, at + self.head_dim)

    def place(self, table, s, j):
        """Page and slot, or None where the table holds no page."""
        page = int(table[s, j // self.page_size])
        return (page, j % self.page_size) if 0 <= page < self.pages else None

    def row(self, pool, side, page, head, slot):
        value = from_bits(pool[self.where(page, head, slot)], self.kind)
        if self.exponents is not None:
            value = value * 2.0 ** (int(self.exponents[page, head, slot, side]) - 127)
        return value

    def sequence(self, table, s, head, n):
        """Keys, values [n, head_dim] in 64 bits and which slots exist."""
        keys, values = np.zeros((n, self.head_dim)), np.zeros((n, self.head_dim))
        there = np.zeros(n, bool)
        for j in range(n):
            at = self.place(table, s, j)
            if at:
                keys[j] = self.row(self.keys, 0, at[0], head, at[1])
                values[j] = self.row(self.values, 1, at[0], head, at[1])
                there[j] = True
        return keys, values, there


def new_rows(lengths, rows, offsets):
    """(sequence, row, rank, of how many) of every new row."""
    for s in range(len(lengths)):
        first, n = (s * rows, rows) if offsets is None else (offsets[s], min(rows, offsets[s + 1] - offsets[s]))
        for i in range(max(0, n)):
            yield s, first + i, i, n


def append(cache, table, lengths, rows, offsets, keys, values, seen=None, weights=None, positions=None):
    """Writes into `cache`, weights and positions; keys, values [total, kv_heads, head_dim]."""
    for s, row, i, n in new_rows(lengths, rows, offsets):
        j = int(lengths[s]) - n + i
        if j < 0 or not 0 <= row < len(keys):
            continue
        if weights is not None:
            weights[s, :, j] = 0
        if positions is not None:
            positions[s, :, j] = (lengths if seen is None else seen)[s] - n + i
        at = cache.place(table, s, j)
        if at is None:
            continue
        for head in range(cache.kv_heads):
            for side, (pool, new) in enumerate(((cache.keys, keys), (cache.values, values))):
                if cache.kind == 'e4m3':
                    codes, byte = quantise(new[row, head])
                    pool[cache.where(at[0], head, at[1])] = codes
                    cache.exponents[at[0], head, at[1], side] = byte
                else:
                    pool[cache.where(at[0], head, at[1])] = to_bits(new[row, head], cache.kind)


def attention(cache, table, lengths, rows, offsets, q, scale, out, weights=None):
    """q, out [total, query_heads, head_dim]; returns (out, tolerance, weights,
    weight tolerance) in 64 bits; `out` gives the rows that no sequence has.

    Tolerances, to first order with u = 2^-24. The scores' operands are exact
    sums of two or three parts (2^-22 of a query in FP16 pairs), products are
    exact, and sums of D terms in FP32 lose at most D + 4 roundings of the sum of
    magnitudes: a score is off by e = scale * sum |q k| * (D + 8) u, and by
    its own rounding where the largest is taken off it. A weight p is then off by
    2 e relative (its own score and the sum's), plus its exponential, its two or
    three parts and the sum of up to N terms taken in blocks: 2^-20 in all. An
    output adds N products in blocks of 32 a wave: (N / 32 + 40) u of sum p |v|.
    """
    out, tolerance = out.astype(np.float64).copy(), np.zeros(out.shape)
    new_weights = None if weights is None else weights.astype(np.float64).copy()
    weight_tolerance = None if weights is None else np.zeros(weights.shape)
    u, heads = 2.0 ** -24, q.shape[1]
    group, dim = heads // cache.kv_heads, cache.head_dim
    views = {}
    for s, row, i, n in new_rows(lengths, rows, offsets):
        if not 0 <= row < len(q):
            continue
        sees = int(lengths[s]) - n + i + 1
        for h in range(heads):
            kv = h // group
            if sees <= 0:
                out[row, h] = 0
                continue
            if (s, kv) not in views:
                views[s, kv] = cache.sequence(table, s, kv, int(lengths[s]))
            keys, values, there = (x[:sees] for x in views[s, kv])
            keys, values = np.where(there[:, None], keys, 0), np.where(there[:, None], values, 0)
            if not there.any():
                out[row, h] = 0
                continue
            query = q[row, h].astype(np.float64)
            scores = np.where(there, keys @ query * scale, -np.inf)
            off = (abs(scale) * (np.abs(keys) @ np.abs(query)) * (dim + 8) * u)[there].max()
            p = np.exp(scores - scores.max())
            p /= p.sum()
            relative = 2 * off + 2.0 ** -20
            out[row, h] = p @ values
            tolerance[row, h] = (p @ np.abs(values)) * (relative + (sees / 32 + 40) * u) + 1e-30
            if weights is not None:
                new_weights[s, kv, :sees] += p
                weight_tolerance[s, kv, :sees] += p * relative
    if weights is not None:
        weight_tolerance += (rows * group + 1) * u * np.abs(new_weights)  # each addition rounds once
    return out, tolerance, new_weights, weight_tolerance


def evict(cache, table, lengths, keep, sinks, recent, seen, weights, positions):
    """Moves rows in `cache`; returns (new lengths, weights, positions) with
    entries from a sequence's new length on as they were."""
    weights, positions = weights.copy(), positions.copy()
    new_lengths = np.minimum(lengths, keep).astype(np.int32)
    for s, n in enumerate(int(x) for x in lengths):
        if n <= keep:
            continue
        for h in range(cache.kv_heads):
            w, p = weights[s, h, :n].astype(np.float64), positions[s, h, :n].astype(np.int64)
            order = np.where(np.isnan(w), -np.inf, np.maximum(w, -np.finfo(np.float64).max / 2))
            order = np.where(~np.isnan(w) & (w == -np.inf), -np.finfo(np.float64).max, order)
            fixed = (p < sinks) | (p >= int(seen[s]) - recent)
            rank = sorted(range(n), key=lambda j: (not fixed[j], 0 if fixed[j] else -order[j], j))
            chosen = np.zeros(n, bool)
            chosen[rank[:keep]] = True
            holes, late = np.flatnonzero(~chosen[:keep]), keep + np.flatnonzero(chosen[keep:])
            for to, start in zip(holes, late):
                weights[s, h, to], positions[s, h, to] = weights[s, h, start], positions[s, h, start]
                a, b = cache.place(table, s, to), cache.place(table, s, start)
                if a is None or b is None:
                    continue
                cache.keys[cache.where(a[0], h, a[1])] = cache.keys[cache.where(b[0], h, b[1])]
                cache.values[cache.where(a[0], h, a[1])] = cache.values[cache.where(b[0], h, b[1])]
                if cache.exponents is not None:
                    cache.exponents[a[0], h, a[1]] = cache.exponents[b[0], h, b[1]]
    return new_lengths, weights, positions

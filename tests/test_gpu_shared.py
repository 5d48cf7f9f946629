"""Attention behind shared prefixes on the GPU against plain NumPy in 64 bits,
every sequence by itself (paged_reference.attention, whose tolerances hold
here too: the same products, and sums in blocks of 32 positions a wave, joined
over fewer parts than there are such blocks), and a whole step: pages, rotation, append,
attention, verification."""
import ctypes
import sys
from pathlib import Path

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import paged_reference as ref  # noqa: E402
import step_reference as steps  # noqa: E402
from test_gpu_paged import Call, Hip  # noqa: E402

pytestmark = pytest.mark.gpu


def shared_table(rng, page, groups, lengths, prefixes, spare=2):
    """Tables of sequences whose groups (first sequences) share the whole pages of their prefixes; the positions of a
    prefix' last page are copied by share_rest."""
    n, used = len(lengths), [-(-x // page) for x in lengths]
    table, at = np.full((n, max(1, max(used))), -1, np.int32), 0
    order = rng.permutation(sum(used) + spare)
    for s in sorted(range(n), key=lambda i: -lengths[i]):  # a group's longest first
        g = next((i for i, (a, b) in enumerate(zip(groups, groups[1:])) if a <= s < b), None)
        source = s if g is None else longest(groups, lengths, g)
        whole = 0 if s == source else min(prefixes[g] // page, used[s])
        table[s, :whole] = table[source, :whole]
        table[s, whole:used[s]] = order[at:at + used[s] - whole]
        at += used[s] - whole
    return table, len(order)


def longest(groups, lengths, g):
    return max(range(groups[g], groups[g + 1]), key=lambda s: lengths[s])


def share_rest(cache, table, groups, lengths, prefixes):
    """Equal keys and values in all of a group's copies of its prefix."""
    for g, (first, last) in enumerate(zip(groups, groups[1:])):
        a = longest(groups, lengths, g) if last > first else first
        for s in range(first, last):
            for j in range(min(prefixes[g], lengths[s])):
                one, two = cache.place(table, a, j), cache.place(table, s, j)
                if one is None or two is None or one == two:
                    continue
                for h in range(cache.kv_heads):
                    for pool in (cache.keys, cache.values):
                        pool[cache.where(two[0], h, two[1])] = pool[cache.where(one[0], h, one[1])]
                    if cache.exponents is not None:
                        cache.exponents[two[0], h, two[1]] = cache.exponents[one[0], h, one[1]]


class Shared:
    """A call on a paged batch whose groups share prefixes."""

    def __init__(self, q, cache, table, lengths, prefixes, groups=None, max_prefix=None, max_rest=None, **batch):
        self.call = Call(q, cache, table, lengths, **batch)
        self.q, self.lib = q, self.call.lib
        make = lambda x: q.DeviceBuffer.from_array(np.asarray(x, np.int32))  # noqa: E731
        self.lengths, self.groups = make(prefixes), make(groups) if groups is not None else None
        most = self.call.b.max_length
        self.p = q.PagedPrefix(self.lengths.ptr, self.groups.ptr if groups is not None else None, len(prefixes),
                               min(most, max(0, max(prefixes))) if max_prefix is None else max_prefix,
                               most if max_rest is None else max_rest)

    def workspace(self, heads):
        need = ctypes.c_size_t()
        self.call.check(self.lib.qwen_gpu_op_paged_shared_workspace(ctypes.byref(self.call.c), ctypes.byref(self.call.b),
                                                                    ctypes.byref(self.p), heads, ctypes.byref(need)))
        return self.q.DeviceBuffer.from_array(np.full(need.value, 0xc5, np.uint8))

    def enqueue(self, queries, q_stride, heads, scale, out, out_stride, space, stream=None):
        self.call.check(self.lib.qwen_gpu_op_paged_attention_shared(
            ctypes.byref(self.call.c), ctypes.byref(self.call.b), ctypes.byref(self.p), queries, q_stride, heads, scale, out,
            out_stride, space.ptr, space.nbytes, stream))

    def __call__(self, queries, heads, scale, out, space=None):
        space = space or self.workspace(heads)
        qd, od = self.q.DeviceBuffer.from_array(queries), self.q.DeviceBuffer.from_array(out)
        self.enqueue(qd.ptr, queries.shape[1], heads, scale, od.ptr, out.shape[1], space)
        self.q.synchronize()
        return od.to_array(np.float32, out.size).reshape(out.shape)


def attend(q, cache, table, lengths, prefixes, heads, *, rng, groups=None, counts=None, rows=1, total=None, sharp=1.0, pad=0,
           **more):
    dim = cache.head_dim
    offsets = None if counts is None else np.concatenate(([0], np.cumsum(counts)))
    rows = rows if counts is None else max(1, max(counts))
    total = total if total is not None else len(lengths) * rows if counts is None else int(offsets[-1])
    queries = (sharp * rng.standard_normal((max(1, total) + 2, heads * dim + pad))).astype(np.float32)
    out = np.full(queries.shape, 7.5, np.float32)
    scale = dim ** -0.5
    call = Shared(q, cache, table, lengths, prefixes, groups, rows=rows, offsets=offsets, total=total, **more)
    got = call(queries, heads, scale, out)
    cut = [x[:total, :heads * dim].reshape(total, heads, dim) for x in (queries, out)]
    want, tolerance, _, _ = ref.attention(cache, table, lengths, rows, offsets, cut[0], scale, cut[1])
    off = np.abs(got[:total, :heads * dim].reshape(want.shape) - want)
    assert not np.isnan(off).any()
    assert (off <= tolerance).all(), (float((off - tolerance).max()), np.argwhere(off > tolerance)[:4])
    assert (got[total:] == 7.5).all() and (got[:, heads * dim:] == 7.5).all()
    return call, got


def made(rng, kind, kv, dim, page, layout, groups, lengths, prefixes):
    table, pages = shared_table(rng, page, groups, lengths, prefixes)
    cache = ref.Cache(kind, pages, page, kv, dim, layout, rng=rng)
    share_rest(cache, table, groups, lengths, prefixes)
    return cache, table


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('kv,group,dim,page,layout,sequences', [
    (8, 2, 128, 16, 'head', 5), (2, 1, 64, 7, 'slot', 3), (1, 16, 128, 1, 'head', 2), (3, 5, 256, 24, 'slab', 7),
    (2, 9, 64, 64, 'head', 9), (1, 40, 256, 33, 'slot', 2), (2, 2, 128, 16, 'slab', 33)])
def test_one_group(qpkg, kind, kv, group, dim, page, layout, sequences):
    """One row each behind prefixes of one position, around the tiles and long; rests of one position and more."""
    rng = np.random.default_rng(7)
    for prefix in (1, 31, 129, 300):
        lengths = [prefix + 1 + int(x) for x in rng.integers(0, 40, sequences)]
        lengths[-1] = prefix + 1
        cache, table = made(rng, kind, kv, dim, page, layout, [0, sequences], lengths, [prefix])
        attend(qpkg, cache, table, lengths, [prefix], kv * group, rng=rng, pad=3)


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('kv,group,dim', [(2, 2, 128), (1, 4, 64), (2, 3, 256), (1, 20, 128)])
def test_groups_and_ragged_rows(qpkg, kind, kv, group, dim):
    """Groups of several sizes, an empty one, one without new rows, sequences of no group before and behind; prefixes of no
    position, longer than what a sequence had before its new rows, and longer than its text."""
    rng = np.random.default_rng(11)
    groups, prefixes = [1, 4, 4, 6, 8, 11], [100, 50, 70, 0, 10 ** 6]
    lengths = [20, 140, 101, 260, 75, 72, 33, 5, 200, 200, 203, 64]
    counts = [3, 1, 1, 40, 0, 0, 5, 5, 1, 7, 2, 1]
    cache, table = made(rng, kind, kv, dim, 16, 'head', groups, lengths, prefixes)
    attend(qpkg, cache, table, lengths, prefixes, kv * group, groups=groups, counts=counts, rng=rng)
    counts = [30, 200, 1, 0, 100, 0, 33, 6, 1, 250, 0, 0]  # more new rows than positions
    attend(qpkg, cache, table, lengths, [100, 50, 70, 0, 200], kv * group, groups=groups, counts=counts, rng=rng)


@pytest.mark.parametrize('rows,group', [(1, 1), (4, 2), (9, 2), (5, 16), (40, 3)])
def test_tiles_of_a_group(qpkg, rows, group):
    """Groups of fewer and more query rows than a tile of 16, 32 and 64 has, all with the same new rows."""
    rng = np.random.default_rng(12)
    for sequences in (1, 2, 8):
        lengths = [257 + rows + 3 * s for s in range(sequences)]
        cache, table = made(rng, 'f16', 2, 128, 16, 'head', [0, sequences], lengths, [257])
        attend(qpkg, cache, table, lengths, [257], 2 * group, rows=rows, rng=rng)


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
def test_many_groups(qpkg, kind):
    """More groups and sequences than a wave has lanes, of which some are empty."""
    rng = np.random.default_rng(13)
    sizes = rng.integers(0, 4, 150)
    groups = np.concatenate(([3], 3 + np.cumsum(sizes))).tolist()
    n = groups[-1] + 2
    prefixes = rng.integers(0, 60, 150).tolist()
    lengths = rng.integers(0, 90, n).tolist()
    counts = np.minimum(rng.integers(0, 3, n), lengths).tolist()
    cache, table = made(rng, kind, 1, 64, 8, 'head', groups, lengths, prefixes)
    attend(qpkg, cache, table, lengths, prefixes, 2, groups=groups, counts=counts, rng=rng)


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
def test_long_prefix(qpkg, kind):
    """Prefixes in many parts, of more positions than the launch was sized for, and fewer."""
    rng = np.random.default_rng(14)
    lengths = [5000 + 20 + s for s in range(4)]
    cache, table = made(rng, kind, 1, 128, 16, 'head', [0, 4], lengths, [5000])
    results = []
    for sizes in ({}, dict(max_prefix=0), dict(max_prefix=300, max_rest=1), dict(max_prefix=5008, max_rest=30),
                  dict(max_prefix=5008, max_rest=5008)):
        _, got = attend(qpkg, cache, table, lengths, [5000], 4, rng=np.random.default_rng(3), **sizes)
        results.append(got)
    assert all(np.abs(x - results[0]).max() < 1e-4 for x in results)


@pytest.mark.parametrize('sharp', [1e-30, 30.0, 1e4])
@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
def test_query_sizes(qpkg, kind, sharp):
    """Scores next to 0, and so large that one position has all the weight, wherever it lies."""
    rng = np.random.default_rng(15)
    lengths = [700, 640, 900]
    cache, table = made(rng, kind, 2, 64, 16, 'head', [0, 3], lengths, [600])
    attend(qpkg, cache, table, lengths, [600], 4, counts=[3, 1, 4], rng=rng, sharp=sharp)


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
def test_takes_nothing_from_what_it_does_not_attend(qpkg, kind):
    """NaN and infinities in slots behind the lengths, in later new rows, and pages of no number, within the prefix and
    behind it."""
    rng, q = np.random.default_rng(16), qpkg
    page, dim, prefix = 4, 64, 70
    lengths = [prefix + 30, prefix + 9, prefix + 41]
    cache, table = made(rng, kind, 2, dim, page, 'head', [0, 3], lengths, [prefix])
    table[:, 5], table[1, 18], table[2, 20] = -1, 10 ** 6, -5  # a page of the prefix, and of two rests
    heads, rows = 10, 7
    queries = rng.standard_normal((3 * rows, heads * dim)).astype(np.float32)
    zeros = np.zeros_like(queries)
    clean = Shared(q, cache, table, lengths, [prefix], rows=rows)(queries, heads, 0.125, zeros)
    want, tolerance, _, _ = ref.attention(cache, table, lengths, rows, None, queries.reshape(-1, heads, dim), 0.125,
                                          zeros.reshape(-1, heads, dim))
    assert (np.abs(clean.reshape(want.shape) - want) <= tolerance).all()
    bad = {'f16': [0x7c00, 0xfc00, 0x7e01], 'bf16': [0x7f80, 0xff80, 0x7fc1], 'e4m3': [0x7f, 0xff, 0x7f]}[kind]
    spoilt = cache.copy()
    used = {cache.place(table, s, j) for s in range(3) for j in range(lengths[s])}
    for p in range(cache.pages):
        for i in range(page):
            if (p, i) not in used:
                for h in range(2):
                    for pool in (spoilt.keys, spoilt.values):
                        pool[cache.where(p, h, i)] = rng.choice(bad, dim)
                    if spoilt.exponents is not None:
                        spoilt.exponents[p, h, i] = 254
    # The last two new rows' values, which the first five do not attend.
    for s in range(3):
        for j in (lengths[s] - 2, lengths[s] - 1):
            p, i = cache.place(table, s, j)
            spoilt.values[cache.where(p, 1, i)][::3] = bad[0]
    got = Shared(q, spoilt, table, lengths, [prefix], rows=rows)(queries, heads, 0.125, zeros)
    early = np.arange(3 * rows) % rows < rows - 2
    assert np.array_equal(got[early].view(np.uint32), clean[early].view(np.uint32))
    second = got.reshape(-1, heads, dim)[~early][:, 5:]  # heads of KV head 1
    assert not np.isfinite(second[..., ::3]).any() and np.isfinite(second[..., 1::3]).all()
    assert np.array_equal(got.reshape(-1, heads, dim)[:, :5], clean.reshape(-1, heads, dim)[:, :5])


def test_bounds_what_the_device_holds(qpkg):
    """Lengths, offsets and groups out of range are bounded; what is left is finite and the rest stays."""
    rng, q, heads, dim = np.random.default_rng(17), qpkg, 4, 64
    lengths = [50, 60, 40, 30]
    cache, table = made(rng, 'bf16', 2, dim, 8, 'head', [0, 4], lengths, [24])
    queries = rng.standard_normal((12, heads * dim)).astype(np.float32)
    out = np.full_like(queries, 7.5)
    big = 2 ** 31 - 1
    for groups, prefixes in (([0, 2, 4], [24, -5]), ([-9, 1, big], [24, 24]), ([0, 4, 4], [big, -big]), ([2, 2, 3], [24, 24])):
        call = Shared(q, cache, table, lengths, prefixes, groups, rows=3)
        want, tolerance, _, _ = ref.attention(cache, table, lengths, 3, None, queries.reshape(-1, heads, dim), 0.125,
                                              out.reshape(-1, heads, dim))
        got = call(queries, heads, 0.125, out)
        if max(prefixes) < big:
            assert (np.abs(got.reshape(want.shape) - want) <= tolerance).all(), groups
        else:
            assert np.isfinite(got).all()  # a prefix of all rows before the new ones, which differ
    for groups in ([4, 0, 2], [big, -big, 3], [1, -4, 9]):  # falling: which sequences share is open
        got = Shared(q, cache, table, lengths, [24, 24], groups, rows=3)(queries, heads, 0.125, out)
        assert np.isfinite(got).all()
    strange = Shared(q, cache, table, [-7, 2, big, 2], [24], rows=3, offsets=np.array([5, -3, big, -2 ** 31, 4]), total=10)
    got = strange(queries, heads, 0.125, out)
    assert (got[10:] == 7.5).all() and np.isfinite(got).all()


def test_offsets_past_32_bits(qpkg):
    """Pages 6 GiB apart, in one allocation of 18 GiB of which a few rows are used."""
    rng, dim, page = np.random.default_rng(18), 64, 16
    stride = 3 << 30  # elements of 2 bytes
    cache = ref.Cache('f16', 4, page, 1, dim, rng=rng)
    table, lengths = np.array([[3, 0, 2], [3, 0, 1]], np.int32), [45, 40]
    call = Shared(qpkg, cache, table, lengths, [32])
    big = qpkg.DeviceBuffer((3 * stride + page * dim * 4) * 2)
    lib, rows = qpkg.load_library(), page * dim
    for p in range(4):
        for name, shift in (('keys', 0), ('values', rows)):
            part = np.ascontiguousarray(getattr(cache, name)[p * rows:(p + 1) * rows])
            assert lib.qwen_gpu_memcpy_to_device(big.ptr.value + 2 * (p * stride + shift), part.ctypes.data, part.nbytes) == 0
    call.call.c.keys, call.call.c.values, call.call.c.page_stride = big.ptr.value, big.ptr.value + 2 * rows, stride
    queries = rng.standard_normal((2, 2 * dim)).astype(np.float32)
    got = call(queries, 2, 0.125, np.zeros_like(queries))
    want, tolerance, _, _ = ref.attention(cache, table, lengths, 1, None, queries.reshape(2, 2, dim), 0.125,
                                          np.zeros((2, 2, dim)))
    assert (np.abs(got.reshape(want.shape) - want) <= tolerance).all()
    big.free()


def test_in_place_and_repeated(qpkg):
    """Outputs over their queries; the same bits every time, whatever the workspace held."""
    rng, heads, dim = np.random.default_rng(19), 6, 128
    lengths = [400 + 10 * s for s in range(6)]
    cache, table = made(rng, 'bf16', 2, dim, 16, 'slot', [0, 4, 6], lengths, [380, 128])
    call = Shared(qpkg, cache, table, lengths, [380, 128], [0, 4, 6], rows=2)
    queries = rng.standard_normal((12, heads * dim)).astype(np.float32)
    space = call.workspace(heads)
    first = call(queries, heads, 0.1, np.zeros_like(queries), space)
    for _ in range(3):
        both = qpkg.DeviceBuffer.from_array(queries)
        call.enqueue(both.ptr, heads * dim, heads, 0.1, both.ptr, heads * dim, space)
        qpkg.synchronize()
        assert np.array_equal(both.to_array(np.uint32, queries.size), first.reshape(-1).view(np.uint32))
    other = call(queries, heads, 0.1, np.zeros_like(queries))
    assert np.array_equal(other, first)


def test_wrapper(qpkg):
    """PagedKV.attention_shared gives what attention gives."""
    rng = np.random.default_rng(20)
    cache = qpkg.PagedKV(sequences=5, pages=40, max_pages=12, page_size=8, kv_heads=2, head_dim=64)
    cache.table[:, :4] = [0, 1, 2, 3]
    cache.table[:, 4:11] = 4 + np.arange(35).reshape(5, 7)
    # Every sequence writes the same prefix into the pages that all share.
    prefix = rng.standard_normal((2, 32, 2, 64)).astype(np.float32)
    for s in range(5):
        cache.append(prefix[0], prefix[1], counts=[32 * (i == s) for i in range(5)])
    counts = [3, 0, 17, 5, 1]
    for _ in range(3):
        keys, values = rng.standard_normal((2, sum(counts), 2, 64)).astype(np.float32)
        cache.append(keys, values, counts)
        queries = rng.standard_normal((sum(counts), 6, 64)).astype(np.float32)
        want = cache.attention(queries)
        for lengths, sizes in ((32, None), ([32, 20], [2, 3]), ([10 ** 6], [1]), ([0], [5])):
            got = cache.attention_shared(queries, lengths, sizes)
            # Twice the distance of either from 64 bits, which the tests above hold to less.
            assert np.abs(got - want).max() < 2e-5
    assert cache.attention_shared(queries, 32, scale=0.5).shape == queries.shape


# ---- a whole step ----

class Server:
    """A cache whose sequences share a prefix and whose pages, lengths and rows never leave the device: each step's
    drafted tokens are given pages, rotated, appended, attended and verified, and those refused are taken back."""

    def __init__(self, q, rng, kind='bf16', n=5, drafts=3, page=4, prefix=18, kv=2, heads=6, dim=64, vocabulary=40):
        self.q, self.lib, self.kv, self.heads, self.dim, self.n, self.vocabulary = q, q.load_library(), kv, heads, dim, n, vocabulary
        self.page, self.rows, self.kind = page, drafts + 1, kind
        self.pages, self.width, whole = 90, 14, -(-prefix // page)
        make = lambda x, dtype=np.int32: q.DeviceBuffer.from_array(np.asarray(x, dtype))  # noqa: E731
        # The prefix' pages belong to all; its last one is full, so that nobody appends to it.
        prefix = whole * page
        self.prefix, self.cache = prefix, ref.Cache(kind, self.pages, page, kv, dim, fill=0)
        order = rng.permutation(self.pages)
        table = np.full((n, self.width), -1, np.int32)
        table[:, :whole] = order[:whole]
        for name in ('keys', 'values'):
            rows = ref.to_bits(rng.standard_normal((whole * page * kv, dim)), kind)
            for j in range(prefix):
                for h in range(kv):
                    getattr(self.cache, name)[self.cache.where(order[j // page], h, j % page)] = rows[j * kv + h]
        stack = np.full(self.pages, -1, np.int32)
        stack[:self.pages - whole] = order[whole:]
        self.state = dict(table=table, held=np.full(n, whole), free=order[whole:], lengths=np.full(n, prefix),
                          page_size=page, pages=self.pages, shared=np.full(n, whole))
        room = n * self.rows
        self.on = {'table': make(table), 'stack': make(stack), 'held': make(np.full(n, whole)),
                   'count': make([self.pages - whole]), 'shared': make(np.full(n, whole)), 'lengths': make(np.full(n, prefix)),
                   'changes': make(np.zeros(n)), 'offsets': make(np.zeros(n + 1)), 'positions': make(np.zeros(room)),
                   'keys': make(self.cache.keys, None), 'values': make(self.cache.values, None),
                   'prefix': make([prefix]), 'qkv': make(np.zeros((room, (heads + 2 * kv) * dim)), np.float32),
                   'norm': make(np.linspace(0.5, 1.5, dim), np.float32),
                   'frequencies': make(1e4 ** (-np.arange(dim // 2) / (dim // 2)), np.float64),
                   'logits': make(np.zeros((room, vocabulary)), np.float32), 'tokens': make(np.zeros(room)),
                   'accept': make(np.zeros(room), np.float32), 'sample': make(np.zeros(n), np.float32),
                   'accepted': make(np.zeros(n)), 'next': make(np.zeros(n)), 'back': make(np.zeros(n))}
        at = {name: buffer.ptr.value for name, buffer in self.on.items()}
        self.pool = q.PagedPool(at['table'], at['stack'], at['held'], at['count'], at['shared'], self.pages, page, n, self.width)
        more = self._more(n + 1)  # the second call's offsets, which nobody reads
        self.grow, self.shrink = (q.PagedGrowth(at['lengths'], None, at[change], at['lengths'], None, at['held'], at['count'],
                                                offsets, None, positions, None, rows)
                                  for change, offsets, positions, rows in (('changes', at['offsets'], at['positions'], room),
                                                                           ('back', more, None, 0)))
        self.c = q.PagedCache(at['keys'], at['values'], None, *self.cache.strides, self.pages, page, kv, dim, q.PAGED_TYPES[kind])
        self.b = q.PagedBatch(at['table'], at['lengths'], at['offsets'], None, None, None, 0, n, self.width,
                              self.width * page, self.rows, room)
        self.p = q.PagedPrefix(at['prefix'], None, 1, prefix, self.width * page - prefix)
        row = (heads + 2 * kv) * dim
        self.row = row
        self.rotary = q.Rotary(at['frequencies'], dim, 0, dim, 0, 1, 1e-6)
        self.sides = [q.RotaryHeads(at['qkv'] + 4 * shift, at['qkv'] + 4 * shift, at['norm'], row, dim, row, dim, count)
                      for shift, count in ((0, heads), (heads * dim, kv))]
        self.draft = q.Draft(at['logits'], None, at['tokens'], at['offsets'], None, at['accept'], at['sample'], vocabulary, 0, 0,
                             vocabulary, n, self.rows, room)
        need = ctypes.c_size_t()
        self.ok(self.lib.qwen_gpu_op_paged_shared_workspace(self.c, self.b, self.p, heads, ctypes.byref(need)))
        self.space = make(np.full(need.value, 0x5a), np.uint8)
        self.ok(self.lib.qwen_gpu_op_verify_workspace(self.draft, ctypes.byref(need)))
        self.space2 = make(np.full(need.value, 0x5a), np.uint8)

    def _more(self, count):
        self.extra = self.q.DeviceBuffer.from_array(np.zeros(count, np.int32))
        return self.extra.ptr.value

    def ok(self, status):
        if status:
            raise RuntimeError(self.lib.qwen_gpu_last_error().decode())

    def give(self, **arrays):
        for name, array in arrays.items():
            array = np.ascontiguousarray(array)
            self.ok(self.lib.qwen_gpu_memcpy_to_device(self.on[name].ptr, array.ctypes.data, array.nbytes))

    def get(self, name, dtype, count):
        return self.on[name].to_array(dtype, count)

    def enqueue(self, stream=None):
        """One step; out takes the queries' place."""
        lib, at, row, dim = self.lib, self.on['qkv'].ptr.value, self.row, self.dim
        keys, values = at + 4 * self.heads * dim, at + 4 * (self.heads + self.kv) * dim
        self.ok(lib.qwen_gpu_op_paged_reserve(self.pool, self.grow, stream))
        self.ok(lib.qwen_gpu_op_rotate(self.rotary, self.sides[0], self.sides[1], self.on['positions'].ptr,
                                       self.n * self.rows, stream))
        self.ok(lib.qwen_gpu_op_paged_append(self.c, self.b, keys, row, values, row, stream))
        self.ok(lib.qwen_gpu_op_paged_attention_shared(self.c, self.b, self.p, at, row, self.heads, 0.125, at, row,
                                                       self.space.ptr, self.space.nbytes, stream))
        self.ok(lib.qwen_gpu_op_verify_draft(self.draft, self.on['accepted'].ptr, self.on['next'].ptr, self.on['back'].ptr,
                                             self.space2.ptr, self.space2.nbytes, stream))
        self.ok(lib.qwen_gpu_op_paged_reserve(self.pool, self.shrink, stream))

    def inputs(self, rng):
        room = self.n * self.rows
        counts = rng.integers(0, self.rows + 1, self.n)
        logits = 2 * rng.standard_normal((room, self.vocabulary))
        tokens = rng.integers(0, self.vocabulary, room)
        tokens[1:] = np.where(rng.random(room - 1) < 0.6, logits[:-1].argmax(1), tokens[1:])
        return dict(changes=counts.astype(np.int32), qkv=rng.standard_normal((room, self.row)).astype(np.float32),
                    logits=logits.astype(np.float32), tokens=tokens.astype(np.int32),
                    accept=rng.random(room).astype(np.float32), sample=rng.random(self.n).astype(np.float32))

    def expect(self, given):
        """The step's results against the oracles, which carry the state on."""
        room, n, dim, heads, kv = self.n * self.rows, self.n, self.dim, self.heads, self.kv
        there = steps.reserve(**self.state, changes=given['changes'], room=room)
        total = int(there['offsets'][-1])
        assert np.array_equal(self.get('positions', np.int32, room), there['positions'])
        qkv = given['qkv'].reshape(room, heads + 2 * kv, dim)
        norm = np.linspace(0.5, 1.5, dim).astype(np.float32)
        turned, _ = steps.rotate(qkv[:total, :heads + kv], there['positions'][:total],
                                 1e4 ** (-np.arange(dim // 2) / (dim // 2)), False, 1.0, norm, np.float32(1e-6))
        # What the kernels wrote is within a rounding of these; the attention is held against the device's own keys.
        pools = {name: self.get(name, np.uint16, self.cache.keys.size) for name in ('keys', 'values')}
        expected = self.cache.copy()
        ref.append(expected, there['table'], there['lengths'], self.rows, there['offsets'], turned[:, heads:].astype(np.float32),
                   qkv[:total, heads + kv:])
        assert np.array_equal(expected.values, pools['values'])
        got, want = (ref.from_bits(x, self.kind) for x in (pools['keys'], expected.keys))
        # 27 u of two channels, then BF16's half step: a value next to a border may go the other way.
        assert (np.abs(got - want) <= 2.0 ** -7 * np.abs(want) + 1e-4).all()
        self.cache.keys, self.cache.values = pools['keys'], pools['values']
        queries = turned[:, :heads].astype(np.float32)
        out, tolerance, _, _ = ref.attention(self.cache, there['table'], there['lengths'], self.rows, there['offsets'], queries,
                                             0.125, queries)
        after = self.get('qkv', np.float32, room * self.row).reshape(room, heads + 2 * kv, dim)
        off = np.abs(after[:total, :heads] - out)
        # Queries are off by 27 u of up to 2 * sqrt(64) * 1.5: scores by 1e-4 at most, weights and outputs by as much.
        assert (off <= tolerance + 4e-4).all(), off.max()
        assert np.array_equal(after[total:].view(np.uint32), qkv[total:].view(np.uint32))
        counts = np.diff(there['offsets'])
        accepted, following = steps.verify(given['logits'][:total], given['tokens'][:total], given['accept'][:total],
                                           given['sample'], None, counts)
        assert np.array_equal(self.get('accepted', np.int32, n), accepted)
        assert np.array_equal(self.get('next', np.int32, n), following)
        back = accepted - np.maximum(counts - 1, 0)
        assert np.array_equal(self.get('back', np.int32, n), back)
        done = steps.reserve(there['table'], there['held'], there['free'], there['lengths'], back, self.page, self.pages, 0,
                             shared=self.state['shared'])
        self.state.update({name: done[name] for name in ('table', 'held', 'free', 'lengths')})
        for name, size in (('held', n), ('lengths', n)):
            assert np.array_equal(self.get(name, np.int32, size), done[name]), name
        assert np.array_equal(self.get('table', np.int32, done['table'].size).reshape(done['table'].shape), done['table'])
        count = int(self.get('count', np.int32, 1)[0])
        assert np.array_equal(self.get('stack', np.int32, self.pages)[:count], done['free'])


@pytest.mark.parametrize('kind', ['f16', 'bf16'])
def test_steps(qpkg, kind):
    """Eight steps of a server, to where sequences run into the ends of their tables."""
    rng = np.random.default_rng(31)
    server = Server(qpkg, rng, kind)
    for _ in range(8):
        given = server.inputs(rng)
        server.give(**given)
        server.enqueue()
        qpkg.synchronize()
        server.expect(given)


def test_captured_steps(qpkg):
    """A step captured once and replayed, eager steps on another server between the replays; then two graphs of two
    servers, each with workspaces of its own, in flight at once."""
    hip, rng = Hip(), np.random.default_rng(32)
    servers = [Server(qpkg, np.random.default_rng(33)) for _ in range(3)]
    streams, runs, graphs = [ctypes.c_void_p() for _ in range(2)], [ctypes.c_void_p() for _ in range(2)], []
    for stream, run, server in zip(streams, runs, servers):
        graph = ctypes.c_void_p()
        hip.hipStreamCreate(ctypes.byref(stream))
        hip.hipStreamBeginCapture(stream, 0)
        server.enqueue(stream)
        hip.hipStreamEndCapture(stream, ctypes.byref(graph))
        hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0)
        graphs.append(graph)
    for turn in range(6):
        given = [server.inputs(rng) for server in servers]
        for server, arrays in zip(servers, given):
            server.give(**arrays)
        if turn % 2:
            for stream, run in zip(streams, runs):
                hip.hipGraphLaunch(run, stream)
            servers[2].enqueue()
        else:
            for stream, run in zip(streams, runs):
                hip.hipGraphLaunch(run, stream)
                hip.hipStreamSynchronize(stream)
                if run is runs[0]:
                    servers[2].enqueue()
        for stream in streams:
            hip.hipStreamSynchronize(stream)
        qpkg.synchronize()
        for server, arrays in zip(servers, given):
            server.expect(arrays)
    for stream, run, graph in zip(streams, runs, graphs):
        hip.hipGraphExecDestroy(run)
        hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(stream)


class Poisoned(Shared):
    """A call whose workspace holds NaN, so that whatever nobody wrote shows."""

    def workspace(self, heads):
        return self.q.DeviceBuffer.from_array(np.full(super().workspace(heads).nbytes, 0xff, np.uint8))


@pytest.fixture
def poisoned(monkeypatch):
    monkeypatch.setattr(sys.modules[__name__], 'Shared', Poisoned)


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('below,total,rows,sequences', [(0, 50, 1, 200), (0, 1, 1, 256), (70, 50, 1, 200), (130, 77, 3, 130)])
def test_offsets_past_the_rows(qpkg, poisoned, kind, below, total, rows, sequences):
    """Many sequences whose offsets rise past total_rows, from below 0 too: the rows that are there get all of their KV
    heads, of the prefix and of what is behind it, and all others stay."""
    rng = np.random.default_rng(41)
    prefix, kv, group, dim = 16, 8, 2, 64
    counts = np.full(sequences, rows)
    offsets = np.concatenate(([0], np.cumsum(counts))) - below
    lengths = [prefix + rows + int(x) for x in rng.integers(0, 40, sequences)]
    cache, table = made(rng, kind, kv, dim, 16, 'head', [0, sequences], lengths, [prefix])
    queries = rng.standard_normal((total + 3, kv * group * dim)).astype(np.float32)
    out = np.full(queries.shape, 7.5, np.float32)
    call = Shared(qpkg, cache, table, lengths, [prefix], rows=rows, offsets=offsets, total=total, max_rest=64, max_prefix=16)
    got = call(queries, kv * group, 0.125, out)
    want, tolerance, _, _ = ref.attention(cache, table, lengths, rows, offsets, queries[:total].reshape(total, -1, dim), 0.125,
                                          out[:total].reshape(total, -1, dim))
    assert (np.abs(got[:total].reshape(want.shape) - want) <= tolerance).all()
    assert (got[total:] == 7.5).all()


@pytest.mark.parametrize('kind', ['f16', 'e4m3'])
def test_rests_far_shorter_than_they_may_be(qpkg, poisoned, kind):
    """A launch sized for rests of 131072 positions, whose parts the workspace bounds: one that has three of them, others of
    a few positions."""
    rng = np.random.default_rng(42)
    prefix, kv, group, dim, rows, page = 100, 2, 16, 64, 4, 16
    lengths = [prefix + 3000] + [prefix + rows + int(x) for x in rng.integers(0, 40, 63)]
    cache, table = made(rng, kind, kv, dim, page, 'head', [0, 64], lengths, [prefix])
    table = np.pad(table, ((0, 0), (0, 131072 // page)), constant_values=-1)
    call, _ = attend(qpkg, cache, table, lengths, [prefix], kv * group, rows=rows, rng=rng, max_rest=131072)
    assert 200 << 20 < call.workspace(kv * group).nbytes < 300 << 20


def test_rows_of_no_sequence(qpkg, poisoned):
    """Rows between a first sequence's, which lie as far below 0 as they can, and the next one's stay."""
    rng, dim = np.random.default_rng(44), 64
    lengths, offsets = [40, 50, 60], np.array([-2 ** 31, 4, 7, 10])
    cache, table = made(rng, 'f16', 2, dim, 16, 'head', [0, 3], lengths, [30])
    queries = rng.standard_normal((12, 4 * dim)).astype(np.float32)
    out = np.full_like(queries, 7.5)
    got = Shared(qpkg, cache, table, lengths, [30], rows=3, offsets=offsets, total=12)(queries, 4, 0.125, out)
    want, tolerance, _, _ = ref.attention(cache, table, lengths, 3, offsets, queries.reshape(12, 4, dim), 0.125,
                                          out.reshape(12, 4, dim))
    assert (np.abs(got.reshape(want.shape) - want) <= tolerance).all()
    assert (got[:4] == 7.5).all() and (got[10:] == 7.5).all()


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
def test_reads_nothing_that_nobody_wrote(qpkg, poisoned, kind):
    """Ragged rows, many groups, launches of other sizes and what the device may hold, again, where every place of the
    workspace that a call does not write is NaN."""
    test_groups_and_ragged_rows(qpkg, kind, 2, 3, 128)
    test_many_groups(qpkg, kind)
    test_long_prefix(qpkg, kind)
    test_bounds_what_the_device_holds(qpkg)


def test_calls_on_streams(qpkg):
    """Three calls of other sizes on streams of their own, each with its workspace, all in flight at once, give what each
    gives alone."""
    hip, rng, calls = Hip(), np.random.default_rng(43), []
    for kind, sequences, rows, heads in (('f16', 64, 1, 16), ('bf16', 9, 5, 8), ('e4m3', 2, 1, 8)):
        prefix = 700
        lengths = [prefix + rows + 30 * s for s in range(sequences)]
        cache, table = made(rng, kind, 2, 128, 16, 'head', [0, sequences], lengths, [prefix])
        call = Shared(qpkg, cache, table, lengths, [prefix], rows=rows)
        queries = rng.standard_normal((sequences * rows, heads * 128)).astype(np.float32)
        want = call(queries, heads, 0.1, np.zeros_like(queries))
        stream = ctypes.c_void_p()
        hip.hipStreamCreate(ctypes.byref(stream))
        calls.append((call, stream, want, heads, call.workspace(heads), qpkg.DeviceBuffer.from_array(queries),
                      qpkg.DeviceBuffer.from_array(np.zeros_like(queries))))
    for _ in range(8):
        for call, stream, want, heads, space, queries, out in calls:
            call.enqueue(queries.ptr, heads * 128, heads, 0.1, out.ptr, heads * 128, space, stream)
    for call, stream, want, heads, space, queries, out in calls:
        hip.hipStreamSynchronize(stream)
        assert np.array_equal(out.to_array(np.float32, want.size).view(np.uint32), want.reshape(-1).view(np.uint32))
        hip.hipStreamDestroy(stream)

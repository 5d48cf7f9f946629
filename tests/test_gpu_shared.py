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

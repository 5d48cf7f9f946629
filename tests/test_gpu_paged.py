"""Paged key-value cache on the GPU against plain NumPy in 64 bits
(paged_reference.py): append and eviction byte for byte over the whole pools,
attention within tolerances that paged_reference.attention derives."""
import ctypes
import sys
from pathlib import Path

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import paged_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu


class Call:
    """One batch on the device, laid out as a caller would."""

    def __init__(self, q, cache, table, lengths, rows=1, offsets=None, total=None, seen=None, weights=None,
                 positions=None, max_length=None):
        self.q, self.lib, self.cache = q, q.load_library(), cache
        self.table, self.lengths = np.asarray(table, np.int32), np.asarray(lengths, np.int32)
        self.rows, self.offsets, self.seen, self.weights, self.positions = rows, offsets, seen, weights, positions
        self.total = len(lengths) * rows if total is None else total
        self.buffers = {}
        for name, array in (('table', self.table), ('lengths', self.lengths), ('offsets', offsets), ('seen', seen),
                            ('weights', weights), ('positions', positions), ('keys', cache.keys),
                            ('values', cache.values), ('exponents', cache.exponents)):
            if array is not None:
                kind = np.int32 if name in ('table', 'lengths', 'offsets', 'seen', 'positions') else None
                self.buffers[name] = q.DeviceBuffer.from_array(np.asarray(array, kind))
        at = lambda name: self.buffers[name].ptr if name in self.buffers else None  # noqa: E731
        self.c = q.PagedCache(at('keys'), at('values'), at('exponents'), *cache.strides, cache.pages, cache.page_size,
                              cache.kv_heads, cache.head_dim, q.PAGED_TYPES[cache.kind])
        stride = next((x.shape[2] for x in (weights, positions) if x is not None), 0)
        most = self.table.shape[1] * cache.page_size
        self.b = q.PagedBatch(at('table'), at('lengths'), at('offsets'), at('seen'), at('weights'), at('positions'),
                              stride, len(self.lengths), self.table.shape[1],
                              max_length or (min(most, stride) if stride else most), rows, self.total)

    def check(self, status):
        if status:
            raise RuntimeError(self.lib.qwen_gpu_last_error().decode())

    def workspace(self, query_heads):
        need = ctypes.c_size_t()
        self.check(self.lib.qwen_gpu_op_paged_workspace(ctypes.byref(self.c), ctypes.byref(self.b), query_heads,
                                                        ctypes.byref(need)))
        return self.q.DeviceBuffer.from_array(np.zeros(need.value, np.uint8))

    def append(self, keys, values, stream=None):
        """keys, values [total, row]: rows may be longer than the heads."""
        self.k, self.v = self.q.DeviceBuffer.from_array(keys), self.q.DeviceBuffer.from_array(values)
        self.check(self.lib.qwen_gpu_op_paged_append(ctypes.byref(self.c), ctypes.byref(self.b), self.k.ptr,
                                                     keys.shape[1], self.v.ptr, values.shape[1], stream))
        self.q.synchronize()

    def attention(self, q, heads, scale, out, space=None, stream=None):
        self.space = space or self.workspace(heads)
        self.qd, self.od = self.q.DeviceBuffer.from_array(q), self.q.DeviceBuffer.from_array(out)
        self.check(self.lib.qwen_gpu_op_paged_attention(ctypes.byref(self.c), ctypes.byref(self.b), self.qd.ptr,
                                                        q.shape[1], heads, scale, self.od.ptr, out.shape[1],
                                                        self.space.ptr, self.space.nbytes, stream))
        self.q.synchronize()
        return self.od.to_array(np.float32, out.size).reshape(out.shape)

    def evict(self, keep, sinks, recent, new_weights=None, new_positions=None):
        space = self.workspace(self.cache.kv_heads)
        n = self.q.DeviceBuffer.from_array(np.full(len(self.lengths), -5, np.int32))
        w = self.buffers['weights'] if new_weights is None else self.q.DeviceBuffer.from_array(new_weights)
        p = self.buffers['positions'] if new_positions is None else self.q.DeviceBuffer.from_array(new_positions)
        self.check(self.lib.qwen_gpu_op_paged_evict(ctypes.byref(self.c), ctypes.byref(self.b), keep, sinks, recent,
                                                    n.ptr, w.ptr, p.ptr, space.ptr, space.nbytes, None))
        self.q.synchronize()
        return (n.to_array(np.int32, len(self.lengths)),
                w.to_array(np.float32, self.weights.size).reshape(self.weights.shape),
                p.to_array(np.int32, self.positions.size).reshape(self.positions.shape))

    def get(self, name, like):
        return self.buffers[name].to_array(like.dtype, like.size).reshape(like.shape)

    def expect_pools(self, cache):
        for name in ('keys', 'values', 'exponents'):
            want = getattr(cache, name)
            if want is not None:
                got = self.get(name, want)
                wrong = np.flatnonzero((got != want).reshape(-1))
                assert wrong.size == 0, (name, wrong.size, wrong[:4])


def make_table(rng, lengths, page_size, spare=2, width=None):
    used = [-(-n // page_size) for n in lengths]
    pages = sum(used) + spare
    order, table, at = rng.permutation(pages), np.full((len(lengths), width or max(1, max(used))), -1, np.int32), 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pages


# ---- append ----

@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('heads,dim,page,layout,pad', [(8, 128, 16, 'head', 0), (3, 64, 5, 'slot', 0),
                                                       (5, 256, 1, 'slab', 16), (1, 64, 64, 'head', 32)])
def test_append(qpkg, kind, heads, dim, page, layout, pad):
    """Ragged new rows (none, some, more than the cache has room for), strided
    sources, untouched bytes everywhere else, tracked slots."""
    rng = np.random.default_rng(3)
    lengths, counts = [37, 1, 12, 0, 130], [5, 1, 0, 3, 130]
    table, pages = make_table(rng, lengths, page)
    offsets = np.concatenate(([0], np.cumsum(counts)))
    cache = ref.Cache(kind, pages, page, heads, dim, layout, pad, fill=7)
    total = int(offsets[-1])
    keys, values = (rng.standard_normal((total + 2, heads * dim + 12)).astype(np.float32) * 3 for _ in range(2))
    seen = np.asarray(lengths) + [0, 5, 0, 0, 1000]
    tracked = (len(lengths), heads, 140)
    weights, positions = rng.random(tracked).astype(np.float32), np.full(tracked, -9, np.int32)
    call = Call(qpkg, cache, table, lengths, 130, offsets, total, seen, weights, positions, max_length=130)
    call.append(keys, values)
    cut = [x[:total, :heads * dim].reshape(total, heads, dim) for x in (keys, values)]
    ref.append(cache, table, lengths, 130, offsets, *cut, seen, weights, positions)
    call.expect_pools(cache)
    assert np.array_equal(call.get('weights', weights), weights)
    assert np.array_equal(call.get('positions', positions), positions)


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
def test_append_special_values(qpkg, kind):
    """Ties, subnormals, zeros, the types' limits, infinities and NaN."""
    dim = 64
    rows = np.zeros((9, 1, dim), np.float32)
    rows[0, 0] = np.linspace(-1, 1, dim)
    rows[1, 0, :8] = [448, -448, 17, 18, 19, 0.0009765625, 1.0625, -1.1875]   # E4M3: ties and a subnormal
    rows[2, 0, :6] = [449, 464, -17, 2.0 ** -9, 3 * 2.0 ** -10, -0.0]
    rows[3, 0, :8] = [1e-45, -1e-45, 1e-39, 1e-41, 0, 0, 0, 2e-40]
    rows[4, 0, :5] = [3.4e38, -3.4e38, 1, 65504, 65520]
    rows[5, 0, :4] = [np.inf, 2, -3, 4]
    rows[6, 0, :4] = [np.nan, -np.inf, 300, 0.3]
    rows[7, 0, :4] = [1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11]  # 16-bit ties
    table = np.arange(3, dtype=np.int32)[None]
    cache = ref.Cache(kind, 3, 3, 1, dim, fill=1)
    call = Call(qpkg, cache, table, [9], 9)
    call.append(rows.reshape(9, dim), -rows.reshape(9, dim))
    ref.append(cache, table, [9], 9, None, rows, -rows)
    for name in ('keys', 'values'):
        got, want = (ref.from_bits(x, kind) for x in (call.get(name, cache.keys), getattr(cache, name)))
        assert np.array_equal(got, want, equal_nan=True), name
        assert np.array_equal(np.signbit(got[~np.isnan(got)]), np.signbit(want[~np.isnan(want)])), name
    if kind == 'e4m3':
        assert np.array_equal(call.get('exponents', cache.exponents), cache.exponents)


def test_append_bounds_what_the_device_holds(qpkg):
    """Pages and rows out of range are left out, lengths beyond max_length are taken as that."""
    rng = np.random.default_rng(5)
    cache = ref.Cache('f16', 4, 8, 2, 64, fill=3)
    table = np.array([[0, -1, 7], [2, 1, 2 ** 31 - 1], [3, -2 ** 31, 4]], np.int32)
    lengths, offsets = np.array([20, 50, 9]), np.array([0, 20, 25, 40])
    keys, values = (rng.standard_normal((30, 128)).astype(np.float32) for _ in range(2))
    call = Call(qpkg, cache, table, lengths, 24, offsets, 30)  # rows 30 .. 39 do not exist
    call.append(keys, values)
    cut = [x.reshape(30, 2, 64) for x in (keys, values)]
    ref.append(cache, table, np.minimum(lengths, 24), 24, offsets, *cut)
    call.expect_pools(cache)
    # Offsets that fall: which rows a sequence gets is open, but only its slots are written (the third's, page 3).
    call = Call(qpkg, cache, table, [-3, 8, 8], 8, np.array([-4, 2, 1, 2 ** 31 - 1]), 30)
    call.append(keys, values)
    for name in ('keys', 'values'):
        want = getattr(cache, name)
        page = want.size // 4
        assert np.array_equal(call.get(name, want)[:3 * page], want[:3 * page])


# ---- attention ----

def attend(q, cache, table, lengths, rows, heads, *, offsets=None, total=None, weights=None, rng, sharp=1.0, scale=None,
           pad=0, max_length=None):
    total = len(lengths) * rows if total is None else total
    stored = max(1, total) + 2
    dim = cache.head_dim
    queries = (sharp * rng.standard_normal((stored, heads * dim + pad))).astype(np.float32)
    out = np.full((stored, heads * dim + pad), 7.5, np.float32)
    scale = dim ** -0.5 if scale is None else scale
    call = Call(q, cache, table, lengths, rows, offsets, total, weights=weights, max_length=max_length)
    got = call.attention(queries, heads, scale, out)
    cut = [x[:total, :heads * dim].reshape(total, heads, dim) for x in (queries, out)]
    want, tolerance, new_weights, weight_tolerance = ref.attention(cache, table, lengths, rows, offsets, cut[0], scale,
                                                                   cut[1], weights)
    result = got[:total, :heads * dim].reshape(want.shape)
    off = np.abs(result - want)
    assert not np.isnan(off).any()
    assert (off <= tolerance).all(), (float((off - tolerance).max()), np.argwhere(off > tolerance)[:4])
    assert (got[total:] == 7.5).all() and (got[:, heads * dim:] == 7.5).all()
    # The bounds above are for the worst case; the root mean square stays far
    # below: 2^-24 a rounding, of which a weight and an output see about ten.
    norm = np.sqrt(np.mean(want ** 2))
    assert np.sqrt(np.mean(off ** 2)) <= 2e-6 * max(1.0, sharp) * norm + 1e-30
    if weights is not None:
        got_weights = call.get('weights', weights)
        off = np.abs(got_weights - new_weights)
        assert (off <= weight_tolerance).all(), float((off - weight_tolerance).max())
    return call, result


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('kv,group,dim,page,layout', [(8, 2, 128, 16, 'head'), (2, 1, 64, 7, 'slot'),
                                                      (1, 16, 128, 1, 'head'), (3, 5, 256, 24, 'slab'),
                                                      (2, 9, 64, 64, 'head'), (1, 40, 256, 33, 'slot')])
def test_attention_one_row(qpkg, kind, kv, group, dim, page, layout):
    """Lengths of none, one, around the tiles of 16, 32 and 128 positions, and odd ones."""
    rng = np.random.default_rng(7)
    lengths = [0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 300, 2]
    table, pages = make_table(rng, lengths, page)
    cache = ref.Cache(kind, pages, page, kv, dim, layout, rng=rng)
    attend(qpkg, cache, table, lengths, 1, kv * group, rng=rng, pad=3)


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('kv,group,dim,rows', [(2, 2, 128, 2), (1, 4, 64, 3), (2, 3, 256, 8), (1, 8, 128, 5)])
def test_attention_new_rows_are_causal(qpkg, kind, kv, group, dim, rows):
    """Ragged new rows, more of them than cached rows (empty rows give 0),
    none at all, weights tracked; rows of no sequence stay."""
    rng = np.random.default_rng(11)
    lengths, counts = [300, 1, 64, 0, 40, 130, 33], [rows, rows, 1, rows, 0, rows - 1, rows]
    offsets = np.concatenate(([0], np.cumsum(counts)))
    table, pages = make_table(rng, lengths, 16)
    cache = ref.Cache(kind, pages, 16, kv, dim, rng=rng)
    weights = rng.random((len(lengths), kv, 310)).astype(np.float32)
    attend(qpkg, cache, table, lengths, rows, kv * group, offsets=offsets, total=int(offsets[-1]), weights=weights,
           rng=rng)


@pytest.mark.parametrize('kind,lengths', [('f16', [5000]), ('bf16', [4097, 3]), ('e4m3', [2500, 4999, 1, 700]),
                                          ('f16', [1, 0, 4100] + [50] * 70)])
@pytest.mark.parametrize('tracked', [False, True])
def test_attention_long_and_ragged(qpkg, kind, lengths, tracked):
    """Lengths that are split over many workgroups beside short ones, more than
    64 sequences, sharp and flat softmax."""
    rng = np.random.default_rng(13)
    table, pages = make_table(rng, lengths, 64)
    cache = ref.Cache(kind, pages, 64, 2, 128, rng=rng)
    weights = np.zeros((len(lengths), 2, max(lengths)), np.float32) if tracked else None
    attend(qpkg, cache, table, lengths, 2, 4, rng=rng, sharp=3.0, weights=weights, max_length=max(lengths))


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('size', [1e-30, 1e-6, 1e5, 3e8])
def test_attention_query_sizes(qpkg, kind, size):
    """Queries far below and beyond 16-bit ranges; the scale brings scores back."""
    rng = np.random.default_rng(17)
    table, pages = make_table(rng, [150, 40], 16)
    cache = ref.Cache(kind, pages, 16, 2, 64, rng=rng)
    dim, heads = 64, 4
    queries = (size * rng.standard_normal((2, heads * dim))).astype(np.float32)
    scale = float(np.float32(0.1 / size))
    call = Call(qpkg, cache, table, [150, 40])
    got = call.attention(queries, heads, scale, np.zeros_like(queries))
    want, tolerance, _, _ = ref.attention(cache, table, [150, 40], 1, None, queries.reshape(2, heads, dim), scale,
                                          np.zeros((2, heads, dim)))
    assert (np.abs(got.reshape(want.shape) - want) <= tolerance).all()


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('scale', [0.0, -0.2, 40.0])
def test_attention_scales(qpkg, kind, scale):
    """Equal weights, negated scores, and scores of thousands (one row takes all)."""
    rng = np.random.default_rng(19)
    table, pages = make_table(rng, [200, 33], 16)
    cache = ref.Cache(kind, pages, 16, 2, 128, rng=rng)
    dim, heads = 128, 2
    queries = rng.standard_normal((2, heads * dim)).astype(np.float32)
    call = Call(qpkg, cache, table, [200, 33])
    got = call.attention(queries, heads, scale, np.zeros_like(queries))
    scale = float(np.float32(scale))
    want, tolerance, _, _ = ref.attention(cache, table, [200, 33], 1, None, queries.reshape(2, heads, dim), scale,
                                          np.zeros((2, heads, dim)))
    assert (np.abs(got.reshape(want.shape) - want) <= tolerance).all()


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
def test_attention_takes_nothing_from_what_it_does_not_attend(qpkg, kind):
    """NaN and infinities behind a sequence's end, on foreign pages, and in new
    rows that earlier ones of the same call do not see."""
    rng = np.random.default_rng(23)
    lengths, rows, page, kv, dim, heads = [37, 130, 3], 3, 16, 2, 64, 4
    table, pages = make_table(rng, lengths, page)
    clean = ref.Cache(kind, pages, page, kv, dim, rng=rng)
    dirty = clean.copy()
    bad = {'f16': (0x7e00, 0x7c00), 'bf16': (0x7fc0, 0xff80), 'e4m3': (0x7f, 0xff)}[kind]
    used = {(int(table[s, j // page]), j % page) for s, n in enumerate(lengths) for j in range(n - 1)}
    for p in range(pages):
        for slot in range(page):
            if (p, slot) not in used:
                for h in range(kv):
                    dirty.keys[dirty.where(p, h, slot)] = bad[slot % 2]
                    dirty.values[dirty.where(p, h, slot)] = bad[(slot + 1) % 2]
    queries = rng.standard_normal((9, heads * dim)).astype(np.float32)
    out = np.zeros_like(queries)
    results = [Call(qpkg, c, table, lengths, rows).attention(queries, heads, 0.125, out) for c in (clean, dirty)]
    for s in range(3):  # the last row of a sequence sees its own, spoilt key and value
        assert np.array_equal(results[0][3 * s:3 * s + 2], results[1][3 * s:3 * s + 2])
        assert not np.isfinite(results[1][3 * s + 2]).any()


@pytest.mark.parametrize('byte', [0, 1, 245, 246, 247, 248, 254, 255])
@pytest.mark.parametrize('heads,dim', [(4, 64), (2, 256), (20, 128)])
def test_attention_takes_nothing_from_exponents_it_does_not_attend(qpkg, byte, heads, dim):
    """Finite codes that their row's exponent carries past what a float holds, and exponents that no row is written
    with, where the test above has codes that are NaN."""
    rng = np.random.default_rng(127)
    lengths, rows, page, kv = [37, 130, 3], 3, 16, 2
    table, pages = make_table(rng, lengths, page)
    clean = ref.Cache('e4m3', pages, page, kv, dim, rng=rng)
    dirty = clean.copy()
    used = {(int(table[s, j // page]), j % page) for s, n in enumerate(lengths) for j in range(n - 1)}
    for p in range(pages):
        for slot in range(page):
            if (p, slot) not in used:
                dirty.exponents[p, :, slot] = byte
                for h in range(kv):
                    dirty.values[dirty.where(p, h, slot)][slot % dim] = 0x7e - 128 * -(slot % 2)  # 448 or -448
    queries = rng.standard_normal((9, heads * dim)).astype(np.float32)
    out = np.zeros_like(queries)
    results = [Call(qpkg, c, table, lengths, rows).attention(queries, heads, 0.125, out) for c in (clean, dirty)]
    for s in range(3):  # the last row of a sequence sees its own key and value
        assert np.isfinite(results[1][3 * s:3 * s + 2]).all()
        assert np.array_equal(results[0][3 * s:3 * s + 2], results[1][3 * s:3 * s + 2])


@pytest.mark.parametrize('kind,kv,group,dim', [('f16', 2, 2, 64), ('bf16', 1, 4, 128), ('e4m3', 2, 1, 256)])
@pytest.mark.parametrize('lengths,offsets,total', [
    ([300, 40, 700, 0, 9], [-1, 1, 2, 4, 4, 7], 6),              # few rows, the first and the last of which do not exist
    ([2500, 40, 2900, 0, 60], [-1, 1, 2, 4, 4, 6], 5),           # behind many positions
    ([1100, 60, 70, 300, 5], [-2, 43, 44, 45, 45, 60], 50),      # a prompt among sequences with a row or none
    ([80, 60, 1, 300, 5], [0, 1, 2, 3, 39, 39], 30)])
def test_tracked_rows_lie_by_their_number(qpkg, kind, kv, group, dim, lengths, offsets, total):
    """Weights of batches whose sequences have very different numbers of new rows, some of which do not exist."""
    rng = np.random.default_rng(131)
    table, pages = make_table(rng, lengths, 16)
    cache = ref.Cache(kind, pages, 16, kv, dim, rng=rng)
    weights = rng.random((len(lengths), kv, max(lengths) + 5)).astype(np.float32)
    rows, heads, scale = int(max(np.diff(offsets))), kv * group, float(np.float32(dim ** -0.5))
    queries = rng.standard_normal((total, heads * dim)).astype(np.float32)
    out = np.full_like(queries, 2.5)
    call = Call(qpkg, cache, table, lengths, rows, np.array(offsets), total, weights=weights)
    got = call.attention(queries, heads, scale, out)
    want, tolerance, new_weights, weight_tolerance = ref.attention(
        cache, table, lengths, rows, np.array(offsets), queries.reshape(total, heads, dim), scale,
        out.reshape(total, heads, dim), weights)
    assert (np.abs(got.reshape(want.shape) - want) <= tolerance).all()
    assert (np.abs(call.get('weights', weights) - new_weights) <= weight_tolerance).all()


def test_attention_bounds_what_the_device_holds(qpkg):
    """Slots without a page are not attended (all of them: 0), rows that do not
    exist are left alone, lengths beyond max_length are taken as that."""
    rng = np.random.default_rng(29)
    cache = ref.Cache('bf16', 6, 16, 2, 128, rng=rng)
    table = np.array([[0, -1, 3, 9], [2, 1, 2 ** 31 - 1, 4], [-1, -2 ** 31, 6, 7], [5, 5, 5, 5]], np.int32)
    lengths, offsets = [64, 60, 64, 999], np.array([0, 2, 3, 6, 9])
    weights = np.zeros((4, 2, 64), np.float32)
    dim, heads, total = 128, 4, 8
    queries = rng.standard_normal((total, heads * dim)).astype(np.float32)
    out = np.full_like(queries, 3.5)
    call = Call(qpkg, cache, table, lengths, 3, offsets, total, weights=weights)
    got = call.attention(queries, heads, 0.1, out)
    bounded = np.minimum(lengths, 64)
    scale = float(np.float32(0.1))
    want, tolerance, new_weights, weight_tolerance = ref.attention(
        cache, table, bounded, 3, offsets, queries.reshape(total, heads, dim), scale,
        out.reshape(total, heads, dim), weights)
    assert (np.abs(got.reshape(want.shape) - want) <= tolerance).all()
    assert (np.abs(call.get('weights', weights) - new_weights) <= weight_tolerance).all()
    strange = Call(qpkg, cache, table, [-7, 2, 2, 2], 3, np.array([5, -3, 2 ** 31 - 1, -2 ** 31, 4]), total)
    got = strange.attention(queries, heads, 0.1, out)
    assert np.isfinite(got).all()


def test_attention_offsets_past_32_bits(qpkg):
    """Pages 6 GiB apart, in one allocation of 18 GiB of which a few rows are used."""
    rng = np.random.default_rng(31)
    dim, page = 64, 16
    stride = 3 << 30  # elements of 2 bytes
    cache = ref.Cache('f16', 4, page, 1, dim, rng=rng)
    table, lengths = np.array([[3, 0, 2]], np.int32), [45]
    call = Call(qpkg, cache, table, lengths)
    big = qpkg.DeviceBuffer((3 * stride + page * dim * 4) * 2)
    lib = qpkg.load_library()
    rows = page * dim
    for p in range(4):
        for name, shift in (('keys', 0), ('values', rows)):
            part = np.ascontiguousarray(getattr(cache, name)[p * rows:(p + 1) * rows])
            assert lib.qwen_gpu_memcpy_to_device(big.ptr.value + 2 * (p * stride + shift), part.ctypes.data,
                                                 part.nbytes) == 0
    call.c.keys, call.c.values, call.c.page_stride = big.ptr.value, big.ptr.value + 2 * rows, stride
    queries = rng.standard_normal((1, 2 * dim)).astype(np.float32)
    got = call.attention(queries, 2, 0.125, np.zeros_like(queries))
    want, tolerance, _, _ = ref.attention(cache, table, lengths, 1, None, queries.reshape(1, 2, dim), 0.125,
                                          np.zeros((1, 2, dim)))
    assert (np.abs(got.reshape(want.shape) - want) <= tolerance).all()
    new = rng.standard_normal((1, dim)).astype(np.float32)
    call.append(new, -new)  # slot 44 lies on page 2
    word = np.zeros(dim, np.uint16)
    assert lib.qwen_gpu_memcpy_to_host(word.ctypes.data, big.ptr.value + 2 * (2 * stride + 12 * dim), word.nbytes) == 0
    assert np.array_equal(word, ref.to_bits(new[0], 'f16'))
    big.free()


def test_attention_shared_pages_and_repeated_runs(qpkg):
    """Sequences on the same pages give what each gives on pages of its own,
    with weights of its own, and the same bits every time."""
    rng = np.random.default_rng(37)
    page, kv, dim, heads, lengths = 16, 2, 128, 4, [90, 90, 75]
    table, pages = make_table(rng, [90], page)
    cache = ref.Cache('f16', pages, page, kv, dim, rng=rng)
    queries = rng.standard_normal((3, heads * dim)).astype(np.float32)
    weights = np.zeros((3, kv, 96), np.float32)
    runs = []
    for _ in range(2):
        call = Call(qpkg, cache, np.repeat(table, 3, 0), lengths, weights=weights)
        runs.append((call.attention(queries, heads, 0.1, np.zeros_like(queries)), call.get('weights', weights)))
    assert np.array_equal(runs[0][0], runs[1][0]) and np.array_equal(runs[0][1], runs[1][1])
    for s in range(3):
        call = Call(qpkg, cache, table, lengths[s:s + 1], weights=weights[:1])
        alone = call.attention(queries[s:s + 1], heads, 0.1, np.zeros_like(queries[:1]))
        assert np.allclose(alone, runs[0][0][s:s + 1], rtol=0, atol=2e-6)  # split elsewhere, perhaps
        assert np.allclose(call.get('weights', weights[:1]), runs[0][1][s:s + 1], rtol=0, atol=2e-6)


@pytest.mark.parametrize('kind,kv,group,dim,rows', [('f16', 16, 1, 64, 1), ('bf16', 16, 2, 64, 2),
                                                    ('e4m3', 12, 9, 64, 2), ('f16', 3, 2, 128, 1)])
@pytest.mark.parametrize('tracked', [False, True])
def test_attention_runs_across_units(qpkg, kind, kv, group, dim, rows, tracked):
    """More blocks of 128 positions than workgroups get one by one: they take
    runs that begin and end inside units and hold whole ones, of one tile of query
    rows and of several, and of sequences without positions."""
    rng = np.random.default_rng(67)
    count = 2600 // kv // (3 if group == 9 else 1)
    lengths = [int(x) for x in rng.integers(0, 300 if kv > 3 else 140, count)]
    lengths[3], lengths[5:8] = 1500, [0, 0, 128]
    table, pages = make_table(rng, lengths, 32)
    cache = ref.Cache(kind, pages, 32, kv, dim, rng=rng)
    weights = rng.random((count, kv, 1500)).astype(np.float32) if tracked else None
    attend(qpkg, cache, table, lengths, rows, kv * group, rng=rng, weights=weights, max_length=1500)


@pytest.mark.parametrize('lengths,counts,kv,group', [
    ([10599, 6551, 2503, 9053, 5005], [8, 7, 6, 5, 3], 1, 16),
    ([2600, 5100, 9800, 9800, 6000], [1, 1, 4, 1, 1], 2, 16),
    ([9000, 9000, 9000, 9000], [1, 2, 2, 4], 4, 8),
    ([520] * 280 + [3000], [1] * 200 + [4, 0] * 40 + [3], 1, 8)])
@pytest.mark.parametrize('kind,tracked', [('f16', False), ('bf16', True)])
def test_attention_runs_and_parts_in_one_call(qpkg, kind, tracked, lengths, counts, kv, group):
    """A head's first tile of query rows has more than 4 blocks a share and is dealt in runs, later tiles, whose
    rows only some sequences have, in parts; the same again with the workspace as the first call left it."""
    rng = np.random.default_rng(113)
    rows, offsets = max(counts), np.concatenate(([0], np.cumsum(counts)))
    tiles = -(-rows * group // 16)
    blocks = [sum(-(-n // 128) for n, c in zip(lengths, counts) if c * group > 16 * t) * tiles * kv
              for t in range(tiles)]
    assert blocks[0] > 4 * 512 >= blocks[-1]
    table, pages = make_table(rng, lengths, 32)
    cache = ref.Cache(kind, pages, 32, kv, 64, rng=rng)
    weights = rng.random((len(lengths), kv, max(lengths))).astype(np.float32) if tracked else None
    call, result = attend(qpkg, cache, table, lengths, rows, kv * group, offsets=offsets, total=sum(counts), rng=rng,
                          weights=weights, max_length=max(lengths))
    queries = call.qd.to_array(np.float32, (sum(counts) + 2) * kv * group * 64).reshape(-1, kv * group * 64)
    again = call.attention(queries, kv * group, 0.125, np.full_like(queries, 7.5), space=call.space)
    assert np.array_equal(again[:sum(counts)].reshape(result.shape), result)


@pytest.mark.parametrize('count', [64, 65, 130, 700, 1100])
@pytest.mark.parametrize('ragged', [False, True])
def test_attention_many_sequences(qpkg, count, ragged):
    rng = np.random.default_rng(71)
    lengths = [int(x) for x in rng.integers(0, 40, count)]
    lengths[count // 2], lengths[-1] = 700, 300
    counts = [int(x) for x in rng.integers(0, 3, count)] if ragged else [1] * count
    offsets = np.concatenate(([0], np.cumsum(counts))) if ragged else None
    table, pages = make_table(rng, lengths, 16)
    cache = ref.Cache('f16', pages, 16, 2, 64, rng=rng)
    attend(qpkg, cache, table, lengths, 2 if ragged else 1, 4, offsets=offsets, total=sum(counts), rng=rng)


def test_workspace_serves_calls_of_different_shapes(qpkg):
    """One workspace, zeroed once, for calls that split differently, with an eviction in between: the
    same bits as with fresh ones, and its counters are 0 again after each."""
    rng = np.random.default_rng(73)
    shapes = [([4000], 2, 4, 1), ([100] * 20, 2, 4, 2), ([900, 3, 2000], 8, 16, 1), ([4000], 2, 4, 1)]
    shapes.append(([300] * 60, 16, 16, 1))
    calls = []
    for lengths, kv, heads, rows in shapes:
        table, pages = make_table(rng, lengths, 16)
        cache = ref.Cache('f16', pages, 16, kv, 64, rng=rng)
        tracked = (len(lengths), kv, max(lengths))
        weights, positions = rng.random(tracked).astype(np.float32), np.zeros(tracked, np.int32)
        calls.append((Call(qpkg, cache, table, lengths, rows, weights=weights, positions=positions), heads))
    space = max((call.workspace(heads) for call, heads in calls), key=lambda x: x.nbytes)
    for call, heads in calls:
        queries = rng.standard_normal((call.total, heads * 64)).astype(np.float32)
        fresh = call.attention(queries, heads, 0.125, np.zeros_like(queries))
        shared = call.attention(queries, heads, 0.125, np.zeros_like(queries), space)
        assert np.array_equal(fresh, shared)
        assert not space.to_array(np.uint8, 98304).any()
        n = qpkg.DeviceBuffer(4 * len(call.lengths))
        keep = max(1, int(call.lengths.max()) // 2)
        call.check(call.lib.qwen_gpu_op_paged_evict(ctypes.byref(call.c), ctypes.byref(call.b), keep, 0, 1, n.ptr,
                                                    call.b.weights, call.b.positions, space.ptr, space.nbytes, None))
        qpkg.synchronize()
        assert not space.to_array(np.uint8, 98304).any()


def test_workspace_needs_its_counters_zeroed_and_nothing_else(qpkg):
    """The rest may hold anything, and after each call all of the counters are 0."""
    rng = np.random.default_rng(137)
    for lengths, kv, heads, rows, dim in (([4000, 3], 2, 4, 1, 64), ([700] * 3, 1, 12, 40, 128), ([300] * 90, 16, 16, 1, 256),
                                          ([17000] + [100] * 600, 1, 9, 1, 64)):
        table, pages = make_table(rng, lengths, 16)
        cache = ref.Cache('f16', pages, 16, kv, dim, rng=rng)
        tracked = (len(lengths), kv, max(lengths))
        weights, positions = rng.random(tracked).astype(np.float32), np.zeros(tracked, np.int32)
        results = []
        for fill in (0, 255):
            call = Call(qpkg, cache, table, lengths, rows, weights=weights, positions=positions)
            held = np.full(call.workspace(heads).nbytes, fill, np.uint8)
            held[:qpkg.PAGED_COUNTER_BYTES] = 0
            space = qpkg.DeviceBuffer.from_array(held)
            queries = np.random.default_rng(139).standard_normal((call.total, heads * dim)).astype(np.float32)
            results.append((call.attention(queries, heads, 0.125, np.zeros_like(queries), space),
                            call.get('weights', weights)))
            assert not space.to_array(np.uint8, qpkg.PAGED_COUNTER_BYTES).any()
            n = qpkg.DeviceBuffer(4 * len(lengths))
            call.check(call.lib.qwen_gpu_op_paged_evict(ctypes.byref(call.c), ctypes.byref(call.b), 100, 0, 1, n.ptr,
                                                        call.b.weights, call.b.positions, space.ptr, space.nbytes, None))
            qpkg.synchronize()
            assert not space.to_array(np.uint8, qpkg.PAGED_COUNTER_BYTES).any()
        for a, b in zip(*results):
            assert np.isfinite(a).all() and np.array_equal(a, b)


def test_attention_most_sequences(qpkg):
    rng = np.random.default_rng(97)
    lengths = [int(x) for x in rng.integers(0, 6, 4096)]
    lengths[4095], lengths[2222] = 400, 90
    counts = [int(x) for x in rng.integers(0, 2, 4096)]
    offsets = np.concatenate(([0], np.cumsum(counts)))
    table, pages = make_table(rng, lengths, 4)
    cache = ref.Cache('f16', pages, 4, 1, 64, rng=rng)
    attend(qpkg, cache, table, lengths, 1, 2, offsets=offsets, total=sum(counts), rng=rng)


def test_calls_on_streams(qpkg):
    """Two sequences of calls in flight at once, on streams and workspaces of their own."""
    hip, rng = Hip(), np.random.default_rng(101)
    lengths, heads, dim = [3000, 100], 4, 64
    table, pages = make_table(rng, lengths, 16)
    cache = ref.Cache('f16', pages, 16, 2, dim, rng=rng)
    sides = []
    for side in range(2):
        call = Call(qpkg, cache, table, lengths)
        queries = rng.standard_normal((2, heads * dim)).astype(np.float32)
        want = call.attention(queries, heads, 0.125, np.zeros_like(queries))
        stream = ctypes.c_void_p()
        hip.hipStreamCreate(ctypes.byref(stream))
        sides.append((call, want, stream, qpkg.DeviceBuffer(want.nbytes)))
    for _ in range(20):
        for call, want, stream, out in sides:
            call.check(call.lib.qwen_gpu_op_paged_attention(
                ctypes.byref(call.c), ctypes.byref(call.b), call.qd.ptr, heads * dim, heads, 0.125, out.ptr, heads * dim,
                call.space.ptr, call.space.nbytes, stream))
    qpkg.synchronize()
    for call, want, stream, out in sides:
        assert np.array_equal(out.to_array(np.float32, want.size).reshape(want.shape), want)
        hip.hipStreamDestroy(stream)


def test_more_new_rows_than_any_sequence_holds(qpkg):
    """Of eight new rows the last two are cached and see anything."""
    rng = np.random.default_rng(89)
    table, pages = make_table(rng, [2, 1], 16)
    cache = ref.Cache('f16', pages, 16, 2, 64, fill=0)
    call = Call(qpkg, cache, table, [2, 1], 8, max_length=2)
    keys, values = (rng.standard_normal((16, 128)).astype(np.float32) for _ in range(2))
    call.append(keys, values)
    ref.append(cache, table, [2, 1], 8, None, keys.reshape(16, 2, 64), values.reshape(16, 2, 64))
    call.expect_pools(cache)
    call, result = attend(qpkg, cache, table, [2, 1], 8, 4, rng=rng, max_length=2)
    assert not result[:6].any() and result[6:8].any(axis=(1, 2)).all()


@pytest.mark.parametrize('lengths,kv,heads,rows', [([5000, 40], 2, 16, 2), ([4300], 1, 1, 1),
                                                   ([17000] + [100] * 2000, 1, 3, 1), ([17000] + [100] * 2000, 1, 9, 1)])
def test_attention_joined_in_groups(qpkg, lengths, kv, heads, rows):
    """Units of more parts than one workgroup adds, dealt in parts and in runs, 8 and 16 rows a tile."""
    rng = np.random.default_rng(83)
    table, pages = make_table(rng, lengths, 64)
    cache = ref.Cache('f16', pages, 64, kv, 64, rng=rng)
    attend(qpkg, cache, table, lengths, rows, heads, rng=rng)


@pytest.mark.parametrize('kind', ['bf16', 'e4m3'])
@pytest.mark.parametrize('lengths,kv,heads,rows', [([5000, 40], 2, 16, 2), ([4300], 1, 1, 1),
                                                   ([17000] + [100] * 2000, 1, 9, 1)])
def test_attention_of_other_types_joined_in_groups(qpkg, kind, lengths, kv, heads, rows):
    rng = np.random.default_rng(83)
    table, pages = make_table(rng, lengths, 64)
    cache = ref.Cache(kind, pages, 64, kv, 64, rng=rng)
    attend(qpkg, cache, table, lengths, rows, heads, rng=rng)


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
@pytest.mark.parametrize('tracked', [False, True])
@pytest.mark.parametrize('dealt,lengths,counts,kv,group', [
    ('1', [5000, 40], [1, 1], 1, 2),                             # 40 parts, joined in groups, tiles of 8 rows
    ('1', [2600, 300], [2, 1], 1, 8),                            # 21 parts, tiles of 16 rows
    ('1', [2600, 300], [2, 1], 1, 9),                            # two tiles
    ('2', [9000, 7000, 50], [1, 2, 1], 3, 2),
    ('4', [9000, 7000, 6000], [1, 1, 1], 5, 3),
    ('runs', [2000, 0, 0, 128] + [17 * i % 290 for i in range(130)], [1] * 134, 8, 1),
    ('runs', [17000] + [100] * 1000, [1] * 1001, 1, 2),          # a unit of many runs, joined in groups
    ('both', [5300, 3300, 1300, 4500, 2500], [8, 7, 6, 5, 3], 1, 16)])
def test_attention_deals_heads_of_256(qpkg, kind, tracked, dealt, lengths, counts, kv, group):
    """Half as many workgroups as with smaller heads: parts of 1, 2 and 4 blocks, runs, and both in one call."""
    rows, offsets = max(counts), np.concatenate(([0], np.cumsum(counts)))
    tile = 8 if rows * group <= 8 else 16
    tiles = -(-rows * group // tile)
    blocks = [sum(max(1, -(-n // 128)) for n, c in zip(lengths, counts) if c * group > tile * t) * tiles * kv
              for t in range(tiles)]
    ways = ['1' if n <= 256 else '2' if n <= 512 else '4' if n <= 1024 else 'runs' for n in blocks]
    assert ways[0] == dealt or (dealt == 'both' and ways[0] == 'runs' != ways[-1])
    rng = np.random.default_rng(149)
    table, pages = make_table(rng, lengths, 32)
    cache = ref.Cache(kind, pages, 32, kv, 256, rng=rng)
    weights = rng.random((len(lengths), kv, max(lengths))).astype(np.float32) if tracked else None
    attend(qpkg, cache, table, lengths, rows, kv * group, offsets=offsets, total=sum(counts), rng=rng, weights=weights,
           max_length=max(lengths))


def test_attention_in_place_of_its_queries(qpkg):
    """out may be the queries' own memory."""
    rng = np.random.default_rng(79)
    lengths, heads, dim = [1000, 5, 300], 24, 64
    table, pages = make_table(rng, lengths, 16)
    cache = ref.Cache('bf16', pages, 16, 2, dim, rng=rng)
    queries = rng.standard_normal((6, heads * dim)).astype(np.float32)
    call = Call(qpkg, cache, table, lengths, 2)
    want = call.attention(queries, heads, 0.125, np.zeros_like(queries))
    both = qpkg.DeviceBuffer.from_array(queries)
    call.check(call.lib.qwen_gpu_op_paged_attention(ctypes.byref(call.c), ctypes.byref(call.b), both.ptr, heads * dim,
                                                    heads, 0.125, both.ptr, heads * dim, call.space.ptr,
                                                    call.space.nbytes, None))
    qpkg.synchronize()
    assert np.array_equal(both.to_array(np.float32, queries.size).reshape(queries.shape), want)


# ---- eviction ----

@pytest.mark.parametrize('kind,heads,dim,page,layout', [('f16', 8, 128, 16, 'head'), ('bf16', 3, 64, 5, 'slot'),
                                                        ('e4m3', 2, 256, 1, 'slab')])
@pytest.mark.parametrize('keep,sinks,recent', [(1, 0, 0), (1, 0, 1), (32, 4, 8), (32, 16, 16), (129, 0, 40),
                                               (300, 4, 100), (1024, 2, 1000)])
@pytest.mark.parametrize('in_place', [False, True])
def test_evict(qpkg, kind, heads, dim, page, layout, keep, sinks, recent, in_place):
    rng = np.random.default_rng(41)
    lengths = np.array([keep + 1, 0, keep, 2 * keep + 77, max(1, keep - 1), keep + 500], np.int32)
    table, pages = make_table(rng, lengths, page)
    cache = ref.Cache(kind, pages, page, heads, dim, layout, rng=rng)
    tracked = (len(lengths), heads, int(max(lengths)) + 3)
    weights = np.exp(rng.standard_normal(tracked)).astype(np.float32)
    positions = np.sort(rng.permuted(np.broadcast_to(np.arange(tracked[2] + 60), tracked[:2] + (tracked[2] + 60,)),
                                     axis=2)[:, :, :tracked[2]], axis=2).astype(np.int32)
    positions = rng.permuted(positions, axis=2)  # as earlier evictions leave them
    seen = lengths + 60
    call = Call(qpkg, cache, table, lengths, seen=seen, weights=weights, positions=positions)
    fresh = (weights, positions) if in_place else (np.full_like(weights, -1), np.full_like(positions, -1))
    got = call.evict(keep, sinks, recent, *((None, None) if in_place else fresh))
    want = ref.evict(cache, table, lengths, keep, sinks, recent, seen, weights, positions)
    assert np.array_equal(got[0], want[0])
    for mine, whole, before in ((got[1], want[1], fresh[0]), (got[2], want[2], fresh[1])):
        for s, n in enumerate(want[0]):
            assert np.array_equal(mine[s, :, :n], whole[s, :, :n])
            assert np.array_equal(mine[s, :, n:], before[s, :, n:])
    call.expect_pools(cache)
    if not in_place:
        assert np.array_equal(call.get('weights', weights), weights)
        assert np.array_equal(call.get('positions', positions), positions)


@pytest.mark.parametrize('values', [[0.0], [-0.0, 0.0], [np.nan, 1.0], [np.inf, np.nan, -np.inf, 0.5],
                                    [1.0, 1.0 + 2 ** -23], [-1.0, -2.0, 1e-45, -1e-45], [3.4e38, 0.0, -3.4e38]])
@pytest.mark.parametrize('length,keep', [(50, 20), (2100, 1030), (65, 64)])
def test_evict_ties_and_odd_weights(qpkg, values, length, keep):
    """Equal weights go by the lowest slot; NaN is the lowest weight, -0 is 0."""
    rng = np.random.default_rng(43)
    table, pages = make_table(rng, [length], 16)
    cache = ref.Cache('f16', pages, 16, 2, 64, rng=rng)
    weights = rng.choice(np.array(values, np.float32), (1, 2, length)).astype(np.float32)
    positions = np.broadcast_to(np.arange(length, dtype=np.int32), weights.shape).copy()
    call = Call(qpkg, cache, table, [length], weights=weights, positions=positions)
    got = call.evict(keep, 1, 2)
    want = ref.evict(cache, table, [length], keep, 1, 2, [length], weights, positions)
    assert np.array_equal(got[2][..., :keep], want[2][..., :keep])
    assert np.array_equal(got[1][..., :keep], want[1][..., :keep], equal_nan=True)
    call.expect_pools(cache)


@pytest.mark.parametrize('length,keep', [(20000, 9000), (40001, 40000), (17000, 3)])
def test_evict_long(qpkg, length, keep):
    rng = np.random.default_rng(47)
    table, pages = make_table(rng, [length], 64)
    cache = ref.Cache('e4m3', pages, 64, 1, 64, rng=rng)
    weights = rng.random((1, 1, length)).astype(np.float32)
    weights[0, 0, ::3] = weights[0, 0, 1]
    positions = np.arange(length, dtype=np.int32)[None, None].copy()
    call = Call(qpkg, cache, table, [length], weights=weights, positions=positions)
    got = call.evict(keep, 1, 2)
    want = ref.evict(cache, table, [length], keep, 1, 2, [length], weights, positions)
    assert np.array_equal(got[2][..., :keep], want[2][..., :keep])
    call.expect_pools(cache)


def test_evict_bounds_what_the_device_holds(qpkg):
    """Positions that protect more rows than stay, extreme counts of seen tokens, and missing pages."""
    rng = np.random.default_rng(53)
    cache = ref.Cache('f16', 8, 16, 1, 64, rng=rng)
    table = np.array([[0, 9, 2, 3], [4, 5, -1, 7]], np.int32)
    weights = rng.random((2, 1, 64)).astype(np.float32)
    positions = np.zeros((2, 1, 64), np.int32)
    positions[1] = 2 ** 31 - 1
    for seen in ([0, 0], [2 ** 31 - 1, -2 ** 31]):
        call = Call(qpkg, cache, table, [64, 999], seen=np.array(seen), weights=weights, positions=positions)
        got = call.evict(20, 5, 10)
        want = ref.evict(cache, table, [64, 64], 20, 5, 10, seen, weights, positions)
        for a, b in zip(got, want):
            assert np.array_equal(a[..., :20], b[..., :20])
        call.expect_pools(cache)


# ---- together ----

@pytest.mark.parametrize('kind', ['f16', 'bf16', 'e4m3'])
def test_bounded_decoding(qpkg, kind):
    """Prompts of three lengths, then steps of one and two tokens: append, attention with weights, eviction to 40 rows.
    What is cached is followed byte for byte, outputs and weights within the
    derived tolerances; the eviction's choice is checked on the weights that the device has."""
    rng = np.random.default_rng(59)
    sequences, kv, group, dim, page, keep, slots = 3, 2, 2, 128, 8, 40, 64
    width = slots // page
    paged = qpkg.PagedKV(sequences, sequences * width, width, page, kv, dim, kind, track=True)
    paged.table[:] = rng.permutation(sequences * width).reshape(sequences, width)
    cache = ref.Cache(kind, sequences * width, page, kv, dim, fill=0)
    if kind == 'e4m3':
        cache.exponents[:] = 0
    weights, positions = np.zeros((sequences, kv, slots), np.float32), np.zeros((sequences, kv, slots), np.int32)
    lengths, seen = np.zeros(sequences, np.int64), np.zeros(sequences, np.int64)
    for step in range(14):
        counts = np.array([50, 1, 33]) if step == 0 else np.full(3, 1 + step % 2)
        offsets, total = np.concatenate(([0], np.cumsum(counts))), int(counts.sum())
        keys, values, queries = (rng.standard_normal((total, n, dim)).astype(np.float32) for n in (kv, kv, kv * group))
        paged.append(keys, values, counts)
        lengths, seen = lengths + counts, seen + counts
        ref.append(cache, paged.table, lengths, int(counts.max()), offsets, keys, values, seen, weights, positions)
        got = paged.attention(queries)
        want, tolerance, new_weights, weight_tolerance = ref.attention(
            cache, paged.table, lengths, int(counts.max()), offsets, queries, dim ** -0.5, np.zeros(queries.shape), weights)
        assert (np.abs(got - want) <= tolerance).all(), step
        weights = paged.weights()
        assert (np.abs(weights - new_weights) <= weight_tolerance).all(), step
        paged.evict(keep, sinks=2, recent=10)
        new_lengths, weights, positions = ref.evict(cache, paged.table, lengths, keep, 2, 10, seen, weights, positions)
        assert np.array_equal(paged.lengths, new_lengths), step
        lengths = new_lengths.astype(np.int64)
        assert np.array_equal(paged.seen, seen)
        for s, n in enumerate(lengths):
            assert np.array_equal(paged.positions()[s, :, :n], positions[s, :, :n]), step
            assert np.array_equal(paged.weights()[s, :, :n], weights[s, :, :n]), step
        size = cache.keys.size
        assert np.array_equal(paged._keys.to_array(cache.keys.dtype, size), cache.keys), step
        assert np.array_equal(paged._values.to_array(cache.keys.dtype, size), cache.values), step
    assert all(0 in p and 1 in p and int(t) - 1 in p for s, t in enumerate(seen) for p in positions[s, :, :lengths[s]])


class Hip:
    """The runtime that the library has loaded already, for streams and graphs."""

    def __init__(self):
        self.lib = ctypes.CDLL('libamdhip64.so.7')

    def __getattr__(self, name):
        call = getattr(self.lib, name)

        def checked(*args):
            assert call(*args) == 0, name
        return checked


def test_captured_steps_follow_the_lengths(qpkg):
    """A step (append, attention with weights, eviction) captured once and
    replayed with new rows and lengths in the same device arrays, with eager calls on the same
    workspace between the replays, against eager calls on a second cache."""
    hip, rng = Hip(), np.random.default_rng(61)
    kv, dim, heads, page, keep = 2, 128, 4, 16, 300
    table = rng.permutation(42).reshape(2, 21).astype(np.int32)
    start = ref.Cache('f16', 42, page, kv, dim, rng=rng)
    tracked = (2, kv, 336)
    weights = np.exp(rng.standard_normal(tracked)).astype(np.float32)
    positions = np.broadcast_to(np.arange(336, dtype=np.int32), tracked).copy()
    calls = [Call(qpkg, start.copy(), table, [301, 200], seen=np.array([301, 200]), weights=weights,
                  positions=positions) for _ in range(2)]
    stream = ctypes.c_void_p()
    hip.hipStreamCreate(ctypes.byref(stream))
    sides = []
    for call in calls:
        side = {name: qpkg.DeviceBuffer(2 * heads * dim * 4) for name in ('q', 'k', 'v', 'out')}
        side['lengths'] = qpkg.DeviceBuffer(8)
        side['space'] = call.workspace(heads)
        sides.append(side)

    def step(call, side, on):
        lib, c, b, row = call.lib, ctypes.byref(call.c), ctypes.byref(call.b), kv * dim
        call.check(lib.qwen_gpu_op_paged_append(c, b, side['k'].ptr, row, side['v'].ptr, row, on))
        call.check(lib.qwen_gpu_op_paged_attention(c, b, side['q'].ptr, heads * dim, heads, 0.1, side['out'].ptr,
                                                   heads * dim, side['space'].ptr, side['space'].nbytes, on))
        call.check(lib.qwen_gpu_op_paged_evict(c, b, keep, 2, 20, side['lengths'].ptr, call.b.weights,
                                               call.b.positions, side['space'].ptr, side['space'].nbytes, on))

    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    hip.hipStreamBeginCapture(stream, 0)
    step(calls[0], sides[0], stream)
    hip.hipStreamEndCapture(stream, ctypes.byref(graph))
    hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0)
    lib = qpkg.load_library()
    lengths, seen = np.array([301, 200], np.int32), np.array([301, 200], np.int32)
    for turn in range(6):
        fresh = {name: rng.standard_normal(2 * n * dim).astype(np.float32)
                 for name, n in (('q', heads), ('k', kv), ('v', kv))}
        for call, side in zip(calls, sides):
            for name, array in list(fresh.items()):
                assert lib.qwen_gpu_memcpy_to_device(side[name].ptr, array.ctypes.data, array.nbytes) == 0
            for name, array in (('lengths', lengths), ('seen', seen)):
                assert lib.qwen_gpu_memcpy_to_device(call.buffers[name].ptr, array.ctypes.data, array.nbytes) == 0
        hip.hipGraphLaunch(run, stream)
        hip.hipStreamSynchronize(stream)
        step(calls[1], sides[1], None)
        qpkg.synchronize()
        outs = [side['out'].to_array(np.uint32, 2 * heads * dim) for side in sides]
        assert np.array_equal(*outs), turn
        for name, like in (('weights', weights), ('positions', positions), ('keys', start.keys), ('values', start.values)):
            a, b = (call.get(name, like) for call in calls)
            assert np.array_equal(a, b), (turn, name)
        cut = [side['lengths'].to_array(np.int32, 2) for side in sides]
        assert np.array_equal(*cut) and np.array_equal(cut[0], np.minimum(lengths, keep))
        lengths, seen = cut[0] + 1, seen + 1
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
    hip.hipStreamDestroy(stream)

"""What a step needs around a paged cache, on the GPU against plain NumPy in 64
bits (step_reference.py): heads normed and turned within tolerances derived
there, pages, rows and verified drafts number for number."""
import ctypes
import sys
from pathlib import Path

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import step_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu


class Hip:
    """The runtime that the library has loaded already, for streams and graphs."""

    def __init__(self):
        self.lib = ctypes.CDLL('libamdhip64.so.7')

    def __getattr__(self, name):
        call = getattr(self.lib, name)

        def checked(*args):
            assert call(*args) == 0, name
        return checked


def ok(q, status):
    if status:
        raise RuntimeError(q.load_library().qwen_gpu_last_error().decode())


# ---- rotation ----

class Heads:
    """Rows of heads inside a larger array: [rows][stride] elements with the heads from `first` on, or [head][row][d]."""

    def __init__(self, q, raw, heads, dim, first, by_head=False, out=None):
        self.q, self.raw, self.heads, self.dim, self.first, self.by_head = q, raw, heads, dim, first, by_head
        self.buffer = q.DeviceBuffer.from_array(raw)
        self.out = q.DeviceBuffer.from_array(out) if out is not None else self.buffer
        self.out_raw = raw if out is None else out

    def strides(self, raw):
        return (self.dim, raw.shape[1] * self.dim) if self.by_head else (raw.shape[1], self.dim)

    def place(self, raw):
        """The heads in an array like raw, [rows, heads, dim]."""
        if self.by_head:
            return raw.reshape(-1, raw.shape[1], self.dim)[:self.heads].transpose(1, 0, 2)
        return raw[:, self.first:self.first + self.heads * self.dim].reshape(raw.shape[0], self.heads, self.dim)

    def given(self, norm):
        size, skip = self.raw.itemsize, 0 if self.by_head else self.first
        r, h = self.strides(self.raw)
        out_r, out_h = self.strides(self.out_raw)
        return self.q.RotaryHeads(self.buffer.ptr.value + skip * size, self.out.ptr.value + skip * size,
                                  norm.ptr if norm else None, r, h, out_r, out_h, self.heads)

    def result(self):
        return self.out.to_array(self.out_raw.dtype, self.out_raw.size).reshape(self.out_raw.shape)


def rotate(q, sides, norms, positions, frequencies, interleaved, magnitude, kind, stream=None):
    """One call; sides: one or two Heads. Returns what the outs hold afterwards."""
    held = [q.DeviceBuffer.from_array(np.asarray(x, np.float32)) if x is not None else None for x in norms]
    place = q.DeviceBuffer.from_array(np.asarray(positions, np.int32))
    turns = q.DeviceBuffer.from_array(frequencies) if len(frequencies) else None
    rotary = q.Rotary(turns.ptr if turns else None, 2 * len(frequencies), int(interleaved), sides[0].dim, q.TYPES[kind],
                      magnitude, 1e-6)
    heads = [side.given(norm) for side, norm in zip(sides, held)]
    ok(q, q.load_library().qwen_gpu_op_rotate(rotary, heads[0], heads[1] if len(heads) > 1 else None, place.ptr,
                                              len(positions), stream))
    q.synchronize()
    return [side.result() for side in sides]


def expect_rotated(side, got, norm, positions, frequencies, interleaved, magnitude, kind):
    """Heads within their tolerance, all other elements as they were."""
    positions = np.asarray(positions)
    want, tolerance = ref.rotate(ref.decode(np.ascontiguousarray(side.place(side.raw)), kind), positions, frequencies,
                                 interleaved, np.float32(magnitude), norm, np.float32(1e-6), kind)
    off = np.abs(ref.decode(np.ascontiguousarray(side.place(got)), kind) - want)
    live = positions >= 0
    assert (off[live] <= tolerance[live]).all(), (off[live] / tolerance[live]).max()
    rest = side.out_raw.copy()
    side.place(rest)[live] = side.place(got)[live]
    assert np.array_equal(rest, got)


CASES = [  # head_dim, dims, heads of queries and keys, rows, extra elements of a row
    (128, 128, 16, 8, 5, 0), (128, 64, 7, 1, 3, 4), (64, 64, 3, 3, 1, 0), (80, 20, 4, 2, 9, 7), (256, 256, 2, 1, 4, 1),
    (96, 48, 5, 5, 2, 0), (512, 510, 1, 1, 3, 3), (512, 512, 2, 1, 2, 8), (2, 2, 1, 1, 7, 0), (6, 0, 2, 1, 3, 1),
    (192, 4, 1, 40, 2, 0), (34, 34, 2, 2, 4100, 0)]


@pytest.mark.parametrize('kind', ref.TYPES)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dim,dims,heads,kv,rows,extra', CASES)
def test_rotate(qpkg, kind, interleaved, dim, dims, heads, kv, rows, extra):
    """Queries and keys in place in the rows of a projection whose other elements stay; odd sizes and alignments."""
    rng = np.random.default_rng(5)
    raw = ref.encode(rng.standard_normal((rows, (heads + 2 * kv) * dim + extra)) * np.exp(rng.standard_normal((rows, 1))),
                     kind)
    norms = [1 + 0.3 * rng.standard_normal(dim).astype(np.float32) for _ in range(2)]
    positions = rng.integers(0, 5000, rows)
    positions[0] = 0
    frequencies = 1e4 ** (-2.0 * np.arange(dims // 2) / max(2, dims))
    side = Heads(qpkg, raw, heads, dim, 0)
    keys = Heads(qpkg, raw, kv, dim, heads * dim)
    keys.buffer = keys.out = side.buffer
    got, _ = rotate(qpkg, [side, keys], norms, positions, frequencies, interleaved, 1.25, kind)
    for which, norm, other in ((side, norms[0], keys), (keys, norms[1], side)):
        mine = raw.copy()
        which.place(mine)[:] = which.place(got)
        other_kept = got.copy()
        other.place(other_kept)[:] = other.place(raw)
        assert np.array_equal(other_kept, mine)
        expect_rotated(which, mine, norm, positions, frequencies, interleaved, 1.25, kind)


@pytest.mark.parametrize('kind', ref.TYPES)
@pytest.mark.parametrize('norms', [(False, False), (True, False), (False, True)])
def test_rotate_into_other_arrays(qpkg, kind, norms):
    """Out of place, queries of [head][row] into [row][head], keys the other way; norms of one side alone; rows of a
    negative position left as they were."""
    rng, dim, rows = np.random.default_rng(6), 64, 6
    query = Heads(qpkg, ref.encode(rng.standard_normal((5, rows, dim)), kind), 5, dim, 0, by_head=True)
    query.out_raw = ref.encode(rng.standard_normal((rows, 5 * dim + 3)), kind)
    key = Heads(qpkg, ref.encode(rng.standard_normal((rows, 2 * dim)), kind), 2, dim, 0)
    key.out_raw = ref.encode(rng.standard_normal((2, rows, dim)), kind)
    weights = [rng.standard_normal(dim).astype(np.float32) if x else None for x in norms]
    positions, frequencies = np.array([0, -1, 7, 123456, -2 ** 31, 2 ** 24]), 5e5 ** (-np.arange(16) / 16)
    given = []
    buffers = []
    for side, norm in zip((query, key), weights):
        side.out = qpkg.DeviceBuffer.from_array(side.out_raw)
        buffers.append(qpkg.DeviceBuffer.from_array(norm) if norm is not None else None)
        row_in, head_in = (dim, rows * dim) if side.by_head else (side.raw.shape[1], dim)
        row_out, head_out = (dim, rows * dim) if not side.by_head else (side.out_raw.shape[1], dim)
        given.append(qpkg.RotaryHeads(side.buffer.ptr, side.out.ptr, buffers[-1].ptr if norm is not None else None, row_in,
                                      head_in, row_out, head_out, side.heads))
    turns, place = qpkg.DeviceBuffer.from_array(frequencies), qpkg.DeviceBuffer.from_array(positions.astype(np.int32))
    rotary = qpkg.Rotary(turns.ptr, 32, 1, dim, qpkg.TYPES[kind], 1, 1e-6)
    ok(qpkg, qpkg.load_library().qwen_gpu_op_rotate(rotary, given[0], given[1], place.ptr, rows, None))
    qpkg.synchronize()
    live = positions >= 0
    for side, norm in zip((query, key), weights):
        got = side.out.to_array(side.out_raw.dtype, side.out_raw.size).reshape(side.out_raw.shape)
        if side.by_head:
            x = side.raw.transpose(1, 0, 2)
            y, kept = (z[:, :5 * dim].reshape(rows, 5, dim) for z in (got, side.out_raw))
            assert np.array_equal(got[:, 5 * dim:], side.out_raw[:, 5 * dim:])
        else:
            x, y, kept = side.raw.reshape(rows, 2, dim), got.transpose(1, 0, 2), side.out_raw.transpose(1, 0, 2)
        want, tolerance = ref.rotate(ref.decode(np.ascontiguousarray(x), kind), positions, frequencies, True, 1.0, norm,
                                     np.float32(1e-6), kind)
        off = np.abs(ref.decode(np.ascontiguousarray(y), kind) - want)
        assert (off[live] <= tolerance[live]).all()
        assert np.array_equal(y[~live], kept[~live])


@pytest.mark.parametrize('position', [0, 1, 4095, 2 ** 20 + 1, 2 ** 24 - 1, 2 ** 31 - 1])
def test_rotate_far_positions(qpkg, position):
    """Angles of far positions and plain channels of any size: infinities and NaN behind the turned ones stay there."""
    rng = np.random.default_rng(7)
    frequencies, _ = qpkg.rotary_frequencies(64, 1e6, 'ramp', 64, trained=4096)
    x = rng.standard_normal((2, 3, 96)).astype(np.float32)
    x[0, 0, 64:68] = np.inf, -np.inf, np.nan, 3e38
    got, none = qpkg.rotate(x, None, [position, 3], frequencies, 'interleaved', 1.4158883)
    assert none is None
    with np.errstate(invalid='ignore'):
        want, tolerance = ref.rotate(x, [position, 3], frequencies, True, np.float32(1.4158883), None, 1e-6)
    # The position's own angle in turns, rounded to 64 bits twice.
    tolerance = tolerance + 1.5 * 8 * position * 2.0 ** -52
    assert np.array_equal(got[..., 64:].view(np.uint32), x[..., 64:].view(np.uint32))
    assert (np.abs(got - want)[..., :64] <= tolerance[..., :64]).all()


def test_rotate_rows_past_32_bits(qpkg):
    """Two rows more than 4 GiB apart, read and written."""
    rng, dim = np.random.default_rng(8), 128
    stride = (1 << 30) + 64
    space = qpkg.DeviceBuffer(4 * (stride + dim))
    x = rng.standard_normal((2, 1, dim)).astype(np.float32)
    for r in range(2):
        ok(qpkg, qpkg.load_library().qwen_gpu_memcpy_to_device(space.ptr.value + 4 * r * stride, x[r].ctypes.data, 4 * dim))
    frequencies = 1e4 ** (-np.arange(64) / 64)
    turns, place = qpkg.DeviceBuffer.from_array(frequencies), qpkg.DeviceBuffer.from_array(np.array([5, 9], np.int32))
    heads = qpkg.RotaryHeads(space.ptr, space.ptr, None, stride, dim, stride, dim, 1)
    ok(qpkg, qpkg.load_library().qwen_gpu_op_rotate(qpkg.Rotary(turns.ptr, 128, 0, dim, 0, 1, 1e-6), heads, None, place.ptr, 2,
                                                    None))
    qpkg.synchronize()
    want, tolerance = ref.rotate(x, [5, 9], frequencies, False, 1.0, None, 1e-6)
    for r in range(2):
        got = np.zeros(dim, np.float32)
        ok(qpkg, qpkg.load_library().qwen_gpu_memcpy_to_host(got.ctypes.data, space.ptr.value + 4 * r * stride, 4 * dim))
        assert (np.abs(got - want[r, 0]) <= tolerance[r, 0]).all()


def test_rotate_nothing(qpkg):
    empty = np.zeros((0, 2, 8), np.float32)
    assert qpkg.rotate(empty, empty, [], np.ones(2))[1].shape == (0, 2, 8)


# ---- pages and rows ----

def expect_reserved(got, want):
    for name, value in want.items():
        assert np.array_equal(got[name], value), (name, np.flatnonzero(np.asarray(got[name] != value).reshape(-1))[:5])


def state(rng, n, page, longest, spare, width=None):
    """Tables of sequences with lengths up to `longest`, and the free pages."""
    lengths = rng.integers(0, longest + 1, n)
    lengths[rng.random(n) < 0.2] = 0
    held = -(-lengths // page)
    width = width or int(max(1, held.max() + 3))
    pages = int(held.sum()) + spare
    order, table, at = rng.permutation(pages), np.full((n, width), -1), 0
    for s in range(n):
        table[s, :held[s]] = order[at:at + held[s]]
        at += held[s]
    return dict(table=table, held=held, free=order[at:], lengths=lengths, page_size=page, pages=max(1, pages))


@pytest.mark.parametrize('n,page,longest,spare,room', [
    (1, 16, 40, 3, 8), (3, 1, 9, 20, 50), (8, 4, 30, 0, 20), (64, 16, 500, 40, 100), (64, 7, 100, 5, 64),
    (300, 16, 60, 300, 2000), (1025, 3, 40, 2000, 1000), (4096, 16, 100, 3000, 9000), (4096, 2, 3, 0, 5), (5, 65536, 9, 2, 30)])
def test_reserve(qpkg, n, page, longest, spare, room):
    """Rows wished for, taken back and left, with enough pages and room and without; eviction's emptied pages; text
    positions beyond the cached ones; shared first pages."""
    rng = np.random.default_rng(n + page)
    for turn in range(3):
        given = state(rng, n, page, longest, spare)
        given['changes'] = rng.integers(-longest - 2, longest + 2, n) if turn else np.ones(n, int)
        if turn == 2:
            given['seen'] = given['lengths'] + rng.integers(0, 1000, n)
            given['held'] = np.minimum(given['held'] + rng.integers(0, 2, n), given['table'].shape[1])
            given['shared'] = rng.integers(-1, 4, n)
        expect_reserved(qpkg.paged_reserve(**given, room=room), ref.reserve(**given, room=room))


def test_reserve_gives_back_what_it_took(qpkg):
    """Rows wished for and taken back again leave the lengths, and the same free pages in another order."""
    rng = np.random.default_rng(3)
    given = state(rng, 40, 4, 30, 200)
    changes = rng.integers(0, 9, 40)
    there = qpkg.paged_reserve(**given, changes=changes, room=400)
    back = qpkg.paged_reserve(there['table'], there['held'], there['free'], there['lengths'], -changes, 4, given['pages'], 0)
    assert np.array_equal(back['lengths'], given['lengths']) and np.array_equal(back['held'], given['held'])
    assert sorted(back['free']) == sorted(given['free'])


def test_reserve_of_nothing(qpkg):
    """No room, no pages, no rows; a page's last slot and the table's last entry."""
    given = dict(table=[[3, 1], [0, 2]], held=[2, 1], free=[], lengths=[8, 3], page_size=4, pages=4)
    for changes, room in (([0, 0], 0), ([1, 1], 0), ([1, 1], 5), ([-8, 2], 5), ([-99, 5], 5), ([-1, 6], 9)):
        expect_reserved(qpkg.paged_reserve(**given, changes=changes, room=room), ref.reserve(**given, changes=changes, room=room))


def test_reserve_bounds_what_the_device_holds(qpkg):
    """Lengths, held pages and counts out of range are taken into it; pages out of range are handed on, without slots; more
    pages given back than the stack has places are dropped."""
    big = 2 ** 31 - 1
    given = dict(table=[[3, 1, 99], [0, 2, -7], [5, 5, 5], [1, 1, 1]], held=[99, -4, 3, 3], free=[77, 4, -3],
                 lengths=[big, -big, 2, 12], changes=[-big - 1, 9, 3, big], page_size=4, pages=6)
    expect_reserved(qpkg.paged_reserve(**given, room=20), ref.reserve(**given, room=20))
    q, n = qpkg, 2
    on = {name: q.DeviceBuffer.from_array(np.asarray(x, np.int32)) for name, x in dict(
        table=[[0, 1], [2, 3]], stack=[9, 9, 9, 9, -55], held=[2, 2], lengths=[5, 5], changes=[-5, 2], offsets=[0] * 3,
        new=[0] * 6).items()}
    for count in (-3, big):  # taken as 0 and as 4: of the two pages given back both or none has a place
        free = q.DeviceBuffer.from_array(np.array([count], np.int32))
        pool = q.PagedPool(on['table'].ptr, on['stack'].ptr, on['held'].ptr, free.ptr, None, 4, 2, n, 2)
        new = on['new'].ptr.value
        growth = q.PagedGrowth(on['lengths'].ptr, None, on['changes'].ptr, new, None, new + 8, new + 16, on['offsets'].ptr, None,
                               None, None, 9)
        ok(q, q.load_library().qwen_gpu_op_paged_reserve(pool, growth, None))
        q.synchronize()
        got = on['new'].to_array(np.int32, 6)
        # Sequence 1's wish of 7 rows passes its table's 4 and counts as none; it keeps its length, taken as 4.
        assert got[:4].tolist() == [0, 4, 0, 2] and got[4] == (2 if count < 0 else 4)
        assert on['stack'].to_array(np.int32, 5)[4] == -55


@pytest.mark.parametrize('n', [2, 30, 1500])
def test_reserve_with_fewer_pages_than_rows(qpkg, n):
    """A sequence that has fewer pages than its rows need takes them all when it grows, and none before."""
    rng = np.random.default_rng(n)
    given = state(rng, n, 4, 30, 3 * n)
    given['held'] = np.maximum(0, given['held'] - rng.integers(0, 3, n))
    given['changes'] = rng.integers(-2, 4, n)
    expect_reserved(qpkg.paged_reserve(**given, room=4 * n), ref.reserve(**given, room=4 * n))


def test_reserve_with_one_array_as_lengths_and_seen(qpkg):
    """Lengths that are the text's positions as well, and their results in the place of one of them."""
    rng, q = np.random.default_rng(5), qpkg
    given = state(rng, 30, 4, 30, 60)
    changes = rng.integers(-6, 6, 30)
    want = ref.reserve(**given, changes=changes, room=0)
    stack = np.full(given['pages'], -1, np.int32)
    stack[:len(given['free'])] = given['free']
    for in_place in ('lengths', 'seen'):
        on = {name: q.DeviceBuffer.from_array(np.asarray(x, np.int32)) for name, x in dict(
            table=given['table'], held=given['held'], lengths=given['lengths'], changes=changes, stack=stack,
            count=[len(given['free'])], other=[0] * 30, offsets=[0] * 31).items()}
        at = {name: buffer.ptr for name, buffer in on.items()}
        pool = q.PagedPool(at['table'], at['stack'], at['held'], at['count'], None, given['pages'], 4, 30,
                           np.asarray(given['table']).shape[1])
        results = (at['lengths'], at['other']) if in_place == 'lengths' else (at['other'], at['lengths'])
        growth = q.PagedGrowth(at['lengths'], at['lengths'], at['changes'], *results, at['held'], at['count'], at['offsets'],
                               None, None, None, 0)
        ok(q, q.load_library().qwen_gpu_op_paged_reserve(pool, growth, None))
        q.synchronize()
        for name in ('lengths', 'other'):
            assert np.array_equal(on[name].to_array(np.int32, 30), want['lengths']), (in_place, name)


def test_reserve_results_apart_from_what_is_given(qpkg):
    """Results in arrays of their own: what was given stays, and the call can be made again."""
    rng, q = np.random.default_rng(4), qpkg
    given = state(rng, 30, 4, 30, 60)
    changes = rng.integers(-6, 6, 30)
    want = ref.reserve(**given, changes=changes, room=70)
    ints = {name: np.asarray(given[name], np.int32) for name in ('table', 'held', 'lengths')}
    stack = np.full(given['pages'], -1, np.int32)
    stack[:len(given['free'])] = given['free']
    ints.update(changes=changes.astype(np.int32), seen=(given['lengths'] + 5).astype(np.int32), stack=stack,
                count=np.array([len(given['free'])], np.int32))
    on = {name: q.DeviceBuffer.from_array(x) for name, x in ints.items()}
    out = {name: q.DeviceBuffer(4 * size) for name, size in
           (('lengths', 30), ('seen', 30), ('held', 30), ('count', 1), ('offsets', 31), ('positions', 70))}
    pool = q.PagedPool(on['table'].ptr, on['stack'].ptr, on['held'].ptr, on['count'].ptr, None, given['pages'], 4, 30,
                       ints['table'].shape[1])
    growth = q.PagedGrowth(on['lengths'].ptr, on['seen'].ptr, on['changes'].ptr, out['lengths'].ptr, out['seen'].ptr,
                           out['held'].ptr, out['count'].ptr, out['offsets'].ptr, None, out['positions'].ptr, None, 70)
    for _ in range(3):
        ok(q, q.load_library().qwen_gpu_op_paged_reserve(pool, growth, None))
        q.synchronize()
        for name in ('lengths', 'held', 'offsets'):
            assert np.array_equal(out[name].to_array(np.int32, want[name].size), want[name]), name
        assert np.array_equal(out['seen'].to_array(np.int32, 30), want['seen'] + 5)
        assert out['count'].to_array(np.int32, 1)[0] == len(want['free'])
        rows = want['offsets'][-1]
        assert np.array_equal(out['positions'].to_array(np.int32, 70)[:rows], want['positions'][:rows] + 5)
        assert np.array_equal(on['table'].to_array(np.int32, ints['table'].size).reshape(ints['table'].shape), want['table'])
        for name in ('held', 'lengths', 'changes', 'seen', 'count'):
            assert np.array_equal(on[name].to_array(np.int32, ints[name].size), ints[name]), name


# ---- drafts ----

class Drafts:
    """A call's arrays on the device."""

    def __init__(self, q, logits, tokens, accept, sample, draft=None, counts=None, temperature=None, kind='f32', pad=0,
                 vocabulary=None, rows=None, offsets=None):
        self.q, self.n = q, len(sample)
        total, width = logits.shape
        self.vocabulary = vocabulary or width - pad
        if counts is not None and offsets is None:
            offsets = np.concatenate(([0], np.cumsum(counts)))
        self.rows = rows or (max(1, int(max(counts))) if counts is not None else total // self.n)
        make = lambda x, dtype: q.DeviceBuffer.from_array(np.asarray(x, dtype)) if x is not None else None  # noqa: E731
        self.held = [q.DeviceBuffer.from_array(logits), make(draft, np.float32), make(tokens, np.int32), make(offsets, np.int32),
                     make(temperature, np.float32), make(accept, np.float32), make(sample, np.float32)]
        self.given = q.Draft(*[x.ptr if x is not None else None for x in self.held], width,
                             draft.shape[1] if draft is not None else 0, q.TYPES[kind], self.vocabulary, self.n, self.rows, total)
        need = ctypes.c_size_t()
        ok(q, q.load_library().qwen_gpu_op_verify_workspace(self.given, ctypes.byref(need)))
        self.space = q.DeviceBuffer.from_array(np.full(need.value, 0xa5, np.uint8))
        self.out = [q.DeviceBuffer.from_array(np.full(self.n, -9, np.int32)) for _ in range(3)]

    def enqueue(self, stream=None):
        ok(self.q, self.q.load_library().qwen_gpu_op_verify_draft(self.given, *[x.ptr for x in self.out], self.space.ptr,
                                                                  self.space.nbytes, stream))

    def results(self):
        return [x.to_array(np.int32, self.n) for x in self.out]

    def __call__(self):
        self.enqueue()
        self.q.synchronize()
        return self.results()


def random_drafts(rng, n, rows, vocabulary, ragged=False, draft=True, filtered=False, hot=1.0):
    counts = rng.integers(1, rows + 1, n) if ragged else np.full(n, rows)
    total = int(counts.sum())
    logits = 3 * rng.standard_normal((total, vocabulary)) + 2 * rng.standard_normal(vocabulary)
    guess = logits + rng.standard_normal((total, vocabulary))
    if filtered:
        logits = np.where(logits >= np.sort(logits, -1)[:, -min(20, vocabulary)][:, None], logits, -np.inf)
    guess = np.exp((guess - guess.max(-1, keepdims=True)) / hot)
    guess = (guess / guess.sum(-1, keepdims=True)).astype(np.float32)
    tokens = np.zeros(total, int)
    for r in range(total - 1):
        if draft:
            p = guess[r].astype(np.float64)
            tokens[r + 1] = rng.choice(vocabulary, p=p / p.sum())
        else:
            tokens[r + 1] = logits[r].argmax() if rng.random() < 0.6 else rng.integers(vocabulary)
    return dict(logits=logits.astype(np.float32), tokens=tokens, accept=rng.random(total).astype(np.float32),
                sample=rng.random(n).astype(np.float32), draft=guess if draft else None, counts=counts)


@pytest.mark.parametrize('kind', ref.TYPES)
@pytest.mark.parametrize('n,rows,vocabulary,ragged,draft,filtered', [
    (1, 2, 1000, False, False, False), (3, 1, 7, False, False, False), (5, 4, 4097, True, True, False),
    (9, 6, 12289, True, True, True), (40, 3, 257, True, False, True), (2, 3, 151936, False, True, False),
    (300, 2, 2, False, True, False), (4, 3, 1, True, True, False), (1, 40, 100, False, True, False),
    (2, 2, 1100000, False, True, False)])
def test_verify(qpkg, kind, n, rows, vocabulary, ragged, draft, filtered):
    """Greedy and warm sequences together, rows with padding behind the vocabulary that no token stands for."""
    rng = np.random.default_rng(n + vocabulary)
    given = random_drafts(rng, n, rows, vocabulary, ragged, draft, filtered)
    temperature = np.where(rng.random(n) < 0.3, 0, 0.3 + rng.random(n)).astype(np.float32)
    raw = ref.encode(given['logits'], kind)
    given['logits'] = ref.decode(raw, kind)
    want = ref.verify(**given, temperature=temperature)
    pad = 3
    raw = np.concatenate((raw, ref.encode(np.full((len(raw), pad), 1e4, np.float32), kind)), 1)
    given['logits'] = raw
    accepted, following, back = Drafts(qpkg, **given, temperature=temperature, kind=kind, pad=pad)()
    assert np.array_equal(accepted, want[0]) and np.array_equal(following, want[1])
    assert np.array_equal(back, want[0] - (given['counts'] - 1))


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('n,rows,vocabulary', [(1, 1, 151936), (1, 2, 151936), (3, 4, 20000), (64, 7, 20000), (200, 8, 12289),
                                               (385, 2, 32769)])
def test_verify_certain_drafts(qpkg, kind, n, rows, vocabulary):
    """Without probabilities of their own: a row's sums are added once, in ranges of one chunk, of several, and of more than
    a workgroup goes through."""
    rng = np.random.default_rng(n + vocabulary)
    given = random_drafts(rng, n, rows, vocabulary, draft=False)
    raw = ref.encode(given['logits'], kind)
    given['logits'] = ref.decode(raw, kind)
    temperature = (0.3 + rng.random(n)).astype(np.float32)
    want = ref.verify(**given, temperature=temperature)
    given['logits'] = raw
    accepted, following, _ = Drafts(qpkg, **given, temperature=temperature, kind=kind)()
    assert np.array_equal(accepted, want[0]) and np.array_equal(following, want[1])


@pytest.mark.parametrize('many', [1, 50])
def test_verify_certain_drafts_at_borders(qpkg, many):
    """Equal logits again, the drafted token refused: the others' weights are whole numbers on either side of it. Rows
    of 400 sequences are one range, of three chunks."""
    vocabulary, token = 8192 + 1, 5000
    share = np.array([0, 1, 4095, 4096, 4999, 5000, 8191, 8190])
    n, sample = 8 * many, np.tile(share / 8192, many).astype(np.float32)
    logits = np.full((2 * n, vocabulary), -2.5, np.float32)
    tokens = np.zeros(2 * n, int)
    tokens[1::2] = token
    accepted, following, _ = Drafts(qpkg, logits, tokens, np.full(2 * n, 0.5, np.float32), sample)()
    want = np.tile(share + (share >= token), n // 8)
    assert not accepted.any() and np.array_equal(following, want)


def test_verify_wrapper(qpkg):
    rng = np.random.default_rng(9)
    given = random_drafts(rng, 6, 4, 500, ragged=True)
    for more in ({}, {'temperature': np.array([0, 1, 0.5, 2, 0, 1], np.float32)}):
        want = ref.verify(**given, **more)
        got = qpkg.verify_draft(**given, **more)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    one = qpkg.verify_draft(given['logits'][:4], given['tokens'][:4], given['accept'][:4], given['sample'][:2])
    assert np.array_equal(one[1], ref.verify(given['logits'][:4], given['tokens'][:4], given['accept'][:4], given['sample'][:2])[1])


@pytest.mark.parametrize('vocabulary', [1, 64, 4096, 8192, 65536])
def test_verify_at_borders(qpkg, vocabulary):
    """Equal logits of a power of two: every sum is exact, so numbers on the borders fall where the definition has them."""
    n = 8
    share = np.array([0, 1, vocabulary // 2, vocabulary - 1, 0, 1, 5, vocabulary - 1]) % vocabulary
    sample = (share / vocabulary).astype(np.float32)
    logits = np.full((2 * n, vocabulary), 7.5, np.float32)
    tokens = np.zeros(2 * n, int)
    tokens[1::2] = vocabulary - 1
    q = np.full((2 * n, vocabulary), 1 / vocabulary, np.float32)
    q[:, -1] = 2 / vocabulary
    accept = np.zeros(2 * n, np.float32)
    accept[::2] = [0.5, 0.499, 0.5, 0.25, 0, 0.75, np.float32(1 - 2 ** -24), 0.5]  # p / q is a half
    accepted, following, _ = Drafts(qpkg, logits, tokens, accept, sample, q)()
    assert accepted.tolist() == [0, 1, 0, 1, 1, 0, 0, 0]
    # Refused: max(p - q, 0) is 0 throughout, so p; accepted: the last row's p. Both are even.
    assert following.tolist() == share.tolist()


def test_verify_odd_rows(qpkg):
    """Filtered, NaN and infinite logits, rows without a token, equal largest logits, tokens outside the vocabulary,
    probabilities that are 0, negative or NaN, numbers beyond [0, 1)."""
    inf, nan, v = np.inf, np.nan, 6
    rows = [[-inf] * v, [nan] * v, [nan, 2, -inf, 2, nan, 1], [inf, 1, 2, inf, -inf, 0], [3e38, -3e38, 0, 1, 2, 3e38],
            [-inf, -inf, 5, -inf, -inf, -inf], [0, 0, 1, 1, 1, 0], [-1e-45, 0, -0.0, 1e-45, 0, 0]]
    rng = np.random.default_rng(10)
    drafts = [[0.1, 0.2, 0.3, 0.4, 0, 0], [0] * v, [-1, nan, 0.5, 0.5, inf, 0], [1, 0, 0, 0, 0, 0]]
    logits, tokens, accept, sample, draft, heat = [], [], [], [], [], []
    for row in rows:
        for guess in drafts:
            for token in (0, 2, 3, -1, 6, 2 ** 31 - 1):
                for t in (0.0, 1.0, 1e-3, -1.0, nan, 1e-45, inf):
                    logits += [row, rng.standard_normal(v)]
                    draft += [guess, [0.5] * v]
                    tokens += [0, token]
                    accept += [rng.choice([0, 0.3, 0.99, nan, 2.0]), nan]
                    sample.append(rng.choice([0, 0.5, 0.999, 1.5, -1.0, nan]))
                    heat.append(t)
    n = len(sample)
    logits, draft = np.asarray(logits, np.float32), np.asarray(draft, np.float32)
    half = n // 2  # of them with a draft's probabilities, the others certain
    for part, q in ((slice(0, half), draft), (slice(half, n), None)):
        two = slice(2 * part.start, 2 * part.stop)
        given = (logits[two], np.asarray(tokens)[two], np.asarray(accept, np.float32)[two], np.asarray(sample, np.float32)[part],
                 q[two] if q is not None else None)
        with np.errstate(all='ignore'):
            want = ref.verify(*given, temperature=np.asarray(heat, np.float32)[part])
        accepted, following, _ = Drafts(qpkg, *given, temperature=np.asarray(heat, np.float32)[part])()
        assert np.array_equal(accepted, want[0])
        assert np.array_equal(following, want[1]), np.flatnonzero(following != want[1])[:5]


def test_verify_bounds_what_the_device_holds(qpkg):
    """Offsets out of range leave rows out; sequences without rows draw nothing."""
    rng = np.random.default_rng(11)
    given = random_drafts(rng, 4, 3, 50, draft=False)
    del given['counts']
    offsets = [0, 3, 3, 6, 99]  # the fourth has the rows that there are: 6 .. 11, of which a sequence has three at most
    accepted, following, back = Drafts(qpkg, **given, offsets=offsets, rows=3)()
    trimmed = {name: x[:9] if name in ('logits', 'tokens', 'accept') else x for name, x in given.items()}
    want = ref.verify(**trimmed, counts=[3, 0, 3, 3])
    assert np.array_equal(accepted, want[0]) and np.array_equal(following, want[1])
    assert back[1] == 0
    accepted, following, back = Drafts(qpkg, **given, offsets=[-5, -1, 200, 300, 100], rows=3)()
    assert accepted.tolist() == [0] * 4 and following.tolist() == [-1] * 4 and back.tolist() == [0] * 4


def test_verify_offsets_past_32_bits(qpkg):
    """Rows of logits and of the draft more than 4 GiB apart."""
    rng, v, stride = np.random.default_rng(12), 3000, (1 << 30) + 64
    given = random_drafts(rng, 1, 3, v)
    lib = qpkg.load_library()
    spaces = [qpkg.DeviceBuffer(4 * (2 * stride + v)) for _ in range(2)]
    for space, rows in zip(spaces, (given['logits'], given['draft'])):
        for r in range(3):
            row = np.ascontiguousarray(rows[r])
            ok(qpkg, lib.qwen_gpu_memcpy_to_device(space.ptr.value + 4 * r * stride, row.ctypes.data, 4 * v))
    for accept in (np.zeros(3, np.float32), given['accept'], np.ones(3, np.float32)):
        given['accept'] = accept
        call = Drafts(qpkg, **given)
        call.given.logits, call.given.draft = spaces[0].ptr, spaces[1].ptr
        call.given.logit_stride = call.given.draft_stride = stride
        want = ref.verify(**given)
        accepted, following, _ = call()
        assert np.array_equal(accepted, want[0]) and np.array_equal(following, want[1])


def test_verify_repeats(qpkg):
    """The same numbers every time, on a workspace that held another call's."""
    rng = np.random.default_rng(13)
    calls = [Drafts(qpkg, **random_drafts(rng, n, rows, v, ragged=True)) for n, rows, v in ((5, 4, 9000), (9, 2, 300))]
    big = max((c.space for c in calls), key=lambda s: s.nbytes)
    for call in calls:
        call.space = big
    first = [call() for call in calls]
    for _ in range(3):
        for call, want in zip(calls, first):
            assert all(np.array_equal(a, b) for a, b in zip(call(), want))


# ---- calls at once, streams, graphs ----

def test_calls_on_streams(qpkg):
    """Every operator on a stream of its own, all in flight at once, against the same calls one after the other; the
    runtime's stand-in handles are refused."""
    q, hip, rng = qpkg, Hip(), np.random.default_rng(21)
    lib, streams = q.load_library(), []
    for _ in range(4):
        streams.append(ctypes.c_void_p())
        hip.hipStreamCreate(ctypes.byref(streams[-1]))
    drafts = [Drafts(q, **random_drafts(rng, 5, 4, 9000, ragged=True)) for _ in range(2)]
    alone = [call() for call in drafts]
    x = [rng.standard_normal((200, 6 * 64)).astype(np.float32) for _ in range(2)]
    frequencies, positions = 1e4 ** (-np.arange(32) / 32), rng.integers(0, 9999, 200)
    place, turns = q.DeviceBuffer.from_array(positions.astype(np.int32)), q.DeviceBuffer.from_array(frequencies)
    rotary = q.Rotary(turns.ptr, 64, 0, 64, 0, 1, 1e-6)
    want = []
    for array in x:
        side = Heads(q, array, 6, 64, 0)
        want.append(rotate(q, [side], [None], positions, frequencies, False, 1.0, 'f32')[0])
    on = [q.DeviceBuffer.from_array(array) for array in x]
    for turn in range(2):
        for call, stream in zip(drafts, streams):
            call.enqueue(stream)
        for buffer, stream in zip(on, streams[2:]):
            if turn == 0:
                heads = q.RotaryHeads(buffer.ptr, buffer.ptr, None, 384, 64, 384, 64, 6)
                ok(q, lib.qwen_gpu_op_rotate(rotary, heads, None, place.ptr, 200, stream))
    for stream in streams:
        hip.hipStreamSynchronize(stream)
    for call, given in zip(drafts, alone):
        assert all(np.array_equal(a, b) for a, b in zip(call.results(), given))
    for buffer, given in zip(on, want):
        assert np.array_equal(buffer.to_array(np.float32, given.size), given.reshape(-1))
    for handle in (1, 2):
        with pytest.raises(RuntimeError, match='The stream must be NULL'):
            drafts[0].enqueue(ctypes.c_void_p(handle))
    for stream in streams:
        hip.hipStreamDestroy(stream)


def test_host_memory_is_refused(qpkg):
    """Plain host arrays, which a kernel cannot read, are found before anything is launched."""
    call = Drafts(qpkg, **random_drafts(np.random.default_rng(22), 2, 2, 50))
    host = np.zeros(100, np.float32)
    call.given.sample = host.ctypes.data
    with pytest.raises(RuntimeError, match='Not device memory: sample'):
        call()


@pytest.mark.parametrize('kind', ref.TYPES)
@pytest.mark.parametrize('vocabulary', [1, 6, 300, 70000])
def test_verify_infinite_temperatures(qpkg, kind, vocabulary):
    """At temperatures at which all finite logits are as likely, infinite ones still have all of p, also where no other
    token of their row is left: alone, at both ends, throughout, beside finite ones and beside NaN."""
    inf, v = np.inf, vocabulary
    rng = np.random.default_rng(v)
    rows = [np.full(v, x, np.float32) for x in (-inf, -inf, -inf, inf, 0.0, np.nan, -inf, -inf)]
    rows[0][0] = rows[1][-1] = rows[2][0] = rows[2][-1] = rows[4][v // 2] = rows[5][v // 3] = inf
    rows[6][v // 2] = 3.0  # the last one has no token
    logits, tokens, accept, sample, heat = [], [], [], [], []
    for row in rows:
        for token in (0, v - 1, v // 2):
            for t in (inf, 3.4e38, 6e36, 5e36, 1.0):
                logits += [row, rng.standard_normal(v).astype(np.float32)]
                tokens += [0, token]
                accept += [0.25, 0.5]
                sample.append(rng.choice([0, 0.51237, 0.99917]))  # on no border between equal weights
                heat.append(t)
    raw = ref.encode(np.asarray(logits, np.float32), kind)
    given = dict(logits=ref.decode(raw, kind), tokens=np.asarray(tokens), accept=np.asarray(accept, np.float32),
                 sample=np.asarray(sample, np.float32))
    heat = np.asarray(heat, np.float32)
    draft = np.full(raw.shape, 1 / v, np.float32)
    for q in (None, draft):
        with np.errstate(all='ignore'):
            want = ref.verify(**given, draft=q, temperature=heat)
        accepted, following, _ = Drafts(qpkg, raw, given['tokens'], given['accept'], given['sample'], q, temperature=heat,
                                        kind=kind)()
        assert np.array_equal(accepted, want[0])
        assert np.array_equal(following, want[1]), np.flatnonzero(following != want[1])[:5]


@pytest.mark.parametrize('rows', [(1 << 24) - 1, 1 << 24])
def test_rotate_the_most_rows(qpkg, rows):
    """As many rows as a call has at most, of which a few are there; all others, of negative positions, stay."""
    rng = np.random.default_rng(25)
    live = np.unique(np.concatenate(([0, 1, (1 << 23) - 1, 1 << 23, rows - 2, rows - 1], rng.integers(0, rows, 2000))))
    positions = np.full(rows, -1, np.int32)
    positions[live] = rng.integers(0, 5000, live.size)
    raw = np.full((rows, 2), 0x3c00, np.uint16)  # ones
    raw[live] = ref.encode(rng.standard_normal((live.size, 2)), 'f16')
    side = Heads(qpkg, raw, 1, 2, 0)
    got, = rotate(qpkg, [side], [None], positions, np.array([0.37]), False, 1.0, 'f16')
    x = ref.decode(raw[live], 'f16').reshape(-1, 1, 2)
    want, tolerance = ref.rotate(x, positions[live], np.array([0.37]), False, np.float32(1), None, np.float32(1e-6), 'f16')
    off = np.abs(ref.decode(got[live], 'f16').reshape(want.shape) - want)
    assert (off <= tolerance).all(), (off / tolerance).max()
    rest = got.copy()
    rest[live] = raw[live]
    assert np.array_equal(rest, raw)


def test_reservations_on_streams(qpkg):
    """Pages of two pools reserved on streams of their own, beside rotations and verifications, step after step."""
    q, hip, rng = qpkg, Hip(), np.random.default_rng(26)
    lib, n, streams, pools, want = q.load_library(), 300, [], [], []
    for _ in range(2):
        streams.append(ctypes.c_void_p())
        hip.hipStreamCreate(ctypes.byref(streams[-1]))
        given = state(rng, n, 4, 30, 2000, width=40)
        steps = [rng.integers(-5, 6, n) for _ in range(6)]
        on = {name: q.DeviceBuffer.from_array(np.asarray(x, np.int32)) for name, x in dict(
            table=given['table'], held=given['held'], lengths=given['lengths'], count=[len(given['free'])],
            stack=np.pad(given['free'], (0, given['pages'] - len(given['free'])), constant_values=-1),
            offsets=np.zeros(n + 1), positions=np.zeros(3000)).items()}
        changes = [q.DeviceBuffer.from_array(np.asarray(x, np.int32)) for x in steps]
        pools.append((on, changes, q.PagedPool(on['table'].ptr, on['stack'].ptr, on['held'].ptr, on['count'].ptr, None,
                                               given['pages'], 4, n, 40)))
        for x in steps:
            there = ref.reserve(**given, changes=x, room=3000)
            given.update({name: there[name] for name in ('table', 'held', 'free', 'lengths')})
        want.append(there)
    draft = Drafts(q, **random_drafts(rng, 5, 4, 9000, ragged=True))
    alone = draft()
    turned = q.DeviceBuffer.from_array(rng.standard_normal((200, 384)).astype(np.float32))
    place, turns = q.DeviceBuffer.from_array(np.full(200, 7, np.int32)), q.DeviceBuffer.from_array(np.full(32, 0.3))
    for i in range(6):
        for stream, (on, changes, pool) in zip(streams, pools):
            growth = q.PagedGrowth(on['lengths'].ptr, None, changes[i].ptr, on['lengths'].ptr, None, on['held'].ptr,
                                   on['count'].ptr, on['offsets'].ptr, None, on['positions'].ptr, None, 3000)
            ok(q, lib.qwen_gpu_op_paged_reserve(pool, growth, stream))
        draft.enqueue(streams[0])
        heads = q.RotaryHeads(turned.ptr, turned.ptr, None, 384, 64, 384, 64, 6)
        ok(q, lib.qwen_gpu_op_rotate(q.Rotary(turns.ptr, 64, 0, 64, 0, 1, 1e-6), heads, None, place.ptr, 200, streams[1]))
    for stream in streams:
        hip.hipStreamSynchronize(stream)
    assert all(np.array_equal(a, b) for a, b in zip(draft.results(), alone))
    for (on, _, _), there in zip(pools, want):
        for name in ('held', 'lengths', 'offsets', 'positions'):
            assert np.array_equal(on[name].to_array(np.int32, there[name].size), there[name]), name
        assert np.array_equal(on['table'].to_array(np.int32, n * 40).reshape(n, 40), there['table'])
        count = int(on['count'].to_array(np.int32, 1)[0])
        assert np.array_equal(on['stack'].to_array(np.int32, on['stack'].nbytes // 4)[:count], there['free'])
    for stream in streams:
        hip.hipStreamDestroy(stream)

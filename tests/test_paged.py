"""What the paged cache's entry points refuse (CPU: every check of arguments
comes before the device is used), and the arithmetic of their NumPy oracle."""
import ctypes
import sys
from pathlib import Path

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import paged_reference as ref  # noqa: E402

AT = 1 << 20  # stands for device memory; never used


def cache(q, **more):
    fields = dict(keys=AT, values=AT, exponents=None, page_stride=8 * 16 * 128, head_stride=16 * 128, slot_stride=128,
                  pages=4, page_size=16, kv_heads=8, head_dim=128, type=0)
    fields.update(more)
    return q.PagedCache(**fields)


def batch(q, **more):
    fields = dict(table=AT, lengths=AT, offsets=None, seen=None, weights=AT, positions=AT, track_stride=64,
                  sequences=2, table_stride=4, max_length=64, rows=1, total_rows=2)
    fields.update(more)
    return q.PagedBatch(**fields)


def refused(package, message, c=None, b=None, op='append', **call):
    lib = package.load_library()
    c, b = c if c is not None else cache(package), b if b is not None else batch(package)
    given = dict(k=AT, v=AT, k_stride=1024, v_stride=1024, q=AT, q_stride=2048, heads=16, out=AT, out_stride=2048,
                 space=AT, bytes=1 << 30, keep=8, sinks=1, recent=1, n=2 * AT, w=AT, p=AT)
    given.update(call)
    g = given
    if op == 'append':
        status = lib.qwen_gpu_op_paged_append(c, b, g['k'], g['k_stride'], g['v'], g['v_stride'], None)
    elif op == 'attention':
        status = lib.qwen_gpu_op_paged_attention(c, b, g['q'], g['q_stride'], g['heads'], 0.1, g['out'], g['out_stride'],
                                                 g['space'], g['bytes'], None)
    else:
        status = lib.qwen_gpu_op_paged_evict(c, b, g['keep'], g['sinks'], g['recent'], g['n'], g['w'], g['p'],
                                             g['space'], g['bytes'], None)
    assert status == 1
    error = lib.qwen_gpu_last_error().decode()
    assert message in error, error


@pytest.mark.parametrize('op', ['append', 'attention', 'evict'])
@pytest.mark.parametrize('message,fields', [
    ('Null argument: keys', dict(keys=None)), ('Null argument: values', dict(values=None)),
    ('Null argument: exponents', dict(type=2)), ('Unknown paged cache type', dict(type=3)),
    ('head_dim must be', dict(head_dim=96)), ('head_dim must be', dict(head_dim=0)),
    ('Page size must be', dict(page_size=0)), ('Page size must be', dict(page_size=65537)),
    ('needs pages', dict(pages=0)), ('kv_heads must be', dict(kv_heads=0)), ('kv_heads must be', dict(kv_heads=1025)),
    ('let rows overlap', dict(slot_stride=120)), ('let rows overlap', dict(head_stride=15 * 128)),
    ('let rows overlap', dict(page_stride=0)), ('let rows overlap', dict(slot_stride=-128)),
    ('let rows overlap', dict(page_stride=1 << 41)), ('multiples of 16 bytes', dict(page_stride=8 * 16 * 128 + 4))])
def test_caches_refused(qpkg, op, message, fields):
    refused(qpkg, message, cache(qpkg, **fields), op=op)


@pytest.mark.parametrize('op', ['append', 'attention', 'evict'])
@pytest.mark.parametrize('fields', [
    dict(page_stride=1 << 34, pages=1 << 30), dict(page_stride=1 << 40, pages=1 << 24),
    dict(page_stride=1 << 34, pages=(1 << 30) + 1, head_stride=1 << 36),
    dict(page_stride=1 << 40, pages=(1 << 24) + 1, kv_heads=2, head_stride=1 << 40),
    dict(page_stride=1 << 24, pages=(1 << 20) + 1)])
def test_pools_past_64_bits_refused(qpkg, op, fields):
    """Rows further apart than any memory, the products of stride and count that pass 64 bits among them."""
    refused(qpkg, 'let rows overlap or run too far', cache(qpkg, **fields), op=op)


@pytest.mark.parametrize('op', ['append', 'attention', 'evict'])
@pytest.mark.parametrize('message,fields', [
    ('Null argument: table', dict(table=None)), ('Null argument: lengths', dict(lengths=None)),
    ('sequences must be', dict(sequences=0)), ('sequences must be', dict(sequences=65537)),
    ('table needs entries', dict(table_stride=0)), ('max_length must be', dict(max_length=0)),
    ('max_length must be', dict(max_length=65)), ('max_length must be', dict(max_length=1 << 25, table_stride=1 << 25)),
    ('track_stride is below', dict(track_stride=63)), ('track_stride is too large', dict(track_stride=1 << 33))])
def test_batches_refused(qpkg, op, message, fields):
    refused(qpkg, message, b=batch(qpkg, **fields), op=op)


@pytest.mark.parametrize('op', ['append', 'attention'])
@pytest.mark.parametrize('message,fields', [
    ('rows must be', dict(rows=0)), ('rows must be', dict(rows=(1 << 24) + 1)), ('total_rows must be', dict(total_rows=3)),
    ('total_rows must be', dict(total_rows=-1, offsets=AT)),
    ('total_rows must be', dict(total_rows=(1 << 24) + 1, offsets=AT))])
def test_new_rows_refused(qpkg, op, message, fields):
    refused(qpkg, message, b=batch(qpkg, **fields), op=op)


@pytest.mark.parametrize('op,message,call', [
    ('append', 'Null argument: new keys', dict(k=None)), ('append', 'Null argument: new values', dict(v=None)),
    ('append', 'stride below', dict(k_stride=1023)), ('append', 'stride below', dict(v_stride=-1)),
    ('append', 'too large', dict(k_stride=1 << 33)),
    ('attention', 'Null argument: queries', dict(q=None)), ('attention', 'Null argument: out', dict(out=None)),
    ('attention', 'multiple of kv_heads', dict(heads=12)), ('attention', 'multiple of kv_heads', dict(heads=0)),
    ('attention', 'stride below', dict(q_stride=2047)), ('attention', 'stride below', dict(out_stride=0)),
    ('evict', 'Null argument: new_lengths', dict(n=None)), ('evict', 'Null argument: new_weights', dict(w=None)),
    ('evict', 'Null argument: new_positions', dict(p=None)), ('evict', 'keep must be', dict(keep=0)),
    ('evict', 'sinks + recent <= keep', dict(sinks=5, recent=4)), ('evict', 'sinks + recent <= keep', dict(sinks=-1)),
    ('evict', 'sinks + recent <= keep', dict(recent=2 ** 31 - 1)), ('evict', 'overlaps lengths', dict(n=AT)),
    ('evict', 'overlaps lengths', dict(n=AT + 4)), ('evict', 'overlaps weights', dict(w=AT + 4)),
    ('evict', 'overlaps positions', dict(p=AT - 4))])
def test_calls_refused(qpkg, op, message, call):
    refused(qpkg, message, op=op, **call)


@pytest.mark.parametrize('scale', [np.inf, -np.inf, np.nan])
def test_scale_refused(qpkg, scale):
    status = qpkg.load_library().qwen_gpu_op_paged_attention(cache(qpkg), batch(qpkg), AT, 2048, 16, scale, AT, 2048, AT,
                                                             1 << 30, None)
    assert status == 1 and 'scale must be finite' in qpkg.load_library().qwen_gpu_last_error().decode()


@pytest.mark.parametrize('scale', [2.4e38, -3.4e38])
def test_scales_refused_whose_power_of_2_overflows(qpkg, scale):
    """Finite, but not times log2(e): a score of 0 would become NaN."""
    lib = qpkg.load_library()
    status = lib.qwen_gpu_op_paged_attention(cache(qpkg), batch(qpkg), AT, 2048, 16, scale, AT, 2048, AT, 1 << 30, None)
    assert status == 1 and 'scale must be finite, times' in lib.qwen_gpu_last_error().decode()


@pytest.mark.parametrize('refuses,out,stride,out_stride', [
    (True, 0, 4096, 4097), (True, 0, 4096, 2048), (True, 4, 4096, 4096), (True, -4, 4096, 4096),
    (True, 4096, 4096, 4096), (True, 2047, 4096, 4096), (True, 2049, 4096, 4096), (True, -4096, 4096, 4096),
    (True, 2 * 4096 + 2047, 4096, 4096), (True, 2048, 4096, 2048), (True, 2 * 4096, 4096, 4096),
    (False, 0, 4096, 4096), (False, 2048, 4096, 4096), (False, -2048, 4096, 4096), (False, 2 * 4096 + 2048, 4096, 2048),
    (False, 3 * 4096, 4096, 4096), (False, -2 * 2048 - 2048, 4096, 2048), (False, 4096 + 2048, 4096, 4096)])
def test_attention_refuses_outputs_over_other_queries(qpkg, refuses, out, stride, out_stride):
    """Three rows of 2048: other rows and heads of the call may still read what is written there."""
    given = dict(q=AT, q_stride=stride, out=AT + 4 * out, out_stride=out_stride, op='attention')
    message = 'out overlaps' if refuses else 'Not device memory: keys'
    refused(qpkg, message, b=batch(qpkg, sequences=3, total_rows=3), **given)


def test_sizes_refused_that_no_launch_holds(qpkg):
    """Grids and indices would pass 32 bits."""
    wide = dict(sequences=4096, total_rows=4096)
    heads = cache(qpkg, kv_heads=1024, page_stride=1024 * 16 * 128)
    for op in ('append', 'attention', 'evict'):
        refused(qpkg, 'Too many sequences', heads, batch(qpkg, **wide), op=op, k_stride=1 << 20, v_stride=1 << 20,
                q_stride=1 << 20, out_stride=1 << 20, heads=1024)
    long = dict(table_stride=1 << 20, max_length=1 << 24, track_stride=1 << 24, sequences=4096, total_rows=4096)
    refused(qpkg, 'Too many new rows or positions', b=batch(qpkg, **long), op='attention')
    refused(qpkg, 'Too many new rows', cache(qpkg, kv_heads=64, page_stride=64 * 16 * 128),
            batch(qpkg, offsets=AT, total_rows=1 << 23), op='append', k_stride=1 << 13, v_stride=1 << 13)


def test_workspace_of_the_eviction_alone(qpkg):
    """Without query heads: no scores of rows that are not attended, and no rows needed."""
    lib, size = qpkg.load_library(), ctypes.c_size_t()
    evicts = dict(sequences=64, rows=0, total_rows=0, table_stride=512, max_length=8192, track_stride=8192)
    assert lib.qwen_gpu_op_paged_workspace(cache(qpkg), batch(qpkg, **evicts), 0, ctypes.byref(size)) == 0
    assert size.value == 131072 + 64 * 8 * (2 * 4096 + 4) * 4 + 16
    assert lib.qwen_gpu_op_paged_workspace(cache(qpkg), batch(qpkg, **evicts), 16, ctypes.byref(size)) == 1
    assert 'rows must be' in lib.qwen_gpu_last_error().decode()


def test_workspace_of_calls_that_no_launch_holds(qpkg):
    """The size of a call that would be refused is an error as well, and no number that has wrapped around."""
    lib, size = qpkg.load_library(), ctypes.c_size_t()
    long = dict(table_stride=1 << 20, max_length=1 << 24, track_stride=1 << 24)
    for c, b, heads in ((cache(qpkg), batch(qpkg, sequences=4096, total_rows=4096, **long), 16),
                        (cache(qpkg), batch(qpkg, sequences=1, rows=1 << 24, total_rows=1 << 24, **long), 8192),
                        (cache(qpkg, kv_heads=1024, page_stride=1024 * 16 * 128),
                         batch(qpkg, sequences=1, rows=1 << 24, total_rows=1 << 24, **long), 1 << 20)):
        assert lib.qwen_gpu_op_paged_workspace(c, b, heads, ctypes.byref(size)) == 1
        assert 'Too many new rows or positions' in lib.qwen_gpu_last_error().decode() and size.value == 0


def test_evict_needs_what_it_goes_by(qpkg):
    refused(qpkg, 'Null argument: weights', b=batch(qpkg, weights=None), op='evict')
    refused(qpkg, 'Null argument: positions', b=batch(qpkg, positions=None), op='evict')


@pytest.mark.parametrize('shift', [-4, 0, 4])
def test_evict_refuses_new_lengths_among_the_seen(qpkg, shift):
    """Each head of a sequence reads seen[s] while the first one writes new_lengths[s]."""
    refused(qpkg, 'new_lengths overlaps seen', b=batch(qpkg, seen=2 * AT + shift), op='evict')


@pytest.mark.parametrize('op', ['append', 'attention', 'evict'])
def test_host_memory_refused(qpkg, op):
    """Pointers that no kernel could read end in an error, not in a fault."""
    host = np.zeros(1 << 16, np.uint8)
    at = host.ctypes.data + (-host.ctypes.data) % 16
    refused(qpkg, 'Not device memory: keys', cache(qpkg, keys=at, values=at), op=op)


@pytest.mark.parametrize('handle', [1, 2])
def test_stand_in_streams_refused(qpkg, handle):
    """Handles that name the legacy and the per-thread stream are no streams to the runtime's queries."""
    lib, c, b = qpkg.load_library(), cache(qpkg), batch(qpkg)
    for status in (lib.qwen_gpu_op_paged_append(c, b, AT, 1024, AT, 1024, handle),
                   lib.qwen_gpu_op_paged_attention(c, b, AT, 2048, 16, 0.1, AT, 2048, AT, 1 << 30, handle),
                   lib.qwen_gpu_op_paged_evict(c, b, 8, 0, 0, 2 * AT, AT, AT, AT, 1 << 30, handle)):
        assert status == 1 and 'must be NULL or a stream' in lib.qwen_gpu_last_error().decode()


def test_null_descriptions_refused(qpkg):
    lib, c, b = qpkg.load_library(), cache(qpkg), batch(qpkg)
    size = ctypes.c_size_t()
    for status in (lib.qwen_gpu_op_paged_append(None, b, AT, 1024, AT, 1024, None),
                   lib.qwen_gpu_op_paged_attention(c, None, AT, 2048, 16, 0.1, AT, 2048, AT, 1 << 30, None),
                   lib.qwen_gpu_op_paged_evict(None, None, 8, 0, 0, AT, AT, AT, AT, 1 << 30, None),
                   lib.qwen_gpu_op_paged_workspace(c, None, 16, ctypes.byref(size)),
                   lib.qwen_gpu_op_paged_workspace(c, b, 16, None)):
        assert status == 1 and 'Null argument' in lib.qwen_gpu_last_error().decode()


def test_workspace_bytes(qpkg):
    """Known without a device, and enough for the lists of half the longest sequence."""
    lib, size = qpkg.load_library(), ctypes.c_size_t()
    assert lib.qwen_gpu_op_paged_workspace(cache(qpkg), batch(qpkg), 16, ctypes.byref(size)) == 0
    assert size.value >= 2 * 8 * 2 * 32 * 4
    assert lib.qwen_gpu_op_paged_workspace(cache(qpkg), batch(qpkg), 12, ctypes.byref(size)) == 1
    assert 'multiple of kv_heads' in lib.qwen_gpu_last_error().decode()


def test_strides_of_single_axes_do_not_matter(qpkg):
    """An axis of one entry is never stepped along."""
    lib, size = qpkg.load_library(), ctypes.c_size_t()
    c = cache(qpkg, pages=1, page_stride=-3, kv_heads=1, head_stride=1, page_size=16)
    assert lib.qwen_gpu_op_paged_workspace(c, batch(qpkg), 4, ctypes.byref(size)) == 0


def test_oracle_conversions():
    """The oracle's roundings against NumPy's own and the E4M3 format's values."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(2000) * np.exp2(rng.integers(-20, 20, 2000))).astype(np.float32)
    bf16 = ref.from_bits(ref.to_bits(x, 'bf16'), 'bf16')
    assert (np.abs(bf16 - x) <= np.abs(x) * 2.0 ** -8).all()
    assert ref.E4M3[0x7e] == 448 and ref.E4M3[1] == 2.0 ** -9 and ref.E4M3[0x38] == 1 and ref.E4M3[0xb8] == -1
    assert np.isnan(ref.E4M3[[0x7f, 0xff]]).all()
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    assert np.array_equal(ref.to_e4m3(ref.E4M3[codes]), codes)
    assert ref.E4M3[ref.to_e4m3([17, 19, 463.9, 464, 2.0 ** -10, 3 * 2.0 ** -10])].tolist()[:3] == [16, 20, 448]
    assert ref.to_e4m3([2.0 ** -10, 3 * 2.0 ** -10]).tolist() == [0, 2]
    codes, byte = ref.quantise(np.array([[448, 1], [449, 1], [0, 0], [0.875, 0.4375]], np.float32))
    assert (byte.astype(int) - 127).tolist() == [0, 1, -126, -9] and codes[0, 0] == 0x7e and codes[3, 0] == 0x7e


def test_wrapper_checks_arguments(qpkg):
    """Python's PagedKV refuses what it can see before it allocates."""
    with pytest.raises(ValueError, match='type must be'):
        qpkg.PagedKV(1, 1, 1, type='f32')
    with pytest.raises(ValueError, match='needs sequences'):
        qpkg.PagedKV(0, 1, 1)


class Memory:
    """Stands for DeviceBuffer where no device is: host arrays."""

    def __init__(self, nbytes):
        self.nbytes, self.array = int(nbytes), np.zeros(int(nbytes), np.uint8)
        self.ptr = ctypes.c_void_p(self.array.ctypes.data)

    @classmethod
    def from_array(cls, array):
        array = np.ascontiguousarray(array)
        made = cls(array.nbytes)
        made.array[:] = array.reshape(-1).view(np.uint8)
        return made

    def to_array(self, dtype, count):
        return self.array.view(dtype)[:count].copy()


class Library:
    """Stands for the library: keeps each call's name and batch, and fails where told to."""

    def __init__(self):
        self.calls, self.fails = [], False

    def __getattr__(self, name):
        def call(cache, batch, *rest):
            b = batch._obj
            self.calls.append((name, b.rows, b.total_rows, b.max_length,
                               np.ctypeslib.as_array(ctypes.cast(b.offsets, ctypes.POINTER(ctypes.c_int32)),
                                                     (b.sequences + 1,)).copy(),
                               np.ctypeslib.as_array(ctypes.cast(b.lengths, ctypes.POINTER(ctypes.c_int32)),
                                                     (b.sequences,)).copy()))
            return int(self.fails)
        return call

    def qwen_gpu_memcpy_to_device(self, to, host, nbytes):
        self.copied = nbytes
        return 0

    def qwen_gpu_last_error(self):
        return b'it fails'


@pytest.fixture
def paged(qpkg, monkeypatch):
    """A PagedKV of two sequences over stand-ins for memory and library."""
    qpkg.load_library()
    library = Library()
    monkeypatch.setattr(qpkg, 'DeviceBuffer', Memory)
    monkeypatch.setattr(qpkg, '_LIB', library)
    monkeypatch.setattr(qpkg, 'synchronize', lambda: None)
    made = qpkg.PagedKV(2, 8, 4, 16, 2, 64, track=True)
    made.table[:] = np.arange(8).reshape(2, 4)
    return made, library


def new(count):
    return np.zeros((count, 2, 64), np.float32)


def test_wrapper_keeps_its_own_counts(paged):
    """The array of counts is the caller's, who may use it again before the attention."""
    cache, library = paged
    counts = np.array([3, 1], np.int32)
    cache.append(new(4), new(4), counts)
    counts[:] = 0
    cache.attention(np.zeros((4, 2, 64), np.float32))
    name, rows, total, _, offsets, lengths = library.calls[-1]
    assert name == 'qwen_gpu_op_paged_attention' and (rows, total) == (3, 4)
    assert offsets.tolist() == [0, 3, 4] and lengths.tolist() == [3, 1]


@pytest.mark.parametrize('fault', ['library', 'memory', 'synchronize', 'table'])
def test_wrapper_stays_as_it_was_where_an_append_fails(qpkg, paged, monkeypatch, fault):
    """No sequence is longer by rows that were not written, and the next append goes where the failed one would have."""
    cache, library = paged
    cache.append(new(5), new(5), [4, 1])

    def fail(*_):
        raise RuntimeError('it fails')

    with monkeypatch.context() as broken:
        if fault == 'library':
            library.fails = True
        elif fault == 'memory':
            broken.setattr(Memory, 'from_array', fail)
        elif fault == 'synchronize':
            broken.setattr(qpkg, 'synchronize', fail)
        else:
            broken.setattr(cache, 'table', cache.table[:1])
        with pytest.raises((RuntimeError, ValueError)):
            cache.append(new(3), new(3), [1, 2])
    library.fails = False
    assert cache.lengths.tolist() == cache.seen.tolist() == [4, 1]
    cache.attention(np.zeros((5, 2, 64), np.float32))
    assert library.calls[-1][1:3] == (4, 5)
    cache.append(new(3), new(3), [1, 2])
    assert library.calls[-1][5].tolist() == cache.lengths.tolist() == [5, 3]
    cache.append(new(0), new(0), [0, 0])
    assert cache.lengths.tolist() == [5, 3] and cache.attention(np.zeros((0, 2, 64), np.float32)).shape == (0, 2, 64)


@pytest.mark.parametrize('rows,sequences', [(4096, 64), (4096, 256), (2000, 64), (500, 64), (100, 512), (8, 4096),
                                            (1, 4096), (1, 1)])
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_workspace_holds_the_parts_of_split_units_alone(qpkg, rows, sequences, dim):
    """Untracked, whatever the number of new rows: four shares' tiles of sums for each of the 512 workgroups (256 with
    heads of 256) at most, none where there are as many tiles as workgroups; and the eviction's lists."""
    lib, size = qpkg.load_library(), ctypes.c_size_t()
    c = cache(qpkg, head_dim=dim, page_stride=8 * 16 * dim, head_stride=16 * dim, slot_stride=dim)
    b = batch(qpkg, weights=None, positions=None, offsets=AT, sequences=sequences, rows=rows,
              total_rows=min(1 << 24, sequences * rows), table_stride=256, max_length=4096)
    assert lib.qwen_gpu_op_paged_workspace(c, b, 16, ctypes.byref(size)) == 0
    fixed, lists, shares = 131072 + 16, sequences * 8 * (4096 + 4) * 4, 256 if dim == 256 else 512
    tile = 8 if rows * 2 <= 8 else 16
    tiles = 8 * -(-rows * 2 // tile)
    partials = 0 if tiles >= shares else 4 * shares * tile * (dim + 4) * 4
    assert size.value <= fixed + max(lists, partials)


@pytest.mark.parametrize('sequences,rows,total', [(64, 512, 575), (256, 2000, 2255), (8, 512, 512), (64, 1, 64), (1, 4001, 4001)])
def test_workspace_of_tracked_calls_goes_by_the_new_rows(qpkg, sequences, rows, total):
    """A score for each new row, query head and position: one prompt among sequences with a row each takes what the
    rows do, not as if each sequence had a prompt."""
    lib, size = qpkg.load_library(), ctypes.c_size_t()
    b = batch(qpkg, offsets=AT, sequences=sequences, rows=rows, total_rows=total, table_stride=256, max_length=4001,
              track_stride=4096)
    assert lib.qwen_gpu_op_paged_workspace(cache(qpkg), b, 16, ctypes.byref(size)) == 0
    fixed, lists, partials = 131072 + 32, sequences * 8 * (4001 + 4) * 4, 4 * 512 * 16 * (128 + 4) * 4
    scores = total * 16 * (4032 * 4 + 8)
    assert scores < size.value <= fixed + max(lists, partials + scores)


def test_wrapper_calls_go_by_the_lengths(paged):
    """The workspace grows with the longest sequence, not with what the table has room for (64 slots)."""
    cache, library = paged
    cache.append(new(5), new(5), [4, 1])
    cache.attention(np.zeros((5, 2, 64), np.float32))
    cache.evict(3)
    assert {name for name, *_ in library.calls} == {'qwen_gpu_op_paged_append', 'qwen_gpu_op_paged_workspace',
                                                    'qwen_gpu_op_paged_attention', 'qwen_gpu_op_paged_evict'}
    assert [call[3] for call in library.calls] == [4] * 5
    cache.lengths = np.array([0, 0], np.int32)
    cache.evict(3)
    assert library.calls[-1][3] == 1


def test_wrapper_zeroes_the_counters_alone(paged, qpkg):
    """Not gigabytes of scores on the host."""
    cache, library = paged
    cache.append(new(5), new(5), [4, 1])
    library.copied = 0
    cache.attention(np.zeros((5, 2, 64), np.float32))
    assert library.copied == qpkg.PAGED_COUNTER_BYTES
    header = (Path(__file__).resolve().parents[1] / 'include' / 'qwen_gpu.h').read_text()
    assert f'#define QWEN_GPU_PAGED_COUNTER_BYTES {qpkg.PAGED_COUNTER_BYTES}\n' in header

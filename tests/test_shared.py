"""What attention behind shared prefixes refuses, and its workspace (CPU: every
check of arguments comes before the device is used)."""
import ctypes
import sys
from pathlib import Path

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
from test_paged import AT, batch, cache  # noqa: E402


def prefix(q, **more):
    return q.PagedPrefix(**{**dict(lengths=AT, offsets=None, groups=1, max_length=32, max_rest=64), **more})


def untracked(q, **more):
    return batch(q, **{**dict(weights=None, positions=None, track_stride=0), **more})


def refused(q, message, c=None, b=None, p=None, **call):
    lib = q.load_library()
    g = {**dict(queries=AT, q_stride=2048, heads=16, scale=0.1, out=AT, out_stride=2048, space=AT, bytes=1 << 30, stream=None), **call}
    status = lib.qwen_gpu_op_paged_attention_shared(c or cache(q), b or untracked(q), p or prefix(q), g['queries'], g['q_stride'],
                                                    g['heads'], g['scale'], g['out'], g['out_stride'], g['space'], g['bytes'],
                                                    g['stream'])
    assert status == 1
    error = lib.qwen_gpu_last_error().decode()
    assert message in error, error


@pytest.mark.parametrize('message,fields', [
    ('Null argument: keys', dict(keys=None)), ('Unknown paged cache type', dict(type=3)), ('head_dim must be', dict(head_dim=96)),
    ('let rows overlap', dict(slot_stride=120)), ('needs pages', dict(pages=0))])
def test_caches_refused(qpkg, message, fields):
    refused(qpkg, message, cache(qpkg, **fields))


@pytest.mark.parametrize('message,fields', [
    ('tracks no weights', dict(weights=AT, track_stride=64)), ('tracks no weights', dict(positions=AT, track_stride=64)),
    ('Null argument: table', dict(table=None)), ('sequences must be', dict(sequences=0)), ('rows must be', dict(rows=0)),
    ('total_rows must be', dict(total_rows=3)), ('total_rows must be', dict(total_rows=-1, offsets=AT)),
    ('Too many new rows', dict(rows=1 << 24, total_rows=1 << 24, offsets=AT, table_stride=1 << 20, max_length=1 << 24))])
def test_batches_refused(qpkg, message, fields):
    refused(qpkg, message, b=untracked(qpkg, **fields), p=prefix(qpkg, max_rest=1), heads=128 if 'Too' in message else 16)


@pytest.mark.parametrize('message,fields', [
    ('lengths of the prefixes', dict(lengths=None)), ('Groups must be', dict(groups=0)), ('Groups must be', dict(groups=2)),
    ('Groups must be', dict(groups=3, offsets=AT)), ("max_length must be in 0..max_length", dict(max_length=-1)),
    ("max_length must be in 0..max_length", dict(max_length=65)), ('max_rest must be', dict(max_rest=0)),
    ('max_rest must be', dict(max_rest=65))])
def test_prefixes_refused(qpkg, message, fields):
    refused(qpkg, message, p=prefix(qpkg, **fields))


@pytest.mark.parametrize('message,call', [
    ('Null argument: queries', dict(queries=None)), ('Null argument: out', dict(out=None)),
    ('multiple of kv_heads', dict(heads=12)), ('multiple of kv_heads', dict(heads=0)),
    ('multiple of kv_heads', dict(heads=8 * 1025, q_stride=1 << 21, out_stride=1 << 21)),
    ('stride below', dict(q_stride=2047)), ('stride below', dict(out_stride=0)), ('too large', dict(q_stride=1 << 33)),
    ('scale must be finite', dict(scale=np.inf)), ('scale must be finite', dict(scale=np.nan)),
    ('scale must be finite', dict(scale=3e38)), ('The stream must be NULL', dict(stream=1))])
def test_calls_refused(qpkg, message, call):
    refused(qpkg, message, **call)


@pytest.mark.parametrize('sequences,rows,heads,max_length,max_rest', [
    (4096, 1, 16, 0, 64), (4096, 8, 16, 64, 64), (1, 1, 8, 64, 1), (2, 4096, 128, 0, 1), (3, 7, 8 * 1024, 64, 64)])
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_workspace(qpkg, sequences, rows, heads, max_length, max_rest, dim):
    """The parts' sums: one part of a prefix and one behind it at least, with outputs, references and sums in FP32."""
    need = ctypes.c_size_t()
    c = cache(qpkg, head_dim=dim, page_stride=8 * 16 * dim, head_stride=16 * dim, slot_stride=dim)
    b = untracked(qpkg, sequences=sequences, rows=rows, total_rows=sequences * rows)
    status = qpkg.load_library().qwen_gpu_op_paged_shared_workspace(c, b, prefix(qpkg, max_length=max_length, max_rest=max_rest),
                                                                    heads, ctypes.byref(need))
    assert status == 0, qpkg.load_library().qwen_gpu_last_error()
    assert need.value == (2 * sequences * rows * heads * 8 + 15) // 16 * 16 + 2 * sequences * rows * heads * dim * 4


@pytest.mark.parametrize('sequences,rows,total,heads,max_rest', [
    (16, 128, 2048, 32, 32768), (1, 8192, 8192, 16, 1 << 17), (64, 4, 256, 32, 131072), (4096, 1, 4096, 32, 131072),
    (64, 4096, 4159, 16, 65536), (1, 1 << 16, 1 << 16, 16, 1 << 20), (3, 5, 0, 16, 1 << 24)])
def test_workspace_of_long_rests(qpkg, sequences, rows, total, heads, max_rest):
    """However long the rests may be, their parts' sums take 256 MiB, or one part's: a prefix of one part here."""
    need, lib = ctypes.c_size_t(), qpkg.load_library()
    b = untracked(qpkg, sequences=sequences, rows=rows, total_rows=total, offsets=AT, max_length=max_rest, table_stride=1 << 20)
    status = lib.qwen_gpu_op_paged_shared_workspace(cache(qpkg), b, prefix(qpkg, max_rest=max_rest), heads, ctypes.byref(need))
    assert status == 0, lib.qwen_gpu_last_error()
    part = total * heads * (128 * 4 + 8)
    assert need.value <= part + max(part, 1 << 28) + 16


@pytest.mark.parametrize('kv,heads,batch_fields', [
    (256, 256, dict(sequences=4096, rows=256, total_rows=4096, offsets=AT)),  # workgroups behind the prefixes
    (1024, 1024, dict(sequences=1, rows=32, total_rows=(1 << 21) - 1, offsets=AT)),  # of the prefixes
    (8, 8, dict(sequences=1, rows=1 << 24, total_rows=1 << 24))])  # a workgroup for each new row
def test_launches_that_cannot_be(qpkg, kv, heads, batch_fields):
    """A launch has less than 2^32 threads, 2^24 workgroups of 256; what is a little smaller is accepted."""
    need, lib = ctypes.c_size_t(), qpkg.load_library()
    c = cache(qpkg, kv_heads=kv, page_stride=kv * 16 * 128)
    p = prefix(qpkg, max_rest=1)
    given = dict(c=c, p=p, heads=heads, q_stride=heads * 128, out_stride=heads * 128, bytes=1 << 60)
    b = untracked(qpkg, **batch_fields)
    assert lib.qwen_gpu_op_paged_shared_workspace(c, b, p, heads, ctypes.byref(need)) == 1 and need.value == 0
    refused(qpkg, 'Too many new rows or positions', b=b, **given)
    fewer = dict(batch_fields, rows=batch_fields['rows'] * 15 // 16, total_rows=batch_fields['total_rows'] * 15 // 16)
    b = untracked(qpkg, **fewer)
    assert lib.qwen_gpu_op_paged_shared_workspace(c, b, p, heads, ctypes.byref(need)) == 0 and need.value
    refused(qpkg, 'Not device memory', b=b, **given)


def test_wrapper_checks(qpkg):
    paged = object.__new__(qpkg.PagedKV)
    paged.lengths, paged._counts, paged.head_dim = np.zeros(3, np.int32), np.array([1, 0, 2]), 64
    queries = np.zeros((3, 4, 64), np.float32)
    for call in (lambda: paged.attention_shared(queries[:2], 5), lambda: paged.attention_shared(queries, [5, 6], [1]),
                 lambda: paged.attention_shared(queries, [5, 6], [2, 2]), lambda: paged.attention_shared(queries, [5], [-1]),
                 lambda: paged.attention_shared(queries, [-5])):
        with pytest.raises(ValueError):
            call()

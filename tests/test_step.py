"""What the entry points of a step around a paged cache refuse (CPU: every
check of arguments comes before the device is used), the frequencies of
scaled rotations, and the arithmetic of the NumPy oracle."""
import ctypes
import math
import sys
from pathlib import Path

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent))
import step_reference as ref  # noqa: E402

AT = 1 << 40  # stands for device memory; never used
FAR = 1 << 32


def refused(package, message, status):
    assert status == 1
    error = package.load_library().qwen_gpu_last_error().decode()
    assert message in error, error


def rotary(q, **more):
    return q.Rotary(**{**dict(frequencies=AT, dims=128, layout=0, head_dim=128, type=0, magnitude=1, epsilon=1e-6), **more})


def heads(q, place=0, **more):
    at = AT + (2 + 2 * place) * FAR
    return q.RotaryHeads(**{**dict(rows=at, out=at + FAR, norm=None, row_stride=4096, head_stride=128,
                                   out_row_stride=4096, out_head_stride=128, heads=8), **more})


def rotate(q, message, first=None, second=None, positions=AT + FAR, rows=10, stream=None, **more):
    refused(q, message, q.load_library().qwen_gpu_op_rotate(rotary(q, **more), first or heads(q), second, positions, rows,
                                                            stream))


@pytest.mark.parametrize('message,fields', [
    ('Unknown type of rows', dict(type=3)), ('head_dim must be even', dict(head_dim=0, dims=0)),
    ('head_dim must be even', dict(head_dim=513)), ('head_dim must be even', dict(head_dim=514)),
    ('dims must be even', dict(dims=130)), ('dims must be even', dict(dims=3)), ('dims must be even', dict(dims=-2)),
    ('Unknown rotary layout', dict(layout=2)), ('magnitude must be finite', dict(magnitude=math.inf)),
    ('epsilon must be above 0', dict(epsilon=0)), ('epsilon must be above 0', dict(epsilon=math.nan)),
    ('Null argument: frequencies', dict(frequencies=None)), ('Null argument: positions', dict(positions=None)),
    ('rows must be in', dict(rows=-1)), ('rows must be in', dict(rows=(1 << 24) + 1)),
    ('The stream must be NULL', dict(stream=1)), ('The stream must be NULL', dict(stream=2))])
def test_rotations_refused(qpkg, message, fields):
    rotate(qpkg, message, **fields)


@pytest.mark.parametrize('message,fields', [
    ('Null argument: queries', dict(rows=None)), ('Null argument: out of queries', dict(out=None)),
    ('heads must be in', dict(heads=0)), ('heads must be in', dict(heads=4097)),
    ('strides must be in', dict(row_stride=-1)), ('strides must be in', dict(head_stride=(1 << 32) + 1)),
    ('let heads of out overlap', dict(out_head_stride=127)), ('let heads of out overlap', dict(out_row_stride=1023)),
    ('let heads of out overlap', dict(out_row_stride=128, out_head_stride=1279)),
    ('let heads of out overlap', dict(out_row_stride=0)),
    # Over what is read: a byte inside, other strides in place, between the heads of its own rows.
    ('overlaps heads that are read', dict(out=AT + 2 * FAR + 4)),
    ('overlaps heads that are read', dict(out=AT + 2 * FAR, out_row_stride=8192)),
    ('overlaps heads that are read', dict(out=AT + 2 * FAR + 4 * 3200)),
    ('overlaps positions', dict(out=AT + FAR - 4)), ('overlaps frequencies', dict(out=AT + 8)),
    ('overlaps the norm', dict(norm=AT + 3 * FAR + 600))])
def test_heads_refused(qpkg, message, fields):
    rotate(qpkg, message, heads(qpkg, **fields))


def test_keys_refused(qpkg):
    rotate(qpkg, 'Null argument: keys', second=heads(qpkg, 1, rows=None))
    rotate(qpkg, 'heads must be in', second=heads(qpkg, 1, heads=0))
    rotate(qpkg, 'outs of queries and keys overlap', second=heads(qpkg, 1, out=AT + 3 * FAR + 4 * 900))
    rotate(qpkg, 'overlaps heads that are read', second=heads(qpkg, 1, rows=AT + 3 * FAR))
    rotate(qpkg, 'overlaps heads that are read', second=heads(qpkg, 1, out=AT + 2 * FAR))


@pytest.mark.parametrize('first,second', [
    # In place side by side in the rows of a projection, and head by head beside each other.
    (dict(out=AT + 2 * FAR), dict(rows=AT + 2 * FAR + 4096, out=AT + 2 * FAR + 4096)),
    (dict(out=AT + 2 * FAR, head_stride=384, out_head_stride=384, row_stride=3840, out_row_stride=3840),
     dict(rows=AT + 2 * FAR + 512, out=AT + 2 * FAR + 512, head_stride=384, out_head_stride=384, row_stride=3840,
          out_row_stride=3840)),
    # Broadcast rows read, [head][row] written; the values' columns of the same rows written.
    (dict(row_stride=0, out_row_stride=128, out_head_stride=1280), None),
    (dict(out=AT + 2 * FAR + 4 * 1024), None)])
def test_heads_that_keep_apart_are_accepted(qpkg, first, second):
    """All checks of arguments pass; what stands for memory is none."""
    rotate(qpkg, 'Not device memory', heads(qpkg, **first), heads(qpkg, **second) if second else None)


@pytest.mark.parametrize('message,call', [
    ('Unknown rotary scaling', (4, 8, 1e4, 2, 100, 1, 32)), ('dims must be even', (0, 0, 1e4, 1, 0, 0, 0)),
    ('dims must be even', (0, 7, 1e4, 1, 0, 0, 0)), ('dims must be even', (0, 514, 1e4, 1, 0, 0, 0)),
    ('base must be above 1', (0, 8, 1.0, 1, 0, 0, 0)), ('base must be above 1', (0, 8, math.nan, 1, 0, 0, 0)),
    ('factor must be 1 or more', (1, 8, 1e4, 0.5, 0, 0, 0)), ('factor must be 1 or more', (2, 8, 1e4, math.inf, 0, 0, 0)),
    ('more than one pair', (2, 2, 1e4, 2, 0, 0, 0)), ('ramp needs', (3, 8, 1e4, 2, 0, 1, 32)),
    ('ramp needs', (3, 8, 1e4, 2, 100, 32, 32)), ('ramp needs', (3, 8, 1e4, 2, 100, 0, 32))])
def test_frequencies_refused(qpkg, message, call):
    to = (ctypes.c_double * 256)()
    refused(qpkg, message, qpkg.load_library().qwen_gpu_rotary_frequencies(*call, to, None))


@pytest.mark.parametrize('dims,base,factor', [(4, 1e10, 1e150), (4, 1e300, 1e5), (512, 1e300, 1e9)])
def test_scaled_bases_that_no_number_holds(qpkg, dims, base, factor):
    """Their last pair would not turn at all, instead of by 1 / factor of its angle."""
    to = (ctypes.c_double * 256)()
    refused(qpkg, 'base must be finite', qpkg.load_library().qwen_gpu_rotary_frequencies(2, dims, base, factor, 0, 0, 0, to, None))


def test_frequencies_need_room(qpkg):
    refused(qpkg, 'Null argument', qpkg.load_library().qwen_gpu_rotary_frequencies(0, 8, 1e4, 1, 0, 0, 0, None, None))


@pytest.mark.parametrize('dims,base', [(128, 1e6), (2, 1e4), (20, 500.0), (512, 1e4)])
def test_frequencies(qpkg, dims, base):
    i = np.arange(dims // 2)
    plain = base ** (-2.0 * i / dims)
    near = dict(rtol=1e-14, atol=0)
    np.testing.assert_allclose(qpkg.rotary_frequencies(dims, base)[0], plain, **near)
    np.testing.assert_allclose(qpkg.rotary_frequencies(dims, base, 'linear', 4)[0], plain / 4, **near)
    if dims > 2:
        grown, magnitude = qpkg.rotary_frequencies(dims, base, 'base', 8)
        assert grown[0] == 1 and magnitude == 1
        np.testing.assert_allclose(grown[-1], plain[-1] / 8, rtol=1e-13)
    ramp, magnitude = qpkg.rotary_frequencies(dims, base, 'ramp', 16, trained=4096, slow=1, fast=32)
    turns = 4096 * plain / (2 * np.pi)
    share = np.clip((turns - 1) / 31, 0, 1)
    np.testing.assert_allclose(ramp, plain * share + plain / 16 * (1 - share), **near)
    assert magnitude == np.float32(0.1 * math.log(16) + 1)
    # A factor of 1 changes nothing.
    np.testing.assert_allclose(qpkg.rotary_frequencies(dims, base, 'ramp', 1, 4096)[0], plain, **near)


def test_rotation_keeps_lengths_and_relative_positions():
    rng = np.random.default_rng(1)
    f = 1e4 ** (-np.arange(8) / 8)
    a, b = rng.standard_normal((2, 1, 1, 16))
    for interleaved in (False, True):
        def turned(x, position):
            return ref.rotate(x, [position], f, interleaved, 1.0, None, 1e-6)[0][0, 0]
        np.testing.assert_allclose(np.linalg.norm(turned(a, 77)), np.linalg.norm(a))
        np.testing.assert_allclose(turned(a, 100) @ turned(b, 93), turned(a, 1007) @ turned(b, 1000), rtol=1e-9)


# ---- pages and rows ----

def pool(q, **more):
    return q.PagedPool(**{**dict(table=AT, free_pages=AT + FAR, held=AT + 2 * FAR, free_count=AT + 3 * FAR, shared=None,
                                 pages=64, page_size=16, sequences=4, table_stride=8), **more})


def growth(q, **more):
    names = ('lengths', 'seen', 'changes', 'new_lengths', 'new_seen', 'new_held', 'new_free_count', 'offsets',
             'row_sequences', 'row_positions', 'row_slots')
    return q.PagedGrowth(**{**{name: AT + (4 + i) * FAR for i, name in enumerate(names)}, 'total_rows': 16, **more})


@pytest.mark.parametrize('message,fields', [
    ('pages must be', dict(pages=0)), ('pages must be', dict(pages=(1 << 30) + 1)), ('Page size must be', dict(page_size=0)),
    ('Page size must be', dict(page_size=65537)), ('sequences must be', dict(sequences=0)),
    ('sequences must be', dict(sequences=4097)), ('table_stride must be', dict(table_stride=0)),
    ('table_stride must be', dict(table_stride=(1 << 24) + 1)), ('Null argument: table', dict(table=None)),
    ('Null argument: free_pages', dict(free_pages=None)), ('Null argument: held', dict(held=None)),
    ('Null argument: free_count', dict(free_count=None)), ('overlaps free_pages', dict(free_pages=AT + 4)),
    ('table overlaps', dict(held=AT + 4 * 8 * 4 - 4)), ('overlaps shared', dict(shared=AT + FAR))])
def test_pools_refused(qpkg, message, fields):
    refused(qpkg, message, qpkg.load_library().qwen_gpu_op_paged_reserve(pool(qpkg, **fields), growth(qpkg), None))


@pytest.mark.parametrize('message,fields', [
    ('Room for rows', dict(total_rows=-1)), ('Room for rows', dict(total_rows=(1 << 24) + 1)),
    ('come together', dict(seen=None)), ('come together', dict(new_seen=None)),
    ('Null argument: lengths', dict(lengths=None)), ('Null argument: changes', dict(changes=None)),
    ('Null argument: new_lengths', dict(new_lengths=None)), ('Null argument: new_held', dict(new_held=None)),
    ('Null argument: new_free_count', dict(new_free_count=None)), ('Null argument: offsets', dict(offsets=None)),
    ('new_lengths overlaps lengths', dict(new_lengths=AT + 4 * FAR + 4)),
    ('new_lengths overlaps changes', dict(new_lengths=AT + 6 * FAR)),
    ('new_lengths overlaps seen', dict(new_lengths=AT + 5 * FAR)),
    ('offsets overlaps lengths', dict(offsets=AT + 4 * FAR - 16)), ('row_slots overlaps', dict(row_slots=AT + 13 * FAR)),
    ('new_lengths overlaps new_held', dict(new_held=AT + 7 * FAR))])
def test_growths_refused(qpkg, message, fields):
    status = qpkg.load_library().qwen_gpu_op_paged_reserve(pool(qpkg), growth(qpkg, **fields), None)
    if message == 'row_slots overlaps':
        message = 'row_positions overlaps row_slots'
    refused(qpkg, message, status)


def test_growths_in_place_are_accepted(qpkg):
    in_place = growth(qpkg, new_lengths=AT + 4 * FAR, new_seen=AT + 5 * FAR, new_held=AT + 2 * FAR,
                      new_free_count=AT + 3 * FAR)
    refused(qpkg, 'Not device memory: table', qpkg.load_library().qwen_gpu_op_paged_reserve(pool(qpkg), in_place, None))


@pytest.mark.parametrize('message,fields', [
    ('new_lengths overlaps new_seen', dict(seen=AT + 4 * FAR, new_seen=AT + 4 * FAR, new_lengths=AT + 4 * FAR)),
    ('new_lengths overlaps new_held', dict(new_lengths=AT + 4 * FAR, new_held=AT + 4 * FAR)),
    ('new_lengths overlaps held', dict(new_lengths=AT + 2 * FAR))])
def test_results_share_no_place(qpkg, message, fields):
    """Two results in the place of one array, also where that array is given twice."""
    refused(qpkg, message, qpkg.load_library().qwen_gpu_op_paged_reserve(pool(qpkg), growth(qpkg, **fields), None))


def test_reserve_oracle():
    """Worked by hand: pages of 4; sequence 0 grows into its page, 1 ends, 2 takes three pages, 3 wants more than are left,
    4 needs none, 5 has no entries."""
    table = np.array([[0, -1, -1, -1], [1, 2, -1, -1], [-1] * 4, [3, -1, -1, -1], [4, -1, -1, -1], [5, 6, 7, 8]])
    got = ref.reserve(table, [1, 2, 0, 1, 1, 4], [9, 10], [3, 7, 0, 4, 1, 15], [1, -7, 10, 5, 2, 2], 4, 16, 20)
    assert got['lengths'].tolist() == [4, 0, 10, 4, 3, 15] and got['held'].tolist() == [1, 0, 3, 1, 1, 4]
    assert got['table'][2].tolist() == [2, 1, 10, -1] and got['free'].tolist() == [9]
    assert got['offsets'].tolist() == [0, 1, 1, 11, 11, 13, 13]
    assert got['slots'][:13].tolist() == [3, 8, 9, 10, 11, 4, 5, 6, 7, 40, 41, 17, 18]
    # Pages that a sequence lacks for the rows that it has are taken when it grows, not before.
    got = ref.reserve([[-1, -1], [7, -1]], [0, 1], [5, 6], [6, 4], [0, 1], 4, 8, 4)
    assert got['held'].tolist() == [0, 2] and got['table'].tolist() == [[-1, -1], [7, 6]] and got['free'].tolist() == [5]
    got = ref.reserve([[-1, -1], [7, -1]], [0, 1], [5, 6], [6, 4], [1, 1], 4, 8, 4)
    assert got['held'].tolist() == [2, 1] and got['table'].tolist() == [[6, 5], [7, -1]] and got['free'].tolist() == []


# ---- drafts ----

def draft(q, **more):
    names = ('logits', 'draft', 'tokens', 'offsets', 'temperature', 'accept', 'sample')
    return q.Draft(**{**{name: AT + i * FAR for i, name in enumerate(names)}, **dict(
        logit_stride=1000, draft_stride=1000, type=0, vocabulary=1000, sequences=2, rows=3, total_rows=6), **more})


def verify(q, message, given=None, accepted=AT + 10 * FAR, following=AT + 11 * FAR, back=AT + 12 * FAR, space=AT + 13 * FAR,
           size=1 << 20):
    refused(q, message, q.load_library().qwen_gpu_op_verify_draft(given or draft(q), accepted, following, back, space, size,
                                                                  None))


@pytest.mark.parametrize('message,fields', [
    ('Unknown type of logits', dict(type=3)), ('vocabulary must be', dict(vocabulary=0)),
    ('vocabulary must be', dict(vocabulary=(1 << 24) + 1)), ('sequences must be', dict(sequences=0)),
    ('sequences must be', dict(sequences=4097)), ('rows must be', dict(rows=0)), ('rows must be', dict(rows=1025)),
    ('total_rows must be', dict(total_rows=-1)), ('total_rows must be', dict(total_rows=(1 << 20) + 1)),
    ('total_rows must be', dict(offsets=None, total_rows=5)),
    ('Too many logits', dict(vocabulary=1 << 24, total_rows=1 << 20)),
    ('Null argument: logits', dict(logits=None)), ('Null argument: tokens', dict(tokens=None)),
    ('Null argument: accept', dict(accept=None)), ('Null argument: sample', dict(sample=None)),
    ('logits overlap', dict(logit_stride=999)), ('draft overlap', dict(draft_stride=999)),
    ('logits overlap', dict(logit_stride=(1 << 32) + 1))])
def test_drafts_refused(qpkg, message, fields):
    verify(qpkg, message, draft(qpkg, **fields))


@pytest.mark.parametrize('message,call', [
    ('Null argument: next', dict(following=None)), ('Null argument: workspace', dict(space=None)),
    ('Workspace is too small', dict(size=0)), ('accepted overlaps next', dict(accepted=AT + 11 * FAR + 4)),
    ('next overlaps tokens', dict(following=AT + 2 * FAR + 20)), ('back overlaps sample', dict(back=AT + 6 * FAR)),
    ('workspace overlaps', dict(space=AT + 12 * FAR)), ('next overlaps logits', dict(following=AT + 5996))])
def test_verifications_refused(qpkg, message, call):
    if message == 'workspace overlaps':
        message = 'back overlaps workspace'
    verify(qpkg, message, **call)


def test_workspace_of_drafts(qpkg):
    need, lib = ctypes.c_size_t(), qpkg.load_library()
    assert lib.qwen_gpu_op_verify_workspace(draft(qpkg), ctypes.byref(need)) == 0 and 0 < need.value < 4096
    assert lib.qwen_gpu_op_verify_workspace(draft(qpkg, vocabulary=0), ctypes.byref(need)) == 1 and need.value == 0


def test_verify_oracle_follows_the_targets_distribution():
    """Whatever the draft's distribution is, accepted and drawn tokens together have the target's."""
    rng = np.random.default_rng(2)
    target, guess, n = rng.standard_normal(5) * 1.5, rng.dirichlet(np.ones(5)), 20000
    p = ref.probabilities(target, 0.8)
    drawn = rng.choice(5, n, p=guess)
    tokens = np.stack((np.zeros(n, int), drawn), 1).reshape(-1)
    accepted, following = ref.verify(np.broadcast_to(target, (2 * n, 5)), tokens, rng.random(2 * n), rng.random(n),
                                     np.broadcast_to(guess, (2 * n, 5)), None, np.full(n, 0.8))
    first = np.where(accepted == 1, drawn, following)
    # Five shares of 20000 draws: six standard deviations.
    np.testing.assert_allclose(np.bincount(first, minlength=5) / n, p, atol=6 * 0.5 / math.sqrt(n))


def test_wrappers_check_shapes(qpkg):
    x = np.zeros((4, 2, 8), np.float32)
    for call in (lambda: qpkg.rotate(x, x[:3], np.zeros(4), np.ones(4)), lambda: qpkg.rotate(x, None, np.zeros(3), np.ones(4)),
                 lambda: qpkg.rotate(x, x, np.zeros(4), np.ones(4), 'other'), lambda: qpkg.rotate(x[0], None, [0, 1], np.ones(4)),
                 lambda: qpkg.rotary_frequencies(8, scaling='other'),
                 lambda: qpkg.paged_reserve(np.zeros((2, 3)), [1], [], [1, 1], [1, 1], 4, 8, 2),
                 lambda: qpkg.paged_reserve(np.zeros((2, 3)), [1, 1], np.arange(9), [1, 1], [1, 1], 4, 8, 2),
                 lambda: qpkg.verify_draft(np.zeros((3, 5)), [0] * 3, [0] * 3, [0, 0]),
                 lambda: qpkg.verify_draft(np.zeros((3, 5)), [0] * 3, [0] * 3, [0], counts=[2]),
                 lambda: qpkg.verify_draft(np.zeros((3, 5)), [0] * 3, [0] * 3, [0], draft=np.zeros((3, 4)))):
        with pytest.raises(ValueError):
            call()

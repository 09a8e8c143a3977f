"""mt_sched_batch_tables against the requests taken one by one on the host:
whole tables, slot maps, positions and offsets, bit for bit."""
import ctypes as ct

import numpy as np
import pytest

from minitorch_amd import paged_ops
from minitorch_amd.runtime import RawDeviceBuffer, runtime
from shared_prefix import upload

pytestmark = pytest.mark.gpu


def plain(table, lengths, tokens, pages, *, rows, page, prefix):
    """(table, slots, positions, cu): one request after the other."""
    table, columns = table.copy(), table.shape[1]
    slots, positions = np.full(rows, -1, np.int64), np.full(rows, np.float32(-7))
    cu, taken = [0], 0
    for r, length in enumerate(int(x) for x in lengths):
        n = 0 if length < 0 else max(0, min(1 if tokens is None else int(tokens[r]), rows))
        if length >= 0:
            first, last = (min(-(-x // page), columns) for x in (length, length + n))
            if length == 0:
                table[r, last:] = -1
            for c in range(first, last):
                table[r, c] = pages[taken] if taken < len(pages) else -1
                taken += 1
            for i in range(n):
                t, p = cu[-1] + i, length + i
                if t < rows:
                    held = int(table[r, p // page]) if p // page < columns else -1
                    slots[t] = held * page + p % page if held >= 0 else -1
                    positions[t] = np.float32(prefix + p)
        cu.append(cu[-1] + n)
    return table, slots, positions, np.minimum(cu, rows).astype(np.int32)


def check(table, lengths, tokens, pages, *, rows, page=16, prefix=0):
    lengths = np.asarray(lengths, np.int32)
    tokens = None if tokens is None else np.asarray(tokens, np.int32)
    pages = np.asarray(pages, np.int32)
    ref = plain(table, lengths, tokens, pages, rows=rows, page=page, prefix=prefix)
    dev = upload(table)
    slots, positions = RawDeviceBuffer(8 * rows), upload(np.full(rows, np.float32(-7)))
    cu = RawDeviceBuffer(4 * (len(lengths) + 1))
    held = [upload(lengths), None if tokens is None else upload(tokens), upload(pages)]
    for _ in range(2):  # a second call finds what it wrote and writes the same
        paged_ops.batch_tables(dev.ptr, slots.ptr, positions.ptr, cu.ptr, held[0].ptr, held[1] and held[1].ptr,
                               held[2].ptr, b=len(lengths), rows=rows, page_count=len(pages), columns=table.shape[1],
                               page_size=page, prefix_tokens=prefix)
        runtime().synchronize()
        got = (dev.download(np.int32, table.size).reshape(table.shape), slots.download(np.int64, rows),
               positions.download(np.float32, rows), cu.download(np.int32, len(lengths) + 1))
        for name, x, y in zip(('table', 'slots', 'positions', 'cu_tokens'), got, ref):
            assert np.array_equal(x, y), (name, np.argwhere(x != y)[:5])


def random_step(seed, b, page, *, most=100, starting=0.3, new=5, spare=0):
    rng = np.random.default_rng(seed)
    lengths = np.where(rng.random(b) < starting, 0, rng.integers(0, most, b))
    tokens = rng.integers(0, new + 1, b)
    first, last = -(-lengths // page), -(-(lengths + tokens) // page)
    columns = max(1, int(last.max())) + spare
    order = rng.permutation(int(last.sum()) + 3)
    table = rng.integers(0, 9999, (b, columns)).astype(np.int32)  # stale entries
    at = 0
    for r in range(b):
        table[r, :first[r]] = order[at:at + first[r]]
        at += first[r]
    return table, lengths, tokens, order[at:at + int((last - first).sum())]


@pytest.mark.parametrize('page', [8, 16, 32])
@pytest.mark.parametrize('b', [1, 2, 63, 255, 256, 257, 700])
def test_random_steps(b, page):
    table, lengths, tokens, pages = random_step(b + page, b, page, spare=b % 3)
    check(table, lengths, tokens, pages, rows=max(1, int(tokens.sum())), page=page, prefix=b)


@pytest.mark.parametrize('b', [1, 64, 300])
def test_one_token_each(b):
    table, lengths, _, _ = random_step(b, b, 16, spare=2)
    pages = 50000 + np.arange(int((lengths % 16 == 0).sum()))
    check(table, lengths, None, pages, rows=b, prefix=11)


@pytest.mark.parametrize('lengths,tokens', [([0], [20000]), ([5, 0, 0], [9000, 0, 3000]), ([0] * 40, [700] * 40)])
def test_long_requests_spread_over_workgroups(lengths, tokens):
    lengths, tokens = np.array(lengths), np.array(tokens)
    need = -(-(lengths + tokens) // 8)
    table = np.full((len(lengths), int(need.max())), 123456, np.int32)
    pages = np.random.default_rng(3).permutation(int(need.sum()))
    check(table, lengths, tokens, pages, rows=int(tokens.sum()) + 5, page=8)


def test_padding_negative_and_empty_requests():
    table = np.arange(7 * 4, dtype=np.int32).reshape(7, 4)
    check(table, [-1, 0, 17, -5, 0, 64, 3], [4, 0, 3, 9, 18, 1, -2], [100, 101, 102], rows=30, prefix=5)


def test_tokens_past_the_rows_are_dropped():
    table = np.full((3, 6), -1, np.int32)
    check(table, [0, 0, 0], [20, 20, 20], np.arange(6), rows=33)


def test_tokens_past_the_table_have_no_slot():
    table = np.full((3, 2), -1, np.int32)
    check(table, [0, 30, 40], [50, 5, 2], np.arange(2), rows=57)


def test_list_exhausted():
    table = np.full((3, 5), 77, np.int32)
    check(table, [0, 16, 0], [40, 20, 3], [9, 8, 7, 6], rows=63)
    check(table, [0, 16, 0], [40, 20, 3], [], rows=63)


def test_missing_entry_of_a_started_page():
    table = np.array([[5, -1, 0], [2, 3, 4]], np.int32)
    check(table, [20, 20], [3, 13], [8], rows=16)


def test_slots_past_32_bits():
    # pages of a pool of 2^31 rows and more: the slot is a 64-bit number
    table = np.array([[2 ** 31 - 2, 7]], np.int32)
    check(table, [3], [20], [2 ** 31 - 1], rows=20, page=16)
    check(table, [3], [40], [2 ** 31 - 1], rows=40, page=32)


def test_positions_far_behind():
    table = np.full((1, 3), -1, np.int32)
    check(table, [0], [33], [4, 5, 6], rows=33, prefix=2 ** 24 - 16)


def test_many_requests():
    rng = np.random.default_rng(8)
    b = 65535
    lengths = rng.integers(-1, 40, b)
    tokens = rng.integers(0, 3, b)
    table = rng.integers(0, 10 ** 6, (b, 3)).astype(np.int32)
    live = lengths >= 0
    pages = rng.integers(0, 10 ** 6, int((-(-(lengths + tokens) // 16) - -(-lengths // 16))[live].sum()))
    check(table, lengths, tokens, pages, rows=int(tokens[live].sum()) + 1)


def test_lengths_and_tokens_at_their_ends():
    table = np.full((300, 4), 9, np.int32)
    most = 2 ** 31 - 1
    lengths = np.array([most, 10, most - 3, 0, 20] + [0] * 295)
    check(table, lengths, [5, 2, most, most, 3] + [most] * 295, np.arange(9), rows=700)
    check(table, [most] * 300, [most] * 300, np.arange(9), rows=2 ** 13, page=32)


def test_captured_call_replays():
    lib = runtime().lib
    lib.mt_graph_end.argtypes = [ct.POINTER(ct.c_void_p)]
    lib.mt_graph_launch.argtypes = lib.mt_graph_destroy.argtypes = [ct.c_void_p]
    b, rows, page, columns = 300, 2000, 16, 16
    table, slots, positions = RawDeviceBuffer(4 * b * columns), RawDeviceBuffer(8 * rows), RawDeviceBuffer(4 * rows)
    cu, lengths, tokens, pages = (RawDeviceBuffer(4 * n) for n in (b + 1, b, b, 900))
    graph = ct.c_void_p()
    for step in range(4):
        t, L, n, p = random_step(50 + step, b, page, new=5 + step)
        t = np.concatenate([t, np.full((b, columns - t.shape[1]), 77, np.int32)], 1)
        p = np.concatenate([p, np.full(900 - len(p), 5, p.dtype)]).astype(np.int32)
        for buffer, x in ((table, t), (lengths, L), (tokens, n), (pages, p), (positions, np.full(rows, np.float32(-7)))):
            buffer.upload(x.astype(np.int32) if x.dtype == np.int64 else x)
        if not graph:
            assert lib.mt_graph_begin() == 0
            paged_ops.batch_tables(table.ptr, slots.ptr, positions.ptr, cu.ptr, lengths.ptr, tokens.ptr, pages.ptr, b=b,
                                   rows=rows, page_count=900, columns=columns, page_size=page, prefix_tokens=3)
            assert lib.mt_graph_end(ct.byref(graph)) == 0
        for _ in range(2):
            assert lib.mt_graph_launch(graph) == 0
        runtime().synchronize()
        ref = plain(t, L, n, p, rows=rows, page=page, prefix=3)
        got = (table.download(np.int32, t.size).reshape(t.shape), slots.download(np.int64, rows),
               positions.download(np.float32, rows), cu.download(np.int32, b + 1))
        for x, y in zip(got, ref):
            assert np.array_equal(x, y)
    assert lib.mt_graph_destroy(graph) == 0

"""Serving a batch behind a shared prefix against 64-bit results: the append
through a slot map, one-token decode and ragged attention (include/mt_shared.h),
and a run of them together. Tolerances are in tests/tolerances.py."""
import ctypes as ct
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

from minitorch_amd import paged_ops
from minitorch_amd.dtypes import storage_numpy_dtype
from minitorch_amd.runtime import RawDeviceBuffer, runtime
from oracle import paged_oracle as po
from shared_prefix import CODES, SIZE, SharedCase, upload
from tolerances import assert_attention_close

pytestmark = pytest.mark.gpu
TYPES = ['float32', 'float16', 'bfloat16']


# ----------------------------------------------------------------- append ---
def append_case(dtype, dim, *, rows=37, heads=3, page=16, blocks=1, shift=0, layers=2, layer=1, seed=0):
    case = SharedCase(seed, prefix=0, lengths=[0], new=[rows], heads=heads, dim=dim, page_size=page, dtype=dtype,
                      blocks=blocks, shift=shift, layers=layers, layer=layer)
    pos = np.arange(rows)
    slots = case.table[0, pos // page].astype(np.int64) * page + pos % page
    return case, slots


def check_append(case, slots):
    dev = upload(slots)
    paged_ops.paged_append_slots(case.row_ptr(1), case.row_ptr(2), case.slab_table.ptr, dev.ptr, rows=len(slots),
                                 kv_stride=case.stride, **case.common())
    runtime().synchronize()
    image = case.image.copy()
    for t, slot in enumerate(slots):
        page, row = int(slot) // case.page, int(slot) % case.page
        if slot < 0 or page >= case.slabs * case.pps or not case.present[page // case.pps]:
            continue
        for kind in (0, 1):
            image[page // case.pps, case.layer, kind, page % case.pps, :, row] = case.block(1 + kind)[t]
    assert np.array_equal(case.pool_image().view(np.uint8), image.view(np.uint8))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim,blocks', [(64, 1), (64, 3), (128, 3), (80, 1), (36, 3), (5, 1), (1, 3)])
def test_append_slots(dtype, dim, blocks):
    check_append(*append_case(dtype, dim, blocks=blocks))


@pytest.mark.parametrize('page', [8, 32])
@pytest.mark.parametrize('shift', [0, 1])
def test_append_slots_page_sizes_and_unaligned_rows(page, shift):
    check_append(*append_case('bfloat16', 64, page=page, shift=shift, rows=100))


def test_append_slots_skips_what_is_not_there():
    case, slots = append_case('float16', 64, rows=60)
    case.drop_slab(int(case.table[0, 1]) // case.pps)
    end = case.slabs * case.pps * case.page
    slots[[3, 7, 11, 30, 31]] = [-1, end, 2 ** 40 + 5, -2 ** 62, 2 ** 63 - 1]
    check_append(case, slots)


def test_append_slots_of_one_row_and_none():
    case, slots = append_case('float32', 64, rows=1)
    check_append(case, slots)
    case, slots = append_case('float32', 64, rows=9)
    check_append(case, np.full(9, -1, np.int64))


def test_append_slots_same_slot_twice_keeps_one_of_the_rows():
    case, slots = append_case('float16', 64, rows=40)
    slots[25] = slots[4]
    dev = upload(slots)
    paged_ops.paged_append_slots(case.row_ptr(1), case.row_ptr(2), case.slab_table.ptr, dev.ptr, rows=40,
                                 kv_stride=case.stride, **case.common())
    image = case.pool_image()
    page, row = int(slots[4]) // 16, int(slots[4]) % 16
    for kind in (0, 1):
        got = image[page // case.pps, 1, kind, page % case.pps, :, row].view(np.uint16).reshape(-1, 8)
        rows = [case.block(1 + kind)[t].view(np.uint16).reshape(-1, 8) for t in (4, 25)]
        assert ((got == rows[0]).all(1) | (got == rows[1]).all(1)).all()


# ----------------------------------------------------------------- decode ---
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('prefix', [0, 1, 16, 100, 1000])
@pytest.mark.parametrize('b', [1, 4, 33, 70, 150])
def test_decode_batches_and_prefixes(dtype, prefix, b):
    lengths = np.random.default_rng(b).integers(0, 90, b)
    lengths[0] = 0
    SharedCase(b + prefix, prefix=prefix, lengths=lengths, new=[1] * b, dtype=dtype, pps=16).check_decode()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [128, 80, 32, 8, 36, 5, 127])
def test_decode_head_dims(dtype, dim):
    for b, prefix in ((3, 70), (40, 300)):
        SharedCase(dim, prefix=prefix, lengths=[(17 * i) % 60 for i in range(b)], new=[1] * b, dim=dim, dtype=dtype,
                   pps=16).check_decode(context=f'{b} rows')


@pytest.mark.parametrize('page', [8, 16, 32])
@pytest.mark.parametrize('prefix', [7, 8, 31, 33, 255, 257, 513])
def test_decode_page_sizes(page, prefix):
    SharedCase(page + prefix, prefix=prefix, lengths=[0, 7, 8, 15, 16, 31, 32, 63], new=[1] * 8, page_size=page,
               dtype='bfloat16', layers=2, layer=1, pps=5).check_decode()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 128])
def test_decode_long_contexts(dtype, dim):
    # own contexts that are cut into pieces, next to empty ones
    SharedCase(9, prefix=700, lengths=[2500, 0, 1023, 1024, 4000, 5], new=[1] * 6, dim=dim, dtype=dtype,
               pps=32).check_decode()


@pytest.mark.parametrize('b', [1, 3, 300])
def test_decode_long_prefix(b):
    SharedCase(b, prefix=9001, lengths=np.arange(b) % 40, new=[1] * b, dtype='float16', heads=1, pps=64).check_decode()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shift,blocks', [(0, 3), (1, 1), (1, 3)])
def test_decode_strides_and_alignment(dtype, shift, blocks):
    SharedCase(4, prefix=90, lengths=[3, 40, 0], new=[1] * 3, dtype=dtype, heads=3, blocks=blocks,
               shift=shift).check_decode()


@pytest.mark.parametrize('heads', [1, 7, 25])
def test_decode_head_counts(heads):
    SharedCase(5, prefix=260, lengths=[5, 0, 33], new=[1] * 3, heads=heads, dtype='float16').check_decode()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 5])
def test_decode_padding_rows_and_rows_past_the_table(dtype, dim):
    # negative offsets: zero rows, nothing written; past the two columns: NaN
    lengths = np.array([-1, 31, 32, 100, -7])
    case = SharedCase(6, prefix=50, lengths=lengths, new=[1] * 5, dim=dim, dtype=dtype, columns=2, pps=16)
    got = case.check_decode()
    assert (got[[0, 4]] == 0).all() and np.isnan(got[[2, 3]]).all() and np.isfinite(got[1]).all()
    case.lengths[3] = 2 ** 31 - 1
    case.dev_lengths.upload(case.lengths)
    case.clear()
    case.decode()
    assert np.isnan(case.result()[3]).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 128, 5])
def test_decode_missing_pages(dtype, dim):
    # of a request (held, then the new token's) and of the prefix
    case = SharedCase(7, prefix=60, lengths=[40, 40, 40, 48], new=[1] * 4, dim=dim, dtype=dtype)
    case.table[1, 0] = -1
    case.table[2, 2] = 10 ** 6
    case.table[3, 3] = -5
    case.tables()
    got = case.check_decode()
    assert np.isnan(got[1:]).all() and np.isfinite(got[0]).all()
    case = SharedCase(8, prefix=60, lengths=[40, -1], new=[1, 1], dim=dim, dtype=dtype)
    case.prefix_table[1] = -1
    case.tables()
    got = case.check_decode()
    assert np.isnan(got[0]).all() and (got[1] == 0).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_decode_absent_slab(dtype):
    case = SharedCase(9, prefix=40, lengths=[20, 50, 90], new=[1] * 3, dtype=dtype, pps=2)
    case.drop_slab(int(case.table[2, 3]) // 2)
    assert np.isnan(case.check_decode()[2]).all()


def poison(case, table_row, position, kind, head, value):
    page = int(table_row[position // case.page])
    case.image[page // case.pps, case.layer, kind, page % case.pps, head, position % case.page, 3] = \
        po.encode(np.array([value], np.float32), CODES[case.dtype])[0]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 128])
def test_decode_non_finite_values(dtype, dim):
    # an Inf or NaN of V reaches its column of the queries that attend it, with
    # whatever weight; stale rows behind a request's last token reach nobody
    case = SharedCase(10, prefix=80, lengths=[40, 41, 42, 43], new=[1] * 4, dim=dim, dtype=dtype)
    poison(case, case.prefix_table, 33, 1, 0, np.inf)
    poison(case, case.table[1], 5, 1, 1, -np.inf)
    poison(case, case.table[2], 7, 1, 1, np.nan)
    poison(case, case.table[3], 47, 1, 1, np.nan)   # behind the last token
    poison(case, case.table[3], 46, 0, 1, np.inf)
    case.upload_image()
    case.clear()
    case.decode()
    got = case.result()
    assert np.isposinf(got[:, 0, 3]).all() and np.isneginf(got[1, 1, 3]) and np.isnan(got[2, 1, 3])
    others = np.ones((4, 2, dim), bool)
    others[:, 0, 3] = others[1, 1, 3] = others[2, 1, 3] = False
    assert np.isfinite(got[others]).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_decode_large_scores(dtype):
    # scores far apart: the running maximum moves and most weights underflow
    for b in (3, 40):
        SharedCase(11, prefix=500, lengths=[(29 * i) % 100 for i in range(b)], new=[1] * b, dtype=dtype, pps=16,
                   scale=8.0).check_decode()


def test_decode_lowest_scores_in_the_prefix():
    # every prefix key scores far below the own ones, past the range of exp
    case = SharedCase(12, prefix=64, lengths=[20] * 2, new=[1] * 2, dtype='float32')
    q = case.block(0)
    for p in range(64):
        page = int(case.prefix_table[p // 16])
        case.image[page // case.pps, 0, 0, page % case.pps, :, p % 16] = -1e3 * q[0]
    case.upload_image()
    case.check_decode()


@pytest.mark.parametrize('dtype', TYPES)
def test_decode_equals_the_unshared_one(dtype):
    # a prefix of whole pages named in every request's own table instead
    case = SharedCase(13, prefix=160, lengths=[7, 100, 0, 33, 64], new=[1] * 5, dtype=dtype, pps=16)
    shared = case.check_decode()
    table = np.concatenate([np.tile(case.prefix_table, (5, 1)), case.table], 1)
    dev, offsets = upload(table), upload((case.lengths + 160).astype(np.int32))
    case.upload_image()
    case.clear()
    paged_ops.paged_decode_batch(case.out_ptr, case.row_ptr(0), case.row_ptr(1), case.row_ptr(2), case.slab_table.ptr,
                                 dev.ptr, offsets.ptr, b=5, columns=table.shape[1], **case.common())
    got, image = case.result(), case.image.copy()
    case.append(image)
    assert_attention_close(got, case.reference(image), dtype)
    assert_attention_close(shared, case.reference(image), dtype)


# -------------------------------------------------------------- attention ---
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('prefix', [0, 1, 100, 600])
@pytest.mark.parametrize('new,lengths', [
    ([1], [0]), ([5] * 9, [3 * i for i in range(9)]), ([0, 33, 1, 0, 64, 65, 2], [0, 10, 70, 5, 0, 31, 200]),
    ([200, 3], [0, 300])])
def test_attention_shapes(dtype, dim, prefix, new, lengths):
    SharedCase(sum(new) + prefix, prefix=prefix, lengths=lengths, new=new, dim=dim, dtype=dtype, appended=True,
               behind=3, pps=16).check_attend()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [80, 8, 36, 5, 127])
def test_attention_head_dims(dtype, dim):
    SharedCase(dim, prefix=75, lengths=[0, 20, 7], new=[40, 5, 1], dim=dim, dtype=dtype, appended=True).check_attend()


@pytest.mark.parametrize('page', [8, 16, 32])
def test_attention_page_sizes(page):
    SharedCase(page, prefix=77, lengths=[0, 7, 8, 9, 31, 33], new=[9, 8, 33, 1, 2, 70], page_size=page, dtype='bfloat16',
               layers=3, layer=2, pps=3, appended=True).check_attend()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shift,blocks', [(0, 3), (1, 1), (1, 3)])
def test_attention_strides_and_alignment(dtype, shift, blocks):
    SharedCase(4, prefix=90, lengths=[3, 0], new=[20, 3], dtype=dtype, heads=3, blocks=blocks, shift=shift,
               appended=True).check_attend()


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_many_rows_and_long_contexts(dtype):
    new = [3, 1, 40, 7] * 12
    SharedCase(5, prefix=1500, lengths=[(97 * i) % 900 for i in range(48)], new=new, dtype=dtype, heads=1, pps=64,
               appended=True).check_attend()


@pytest.mark.parametrize('dim', [64, 128])
def test_attention_long_own_context_is_cut(dim):
    SharedCase(6, prefix=300, lengths=[4500, 0, 2100], new=[3, 40, 33], dim=dim, dtype='float16', pps=64,
               appended=True).check_attend()


@pytest.mark.parametrize('dim', [64, 5])
def test_attention_padding_and_more_tokens_than_promised(dim):
    # a request of negative length has zero rows; tokens past max_tokens are not written
    case = SharedCase(7, prefix=40, lengths=[-1, 5, 9], new=[4, 20, 6], dim=dim, dtype='float16', appended=True)
    got = case.check_attend()
    assert (got[:4] == 0).all()
    case.clear()
    case.attend(max_tokens=8)
    raw, full = case.result(), got
    blank = po.decode(case.blank, CODES['float16']).reshape(full.shape)
    assert np.array_equal(raw[12:24], blank[12:24])
    keep = np.r_[0:12, 24:30]
    assert_attention_close(raw[keep], case.reference(case.image)[keep], 'float16')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 128, 5])
def test_attention_missing_pages_and_past_the_table(dtype, dim):
    # only the queries that attend a missing page are NaN
    case = SharedCase(8, prefix=33, lengths=[0, 20, 10], new=[50, 40, 40], dim=dim, dtype=dtype, appended=True, pps=16)
    case.table[0, 2] = -1
    case.tables()
    got = case.check_attend()
    assert np.isnan(got[32:50]).all() and np.isfinite(got[:32]).all() and np.isfinite(got[50:]).all()
    case = SharedCase(9, prefix=33, lengths=[0, 20], new=[50, 40], dim=dim, dtype=dtype, columns=2, appended=True, pps=16)
    got = case.check_attend()
    assert np.isfinite(got[:32]).all() and np.isnan(got[32:50]).all() and np.isnan(got[62:]).all()
    case = SharedCase(10, prefix=33, lengths=[0, 20], new=[5, 40], dim=dim, dtype=dtype, appended=True)
    case.prefix_table[2] = 10 ** 8
    case.tables()
    assert np.isnan(case.check_attend()).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 128])
def test_attention_non_finite_values_reach_only_their_readers(dtype, dim):
    # V of a new token is Inf: the queries before it do not see it
    case = SharedCase(11, prefix=50, lengths=[10, 0, 3], new=[40, 70, 1], dim=dim, dtype=dtype, appended=True)
    poison(case, case.table[0], 30, 1, 0, np.inf)
    poison(case, case.table[1], 69, 1, 1, np.nan)
    poison(case, case.table[2], 4, 1, 1, np.nan)     # behind the last token
    poison(case, case.prefix_table, 49, 1, 1, -np.inf)
    case.upload_image()
    case.clear()
    case.attend()
    got = case.result()
    assert np.isfinite(got[:20, 0]).all() and np.isposinf(got[20:40, 0, 3]).all()
    assert np.isneginf(got[:109, 1, 3]).all() and np.isnan(got[109, 1, 3]) and np.isneginf(got[110, 1, 3])
    got[20:40, 0, 3] = got[:, 1, 3] = 0
    assert np.isfinite(got).all()


@pytest.mark.parametrize('cu', [[0, 3, 2, 9], [-4, 3, 8, 400], [5, 5, 5, 5], [2 ** 31 - 1, 0, -2 ** 31, 9]])
def test_attention_wild_offsets_stay_in_bounds(cu):
    # offsets that no step has: rows outside q and out are never touched
    case = SharedCase(12, prefix=40, lengths=[5, 6, 7], new=[3, 3, 3], dtype='float16', appended=True, behind=2)
    case.dev_cu.upload(np.array(cu, np.int32))
    case.attend(max_tokens=9)
    runtime().synchronize()
    assert np.array_equal(case.pool_image().view(np.uint8), case.image.view(np.uint8))


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_of_one_token_each_agrees_with_decode(dtype):
    case = SharedCase(13, prefix=333, lengths=[(37 * i) % 140 for i in range(40)], new=[1] * 40, dtype=dtype, pps=16,
                      appended=True)
    one = case.check_attend()
    two = case.check_decode()
    assert_attention_close(one, two, dtype, ref_rounded=True)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [64, 128, 16])
def test_attention_of_many_requests_most_of_few_tokens(dtype, dim):
    # a table far wider than most contexts: the workgroups look up their items
    b = 300
    new = [(i * 7) % 4 for i in range(b)]
    lengths = [(i * 37) % 60 for i in range(b)]
    new[5], new[290], lengths[17], new[17], lengths[33] = 300, 33, 4075, 9, -1
    case = SharedCase(30, prefix=50, lengths=lengths, new=new, heads=8, dim=dim, page_size=8, dtype=dtype, columns=513, pps=64,
                      appended=True, behind=3)
    case.check_attend()
    case.check_attend(max_tokens=case.rows)


@pytest.mark.parametrize('cu', [[0, 3, 2, 9], [-4, 3, 8, 400], [5, 5, 5, 5], [2 ** 31 - 1, 0, -2 ** 31, 9]])
def test_attention_wild_offsets_stay_in_bounds_with_a_wide_table(cu):
    case = SharedCase(31, prefix=40, lengths=[5, 6, 7], new=[3, 3, 3], heads=12, dtype='float16', appended=True, behind=2,
                      page_size=32, columns=8192)
    case.dev_cu.upload(np.array(cu, np.int32))
    case.dev_lengths.upload(np.array([2 ** 31 - 1, 6, -2 ** 31], np.int32))
    case.attend(max_tokens=9)
    runtime().synchronize()
    assert np.array_equal(case.pool_image().view(np.uint8), case.image.view(np.uint8))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [128, 80])
def test_attention_many_rows_of_wide_heads(dtype, dim):
    case = SharedCase(32, prefix=901, lengths=[0, 100, 31, 0], new=[170, 1, 60, 90], heads=3, dim=dim, dtype=dtype, pps=32,
                      appended=True)
    case.check_attend()


@pytest.mark.parametrize('dtype', TYPES)
def test_prefix_shares_that_cross_tiles(dtype):
    # 24 (head, tile) of 25 units, three units a workgroup: pieces end in one tile and
    # start the next
    case = SharedCase(33, prefix=25 * 128 - 5, lengths=[(5 * i) % 19 for i in range(300)], new=[1] * 300, heads=12, dim=32,
                      dtype=dtype, pps=256)
    case.check_decode()


@pytest.mark.parametrize('page', [8, 32])
def test_prefix_pieces_of_the_most_pages(page):
    case = SharedCase(34, prefix=16384 + 3, lengths=[i % 5 for i in range(260)], new=[1] * 260, heads=32, dim=8,
                      dtype='float16', page_size=page, pps=512)
    case.clear()
    case.decode()
    got, image = case.result(), case.image.copy()
    case.append(image)
    for head in (0, 13, 31):
        k0, v0 = po.image_gather(image, CODES['float16'], case.prefix_table, len(case.prefix_table), 0, head, case.prefix)
        for r in (0, 7, 255, 256, 259):
            k1, v1 = po.image_gather(image, CODES['float16'], case.table[r], case.columns, 0, head, int(case.lengths[r]) + 1)
            q = po.decode(case.block(0), CODES['float16']).reshape(260, 32, 8)[r, head]
            ref = po.attention_fp64(q, np.concatenate([k0, k1]), np.concatenate([v0, v1]))
            assert_attention_close(got[r, head], ref, 'float16', context=f'{head} {r}')


# ------------------------------------------------------------ as one uses ---
def test_calls_repeat_bit_for_bit():
    for dtype in TYPES:
        case = SharedCase(14, prefix=900, lengths=[(37 * i) % 140 for i in range(70)], new=[1] * 70, dtype=dtype, pps=16)
        case.decode()
        first = case.raw()
        for _ in range(3):
            case.clear()
            case.decode()
            assert np.array_equal(case.raw().view(np.uint8), first.view(np.uint8))


@pytest.mark.parametrize('kind', ['decode', 'attend'])
def test_captured_calls_replay(kind):
    # two graphs and eager calls on workspaces of their own; lengths change on
    # the device between the replays
    lib = runtime().lib
    lib.mt_graph_end.argtypes = [ct.POINTER(ct.c_void_p)]
    lib.mt_graph_launch.argtypes = lib.mt_graph_destroy.argtypes = [ct.c_void_p]
    new = [1] * 6 if kind == 'decode' else [3, 1, 0, 40, 2, 5]
    cases = [SharedCase(15 + i, prefix=300 + i, lengths=[10, 0, 60, 33, 5, 90], new=new, dtype='float16',
                        appended=kind == 'attend', pps=16) for i in range(2)]
    graphs = []
    for case in cases:
        getattr(case, kind)()
        runtime().synchronize()
        graph = ct.c_void_p()
        assert lib.mt_graph_begin() == 0
        getattr(case, kind)()
        assert lib.mt_graph_end(ct.byref(graph)) == 0
        graphs.append(graph)
    other = SharedCase(17, prefix=500, lengths=[9] * 20, new=[1] * 20, dtype='bfloat16', pps=16)
    for turn in range(4):
        for case, graph in zip(cases, graphs):
            case.upload_image()
            if turn == 2 and kind == 'decode':  # shorter contexts, one of them padding
                case.lengths[:] = [3, 0, 20, -1, 5, 64]
                case.dev_lengths.upload(case.lengths)
            case.clear()
            assert lib.mt_graph_launch(graph) == 0
            replayed = case.raw()
            other.check_decode()
            case.upload_image()
            case.clear()
            getattr(case, kind)()
            assert np.array_equal(case.raw().view(np.uint8), replayed.view(np.uint8))
            image = case.image.copy()
            case.append(image)
            assert_attention_close(case.result(), case.reference(image), 'float16')
    for graph in graphs:
        assert lib.mt_graph_destroy(graph) == 0


def test_two_host_threads_at_once():
    # a stream and a workspace for each
    cases = [SharedCase(40 + i, prefix=700 + i, lengths=[(37 * r) % 140 for r in range(50)], new=[1] * 50, dtype='bfloat16',
                        pps=16) for i in range(2)]
    images = [case.image.copy() for case in cases]
    for case, image in zip(cases, images):
        case.append(image)

    def steps(case):
        outs = []
        for _ in range(20):
            case.clear()
            case.decode()
            outs.append(case.raw())
        return outs
    with ThreadPoolExecutor(2) as pool:
        both = list(pool.map(steps, cases))
    for case, image, outs in zip(cases, images, both):
        for out in outs[1:]:
            assert np.array_equal(out.view(np.uint8), outs[0].view(np.uint8))
        assert_attention_close(po.decode(outs[0], CODES['bfloat16']).reshape(outs[0].shape), case.reference(image), 'bfloat16')


@pytest.mark.parametrize('dtype,page', [('float32', 16), ('float16', 8), ('bfloat16', 32)])
def test_prompts_then_decode_steps(dtype, page):
    """Prompts of different lengths enter behind a shared prefix, then decode
    together: tables and slots, append and attention each step, pages popped
    from one list."""
    rng = np.random.default_rng(20)
    prompts = [30, 1, 17, 64]
    b, steps, columns, capacity = 4, 20, 4 * 32 // page, sum(prompts) + 9
    # a pool with room for every token; the case's own table is not used
    case = SharedCase(21, prefix=45, lengths=[0] * b, new=[n + steps for n in prompts], heads=3, dtype=dtype, page_size=page,
                      pps=16, blocks=3, columns=columns)
    spare = [p for p in rng.permutation(case.slabs * case.pps) if p not in set(case.prefix_table)]
    h, d = 3, 64
    table = RawDeviceBuffer(4 * b * columns)
    slots, positions = RawDeviceBuffer(8 * capacity), RawDeviceBuffer(4 * capacity)
    cu, out = RawDeviceBuffer(4 * (b + 1)), RawDeviceBuffer(SIZE[dtype] * capacity * h * d)
    lengths, host = np.zeros(b, np.int32), np.full((b, columns), -1, np.int32)
    tokens_seen = [[] for _ in range(b)]  # rows of case.qkv, per request
    row, item, image = 0, SIZE[dtype], case.image.copy()
    for step in range(steps):
        tokens = np.array(prompts if step == 0 else [1] * b, np.int32)
        n = int(tokens.sum())
        taken = [spare.pop() for _ in range(int((-(-(lengths + tokens) // page) - -(-lengths // page)).sum()))]
        held = [upload(lengths), upload(tokens), upload(np.array(taken + [-9], np.int32))]
        rows = capacity if step == 0 else b
        paged_ops.batch_tables(table.ptr, slots.ptr, positions.ptr, cu.ptr, held[0].ptr, held[1].ptr, held[2].ptr, b=b,
                               rows=rows, page_count=len(taken), columns=columns, page_size=page, prefix_tokens=45)
        at = [case.row_ptr(i) + row * case.stride * item for i in range(3)]
        sizes = dict(b=b, prefix_tokens=45, columns=columns)
        if step == 0:
            paged_ops.paged_append_slots(at[1], at[2], case.slab_table.ptr, slots.ptr, rows=n, kv_stride=case.stride,
                                         **case.common())
            space = paged_ops.shared_workspace_bytes(rows=n, max_tokens=64, h=h, d=d, page_size=page, dtype=dtype, **sizes)
            scratch = RawDeviceBuffer(max(16, space))
            paged_ops.paged_shared_attention(out.ptr, at[0], case.slab_table.ptr, case.dev_prefix.ptr, table.ptr,
                                             held[0].ptr, cu.ptr, rows=n, max_tokens=64, q_stride=case.stride,
                                             workspace=scratch.ptr, workspace_bytes=space, **sizes, **case.common())
        else:
            space = paged_ops.shared_workspace_bytes(rows=b, max_tokens=1, h=h, d=d, page_size=page, dtype=dtype, **sizes)
            scratch = RawDeviceBuffer(max(16, space))
            paged_ops.paged_shared_decode(out.ptr, *at, case.slab_table.ptr, case.dev_prefix.ptr, table.ptr, held[0].ptr,
                                          qkv_stride=case.stride, workspace=scratch.ptr, workspace_bytes=space, **sizes,
                                          **case.common())
        runtime().synchronize()
        got = po.decode(out.download(storage_numpy_dtype(dtype), n * h * d), CODES[dtype]).reshape(n, h, d)
        # the same on the host
        q, k, v = (po.decode(case.block(i), CODES[dtype]).reshape(-1, h, d) for i in range(3))
        ref, t = np.zeros((n, h, d)), 0
        for r in range(b):
            for i in range(tokens[r]):
                p = int(lengths[r]) + i
                assert positions.download(np.float32, n)[t] == 45 + p
                tokens_seen[r].append(row + t)
                for head in range(h):
                    pk, pv = po.image_gather(image, CODES[dtype], case.prefix_table, len(case.prefix_table), 0, head, 45)
                    ref[t, head] = po.attention_fp64(q[row + t, head], np.concatenate([pk, k[tokens_seen[r], head]]),
                                                     np.concatenate([pv, v[tokens_seen[r], head]]))
                t += 1
        assert_attention_close(got, ref, dtype, context=f'step {step}')
        lengths += tokens
        row += n

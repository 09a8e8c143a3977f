"""The shared-prefix entries and mt_sched_batch_tables load here (no GPU), export
what their header declares and refuse invalid arguments before any launch."""
import ctypes as ct
import re
from pathlib import Path

import pytest

from minitorch_amd import paged_ops
from minitorch_amd.runtime import I, P, Z, library

ROOT = Path(__file__).resolve().parents[1]


def test_header_symbols_exported():
    names = re.findall(r'^\s*int\s+(mt_\w+)\s*\(', (ROOT / 'include' / 'mt_shared.h').read_text(), re.M)
    lib = library('shared_prefix_kernel')
    assert len(names) == 4 and all(hasattr(lib, n) for n in names)


def _call(lib, name, types, args, changes):
    unknown = set(changes) - set(args)
    assert not unknown, unknown
    f = getattr(library(lib), name)
    f.argtypes, f.restype = types, I
    return f(*{**args, **changes}.values())


TABLES = dict(table=16, slots=16, positions=16, cu=16, lengths=16, tokens=16, pages=16, b=4, rows=9, page_count=5,
              columns=8, page_size=16, prefix=0)


@pytest.mark.parametrize('bad', [
    dict(table=None), dict(slots=None), dict(positions=None), dict(cu=None), dict(lengths=None), dict(pages=None),
    dict(b=0), dict(b=65536), dict(rows=0), dict(rows=2 ** 24), dict(page_count=-1),
    dict(page_count=2 ** 30 + 1), dict(columns=0), dict(columns=2 ** 29 + 1),
    dict(page_size=12), dict(page_size=64), dict(prefix=-1), dict(b=65535, columns=32769),
    dict(b=1, columns=2 ** 27, page_size=16)])
def test_batch_tables_refuses(bad):
    assert _call('sched_kernels', 'mt_sched_batch_tables', [P] * 7 + [I] * 6, TABLES, bad) == 1


APPEND = dict(k=16, v=16, slabs=16, slots=16, rows=9, h=12, d=64, page_size=16, pps=4, slabs_n=8, layer=0, layers=1,
              dtype=1, stride=0)


@pytest.mark.parametrize('bad', [
    dict(k=None), dict(v=None), dict(slabs=None), dict(slots=None), dict(rows=0), dict(h=0), dict(d=0), dict(d=129),
    dict(page_size=4), dict(pps=0), dict(slabs_n=0), dict(pps=2 ** 16, slabs_n=2 ** 15), dict(layer=1), dict(layer=-1),
    dict(layers=0), dict(dtype=3), dict(dtype=-1), dict(stride=767), dict(stride=-1), dict(rows=2 ** 22),
    dict(rows=2 ** 20, stride=2 ** 12)])
def test_append_slots_refuses(bad):
    assert _call('shared_prefix_kernel', 'mt_paged_append_slots', [P] * 4 + [I] * 10, APPEND, bad) == 1


SHAPES = [dict(h=0), dict(d=0), dict(d=129), dict(page_size=12), dict(prefix=-1), dict(columns=0), dict(dtype=3),
          dict(dtype=-1), dict(b=0), dict(b=65535), dict(prefix=2 ** 31 - 100), dict(columns=2 ** 28)]
POOL = [dict(pps=0), dict(slabs_n=0), dict(pps=2 ** 16, slabs_n=2 ** 15), dict(layer=1), dict(layer=-1), dict(layers=0)]

SIZE = dict(rows=8, b=4, h=12, d=64, page_size=16, prefix=100, columns=8, max_tokens=3, dtype=1)


@pytest.mark.parametrize('bad', SHAPES + [dict(rows=0), dict(max_tokens=0), dict(max_tokens=9), dict(rows=2 ** 22)])
def test_workspace_refuses(bad):
    size = ct.c_size_t(7)
    args = dict(SIZE, size=ct.byref(size))
    types = [I] * 9 + [ct.POINTER(ct.c_size_t)]
    assert _call('shared_prefix_kernel', 'mt_paged_shared_workspace_bytes', types, args, bad) == 1
    assert size.value == 7


def test_workspace_refuses_no_result():
    assert _call('shared_prefix_kernel', 'mt_paged_shared_workspace_bytes', [I] * 9 + [P], dict(SIZE, size=None), {}) == 1


DECODE = dict(out=16, q=16, k=16, v=16, slabs=16, prefix_table=16, table=16, offsets=16, b=4, h=12, d=64, page_size=16,
              pps=4, slabs_n=8, prefix=100, columns=8, layer=0, layers=1, dtype=1, stride=0, workspace=16,
              size=1 << 40)


@pytest.mark.parametrize('bad', SHAPES + POOL + [
    dict(out=None), dict(q=None), dict(k=None), dict(v=None), dict(slabs=None), dict(prefix_table=None), dict(table=None),
    dict(offsets=None), dict(stride=767), dict(stride=-1), dict(stride=2 ** 30)])
def test_decode_refuses(bad):
    assert _call('shared_prefix_kernel', 'mt_paged_shared_decode', [P] * 8 + [I] * 12 + [P, Z], DECODE, bad) == 1


ATTEND = dict(out=16, q=16, slabs=16, prefix_table=16, table=16, lengths=16, cu=16, b=4, rows=8, max_tokens=3, h=12, d=64,
              page_size=16, pps=4, slabs_n=8, prefix=100, columns=8, layer=0, layers=1, dtype=1, q_stride=0,
              out_stride=0, workspace=16, size=1 << 40)


@pytest.mark.parametrize('bad', SHAPES + POOL + [
    dict(out=None), dict(q=None), dict(slabs=None), dict(prefix_table=None), dict(table=None), dict(lengths=None),
    dict(cu=None), dict(rows=0), dict(max_tokens=0), dict(max_tokens=9), dict(q_stride=767), dict(q_stride=-1),
    dict(out_stride=767), dict(out_stride=-1), dict(rows=2 ** 20, q_stride=2 ** 12), dict(rows=2 ** 20, out_stride=2 ** 12)])
def test_attention_refuses(bad):
    assert _call('shared_prefix_kernel', 'mt_paged_shared_attention', [P] * 7 + [I] * 15 + [P, Z], ATTEND, bad) == 1


@pytest.mark.parametrize('bad', [dict(workspace=None), dict(workspace=24), dict(size=0)])
def test_attentions_refuse_a_workspace_that_does_not_do(bad):
    lib = 'shared_prefix_kernel'
    assert _call(lib, 'mt_paged_shared_decode', [P] * 8 + [I] * 12 + [P, Z], DECODE, bad) == 1
    assert _call(lib, 'mt_paged_shared_attention', [P] * 7 + [I] * 15 + [P, Z], ATTEND, bad) == 1


# Sizes that a launch's workgroups or the counts of its items do not hold, and ones
# just below them.
PLANS = [(dict(rows=2 ** 22, h=16, d=8), dict(rows=2 ** 22 - 1, h=16, d=8)),
         (dict(rows=2 ** 22, max_tokens=2 ** 22, h=1, b=1, columns=2 ** 15, prefix=0),
          dict(rows=2 ** 22, max_tokens=2 ** 22, h=1, b=1, columns=2 ** 15 - 200, prefix=0)),
         (dict(rows=2 ** 22, h=1, b=1, prefix=2 ** 21), dict(rows=2 ** 22, h=1, b=1, prefix=2 ** 20))]


@pytest.mark.parametrize('bad,good', PLANS)
def test_workspace_refuses_more_than_a_launch_has(bad, good):
    types, size = [I] * 9 + [ct.POINTER(ct.c_size_t)], ct.c_size_t(7)
    args = dict(SIZE, size=ct.byref(size))
    assert _call('shared_prefix_kernel', 'mt_paged_shared_workspace_bytes', types, args, bad) == 1
    assert size.value == 7
    assert _call('shared_prefix_kernel', 'mt_paged_shared_workspace_bytes', types, args, good) == 0
    assert size.value > 7


def test_attention_refuses_more_than_a_launch_has():
    for bad, _ in PLANS:
        assert _call('shared_prefix_kernel', 'mt_paged_shared_attention', [P] * 7 + [I] * 15 + [P, Z], ATTEND,
                     dict(bad, size=1 << 60)) == 1


def test_workspace_grows_with_the_batch():
    args = dict(h=12, d=64, page_size=16, prefix_tokens=2000, columns=8, dtype='float16')
    sizes = [paged_ops.shared_workspace_bytes(rows=b, b=b, max_tokens=1, **args) for b in (1, 8, 64)]
    assert 0 < sizes[0] < sizes[1] < sizes[2]
    # rows that are not whole 16-byte chunks use none
    assert paged_ops.shared_workspace_bytes(rows=8, b=8, max_tokens=1, **dict(args, d=63)) == 0


def test_python_reports_a_refusal():
    with pytest.raises(RuntimeError):
        paged_ops.paged_append_slots(16, 16, 16, 16, rows=0, h=12, d=64, page_size=16, pages_per_slab=4, num_slabs=8,
                                     layer=0, layers=1, dtype='float16')
    with pytest.raises(RuntimeError):
        paged_ops.shared_workspace_bytes(rows=4, b=4, h=12, d=200, page_size=16, prefix_tokens=0, columns=8, max_tokens=1,
                                         dtype='float16')

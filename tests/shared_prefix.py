"""Batches behind a shared prefix for the tests: a page pool whose image holds
the prefix's and the requests' K/V, the calls on its device copy, and the
64-bit result (every query's keys in one list, prefix first)."""
import numpy as np

from minitorch_amd import paged_ops
from minitorch_amd.dtypes import encode_host, storage_numpy_dtype
from minitorch_amd.runtime import DeviceTensor, RawDeviceBuffer, runtime
from oracle import paged_oracle as po
from tolerances import assert_attention_close

CODES = {'float32': po.F32, 'float16': po.F16, 'bfloat16': po.BF16}
SIZE = {'float32': 4, 'float16': 2, 'bfloat16': 2}


def upload(array):
    buffer = RawDeviceBuffer(max(16, array.nbytes))
    buffer.upload(array)
    return buffer


class SharedCase:
    """``lengths[r]`` own tokens of request r before its ``new[r]`` new ones,
    behind ``prefix`` shared tokens. The new tokens' K/V are in the image
    where ``appended``; q/k/v rows are token-major, request after request,
    ``blocks`` matrices of h*d columns side by side (3: a fused projection)."""

    def __init__(self, seed, *, prefix, lengths, new, heads=2, dim=64, page_size=16, dtype='float16', pps=4, layers=1,
                 layer=0, columns=None, blocks=1, appended=False, behind=0, scale=1.0, shift=0):
        rng = np.random.default_rng(seed)
        self.prefix, self.heads, self.dim, self.page, self.dtype = prefix, heads, dim, page_size, dtype
        self.lengths, self.new = np.asarray(lengths, np.int32), np.asarray(new, np.int32)
        self.b, self.rows = len(self.lengths), int(self.new.sum()) + behind
        self.pps, self.layers, self.layer = pps, layers, layer
        total = np.maximum(self.lengths, 0) + self.new
        need = -(-total // page_size)
        shared = -(-prefix // page_size)
        self.columns = max(1, int(need.max())) if columns is None else columns
        pool = shared + int(need.sum()) + 3
        self.slabs = -(-pool // pps)
        order = rng.permutation(self.slabs * pps).astype(np.int32)
        self.prefix_table = order[:shared].copy()
        self.table = np.full((self.b, self.columns), -1, np.int32)
        at = shared
        for r in range(self.b):
            n = min(int(need[r]), self.columns)
            self.table[r, :n] = order[at:at + n]
            at += n
        self.image = self._random(rng, (self.slabs, layers, 2, pps, heads, page_size, dim))
        self.present = np.ones(self.slabs, bool)
        hd = heads * dim
        self.stride = blocks * hd
        self.qkv = self._random(rng, (self.rows, 3 * hd), scale)
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        if appended:
            self.append(self.image)
        # device; ``shift`` elements before the rows break their alignment
        self.blocks, self.shift = blocks, shift
        self.dev_rows = []
        for i in range(1 if blocks == 3 else 3):
            rows = self.qkv if blocks == 3 else self.qkv[:, i * hd:(i + 1) * hd]
            flat = np.concatenate([np.zeros(shift, rows.dtype), np.ascontiguousarray(rows).reshape(-1)])
            self.dev_rows.append(upload(flat))
        self.pool = upload(self.image)
        self.slab_bytes = self.image[0].nbytes
        self.slab_table = upload(np.array([self.pool.ptr + s * self.slab_bytes for s in range(self.slabs)], np.uint64))
        self.tables()
        self.dev_lengths, self.dev_cu = upload(self.lengths), upload(self.cu)
        self.blank = np.full(shift + self.rows * hd, 0x1234, np.uint16).astype(storage_numpy_dtype(dtype))
        self.out = upload(self.blank)
        self.scratch = None

    def _random(self, rng, shape, scale=1.0):
        return encode_host((scale * rng.standard_normal(shape)).astype(np.float32), self.dtype).reshape(shape)

    def tables(self):
        """Uploads the tables (after a change to them)."""
        self.dev_prefix, self.dev_table = upload(self.prefix_table), upload(self.table)

    def upload_image(self):
        self.pool.upload(self.image)

    def drop_slab(self, slab):
        self.present[slab] = False
        addresses = np.array([self.pool.ptr + s * self.slab_bytes for s in range(self.slabs)], np.uint64)
        addresses[~self.present] = 0
        self.slab_table.upload(addresses)

    def block(self, i):
        """Rows of q (0), k (1) or v (2) as [rows, heads, dim]."""
        hd = self.heads * self.dim
        return self.qkv[:, i * hd:(i + 1) * hd].reshape(self.rows, self.heads, self.dim)

    def row_ptr(self, i):
        """Device address of the rows of q (0), k (1) or v (2)."""
        item, hd = SIZE[self.dtype], self.heads * self.dim
        if self.blocks == 3:
            return self.dev_rows[0].ptr + (self.shift + i * hd) * item
        return self.dev_rows[i].ptr + self.shift * item

    @property
    def out_ptr(self):
        return self.out.ptr + self.shift * SIZE[self.dtype]

    def append(self, image):
        """The new tokens' K/V written to an image."""
        for r in range(self.b):
            if self.lengths[r] < 0:
                continue
            for i in range(self.new[r]):
                p = int(self.lengths[r]) + i
                column = p // self.page
                page = int(self.table[r, column]) if column < self.columns else -1
                if not 0 <= page < self.slabs * self.pps or not self.present[page // self.pps]:
                    continue
                for kind in (0, 1):
                    image[page // self.pps, self.layer, kind, page % self.pps, :, p % self.page] = \
                        self.block(1 + kind)[self.cu[r] + i]

    def common(self):
        return dict(h=self.heads, d=self.dim, page_size=self.page, pages_per_slab=self.pps, num_slabs=self.slabs,
                    layer=self.layer, layers=self.layers, dtype=self.dtype)

    def workspace(self, rows, max_tokens):
        size = paged_ops.shared_workspace_bytes(rows=rows, b=self.b, h=self.heads, d=self.dim, page_size=self.page,
                                                prefix_tokens=self.prefix, columns=self.columns, max_tokens=max_tokens,
                                                dtype=self.dtype)
        if size and (self.scratch is None or self.scratch.nbytes < size):
            self.scratch = RawDeviceBuffer(size)
            self.scratch.fill_words(0x7FC00000)
        return dict(workspace=self.scratch.ptr if size else None, workspace_bytes=size)

    def decode(self):
        paged_ops.paged_shared_decode(self.out_ptr, self.row_ptr(0), self.row_ptr(1), self.row_ptr(2),
                                      self.slab_table.ptr, self.dev_prefix.ptr, self.dev_table.ptr, self.dev_lengths.ptr,
                                      b=self.b, prefix_tokens=self.prefix, columns=self.columns, qkv_stride=self.stride,
                                      **self.workspace(self.b, 1), **self.common())

    def attend(self, max_tokens=None):
        most = max(1, int(self.new.max())) if max_tokens is None else max_tokens
        paged_ops.paged_shared_attention(self.out_ptr, self.row_ptr(0), self.slab_table.ptr, self.dev_prefix.ptr,
                                         self.dev_table.ptr, self.dev_lengths.ptr, self.dev_cu.ptr, b=self.b,
                                         rows=self.rows, max_tokens=most, prefix_tokens=self.prefix, columns=self.columns,
                                         q_stride=self.stride, **self.workspace(self.rows, most), **self.common())

    def clear(self):
        self.out.upload(self.blank)

    def raw(self):
        runtime().synchronize()
        return self.out.download(storage_numpy_dtype(self.dtype), self.shift + self.rows * self.heads * self.dim)[
            self.shift:].reshape(self.rows, self.heads, self.dim)

    def result(self):
        return po.decode(self.raw(), CODES[self.dtype]).reshape(self.rows, self.heads, self.dim)

    def pool_image(self):
        return self.pool.download(storage_numpy_dtype(self.dtype), self.image.size).reshape(self.image.shape)

    def reference(self, image):
        """The 64-bit result over an image that holds the new tokens' K/V; rows
        of padding zero, rows behind the last request NaN."""
        code = CODES[self.dtype]
        q = po.decode(self.block(0), code).reshape(self.rows, self.heads, self.dim)
        out = np.full((self.rows, self.heads, self.dim), np.nan)
        for h in range(self.heads):
            shared = po.image_gather(image, code, self.prefix_table, len(self.prefix_table), self.layer, h, self.prefix,
                                     self.present)
            for r in range(self.b):
                rows = slice(int(self.cu[r]), int(self.cu[r + 1]))
                if self.lengths[r] < 0:
                    out[rows, h] = 0
                    continue
                keys = int(self.lengths[r] + self.new[r])
                mine = po.image_gather(image, code, self.table[r], self.columns, self.layer, h, keys, self.present)
                for i, row in enumerate(range(rows.start, rows.stop)):
                    top = int(self.lengths[r]) + i + 1
                    k, v = (np.concatenate([s, m[:top]]) for s, m in zip(shared, mine))
                    out[row, h] = po.attention_fp64(q[row, h], k, v)
        return out

    def check_decode(self, context=''):
        """The output and the whole pool after a decode."""
        self.clear()
        self.decode()
        image = self.image.copy()
        self.append(image)
        got = self.result()
        assert np.array_equal(self.pool_image().view(np.uint8), image.view(np.uint8)), context
        assert_attention_close(got, self.reference(image), self.dtype, context=context)
        return got

    def check_attend(self, context='', max_tokens=None):
        """The output of an attention; the rows behind the last request's and
        the pool stay as they were."""
        self.clear()
        self.attend(max_tokens)
        raw, got = self.raw(), self.result()
        last = int(self.cu[-1])
        assert_attention_close(got[:last], self.reference(self.image)[:last], self.dtype, context=context)
        blank = self.blank[self.shift:].reshape(raw.shape)
        assert np.array_equal(raw[last:].view(np.uint8), blank[last:].view(np.uint8)), context
        assert np.array_equal(self.pool_image().view(np.uint8), self.image.view(np.uint8)), context
        return got

"""Serving a batch whose requests share a long prefix, as timed cases.

Four operators, over the sizes that the framework's configurations, tests and
benchmark use:

* ``tables``: a step's block tables, slot map, positions and token offsets from
  the requests' lengths, on the device (``paged_ops.batch_tables``).
* ``append``: a step's K/V rows written to their pages through a slot map
  (``paged_ops.paged_append_slots``).
* ``decode``: one token per request, appended and attended over the shared prefix
  and the request's own pages (``paged_ops.paged_shared_decode``).
* ``attend``: several new tokens per request, already appended, attended over the
  shared prefix and, causally, the request's own pages
  (``paged_ops.paged_shared_attention``).

Where ``own`` is false ``run`` computes them in elementary torch operations.
Lengths are the quantiles of the stated distribution, dealt to the requests in an
order drawn from the seed, so that every seed asks for the same amount of work.
"""
import math

import numpy as np
import torch

own = False

TORCH_DTYPE = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
SIZE = {'float32': 4, 'float16': 2, 'bfloat16': 2}
PAGES_PER_SLAB = 64


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # a decode step of the headline batch: 64 requests, one token each
        dict(name='tables 64 decode', op='tables', kind='decode', batch=64, page=16, columns=64, low=127, high=1023,
             prefix=2048, pad=0),
        # a step of the steady-state serving run: 96 requests decode while 32 prompts enter; padded to a fixed row count
        dict(name='tables 128 mixed', op='tables', kind='mixed', batch=128, page=16, columns=64, low=16, high=512,
             prefix=1000, pad=250),
        # a long-context batch admitted at once: 512 prompts up to 8192 tokens
        dict(name='tables 512 prompts', op='tables', kind='prompts', batch=512, page=16, columns=512, low=1, high=8192,
             prefix=0, pad=0),
        # the decode step's K/V rows, column blocks of a fused projection
        dict(name='append 64 fp16', op='append', tokens=64, heads=12, dim=64, page=16, dtype='float16', fused=True, pad=0),
        # the rows of many prompts together, GPT-2-XL heads, behind them rows of padding
        dict(name='append 5001 bf16', op='append', tokens=5001, heads=25, dim=64, page=32, dtype='bfloat16', fused=False,
             pad=119),
        # the smallest call: four short requests in the default precision behind a short prefix
        dict(name='decode 4 fp32', op='decode', batch=4, heads=12, dim=64, page=16, dtype='float32', prefix=200,
             lengths='uniform', low=7, high=120, fused=False),
        # the headline batch behind a system prompt: GPT-2-small heads
        dict(name='decode 64 fp16', op='decode', batch=64, heads=12, dim=64, page=16, dtype='float16', prefix=2048,
             lengths='uniform', low=1, high=256, fused=True),
        # questions on one long document, of odd length: few own tokens, GPT-2-medium heads
        dict(name='decode 256 bf16', op='decode', batch=256, heads=16, dim=64, page=16, dtype='bfloat16', prefix=16001,
             lengths='lognormal', low=1, high=512, fused=False),
        # the ragged long-context batch behind a prefix: GPT-2-XL heads, own contexts up to 8192
        dict(name='decode 512 bf16 ragged', op='decode', batch=512, heads=25, dim=64, page=32, dtype='bfloat16',
             prefix=8192, lengths='lognormal', low=1, high=8192, fused=False),
        # five tokens per request to be checked at once
        dict(name='attend 32 x 5 fp16', op='attend', batch=32, heads=12, dim=64, page=16, dtype='float16', prefix=2048,
             new_low=5, new_high=5, low=10, high=300),
        # sixteen prompts admitted together behind a system prompt, from empty; DistilGPT-2 heads, default precision
        dict(name='attend 16 prompts fp32', op='attend', batch=16, heads=12, dim=64, page=16, dtype='float32', prefix=700,
             new_low=2, new_high=100, low=0, high=0),
        # longer prompts, wide heads, a long prefix; some requests have a context of their own
        dict(name='attend 24 bf16 wide', op='attend', batch=24, heads=16, dim=128, page=32, dtype='bfloat16', prefix=8100,
             new_low=1, new_high=256, low=0, high=600),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choices(['tables', 'append', 'decode', 'attend'], [3, 2, 5, 4])[0]
    heads, page = rng.choice([12, 16, 25]), rng.choice([8, 16, 16, 32])
    dtype = rng.choice(['float32', 'float16', 'bfloat16'])
    if op == 'tables':
        high = _log(rng, 8, 8192)
        return dict(op=op, kind=rng.choice(['decode', 'mixed', 'prompts']), batch=_log(rng, 1, 512), page=page,
                    columns=-(-(high + 1) // page) + rng.randint(0, 9), low=max(1, high // rng.choice([1, 8, 64])),
                    high=high, prefix=rng.choice([0, _log(rng, 1, 16384)]), pad=rng.choice([0, rng.randint(1, 300)]))
    dim = rng.choice([64, 64, 64, 128, 80, 32, 36 if dtype == 'float32' else 72])
    if op == 'append':
        tokens = _log(rng, 1, 8192)
        while tokens * heads * dim * SIZE[dtype] > 5001 * 25 * 64 * 2:
            tokens = tokens * 2 // 3
        return dict(op=op, tokens=tokens, heads=heads, dim=dim, page=page, dtype=dtype, fused=rng.choice([False, True]),
                    pad=rng.choice([0, rng.randint(1, 100)]))
    if op == 'decode':
        high = _log(rng, 1, 8192)
        case = dict(op=op, batch=_log(rng, 1, 512), heads=heads, dim=dim, page=page, dtype=dtype,
                    prefix=_log(rng, 16, 32768), lengths=rng.choice(['uniform', 'lognormal']),
                    low=max(1, high // rng.choice([1, 8, 64])), high=high, fused=rng.choice([False, True]))
        while case['batch'] > 1 and (work(case)['bytes'] > 1.2e9 or work(case)['flops'] > _most(dtype, 25e9)):
            case['batch'] = case['batch'] * 2 // 3
        return case
    new = _log(rng, 1, 512)
    case = dict(op=op, batch=_log(rng, 1, 64), heads=heads, dim=dim, page=page, dtype=dtype, prefix=_log(rng, 16, 32768),
                new_low=max(1, new // rng.choice([1, 4, 64])), new_high=new, low=0,
                high=rng.choice([0, _log(rng, 1, 2000)]))
    while case['batch'] > 1 and work(case)['flops'] > _most(dtype, 80e9):
        case['batch'] = case['batch'] * 2 // 3
    while case['new_high'] > 1 and work(case)['flops'] > _most(dtype, 80e9):
        case['new_high'] = case['new_high'] * 2 // 3
        case['new_low'] = min(case['new_low'], case['new_high'])
    return case


def _most(dtype, flops):
    """The largest draw of a type: fp32 products run at a sixteenth of the 16-bit rate."""
    return flops / 8 if dtype == 'float32' else flops


# ---------------------------------------------------------------- lengths ---
def _quantiles(n, low, high, kind='uniform'):
    """n lengths in [low, high]: evenly spread, or lognormal about a quarter of
    ``high`` (256 from 1024 tokens on; sigma 1.2 from 4096 on, else 0.8), clipped."""
    u = (np.arange(n) + 0.5) / n
    if kind == 'uniform':
        x = low + u * (high - low)
    else:
        median = 256 if high >= 1024 else max(low, high / 4)
        z = np.array([math.sqrt(2) * _inverse_erf(2 * p - 1) for p in u])
        x = np.exp(math.log(median) + (1.2 if high >= 4096 else 0.8) * z)
        x[-1] = high
    return np.clip(np.round(x), low, high).astype(np.int64)


def _inverse_erf(y):
    """Inverse of erf by bisection."""
    low, high = -4.5, 4.5
    for _ in range(50):
        mid = (low + high) / 2
        low, high = (mid, high) if math.erf(mid) < y else (low, mid)
    return (low + high) / 2


def _requests(case):
    """Committed lengths and new tokens of a case's requests."""
    b = case['batch']
    if case['op'] == 'decode':
        return _quantiles(b, case['low'], case['high'], case['lengths']) - 1, np.ones(b, np.int64)
    if case['op'] == 'attend':
        # the longest new parts belong to the shortest contexts
        return (_quantiles(b, case['low'], case['high']),
                _quantiles(b, case['new_low'], case['new_high'])[::-1].copy())
    kind = 'lognormal' if case['high'] >= 1024 else 'uniform'
    lengths = _quantiles(b, case['low'], case['high'], kind)
    starts = np.zeros(b, bool)
    if case['kind'] == 'mixed':
        starts[::4] = True
    elif case['kind'] == 'prompts':
        starts[:] = True
    return np.where(starts, 0, lengths), np.where(starts, lengths, 1)


def _deal(case, seed):
    lengths, new = _requests(case)
    order = np.random.default_rng([seed, 1]).permutation(len(lengths))
    return lengths[order], new[order]


# ------------------------------------------------------------------- work ---
def work(case):
    if case['op'] == 'append':
        rows = case['tokens']
        return dict(bytes=4 * rows * case['heads'] * case['dim'] * SIZE[case['dtype']] + 8 * (rows + case['pad']), flops=0)
    L, n = _requests(case)
    page, b, rows = case['page'], len(L), int(n.sum())
    if case['op'] == 'tables':
        first, last = -(-L // page), -(-(L + n) // page)
        taken = int((last - first).sum())
        tails = int((case['columns'] - last)[L == 0].sum())
        held = int((L % page != 0).sum())
        # lengths, tokens, pages and the started page's entry read; entries, slots, positions and offsets written
        return dict(bytes=8 * b + 4 * taken + 4 * held + 4 * (taken + tails) + 12 * rows + 8 * case['pad'] + 4 * (b + 1),
                    flops=0)
    s, hd = SIZE[case['dtype']], case['heads'] * case['dim']
    entries = 4 * (-(-case['prefix'] // page) + int((-(-(L + n) // page)).sum()))
    pairs = rows * case['prefix'] + int((n * L + n * (n + 1) // 2).sum())
    if case['op'] == 'decode':
        # cached K and V, q/k/v in, out and the new rows written
        return dict(bytes=(2 * (case['prefix'] + int(L.sum())) + 6 * b) * hd * s + entries + 4 * b, flops=4 * pairs * hd)
    return dict(bytes=(2 * (case['prefix'] + int((L + n).sum())) + 2 * rows) * hd * s + entries + 8 * b, flops=4 * pairs * hd)


# --------------------------------------------------------------- the pool ---
class _Pool:
    """A page pool [slabs, 1 layer, K and V, pages, heads, page, dim] with the
    pages of the prefix and of the requests at random places; cached values
    are N(0, 1)."""

    def __init__(self, case, totals, seed, prefix):
        h, d, page, t = case['heads'], case['dim'], case['page'], TORCH_DTYPE[case['dtype']]
        gen = torch.Generator('cuda').manual_seed(seed)
        need = -(-totals // page)
        shared, mine = -(-prefix // page), int(need.sum())
        self.slabs = -(-(shared + mine + 8) // PAGES_PER_SLAB)
        self.columns = max(1, int(need.max()))
        self.pages = torch.randn((self.slabs, 1, 2, PAGES_PER_SLAB, h, page, d), device='cuda', dtype=t, generator=gen)
        order = torch.randperm(self.slabs * PAGES_PER_SLAB, device='cuda', generator=gen).to(torch.int32)
        table = torch.full((len(totals), self.columns), -1, device='cuda', dtype=torch.int32)
        held = torch.arange(self.columns, device='cuda')[None, :] < torch.from_numpy(need).cuda()[:, None]
        table[held] = order[shared:shared + mine]
        self.table, self.prefix_table = table, order[:max(1, shared)].contiguous()
        slab_bytes = self.pages[0].numel() * self.pages.element_size()
        self.slab_table = (self.pages.data_ptr() + slab_bytes * torch.arange(self.slabs, dtype=torch.int64)).cuda()
        self.gen, self.t, self.page = gen, t, page

    def randn(self, *shape):
        return torch.randn(shape, device='cuda', dtype=self.t, generator=self.gen)

    def common(self, case):
        return dict(h=case['heads'], d=case['dim'], page_size=case['page'], pages_per_slab=PAGES_PER_SLAB,
                    num_slabs=self.slabs, layer=0, layers=1, dtype=case['dtype'])

    def rows(self, table_row, count, kind, dtype, pages=None):
        """K (kind 0) or V (1) [heads, count, dim] of the first tokens of one table row."""
        pos = torch.arange(count, device='cuda')
        page = table_row[pos // self.page].long()
        rows = (self.pages if pages is None else pages)[page // PAGES_PER_SLAB, 0, kind, page % PAGES_PER_SLAB, :,
                                                        pos % self.page]
        return rows.to(dtype).transpose(0, 1).contiguous()


def _write(pages, slot, k, v, page):
    """K/V rows [count, heads, dim] to the pages at the flat slots."""
    physical, row = slot // page, slot % page
    pages[physical // PAGES_PER_SLAB, 0, 0, physical % PAGES_PER_SLAB, :, row] = k
    pages[physical // PAGES_PER_SLAB, 0, 1, physical % PAGES_PER_SLAB, :, row] = v


# ----------------------------------------------------------------- tables ---
def _prepare_tables(case, seed):
    L, n = _deal(case, seed)
    page, b = case['page'], case['batch']
    gen = torch.Generator('cuda').manual_seed(seed)
    first, last = -(-L // page), -(-(L + n) // page)
    order = torch.randperm(int(last.sum()) + 8, device='cuda', generator=gen).to(torch.int32)
    held, rows = int(first.sum()), int(n.sum())
    table = torch.full((b, case['columns']), -1, device='cuda', dtype=torch.int32)
    table[torch.arange(case['columns'], device='cuda')[None, :] < torch.from_numpy(first).cuda()[:, None]] = order[:held]
    taken = int((last - first).sum())
    return dict(op='tables', case=case, table=table, lengths=torch.from_numpy(L.astype(np.int32)).cuda(),
                tokens=torch.from_numpy(n.astype(np.int32)).cuda(), pages=order[held:held + max(1, taken)].contiguous(),
                taken=taken, rows=rows, slots=torch.zeros(rows + case['pad'], device='cuda', dtype=torch.int64),
                positions=torch.zeros(rows + case['pad'], device='cuda'),
                offsets=torch.zeros(b + 1, device='cuda', dtype=torch.int32))


def _run_tables(s):
    case, page = s['case'], s['case']['page']
    out = dict(table=s['table'], slots=s['slots'], positions=s['positions'], offsets=s['offsets'])
    if own:
        from minitorch_amd import paged_ops
        paged_ops.batch_tables(s['table'].data_ptr(), s['slots'].data_ptr(), s['positions'].data_ptr(),
                               s['offsets'].data_ptr(), s['lengths'].data_ptr(), s['tokens'].data_ptr(),
                               s['pages'].data_ptr(), b=case['batch'], rows=s['rows'] + case['pad'],
                               page_count=s['taken'], columns=case['columns'], page_size=page,
                               prefix_tokens=case['prefix'])
        return out
    table, L, n = s['table'], s['lengths'].long(), s['tokens'].long()
    requests = torch.arange(case['batch'], device='cuda')
    first, last = (L + page - 1) // page, (L + n + page - 1) // page
    ends, page_ends = torch.cumsum(n, 0), torch.cumsum(last - first, 0)
    # the requests' new pages, and -1 behind the pages of those that start
    columns = torch.arange(case['columns'], device='cuda')
    table.masked_fill_((L == 0)[:, None] & (columns[None, :] >= last[:, None]), -1)
    if s['taken']:
        r = torch.repeat_interleave(requests, last - first, output_size=s['taken'])
        j = torch.arange(s['taken'], device='cuda') - (page_ends - last + first)[r]
        table[r, first[r] + j] = s['pages'][:s['taken']]
    r = torch.repeat_interleave(requests, n, output_size=s['rows'])
    p = L[r] + torch.arange(s['rows'], device='cuda') - (ends - n)[r]
    s['slots'][:s['rows']] = table[r, p // page].long() * page + p % page
    s['slots'][s['rows']:] = -1
    s['positions'][:s['rows']] = (p + case['prefix']).to(torch.float32)
    s['offsets'][0] = 0
    s['offsets'][1:] = ends
    return out


def _exact_tables(case, s):
    L, n = s['lengths'].cpu().numpy().astype(np.int64), s['tokens'].cpu().numpy().astype(np.int64)
    table, pages, page = s['table'].cpu().numpy().copy(), s['pages'].cpu().numpy(), case['page']
    slots, positions, offsets, taken = [], [], [0], 0
    for r in range(case['batch']):
        first, last = -(-L[r] // page), -(-(L[r] + n[r]) // page)
        if L[r] == 0:
            table[r] = -1
        table[r, first:last] = pages[taken:taken + last - first]
        taken += last - first
        p = np.arange(L[r], L[r] + n[r])
        slots.append(table[r, p // page].astype(np.int64) * page + p % page)
        positions.append(p + case['prefix'])
        offsets.append(offsets[-1] + int(n[r]))
    pad = case['pad']
    return dict(table=torch.from_numpy(table).cuda(),
                slots=torch.from_numpy(np.concatenate(slots + [np.full(pad, -1, np.int64)])).cuda(),
                positions=torch.from_numpy(np.concatenate(positions + [np.zeros(pad)]).astype(np.float64)).cuda(),
                offsets=torch.from_numpy(np.array(offsets, np.int32)).cuda())


# ----------------------------------------------------------------- append ---
def _prepare_append(case, seed):
    tokens, hd = case['tokens'], case['heads'] * case['dim']
    pool = _Pool(case, np.array([tokens]), seed, 0)
    rows = tokens + case['pad']
    # neighbouring tokens of a request lie next to each other in a page; pages lie anywhere
    pos = torch.arange(tokens, device='cuda')
    slots = pool.table[0, pos // case['page']].long() * case['page'] + pos % case['page']
    slots = torch.cat([slots, torch.full((case['pad'],), -1, device='cuda', dtype=torch.int64)])
    blocks = 3 if case['fused'] else 1
    if case['fused']:
        qkv = pool.randn(rows, 3 * hd)
        k, v = qkv[:, hd:2 * hd], qkv[:, 2 * hd:]
    else:
        k, v = pool.randn(rows, hd), pool.randn(rows, hd)
    return dict(op='append', case=case, pool=pool, k=k, v=v, slots=slots, stride=blocks * hd)


def _run_append(s):
    case, pool = s['case'], s['pool']
    rows, h, d = case['tokens'] + case['pad'], case['heads'], case['dim']
    if own:
        from minitorch_amd import paged_ops
        paged_ops.paged_append_slots(s['k'].data_ptr(), s['v'].data_ptr(), pool.slab_table.data_ptr(),
                                     s['slots'].data_ptr(), rows=rows, kv_stride=s['stride'], **pool.common(case))
    else:
        n = case['tokens']
        _write(pool.pages, s['slots'][:n], s['k'][:n].reshape(n, h, d), s['v'][:n].reshape(n, h, d), case['page'])
    return dict(pages=pool.pages)


def _exact_append(case, s):
    pages = s['pool'].pages.clone()
    n, h, d = case['tokens'], case['heads'], case['dim']
    _write(pages, s['slots'][:n], s['k'][:n].reshape(n, h, d), s['v'][:n].reshape(n, h, d), case['page'])
    return dict(pages=pages)


# ------------------------------------------------- attention, plain form ---
def _join(parts):
    """The softmax over keys whose parts are (max, sum, weighted values)."""
    top = parts[0][0]
    for m, _, _ in parts[1:]:
        top = torch.maximum(top, m)
    total = sum(l * torch.exp(m - top) for m, l, _ in parts)
    acc = sum(o * torch.exp(m - top) for m, _, o in parts)
    return acc / total


def _part(q, k, v, hidden=None):
    """Scores of queries [heads, n, dim] over keys [heads, m, dim] as (max, sum, weighted values)."""
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(q.shape[2])
    if hidden is not None:
        scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(2, keepdim=True)
    weights = torch.exp(scores - top)
    return top, weights.sum(2, keepdim=True), torch.bmm(weights, v)


def _flat(counts, total):
    """The request of each of ``total`` items, ``counts`` items a request, and the item's index in it."""
    r = torch.repeat_interleave(torch.arange(len(counts), device='cuda'), counts, output_size=total)
    return r, torch.arange(total, device='cuda') - (torch.cumsum(counts, 0) - counts)[r]


def _gather(pool, r, pos, kind):
    """K (kind 0) or V (1) [.., heads, dim] of tokens ``pos`` of the requests ``r``, in 32 bits."""
    page = pool.table[r, pos // pool.page].clamp(min=0).long()
    return pool.pages[page // PAGES_PER_SLAB, 0, kind, page % PAGES_PER_SLAB, :, pos % pool.page].to(torch.float32)


def _single_rows(pool, q, lengths, keys):
    """One query [heads, dim] per request over its own ``keys`` in all: every
    (request, key) pair in one list, summed by request."""
    r, pos = _flat(lengths + 1, keys)
    scores = (q[r] * _gather(pool, r, pos, 0)).sum(2) / math.sqrt(q.shape[2])
    top = torch.full(q.shape[:2], -math.inf, device='cuda')
    top.scatter_reduce_(0, r[:, None].expand_as(scores), scores, 'amax')
    weights = torch.exp(scores - top[r])
    total = torch.zeros_like(top).index_add_(0, r, weights)
    acc = torch.zeros_like(q).index_add_(0, r, weights[:, :, None] * _gather(pool, r, pos, 1))
    return [x.transpose(0, 1).contiguous() for x in (top[:, :, None], total[:, :, None], acc)]


def _padded_rows(pool, q, lengths, new, most_new, most_keys):
    """Several queries per request over their own keys, causally: requests
    padded to the longest."""
    rows, h, d = q.shape
    b = len(lengths)
    r, i = _flat(new, rows)
    queries = torch.zeros((b, most_new, h, d), device='cuda')
    queries[r, i] = q
    pos = torch.arange(most_keys, device='cuda')[None, :].expand(b, most_keys)
    k, v = (_gather(pool, torch.arange(b, device='cuda')[:, None], pos, kind).transpose(1, 2).reshape(b * h, most_keys, d)
            for kind in (0, 1))
    last = lengths[:, None] + torch.arange(most_new, device='cuda')[None, :]
    hidden = (pos[:, None, :] > last[:, :, None])[:, None].expand(b, h, most_new, most_keys)
    parts = _part(queries.transpose(1, 2).reshape(b * h, most_new, d), k, v,
                  hidden.reshape(b * h, most_new, most_keys))
    return [x.reshape(b, h, most_new, -1)[r, :, i].transpose(0, 1).contiguous() for x in parts]


def _shared_plain(pool, prefix, q, part):
    """Attention of query rows [rows, heads, dim]: the prefix for all rows in
    one product, joined with ``part`` of the rows' own keys."""
    queries = q.transpose(0, 1).contiguous()
    shared = _part(queries, *(pool.rows(pool.prefix_table, prefix, kind, torch.float32) for kind in (0, 1)))
    return _join([shared, part]).transpose(0, 1).to(pool.t)


def _shared_exact(pool, pages, prefix, q, lengths, new):
    """The same rows in 64 bits: each request's keys in one piece, head by head."""
    rows, h, d = q.shape
    out, at = torch.empty((rows, h, d), device='cuda', dtype=torch.float64), 0
    shared = [pool.rows(pool.prefix_table, prefix, kind, torch.float64, pages) for kind in (0, 1)]
    for r, (length, n) in enumerate(zip(lengths, new)):
        k, v = (torch.cat([shared[kind], pool.rows(pool.table[r], length + n, kind, torch.float64, pages)], 1)
                for kind in (0, 1))
        last = prefix + length + torch.arange(n, device='cuda')
        for head in range(h):
            logits = (q[at:at + n, head].double() @ k[head].t().contiguous()) / math.sqrt(d)
            logits.masked_fill_(torch.arange(k.shape[1], device='cuda')[None, :] > last[:, None], -math.inf)
            out[at:at + n, head] = torch.softmax(logits, 1) @ v[head]
        at += n
    return out


# ----------------------------------------------------------------- decode ---
def _prepare_decode(case, seed):
    L, n = _deal(case, seed)
    pool = _Pool(case, L + n, seed, case['prefix'])
    b, h, d = case['batch'], case['heads'], case['dim']
    if case['fused']:
        qkv = pool.randn(b, 3 * h * d)
        q, k, v = (qkv[:, i * h * d:(i + 1) * h * d] for i in range(3))
    else:
        q, k, v = (pool.randn(b, h * d) for _ in range(3))
    s = dict(op='decode', case=case, pool=pool, lengths=[int(x) for x in L], q=q, k=k, v=v,
             offsets=torch.from_numpy(L.astype(np.int32)).cuda(),
             out=torch.empty((b, h, 1, d), device='cuda', dtype=pool.t))
    if own:
        from minitorch_amd import paged_ops
        size = paged_ops.shared_workspace_bytes(rows=b, b=b, h=h, d=d, page_size=case['page'],
                                                prefix_tokens=case['prefix'], columns=pool.columns, max_tokens=1,
                                                dtype=case['dtype'])
        s['workspace'] = torch.empty(max(1, size), device='cuda', dtype=torch.uint8)
        s['args'] = dict(b=b, prefix_tokens=case['prefix'], columns=pool.columns, workspace=s['workspace'].data_ptr(),
                         workspace_bytes=size, qkv_stride=(3 if case['fused'] else 1) * h * d, **pool.common(case))
    return s


def _new_slots(s):
    pool, pos = s['pool'], s['offsets'].long()
    return pool.table[torch.arange(len(pos), device='cuda'), pos // pool.page].long() * pool.page + pos % pool.page


def _run_decode(s):
    case, pool = s['case'], s['pool']
    if own:
        from minitorch_amd import paged_ops
        paged_ops.paged_shared_decode(s['out'].data_ptr(), s['q'].data_ptr(), s['k'].data_ptr(), s['v'].data_ptr(),
                                      pool.slab_table.data_ptr(), pool.prefix_table.data_ptr(), pool.table.data_ptr(),
                                      s['offsets'].data_ptr(), **s['args'])
        return dict(out=s['out'], pages=pool.pages)
    b, h, d = case['batch'], case['heads'], case['dim']
    q, k, v = (s[x].reshape(b, h, d) for x in 'qkv')
    _write(pool.pages, _new_slots(s), k, v, case['page'])
    q = q.to(torch.float32)
    out = _shared_plain(pool, case['prefix'], q, _single_rows(pool, q, s['offsets'].long(), sum(s['lengths']) + b))
    return dict(out=out.reshape(b, h, 1, d), pages=pool.pages)


def _exact_decode(case, s):
    b, h, d = case['batch'], case['heads'], case['dim']
    pages = s['pool'].pages.clone()
    q, k, v = (s[x].reshape(b, h, d) for x in 'qkv')
    _write(pages, _new_slots(s), k, v, case['page'])
    out = _shared_exact(s['pool'], pages, case['prefix'], q, s['lengths'], [1] * b)
    return dict(out=out.reshape(b, h, 1, d), pages=pages)


# ----------------------------------------------------------------- attend ---
def _prepare_attend(case, seed):
    L, n = _deal(case, seed)
    pool = _Pool(case, L + n, seed, case['prefix'])
    rows, h, d = int(n.sum()), case['heads'], case['dim']
    s = dict(op='attend', case=case, pool=pool, lengths=[int(x) for x in L], new=[int(x) for x in n],
             q=pool.randn(rows, h, d), out=torch.empty((rows, h, d), device='cuda', dtype=pool.t),
             committed=torch.from_numpy(L.astype(np.int32)).cuda(),
             offsets=torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).cuda())
    if own:
        from minitorch_amd import paged_ops
        sizes = dict(rows=rows, b=case['batch'], max_tokens=int(n.max()), prefix_tokens=case['prefix'],
                     columns=pool.columns)
        size = paged_ops.shared_workspace_bytes(h=h, d=d, page_size=case['page'], dtype=case['dtype'], **sizes)
        s['workspace'] = torch.empty(max(1, size), device='cuda', dtype=torch.uint8)
        s['args'] = dict(workspace=s['workspace'].data_ptr(), workspace_bytes=size, **sizes, **pool.common(case))
    return s


def _run_attend(s):
    case, pool = s['case'], s['pool']
    if own:
        from minitorch_amd import paged_ops
        paged_ops.paged_shared_attention(s['out'].data_ptr(), s['q'].data_ptr(), pool.slab_table.data_ptr(),
                                         pool.prefix_table.data_ptr(), pool.table.data_ptr(), s['committed'].data_ptr(),
                                         s['offsets'].data_ptr(), **s['args'])
        return s['out']
    q, L = s['q'].to(torch.float32), s['committed'].long()
    most = max(length + n for length, n in zip(s['lengths'], s['new']))
    return _shared_plain(pool, case['prefix'], q,
                         _padded_rows(pool, q, L, s['offsets'].diff().long(), max(s['new']), most))


def _exact_attend(case, s):
    return _shared_exact(s['pool'], s['pool'].pages, case['prefix'], s['q'], s['lengths'], s['new'])


# -------------------------------------------------------------- interface ---
_PREPARE = dict(tables=_prepare_tables, append=_prepare_append, decode=_prepare_decode, attend=_prepare_attend)
_RUN = dict(tables=_run_tables, append=_run_append, decode=_run_decode, attend=_run_attend)
_EXACT = dict(tables=_exact_tables, append=_exact_append, decode=_exact_decode, attend=_exact_attend)


def prepare(case, seed):
    state = _PREPARE[case['op']](case, seed)
    # the framework launches on the calling thread's own stream, torch on its
    # default one: the inputs are there before the first call
    torch.cuda.synchronize()
    return state


def run(state):
    return _RUN[state['op']](state)


def exact(case, seed):
    return _EXACT[case['op']](case, prepare(case, seed))

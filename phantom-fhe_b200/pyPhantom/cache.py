"""A cache of ciphertexts in pages, and the attention products that read it (no counterpart in the reference, whose K/V
ciphertexts are lists kept by its application, and whose attention products, src/attention.cu:10-98, take such lists).

A page is one two-polynomial ciphertext whose slots hold `positions` token positions (slots // d_total, the layout of
`compute_qkt`); a sequence is a list of page numbers, its table. One cache holds the pages of one level in `planes` planes (K and V
of every layer, say): a page number names the same page of every plane, and whatever is done to pages is done to all planes at once:
in one launch up to 480 steps (one a page, one more a cycle), in several, one after another, beyond that. The memory is one tensor data[planes][pages][2][limbs][N].

Forked sequences share their full pages, which are counted; a page held more than once is not written to. A cache serves one
stream at a time; calls work on torch's current stream of the context's device. Page numbers are read at the call: a captured graph
replays the moves of the numbers it was captured with.
"""
import heapq
import math
from array import array
from operator import index

import numpy as np
import torch

from . import _check_plain, _galois_index, _key_table, _multiply_sum, _operands, _rescale_rounded, add, ciphertext, get_elt_from_step, relinearize, rotate
from ._native import LIB, check, current_stream as _stream, on_device


class ciphertext_cache:
    def __init__(self, context, chain_index, pages, planes=1, scale=2.0 ** 40):
        pages, planes = int(pages), int(planes)
        if pages < 1 or planes < 1:
            raise ValueError("ciphertext_cache: at least one page and one plane are wanted")
        if not 1 <= chain_index <= context.size_Q:
            raise ValueError("chain index out of range")
        if not 0 < float(scale) < math.inf:
            raise ValueError("scale out of bounds")
        self.ctx, self._chain_index, self._limbs, self._scale = context, int(chain_index), context.limbs_at(chain_index), float(scale)
        self._planes, self._page_bytes = planes, 16 * self._limbs * context.N
        self.data = context.empty(planes, pages, 2, self._limbs)
        self._held = [0] * pages       # how many tables hold a page
        self._free = list(range(pages))  # a heap: the lowest number goes out first

    # ---- what it is -------------------------------------------------------------------------------------------------
    def chain_index(self):
        return self._chain_index

    def scale(self):
        return self._scale

    def planes(self):
        return self._planes

    def pages(self):
        return len(self._held)

    def free_pages(self):
        return len(self._free)

    def held(self, page):
        """how many tables hold the page"""
        return self._held[self._number(page)]

    def _number(self, page):
        page = index(page)
        if not 0 <= page < len(self._held):
            raise ValueError("ciphertext_cache: page out of range")
        return page

    def _live(self, pages):
        """the page numbers as a list of integers, each of an allocated page"""
        pages = list(map(index, pages))
        held = self._held
        try:
            ok = not pages or (min(pages) >= 0 and all(map(held.__getitem__, pages)))
        except IndexError:
            ok = False
        if not ok:
            for p in pages:
                self._number(p)
            raise ValueError("ciphertext_cache: page is not allocated")
        return pages

    def _plane(self, plane):
        if not 0 <= int(plane) < self._planes:
            raise ValueError("ciphertext_cache: plane out of range")
        return int(plane)

    def page(self, page, plane=0):
        """the page as a ciphertext: a view, not a copy"""
        (page,) = self._live([page])
        return self._view(self.data[self._plane(plane), page])

    def ciphertexts(self, pages, plane=0):
        """the pages as a list of ciphertexts (views), as compute_qkt and score_times_v take them"""
        rows = self.data[self._plane(plane)]
        return [self._view(rows[p]) for p in self._live(pages)]

    def _view(self, data):
        ct = ciphertext()
        ct._chain_index, ct._size, ct._N, ct._limbs, ct._scale, ct.data = self._chain_index, 2, self.ctx.N, self._limbs, self._scale, data
        return ct

    # ---- pages ------------------------------------------------------------------------------------------------------
    def _move(self, dst, src, source=None):
        n = len(dst)
        if not n:
            return
        d, s = array("q", dst), array("q", src)  # half the host time of numpy arrays
        x = self if source is None else source
        with on_device(self.ctx):
            check(LIB.b2_pages_move(self.ctx._h, self._limbs, self._planes, self.data.data_ptr(), len(self._held), x.data.data_ptr(), x._limbs,
                                    len(x._held), n, d.buffer_info()[0], s.buffer_info()[0], _stream()))

    def allocate(self, n=1):
        """n pages that nobody holds, as a table; zeros in every plane"""
        n = int(n)
        if n < 0:
            raise ValueError("ciphertext_cache: a negative number of pages")
        pages = self._take(n)
        try:
            self._move(pages, [-1] * n)
        except Exception:
            self.free(pages)
            raise
        return pages

    def _take(self, n):
        if n > len(self._free):
            raise RuntimeError("ciphertext_cache: out of pages")
        pages = [heapq.heappop(self._free) for _ in range(n)]
        for p in pages:
            self._held[p] = 1
        return pages

    def free(self, table):
        """gives a table back; a page goes when no other table holds it"""
        counts = {}
        for p in self._live(table):
            counts[p] = counts.get(p, 0) + 1
        if any(self._held[p] < k for p, k in counts.items()):
            raise ValueError("ciphertext_cache: a page is given back more often than it is held")
        for p, k in counts.items():
            self._held[p] -= k
            if not self._held[p]:
                heapq.heappush(self._free, p)

    def fork(self, table, copies=1, tail=1):
        """`copies` new tables with the contents of `table`: all pages but the last `tail` are shared, those are copied (the last
        page still takes positions), every plane and every copy at once"""
        table, copies, tail = self._live(table), int(copies), int(tail)
        if copies < 1 or tail < 0:
            raise ValueError("ciphertext_cache: at least one copy and no negative tail are wanted")
        keep = max(0, len(table) - tail)
        new = self._take(copies * (len(table) - keep))
        try:
            self._move(new, table[keep:] * copies)
        except Exception:
            self.free(new)
            raise
        for p in table[:keep]:
            self._held[p] += copies
        n = len(table) - keep
        return [table[:keep] + new[k * n:(k + 1) * n] for k in range(copies)]

    def copy(self, dst, src, source=None):
        """page dst[i] becomes what page src[i] was before the call, for all i at once, in every plane; dst distinct, both
        allocated. `source`: another cache with as many planes, at this level or a higher one (the limbs beyond are dropped, as
        mod_switch_to does)"""
        if len(dst) != len(src):
            raise ValueError("ciphertext_cache: as many sources as destinations are wanted")
        other = self if source is None else source
        if other.ctx is not self.ctx or other._planes != self._planes or other._limbs < self._limbs:
            raise ValueError("ciphertext_cache: the source has another context, other planes or a lower level")
        if not abs(other._scale - self._scale) <= 1e-9 * self._scale:
            raise ValueError("scale mismatch")
        dst = self._live(dst)
        if any(self._held[p] > 1 for p in dst):
            raise ValueError("ciphertext_cache: the page is shared (fork the table first)")
        self._move(dst, other._live(src), source)

    def compact(self, tables):
        """Moves all allocated pages to the front of the pool, those of `tables` first and in their order (a table's pages then
        lie one after another), in place and at once. Returns the tables with their new numbers; every other table that is
        still held is out of date unless it is given too: pages outside `tables` keep their order behind them."""
        tables = [self._live(t) for t in tables]
        order = list(dict.fromkeys(p for t in tables for p in t))
        seen = set(order)
        order += [p for p, k in enumerate(self._held) if k and p not in seen]
        self._move(range(len(order)), order)
        new = {p: i for i, p in enumerate(order)}
        self._held = [self._held[p] for p in order] + [0] * (len(self._held) - len(order))
        self._free = list(range(len(order), len(self._held)))
        return [[new[p] for p in t] for t in tables]

    def resize(self, pages):
        """another number of pages; those allocated have to lie in front of it (`compact`). The pool moves: a graph captured before
        works on memory that was given back, and has to be captured anew; while one is captured this call is refused."""
        pages = int(pages)
        if pages < 1 or any(self._held[pages:]):
            raise ValueError("ciphertext_cache: allocated pages lie behind the new end (compact first)")
        with on_device(self.ctx):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("ciphertext_cache: resize cannot be captured (every replay would read the memory that it gives back)")
        n = min(pages, len(self._held))
        data = self.ctx.empty(self._planes, pages, 2, self._limbs)
        live = array("q", [p for p in range(n) if self._held[p]])
        if live:
            at = live.buffer_info()[0]
            with on_device(self.ctx):
                check(LIB.b2_pages_move(self.ctx._h, self._limbs, self._planes, data.data_ptr(), pages, self.data.data_ptr(), self._limbs, len(self._held),
                                        len(live), at, at, _stream()))
        # the pool may have been made on another stream: its memory goes back only after what this one still does with it
        self.data.record_stream(torch.cuda.current_stream(self.ctx.device))
        self.data = data
        self._held = self._held[:n] + [0] * (pages - n)
        self._free = [p for p, k in enumerate(self._held) if not k]

    # ---- contents -----------------------------------------------------------------------------------------------------
    def _writable(self, page, ct):
        (page,) = self._live([page])
        if self._held[page] > 1:
            raise ValueError("ciphertext_cache: the page is shared (fork the table first)")
        data = ct.data
        if (ct._size != 2 or not ct._is_ntt_form or data.shape != (2, ct._limbs, self.ctx.N) or data.dtype != torch.int64
                or data.get_device() != self.ctx.device):
            raise ValueError("ciphertext_cache: a two-polynomial ciphertext in NTT form on the context's device is wanted")
        if ct._chain_index > self._chain_index or ct._limbs < self._limbs:
            raise ValueError("cannot switch to higher level modulus")
        if not abs(ct._scale - self._scale) <= 1e-9 * self._scale:
            raise ValueError("scale mismatch")
        return page

    def store(self, page, ct, plane=0):
        """page := ct (dropped to the cache's level)"""
        self.data[self._plane(plane), self._writable(page, ct)].copy_(ct.data[:, :self._limbs])

    def append(self, page, ct, plane=0):
        """page += ct (dropped to the cache's level): puts positions into a page where it still holds zeros. The ciphertext is zero
        in every other position, as rotary factors of a masked block or a product with a mask leave it"""
        row = self.data[self._plane(plane), self._writable(page, ct)]
        x = ct.data if ct._limbs == self._limbs and ct.data.is_contiguous() else ct.data[:, :self._limbs].contiguous()
        with on_device(self.ctx):
            check(LIB.b2_ct_op(self.ctx._h, 0, self._limbs, 2, row.data_ptr(), x.data_ptr(), row.data_ptr(), _stream()))

    def multiply_sum(self, scores, pages, plane=0):
        """multiply_sum of `scores` with the pages, read where they lie: sum_t scores[t] x page[pages[t]] as one three-polynomial
        ciphertext at the lower of the two levels. A list of such lists (queries that read the same pages) gives a list."""
        pages = self._live(pages)
        step = self._page_bytes
        base = self.data.data_ptr() + self._plane(plane) * len(self._held) * step
        return _multiply_sum(self.ctx, scores, array("Q", [base + p * step for p in pages]), self._limbs, self._chain_index, self._scale)


# ---- attention products ---------------------------------------------------------------------------------------------------
BATCH = 16  # ciphertexts that go through each kernel together (the products of one call of b2_multiply_relin_rescale_many)


def _nominal(scale, prime):
    """A product keeps its first factor's (nominal) scale, as the lists' forms label it, which is right where the other factor's
    scale is about the prime that the rescale removes. The primes of a size lie within a few per cent of the power of two that such
    a scale is (24 primes of 30 bits for N = 2^17: 6); an eighth away is another size."""
    if not 0.875 < scale / float(prime) < 1.125:
        raise ValueError("scale mismatch")


def _rotate_add_batch(ctx, x, step, galois_key):
    """x[n][2][l][N] += x rotated by `step`, every kernel one launch over the n ciphertexts"""
    n, l = x.shape[0], x.shape[2]
    elt = get_elt_from_step(step, ctx.N)
    key = galois_key.resolve(_galois_index(ctx, elt))
    if key is None:
        raise ValueError("Galois key not present (no owned key, no fallback)")
    tab = _key_table(ctx, key, l)
    nbytes = int(LIB.b2_keyswitch_batch_workspace_bytes(ctx._h, l, n))
    ws, out = torch.empty(max(nbytes // 8, 1), dtype=torch.int64, device=ctx.device), torch.empty_like(x)
    check(LIB.b2_apply_galois_batch(ctx._h, l, elt, n, x.data_ptr(), 2 * l, tab.ctypes.data, len(tab), out.data_ptr(), 2 * l, ws.data_ptr(), nbytes,
                                    _stream()))
    check(LIB.b2_ct_op(ctx._h, 0, l, 2 * n, x.data_ptr(), out.data_ptr(), x.data_ptr(), _stream()))


def cached_qkt(context, relin_key, galois_key, q, cache, pages, d_head, plane=0):
    """compute_qkt (src/attention.cu:10-28) over cached pages: per page q * k, one rescale, the sum over each d_head block; slot
    t * d_total + h * d_head of result j holds Q[h] . K of position t of page pages[j]. The pages are read where they lie, at q's
    level or above it, and every kernel runs over 16 of them at a time; the rescale rounds to nearest, so that the results agree
    with compute_qkt's to rounding, not limb for limb. They keep q's scale: the pages' has to be about the prime that it removes."""
    ctx, pages = context, cache._live(pages)
    plane = cache._plane(plane)
    if d_head == 0 or d_head & (d_head - 1):
        raise ValueError("inner_sum: block_size must be a power of 2")
    if cache.ctx is not ctx:
        raise ValueError("ciphertext_cache: the cache belongs to another context")
    if q._chain_index < cache._chain_index:
        raise ValueError("encrypted1 and encrypted2 parameter mismatch")
    _, table, held = _operands(ctx, [[q]])
    if q._chain_index == ctx.size_Q:
        raise ValueError("end of modulus switching chain reached")
    l, nominal, results = q._limbs, q._scale, []
    _nominal(cache._scale, ctx.primes[l - 1])
    tab = _key_table(ctx, relin_key, l)
    step = cache._page_bytes
    base = cache.data.data_ptr() + plane * cache.pages() * step
    with on_device(ctx):
        for p0 in range(0, len(pages), BATCH):
            part = pages[p0:p0 + BATCH]
            n = len(part)
            a, b = np.full(n, table[0], dtype=np.uint64), np.array([base + p * step for p in part], dtype=np.uint64)
            la, lb = np.full(n, l, dtype=np.uint32), np.full(n, cache._limbs, dtype=np.uint32)
            nbytes = int(LIB.b2_multiply_relin_batch_workspace_bytes(ctx._h, l, n))
            ws, out = torch.empty(nbytes // 8, dtype=torch.int64, device=ctx.device), ctx.empty(n, 2, l - 1)
            check(LIB.b2_multiply_relin_rescale_many(ctx._h, l, n, 1, a.ctypes.data, la.ctypes.data, b.ctypes.data, lb.ctypes.data, 0, tab.ctypes.data,
                                                     len(tab), out.data_ptr(), ws.data_ptr(), nbytes, _stream()))
            del ws
            stride = 1
            while stride < d_head:
                _rotate_add_batch(ctx, out, stride, galois_key)
                stride <<= 1
            results += [q._like(out[i], chain_index=q._chain_index + 1, scale=nominal) for i in range(n)]
    return results


def cached_score_times_v(context, relin_key, galois_key, scores, cache, pages, mask_pt, d_head, d_total, positions_per_ct, plane=0):
    """score_times_v (src/attention.cu:30-98) over cached pages: sum_t score[t] V[t]. The masked scores are spread over their heads
    16 at a time; the products with all pages are summed before they are relinearised, so that one relinearisation, one rescale
    and one fold over the positions serve the whole context (score_times_v makes each of them per chunk). Same levels; the
    rescales round to nearest. The result keeps the scores' scale: the mask's and the pages' have to be about the primes that are
    removed."""
    ctx = context
    if len(scores) == 0:
        raise ValueError("score_times_v: score_cts is empty")
    if len(scores) != len(pages):
        raise ValueError("score_times_v: score_cts and v_cts size mismatch")
    if d_head == 0 or d_head & (d_head - 1):
        raise ValueError("score_times_v: d_head must be a power of 2")
    if positions_per_ct == 0 or positions_per_ct & (positions_per_ct - 1):
        raise ValueError("score_times_v: positions_per_ct must be a power of 2")
    if cache.ctx is not ctx:
        raise ValueError("ciphertext_cache: the cache belongs to another context")
    first, _, _ = _operands(ctx, [scores])
    _check_plain(first, mask_pt)
    if mask_pt.data.shape != (first._limbs, ctx.N) or mask_pt.data.dtype != torch.int64 or mask_pt.data.get_device() != ctx.device:
        raise ValueError("encrypted and plain parameter mismatch")
    mask = mask_pt.data.contiguous()
    l, nominal, spread = first._limbs, first._scale, []
    deep = min(l - 1, cache._limbs)  # of the products
    if l < 3 or deep < 2:
        raise ValueError("end of modulus switching chain reached")
    _nominal(mask_pt._scale, ctx.primes[l - 1])
    _nominal(cache._scale, ctx.primes[deep - 1])
    with on_device(ctx):
        for p0 in range(0, len(scores), BATCH):
            x = torch.stack([s.data for s in scores[p0:p0 + BATCH]])
            n = x.shape[0]
            check(LIB.b2_ct_op(ctx._h, 2, l, 2 * n, x.data_ptr(), mask.data_ptr(), x.data_ptr(), _stream()))
            m, ws = ctx.empty(n, 2, l - 1), ctx.empty(2 * n)
            check(LIB.b2_rescale_rounded_batch(ctx._h, l, n, x.data_ptr(), m.data_ptr(), ws.data_ptr(), ws.numel() * 8, _stream()))
            b = d_head // 2
            while b >= 1:
                _rotate_add_batch(ctx, m, -b, galois_key)
                b >>= 1
            spread += [first._like(m[i], chain_index=first._chain_index + 1, scale=nominal) for i in range(n)]
        total = _rescale_rounded(ctx, relinearize(ctx, cache.multiply_sum(spread, pages, plane), relin_key))
        total.set_scale(nominal)
        stride = d_total
        while stride < positions_per_ct * d_total:
            total = add(ctx, total, rotate(ctx, total, stride, galois_key))
            stride <<= 1
    return total

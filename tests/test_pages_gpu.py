"""The paged cache's operations against a plain model of it, byte for byte."""
import pytest
import torch

import servref as R
from kvc_b200 import attn, pages

pytestmark = pytest.mark.gpu


class Model:
    """What the operations say, on host copies."""

    def __init__(self, c):
        self.page, self.L = c.page, c.layers
        self.K, self.V = c.K.cpu().clone(), c.V.cpu().clone()
        self.beta = None if c.beta is None else c.beta.cpu().clone()
        self.table, self.ref, self.len = c.table.cpu().tolist(), c.ref.cpu().tolist(), c.seq_len.cpu().tolist()
        self.status = 0

    def at(self, slot, r):
        return self.table[slot][r // self.page] * self.page + r % self.page

    def put(self, layer, dst, src, V=None, beta=None):
        p = self.page
        self.K[layer, dst] = self.old[0][layer, src]
        self.V[layer, dst] = self.old[1][layer, src] if V is None else V
        if self.beta is not None:
            self.beta[layer, dst // p, :, dst % p] = self.old[2][layer, src // p, :, src % p] if beta is None else beta

    def plan(self, items):
        """items: (src, dst, whole, length); the table rows they get, or None."""
        free = [i for i, r in enumerate(self.ref) if r == 0]
        rows = []
        for src, dst, whole, length in items:
            need = max(0, -(-length // self.page) - whole)
            if whole + need > len(self.table[0]):
                self.status = -13
                return None
            if need > len(free):
                self.status = -11
                return None
            rows.append(self.table[src][:whole] + free[:need])
            free = free[need:]
        self.old = (self.K.clone(), self.V.clone(), None if self.beta is None else self.beta.clone())
        return rows

    def commit(self, items, rows):
        width = len(self.table[0])
        new = [r + [-1] * (width - len(r)) for r in rows]
        for (src, dst, _, length), row in zip(items, new):
            for p in self.table[dst]:
                if p >= 0:
                    self.ref[p] -= 1
            for p in row:
                if p >= 0:
                    self.ref[p] += 1
        for (src, dst, _, length), row in zip(items, new):
            self.table[dst], self.len[dst] = row, length

    def reserve(self, seqs, add):
        items = [(s, s, -(-self.len[s] // self.page), self.len[s] + n) for s, n in zip(seqs, add)]
        rows = self.plan(items)
        if rows is not None:
            self.commit(items, rows)

    def fork(self, src, dst):
        items = [(s, d, self.len[s] // self.page, self.len[s]) for s, d in zip(src, dst)]
        rows = self.plan(items)
        if rows is None:
            return
        for (s, d, whole, n), row in zip(items, rows):
            for r in range(whole * self.page, n):
                for l in range(self.L):
                    self.put(l, row[whole] * self.page + r % self.page, self.at(s, r))
        self.commit(items, rows)

    def compact(self, src, dst, keep, keep_n, base, v_rows=None, beta_rows=None):
        items = []
        for i, (s, d) in enumerate(zip(src, dst)):
            b, k = min(max(base[i], 0), self.len[s]), min(max(keep_n[i], 0), keep.shape[2])
            items.append((s, d, b // self.page, b + k))
        rows = self.plan(items)
        if rows is None:
            return
        for i, (s, d, whole, n) in enumerate(items):
            b = min(max(base[i], 0), self.len[s])
            for r in range(whole * self.page, n):
                dst_row = rows[i][r // self.page] * self.page + r % self.page
                for l in range(self.L):
                    if r < b:
                        self.put(l, dst_row, self.at(s, r))
                        continue
                    j = r - b
                    want = int(keep[l % keep.shape[0], i, j])
                    if 0 <= want < self.len[s]:
                        self.put(l, dst_row, self.at(s, want), None if v_rows is None else v_rows[l, i, j],
                                 None if beta_rows is None else beta_rows[l, i, :, j])
        self.commit(items, rows)

    def free(self, seqs):
        self.commit([(s, s, 0, 0) for s in seqs], [[] for _ in seqs])

    def same(self, c):
        torch.cuda.synchronize()
        assert c.table.cpu().tolist() == self.table
        assert c.ref.cpu().tolist() == self.ref
        assert c.seq_len.cpu().tolist() == self.len
        assert int(c.status) == self.status
        assert torch.equal(c.K.cpu(), self.K) and torch.equal(c.V.cpu(), self.V)
        if c.beta is not None:
            assert torch.equal(c.beta.cpu(), self.beta)


def cache(lens, page=8, hkv=2, d=64, kt=R.Q8_0, vt=R.F16, layers=2, beta=True, spare=40, slots=8, **kw):
    return R.Cache(lens, hkv, d, d, kt, vt, page, layers=layers, beta=beta, spare=spare, slots=slots, max_pages=48, **kw)


dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731


@pytest.mark.parametrize("kt,vt", [(R.F32, R.Q4_1), (R.F16, R.F16), (R.Q8_0, R.Q4_0)])
@pytest.mark.parametrize("page", [1, 7, 8, 16])
@pytest.mark.parametrize("hkv,d", [(1, 32), (2, 64), (3, 32)])
def test_fork(kvc, page, kt, vt, hkv, d):
    c = cache([21, 16, 0, 5], page=page, kt=kt, vt=vt, hkv=hkv, d=d)
    m, h = Model(c), c.handle(kvc)
    for src, dst in (([0, 0, 1, 2], [4, 5, 6, 7]), ([3], [4]), ([4, 5], [0, 1]), ([2], [5])):
        h.fork(src, dst)
        m.fork(src, dst)
        m.same(c)


@pytest.mark.parametrize("refit", [False, True])
@pytest.mark.parametrize("lists", [1, 2])
@pytest.mark.parametrize("page", [1, 7, 8, 16])
@pytest.mark.parametrize("kt,vt,beta", [(R.Q8_0, R.Q8_0, True), (R.F32, R.F16, False), (R.Q4_0, R.Q4_1, True)])
def test_compact(kvc, refit, lists, page, kt, vt, beta):
    c = cache([40, 17, 9], page=page, kt=kt, vt=vt, beta=beta, hkv=3, d=32, spare=120)
    m, h = Model(c), c.handle(kvc)
    g = torch.Generator().manual_seed(page)
    for src, dst in (([0, 1, 2], [4, 5, 6]), ([0, 1, 2], [0, 1, 2]), ([4], [0]), ([5, 0], [5, 7])):
        n, ld = len(src), 12
        length = [m.len[s] for s in src]
        base = [int(torch.randint(0, x + 1, (1,), generator=g)) for x in length]
        keep = torch.zeros(lists, n, ld, dtype=torch.int32)
        count = [min(ld, x - b) for x, b in zip(length, base)]
        for l in range(lists):
            for i in range(n):
                keep[l, i, :count[i]] = torch.randperm(length[i] - base[i], generator=g)[:count[i]].sort()[0].int() + base[i]
        v = torch.randint(0, 256, (2, n, ld, c.V.shape[2]), generator=g).to(torch.uint8) if refit else None
        b = torch.randn(2, n, 3, ld, generator=g) if refit and beta else None
        h.compact(src, dst, keep.cuda(), dev(count), dev(base), v_rows=None if v is None else v.cuda(),
                  beta_rows=None if b is None else b.cuda())
        m.compact(src, dst, keep, count, base, v, b)
        m.same(c)


def test_compact_odd_lists(kvc):
    """Lists that name a row twice, rows outside the sequence, counts and bases outside their ranges; nothing kept."""
    c = cache([20, 20], page=8)
    m, h = Model(c), c.handle(kvc)
    keep = torch.tensor([[[3, 3, 19, 20, -1, 500, 0, 7]] * 2], dtype=torch.int32)
    for count, base in (([8, 99], [0, 2]), ([3, -4], [-5, 40]), ([0, 0], [0, 13])):
        h.compact([0, 1], [2, 3], keep.cuda(), dev(count), dev(base))
        m.compact([0, 1], [2, 3], keep, count, base)
        m.same(c)
    h.compact([0], [0], torch.zeros(1, 1, 0, dtype=torch.int32, device="cuda"), dev([0]), dev([9]))
    m.compact([0], [0], torch.zeros(1, 1, 0, dtype=torch.int32), [0], [9])
    m.same(c)


@pytest.mark.parametrize("page", [1, 7, 16])
def test_reserve_free_and_reuse(kvc, page):
    c = cache([5, 0, 16], page=page, spare=60)
    m, h = Model(c), c.handle(kvc)
    for seqs, add in (([0, 1], [3, 16]), ([4], [0]), ([2, 0], [1, 1])):
        h.reserve(seqs, add)
        m.reserve(seqs, add)
        m.same(c)
    h.fork([2], [5])
    m.fork([2], [5])
    for seqs in ([2, 7], [5], [0, 1, 2]):
        h.free(seqs)
        m.free(seqs)
        m.same(c)
    h.reserve([3], [page * 3])
    m.reserve([3], [page * 3])
    m.same(c)


def test_a_call_that_cannot_be_done_changes_nothing(kvc):
    c = cache([20, 30], page=8, spare=2)
    m, h = Model(c), c.handle(kvc)
    h.reserve([0, 1], [100, 1])                        # pages
    m.reserve([0, 1], [100, 1])
    assert m.status == -11
    m.same(c)
    with pytest.raises(RuntimeError, match="-11"):
        h.check()
    h.check()
    m.status = 0
    h.reserve([0], [48 * 8])                           # table entries
    m.reserve([0], [48 * 8])
    assert m.status == -13
    m.same(c)
    h.status.zero_()
    h.reserve([0], [2 ** 31 - 1])
    torch.cuda.synchronize()
    assert int(c.status) == -13
    h.status.zero_()
    m.status = 0
    h.fork([0, 0, 0], [2, 3, 4])
    m.fork([0, 0, 0], [2, 3, 4])
    assert m.status == -11
    m.same(c)
    h.status.zero_()
    m.status = 0
    h.fork([0, 0], [2, 3])
    m.fork([0, 0], [2, 3])
    m.same(c)


@pytest.mark.parametrize("add", [[2 ** 30, 2 ** 30], [2 ** 30, 1], [5, 0]])
def test_more_pages_asked_for_than_32_bits_count(kvc, add):
    """Table rows so long that the entries of a call together ask for 2^31 pages (the table is not written)."""
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = torch.zeros(1, 4, 4, dtype=torch.uint8, device="cuda")
    table = torch.empty(2, 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, :8] = -1
    c = pages.PageCache(kvc, rows, rows.clone(), table, z(2), z(4), z(1), 1, 1, 1, 1, 0, 0)
    c.reserve([0, 1], add)
    torch.cuda.synchronize()
    assert int(c.status) == -11 and c.seq_len.tolist() == [0, 0] and int(c.ref_count.abs().sum()) == 0
    assert bool((table[:, :8] == -1).all())


@pytest.mark.parametrize("at", [0, 31, 32, 100, 255])
def test_one_entry_of_many_that_does_not_fit(kvc, at):
    """A table row that is too short in any of 256 entries, or too few pages for all: nothing changes."""
    c = cache([5] * 256, page=4, slots=256, spare=300, hkv=1, d=32)
    m, h = Model(c), c.handle(kvc)
    add = [4] * 256
    add[at] = 48 * 4
    for _ in range(20):
        h.reserve(list(range(256)), add)
        torch.cuda.synchronize()
        assert int(c.status) == -13
        c.status.zero_()
    m.same(c)
    h.reserve(list(range(256)), [9] * 256)             # 512 pages of 300
    m.reserve(list(range(256)), [9] * 256)
    assert m.status == -11
    m.same(c)


@pytest.mark.parametrize("n_pages", [1, 15, 16, 17, 5000, 40001])
def test_lowest_free_pages(kvc, n_pages):
    """Pools around and beyond one step of the scan, with few free pages and far ones."""
    g = torch.Generator().manual_seed(n_pages)
    ref = (torch.rand(n_pages, generator=g) < 0.97).int()
    ref[-1] = 0
    free = (ref == 0).nonzero()[:, 0].tolist()
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    for off in (0, 1):                                 # counts at another alignment
        buf = torch.zeros(n_pages + 1, dtype=torch.int32, device="cuda")
        buf[off:off + n_pages] = ref.cuda()
        rows = torch.zeros(1, n_pages, 4, dtype=torch.uint8, device="cuda")
        c = pages.PageCache(kvc, rows, rows.clone(), z(3, n_pages) - 1, z(3), buf[off:off + n_pages], z(1), 1, 1, 1, 1, 0, 0)
        take = [len(free) // 2, len(free) - len(free) // 2]
        c.reserve([2, 0], take)
        torch.cuda.synchronize()
        assert c.page_table[2, :take[0]].tolist() == free[:take[0]]
        assert c.page_table[0, :take[1]].tolist() == free[take[0]:]
        assert int((c.ref_count == 0).sum()) == 0 and int(c.status) == 0
        c.reserve([1], [1])
        torch.cuda.synchronize()
        assert int(c.status) == -11


@pytest.mark.parametrize("page", [1, 5, 16])
def test_write_and_read(kvc, page):
    c = cache([30, 18, 4], page=page, hkv=3, d=32, kt=R.Q8_0, vt=R.F32)
    m, h = Model(c), c.handle(kvc)
    g = torch.Generator().manual_seed(1)
    seqs, first, count = [1, 0, 1, 2], [0, 7, 15, 3], [5, 23, 10, 0]      # rows 18 and on of sequence 1 do not exist
    n = sum(count)
    k = torch.randint(0, 256, (2, n, c.K.shape[2]), generator=g).to(torch.uint8)
    v = torch.randint(0, 256, (2, n, c.V.shape[2]), generator=g).to(torch.uint8)
    b = torch.randn(2, 3, n, generator=g)
    h.write(seqs, first, count, k.cuda(), v.cuda(), b.cuda())
    want = [torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(b)]
    at = 0
    for s, f, cnt in zip(seqs, first, count):
        for i in range(cnt):
            if f + i < m.len[s]:
                r = m.at(s, f + i)
                m.K[:, r], m.V[:, r], m.beta[:, r // page, :, r % page] = k[:, at], v[:, at], b[:, :, at]
                for w, x, ix in ((want[0], k, (slice(None), at)), (want[1], v, (slice(None), at)),
                                 (want[2], b, (slice(None), slice(None), at))):
                    w[ix] = x[ix]
            at += 1
    m.same(c)
    got = h.read(seqs, first, count)
    torch.cuda.synchronize()
    for a, w in zip(got, want):
        assert torch.equal(a.cpu(), w)
    h.write([0], [0], [3], None, v[:, :3].contiguous().cuda())            # V alone
    for i in range(3):
        m.V[:, m.at(0, i)] = v[:, i]
    m.same(c)
    h.read([0, 0], [2, 2], [3, 3])                                         # a sequence twice
    torch.cuda.synchronize()


def test_write_leaves_shared_pages(kvc):
    c = cache([20], page=8)
    h = c.handle(kvc)
    h.fork([0], [1])
    m = Model(c)
    k = torch.full((2, 20, c.K.shape[2]), 9, dtype=torch.uint8, device="cuda")
    h.write([1], [0], [20], k)
    for r in range(16, 20):                            # the last, partial page is sequence 1's own
        m.K[:, m.at(1, r)] = 9
    m.status = -2
    m.same(c)
    with pytest.raises(RuntimeError, match="-2"):
        h.check()


def test_copy_pages(kvc):
    c = cache([40], page=7, hkv=3, d=32, kt=R.Q4_0, vt=R.Q8_0)
    m, h = Model(c), c.handle(kvc)
    src, dst = [c.table[0, 2].item(), c.table[0, 0].item(), -1, c.n_pages, 3], None
    free = (c.ref == 0).nonzero()[:, 0].tolist()
    dst = [free[1], free[0], free[2], free[3], -5]
    h.copy(dev(src), dev(dst))
    for a, b in zip(src[:2], dst[:2]):
        m.K[:, b * 7:b * 7 + 7], m.V[:, b * 7:b * 7 + 7] = m.K[:, a * 7:a * 7 + 7], m.V[:, a * 7:a * 7 + 7]
        m.beta[:, b] = m.beta[:, a]
    m.same(c)


@pytest.mark.parametrize("page", [1, 3, 16, 70])
@pytest.mark.parametrize("kt,vt,hkv,d", [(R.F16, R.F16, 2, 64), (R.Q8_0, R.F32, 8, 64), (R.F32, R.Q4_0, 32, 256)])
def test_copy_pages_of_16_byte_pieces(kvc, page, kt, vt, hkv, d):
    """Rows that go by bulk copies (the last ones one per CTA): pairs outside the pool and onto themselves among them."""
    c = cache([40], page=page, hkv=hkv, d=d, kt=kt, vt=vt)
    assert c.K.shape[2] % 16 == 0 and c.V.shape[2] % 16 == 0
    m, h = Model(c), c.handle(kvc)
    free = (c.ref == 0).nonzero()[:, 0].tolist()
    used = [p for p in c.table[0].tolist() if p >= 0]
    pairs = list(zip(used, free[:-3])) + [(-1, free[-1]), (c.n_pages, free[-2]), (used[0], -5), (used[0], c.n_pages), (free[-3],) * 2]
    h.copy(dev([a for a, _ in pairs]), dev([b for _, b in pairs]))
    for a, b in zip(used, free[:-3]):
        for store in (m.K, m.V):
            store[:, b * page:(b + 1) * page] = store[:, a * page:(a + 1) * page]
        m.beta[:, b] = m.beta[:, a]
    m.same(c)


@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("parts", [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_write_and_read_of_16_byte_pieces(kvc, page, parts):
    """Some of the arrays alone, of all layers and of one, by bulk copies: what is left out stays as it was."""
    c = R.Cache([90, 18, 4], 8, 64, 64, R.Q8_0, R.F32, page, layers=2, beta=True, spare=20)
    m, h = Model(c), c.handle(kvc)
    g = torch.Generator().manual_seed(2)
    seqs, first, count = [1, 0, 1, 2], [0, 7, 15, 3], [5, 70, 10, 0]
    n, at = sum(count), 0
    rows = [torch.randint(0, 256, (2, n, c.K.shape[2]), generator=g).to(torch.uint8),
            torch.randint(0, 256, (2, n, c.V.shape[2]), generator=g).to(torch.uint8), torch.randn(2, 8, n, generator=g)]
    assert all(r.shape[2] % 16 == 0 for r in rows[:2])
    for layer in (None, 1, 0):
        part = slice(None) if layer is None else slice(layer, layer + 1)
        given = [r[part].contiguous().cuda() if p else None for r, p in zip(rows, parts)]
        h.write(seqs, first, count, *given, layer=layer)
        at = 0
        for s, f, cnt in zip(seqs, first, count):
            for i in range(cnt):
                if f + i < m.len[s]:
                    r = m.at(s, f + i)
                    if parts[0]:
                        m.K[part, r] = rows[0][part, at]
                    if parts[1]:
                        m.V[part, r] = rows[1][part, at]
                    if parts[2]:
                        m.beta[part, r // page, :, r % page] = rows[2][part][:, :, at]
                at += 1
        m.same(c)
        out = [torch.full_like(r[part], 7).cuda() if p else None for r, p in zip(rows, parts)]
        want = [None if o is None else o.cpu() for o in out]
        h._rows("kvc_pages_read", seqs, first, count, *out, layer)
        at = 0
        for s, f, cnt in zip(seqs, first, count):
            for i in range(cnt):
                if f + i < m.len[s]:
                    r = m.at(s, f + i)
                    for w, store in ((want[0], m.K), (want[1], m.V)):
                        if w is not None:
                            w[:, at] = store[part, r]
                    if want[2] is not None:
                        want[2][:, :, at] = m.beta[part, r // page, :, r % page]
                at += 1
        torch.cuda.synchronize()
        for o, w in zip(out, want):
            assert o is None or torch.equal(o.cpu(), w)
        rows = [r.flip(1) if i < 2 else r + 1 for i, r in enumerate(rows)]


@pytest.mark.parametrize("page", [1, 7, 64])
def test_compact_of_16_byte_pieces(kvc, page):
    """Refitted rows and beta with rows that go by bulk copies, more of them than a CTA takes at a time."""
    c = R.Cache([300, 90], 8, 32, 32, R.F16, R.Q8_0, page, layers=2, beta=True, spare=800, slots=8)
    m, h = Model(c), c.handle(kvc)
    g = torch.Generator().manual_seed(page)
    ld = 250
    keep = torch.stack([torch.stack([torch.randperm(n, generator=g)[:ld].sort()[0] if n >= ld else
                                     torch.arange(ld) % n for n in (300, 90)]) for _ in range(2)]).int()
    v = torch.randint(0, 256, (2, 2, ld, c.V.shape[2]), generator=g).to(torch.uint8)
    b = torch.randn(2, 2, 8, ld, generator=g)
    assert c.K.shape[2] % 16 == 0 and c.V.shape[2] % 16 == 0
    for src, dst, base, given in (([0, 1], [2, 3], [5, 0], (v, b)), ([2, 3], [2, 3], [0, 17], (None, None)), ([0, 1], [0, 1], [0, 3], (v, None))):
        h.compact(src, dst, keep.cuda(), dev([ld, 60]), dev(base), *(None if x is None else x.cuda() for x in given))
        m.compact(src, dst, keep, [ld, 60], base, *given)
        m.same(c)


def test_in_a_graph_and_on_a_stream(kvc):
    c = cache([21, 16], page=8)
    m, h = Model(c), c.handle(kvc)
    g = torch.cuda.CUDAGraph()
    src, dst = pages.ids([0, 1]), pages.ids([2, 3])
    with torch.cuda.graph(g):
        h.fork(src, dst)
        h.free([3])
    m.same(c)
    for _ in range(3):
        g.replay()
        m.fork([0, 1], [2, 3])
        m.free([3])
        m.same(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h.fork([0], [5])
    side.synchronize()
    m.fork([0], [5])
    m.same(c)


def test_far_rows(kvc):
    """Rows more than 2^31 bytes into a layer, and layers more than 2^32 bytes apart."""
    page, n_pages, rb = 64, 20000, 2048 * 2
    c = pages.PageCache.empty(kvc, 1, n_pages, page, 3, 8, 8, 256, 256, R.F16, R.F16)
    c.ref_count.fill_(1)
    c.ref_count[-4:] = 0
    c.reserve([0, 1], [100, 60])
    q = torch.randn(1, 8, 256, device="cuda")
    k = torch.randn(1, 100, 8 * 256, device="cuda").half().view(torch.uint8)
    v = torch.randn(1, 100, 8 * 256, device="cuda").half().view(torch.uint8)
    assert c.K.shape[2] == rb and (n_pages - 4) * page * rb > 2 ** 32
    c.write([0], [0], [100], k.contiguous(), v.contiguous())
    got = c.read([0], [0], [100])
    torch.cuda.synchronize()
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    one = lambda *x: dev(list(x))  # noqa: E731
    t = attn.Tree(kvc, c, q, one(0, 1), one(0), max_nodes=1)
    t.run()
    K, V = R.decode(k[0], R.F16).view(100, 8, 256), R.decode(v[0], R.F16).view(100, 8, 256)
    for h in range(8):
        o, _ = R.attend(q[:, h], K[:, h], V[:, h], None, torch.ones(1, 100, dtype=torch.bool, device="cuda"), 256 ** -0.5)
        assert float((t.out[:, h].double() - o).abs().max()) < 1e-4
    c.fork([0], [2])
    c.check()
    got = c.read([2], [0], [100])
    torch.cuda.synchronize()
    assert torch.equal(got[0], k)

"""Attention over prompts and paged caches against the definition in 64 bits.

Tolerances: a score is the sum of products exact to 22 bits (fp16 pieces) added in fp32, so it is off by at most
A 2^-21 with A = max sum |q||k| scale, and x = score + beta and its scaling to base 2 add 2^-22 |x|; the exponential adds
2^-22. A probability's relative error is that sum e, the output's is 2 e max|V| (numerator and denominator). With F16
queries P times the row scale is rounded to fp16 once, 2^-11 (half an eps), the output once more; Q4_1 rounds two such
products and the sum of minimum and centre.
"""
import ctypes
import math
import threading

import pytest
import torch

import servref as R
from kvc_b200 import attn

pytestmark = pytest.mark.gpu


def bounds(q, K, V, x_max, kind_v, f16, scale):
    A = float((q.double().abs().flatten(0, 1) @ K.abs().flatten(0, -2).t()).max()) * scale if K.numel() else 0.0
    e = A * 2.0 ** -21 + (A + x_max) * 2.0 ** -22 + 2.0 ** -21
    v = float(V.abs().max()) if V.numel() else 0.0
    out = 2 * e * v + 2.0 ** -21 * v
    if f16:
        out += (4 if kind_v == R.Q4_1 else 2) * 2.0 ** -11 * v
    return out, 2 * e + 2.0 ** -21


def check(got, want, tol, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    d = (got - want)[~inf & ~torch.isnan(want)].abs()
    assert d.numel() == 0 or float(d.max()) <= tol, f"{what}: {float(d.max()):.3e} > {tol:.3e}"


def tree_case(kvc, lens, nodes, hkv=2, g=4, dk=64, dv=64, kt=R.Q8_0, vt=R.Q8_0, page=16, beta=False, qt=torch.float16, seed=0,
              mask="tree", edit=None, layers=1, layer=0, seqs=None):
    total = [n + m for n, m in zip(lens, nodes)]
    c = R.Cache(total, hkv, dk, dv, kt, vt, page, layers=layers, beta=beta, seed=seed)
    gen = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(sum(nodes), hkv * g, dk, generator=gen).to("cuda", qt)
    cu = [0]
    for m in nodes:
        cu.append(cu[-1] + m)
    words = max(1, -(-max(nodes + [1]) // 32))
    parents = [[int(torch.randint(-1, i, (1,), generator=gen)) if i else -1 for i in range(m)] for m in nodes]
    bits = attn.tree_mask(parents, words) if mask == "tree" else torch.zeros(sum(nodes), words, dtype=torch.int32)
    seqs = list(range(len(lens))) if seqs is None else seqs
    if edit:
        edit(c, q)
    h = c.handle(kvc)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    t = attn.Tree(kvc, h, q, dev(cu), dev(seqs), mask=None if mask is None else bits.cuda(), max_nodes=max(nodes + [1]),
                  scale=dk ** -0.5, layer=layer)

    def see(i, m, n):
        s = torch.ones(m, n, dtype=torch.bool)
        if mask is None:
            return s
        for a in range(m):
            for b in range(m):
                if n - m + b >= 0:
                    s[a, n - m + b] = bool((int(bits[cu[i] + a, b // 32]) >> (b % 32)) & 1)
        return s

    want = c.attend(q, cu, seqs, see, dk ** -0.5, layer)
    return c, q, t, want


def tree_check(kvc, **kw):
    c, q, t, (out, lse) = tree_case(kvc, **kw)
    layer = kw.get("layer", 0)
    K, V = R.decode(c.K[layer], c.kt), R.decode(c.V[layer], c.vt)
    used = torch.cat([c.rows(s) for s in range(len(kw["lens"]))] + [torch.zeros(0, dtype=torch.long, device="cuda")])
    K, V = K[used].view(-1, c.hkv, c.dk), V[used]
    fin = torch.isfinite(K).all() and torch.isfinite(V).all()
    xb = 0.0 if c.beta is None else float(torch.nan_to_num(c.beta, 0.0, 0.0, 0.0).abs().clamp(max=1e4).max())
    K = torch.nan_to_num(K, 0.0, 0.0, 0.0) if not fin else K
    V = torch.nan_to_num(V, 0.0, 0.0, 0.0) if not fin else V
    o_tol, l_tol = bounds(q, K, V, xb, c.vt, q.dtype == torch.float16, c.dk ** -0.5)
    t.out.fill_(7.0)
    t.lse.fill_(7.0)
    t.run()
    torch.cuda.synchronize()
    check(t.out, out, o_tol, "out")
    check(t.lse, lse, l_tol, "lse")
    first = t.out.clone(), t.lse.clone()
    t.run()
    torch.cuda.synchronize()
    assert torch.equal(first[0], t.out) and torch.equal(first[1], t.lse)       # the same bits every time
    assert int(c.status) == 0
    return t


KINDS = [R.F32, R.F16, R.Q8_0, R.Q4_0, R.Q4_1]


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("vt", KINDS)
@pytest.mark.parametrize("kt", KINDS)
def test_tree_types(kvc, kt, vt, qt):
    tree_check(kvc, lens=[130, 0, 7], nodes=[3, 1, 5], kt=kt, vt=vt, qt=qt, beta=kt != vt, seed=kt * 10 + vt)


@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 128), (128, 64), (96, 96), (128, 128), (256, 256), (192, 160), (256, 64)])
@pytest.mark.parametrize("kind", [R.F16, R.Q8_0, R.Q4_1])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
def test_tree_head_sizes(kvc, dk, dv, kind, qt):
    tree_check(kvc, lens=[77, 300], nodes=[1, 9], hkv=2, g=2, dk=dk, dv=dv, kt=kind, vt=kind, qt=qt, beta=True, seed=dk + dv)


@pytest.mark.parametrize("dk,dv", [(8, 8), (40, 24), (1, 3), (250, 33)])
@pytest.mark.parametrize("kind", [R.F16, R.F32])
def test_tree_odd_head_sizes(kvc, dk, dv, kind):
    tree_check(kvc, lens=[50, 3], nodes=[2, 1], hkv=3, g=1, dk=dk, dv=dv, kt=kind, vt=kind, qt=torch.float32, seed=dk)


@pytest.mark.parametrize("hkv", [1, 2, 3, 5, 8, 17])
@pytest.mark.parametrize("g", [1, 3, 8])
def test_tree_heads(kvc, hkv, g):
    tree_check(kvc, lens=[200, 31], nodes=[1, 1], hkv=hkv, g=g, dk=64, dv=64, kt=R.Q8_0, vt=R.Q4_0, beta=True, seed=hkv)
    tree_check(kvc, lens=[40], nodes=[6], hkv=hkv, g=g, dk=64, dv=64, kt=R.F16, vt=R.Q8_0, seed=g)


@pytest.mark.parametrize("page", [1, 3, 8, 12, 16, 24, 40, 64, 100, 256])
@pytest.mark.parametrize("kind", [R.F16, R.Q8_0])
def test_tree_pages(kvc, page, kind):
    for hkv in (4, 3):
        tree_check(kvc, lens=[333, 15, 64], nodes=[2, 1, 17], hkv=hkv, g=2, kt=kind, vt=kind, page=page, beta=True, seed=page)


@pytest.mark.parametrize("n", [0, 1, 15, 16, 17, 63, 64, 65, 1000, 5001])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
def test_tree_lengths(kvc, n, qt):
    tree_check(kvc, lens=[n], nodes=[1], hkv=8, g=4, dk=128, dv=128, page=16, qt=qt, beta=True, seed=n)


@pytest.mark.parametrize("hkv", [1, 3, 5, 8, 11])
@pytest.mark.parametrize("kind,qt,page", [(R.Q8_0, torch.float32, 64), (R.F16, torch.float16, 32), (R.Q4_1, torch.float32, 5)])
def test_tree_long(kvc, hkv, kind, qt, page):
    """Stretches of many tiles per CTA, so that its ring of tiles turns several times, with warps to spare or not."""
    tree_check(kvc, lens=[30000, 25000 // hkv], nodes=[1, 1], hkv=hkv, g=2, dk=128, dv=128, kt=kind, vt=kind, qt=qt, page=page,
               beta=True, seed=hkv)


@pytest.mark.parametrize("kind,qt", [(R.Q8_0, torch.float32), (R.F16, torch.float16), (R.F16, torch.float32)])
def test_tree_many_rows_long(kvc, kind, qt):
    tree_check(kvc, lens=[60000], nodes=[35], hkv=3, g=2, dk=128, dv=128, kt=kind, vt=kind, qt=qt, page=64, beta=True)


@pytest.mark.parametrize("nodes", [[2], [33], [64, 1, 30], [100], [0, 5, 0]])
@pytest.mark.parametrize("g", [1, 4])
def test_tree_nodes(kvc, nodes, g):
    tree_check(kvc, lens=[100] * len(nodes), nodes=nodes, g=g, dk=128, dv=128, kt=R.F16, vt=R.F16, seed=sum(nodes))
    tree_check(kvc, lens=[20] * len(nodes), nodes=nodes, g=g, kt=R.Q4_0, vt=R.Q8_0, qt=torch.float32, seed=sum(nodes))


def test_tree_many_sequences(kvc):
    lens = [(i * 37) % 90 for i in range(150)]
    tree_check(kvc, lens=lens, nodes=[1 + i % 3 for i in range(150)], hkv=1, g=2, kt=R.Q8_0, vt=R.F16, page=8, beta=True)
    tree_check(kvc, lens=lens, nodes=[1] * 150, hkv=4, g=2, kt=R.Q8_0, vt=R.Q8_0, page=32)


def attend_entries(c, q, cu, bits, scale):
    """The definition, an entry at a time over all heads."""
    H, g = c.hkv, q.shape[1] // c.hkv
    out, lse = [], []
    for i in range(len(cu) - 1):
        rows, m = c.rows(i), cu[i + 1] - cu[i]
        K, V = (R.decode(x[0][rows], k).view(len(rows), H, -1) for x, k in ((c.K, c.kt), (c.V, c.vt)))
        x = torch.einsum("mhgd,nhd->mhgn", q[cu[i]:cu[i + 1]].double().view(m, H, g, -1), K) * scale
        if c.beta is not None:
            x = x + c.beta[0, rows // c.page, :, rows % c.page].double().t()[None, :, None]
        see = torch.ones(m, len(rows), dtype=torch.bool)
        see[:, len(rows) - m:] = torch.tensor([[bool((int(bits[cu[i] + a, b // 32]) >> (b % 32)) & 1) for b in range(m)]
                                               for a in range(m)])
        x = x.masked_fill(~see.cuda()[:, None, None], -math.inf)
        lse.append(torch.logsumexp(x, -1).flatten(1))
        out.append(torch.einsum("mhgn,nhd->mhgd", torch.softmax(x, -1), V).flatten(1, 2))
    return torch.cat(out), torch.cat(lse)


@pytest.mark.parametrize("entries", [64, 65, 128, 129])
@pytest.mark.parametrize("hkv,g,d,kind,page,most", [(296, 1, 256, R.F16, 8, 1), (148, 1, 256, R.F16, 8, 1), (296, 1, 256, R.F16, 5, 1),
                                                    (160, 4, 64, R.F16, 16, 40), (160, 2, 64, R.Q8_0, 8, 70)])
def test_tree_many_entries_per_worker(kvc, hkv, g, d, kind, page, most, entries):
    """More entries in a CTA's stretch than its list of pieces holds: with so many heads one CTA (two of 148 heads) has all
    entries of its heads. `most` > 32: the kernel for many query rows, whose entries of several tiles and row blocks are
    among the others."""
    lens = [(i * 37) % (8 if most == 1 else 100) for i in range(entries)]
    nodes = [most if i in (3, entries - 1) else 1 + i % min(2, most) for i in range(entries)]
    c = R.Cache([a + b for a, b in zip(lens, nodes)], hkv, d, d, kind, kind, page, beta=True, seed=entries)
    gen = torch.Generator().manual_seed(entries)
    q = torch.randn(sum(nodes), hkv * g, d, generator=gen).cuda().half()
    cu = [sum(nodes[:i]) for i in range(entries + 1)]
    bits = attn.tree_mask([[int(torch.randint(-1, i, (1,), generator=gen)) if i else -1 for i in range(n)] for n in nodes])
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    t = attn.Tree(kvc, c.handle(kvc), q, dev(cu), dev(list(range(entries))), mask=bits.cuda(), max_nodes=most, scale=d ** -0.5)
    t.out.fill_(7.0)
    t.run()
    out, lse = attend_entries(c, q, cu, bits, d ** -0.5)
    used = torch.cat([c.rows(i) for i in range(entries)])
    # |q||k| per head, row by row of q: A of bounds() without a product over all heads
    A = float((q.double().norm(dim=-1).max() * R.decode(c.K[0][used], kind).view(-1, hkv, d).norm(dim=-1).max())) * d ** -0.5
    v = float(R.decode(c.V[0][used], kind).abs().max())
    e = A * 2.0 ** -21 + (A + float(c.beta.abs().max())) * 2.0 ** -22 + 2.0 ** -21
    check(t.out, out, 2 * e * v + 2.0 ** -21 * v + 2 * 2.0 ** -11 * v, "out")
    check(t.lse, lse, 2 * e + 2.0 ** -21, "lse")
    first = t.out.clone()
    t.run()
    torch.cuda.synchronize()
    assert torch.equal(first, t.out) and int(c.status) == 0


def test_tree_without_mask_sees_all(kvc):
    tree_check(kvc, lens=[40, 3], nodes=[4, 2], mask=None)
    tree_check(kvc, lens=[40, 3], nodes=[4, 2], mask=None, kt=R.F32, vt=R.F32)


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q8_0])
@pytest.mark.parametrize("nodes", [[1, 3], [40, 1]])
def test_tree_mask_without_words(kvc, kind, nodes):
    """Shows no node's own row, as a mask of zeros does."""
    c, q, t, (out, lse) = tree_case(kvc, lens=[40, 3], nodes=nodes, kt=kind, vt=kind, qt=torch.float32, mask="none")
    none = torch.zeros(sum(nodes), 0, dtype=torch.int32, device="cuda")
    u = attn.Tree(kvc, c.handle(kvc), q, t._keep[1], t._keep[2], mask=none, max_nodes=max(nodes), scale=64 ** -0.5)
    u.run()
    t.run()
    torch.cuda.synchronize()
    assert torch.equal(u.out, t.out) and torch.equal(u.lse, t.lse)
    assert float((u.out.double() - out).abs().max()) < 1e-4


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q8_0])
def test_tree_rows_that_see_nothing(kvc, kind):
    """No cached rows and an empty mask, or beta of -inf on every row: output 0, log-sum-exp -inf."""
    t = tree_check(kvc, lens=[0, 20], nodes=[3, 2], kt=kind, vt=kind, mask="none")
    assert float(t.out[:3].abs().max()) == 0.0 and bool((t.lse[:3] == -math.inf).all())
    t = tree_check(kvc, lens=[33, 5], nodes=[1, 1], kt=kind, vt=kind, beta=True,
                   edit=lambda c, q: c.beta.fill_(-math.inf))
    assert float(t.out.abs().max()) == 0.0 and bool((t.lse == -math.inf).all())


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q8_0, R.Q4_1])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
def test_tree_lowest_beta(kvc, kind, qt):
    """beta of the type's lowest value is a finite bias: alone it leaves a plain average, next to others nothing."""
    low = torch.finfo(torch.float32).min
    tree_check(kvc, lens=[40], nodes=[1], kt=kind, vt=kind, qt=qt, beta=True, edit=lambda c, q: c.beta.fill_(low))

    def some(c, q):
        c.beta[..., ::3] = low
    tree_check(kvc, lens=[40], nodes=[1], kt=kind, vt=kind, qt=qt, beta=True, edit=some)


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q8_0, R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 60000.0])
def test_tree_hidden_rows_may_hold_anything(kvc, kind, bad):
    """Rows hidden by beta, by the mask, behind a sequence's end, or in free pages."""
    def edit(c, q):
        rows = c.rows(0)
        hidden = [int(rows[5]), int(rows[16]), int(rows[40])]
        for r in hidden:
            c.beta[0, r // c.page, :, r % c.page] = -math.inf
        own = c.rows(1)[-1:].tolist()                  # the last node's own row: the others do not see it
        free = [r for r in range(c.n_pages * c.page) if r not in set(torch.cat([c.rows(0), c.rows(1)]).tolist())]
        for store, t in ((c.K, c.kt), (c.V, c.vt)):
            for r in hidden + own + free:
                if t == R.F32:
                    store[0, r].view(torch.float32).fill_(bad)
                elif t == R.F16:
                    store[0, r].view(torch.float16).fill_(bad)
                else:
                    b = store[0, r].view(-1, R.BLOCK[t])
                    b[:, :2] = torch.tensor([bad], dtype=torch.float16).view(torch.uint8).to(b.device)
    for qt in (torch.float16, torch.float32):
        c, q, t, (out, lse) = tree_case(kvc, lens=[50, 20], nodes=[1, 4], kt=kind, vt=kind, beta=True, page=16, qt=qt,
                                        edit=edit, seed=3)
        t.run()
        torch.cuda.synchronize()
        # the last node sees its own row and gets what that gives; everybody else is as if it were not there
        ok = torch.ones(5, dtype=torch.bool, device="cuda")
        ok[4] = False
        assert bool(torch.isfinite(t.out[ok]).all()) and bool(torch.isfinite(t.lse[ok]).all())
        assert float((t.out[ok].double() - out[ok]).abs().max()) <= 4 * 2.0 ** -11 * 5
        if not math.isfinite(bad):
            assert not bool(torch.isfinite(t.out[4]).all())


def test_tree_large_and_small_scales(kvc):
    """Block scales from fp16's largest to its subnormals, queries far from 1."""
    for size in (1e-6, 1e-2, 3e3):
        def edit(c, q):
            for store, t in ((c.K, c.kt), (c.V, c.vt)):
                b = store[0].view(-1, R.BLOCK[t])
                d = b[:, :2].contiguous().view(torch.float16).float() * size
                b[:, :2] = d.half().view(torch.uint8)
            q.mul_(1.0 / size)
        for kind in (R.Q8_0, R.Q4_1):
            tree_check(kvc, lens=[100], nodes=[1], kt=kind, vt=kind, qt=torch.float32, edit=edit, seed=11)


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q8_0])
@pytest.mark.parametrize("nodes", [[1, 2], [40, 2]])
def test_tree_huge_queries(kvc, kind, nodes):
    """F32 queries up to 2^120: scores of up to 2^122, of which the largest takes everything."""
    def edit(c, q):
        q[0] *= 2.0 ** 118
    c, q, t, (out, lse) = tree_case(kvc, lens=[90, 33], nodes=nodes, kt=kind, vt=kind, qt=torch.float32, edit=edit)
    t.run()
    torch.cuda.synchronize()
    # one key's values alone: no rounding but the pieces' (2^-21); the score itself is off by 2^-21 of sum |q||k|, which is
    # some 8 times its largest value here, and its product with the scale by 2^-23
    v = float(R.decode(c.V[0], kind).abs().max())
    assert float((t.out[0].double() - out[0]).abs().max()) <= 2.0 ** -20 * v
    assert float((t.lse[0].double() / lse[0] - 1).abs().max()) < 2.0 ** -17
    assert float((t.out[1:].double() - out[1:]).abs().max()) < 1e-4


def test_tree_bad_pages_and_slots(kvc):
    """Entries outside the pool count as no rows; an id outside the cache as an empty sequence."""
    for hkv, page, kt in ((2, 16, R.Q8_0), (3, 16, R.Q8_0), (2, 16, R.F32), (2, 5, R.F16)):
        c, q, t, _ = tree_case(kvc, lens=[60], nodes=[1], hkv=hkv, page=page, kt=kt, vt=kt, qt=torch.float32, beta=True)
        c.table[0, 1], c.table[0, 2] = -1, c.n_pages
        t.run()
        torch.cuda.synchronize()
        n = int(c.seq_len[0])
        keep = [r for r in range(n) if r // page not in (1, 2)]
        table = c.table[0].tolist()
        rows = torch.tensor([table[r // page] * page + r % page for r in keep], device="cuda")
        K, V = R.decode(c.K[0][rows], kt).view(-1, hkv, 64), R.decode(c.V[0][rows], kt).view(-1, hkv, 64)
        for h in range(q.shape[1]):
            bias = c.beta[0, rows // page, h // 4, rows % page]
            o, w = R.attend(q[:, h], K[:, h // 4], V[:, h // 4], bias, torch.ones(1, len(keep), dtype=torch.bool, device="cuda"),
                            64 ** -0.5)
            assert float((t.out[:, h].double() - o).abs().max()) < 1e-4 and float((t.lse[:, h].double() - w).abs().max()) < 1e-4
    c, q, t, _ = tree_case(kvc, lens=[60, 5], nodes=[1, 1], seqs=[0, 1])
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for ids in ([0, 99], [0, -1]):
        u = attn.Tree(kvc, c.handle(kvc), q, dev([0, 1, 2]), dev(ids), max_nodes=1)
        u.out.fill_(3.0)
        u.run()
        torch.cuda.synchronize()
        assert float(u.out[1].abs().max()) == 0.0 and bool((u.lse[1] == -math.inf).all())


def test_tree_layers_strides_and_rows_behind(kvc):
    """Another layer of the cache, queries in a wider tensor, output rows that belong to no entry."""
    tree_check(kvc, lens=[90, 20], nodes=[1, 3], layers=3, layer=2, beta=True)
    c, q, t, (out, lse) = tree_case(kvc, lens=[90, 20], nodes=[1, 3], qt=torch.float32)
    wide = torch.randn(6, 3 * 8, 64, device="cuda")
    wide[:4, 8:16] = q
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    mask = torch.zeros(6, 1, dtype=torch.int32, device="cuda")
    mask[:4] = t._keep[3]
    for view in (wide[:, 8:16], wide.flatten(1)[:, 8 * 64 + 0:16 * 64].view(6, 8, 64)):
        u = attn.Tree(kvc, c.handle(kvc), view, dev([0, 1, 4]), dev([0, 1]), mask=mask, max_nodes=3, scale=64 ** -0.5)
        u.out.fill_(5.0)
        u.lse.fill_(5.0)
        u.run()
        torch.cuda.synchronize()
        assert bool((u.out[4:] == 5.0).all()) and bool((u.lse[4:] == 5.0).all())
        assert float((u.out[:4].double() - out).abs().max()) < 1e-4
    # entries with more nodes than max_nodes are cut to it
    u = attn.Tree(kvc, c.handle(kvc), view, dev([0, 1, 4]), dev([0, 1]), mask=mask, max_nodes=1, scale=64 ** -0.5)
    u.out.fill_(5.0)
    u.run()
    torch.cuda.synchronize()
    assert bool((u.out[2:] == 5.0).all()) and float((u.out[0].double() - out[0]).abs().max()) < 1e-4


def test_tree_on_a_stream_and_in_a_graph(kvc):
    c, q, t, (out, _) = tree_case(kvc, lens=[3000, 100], nodes=[1, 2], qt=torch.float32, hkv=4, dk=128, dv=128)
    t.run()
    torch.cuda.synchronize()
    want = t.out.clone()
    side = torch.cuda.Stream()
    t.out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t.run()
    side.synchronize()
    assert torch.equal(t.out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t.run()
        t.run()
    t.out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(t.out, want)
    # a longer sequence and other queries, the same graph
    c.seq_len[0] = 1500
    q.copy_(torch.randn_like(q))
    g.replay()
    torch.cuda.synchronize()
    bits = t._keep[3].cpu()
    cu = [0, 1, 3]

    def see(i, m, n):
        s = torch.ones(m, n, dtype=torch.bool)
        for a in range(m):
            for b in range(m):
                s[a, n - m + b] = bool((int(bits[cu[i] + a, 0]) >> b) & 1)
        return s
    out, _ = c.attend(q, cu, [0, 1], see, 128 ** -0.5)
    assert float((t.out.double() - out).abs().max()) < 2e-4


def test_tree_refuses_a_small_workspace(kvc):
    c, q, t, _ = tree_case(kvc, lens=[3000], nodes=[1])
    cache, desc, ws, size = t._args
    assert size > 0
    assert t.fn(cache, desc, ws, size - 1, None) == -13
    assert t.fn(cache, desc, None, size, None) == -1
    assert t.fn(cache, desc, ws + 4, size, None) == -13


def test_tree_workspace_of_many_nodes(kvc):
    """The partial results go by the workers, not by the rows of an entry: a worker shares two pieces at most."""
    c, q, t, _ = tree_case(kvc, lens=[100], nodes=[40], hkv=8, g=4, dk=128, dv=128, kt=R.F16, vt=R.F16)
    size = {}
    for n in (40, 1000, 16000):
        t.desc.total, t.desc.max_nodes = n, n
        rc = ctypes.c_int(0)
        size[n] = kvc["_lib"].kvc_attn_tree_workspace(t.cache.ref, t.ref, ctypes.addressof(rc))
        assert rc.value == 0
    assert size[40] < size[1000] < size[16000] < size[40] + 16000 * 4      # meta: two numbers per 128 rows and entry


@pytest.mark.parametrize("kind,qt", [(R.F16, torch.float16), (R.Q8_0, torch.float32)])
def test_tree_several_row_blocks_in_a_stretch(kvc, kind, qt):
    """Row blocks laid end to end over the workers, with entries that start and end anywhere in a worker's stretch."""
    tree_check(kvc, lens=[700, 0, 90, 3000], nodes=[100, 70, 3, 150], hkv=3, g=4, kt=kind, vt=kind, qt=qt, page=16, beta=True)
    tree_check(kvc, lens=[20, 5000], nodes=[300, 65], hkv=1, g=2, kt=kind, vt=kind, qt=qt, page=64)


def many_rows(**kw):
    """Sequences with enough nodes that the kernels for many query rows take them, at head size d too."""
    return dict(dict(lens=[200, 0, 70, 513], nodes=[24, 40, 1, 33], hkv=2, g=4, page=16, beta=True), **kw)


@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("vt", KINDS)
@pytest.mark.parametrize("kt", KINDS)
def test_tree_many_rows_types(kvc, kt, vt, qt):
    tree_check(kvc, **many_rows(kt=kt, vt=vt, qt=qt, seed=kt * 10 + vt))


@pytest.mark.parametrize("dk,dv", [(32, 64), (64, 128), (128, 32), (96, 96), (128, 128)])
@pytest.mark.parametrize("kind", [R.F16, R.Q8_0, R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
def test_tree_many_rows_head_sizes(kvc, dk, dv, kind, qt):
    tree_check(kvc, **many_rows(dk=dk, dv=dv, kt=kind, vt=kind, qt=qt, seed=dk + dv))


@pytest.mark.parametrize("rows", [9, 16, 17, 32, 33, 64, 65, 127, 128, 129, 260])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", [R.F16, R.Q8_0])
def test_tree_row_counts(kvc, rows, d, kind):
    """Each number of query rows on either side of a kernel's rows, with one head to a KV head."""
    tree_check(kvc, lens=[300, 40], nodes=[rows, 3], hkv=2, g=1, dk=d, dv=d, kt=kind, vt=kind, page=24, seed=rows)


@pytest.mark.parametrize("page", [1, 7, 64, 100, 256])
@pytest.mark.parametrize("kind", [R.F16, R.Q8_0])
def test_tree_many_rows_pages(kvc, page, kind):
    tree_check(kvc, **many_rows(page=page, kt=kind, vt=kind, hkv=3, g=5, seed=page))


@pytest.mark.parametrize("kind", [R.F16, R.Q8_0, R.Q4_1])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
def test_tree_many_rows_that_see_nothing(kvc, kind, qt):
    t = tree_check(kvc, lens=[0, 20], nodes=[30, 2], kt=kind, vt=kind, qt=qt, mask="none")
    assert float(t.out[:30].abs().max()) == 0.0 and bool((t.lse[:30] == -math.inf).all())
    t = tree_check(kvc, **many_rows(kt=kind, vt=kind, qt=qt, edit=lambda c, q: c.beta.fill_(-math.inf)))
    assert float(t.out.abs().max()) == 0.0 and bool((t.lse == -math.inf).all())
    low = torch.finfo(torch.float32).min
    tree_check(kvc, **many_rows(kt=kind, vt=kind, qt=qt, edit=lambda c, q: c.beta.fill_(low)))


@pytest.mark.parametrize("kind", [R.F16, R.Q8_0, R.Q4_0, R.Q4_1])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
def test_tree_many_rows_hidden_rows_may_hold_anything(kvc, kind, bad, qt):
    """As above where 128 query rows share a tile: rows behind beta, the last node's own row, free pages."""
    def edit(c, q):
        rows = c.rows(0)
        hidden = [int(rows[i]) for i in (0, 5, 63, 64, 130)]
        for r in hidden:
            c.beta[0, r // c.page, :, r % c.page] = -math.inf
        used = torch.cat([c.rows(i) for i in range(3)])
        free = sorted(set(range(c.n_pages * c.page)) - set(used.tolist()))
        for store, t in ((c.K, c.kt), (c.V, c.vt)):
            for r in hidden + c.rows(0)[-1:].tolist() + free:
                if t == R.F16:
                    store[0, r].view(torch.float16).fill_(bad)
                else:
                    b = store[0, r].view(-1, R.BLOCK[t])
                    b[:, :2] = torch.tensor([bad], dtype=torch.float16).view(torch.uint8).to(b.device)
    nodes = [40, 3, 20]
    c, q, t, (out, lse) = tree_case(kvc, lens=[150, 20, 64], nodes=nodes, kt=kind, vt=kind, beta=True, page=16, qt=qt, edit=edit)
    used = torch.cat([c.rows(i) for i in range(3)])
    K, V = (R.decode(x[0][used], kind).nan_to_num(0.0, 0.0, 0.0) for x in (c.K, c.V))
    t.run()
    torch.cuda.synchronize()
    ok = torch.ones(sum(nodes), dtype=torch.bool, device="cuda")
    ok[nodes[0] - 1] = False                           # only the last node sees the bad row of its own
    o_tol, l_tol = bounds(q, K.view(-1, c.hkv, c.dk), V, float(c.beta[c.beta.isfinite()].abs().max()), kind,
                          qt == torch.float16, c.dk ** -0.5)
    check(t.out[ok], out[ok], o_tol, "out")
    check(t.lse[ok], lse[ok], l_tol, "lse")
    assert not bool(torch.isfinite(t.out[nodes[0] - 1]).all())


def test_tree_many_rows_large_and_small_scales(kvc):
    for size in (1e-6, 1e-2, 3e3):
        def edit(c, q):
            for store, t in ((c.K, c.kt), (c.V, c.vt)):
                b = store[0].view(-1, R.BLOCK[t])
                d = b[:, :2].contiguous().view(torch.float16).float() * size
                b[:, :2] = d.half().view(torch.uint8)
            q.mul_(1.0 / size)
        for kind in (R.Q8_0, R.Q4_1):
            tree_check(kvc, lens=[100], nodes=[36], kt=kind, vt=kind, qt=torch.float32, edit=edit, seed=11)


def test_tree_many_rows_bad_pages(kvc):
    for kt in (R.F16, R.Q8_0):
        c, q, t, _ = tree_case(kvc, lens=[200], nodes=[36], hkv=2, page=16, kt=kt, vt=kt, qt=torch.float32, beta=True,
                               mask=None)
        c.table[0, 1], c.table[0, 4] = -1, c.n_pages
        t.run()
        torch.cuda.synchronize()
        n = int(c.seq_len[0])
        keep = [r for r in range(n) if r // 16 not in (1, 4)]
        table = c.table[0].tolist()
        rows = torch.tensor([table[r // 16] * 16 + r % 16 for r in keep], device="cuda")
        K, V = R.decode(c.K[0][rows], kt).view(-1, 2, 64), R.decode(c.V[0][rows], kt).view(-1, 2, 64)
        for h in range(q.shape[1]):
            see = torch.ones(36, len(keep), dtype=torch.bool, device="cuda")
            o, w = R.attend(q[:, h], K[:, h // 4], V[:, h // 4], c.beta[0, rows // 16, h // 4, rows % 16], see, 64 ** -0.5)
            assert float((t.out[:, h].double() - o).abs().max()) < 1e-4 and float((t.lse[:, h].double() - w).abs().max()) < 1e-4


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q8_0])
@pytest.mark.parametrize("nodes", [[2, 2, 1], [40, 40, 3]])
def test_tree_one_sequence_read_twice(kvc, kind, nodes):
    """Several entries over one sequence (the same slot more than once)."""
    tree_check(kvc, lens=[300 - nodes[0], 20 - nodes[1] % 20, 7], nodes=nodes, seqs=[0, 0, 0], kt=kind, vt=kind, beta=True)


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q8_0])
@pytest.mark.parametrize("nodes", [6, 40])
def test_tree_shorter_than_its_nodes(kvc, kind, nodes):
    """A sequence with fewer rows than the entry has nodes: the rows belong to the last nodes."""
    tree_check(kvc, lens=[3 - nodes, 50], nodes=[nodes, 2], kt=kind, vt=kind, qt=torch.float32, beta=True)


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q8_0])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
@pytest.mark.parametrize("nodes", [[1, 3], [40, 3]])
def test_tree_a_bad_query_spoils_its_own_rows(kvc, kind, qt, nodes):
    for bad in (math.nan, math.inf):
        c, q, t, (out, lse) = tree_case(kvc, lens=[90, 33], nodes=nodes, kt=kind, vt=kind, qt=qt, beta=True)
        q[1, 5] = bad
        t.run()
        torch.cuda.synchronize()
        ok = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
        ok[1, 5] = False
        used = torch.cat([c.rows(0), c.rows(1)])
        K, V = (R.decode(x[0][used], kind) for x in (c.K, c.V))
        good = torch.where(ok[..., None], q, torch.zeros_like(q))
        o_tol, l_tol = bounds(good, K.view(-1, c.hkv, c.dk), V, float(c.beta.abs().max()), kind, qt == torch.float16, c.dk ** -0.5)
        check(t.out[ok], out[ok], o_tol, "out")
        check(t.lse[ok], lse[ok], l_tol, "lse")


@pytest.mark.parametrize("kt,vt", [(R.Q8_0, R.Q8_0), (R.Q4_0, R.Q8_0), (R.Q4_1, R.Q4_0)])
@pytest.mark.parametrize("nodes", [[1, 2], [40, 2]])
def test_tree_rows_of_odd_blocks(kvc, kt, vt, nodes):
    """Rows whose size is no multiple of four bytes."""
    for hkv in (1, 3):
        tree_check(kvc, lens=[90, 20], nodes=nodes, hkv=hkv, dk=32, dv=32, kt=kt, vt=vt, qt=torch.float32, page=7, beta=True)


@pytest.mark.parametrize("kind", [R.F32, R.F16, R.Q4_0])
def test_tree_more_heads_than_workers(kvc, kind):
    tree_check(kvc, lens=[70, 0], nodes=[1, 0], hkv=320, g=1, dk=32, dv=32, kt=kind, vt=kind)
    tree_check(kvc, lens=[70, 0], nodes=[40, 0], hkv=160, g=1, dk=32, dv=32, kt=kind, vt=kind)


def test_tree_calls_side_by_side(kvc):
    """Two calls over one cache on two streams, each with its own workspace; a graph next to them."""
    c, q, t, (out, _) = tree_case(kvc, lens=[5000, 300], nodes=[2, 40], qt=torch.float32, hkv=4)
    t.run()
    torch.cuda.synchronize()
    want = t.out.clone()
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    calls = [attn.Tree(kvc, c.handle(kvc), q, dev([0, 2, 42]), dev([0, 1]), mask=t._keep[3], max_nodes=40, scale=64 ** -0.5)
             for _ in range(3)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        calls[2].run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, u in zip(streams, calls):
            with torch.cuda.stream(s):
                u.run()
        g.replay()
    torch.cuda.synchronize()
    for u in calls:
        assert torch.equal(u.out, want)


def test_calls_from_host_threads(kvc):
    """Calls of the general kernel with different head sizes from several host threads, each on a stream of its own. (The
    C calls are made directly, so that they meet; a call that is refused gives its code.)"""
    sizes = [(256, 100), (32, 100), (200, 100), (32, 66)]
    gate, failed = threading.Barrier(len(sizes)), []

    def worker(dk, dv):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                c, q, t, _ = tree_case(kvc, lens=[4], nodes=[1], hkv=1, g=1, dk=dk, dv=dv, kt=R.F32, vt=R.F32, qt=torch.float32)
                t.run()
                torch.cuda.current_stream().synchronize()
                want, st = t.out.clone(), torch.cuda.current_stream().cuda_stream
                gate.wait(60)
                codes = {t.fn(*t._args, st) for _ in range(20000)}
                torch.cuda.current_stream().synchronize()
                assert codes == {0} and torch.equal(t.out, want)
        except Exception as e:  # noqa: BLE001
            gate.abort()
            failed.append(f"{dk}, {dv}: {e}")

    threads = [threading.Thread(target=worker, args=a) for a in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("kind,page,nodes", [(R.F16, 16, [1, 2]), (R.F16, 16, [40, 2]), (R.F16, 5, [1, 2]), (R.F32, 16, [1, 2])])
def test_tree_far_rows(kvc, kind, page, nodes):
    """Pages more than 4 GiB into the pool."""
    c, q, t, (out, lse) = tree_case(kvc, lens=[200, 33], nodes=nodes, hkv=8, dk=128, dv=128, kt=kind, vt=kind, page=page,
                                    qt=torch.float32)
    t.run()
    torch.cuda.synchronize()
    rb, rows = c.K.shape[2], c.K.shape[1]
    far = (-(-(2 ** 32 + 2 ** 20) // rb) // page + 1) * page
    K, V = (torch.empty(1, far + rows, rb, dtype=torch.uint8, device="cuda") for _ in range(2))
    K[:, far:], V[:, far:] = c.K, c.V
    c.K, c.V = K, V
    c.table[c.table >= 0] += far // page
    c.ref = torch.zeros((far + rows) // page, dtype=torch.int32, device="cuda")
    u = attn.Tree(kvc, c.handle(kvc), q, t._keep[1], t._keep[2], mask=t._keep[3], max_nodes=max(nodes), scale=128 ** -0.5)
    u.run()
    torch.cuda.synchronize()
    assert torch.equal(u.out, t.out) and torch.equal(u.lse, t.lse)
    assert float((u.out.double() - out).abs().max()) < 1e-4


@pytest.mark.parametrize("kind,nodes,cut", [(R.F32, [1, 3], 1), (R.F32, [1, 20], 9), (R.Q8_0, [1, 3], 1), (R.F16, [2, 9], 5),
                                            (R.F16, [1, 60], 40), (R.Q8_0, [3, 80], 36)])
@pytest.mark.parametrize("qt", [torch.float16, torch.float32])
def test_tree_cut_entries(kvc, kind, nodes, cut, qt):
    """An entry with more nodes than max_nodes: the nodes that are left see what they would see beside the others (whose
    own rows are in the cache all the same), and the rows of the others are left as they were."""
    c, q, t, (out, lse) = tree_case(kvc, lens=[90, 70], nodes=nodes, kt=kind, vt=kind, qt=qt, beta=True, seed=cut)
    u = attn.Tree(kvc, c.handle(kvc), q, t._keep[1], t._keep[2], mask=t._keep[3], max_nodes=cut, scale=64 ** -0.5)
    u.out.fill_(5.0)
    u.lse.fill_(5.0)
    u.run()
    torch.cuda.synchronize()
    used = torch.cat([c.rows(0), c.rows(1)])
    K, V = (R.decode(x[0][used], kind) for x in (c.K, c.V))
    o_tol, l_tol = bounds(q, K.view(-1, c.hkv, c.dk), V, float(c.beta.abs().max()), kind, qt == torch.float16, c.dk ** -0.5)
    for first, n in ((0, min(nodes[0], cut)), (nodes[0], min(nodes[1], cut))):
        check(u.out[first:first + n], out[first:first + n], o_tol, "out")
        check(u.lse[first:first + n], lse[first:first + n], l_tol, "lse")
    behind = slice(nodes[0] + cut, None)
    assert bool((u.out[behind] == 5.0).all()) and bool((u.lse[behind] == 5.0).all())


def test_tree_max_nodes_left_out(kvc):
    """Where max_nodes is not given, a mask or more rows than entries make it the number of rows; else it is 1."""
    c, q, t, (out, _) = tree_case(kvc, lens=[40, 9], nodes=[1, 5], qt=torch.float32)
    u = attn.Tree(kvc, c.handle(kvc), q, t._keep[1], t._keep[2], mask=t._keep[3], scale=64 ** -0.5)
    u.run()
    torch.cuda.synchronize()
    assert u.desc.max_nodes == 6 and float((u.out.double() - out).abs().max()) < 1e-4
    assert attn.Tree(kvc, c.handle(kvc), q, t._keep[1], t._keep[2]).desc.max_nodes == 6
    assert attn.Tree(kvc, c.handle(kvc), q[:2], t._keep[1], t._keep[2], mask=t._keep[3][:2]).desc.max_nodes == 2
    assert attn.Tree(kvc, c.handle(kvc), q[:2], t._keep[1], t._keep[2]).desc.max_nodes == 1


# ---- prompts ------------------------------------------------------------------------------

def prompt_case(new, past, hkv=2, g=4, dk=64, dv=64, dtype=torch.float16, causal=True, seed=0, wide=False, scale=None, edit=None):
    gen = torch.Generator().manual_seed(seed)
    nk = [a + b for a, b in zip(new, past)]
    rnd = lambda *s: torch.randn(*s, generator=gen).to("cuda", dtype)  # noqa: E731
    q, k, v = rnd(sum(new), hkv * g, dk), rnd(sum(nk), hkv, dk), rnd(sum(nk), hkv, dv)
    if wide:                                           # slices of one fused projection
        fused = rnd(sum(new), hkv * (g * dk + dk + dv))
        fused[:, :hkv * g * dk] = q.flatten(1)
        fused[:, hkv * g * dk:hkv * (g + 1) * dk] = k.flatten(1)
        fused[:, hkv * (g + 1) * dk:] = v.flatten(1)
        q = fused[:, :hkv * g * dk].unflatten(1, (hkv * g, dk))
        k = fused[:, hkv * g * dk:hkv * (g + 1) * dk].unflatten(1, (hkv, dk))
        v = fused[:, hkv * (g + 1) * dk:].unflatten(1, (hkv, dv))
    if edit:
        edit(q, k, v)
    cum = lambda x: torch.tensor([sum(x[:i]) for i in range(len(x) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
    scale = dk ** -0.5 if scale is None else scale
    out = torch.zeros(sum(new), hkv * g, dv, dtype=torch.float64, device="cuda")
    lse = torch.zeros(sum(new), hkv * g, dtype=torch.float64, device="cuda")
    a0 = b0 = 0
    for a, b in zip(new, nk):
        i, j = torch.arange(a, device="cuda")[:, None], torch.arange(b, device="cuda")[None]
        see = (j <= i + b - a) if causal else (j >= 0) & (i >= 0)
        for h in range(hkv * g):
            out[a0:a0 + a, h], lse[a0:a0 + a, h] = R.attend(q[a0:a0 + a, h], k[b0:b0 + b, h // g].double(),
                                                            v[b0:b0 + b, h // g].double(), None, see, scale)
        a0, b0 = a0 + a, b0 + b
    return q, k, v, cum(new), cum(nk), scale, out, lse


def prompt_check(kvc, *args, **kw):
    q, k, v, cu_q, cu_k, scale, out, lse = prompt_case(*args, **kw)
    p = attn.Prompt(kvc, q, k, v, cu_q, cu_k, scale=scale, causal=kw.get("causal", True))
    o_tol, l_tol = bounds(q, k.double(), v.double(), 0.0, R.F16, q.dtype == torch.float16, abs(scale))
    p.out.fill_(7.0)
    p.run()
    torch.cuda.synchronize()
    check(p.out, out, o_tol, "out")
    check(p.lse, lse, l_tol, "lse")
    first = p.out.clone()
    p.run()
    torch.cuda.synchronize()
    assert torch.equal(first, p.out)
    return p


@pytest.mark.parametrize("d", [8, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("g", [1, 3, 4])
def test_prompt_head_sizes(kvc, d, g):
    prompt_check(kvc, [130, 1, 70], [0, 0, 0], g=g, dk=d, dv=d, seed=d)


@pytest.mark.parametrize("dk,dv", [(64, 128), (128, 64), (32, 96), (136, 64), (256, 256), (20, 20), (7, 5)])
def test_prompt_other_head_sizes(kvc, dk, dv):
    prompt_check(kvc, [50, 20], [10, 0], dk=dk, dv=dv, seed=dk)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 600])
def test_prompt_lengths(kvc, n):
    prompt_check(kvc, [n], [0], dk=128, dv=128, seed=n)
    prompt_check(kvc, [n], [0], g=1, seed=n, causal=False)


@pytest.mark.parametrize("past", [1, 100, 128, 511])
def test_prompt_on_past_rows(kvc, past):
    prompt_check(kvc, [65, 3, 1], [past, 0, past + 1], dk=128, dv=128, seed=past)


@pytest.mark.parametrize("g", [1, 2, 5, 7, 16, 128, 130])
def test_prompt_groups(kvc, g):
    prompt_check(kvc, [40, 9], [5, 0], hkv=1, g=g, seed=g)


def test_prompt_many_sequences(kvc):
    new = [(i * 29) % 50 for i in range(90)]
    prompt_check(kvc, new, [(i * 7) % 13 for i in range(90)], hkv=2, g=2)


@pytest.mark.parametrize("d,causal", [(64, True), (128, True), (64, False)])
def test_prompt_long_sequence(kvc, d, causal):
    """One sequence long enough that a CTA takes two tiles; some rows of some heads against the definition."""
    gen = torch.Generator().manual_seed(d)
    n, past, hkv, g = 4801, 77, 8, 4
    rnd = lambda *s: torch.randn(*s, generator=gen).to("cuda", torch.float16)  # noqa: E731
    q, k, v = rnd(n, hkv * g, d), rnd(n + past, hkv, d), rnd(n + past, hkv, d)
    cu = lambda x: torch.tensor([0, x], dtype=torch.int32, device="cuda")  # noqa: E731
    p = attn.Prompt(kvc, q, k, v, cu(n), cu(n + past), scale=d ** -0.5, causal=causal)
    p.out.fill_(7.0)
    p.run()
    torch.cuda.synchronize()
    at = torch.tensor([0, 1, 31, 32, 63, 64, 65, 2047, 2048, 4735, 4736, 4767, 4768, 4799, 4800], device="cuda")
    j = torch.arange(n + past, device="cuda")[None]
    see = (j <= at[:, None] + past) if causal else (j >= 0).expand(len(at), -1)
    o_tol, l_tol = bounds(q, k.double(), v.double(), 0.0, R.F16, True, d ** -0.5)
    for h in (0, 3, 13, 31):
        o, w = R.attend(q[at, h], k[:, h // g].double(), v[:, h // g].double(), None, see, d ** -0.5)
        check(p.out[at, h], o, o_tol, "out")
        check(p.lse[at, h], w, l_tol, "lse")
    first = p.out.clone()
    p.run()
    torch.cuda.synchronize()
    assert torch.equal(first, p.out) and bool(torch.isfinite(p.lse).all())


@pytest.mark.parametrize("d,causal", [(64, True), (128, True), (64, False), (128, False)])
@pytest.mark.parametrize("n", [5999, 6000, 6113])
def test_prompt_either_side_of_two_tiles(kvc, d, causal, n):
    """Sequences of just less and of as many tokens as make a CTA take two tiles; some rows of some heads."""
    gen = torch.Generator().manual_seed(n + d)
    past, hkv, g = 77, 8, 4
    rnd = lambda *s: torch.randn(*s, generator=gen).to("cuda", torch.float16)  # noqa: E731
    q, k, v = rnd(n, hkv * g, d), rnd(n + past, hkv, d), rnd(n + past, hkv, d)
    cu = lambda x: torch.tensor([0, x], dtype=torch.int32, device="cuda")  # noqa: E731
    p = attn.Prompt(kvc, q, k, v, cu(n), cu(n + past), scale=d ** -0.5, causal=causal)
    p.out.fill_(7.0)
    p.run()
    torch.cuda.synchronize()
    at = torch.tensor([0, 31, 32, 63, 64, 127, 128, 2047, 2048, n - 66, n - 65, n - 64, n - 33, n - 32, n - 2, n - 1], device="cuda")
    j = torch.arange(n + past, device="cuda")[None]
    see = (j <= at[:, None] + past) if causal else (j >= 0).expand(len(at), -1)
    o_tol, l_tol = bounds(q, k.double(), v.double(), 0.0, R.F16, True, d ** -0.5)
    for h in (0, 3, 13, 31):
        o, w = R.attend(q[at, h], k[:, h // g].double(), v[:, h // g].double(), None, see, d ** -0.5)
        check(p.out[at, h], o, o_tol, "out")
        check(p.lse[at, h], w, l_tol, "lse")
    first = p.out.clone()
    p.run()
    torch.cuda.synchronize()
    assert torch.equal(first, p.out) and bool(torch.isfinite(p.lse).all())


def test_prompt_fewer_keys_than_queries(kvc):
    """Queries that lie before the first key see nothing; a sequence without keys as well."""
    p = prompt_check(kvc, [100, 5], [-60, -5], dk=128, dv=128)
    assert float(p.out[:60].abs().max()) == 0.0 and bool((p.lse[:60] == -math.inf).all())
    assert float(p.out[100:].abs().max()) == 0.0
    prompt_check(kvc, [7], [-7])
    prompt_check(kvc, [100, 5], [-60, -5], dtype=torch.float32)


def test_prompt_strides(kvc):
    prompt_check(kvc, [70, 20], [0, 0], dk=64, dv=64, wide=True)
    prompt_check(kvc, [70, 20], [0, 0], hkv=1, g=2, dk=24, dv=8, wide=True)
    prompt_check(kvc, [70, 20], [0, 0], hkv=3, g=1, dk=12, dv=4, wide=True)       # strides that are no multiple of 16 bytes


def test_prompt_f32_and_scales(kvc):
    prompt_check(kvc, [70, 20], [3, 0], dtype=torch.float32, dk=96, dv=128)
    for scale in (0.0, -0.3, 1.0):
        prompt_check(kvc, [70, 20], [3, 0], scale=scale)


def test_prompt_growing_maximum(kvc):
    """Scores that rise along the keys move the reference maximum at every step."""
    def edit(q, k, v):
        q.abs_()
        k.abs_()
        k.mul_(torch.linspace(0, 6, k.shape[0], device="cuda")[:, None, None].half())
    prompt_check(kvc, [700], [0], dk=64, dv=64, scale=0.5, edit=edit)


def test_prompt_neighbours_never_matter(kvc):
    """A sequence between others full of NaN and infinities, and rows behind the last one."""
    q, k, v, cu_q, cu_k, scale, out, lse = prompt_case([40, 70, 33], [0, 20, 0], dk=128, dv=128)
    for bad in (math.nan, math.inf):
        for t in (q, k, v):
            t[:40] = bad
            t[-33:] = bad
        p = attn.Prompt(kvc, q, k, v, cu_q, cu_k, scale=scale)
        p.run()
        torch.cuda.synchronize()
        assert float((p.out[40:110].double() - out[40:110]).abs().max()) < 2 * 2.0 ** -11 * 5
        assert bool(torch.isfinite(p.lse[40:110]).all())
    cu_q[3], cu_k[3] = cu_q[2], cu_k[2]                # the last sequence is empty: its rows are nobody's
    p.out.fill_(9.0)
    p.run()
    torch.cuda.synchronize()
    assert bool((p.out[110:] == 9.0).all())


def test_prompt_on_a_stream_and_in_a_graph(kvc):
    q, k, v, cu_q, cu_k, scale, out, lse = prompt_case([300, 20], [0, 0], dk=128, dv=128)
    p = attn.Prompt(kvc, q, k, v, cu_q, cu_k, scale=scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.run()
    side.synchronize()
    want = p.out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.run()
    p.out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(p.out, want) and float((want.double() - out).abs().max()) < 2 * 2.0 ** -11 * 5


@pytest.mark.parametrize("n,d", [(300, 64), (70, 24)])
def test_prompt_far_rows(kvc, n, d):
    """Strides that put the last rows more than 2^31 elements behind the first."""
    wide = torch.empty(n, 2 ** 31 // n // 8 * 8 + 4096, dtype=torch.float16, device="cuda")
    gen = torch.Generator().manual_seed(n)
    q, k, v = (wide[:, i * 8 * d:i * 8 * d + h * d].unflatten(1, (h, d)) for i, h in ((0, 8), (1, 2), (2, 2)))
    for x in (q, k, v):
        x.copy_(torch.randn(x.shape, generator=gen))
    cu = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
    far, near = attn.Prompt(kvc, q, k, v, cu), attn.Prompt(kvc, q.contiguous(), k.contiguous(), v.contiguous(), cu)
    far.run()
    near.run()
    torch.cuda.synchronize()
    assert torch.equal(far.out, near.out) and bool(torch.isfinite(far.out).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prompt_a_bad_query_spoils_its_own_rows(kvc, dtype):
    q, k, v, cu_q, cu_k, scale, out, lse = prompt_case([140, 20], [3, 0], dk=128, dv=128, dtype=dtype)
    q[77, 3] = math.nan
    p = attn.Prompt(kvc, q, k, v, cu_q, cu_k, scale=scale)
    p.run()
    torch.cuda.synchronize()
    ok = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    ok[77, 3] = False
    q = torch.where(ok[..., None], q, torch.zeros_like(q))
    o_tol, l_tol = bounds(q, k.double(), v.double(), 0.0, R.F16, dtype == torch.float16, scale)
    check(p.out[ok], out[ok], o_tol, "out")
    check(p.lse[ok], lse[ok], l_tol, "lse")


def test_prompt_shared_heads_by_stride(kvc):
    """Keys and values expanded over the KV heads (a head stride of 0)."""
    q, k, v, cu_q, cu_k, scale, out, lse = prompt_case([90, 9], [0, 0], hkv=1, g=4)
    p = attn.Prompt(kvc, q, k.expand(-1, 4, -1), v.expand(-1, 4, -1), cu_q, cu_k, scale=scale)
    p.run()
    torch.cuda.synchronize()
    o_tol, l_tol = bounds(q, k.double(), v.double(), 0.0, R.F16, True, scale)
    check(p.out, out, o_tol, "out")
    check(p.lse, lse, l_tol, "lse")


def test_wrappers_check_their_tensors(kvc):
    q, k = torch.randn(4, 4, 64, device="cuda").half(), torch.randn(4, 2, 64, device="cuda").half()
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    for args in ((q.bfloat16(), k.bfloat16(), k.bfloat16(), cu), (q, k.float(), k, cu), (q, k, k, cu.long()),
                 (q, k[:3], k, cu), (q[:, :3], k, k, cu), (q.cpu(), k, k, cu), (q, k, k, cu, cu[:1]),
                 (q.transpose(1, 2), k, k, cu)):
        with pytest.raises(ValueError):
            attn.Prompt(kvc, *args)
    c = R.Cache([10], 2, 64, 64, R.Q8_0, R.Q8_0, 16)
    h, s = c.handle(kvc), torch.zeros(1, dtype=torch.int32, device="cuda")
    for args, kw in (((q[..., :32], cu, s), {}), ((q, cu[:1], s), {}), ((q, cu, s.long()), {}), ((q.bfloat16(), cu, s), {}),
                     ((q, cu, s), dict(mask=torch.zeros(3, 1, dtype=torch.int32, device="cuda"))),
                     ((q, cu, s), dict(out=torch.empty(4, 4, 64, device="cuda")))):
        with pytest.raises(ValueError):
            attn.Tree(kvc, h, *args, max_nodes=4, **kw)
    with pytest.raises(RuntimeError):
        attn.Tree(kvc, h, q, cu, s, max_nodes=4, layer=1)

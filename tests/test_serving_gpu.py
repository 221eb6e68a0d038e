"""The serving operators together, as a server uses them: a prompt is attended to and cached, its cache compacted by the
library, continued by drafted tokens, of which some are kept."""
import pytest
import torch

import servref as R
from kvc_b200 import abi, attn, lib as kvclib, pages

pytestmark = pytest.mark.gpu

L, H, G, D, PAGE = 2, 2, 4, 64, 16


def test_a_conversation(kvc):
    gen = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    n, kind = 1300, R.Q8_0
    cache = pages.PageCache.empty(kvc, L, 400, PAGE, 6, 120, H, D, D, kind, kind, beta=True)
    K, V, Q = rnd(L, n, H * D), rnd(L, n, H * D), rnd(n, H * G, D)

    # the prompt: attended to in one pass, its rows quantised into the cache
    q, k, v = Q.half(), K[0].view(n, H, D).half(), V[0].view(n, H, D).half()
    p = attn.Prompt(kvc, q, k, v, dev([0, n]))
    p.run()
    cache.reserve([0], [n])
    rows = [torch.stack([kvclib.quantize_dev(kvc, x[l].contiguous(), kind) for l in range(L)]) for x in (K, V)]
    cache.write([0], [0], [n], rows[0], rows[1], torch.zeros(L, H, n, device="cuda"))

    # one more token from the cache: what the prompt's last row saw, up to the quantisation
    t = attn.Tree(kvc, cache, Q[n - 1:n].contiguous(), dev([0, 1]), dev([0]))
    t.run()
    cache.check()
    assert float((t.out[0].double() - p.out[n - 1].double()).abs().max()) < 0.05

    # compaction of the rows, read back from the pages, to 30 %
    kr, vr, _ = cache.read([0], [0], [n])
    params = abi.make_params(kvc, target_ratio=0.3, skip_beta=0)
    q_ref = rnd(32, H * D)
    m = kvclib.BatchedModel(kvc, [kr[l] for l in range(L)], [vr[l] for l in range(L)], [q_ref] * L, n, H, D, D, kind, kind,
                            params)
    m.run()
    torch.cuda.synchronize()
    keep = m.t[0]
    assert m.t == [keep] * L and 0 < keep < n
    sel = torch.stack([m.sel[l][:keep] for l in range(L)]).view(L, 1, keep).contiguous()
    v_out = torch.stack([m.vout[l].view(keep, -1) for l in range(L)]).view(L, 1, keep, -1).contiguous()
    beta = torch.stack([m.beta[l].view(H, keep) for l in range(L)]).view(L, 1, H, keep).contiguous()
    before = int((cache.ref_count > 0).sum())
    cache.compact([0], [0], sel, dev([keep]), dev([0]), v_rows=v_out, beta_rows=beta)
    cache.check()
    assert int(cache.seq_len[0]) == keep and int((cache.ref_count > 0).sum()) == -(-keep // PAGE) < before
    got = cache.read([0], [0], [keep])
    for l in range(L):
        assert torch.equal(got[0][l], m.kout[l].view(keep, -1)) and torch.equal(got[1][l], m.vout[l].view(keep, -1))
        assert torch.equal(got[2][l], m.beta[l].view(H, keep))

    # a fork continues with a drafted tree of 5 nodes; rows of the nodes are appended, then verified in one pass
    cache.fork([0], [1])
    cache.reserve([1], [5])
    parents = [[-1, 0, 0, 1, 2]]
    nk, nv = (torch.stack([kvclib.quantize_dev(kvc, rnd(5, H * D), kind) for _ in range(L)]) for _ in range(2))
    cache.write([1], [keep], [5], nk, nv, torch.zeros(L, H, 5, device="cuda"))
    nq = rnd(5, H * G, D)
    mask = attn.tree_mask(parents).cuda()
    for layer in range(L):
        t = attn.Tree(kvc, cache, nq, dev([0, 5]), dev([1]), mask=mask, max_nodes=5, layer=layer)
        t.run()
        cache.check()
        kk, vv, bb = cache.read([1], [0], [keep + 5])
        Kd, Vd = R.decode(kk[layer], kind).view(-1, H, D), R.decode(vv[layer], kind).view(-1, H, D)
        see = torch.ones(5, keep + 5, dtype=torch.bool, device="cuda")
        see[:, keep:] = torch.tensor([[bool((int(mask[a, 0]) >> b) & 1) for b in range(5)] for a in range(5)], device="cuda")
        for h in range(H * G):
            o, w = R.attend(nq[:, h], Kd[:, h // G], Vd[:, h // G], bb[layer, h // G], see, D ** -0.5)
            # scores within +-20 and |V| < 8: 2 (20 2^-20 + 2^-21) 8
            assert float((t.out[:, h].double() - o).abs().max()) < 4e-4 and float((t.lse[:, h].double() - w).abs().max()) < 1e-4

    # nodes 0, 2 and 4 were accepted: the cached rows stay where they are, the accepted path follows
    cache.compact([1], [1], dev([[[keep, keep + 2, keep + 4]]]), dev([3]), dev([keep]))
    cache.check()
    assert int(cache.seq_len[1]) == keep + 3
    path, _, _ = cache.read([1], [keep], [3])
    torch.cuda.synchronize()
    assert torch.equal(path, nk[:, [0, 2, 4]])
    shared = cache.page_table[0, :keep // PAGE].tolist()
    assert cache.page_table[1, :keep // PAGE].tolist() == shared and all(int(cache.ref_count[p]) == 2 for p in shared)
    cache.free([0, 1])
    cache.check()
    assert int(cache.ref_count.abs().sum()) == 0 and cache.seq_len.tolist() == [0] * 6


def test_a_whole_step_in_a_graph(kvc):
    """Append a row, attend to it, for a batch: captured once, replayed."""
    gen = torch.Generator().manual_seed(4)
    c = R.Cache([30, 100, 16], H, D, D, R.Q8_0, R.Q8_0, PAGE, spare=40, max_pages=16)
    h = c.handle(kvc)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(3, H * G, D, generator=gen).cuda()
    t = attn.Tree(kvc, h, q, dev([0, 1, 2, 3]), dev([0, 1, 2]))
    seqs, one = pages.ids([0, 1, 2]), pages.ids([1, 1, 1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h.reserve(seqs, one)
        t.run()
    for step in range(40):
        q.copy_(torch.randn(3, H * G, D, generator=gen))
        g.replay()
        h.check()
        if step % 13 == 0:
            out, _ = c.attend(q, [0, 1, 2, 3], [0, 1, 2], lambda i, m, n: torch.ones(m, n, dtype=torch.bool), D ** -0.5)
            assert float((t.out.double() - out).abs().max()) < 4e-4
    assert c.seq_len.tolist()[:3] == [70, 140, 56]


@pytest.mark.parametrize("nodes", [1, 3])
def test_a_decoder_writes_layer_by_layer(kvc, nodes):
    """A row per token, layer by layer: a layer's K and V come from the output of the layer before. In one graph."""
    gen = torch.Generator().manual_seed(6)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    layers, lens = 3, [30, 100, 15]
    c = R.Cache(lens, H, D, D, R.F16, R.F16, PAGE, layers=layers, spare=40, beta=True, max_pages=16)
    h, n = c.handle(kvc), 3 * nodes
    x = torch.randn(n, H * G * D, generator=gen).cuda()
    proj = [[(torch.randn(H * G * D, w, generator=gen) * 0.1).cuda() for w in (H * G * D, H * D, H * D)] for _ in range(layers)]
    mask = attn.tree_mask([list(range(-1, nodes - 1))] * 3).cuda()            # a chain: each node sees those before it
    seqs, first, one = pages.ids([0, 1, 2]), pages.ids(lens), pages.ids([nodes] * 3)
    cu = dev([0, nodes, 2 * nodes, 3 * nodes])
    q = torch.zeros(n, H * G, D, device="cuda")
    trees = [attn.Tree(kvc, h, q, cu, dev([0, 1, 2]), mask=mask, max_nodes=nodes, layer=l) for l in range(layers)]
    zero = torch.zeros(1, H, n, device="cuda")
    kept = []

    def step():
        y = x
        h.reserve(seqs, one)
        for l in range(layers):
            q.copy_((y @ proj[l][0]).view(n, H * G, D))
            rows = [(y @ p).half().view(1, n, H * D) for p in proj[l][1:]]
            kept.append(rows)
            h.write(seqs, first, one, *(r.view(torch.uint8) for r in rows), zero, layer=l)
            y = trees[l].run().flatten(1)
        return y

    for p in proj[0]:
        x @ p                                              # cuBLAS sets itself up outside the capture
    before = [t.clone() for t in (c.K, c.V, c.beta)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    g.replay()
    h.check()
    assert c.seq_len.tolist()[:3] == [m + nodes for m in lens]
    y = x
    for l in range(layers):
        ql = (y @ proj[l][0]).view(n, H * G, D)
        k, v, b = h.read(seqs, first, one, layer=l)
        torch.cuda.synchronize()
        assert torch.equal(k, kept[l][0].view(torch.uint8)) and torch.equal(v, kept[l][1].view(torch.uint8)) and torch.equal(b, zero)

        def see(i, m, rows):
            s = torch.ones(m, rows, dtype=torch.bool)
            s[:, rows - m:] = torch.tril(torch.ones(m, m, dtype=torch.bool))
            return s
        out, _ = c.attend(ql, cu.tolist(), [0, 1, 2], see, D ** -0.5, l)
        # scores within +-60 and |V| < 16, as above: 2 (60 2^-20 + 2^-21) 16
        assert float((trees[l].out.double() - out).abs().max()) < 2e-3
        y = trees[l].out.flatten(1)
    # nothing else was written: rows of the other tokens and layers are as before
    new = torch.cat([c.rows(s)[m:] for s, m in enumerate(lens)])
    old = torch.ones(c.K.shape[1], dtype=torch.bool, device="cuda")
    old[new] = False
    assert torch.equal(c.K[:, old], before[0][:, old]) and torch.equal(c.V[:, old], before[1][:, old])
    for bad in (-1, layers):
        with pytest.raises(ValueError):
            h.write(seqs, first, one, layer=bad)
        with pytest.raises(ValueError):
            h.read(seqs, first, one, layer=bad)
    with pytest.raises(ValueError):
        h.write(seqs, first, one, torch.zeros(layers, n, c.K.shape[2], dtype=torch.uint8, device="cuda"), layer=0)


def test_launches_are_counted(kvc):
    c = R.Cache([30], H, D, D, R.Q8_0, R.Q8_0, PAGE)
    h = c.handle(kvc)
    at = kvc["_lib"].kvc_launch_count()
    h.free([1])
    assert kvc["_lib"].kvc_launch_count() > at

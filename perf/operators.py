"""Cases of the library's serving operators, their plain forms and their 64-bit definitions.

  prompt   attention over whole prompts: packed sequences, grouped heads, causal from the end
  tree     attention of drafted tokens (or of one token) over a paged, stored-type cache with beta
  copy     copies of whole pages of a cache
  fork     a sequence that shares another one's pages
  compact  a sequence packed down to its kept rows, with refitted values where they are given

Where `own` is true run() makes the library's calls (kvc_b200.attn, kvc_b200.pages); else it
computes the same in elementary torch operations.
"""
import math
import os
import sys

import torch

own = False

F32, F16, Q4_0, Q4_1, Q8_0 = 0, 1, 2, 3, 8          # the library's KV_TYPE_* values
BLOCK_BYTES = {Q8_0: 34, Q4_0: 18, Q4_1: 20}
NAMES = {"f32": F32, "f16": F16, "q4_0": Q4_0, "q4_1": Q4_1, "q8_0": Q8_0}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(v) for v in values)


def listed():
    return [
        # a chat turn's first tokens on a small model: launch latency
        dict(name="prompt_short", op="prompt", new="33", past="0", hkv=4, group=2, d=64),
        # prompts that arrived together, packed without padding, lengths from one token up
        dict(name="prompt_packed", op="prompt", new="1,700,129,64,2047,333,1200,5,513,90", past="0,0,0,0,0,0,0,0,0,0",
             hkv=8, group=4, d=128),
        # the next chunk of two long prompts: the queries are the last rows of the keys
        dict(name="prompt_chunk", op="prompt", new="512,300", past="7000,3333", hkv=8, group=4, d=128),
        # one long document
        dict(name="prompt_long", op="prompt", new="8192", past="0", hkv=8, group=4, d=128),
        # one token of one conversation: launch latency
        dict(name="decode_one", op="tree", rows="1000", nodes="1", hkv=8, group=4, dk=128, dv=128, kt="f16", vt="f16",
             page=16, beta=False, q="f16"),
        # a token for each of 8 sequences over compacted caches (20,000 rows kept of 100,000), beta fitted
        dict(name="decode_compacted", op="tree", rows=_text([20000] * 8), nodes=_text([1] * 8), hkv=8, group=4, dk=128,
             dv=128, kt="q8_0", vt="q8_0", page=64, beta=True, q="f32"),
        # a token for each of a batch of ragged lengths, one of them the whole long cache
        dict(name="decode_ragged", op="tree", rows="100000,17,4096,60001,333,25000,9,1", nodes="1,1,1,1,1,1,1,1", hkv=8,
             group=4, dk=128, dv=128, kt="q8_0", vt="q8_0", page=32, beta=False, q="f16"),
        # drafted trees of a batch, verified in one pass
        dict(name="tree_batch", op="tree", rows="8000,5000,12345,777", nodes="60,31,16,44", hkv=8, group=4, dk=128, dv=128,
             kt="f16", vt="f16", page=16, beta=False, q="f16"),
        # one drafted tree over a 4-bit compacted cache, in the queries' own 32 bits
        dict(name="tree_q4", op="tree", rows="30000", nodes="25", hkv=4, group=8, dk=64, dv=64, kt="q4_0", vt="q4_1",
             page=24, beta=True, q="f32"),
        # pages copied out of the way of writers, every layer
        dict(name="copy_pages", op="copy", count=400, layers=12, hkv=8, d=128, kt="q8_0", vt="q8_0", page=16),
        # four continuations of one conversation
        dict(name="fork_beams", op="fork", rows="5003", to=4, layers=12, hkv=8, d=128, kt="f16", vt="f16", page=64),
        # a long sequence cut to the fifth that compaction kept in each layer, with its refitted values
        dict(name="compact_kept", op="compact", rows="32768", base="64", keep="6540", layers=12, hkv=8, d=128, kt="q8_0",
             vt="q8_0", page=64, refit=True, per_layer=True),
    ]


def draw(rng):
    while True:
        case = _drawn(rng)
        w = work(case)
        if case["op"] == "prompt":
            new, past = _ints(case["new"]), _ints(case["past"])
            scores = len(new) * max(new) * max(a + b for a, b in zip(new, past)) * case["hkv"] * case["group"]
            if scores <= 1.5e9:
                return case
        elif case["op"] == "tree":
            rows, nodes = _ints(case["rows"]), _ints(case["nodes"])
            scores = len(rows) * max(nodes) * max(rows) * case["hkv"] * case["group"]
            if scores <= 1e8 and w["bytes"] <= 3.5e8:
                return case
        elif w["bytes"] <= 3e8 and (case["op"] != "compact" or sum(_ints(case["rows"])) * case["layers"] * case["hkv"] <= 3.2e6):
            return case


def _drawn(rng):
    def logu(a, b):
        return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 1)))))))

    op = rng.choice(["prompt", "prompt", "tree", "tree", "tree", "copy", "fork", "compact"])
    hkv = rng.choice([1, 2, 3, 4, 8])
    if op == "prompt":
        n = logu(1, 12)
        new = [logu(1, 4000) for _ in range(n)]
        past = [rng.choice([0, 0, logu(1, 4000)]) for _ in range(n)]
        return dict(op="prompt", new=_text(new), past=_text(past), hkv=hkv, group=rng.choice([1, 2, 3, 4]),
                    d=rng.choice([64, 128, 128, 72, 96, 40]))
    page = rng.choice([16, 32, 64, 1, 7, 24, 128, logu(1, 200)])
    kinds = ["f16", "q8_0", "q8_0", "q4_0", "q4_1", "f32"]
    if op == "tree":
        n = logu(1, 12)
        rows = [logu(1, 100000 // n) for _ in range(n)]
        nodes = [rng.choice([1, logu(1, 64)]) for _ in range(n)] if rng.random() < 0.6 else [1] * n
        dk = rng.choice([64, 128, 128, 256, 96])
        return dict(op="tree", rows=_text(rows), nodes=_text(nodes), hkv=hkv, group=rng.choice([1, 2, 4, 7, 8]), dk=dk,
                    dv=rng.choice([dk, dk, dk, 64, 128]), kt=rng.choice(kinds), vt=rng.choice(kinds), page=page,
                    beta=rng.random() < 0.5, q=rng.choice(["f16", "f32"]))
    base = dict(layers=logu(1, 12), hkv=hkv, d=rng.choice([64, 128, 96]), kt=rng.choice(kinds), vt=rng.choice(kinds), page=page)
    if op == "copy":
        return dict(op="copy", count=logu(1, 400), **base)
    if op == "fork":
        return dict(op="fork", rows=_text([logu(1, 6000) for _ in range(logu(1, 3))]), to=rng.choice([1, 2, 3, 4]), **base)
    n = logu(1, 6)
    rows = [logu(1, 32768 // n) for _ in range(n)]
    at = [rng.randint(0, r) for r in rows]
    keep = [rng.randint(0, r - b) for r, b in zip(rows, at)]
    return dict(op="compact", rows=_text(rows), base=_text(at), keep=_text(keep), refit=rng.random() < 0.5,
                per_layer=rng.random() < 0.5, **base)


# ---------------------------------------------------------------------------------------------
# stored rows
# ---------------------------------------------------------------------------------------------
def _row_bytes(kind, n):
    return n * 4 if kind == F32 else n * 2 if kind == F16 else n // 32 * BLOCK_BYTES[kind]


def _encode(x, kind):
    """f32 [rows, n] -> the stored bytes, uint8 [rows, row bytes]."""
    rows, n = x.shape
    if kind in (F32, F16):
        return (x if kind == F32 else x.half()).contiguous().view(torch.uint8).view(rows, -1)
    b = x.view(rows, n // 32, 32)
    if kind == Q4_1:
        lo, hi = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
        d, m = ((hi - lo) / 15).half(), lo.half()
        q = ((b - lo) / (hi - lo).clamp_min(1e-20) * 15).round().clamp(0, 15).to(torch.uint8)
        head = torch.cat([d, m], -1).view(torch.uint8)
    else:
        top = 127 if kind == Q8_0 else 7
        a = b.abs().amax(-1, keepdim=True)
        q = (b / a.clamp_min(1e-20) * top).round()
        head = (a / top).half().view(torch.uint8)
        if kind == Q8_0:
            return torch.cat([head, q.to(torch.int8).view(torch.uint8)], -1).view(rows, -1)
        q = (q + 8).clamp(0, 15).to(torch.uint8)
    return torch.cat([head, q[..., 0::2] | (q[..., 1::2] << 4)], -1).view(rows, -1)


def _decode(rows, kind, n):
    """Stored bytes uint8 [..., row bytes] -> the values they stand for, f32 [..., n]."""
    if kind == F32:
        return rows.contiguous().view(torch.float32)
    if kind == F16:
        return rows.contiguous().view(torch.float16).float()
    b = rows.reshape(*rows.shape[:-1], n // 32, BLOCK_BYTES[kind])
    d = b[..., :2].contiguous().view(torch.float16).float()
    if kind == Q8_0:
        return (b[..., 2:].contiguous().view(torch.int8).float() * d).view(*rows.shape[:-1], n)
    q = b[..., 2 if kind == Q4_0 else 4:]
    q = torch.stack([q & 15, q >> 4], -1).flatten(-2).float()
    q = (q - 8) * d if kind == Q4_0 else q * d + b[..., 2:4].contiguous().view(torch.float16).float()
    return q.view(*rows.shape[:-1], n)


def _keys(rows, hkv, d, g, dev):
    """Keys as the benchmark's caches have them: a rank-32 part and noise."""
    u = torch.randn(rows, 32, generator=g, device=dev)
    w = torch.randn(32, hkv * d, generator=g, device=dev)
    return (u @ w) / math.sqrt(32.0) + 0.05 * torch.randn(rows, hkv * d, generator=g, device=dev)


# ---------------------------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------------------------
def _package():
    at = os.path.join(os.getcwd(), "kv-compact_b200", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    from kvc_b200 import attn, lib, pages
    return lib.load(), attn, pages


def _cache(g, dev, layers, lens, hkv, dk, dv, kt, vt, page, spare, slots, beta):
    """A pool whose pages are handed out in a shuffled order, as a server's are after a while."""
    need = [-(-r // page) for r in lens]
    n_pages = sum(need) + spare
    width = max(need) + 2
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((slots, width), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    ref = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    ref[order[:at].long()] = 1
    seq_len = torch.zeros(slots, dtype=torch.int32, device=dev)
    seq_len[:len(lens)] = torch.tensor(lens, dtype=torch.int32, device=dev)
    total = n_pages * page
    K = torch.empty(layers, total, _row_bytes(kt, hkv * dk), dtype=torch.uint8, device=dev)
    V = torch.empty(layers, total, _row_bytes(vt, hkv * dv), dtype=torch.uint8, device=dev)
    for l in range(layers):
        K[l] = _encode(_keys(total, hkv, dk, g, dev), kt)
        V[l] = _encode(torch.randn(total, hkv * dv, generator=g, device=dev), vt)
    b = None
    if beta:
        b = 0.7 * torch.randn(layers, n_pages, hkv, page, generator=g, device=dev)
    return dict(K=K, V=V, beta=b, table=table, seq_len=seq_len, ref=ref, status=torch.zeros(1, dtype=torch.int32, device=dev),
                page=page, hkv=hkv, dk=dk, dv=dv, kt=kt, vt=vt)


def _handle(pages, fns, c):
    return pages.PageCache(fns, c["K"], c["V"], c["table"], c["seq_len"], c["ref"], c["status"], c["page"], c["hkv"],
                           c["dk"], c["dv"], c["kt"], c["vt"], beta=c["beta"])


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    s = dict(op=op)
    if op == "prompt":
        new, past = _ints(case["new"]), _ints(case["past"])
        nk = [a + b for a, b in zip(new, past)]
        hkv, hq, d = case["hkv"], case["hkv"] * case["group"], case["d"]
        cu = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device=dev)  # noqa: E731
        s.update(q=torch.randn(sum(new), hq, d, generator=g, device=dev).half(),
                 k=_keys(sum(nk), hkv, d, g, dev).view(-1, hkv, d).half(),
                 v=torch.randn(sum(nk), hkv, d, generator=g, device=dev).half(), cu_q=cu(new), cu_k=cu(nk),
                 max_q=max(new), max_k=max(nk), scale=d ** -0.5)
        if own:
            fns, attn, _ = _package()
            s["call"] = attn.Prompt(fns, s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], scale=s["scale"], causal=True)
        return s
    if op == "tree":
        past, nodes = _ints(case["rows"]), _ints(case["nodes"])
        n, hkv, hq = len(past), case["hkv"], case["hkv"] * case["group"]
        lens = [p + m for p, m in zip(past, nodes)]
        c = _cache(g, dev, 1, lens, hkv, case["dk"], case["dv"], NAMES[case["kt"]], NAMES[case["vt"]], case["page"], 3, n + 1,
                   case["beta"])
        most, total = max(nodes), sum(nodes)
        words = -(-most // 32)
        # drafted trees: each node hangs under an earlier one; a node sees its ancestors and itself
        vis = torch.zeros(total, words * 32, dtype=torch.bool)
        cg = torch.Generator().manual_seed(seed)
        at = 0
        for m in nodes:
            for i in range(m):
                if i:
                    p = int(torch.randint(max(0, i - 6), i, (1,), generator=cg))
                    vis[at + i] = vis[at + p]
                vis[at + i, i] = True
            at += m
        bit = (vis.view(total, words, 32).long() << torch.arange(32)).sum(-1)
        mask = torch.where(bit >= 2 ** 31, bit - 2 ** 32, bit).to(torch.int32).to(dev)
        cu = torch.tensor([sum(nodes[:i]) for i in range(n + 1)], dtype=torch.int32, device=dev)
        seqs = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=dev) if n > 1 and min(nodes) == most else torch.arange(
            n, dtype=torch.int32, device=dev)
        qt = torch.float16 if case["q"] == "f16" else torch.float32
        s.update(cache=c, q=torch.randn(total, hq, case["dk"], generator=g, device=dev).to(qt), cu=cu, seqs=seqs, mask=mask,
                 most=most, rows=max(lens), scale=case["dk"] ** -0.5)
        if own:
            fns, attn, pages = _package()
            s["call"] = attn.Tree(fns, _handle(pages, fns, c), s["q"], cu, seqs, mask=mask, max_nodes=most, scale=s["scale"])
        return s
    kt, vt, L, hkv, d, page = NAMES[case["kt"]], NAMES[case["vt"]], case["layers"], case["hkv"], case["d"], case["page"]
    if op == "copy":
        n = case["count"]
        c = _cache(g, dev, L, [n * page], hkv, d, d, kt, vt, page, n, 2, True)
        s.update(cache=c, src=c["table"][0, :n].contiguous(), dst=(c["ref"] == 0).nonzero()[:, 0].to(torch.int32).contiguous())
    elif op == "fork":
        lens, to = _ints(case["rows"]), case["to"]
        src = [i for i in range(len(lens)) for _ in range(to)]
        dst = [len(lens) + i for i in range(len(src))]
        c = _cache(g, dev, L, lens, hkv, d, d, kt, vt, page, 2 * len(src) + 1, len(lens) + len(src), True)
        s.update(cache=c, src=src, dst=dst, src_d=torch.tensor(src, device=dev), dst_d=torch.tensor(dst, device=dev))
    else:
        lens, base, keep = _ints(case["rows"]), _ints(case["base"]), _ints(case["keep"])
        n, ld = len(lens), max(1, max(keep))
        spare = 2 * sum(-(-(b + k) // page) for b, k in zip(base, keep)) + 1
        c = _cache(g, dev, L, lens, hkv, d, d, kt, vt, page, spare, 2 * n, True)
        lists = L if case["per_layer"] else 1
        idx = torch.zeros(lists, n, ld, dtype=torch.int32, device=dev)
        for l in range(lists):
            for i in range(n):
                pick = torch.randperm(lens[i] - base[i], generator=g, device=dev)[:keep[i]].sort()[0] + base[i]
                idx[l, i, :keep[i]] = pick.to(torch.int32)
        s.update(cache=c, src=list(range(n)), dst=list(range(n, 2 * n)), src_d=torch.arange(n, device=dev),
                 dst_d=torch.arange(n, 2 * n, device=dev), idx=idx, keep_n=torch.tensor(keep, dtype=torch.int32, device=dev),
                 base=torch.tensor(base, dtype=torch.int32, device=dev), v_rows=None, beta_rows=None)
        if case["refit"]:
            s["v_rows"] = _encode(torch.randn(L * n * ld, hkv * d, generator=g, device=dev), vt).view(L, n, ld, -1)
            s["beta_rows"] = torch.randn(L, n, hkv, ld, generator=g, device=dev)
    if own:
        fns, attn, pages = _package()
        s["call"] = _handle(pages, fns, s["cache"])
        if op != "copy":
            s["src"], s["dst"] = pages.ids(s["src"]), pages.ids(s["dst"])
    return s


# ---------------------------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------------------------
def _softmax_product(x, see, V):
    """softmax of the scores x [..., q, k] over the keys that `see` shows, times V [..., k, d]; and its log-sum-exp."""
    x = x.masked_fill(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(x - m)
    l = e.sum(-1, keepdim=True)
    o = (e @ V) / torch.where(l == 0, torch.ones_like(l), l)
    return o, (m + torch.log(l))[..., 0]


def _padded(cu, most, total):
    """Packed rows as [sequences, most]: the index of each, and which are rows."""
    pos = torch.arange(most, device=cu.device)
    at = cu[:-1, None].long() + pos
    return at.clamp(max=max(total - 1, 0)), pos < (cu[1:] - cu[:-1])[:, None]


def _prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    (tq, hq, d), (tk, hkv, _) = q.shape, k.shape
    iq, oq = _padded(s["cu_q"], s["max_q"], tq)
    ik, ok = _padded(s["cu_k"], s["max_k"], tk)
    n, g = iq.shape[0], hq // hkv
    Q = q[iq].float().view(n, s["max_q"], hkv, g, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * s["max_q"], d)
    K = k[ik].float().permute(0, 2, 3, 1)
    V = (v[ik].float() * ok[..., None, None]).permute(0, 2, 1, 3)
    x = ((Q @ K) * s["scale"]).view(n, hkv, g, s["max_q"], s["max_k"])
    nq, nk = (s["cu_q"][1:] - s["cu_q"][:-1]), (s["cu_k"][1:] - s["cu_k"][:-1])
    last = torch.arange(s["max_q"], device=q.device)[None] + (nk - nq)[:, None]
    see = (torch.arange(s["max_k"], device=q.device) <= last[..., None]) & ok[:, None, :]
    o, lse = _softmax_product(x, see[:, None, None], V[:, :, None])
    out = torch.empty(tq, hq, d, dtype=q.dtype, device=q.device)
    out[iq[oq]] = o.permute(0, 3, 1, 2, 4).reshape(n, s["max_q"], hq, d)[oq].to(q.dtype)
    low = torch.empty(tq, hq, dtype=torch.float32, device=q.device)
    low[iq[oq]] = lse.permute(0, 3, 1, 2).reshape(n, s["max_q"], hq)[oq]
    return out, low


def _tree(s):
    c, q = s["cache"], s["q"]
    hkv, dk, dv, page, R, M = c["hkv"], c["dk"], c["dv"], c["page"], s["rows"], s["most"]
    tq, hq, _ = q.shape
    seqs = s["seqs"].long()
    pos = torch.arange(R, device=q.device)
    at = c["table"][seqs][:, pos // page].clamp(min=0).long()
    ln = c["seq_len"][seqs]
    there = pos < ln[:, None]
    rows = at * page + pos % page
    n, g = rows.shape[0], hq // hkv
    K = _decode(c["K"][0][rows], c["kt"], hkv * dk).view(n, R, hkv, dk).permute(0, 2, 3, 1)
    V = (_decode(c["V"][0][rows], c["vt"], hkv * dv).view(n, R, hkv, dv) * there[..., None, None]).permute(0, 2, 1, 3)
    iq, oq = _padded(s["cu"], M, tq)
    Q = q[iq].float().view(n, M, hkv, g, dk).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * M, dk)
    x = ((Q @ K) * s["scale"]).view(n, hkv, g, M, R)
    if c["beta"] is not None:
        x = x + c["beta"][0][at, :, pos % page].permute(0, 2, 1)[:, :, None, None, :]
    cnt = (s["cu"][1:] - s["cu"][:-1])
    j = pos[None] - (ln - cnt)[:, None]                       # the drafted row's number, negative for cached rows
    word = s["mask"][iq].gather(2, (j.clamp(min=0) // 32).clamp(max=s["mask"].shape[1] - 1)[:, None, :].expand(n, M, R).long())
    see = ((j < 0)[:, None, :] | (((word >> (j.clamp(min=0) % 32)[:, None, :]) & 1) != 0)) & there[:, None, :]
    o, lse = _softmax_product(x, see[:, None, None], V[:, :, None])
    out = torch.empty(tq, hq, dv, dtype=q.dtype, device=q.device)
    out[iq[oq]] = o.permute(0, 3, 1, 2, 4).reshape(n, M, hq, dv)[oq].to(q.dtype)
    low = torch.empty(tq, hq, dtype=torch.float32, device=q.device)
    low[iq[oq]] = lse.permute(0, 3, 1, 2).reshape(n, M, hq)[oq]
    return out, low


def _cache_out(c):
    return dict(K=c["K"], V=c["V"], beta=c["beta"], table=c["table"], seq_len=c["seq_len"], ref=c["ref"], status=c["status"])


def _copy(s):
    c = s["cache"]
    at = lambda p: (p.long()[:, None] * c["page"] + torch.arange(c["page"], device=p.device)).flatten()  # noqa: E731
    a, b = at(s["src"]), at(s["dst"])
    c["K"][:, b] = c["K"][:, a]
    c["V"][:, b] = c["V"][:, a]
    c["beta"][:, s["dst"].long()] = c["beta"][:, s["src"].long()]
    return _cache_out(c)


def _new_pages(c, src, dst, whole, need, length):
    """The table rows of dst: the first `whole` pages of src shared, then `need` of the lowest free pages; the pages that
    dst had are given back. All counts are per sequence."""
    col = torch.arange(c["table"].shape[1], device=src.device)
    free = (c["ref"] != 0).to(torch.uint8).argsort(stable=True).to(torch.int32)
    first = torch.cumsum(need, 0) - need
    fresh = free[(first[:, None] + (col - whole[:, None])).clamp(0, free.numel() - 1).long()]
    row = torch.where(col < whole[:, None], c["table"][src], torch.where(col < (whole + need)[:, None], fresh, -1))
    old = c["table"][dst]
    n = c["ref"].numel()
    for t, by in ((old, -1), (row, 1)):
        c["ref"] += by * torch.bincount(torch.where(t < 0, n, t).flatten(), minlength=n + 1)[:n].to(torch.int32)
    before = c["table"][src]
    c["table"][dst] = row
    c["seq_len"][dst] = length.to(torch.int32)
    return before, row


def _fork(s):
    c, src, dst, page = s["cache"], s["src_d"], s["dst_d"], s["cache"]["page"]
    length = c["seq_len"][src].long()
    whole, rest = length // page, length % page
    before, row = _new_pages(c, src, dst, whole, (rest > 0).long(), length)
    off = torch.arange(page, device=src.device)
    pick = off < rest[:, None]
    at = whole.clamp(max=row.shape[1] - 1)[:, None]
    a = (before.gather(1, at) * page + off)[pick].long()
    b = (row.gather(1, at) * page + off)[pick].long()
    _move(c, a, b)
    return _cache_out(c)


def _move(c, a, b):
    page = c["page"]
    c["K"][:, b] = c["K"][:, a]
    c["V"][:, b] = c["V"][:, a]
    c["beta"][:, b // page, :, b % page] = c["beta"][:, a // page, :, a % page]


def _compact(s):
    c, src, dst, page = s["cache"], s["src_d"], s["dst_d"], s["cache"]["page"]
    base, keep = s["base"].long(), s["keep_n"].long()
    length = base + keep
    whole = base // page
    before, row = _new_pages(c, src, dst, whole, (length + page - 1) // page - whole, length)
    # the rows of the base's last page that stay
    off = torch.arange(page, device=src.device)
    pick = off < (base % page)[:, None]
    at = whole.clamp(max=row.shape[1] - 1)[:, None]
    _move(c, (before.gather(1, at) * page + off)[pick].long(), (row.gather(1, at) * page + off)[pick].long())
    # the kept rows
    L, ld = c["K"].shape[0], s["idx"].shape[2]
    j = torch.arange(ld, device=src.device)
    pick = (j < keep[:, None]).nonzero()
    i, j = pick[:, 0], pick[:, 1]
    to = base[i] + j
    b = row[i, to // page].long() * page + to % page
    idx = s["idx"].long()[:, i, j]
    a = before[i[None], idx // page].long() * page + idx % page
    if a.shape[0] == 1:
        a = a.expand(L, -1)
    l = torch.arange(L, device=src.device)[:, None]
    c["K"][:, b] = c["K"][l, a]
    c["V"][:, b] = c["V"][l, a] if s["v_rows"] is None else s["v_rows"][:, i, j]
    # (the index arrays lead the result: [L, rows, heads])
    new = c["beta"][l, a // page, :, a % page] if s["beta_rows"] is None else s["beta_rows"][:, i, :, j].transpose(0, 1)
    c["beta"][l, b // page, :, b % page] = new
    return _cache_out(c)


def run(state):
    op = state["op"]
    if own:
        call = state["call"]
        if op in ("prompt", "tree"):
            call.run()
            return call.out, call.lse
        if op == "copy":
            call.copy(state["src"], state["dst"])
        elif op == "fork":
            call.fork(state["src"], state["dst"])
        else:
            call.compact(state["src"], state["dst"], state["idx"], state["keep_n"], state["base"], v_rows=state["v_rows"],
                         beta_rows=state["beta_rows"])
        return _cache_out(state["cache"])
    return {"prompt": _prompt, "tree": _tree, "copy": _copy, "fork": _fork, "compact": _compact}[op](state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    op, hkv = case["op"], case["hkv"]
    if op == "prompt":
        new, past, hq, d = _ints(case["new"]), _ints(case["past"]), hkv * case["group"], case["d"]
        pairs = sum(a * p + a * (a + 1) // 2 for a, p in zip(new, past))
        rows_k = sum(new) + sum(past)
        return {"bytes": 2 * d * (2 * sum(new) * hq + 2 * rows_k * hkv) + 4 * sum(new) * hq, "flops": 4 * d * hq * pairs}
    kt, vt, page = NAMES[case["kt"]], NAMES[case["vt"]], case["page"]
    if op == "tree":
        past, nodes, hq = _ints(case["rows"]), _ints(case["nodes"]), hkv * case["group"]
        rows, size = sum(past) + sum(nodes), 2 if case["q"] == "f16" else 4
        stored = _row_bytes(kt, hkv * case["dk"]) + _row_bytes(vt, hkv * case["dv"]) + (4 * hkv if case["beta"] else 0)
        pairs = sum(m * (p + 1) for p, m in zip(past, nodes))  # a node sees the cache and itself at least
        return {"bytes": rows * stored + sum(nodes) * hq * ((case["dk"] + case["dv"]) * size + 4),
                "flops": 2 * (case["dk"] + case["dv"]) * hq * pairs}
    d, L = case["d"], case["layers"]
    stored = _row_bytes(kt, hkv * d) + _row_bytes(vt, hkv * d) + 4 * hkv
    if op == "copy":
        return {"bytes": 2 * L * case["count"] * page * stored, "flops": 0}
    lens = _ints(case["rows"])
    if op == "fork":
        pages = sum(-(-r // page) for r in lens)
        return {"bytes": case["to"] * (2 * L * sum(r % page for r in lens) * stored + 3 * 4 * pages), "flops": 0}
    base, keep = _ints(case["base"]), _ints(case["keep"])
    rows = sum(b % page + k for b, k in zip(base, keep))
    lists = (L if case["per_layer"] else 1) * sum(keep)
    return {"bytes": 2 * L * rows * stored + 4 * lists + 3 * 4 * sum(-(-(b + k) // page) for b, k in zip(base, keep)),
            "flops": 0}


# ---------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def _stored64(raw, kind):
    """The values of stored rows [r, bytes] by the formats' definitions."""
    if kind == F32:
        return raw.contiguous().view(torch.float32).double()
    if kind == F16:
        return raw.contiguous().view(torch.float16).double()
    size = BLOCK_BYTES[kind]
    raw = raw.reshape(raw.shape[0], -1, size)
    half = lambda a: raw[:, :, a:a + 2].contiguous().view(torch.float16).double()  # noqa: E731
    out = torch.empty(raw.shape[0], raw.shape[1], 32, dtype=torch.float64, device=raw.device)
    if kind == Q8_0:
        code = raw[:, :, 2:].double()
        out[:] = half(0) * torch.where(code > 127, code - 256, code)
    else:
        code = raw[:, :, size - 16:]
        low, high = (code % 16).double(), (code // 16).double()
        for part, x in ((0, low), (1, high)):
            out[:, :, part::2] = half(0) * (x - 8) if kind == Q4_0 else half(0) * x + half(2)
    return out.reshape(raw.shape[0], -1)


def _attend64(q, K, V, bias, see, scale):
    """q [r, d], K [k, d], V [k, dv]; bias [k] or None, see [r, k]."""
    x = torch.einsum("rd,kd->rk", q.double(), K) * scale
    if bias is not None:
        x = x + bias.double()
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    lse = torch.logsumexp(x, 1)
    w = torch.where(see, torch.exp(x - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None]), torch.zeros_like(x))
    return w @ V, lse


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    op = case["op"]
    if op == "prompt":
        out = torch.zeros(*s["q"].shape, dtype=torch.float64, device=s["q"].device)
        lse = torch.zeros(*s["q"].shape[:2], dtype=torch.float64, device=s["q"].device)
        a0 = b0 = 0
        for a, p in zip(_ints(case["new"]), _ints(case["past"])):
            b = a + p
            dev = out.device
            see = torch.arange(b, device=dev)[None, :] <= torch.arange(a, device=dev)[:, None] + p
            for h in range(s["q"].shape[1]):
                kv = h // case["group"]
                out[a0:a0 + a, h], lse[a0:a0 + a, h] = _attend64(s["q"][a0:a0 + a, h], s["k"][b0:b0 + b, kv].double(),
                                                                 s["v"][b0:b0 + b, kv].double(), None, see, s["scale"])
            a0, b0 = a0 + a, b0 + b
        return out, lse
    c = s["cache"]
    page = c["page"]
    if op == "tree":
        q, hkv, g = s["q"], case["hkv"], case["group"]
        dev = q.device
        out = torch.zeros(q.shape[0], q.shape[1], case["dv"], dtype=torch.float64, device=dev)
        lse = torch.zeros(*q.shape[:2], dtype=torch.float64, device=dev)
        cu, table = s["cu"].tolist(), c["table"].tolist()
        for i, slot in enumerate(s["seqs"].tolist()):
            n, m = int(c["seq_len"][slot]), cu[i + 1] - cu[i]
            rows = torch.tensor([table[slot][r // page] * page + r % page for r in range(n)], device=dev)
            K = _stored64(c["K"][0][rows], c["kt"]).view(n, hkv, -1)
            V = _stored64(c["V"][0][rows], c["vt"]).view(n, hkv, -1)
            see = torch.ones(m, n, dtype=torch.bool, device=dev)
            words = s["mask"][cu[i]:cu[i + 1]].cpu().tolist()
            see[:, n - m:] = torch.tensor([[bool((words[a][b // 32] >> (b % 32)) & 1) for b in range(m)] for a in range(m)],
                                          device=dev)
            for h in range(hkv * g):
                bias = None if c["beta"] is None else c["beta"][0, rows // page, h // g, rows % page]
                o, w = _attend64(q[cu[i]:cu[i + 1], h], K[:, h // g], V[:, h // g], bias, see, s["scale"])
                out[cu[i]:cu[i + 1], h], lse[cu[i]:cu[i + 1], h] = o, w
        return out, lse
    # page operations move values: beta is the one floating output
    beta = c["beta"].double().cpu()
    if op == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            beta[:, b] = c["beta"][:, a].double().cpu()
    else:
        ref, table = c["ref"].tolist(), c["table"].tolist()
        free = iter([p for p, r in enumerate(ref) if r == 0])
        old = beta.clone()
        for i, src in enumerate(s["src"]):
            n = int(c["seq_len"][src])
            if op == "fork":
                base, kept, new = n // page * page, list(range(n // page * page, n)), None
                lists = torch.tensor(kept, dtype=torch.long)[None]
            else:
                base, k = int(s["base"][i]), int(s["keep_n"][i])
                lists = s["idx"][:, i, :k].long().cpu()
                head = torch.arange(base // page * page, base).expand(lists.shape[0], -1)
                lists, base, new = torch.cat([head, lists], 1), base // page * page, s["beta_rows"]
            count = lists.shape[1]
            pages = torch.tensor([next(free) for _ in range(-(-count // page))], dtype=torch.long)
            to = torch.arange(count)
            for l in range(beta.shape[0]):
                r = lists[l % lists.shape[0]]
                at = torch.tensor(table[src])[r // page]
                got = old[l, at, :, r % page]
                if new is not None:
                    got[count - k:] = new[l, i, :, :k].double().cpu().t()
                beta[l, pages[to // page], :, to % page] = got
    return dict(K=None, V=None, beta=beta, table=None, seq_len=None, ref=None, status=None)

"""Plain 64-bit forms of the serving operators, and caches to run them on."""
import math

import torch

F32, F16, Q4_0, Q4_1, Q8_0 = 0, 1, 2, 3, 8
BLOCK = {Q8_0: 34, Q4_0: 18, Q4_1: 20}


def row_bytes(kind, n):
    return 4 * n if kind == F32 else 2 * n if kind == F16 else n // 32 * BLOCK[kind]


def encode(x, kind):
    """f32 [rows, n] -> stored bytes (any valid encoding will do: the tests start from the bytes)."""
    rows, n = x.shape
    if kind == F32:
        return x.contiguous().view(torch.uint8).view(rows, -1)
    if kind == F16:
        return x.half().contiguous().view(torch.uint8).view(rows, -1)
    b = x.view(rows, n // 32, 32)
    if kind == Q4_1:
        lo, hi = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
        q = ((b - lo) / (hi - lo).clamp_min(1e-20) * 15).round().clamp(0, 15).to(torch.uint8)
        head = torch.cat([((hi - lo) / 15).half(), lo.half()], -1).view(torch.uint8)
    else:
        top = 127 if kind == Q8_0 else 7
        a = b.abs().amax(-1, keepdim=True)
        q = (b / a.clamp_min(1e-20) * top).round()
        head = (a / top).half().view(torch.uint8)
        if kind == Q8_0:
            return torch.cat([head, q.to(torch.int8).view(torch.uint8)], -1).view(rows, -1)
        q = (q + 8).clamp(0, 15).to(torch.uint8)
    return torch.cat([head, q[..., 0::2] | (q[..., 1::2] << 4)], -1).view(rows, -1)


def decode(raw, kind):
    """Stored bytes [rows, bytes] -> the values they stand for, f64 [rows, n]."""
    raw = raw.contiguous()
    if kind == F32:
        return raw.view(torch.float32).double()
    if kind == F16:
        return raw.view(torch.float16).double()
    b = raw.view(raw.shape[0], raw.shape[1] // BLOCK[kind], BLOCK[kind])
    d = b[..., :2].contiguous().view(torch.float16).double()
    if kind == Q8_0:
        return (b[..., 2:].contiguous().view(torch.int8).double() * d).flatten(1)
    q = b[..., BLOCK[kind] - 16:]
    q = torch.stack([q & 15, q >> 4], -1).flatten(-2).double()
    if kind == Q4_0:
        return ((q - 8) * d).flatten(1)
    return (q * d + b[..., 2:4].contiguous().view(torch.float16).double()).flatten(1)


def attend(q, K, V, bias, see, scale):
    """q [r, d], K [n, d], V [n, dv], bias [n] or None, see [r, n]: output and log-sum-exp by the definition. Keys that a
    row does not see count for nothing, whatever they hold."""
    x = q.double() @ K.t() * scale
    if bias is not None:
        x = x + bias.double()
        see = see & (bias != -math.inf)
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    m = x.amax(1, keepdim=True) if x.shape[1] else x.new_full((x.shape[0], 1), -math.inf)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.where(see, torch.exp(x - m), torch.zeros_like(x))
    l = p.sum(1, keepdim=True)
    o = torch.zeros(q.shape[0], V.shape[1], dtype=torch.float64, device=q.device)
    for r in range(q.shape[0]):                      # only the rows that are seen enter the sum
        at = p[r] != 0
        o[r] = p[r][at] @ V[at]
    o = torch.where(l > 0, o / torch.where(l > 0, l, torch.ones_like(l)), torch.zeros_like(o))
    return o, (m + torch.log(l))[:, 0]


class Cache:
    """A cache whose sequences lie on shuffled pages; slot i has lens[i] rows."""

    def __init__(self, lens, hkv, dk, dv, kt, vt, page, layers=1, spare=4, slots=None, beta=False, seed=0, device="cuda",
                 max_pages=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        slots = slots or len(lens) + 1
        width = max_pages or max(need + [0]) + 2
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        table = torch.full((slots, width), -1, dtype=torch.int32)
        ref = torch.zeros(self.n_pages, dtype=torch.int32)
        at = 0
        for s, k in enumerate(need):
            table[s, :k] = order[at:at + k]
            ref[order[at:at + k].long()] = 1
            at += k
        seq = torch.zeros(slots, dtype=torch.int32)
        seq[:len(lens)] = torch.tensor(lens, dtype=torch.int32)
        rows = self.n_pages * page
        enc = lambda d, kind: torch.stack([encode(torch.randn(rows, hkv * d, generator=g), kind) for _ in range(layers)])  # noqa: E731
        self.K, self.V = enc(dk, kt).to(device), enc(dv, vt).to(device)
        self.beta = torch.randn(layers, self.n_pages, hkv, page, generator=g).to(device) if beta else None
        self.table, self.ref, self.seq_len = table.to(device), ref.to(device), seq.to(device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.page, self.hkv, self.dk, self.dv, self.kt, self.vt, self.layers = page, hkv, dk, dv, kt, vt, layers

    def handle(self, kvc):
        from kvc_b200 import pages
        return pages.PageCache(kvc, self.K, self.V, self.table, self.seq_len, self.ref, self.status, self.page, self.hkv,
                               self.dk, self.dv, self.kt, self.vt, beta=self.beta)

    def rows(self, slot):
        n, t = int(self.seq_len[slot]), self.table[slot].tolist()
        return torch.tensor([t[r // self.page] * self.page + r % self.page for r in range(n)], dtype=torch.long,
                            device=self.K.device)

    def attend(self, q, cu, seqs, see_of, scale, layer=0):
        """The definition for a batch; see_of(entry, nodes, rows) -> bool [nodes, rows]."""
        out = torch.zeros(q.shape[0], q.shape[1], self.dv, dtype=torch.float64, device=q.device)
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
        g = q.shape[1] // self.hkv
        for i, slot in enumerate(seqs):
            a, b = cu[i], cu[i + 1]
            rows = self.rows(slot)
            K = decode(self.K[layer][rows], self.kt).view(-1, self.hkv, self.dk)
            V = decode(self.V[layer][rows], self.vt).view(-1, self.hkv, self.dv)
            see = see_of(i, b - a, len(rows)).to(q.device)
            for h in range(q.shape[1]):
                bias = None if self.beta is None else self.beta[layer, rows // self.page, h // g, rows % self.page]
                out[a:b, h], lse[a:b, h] = attend(q[a:b, h], K[:, h // g], V[:, h // g], bias, see, scale)
        return out, lse

"""Attention over prompts and over paged caches, on torch tensors
(include/kvc-attn.h).

``Prompt`` and ``Tree`` hold the tensors and buffers of one call shape;
``run()`` queues the kernels on the current stream of the tensors' device and
returns the output without waiting. The tensors are read at every run, so a
program refills them in place (or captures the run into a graph). Runs of one
object write its output and workspace: order them, or make an object for each
stream. Its tensors must live until the queued work is done.
"""
import ctypes
from ctypes import Structure, c_float, c_int, c_longlong, c_void_p

from . import abi
from .pages import need, on_device


class PromptDesc(Structure):
    _fields_ = [("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("out", c_void_p), ("lse", c_void_p),
                ("cu_q", c_void_p), ("cu_k", c_void_p), ("type", c_int), ("n_seqs", c_int), ("total_q", c_int),
                ("total_k", c_int), ("n_head", c_int), ("n_head_kv", c_int), ("d_k", c_int), ("d_v", c_int),
                ("causal", c_int), ("scale", c_float), ("q_stride", c_longlong), ("q_head_stride", c_longlong),
                ("k_stride", c_longlong), ("k_head_stride", c_longlong), ("v_stride", c_longlong),
                ("v_head_stride", c_longlong)]


class TreeDesc(Structure):
    _fields_ = [("q", c_void_p), ("out", c_void_p), ("lse", c_void_p), ("cu", c_void_p), ("seqs", c_void_p),
                ("mask", c_void_p), ("q_type", c_int), ("mask_words", c_int), ("n_seqs", c_int), ("total", c_int),
                ("max_nodes", c_int), ("n_head", c_int), ("layer", c_int), ("scale", c_float), ("q_stride", c_longlong)]


def _kind(dtype):
    import torch
    kinds = {torch.float32: abi.KV_TYPE_F32, torch.float16: abi.KV_TYPE_F16}
    if dtype not in kinds:
        raise ValueError(f"{dtype}: float16 or float32 is wanted")
    return kinds[dtype]


def _strided(t, what, like):
    if t.device != like.device or t.dtype != like.dtype or t.dim() != 3:
        raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{what}: the last dimension is not contiguous")
    return t


class Prompt:
    """Causal (or full) attention over packed sequences.

    q [total_q, heads, d_k], k [total_k, kv heads, d_k], v [total_k, kv heads, d_v]: float16 or float32 CUDA tensors, any
    strides with a contiguous last dimension (slices of a fused projection); cu_q, cu_k: int32 [n + 1] cumulative lengths
    (cu_k None: cu_q). out [total_q, heads, d_v] and lse [total_q, heads] are made here unless given (lse=False: none)."""

    def __init__(self, fns, q, k, v, cu_q, cu_k=None, scale=None, causal=True, out=None, lse=None):
        import torch
        if q.device.type != "cuda":
            raise ValueError(f"q: on {q.device}")
        _strided(q, "q", q), _strided(k, "k", q), _strided(v, "v", q)
        cu_k = cu_q if cu_k is None else cu_k
        need(cu_q, "cu_q", (torch.int32,), q.device, (None,))
        need(cu_k, "cu_k", (torch.int32,), q.device, (cu_q.shape[0],))
        (tq, h, dk), (tk, hkv, dk2), (tv, hkv2, dv) = q.shape, k.shape, v.shape
        if dk != dk2 or tk != tv or hkv != hkv2 or hkv == 0 or h % hkv or cu_q.shape[0] < 1:
            raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, cu_q {tuple(cu_q.shape)}")
        self.out = torch.empty(tq, h, dv, dtype=q.dtype, device=q.device) if out is None else need(
            out, "out", (q.dtype,), q.device, (tq, h, dv))
        self.lse = None if lse is False else torch.empty(tq, h, device=q.device) if lse is None else need(
            lse, "lse", (torch.float32,), q.device, (tq, h))
        self.fn, self.index = fns["_lib"].kvc_attn_prompt, q.device.index
        self._keep = (q, k, v, cu_q, cu_k)
        self.desc = PromptDesc(q.data_ptr(), k.data_ptr(), v.data_ptr(), self.out.data_ptr(),
                               self.lse.data_ptr() if self.lse is not None else None, cu_q.data_ptr(), cu_k.data_ptr(),
                               _kind(q.dtype), cu_q.shape[0] - 1, tq, tk, h, hkv, dk, dv, 1 if causal else 0,
                               dk ** -0.5 if scale is None else scale, q.stride(0), q.stride(1), k.stride(0), k.stride(1),
                               v.stride(0), v.stride(1))
        self.ref = ctypes.addressof(self.desc)

    def run(self):
        rc = on_device(self.index, self.fn, self.ref)
        if rc != 0:
            raise RuntimeError(f"kvc_attn_prompt failed: {rc}")
        return self.out


class Tree:
    """Attention of drafted tokens over a pages.PageCache; one token per sequence is a tree of one node.

    q [total, heads, d_k] float16 or float32; cu int32 [n + 1]: entry s has the rows cu[s] .. cu[s+1]-1 of q; seqs int32
    [n]: its sequence, whose last rows are the nodes' own; mask int32 [total, words]: bit j of a node's words shows it the
    row of its entry's node j (None: all); max_nodes: most nodes of an entry (left out: 1 for a row of q per entry and no
    mask, else all rows of q, which always suffices but costs time). out [total, heads, d_v] (of q's type) and lse
    [total, heads] are made here unless given (lse=False: none)."""

    def __init__(self, fns, cache, q, cu, seqs, mask=None, max_nodes=None, scale=None, layer=0, out=None, lse=None):
        import torch
        dev, c = cache.device, cache.desc
        _kind(q.dtype)
        if q.device != dev or q.dim() != 3 or q.shape[2] != c.d_k or q.stride(2) != 1 or q.stride(1) != c.d_k:
            raise ValueError(f"q: {tuple(q.shape)} on {q.device} with strides {q.stride()}")
        n = seqs.shape[0]
        need(seqs, "seqs", (torch.int32,), dev, (None,))
        need(cu, "cu", (torch.int32,), dev, (n + 1,))
        if mask is not None:
            need(mask, "mask", (torch.int32,), dev, (q.shape[0], None))
        total, h = q.shape[0], q.shape[1]
        if max_nodes is None:
            max_nodes = 1 if mask is None and total <= n else total
        self.out = torch.empty(total, h, c.d_v, dtype=q.dtype, device=dev) if out is None else need(
            out, "out", (q.dtype,), dev, (total, h, c.d_v))
        self.lse = None if lse is False else torch.empty(total, h, device=dev) if lse is None else need(
            lse, "lse", (torch.float32,), dev, (total, h))
        # a mask without words shows no node's own row; an empty tensor's null pointer would be no mask at all
        at = None if mask is None else mask.data_ptr() or cu.data_ptr()
        lib = fns["_lib"]
        self.fn, self.index, self.cache = lib.kvc_attn_tree, dev.index, cache
        self._keep = (q, cu, seqs, mask)
        self.desc = TreeDesc(q.data_ptr(), self.out.data_ptr(), self.lse.data_ptr() if self.lse is not None else None,
                             cu.data_ptr(), seqs.data_ptr(), at,
                             _kind(q.dtype), mask.shape[1] if mask is not None else 0, n, total, max_nodes, h, layer,
                             c.d_k ** -0.5 if scale is None else scale, q.stride(0) if total > 1 else h * c.d_k)
        self.ref = ctypes.addressof(self.desc)
        rc = c_int(0)
        with torch.cuda.device(dev):
            size = lib.kvc_attn_tree_workspace(cache.ref, self.ref, ctypes.addressof(rc))
        if rc.value != 0:
            raise RuntimeError(f"kvc_attn_tree_workspace failed: {rc.value}")
        self.workspace = torch.empty(size, dtype=torch.uint8, device=dev)
        self._args = (cache.ref, self.ref, self.workspace.data_ptr() if size else None, size)

    def run(self):
        rc = on_device(self.index, self.fn, *self._args)
        if rc != 0:
            raise RuntimeError(f"kvc_attn_tree failed: {rc}")
        return self.out


def tree_mask(parents, words=None):
    """Visibility words of drafted trees from parent lists, one list per entry: parents[i] is the number of node i's
    parent within its entry, negative for a root. Node i sees its ancestors and itself. Returns int32 [total, words] (CPU)."""
    import torch
    words = words or max(1, -(-max((len(p) for p in parents), default=1) // 32))
    rows = []
    for p in parents:
        seen = []
        for i, up in enumerate(p):
            if up >= i:
                raise ValueError(f"node {i}: parent {up} comes after it")
            seen.append((seen[up] if up >= 0 else 0) | (1 << i))
        rows += seen
    full = 2 ** 32 - 1
    signed = lambda w: w - 2 ** 32 if w >= 2 ** 31 else w  # noqa: E731
    return torch.tensor([[signed((r >> (32 * w)) & full) for w in range(words)] for r in rows],
                        dtype=torch.int32).view(-1, words)

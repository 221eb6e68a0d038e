"""A paged KV cache of stored rows over torch tensors (include/kvc-pages.h).

The cache's memory is the caller's tensors; the methods queue kernels on the
current stream of the cache's device and return without waiting, so they can
be captured into a graph. ``check()`` reads the status word.
"""
import ctypes
from ctypes import Structure, c_int, c_size_t, c_void_p

KINDS = {0: (1, 4), 1: (1, 2), 2: (32, 18), 3: (32, 20), 8: (32, 34)}     # KV_TYPE_* -> values, bytes of a block


class PageCacheDesc(Structure):
    _fields_ = [("n_layers", c_int), ("n_pages", c_int), ("page_size", c_int), ("n_slots", c_int),
                ("max_pages", c_int), ("n_head_kv", c_int), ("d_k", c_int), ("d_v", c_int), ("k_type", c_int),
                ("v_type", c_int), ("k_row_bytes", c_size_t), ("v_row_bytes", c_size_t), ("K", c_void_p),
                ("V", c_void_p), ("beta", c_void_p), ("page_table", c_void_p), ("seq_len", c_void_p),
                ("ref_count", c_void_p), ("status", c_void_p)]


def ids(values):
    """A host list of sequence ids or counts, as the calls take it (built once, passed often)."""
    if isinstance(values, ctypes.Array) and values._type_ is c_int:
        return values
    values = [int(v) for v in values]
    return (c_int * len(values))(*values)


def raw_stream(index):
    """Handle of the current stream of device `index`."""
    import torch
    return torch._C._cuda_getCurrentRawStream(index)


def on_device(index, fn, *args):
    """fn(*args, stream) with device `index` current."""
    import torch
    if torch.cuda.current_device() == index:
        return fn(*args, raw_stream(index))
    with torch.cuda.device(index):
        return fn(*args, raw_stream(index))


def need(t, what, dtypes, device, shape=None):
    """Argument check: a contiguous CUDA tensor of one of `dtypes` on `device`, of `shape` (None entries free)."""
    if t.device != device:
        raise ValueError(f"{what}: on {t.device}, not {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what}: {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: not contiguous")
    if shape is not None and (t.dim() != len(shape) or any(w is not None and w != h for w, h in zip(shape, t.shape))):
        raise ValueError(f"{what}: shape {tuple(t.shape)}, not {shape}")
    return t


def row_bytes(kind, n):
    per, size = KINDS[kind]
    if n % per:
        raise ValueError(f"rows of {n} values are no whole blocks of type {kind}")
    return n // per * size


class PageCache:
    """K, V: uint8 CUDA tensors [n_layers, n_pages*page_size, row bytes]; page_table: int32 [n_slots, max_pages], unused
    entries negative; seq_len: int32 [n_slots]; ref_count: int32 [n_pages]; status: int32 [1]; beta: float32
    [n_layers, n_pages, n_head_kv, page_size] or None. The tensors stay the caller's and are read and written in place."""

    def __init__(self, fns, K, V, page_table, seq_len, ref_count, status, page_size, n_head_kv, d_k, d_v, k_type, v_type,
                 beta=None):
        import torch
        dev = K.device
        if dev.type != "cuda":
            raise ValueError(f"K: on {dev}")
        if k_type not in KINDS or v_type not in KINDS:
            raise ValueError(f"types {k_type}, {v_type}")
        need(ref_count, "ref_count", (torch.int32,), dev, (None,))
        n_pages = ref_count.shape[0]
        rows = n_pages * page_size
        need(K, "K", (torch.uint8,), dev, (None, rows, row_bytes(k_type, n_head_kv * d_k)))
        need(V, "V", (torch.uint8,), dev, (K.shape[0], rows, row_bytes(v_type, n_head_kv * d_v)))
        need(page_table, "page_table", (torch.int32,), dev, (None, None))
        need(seq_len, "seq_len", (torch.int32,), dev, (page_table.shape[0],))
        need(status, "status", (torch.int32,), dev, (1,))
        if beta is not None:
            need(beta, "beta", (torch.float32,), dev, (K.shape[0], n_pages, n_head_kv, page_size))
        self.fns, self.lib, self.device, self.index = fns, fns["_lib"], dev, dev.index
        self.K, self.V, self.beta, self.page_table = K, V, beta, page_table
        self.seq_len, self.ref_count, self.status, self.page_size = seq_len, ref_count, status, page_size
        self.desc = PageCacheDesc(K.shape[0], n_pages, page_size, page_table.shape[0], page_table.shape[1], n_head_kv, d_k,
                                  d_v, k_type, v_type, K.shape[2], V.shape[2], K.data_ptr(), V.data_ptr(),
                                  beta.data_ptr() if beta is not None else None, page_table.data_ptr(),
                                  seq_len.data_ptr(), ref_count.data_ptr(), status.data_ptr())
        self.ref, self._layers = ctypes.addressof(self.desc), {}
        size = self.lib.kvc_pages_workspace(self.ref)
        if size == 0:
            raise ValueError("kvc_pages_workspace: the cache's sizes are outside the limits")
        self.workspace = torch.empty(size, dtype=torch.uint8, device=dev)
        self._ws = (self.workspace.data_ptr(), size)

    @classmethod
    def empty(cls, fns, n_layers, n_pages, page_size, n_slots, max_pages, n_head_kv, d_k, d_v, k_type, v_type,
              device="cuda", beta=False):
        """A cache with tensors of its own, every page free."""
        import torch
        dev = torch.device(device)
        if dev.index is None:
            dev = torch.device(dev.type, torch.cuda.current_device())
        z = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=dev)  # noqa: E731
        rows = n_pages * page_size
        K = torch.zeros(n_layers, rows, row_bytes(k_type, n_head_kv * d_k), dtype=torch.uint8, device=dev)
        V = torch.zeros(n_layers, rows, row_bytes(v_type, n_head_kv * d_v), dtype=torch.uint8, device=dev)
        b = torch.zeros(n_layers, n_pages, n_head_kv, page_size, device=dev) if beta else None
        return cls(fns, K, V, z(n_slots, max_pages) - 1, z(n_slots), z(n_pages), z(1), page_size, n_head_kv, d_k, d_v,
                   k_type, v_type, beta=b)

    def _layer(self, layer):
        """The description of one layer alone (write and read take it, calls that change tables do not)."""
        if not 0 <= layer < self.desc.n_layers:
            raise ValueError(f"layer {layer} of {self.desc.n_layers}")
        if layer not in self._layers:
            d = PageCacheDesc.from_buffer_copy(self.desc)
            d.n_layers, d.K, d.V = 1, self.K[layer].data_ptr(), self.V[layer].data_ptr()
            d.beta = self.beta[layer].data_ptr() if self.beta is not None else None
            self._layers[layer] = d
        return self._layers[layer]

    def _call(self, name, *args, desc=None):
        rc = on_device(self.index, getattr(self.lib, name), ctypes.addressof(desc or self.desc), *args)
        if rc != 0:
            raise RuntimeError(f"{name} failed: {rc}")

    def check(self):
        """Wait for the queued calls and raise if one of them could not be done (-11 no free pages, -13 too many rows for
        the table, -2 a write into a shared page, -12 a kernel's wait at its limit: rows or outputs since the last check mean
        nothing); clears the status."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError(f"page cache: status {code}")

    def reserve(self, seqs, add):
        """Append add[i] rows to sequence seqs[i]."""
        seqs, add = ids(seqs), ids(add)
        if len(seqs) != len(add):
            raise ValueError("seqs and add differ in length")
        self._call("kvc_pages_reserve", seqs, add, len(seqs), *self._ws)

    def _rows(self, name, seqs, first, count, k_rows, v_rows, beta_rows, layer):
        import torch
        seqs, first, count = ids(seqs), ids(first), ids(count)
        if not len(seqs) == len(first) == len(count):
            raise ValueError("seqs, first and count differ in length")
        n, d = sum(count), self.desc if layer is None else self._layer(layer)
        for t, what, kind, shape in ((k_rows, "k_rows", torch.uint8, (d.n_layers, n, d.k_row_bytes)),
                                     (v_rows, "v_rows", torch.uint8, (d.n_layers, n, d.v_row_bytes)),
                                     (beta_rows, "beta_rows", torch.float32, (d.n_layers, d.n_head_kv, n))):
            if t is not None:
                need(t, what, (kind,), self.device, shape)
        at = [t.data_ptr() if t is not None else None for t in (k_rows, v_rows, beta_rows)]
        self._call(name, seqs, first, count, len(seqs), *at, desc=d)

    def write(self, seqs, first, count, k_rows=None, v_rows=None, beta_rows=None, layer=None):
        """Rows first[i] .. first[i]+count[i]-1 of sequence seqs[i] from packed rows: k_rows, v_rows uint8 [n_layers, sum of
        count, row bytes], beta_rows float32 [n_layers, n_head_kv, sum of count]. With a layer given (a decoder has its rows
        only after the layer before), that one's alone: [1, ...]. An array left out is not written: a cache with beta wants it for
        new rows, whose pages hold what was there before."""
        self._rows("kvc_pages_write", seqs, first, count, k_rows, v_rows, beta_rows, layer)

    def read(self, seqs, first, count, layer=None):
        """The packed rows (K, V, beta or None) of the given stretches, of all layers or of one ([1, ...]); rows past a
        sequence's end are zero."""
        import torch
        seqs, first, count = ids(seqs), ids(first), ids(count)
        n, d = sum(count), self.desc if layer is None else self._layer(layer)
        k = torch.zeros(d.n_layers, n, d.k_row_bytes, dtype=torch.uint8, device=self.device)
        v = torch.zeros(d.n_layers, n, d.v_row_bytes, dtype=torch.uint8, device=self.device)
        b = torch.zeros(d.n_layers, d.n_head_kv, n, device=self.device) if self.beta is not None else None
        self._rows("kvc_pages_read", seqs, first, count, k, v, b, layer)
        return k, v, b

    def copy(self, src_pages, dst_pages):
        """Pages src_pages[i] -> dst_pages[i] (int32 CUDA tensors) in every layer."""
        import torch
        need(src_pages, "src_pages", (torch.int32,), self.device, (None,))
        need(dst_pages, "dst_pages", (torch.int32,), self.device, (src_pages.shape[0],))
        self._call("kvc_pages_copy", src_pages.data_ptr(), dst_pages.data_ptr(), src_pages.shape[0])

    def fork(self, src, dst):
        """Sequence dst[i] shares the rows of src[i]."""
        src, dst = ids(src), ids(dst)
        if len(src) != len(dst):
            raise ValueError("src and dst differ in length")
        self._call("kvc_pages_fork", src, dst, len(src), *self._ws)

    def compact(self, src, dst, keep, keep_n, base, v_rows=None, beta_rows=None):
        """Sequence dst[i] becomes the first base[i] rows of src[i] and its rows keep[.., i, :keep_n[i]] (src[i] == dst[i]:
        in place). keep: int32 [1 or n_layers, n, ld]; keep_n, base: int32 [n]; v_rows [n_layers, n, ld, row bytes] and
        beta_rows [n_layers, n, n_head_kv, ld] replace the kept rows' V and beta. All CUDA tensors."""
        import torch
        src, dst = ids(src), ids(dst)
        n, d = len(src), self.desc
        if len(dst) != n:
            raise ValueError("src and dst differ in length")
        need(keep, "keep", (torch.int32,), self.device, (None, n, None))
        lists, ld = keep.shape[0], keep.shape[2]
        if lists not in (1, d.n_layers):
            raise ValueError(f"keep: {lists} lists for {d.n_layers} layers")
        need(keep_n, "keep_n", (torch.int32,), self.device, (n,))
        need(base, "base", (torch.int32,), self.device, (n,))
        if v_rows is not None:
            need(v_rows, "v_rows", (torch.uint8,), self.device, (d.n_layers, n, ld, d.v_row_bytes))
        if beta_rows is not None:
            need(beta_rows, "beta_rows", (torch.float32,), self.device, (d.n_layers, n, d.n_head_kv, ld))
        self._call("kvc_pages_compact", src, dst, n, base.data_ptr(), keep_n.data_ptr(), keep.data_ptr(), ld,
                   n * ld if lists > 1 else 0, v_rows.data_ptr() if v_rows is not None else None,
                   beta_rows.data_ptr() if beta_rows is not None else None, *self._ws)

    def free(self, seqs):
        """Give back the pages of the sequences."""
        seqs = ids(seqs)
        self._call("kvc_pages_free", seqs, len(seqs), *self._ws)

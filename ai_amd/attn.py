"""Attention of one layer through librv12.so: q/k head RMSNorm, RoPE at a
device-side position, K/V into the cache, grouped-query attention.  One token
(rv12_rope_attn: the reference's rope_attn_k,
ramvi/engine/ramvi_engine/kernels/tkernels.py:164-213) or a batch of up to 16
tokens of one sequence, each attending causally (rv12_rope_attn_batch: the
reference's qk_rope_cache_k + attn_k, tkernels.py:82-150), or a whole prompt
block (rv12_prefill_rope_attn: qk_rope_cache_k + att_k of the blocked prefill,
ramvi/engine/ramvi_engine/kernels/prefill.py:100-103,
prefill_kernels.py:29-54).  Many sequences share a cache in pages
(PagedRopeAttn: rv12_paged_append, rv12_paged_attend)."""
import ctypes

import torch

from ._lib import Attn, Paged, check, lib, on
from .wcomp import _ptr, _stream


SPAN = 80  # positions one workgroup covers at most
LONG_SPAN = 256  # one split per kv head covers up to this many (no combine pass)
MAX_SPLITS = 128


def default_splits(n_kv, maxt, kv_bf16=True, head_dim=128):
    """Position splits: one for a context of up to 256 positions (one
    workgroup per kv head, no combine launch; not for float32 caches of
    128-dim heads, whose long-span workgroup would spill registers); else
    each workgroup covers at most 80 positions, and there are at least 256
    workgroups while each keeps >= 16 positions."""
    if maxt <= LONG_SPAN and (kv_bf16 or head_dim <= 64):
        return 1
    need = -(-maxt // SPAN)
    want = min(-(-256 // n_kv), -(-maxt // 16))
    s = max(1, need, want)
    if s > MAX_SPLITS:
        raise ValueError("the attention kernel covers at most 10240 positions")
    return int(s)


class RopeAttn:
    """Launch parameters and workspace for one model's caches."""

    def __init__(self, n_heads, n_kv, head_dim, maxt, kv_dtype, eps, device, splits=None):
        if kv_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("the cache must be float32 or bfloat16")
        bf16 = kv_dtype == torch.bfloat16
        self.a = Attn(n_heads, n_kv, head_dim, maxt, 1 if bf16 else 0,
                      splits or default_splits(n_kv, maxt, bf16, head_dim), float(eps), float(head_dim ** -0.5))
        need = lib().rv12_attn_workspace_bytes(ctypes.byref(self.a))
        self.ws = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
        need = lib().rv12_attn_batch_workspace_bytes(ctypes.byref(self.a), 16)
        self.wsb = torch.empty(max(need, 16), dtype=torch.uint8, device=device)

    def _check(self, qkv, qn, kn, inv, pos, kc, vc, out, T):
        """The tensors' dtypes, layouts, sizes and device: the C ABI sees only
        pointers, so a cache of another dtype or shape than this object's
        would be written out of bounds."""
        a = self.a
        for t in (qkv, qn, kn, inv, out):
            if t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError("qkv, qn, kn, inv and out must be contiguous float32")
        if pos.dtype != torch.int64 or pos.numel() < 1:
            raise ValueError("pos must be int64")
        dev = qkv.device
        if any(t.device != dev for t in (qn, kn, inv, pos, kc, vc, out)):
            raise ValueError("every tensor must be on the device of qkv")
        if qkv.numel() < T * (a.n_heads + 2 * a.n_kv) * a.head_dim or out.numel() < T * a.n_heads * a.head_dim:
            raise ValueError(f"qkv and out need {T} rows")
        if qn.numel() < a.head_dim or kn.numel() < a.head_dim or inv.numel() < a.head_dim // 2:
            raise ValueError("qn, kn need head_dim entries and inv head_dim / 2")
        want = torch.bfloat16 if a.kv_bf16 else torch.float32
        for c in (kc, vc):
            if c.dtype != want or not c.is_contiguous() or tuple(c.shape) != (a.n_kv, a.maxt, a.head_dim):
                raise ValueError(f"kc and vc must be contiguous {want} caches of shape "
                                 f"({a.n_kv}, {a.maxt}, {a.head_dim})")

    def __call__(self, qkv, qn, kn, inv, pos, kc, vc, out):
        self._check(qkv, qn, kn, inv, pos, kc, vc, out, 1)
        p = lambda t: ctypes.c_void_p(t.data_ptr())
        rc = lib().rv12_rope_attn(ctypes.byref(self.a), p(qkv), p(qn), p(kn), p(inv), p(pos), p(kc), p(vc), p(out),
                                  p(self.ws), self.ws.numel(),
                                  ctypes.c_void_p(torch.cuda.current_stream(qkv.device).cuda_stream))
        check(rc, "rope_attn")

    def batch(self, qkv, qn, kn, inv, pos, kc, vc, out, T):
        """T <= 16 tokens at positions pos .. pos + T - 1: rows of qkv in, rows
        of out written; K/V of the T positions into the caches."""
        self._check(qkv, qn, kn, inv, pos, kc, vc, out, int(T))
        p = lambda t: ctypes.c_void_p(t.data_ptr())
        rc = lib().rv12_rope_attn_batch(ctypes.byref(self.a), int(T), p(qkv), p(qn), p(kn), p(inv), p(pos), p(kc),
                                        p(vc), p(out), p(self.wsb), self.wsb.numel(),
                                        ctypes.c_void_p(torch.cuda.current_stream(qkv.device).cuda_stream))
        check(rc, "rope_attn_batch")

    def prefill(self, qkv, qn, kn, inv, pos, kc, vc, out, T):
        """A prompt block of T tokens at positions pos .. pos + T - 1 (pos a
        device int64): rows of qkv in, rows of out written; K/V of the T
        positions into the caches.  The q rows live in a workspace kept for
        the largest T seen."""
        self._check(qkv, qn, kn, inv, pos, kc, vc, out, int(T))
        L = lib()
        need = L.rv12_prefill_attn_workspace_bytes(ctypes.byref(self.a), int(T))
        if need == 0:
            raise ValueError("prefill attention: unsupported block (tokens, context or head size)")
        ws = getattr(self, "wsp", None)
        if ws is None or ws.numel() < need:
            ws = self.wsp = torch.empty(need, dtype=torch.uint8, device=qkv.device)
        p = lambda t: ctypes.c_void_p(t.data_ptr())
        rc = L.rv12_prefill_rope_attn(ctypes.byref(self.a), int(T), p(qkv), p(qn), p(kn), p(inv), p(pos), p(kc),
                                      p(vc), p(out), p(ws), ws.numel(),
                                      ctypes.c_void_p(torch.cuda.current_stream(qkv.device).cuda_stream))
        check(rc, "prefill_rope_attn")


_TOO_MANY = ("paged attention: at most 65536 rows, 2^30 positions in a table row, 2^35 of both multiplied and 2^40 times "
             "n_kv")


class PagedRopeAttn:
    """Attention over a cache of many sequences in pages (rv12_paged_append,
    rv12_paged_attend).  A pass has T token rows; row r is position pos[r] of
    sequence seq[r].  Rows may be of different sequences (one new token each) or
    of one (a chunk of its prompt, speculated tokens), in any order; those of
    one sequence run faster next to each other.  The tensors of a call, all on
    one GPU, contiguous but for the table's rows:

        qkv    float32 [T, (n_heads + 2 n_kv) head_dim], the qkv linear's output
        q, out float32 [T, n_heads head_dim]
        seq    int32 [T], or None: row r is of sequence r
        pos    int64 [T]
        table  int32 [sequences, pages of one], the page ids of each sequence
               (any stride between its rows)
        kc, vc [pages, n_kv, page, head_dim] of kv_dtype

    At most 65536 rows and 2^30 positions in a row of the table; for attend, rows
    times these at most 2^35 (and times n_kv 2^40: split a larger pass's rows).

    A row with seq or pos outside the table (-1 for padding a pass to a fixed
    size) is padding: its q and out are zeros and it writes nothing.  A page id
    outside the cache (-1) is no page: its positions take no part in the
    attention, a key or value for it is dropped.  A row that sees an infinite key
    or value may be NaN.  Rows that name one slot together leave it with either's
    key and value.  seq, pos and table are read on the device, so a call can be
    captured in a HIP graph; every call has a workspace of its own.  The rotation
    angle is formed in 64 bits (RopeAttn's in float32: the two agree to float32
    rounding times the position)."""

    def __init__(self, n_heads, n_kv, head_dim, page, kv_dtype, eps, scale=None):
        if kv_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("the cache must be float32 or bfloat16")
        self.kv_dtype = kv_dtype
        self.n_heads, self.n_kv, self.head_dim, self.page = (int(v) for v in (n_heads, n_kv, head_dim, page))
        self.eps = float(eps)
        self.scale = float(self.head_dim ** -0.5 if scale is None else scale)
        self._page_shape = (self.n_kv, self.page, self.head_dim)
        self._structs = {}  # sizes of the table and the caches -> argument struct
        if lib().rv12_paged_attend_workspace_bytes(self._struct(1, 1, 1, 1), 1) == 0:
            raise ValueError("paged attention: head_dim must be 64 or 128, n_heads 1 to 16 times n_kv, page a power of "
                             "two from 16 to 1024")

    def _struct(self, *sizes):
        """The argument struct of n_seq, max_pages, table_stride, n_pages."""
        a = self._structs.get(sizes)
        if a is None:
            if len(self._structs) >= 256:
                self._structs.clear()
            a = self._structs[sizes] = ctypes.byref(Paged(
                self.n_heads, self.n_kv, self.head_dim, self.page, 1 if self.kv_dtype == torch.bfloat16 else 0, *sizes,
                self.eps, self.scale))
        return a

    def _rows(self, dev, rows, seq, pos, table, kc, vc):
        """The argument struct of a call and its row count; rows: (tensor,
        floats of one row) pairs.  dev: index of the GPU."""
        if dev < 0:
            raise ValueError("the tensors must be on the GPU")
        T = pos.numel()
        if pos.dtype != torch.int64 or pos.dim() != 1 or not pos.is_contiguous() or pos.get_device() != dev:
            raise ValueError("pos must be a contiguous int64 vector on the rows' device")
        if seq is not None and (seq.dtype != torch.int32 or seq.dim() != 1 or seq.numel() != T
                                or not seq.is_contiguous() or seq.get_device() != dev):
            raise ValueError("seq must be a contiguous int32 vector with an entry for every row, on the rows' device")
        for t, n in rows:
            if t.dtype != torch.float32 or t.numel() != T * n or not t.is_contiguous() or t.get_device() != dev:
                raise ValueError(f"qkv, q and out must be contiguous float32 with {T} rows, on one device")
        if table.dtype != torch.int32 or table.dim() != 2 or table.get_device() != dev:
            raise ValueError("table must be int32 [sequences, pages], on the rows' device")
        n_seq, max_pages = table.shape
        stride, one = table.stride()
        if n_seq == 1:
            stride = max_pages
        if n_seq < 1 or max_pages < 1 or (one != 1 and max_pages > 1) or stride < max_pages:
            raise ValueError("the table's rows must be contiguous, not empty and not overlap")
        n_pages = kc.shape[0]
        want, shape = self.kv_dtype, (n_pages,) + self._page_shape
        if (kc.dtype != want or vc.dtype != want or kc.shape != shape or vc.shape != shape or not kc.is_contiguous()
                or not vc.is_contiguous() or kc.get_device() != dev or vc.get_device() != dev):
            raise ValueError(f"kc and vc must be contiguous {want} caches of shape "
                             f"(pages, {self.n_kv}, {self.page}, {self.head_dim})")
        return self._struct(n_seq, max_pages, stride, n_pages), T

    def append(self, qkv, qn, kn, inv, seq, pos, table, kc, vc, q):
        """Head norms and rotation of the rows' q and k: q to q, k and v to
        their pages."""
        dev = qkv.get_device()
        a, T = self._rows(dev, ((qkv, (self.n_heads + 2 * self.n_kv) * self.head_dim), (q, self.n_heads * self.head_dim)),
                          seq, pos, table, kc, vc)
        for t, n in ((qn, self.head_dim), (kn, self.head_dim), (inv, self.head_dim // 2)):
            if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous() or t.get_device() != dev:
                raise ValueError("qn, kn and inv must be contiguous float32 of head_dim, head_dim and head_dim / 2 "
                                 "entries, on the rows' device")
        if T == 0:
            return
        with on(qkv.device):
            check(lib().rv12_paged_append(a, T, _ptr(qkv), _ptr(qn), _ptr(kn), _ptr(inv), _ptr(seq), _ptr(pos),
                                          _ptr(table), _ptr(kc), _ptr(vc), _ptr(q), _stream(qkv.device)), "paged_append")

    def attend(self, q, seq, pos, table, kc, vc, out):
        """The attention of the rows (q as append leaves it) over their
        sequences' positions 0 .. pos, the rows' own among them."""
        n = self.n_heads * self.head_dim
        a, T = self._rows(q.get_device(), ((q, n), (out, n)), seq, pos, table, kc, vc)
        if T == 0:
            return
        L = lib()
        with on(q.device):
            need = L.rv12_paged_attend_workspace_bytes(a, T)
            if need == 0:
                raise ValueError(_TOO_MANY)
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            check(L.rv12_paged_attend(a, T, _ptr(q), _ptr(seq), _ptr(pos), _ptr(table), _ptr(kc), _ptr(vc), _ptr(out),
                                      _ptr(ws), need, _stream(q.device)), "paged_attend")

    def __call__(self, qkv, qn, kn, inv, seq, pos, table, kc, vc, out):
        """append, then attend (nothing is appended where attend would refuse)."""
        n = pos.numel() * table.shape[-1:].numel() * self.page
        if n > 1 << 35 or (n >> 10) * self.n_kv > 1 << 30:
            raise ValueError(_TOO_MANY)
        q = torch.empty_like(out)
        self.append(qkv, qn, kn, inv, seq, pos, table, kc, vc, q)
        self.attend(q, seq, pos, table, kc, vc, out)

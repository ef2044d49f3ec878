"""Low-rank adapters of many requests beside a shared 12-bit projection
(rv12_lora_apply): the frozen linear runs once for all rows (wcomp.gemvc1,
gemvc_tc, prefill.matrix), then every row gets its own request's adapter.

    wcomp.gemvc_tc(x, W, y, 0, T, lnw=ln1)
    adapters.apply(x, y, idx, lnw=ln1)          # y[t] += scale B (A x'[t])
"""
import ctypes

import torch

from ._lib import Lora, check, lib, on
from .wcomp import _ptr, _stream


class Adapters:
    """The adapters of one linear W [N, K], one bank on one GPU.

    A      bf16 [count, R, K], B bf16 [count, N, R] (R up to 128, K a multiple of
           32; a rank that is no multiple of 8 is padded with zeros once, here)
    scale  float32 [count]: alpha / rank of each
    ranks  None (R each), or a sequence of each adapter's rank: what A and B hold
           past it is not used (cleared once, here)"""

    def __init__(self, A, B, scale, ranks=None):
        for t, name in ((A, "A"), (B, "B")):
            if not torch.is_tensor(t) or not t.is_cuda or t.dtype != torch.bfloat16 or t.dim() != 3:
                raise ValueError(f"{name} must be a 3-D bfloat16 tensor on the GPU")
        count, R, K = A.shape
        N = B.shape[1]
        if B.shape[0] != count or B.shape[2] != R or B.device != A.device:
            raise ValueError("A must be [count, R, K] and B [count, N, R], on one device")
        if count < 1 or N < 1 or not 1 <= R <= 128 or K < 32 or K % 32:
            raise ValueError("Adapters: at least one adapter and output row, rank 1 to 128, K a multiple of 32")
        if (not torch.is_tensor(scale) or scale.dtype != torch.float32 or tuple(scale.shape) != (count,)
                or scale.device != A.device):
            raise ValueError("scale must be float32 [count] on the adapters' device")
        self.ranks = None
        if ranks is not None:
            ranks = [int(r) for r in ranks]
            if len(ranks) != count or min(ranks) < 0 or max(ranks) > R:
                raise ValueError("ranks must have an entry from 0 to R for every adapter")
            self.ranks = torch.tensor(ranks, dtype=torch.int32, device=A.device)
            keep = torch.arange(R, device=A.device)[None, :] < self.ranks[:, None]
            A, B = A.masked_fill(~keep[:, :, None], 0), B.masked_fill(~keep[:, None, :], 0)
        if R % 8:
            pad = 8 - R % 8
            A = torch.cat([A, A.new_zeros(count, pad, K)], 1)
            B = torch.cat([B, B.new_zeros(count, N, pad)], 2)
        self.A, self.B, self.scale = A.contiguous(), B.contiguous(), scale.contiguous()
        self.count, self.N, self.K, self.R, self.device = count, N, K, R, A.device
        self._index, self._r = A.get_device(), self.A.shape[1]
        self._a = ctypes.byref(Lora(_ptr(self.A), _ptr(self.B), _ptr(self.scale), _ptr(self.ranks), N, K, self._r, count))

    @classmethod
    def from_pairs(cls, pairs, device="cuda"):
        """From (A [r, K], B [N, r], alpha) of each adapter, ranks as they are; the
        weights rounded to bf16, scale = alpha / r."""
        pairs = list(pairs)
        if not pairs:
            raise ValueError("Adapters: at least one adapter")
        R = max(a.shape[0] for a, _, _ in pairs)
        K, N = pairs[0][0].shape[1], pairs[0][1].shape[0]
        A = torch.zeros(len(pairs), R, K, dtype=torch.bfloat16, device=device)
        B = torch.zeros(len(pairs), N, R, dtype=torch.bfloat16, device=device)
        for i, (a, b, _) in enumerate(pairs):
            if a.shape[1] != K or b.shape != (N, a.shape[0]) or a.shape[0] < 1:
                raise ValueError("every adapter must have A [r, K] and B [N, r] of one N and K")
            A[i, :a.shape[0]], B[i, :, :a.shape[0]] = a.to(A), b.to(B)
        scale = torch.tensor([float(s) / a.shape[0] for a, _, s in pairs], dtype=torch.float32, device=device)
        return cls(A, B, scale, [a.shape[0] for a, _, _ in pairs])

    def apply(self, x, y, idx, mode=0, lnw=None, eps=1e-6, out=None):
        """out[t] = y[t] + scale B (A x'[t]) of adapter idx[t], for the T <= 65536
        rows of x; out None: into y; a given out is y or does not overlap it.  mode,
        lnw and eps give x' as the shared linear's call has it (wcomp.gemvc1): modes
        0 and 1 x' = x (float32 [T, K]), with lnw (bf16 [K]) its RMSNorm; mode 2
        x' = silu(x[:, :K]) * x[:, K:].  idx: int32 [T], outside [0, count) (-1) no
        adapter: out[t] = y[t].  y and out: float32 [T, N], rows contiguous, any
        stride between them (a slice of a fused projection's output).  Can be
        captured in a HIP graph."""
        dev, K, N = self._index, self.K, self.N
        if mode not in (0, 1, 2):
            raise ValueError("apply: mode must be 0, 1 or 2")
        if (not torch.is_tensor(idx) or idx.dtype != torch.int32 or idx.dim() != 1 or not idx.is_contiguous()
                or idx.get_device() != dev):
            raise ValueError("apply: idx must be a contiguous int32 vector on the adapters' device")
        T = idx.numel()
        width = 2 * K if mode == 2 else K
        if x.dtype != torch.float32 or x.shape != (T, width) or not x.is_contiguous() or x.get_device() != dev:
            raise ValueError(f"apply: x must be contiguous float32 [{T}, {width}] on the adapters' device")
        ys = self._stride(y, T)
        out, os = (y, ys) if out is None else (out, self._stride(out, T))
        if lnw is not None:
            if mode == 2:
                raise ValueError("apply: the RMSNorm goes with modes 0 and 1")
            if lnw.dtype != torch.bfloat16 or lnw.shape != (K,) or not lnw.is_contiguous() or lnw.get_device() != dev:
                raise ValueError("apply: lnw must be a contiguous bf16 vector of K entries on the adapters' device")
        if T == 0:
            return out
        L = lib()
        with on(self.device):
            need = L.rv12_lora_workspace_bytes(self._r, K, T)
            if need == 0:
                raise ValueError("apply: at most 65536 rows")
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            check(L.rv12_lora_apply(self._a, _ptr(x), _ptr(y), ys, _ptr(out), os, _ptr(idx), T, _ptr(lnw), float(eps), mode,
                                    _ptr(ws), need, _stream(self.device)), "lora_apply")
        return out

    def _stride(self, t, T):
        """Stride between the rows of y or out."""
        if t.dtype != torch.float32 or t.shape != (T, self.N) or t.get_device() != self._index:
            raise ValueError(f"apply: y and out must be float32 [{T}, {self.N}] on the adapters' device")
        stride, one = t.stride()
        if (one != 1 and self.N > 1) or (T > 1 and stride < self.N):
            raise ValueError("apply: the rows of y and out must be contiguous and not overlap")
        return stride if T > 1 else self.N

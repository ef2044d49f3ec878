"""Rules on logits before the pick, for many requests at once (rv12_logits_adjust):
penalties for repeated tokens, biases, grammar masks, and the greedy pick of
what they leave.  Head.pick applies them between the head and the pick."""
import ctypes

import torch

from ._lib import Rules, check, lib, on
from .wcomp import _ptr, _stream


def _rows(t, name, dtype, T, n, dev):
    """Stride between the rows of t: [T, n] (n None: any), each contiguous."""
    if not torch.is_tensor(t) or t.dtype != dtype or t.dim() != 2 or t.get_device() != dev:
        raise ValueError(f"adjust: {name} must be a 2-D {dtype} tensor on the device of x")
    rows, m = t.shape
    stride, one = t.stride()
    if rows != T or (n is not None and m != n) or (one != 1 and m > 1):
        raise ValueError(f"adjust: {name} must have {T} rows" + ("" if n is None else f" of {n}") + ", contiguous each")
    return stride if T > 1 else m


def _vector(t, name, dtype, T, dev):
    if (not torch.is_tensor(t) or t.dtype != dtype or t.dim() != 1 or t.numel() != T or not t.is_contiguous()
            or t.get_device() != dev):
        raise ValueError(f"adjust: {name} must be a contiguous {dtype} vector of {T} entries on the device of x")


def adjust(x, out=None, tokens=None, length=None, prompt=None, penalties=None, bias_ids=None, bias=None, mask=None,
           ids=None):
    """The rules on the logits x (float32 [T, V]) into out (None: in place; a given
    out is x or does not overlap it), which is returned.  Per row and id n, in
    float32 and this order:

        n among the row's tokens:            l = l / repetition if l > 0 else l * repetition
        n generated c > 0 times:             l -= frequency * c + presence
        n in bias_ids:                       l += its bias
        n not allowed:                       l = -inf, whatever it was

    tokens     int64 [T, L] with length (int32 [T]): row r's tokens are the first
               length[r]; prompt (int32 [T]): the first prompt[r] of them are the
               prompt, the others generated (None: all of them generated)
    penalties  float32 [T, 3]: repetition, frequency, presence (with tokens)
    bias_ids   int64 [T, M], bias float32 [T, M]; of several entries of one id the
               last counts
    mask       int32 [T, ceil(V / 32)]: bit n % 32 of word n // 32 set where id n
               is allowed
    ids        int64 [T], written: the id of the largest allowed logit, the
               smallest on ties, NaN counting as the largest, -1 where the mask
               allows none

    T is at most 65535, V below 2^31 - 65536, L below 2^20 (whatever the lengths) and
    M below 2^11.  Ids outside [0, V), such as the -1 of an unused entry, are passed
    over.  All on one GPU; nothing is read back, so a call can be captured in a HIP
    graph."""
    if not torch.is_tensor(x) or not x.is_cuda:
        raise ValueError("adjust: x must be a tensor on the GPU")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError("adjust: x must be [T, V]")
    T, V = x.shape
    dev = x.get_device()
    xs = _rows(x, "x", torch.float32, T, V, dev)
    out, ys = (x, xs) if out is None else (out, _rows(out, "out", torch.float32, T, V, dev))
    if T > 1 and ys < V:
        raise ValueError("adjust: the rows of out must not overlap")
    n_tokens = n_bias = ts = bs = ms = 0
    if tokens is not None:
        ts = _rows(tokens, "tokens", torch.int64, T, None, dev)
        n_tokens = tokens.shape[1]
        _vector(length, "length", torch.int32, T, dev)
        if prompt is not None:
            _vector(prompt, "prompt", torch.int32, T, dev)
        if (not torch.is_tensor(penalties) or penalties.dtype != torch.float32 or penalties.shape != (T, 3)
                or not penalties.is_contiguous() or penalties.get_device() != dev):
            raise ValueError(f"adjust: penalties must be contiguous float32 [{T}, 3] on the device of x")
    elif length is not None or prompt is not None or penalties is not None:
        raise ValueError("adjust: length, prompt and penalties go with tokens")
    if bias_ids is not None or bias is not None:
        bs = _rows(bias_ids, "bias_ids", torch.int64, T, None, dev)
        n_bias = bias_ids.shape[1]
        if _rows(bias, "bias", torch.float32, T, n_bias, dev) != bs:
            raise ValueError("adjust: bias_ids and bias must have one layout")
    if mask is not None:
        ms = _rows(mask, "mask", torch.int32, T, -(-V // 32), dev)
    if ids is not None:
        _vector(ids, "ids", torch.int64, T, dev)
    if T == 0:
        return out
    if not n_tokens:
        tokens = length = prompt = penalties = None
    if not n_bias:
        bias_ids = bias = None
    a = Rules(_ptr(tokens), _ptr(length), _ptr(prompt), _ptr(penalties), _ptr(bias_ids), _ptr(bias), _ptr(mask), ts, bs,
              ms, n_tokens, n_bias)
    L = lib()
    device = x.device
    with on(device):
        need, ws = 0, None
        if ids is not None:
            need = L.rv12_logits_workspace_bytes(V, T)
            ws = torch.empty(need, dtype=torch.uint8, device=device)
        check(L.rv12_logits_adjust(ctypes.byref(a), _ptr(x), xs, _ptr(out), ys, V, T, _ptr(ids), _ptr(ws), need,
                                   _stream(device)), "adjust")
    return out

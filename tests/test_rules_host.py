"""The refusals of the logit rules and the adapters that need no GPU: the C ABI's
argument checks, all before any device work."""
import ctypes

import pytest
import torch

P = 4096  # never dereferenced: the checks come first


def test_rules_abi():
    from ai_amd import _lib
    L = _lib.lib()
    call = lambda r, x=P, xs=100, y=P, ys=100, v=100, t=2, ids=P, ws=P, n=1 << 20: L.rv12_logits_adjust(
        None if r is None else ctypes.byref(r), x, xs, y, ys, v, t, ids, ws, n, None)
    ok = _lib.Rules()
    assert L.rv12_logits_workspace_bytes(100, 2) > 0
    assert call(None) == _lib.RV12_E_NULL and call(ok, x=None) == _lib.RV12_E_NULL and call(ok, y=None) == _lib.RV12_E_NULL
    for kw in (dict(t=0), dict(t=65536), dict(v=0), dict(v=(1 << 31) - 65536), dict(ys=99), dict(xs=-1)):
        assert call(ok, **kw) == _lib.RV12_E_RULES, kw
    assert call(ok, ws=None) == _lib.RV12_E_WORKSPACE and call(ok, n=3) == _lib.RV12_E_WORKSPACE
    for kw in (dict(ids=P + 4), dict(x=P + 2), dict(y=P + 1), dict(ws=P + 4)):
        assert call(ok, **kw) == _lib.RV12_E_ALIGN, kw
    for f in ("max_tokens", "n_bias", "tokens_stride", "bias_stride", "mask_stride"):
        r = _lib.Rules()
        setattr(r, f, -1)
        assert call(r) == _lib.RV12_E_RULES, f
    for kw in (dict(max_tokens=1 << 20), dict(n_bias=2048)):
        assert call(_lib.Rules(**kw)) == _lib.RV12_E_RULES
    r = _lib.Rules(tokens=P, max_tokens=4)
    assert call(r) == _lib.RV12_E_NULL  # no length, no penalties
    r = _lib.Rules(n_bias=4, bias_ids=P)
    assert call(r) == _lib.RV12_E_NULL
    for f in ("tokens", "bias_ids"):
        r = _lib.Rules(length=P, penalties=P)
        setattr(r, f, P + 4)
        assert call(r) == _lib.RV12_E_ALIGN
    for f in ("length", "prompt", "penalties", "bias", "mask"):
        r = _lib.Rules()
        setattr(r, f, P + 2)
        assert call(r) == _lib.RV12_E_ALIGN


def test_lora_abi():
    from ai_amd import _lib
    L = _lib.lib()
    d = dict(a=P, b=P, scale=P, ranks=None, n=64, k=64, r=16, count=2)
    mk = lambda **kw: _lib.Lora(**{**d, **kw})
    call = lambda a, x=P, y=P, ys=64, o=P, os=64, idx=P, t=2, lnw=None, mode=0, ws=P, n=1 << 30: L.rv12_lora_apply(
        None if a is None else ctypes.byref(a), x, y, ys, o, os, idx, t, lnw, 1e-6, mode, ws, n, None)
    need = L.rv12_lora_workspace_bytes(16, 64, 2)
    assert need > 0
    for r, k, t in ((0, 64, 2), (12, 64, 2), (136, 64, 2), (16, 0, 2), (16, 40, 2), (16, 64, 0), (16, 64, 65537)):
        assert L.rv12_lora_workspace_bytes(r, k, t) == 0
    for kw in (dict(r=12), dict(r=136), dict(k=40), dict(n=0), dict(count=0)):
        assert call(mk(**kw)) == _lib.RV12_E_LORA, kw
    for kw in (dict(t=0), dict(t=65537), dict(ys=63), dict(os=63), dict(os=80)):
        assert call(mk(), **kw) == _lib.RV12_E_LORA, kw
    for kw in (dict(mode=3), dict(mode=-1), dict(mode=2, lnw=P)):
        assert call(mk(), **kw) == _lib.RV12_E_MODE, kw
    assert call(None) == _lib.RV12_E_NULL
    for f in ("a", "b", "scale"):
        assert call(mk(**{f: None})) == _lib.RV12_E_NULL
    for kw in (dict(x=None), dict(y=None), dict(o=None), dict(idx=None)):
        assert call(mk(), **kw) == _lib.RV12_E_NULL, kw
    for kw in (dict(x=P + 8), dict(lnw=P + 8), dict(ws=P + 8), dict(idx=P + 2), dict(y=P + 2, o=P + 2)):
        assert call(mk(), **kw) == _lib.RV12_E_ALIGN, kw
    assert call(mk(a=P + 8)) == _lib.RV12_E_ALIGN and call(mk(ranks=P + 1)) == _lib.RV12_E_ALIGN
    assert call(mk(), n=need - 1) == _lib.RV12_E_WORKSPACE and call(mk(), ws=None) == _lib.RV12_E_WORKSPACE


def test_cpu_tensors_are_refused():
    from ai_amd import logits
    from ai_amd.lora import Adapters
    with pytest.raises(ValueError):
        logits.adjust(torch.zeros(1, 8))
    with pytest.raises(ValueError):
        Adapters(torch.zeros(1, 8, 32, dtype=torch.bfloat16), torch.zeros(1, 4, 8, dtype=torch.bfloat16), torch.zeros(1))


def test_head_pick_refuses_outputs_among_the_rules():
    """The rules that Head.pick passes on are inputs: logits sent elsewhere would
    leave a sampled pick without the rules."""
    from ai_amd.head import Head
    head = Head.__new__(Head)  # refused before the head's matrix is looked at
    h = torch.zeros(1, 8)
    for rules in ({"out": torch.zeros(1, 100)}, {"ids": torch.zeros(1, dtype=torch.int64)}, {"x": h},
                  {"mask": None, "out": None}, {"penalty": None}):
        for temperature in (0.0, 1.0):
            with pytest.raises(ValueError, match="rules"):
                head.pick(h, 1, temperature=temperature, rules=rules)

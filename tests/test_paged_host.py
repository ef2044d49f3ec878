"""The paged cache's refusals that need no GPU: the object's and the C ABI's
argument checks, all before any device work."""
import ctypes

import pytest
import torch


def _paged(**kw):
    from ai_amd import _lib
    d = dict(n_heads=32, n_kv=8, head_dim=128, page=16, kv_bf16=1, n_seq=4, max_pages=8, table_stride=8, n_pages=40,
             eps=1e-6, scale=0.1)
    d.update(kw)
    return _lib.Paged(*(d[n] for n, _ in _lib.Paged._fields_))


BAD = [dict(head_dim=96), dict(n_heads=31), dict(n_kv=0), dict(n_heads=136), dict(page=8), dict(page=48), dict(page=2048),
       dict(n_seq=0), dict(max_pages=0), dict(n_pages=0), dict(table_stride=7), dict(max_pages=1 << 27, table_stride=1 << 27)]


@pytest.mark.parametrize("kw", BAD)
def test_abi_refuses_geometry(kw):
    from ai_amd import _lib
    L = _lib.lib()
    a = _paged(**kw)
    p = 4096  # never dereferenced: the checks come first
    assert L.rv12_paged_attend_workspace_bytes(ctypes.byref(a), 4) == 0
    assert L.rv12_paged_attend(ctypes.byref(a), 4, p, p, p, p, p, p, p, p, 1 << 30, None) == _lib.RV12_E_PAGED
    assert L.rv12_paged_append(ctypes.byref(a), 4, p, p, p, p, p, p, p, p, p, p, None) == _lib.RV12_E_PAGED


def test_abi_refuses_arguments():
    from ai_amd import _lib
    L = _lib.lib()
    a = _paged()
    need = L.rv12_paged_attend_workspace_bytes(ctypes.byref(a), 4)
    assert need > 0
    p = 4096
    for t in (0, -1, 65537):
        assert L.rv12_paged_attend(ctypes.byref(a), t, p, p, p, p, p, p, p, p, 1 << 40, None) == _lib.RV12_E_PAGED
    assert L.rv12_paged_attend(None, 4, p, p, p, p, p, p, p, p, need, None) == _lib.RV12_E_NULL
    full = [p] * 8
    for i in (0, 2, 3, 4, 5, 6):  # seq may be NULL
        b = list(full)
        b[i] = None
        assert L.rv12_paged_attend(ctypes.byref(a), 4, *b, need, None) == _lib.RV12_E_NULL
    for i in (0, 4, 5, 6, 7):
        b = list(full)
        b[i] = p + 8
        assert L.rv12_paged_attend(ctypes.byref(a), 4, *b, need, None) == _lib.RV12_E_ALIGN
    assert L.rv12_paged_attend(ctypes.byref(a), 4, *full, need - 1, None) == _lib.RV12_E_WORKSPACE
    assert L.rv12_paged_attend(ctypes.byref(a), 4, *full[:7], None, need, None) == _lib.RV12_E_WORKSPACE
    for i in (0, 1, 2, 3, 5, 6, 7, 8, 9):
        b = [p] * 10
        b[i] = None
        assert L.rv12_paged_append(ctypes.byref(a), 4, *b, None) == _lib.RV12_E_NULL
    for i in (0, 1, 2, 7, 8, 9):
        b = [p] * 10
        b[i] = p + 8
        assert L.rv12_paged_append(ctypes.byref(a), 4, *b, None) == _lib.RV12_E_ALIGN
    assert "paged" in _lib.strerror(_lib.RV12_E_PAGED)


def test_object_refusals():
    from ai_amd.attn import PagedRopeAttn
    for args in ((32, 8, 128, 16, torch.float16), (32, 8, 96, 16, torch.float32), (32, 8, 128, 24, torch.float32),
                 (30, 8, 128, 16, torch.float32), (136, 8, 128, 16, torch.float32)):
        with pytest.raises(ValueError):
            PagedRopeAttn(*args, 1e-6)
    p = PagedRopeAttn(8, 4, 64, 16, torch.float32, 1e-6)
    z = torch.zeros
    with pytest.raises(ValueError):  # CPU tensors
        p.attend(z(1, 512), None, z(1, dtype=torch.int64), z(1, 1, dtype=torch.int32), z(1, 4, 16, 64), z(1, 4, 16, 64),
                 z(1, 512))

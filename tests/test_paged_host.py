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
       dict(n_seq=0), dict(max_pages=0), dict(n_pages=0), dict(table_stride=7), dict(max_pages=1 << 27, table_stride=1 << 27),
       dict(max_pages=(1 << 26) + 1, table_stride=1 << 27)]


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


def _plan(lens, n_kv, grain, target=1024):
    """The attention's plan as the kernel forms it: chunk length, chunks per row."""
    total = sum((n + 31) // 32 for n in lens)
    up = lambda a, b: -(-a // b)
    half = up(total * n_kv, target // 2) * 32
    c = half if half <= 512 else max(up(total * n_kv, target) * 32, 512)
    C = up(max(c, 1), grain) * grain
    return C, [max(1, up(n, C)) for n in lens]


@pytest.mark.parametrize("n_kv", [1, 2, 3, 5, 7, 8, 11, 16, 100, 256])
@pytest.mark.parametrize("bf16", [0, 1])
def test_workspace_holds_every_plan(n_kv, bf16):
    """Whatever the lengths, the partials of the rows in several chunks fit the
    workspace, and the grid's workgroups cover every chunk (rows just past a
    chunk's end need the most of both)."""
    import random
    from ai_amd import _lib
    L = _lib.lib()
    rng = random.Random(n_kv)
    worst, grain = 0, 128 if bf16 else 64
    for _ in range(400):
        T = rng.choice([1, 2, 3, 17, 64, 65, 200, 700])
        pages = rng.choice([1, 9, 300, 4000])
        cap = pages * 16
        a = _paged(n_heads=n_kv, n_kv=n_kv, kv_bf16=bf16, max_pages=pages, table_stride=pages)
        need = L.rv12_paged_attend_workspace_bytes(ctypes.byref(a), T)
        assert need > 0
        per_slot = n_kv * 16 * (128 + 4) * 4
        items, rows = min(1024 // n_kv + T, T * -(-cap // grain)), min(T, 1024 // n_kv) if cap > grain else 0
        room, rest = divmod(need - 16 - (32 * (1 + items + rows) if T > 64 else 0), per_slot)
        assert rest == 0
        base = rng.choice([0, rng.randint(1, cap), cap])
        lens = [min(cap, max(0, rng.choice([base, base + 1, rng.randint(0, cap)]))) for _ in range(T)]
        C, chunks = _plan(lens, n_kv, grain)
        # the rows' lengths just past multiples of that chunk length
        for _ in range(3):
            split = [c for c in chunks if c > 1]
            assert sum(split) <= room and len(split) <= rows
            assert sum(chunks) <= items
            worst = max(worst, sum(split) / max(room, 1))
            lens = [min(cap, C * rng.randint(1, 2) + 1) for _ in range(T)]
            C, chunks = _plan(lens, n_kv, grain)
    assert worst > 0.4  # the draws come near the bound


@pytest.mark.parametrize("bf16", [0, 1])
def test_workspace_of_few_positions(bf16):
    """A call needs no more partials than its rows' positions can have chunks, so a
    few short rows do not hold what 1024 workgroups would."""
    from ai_amd import _lib
    L = _lib.lib()
    grain = 128 if bf16 else 64
    per_slot = 8 * 16 * (128 + 4) * 4
    for T, pages in ((1, 1), (1, 16), (1, 17), (3, 40), (16, 64), (64, 8), (1, 4096), (64, 4096)):
        a = _paged(kv_bf16=bf16, max_pages=pages, table_stride=pages)
        chunks = T * -(-16 * pages // grain) if 16 * pages > grain else 0
        assert L.rv12_paged_attend_workspace_bytes(ctypes.byref(a), T) == 16 + min(chunks, 256) * per_slot, (T, pages)


def test_rows_times_positions_bounds_the_attention_alone():
    """The plan's sums hold 2^35 row positions (2^40 times the kv heads); the append
    has no plan, and takes as many rows as any table."""
    from ai_amd import _lib
    L = _lib.lib()
    p = 4096
    for T, pages, n_kv, fits in ((32, 1 << 20, 8, True), (33, 1 << 20, 8, False), (65536, 512, 8, True), (65536, 513, 8, False),
                                 (32, 1 << 20, 32, True), (32, 1 << 20, 33, False), (65536, 1 << 20, 256, False)):
        a = _paged(n_heads=n_kv, n_kv=n_kv, page=1024, max_pages=pages, table_stride=pages)
        assert (L.rv12_paged_attend_workspace_bytes(ctypes.byref(a), T) > 0) == fits, (T, pages, n_kv)
        rc = L.rv12_paged_attend(ctypes.byref(a), T, p, p, p, p, p, p, p, None, 1 << 50, None)
        assert rc == (_lib.RV12_E_WORKSPACE if fits else _lib.RV12_E_PAGED)
        # past the size checks: the next one is for the pointers
        assert L.rv12_paged_append(ctypes.byref(a), T, None, p, p, p, p, p, p, p, p, p, None) == _lib.RV12_E_NULL
    assert "2^35" in _lib.strerror(_lib.RV12_E_PAGED)


def test_call_refuses_shapeless_tables():
    """append and attend in one call look at the table's size first: a table of no
    dimension is refused as by append."""
    from ai_amd.attn import PagedRopeAttn
    p = PagedRopeAttn(8, 4, 64, 16, torch.float32, 1e-6)
    z = torch.zeros
    pos = z(1, dtype=torch.int64)
    for table in (torch.tensor(0, dtype=torch.int32), z(3, dtype=torch.int32), z(0, 0, dtype=torch.int32)):
        with pytest.raises(ValueError):
            p(z(1, 1024), z(64), z(64), z(32), None, pos, table, z(1, 4, 16, 64), z(1, 4, 16, 64), z(1, 512))

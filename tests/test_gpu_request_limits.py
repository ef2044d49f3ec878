"""The operators for several requests at their largest row and head counts, and the
plan of more than 64 rows in a captured graph, against the same formulas in float64
with the tolerances of their own tests (test_gpu_paged, test_gpu_logits,
test_gpu_lora)."""
import numpy as np
import pytest
import torch

import test_gpu_logits as tl
import test_gpu_lora as ta
import test_gpu_paged as tp

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _one_page_ref(q, own, table, kc, vc, H, KV, HD, n):
    """(out, bound) of rows that see the first n[r] <= page positions of one page."""
    G, page = H // KV, kc.shape[2]
    K, V = kc.double()[table[own, 0].long()], vc.double()[table[own, 0].long()]
    qd = q.double().view(-1, KV, G, HD)
    dead = torch.arange(page, device="cuda")[None, :] >= n[:, None]
    dead = dead[:, None, None, :]
    z = torch.matmul(qd, K.transpose(2, 3).contiguous()) * HD ** -0.5
    za = (torch.matmul(qd.abs(), K.abs().transpose(2, 3).contiguous()) * HD ** -0.5).masked_fill(dead, 0)
    w = torch.softmax(z.masked_fill(dead, -float("inf")), -1)
    rel = 4 * (HD + 4) * U * za.amax(-1, keepdim=True) + 2.0 ** -21 + (112 + 64) * U
    return torch.matmul(w, V).reshape(-1, H, HD), (rel * torch.matmul(w, V.abs())).reshape(-1, H, HD)


@pytest.mark.parametrize("kv", tp.KV_TYPES)
def test_paged_65536_rows(kv):
    """The most rows of a pass: 40000 sequences of one row, 1250 of 20, padding."""
    from ai_amd.attn import PagedRopeAttn
    H, KV, HD, page, n_seq = 2, 1, 64, 16, 41250
    g = tp._gen(20)
    own = torch.cat([torch.arange(40000), torch.arange(40000, n_seq).repeat_interleave(20), torch.full((536,), -1)]).int().cuda()
    pos = torch.cat([torch.randint(0, 16, (40000,)), torch.arange(20).repeat(1250) % 16, torch.zeros(536, dtype=torch.long)]).cuda()
    T = len(own)
    assert T == 65536
    table = torch.randperm(n_seq, generator=g, device="cuda").int()[:, None].contiguous()
    kc, vc = tp._randn(g, n_seq, KV, page, HD).to(kv), tp._randn(g, n_seq, KV, page, HD).to(kv)
    q = tp._randn(g, T, H * HD) * 2
    p = PagedRopeAttn(H, KV, HD, page, kv, tp.EPS)
    out = torch.full_like(q, float("nan"))
    p.attend(q, own, pos, table, kc, vc, out)
    torch.cuda.synchronize()
    live = own >= 0
    ref, bound = _one_page_ref(q[live], own[live].long(), table, kc, vc, H, KV, HD, pos[live] + 1)
    assert bool(((out[live].double().view(-1, H, HD) - ref).abs() <= bound).all())
    assert torch.equal(out[~live], torch.zeros_like(out[~live]))
    # the append of as many rows: values land in their slots, rows of one slot agree
    qkv = tp._randn(g, T, (H + 2 * KV) * HD)
    qkv[~live] = 0
    ones = torch.ones(HD, device="cuda")
    q2 = torch.full_like(q, float("nan"))
    p.append(qkv, ones, ones, tp._inv(HD), own, pos, table, kc, vc, q2)
    torch.cuda.synchronize()
    rq, rk, rv, bq, bk = tp._append_ref(qkv, ones, ones, tp._inv(HD), pos, H, KV, HD)
    assert bool(((q2[live].double().view(-1, H, HD) - rq[live]).abs() <= bq[live]).all()) and not bool(q2[~live].any())
    first = slice(0, 40000)  # rows with a slot of their own
    pid, at = table[own[first].long(), 0].long(), pos[first]
    half = torch.finfo(kv).eps / 2
    assert torch.equal(vc[pid, :, at], rv[first].to(kv))
    assert bool(((kc[pid, :, at].double() - rk[first]).abs() <= bk[first] + half * (rk[first].abs() + bk[first])).all())
    with pytest.raises(ValueError):
        p.attend(torch.zeros(T + 1, H * HD, device="cuda"), None, torch.zeros(T + 1, dtype=torch.long, device="cuda"), table,
                 kc, vc, torch.zeros(T + 1, H * HD, device="cuda"))


@pytest.mark.parametrize("kv", tp.KV_TYPES)
@pytest.mark.parametrize("H,KV,HD,page", [(256, 256, 64, 16), (100, 100, 128, 32), (48, 3, 128, 1024), (44, 11, 64, 512)])
def test_paged_head_counts_and_large_pages(H, KV, HD, page, kv):
    """Up to 256 kv heads, 16 query heads each, pages longer than a chunk."""
    from ai_amd.attn import PagedRopeAttn
    g = tp._gen(H, page, 21)
    lens = [1, 700, 2100, 33]
    print("case", H, KV, HD, page, kv, flush=True)
    table, n_pages = tp._table(lens, page, g)
    kc, vc = (tp._randn(g, n_pages, KV, page, HD).to(kv) for _ in range(2))
    rows = [(0, 0), (1, 699), (2, 2097), (2, 2098), (2, 2099), (3, 32), (-1, 0), (2, 1023), (2, 1024)]
    seq = torch.tensor([r[0] for r in rows], dtype=torch.int32, device="cuda")
    pos = torch.tensor([r[1] for r in rows], device="cuda")
    q = tp._randn(g, len(rows), H * HD)
    tp._check(PagedRopeAttn(H, KV, HD, page, kv, tp.EPS), q, seq, pos, table, kc, vc)


@pytest.mark.parametrize("kv", tp.KV_TYPES)
def test_append_under_the_largest_table(kv):
    """Rows up to the last of 2^30 positions, more of them than the attention takes
    with such a table: appended alone, and refused before anything is written where
    the attention is to follow."""
    from ai_amd.attn import PagedRopeAttn
    H, KV, HD, page, T = 4, 2, 64, 1024, 40
    g = tp._gen(25)
    table = torch.full((1, 1 << 20), -1, dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(20), torch.arange((1 << 30) - 20, 1 << 30)]).cuda()
    table[0, 0], table[0, -1] = 2, 0
    kc, vc = (tp._randn(g, 3, KV, page, HD).to(kv) for _ in range(2))
    kc0, vc0 = kc.clone(), vc.clone()
    qkv, ones, seq = tp._randn(g, T, (H + 2 * KV) * HD), torch.ones(HD, device="cuda"), torch.zeros(T, dtype=torch.int32).cuda()
    p = PagedRopeAttn(H, KV, HD, page, kv, tp.EPS)
    q, out = torch.full((T, H * HD), float("nan"), device="cuda"), torch.zeros(T, H * HD, device="cuda")
    args = (qkv, ones, ones, tp._inv(HD), seq, pos, table, kc, vc)
    for call in (lambda: p(*args, out), lambda: p.attend(q, seq, pos, table, kc, vc, out)):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)
    p.append(*args, q)
    torch.cuda.synchronize()
    rq, rk, rv, bq, bk = tp._append_ref(qkv, ones, ones, tp._inv(HD), pos, H, KV, HD)
    assert bool(((q.double().view(T, H, HD) - rq).abs() <= bq).all())
    pid, at = torch.tensor([2] * 20 + [0] * 20, device="cuda"), pos % page
    half = torch.finfo(kv).eps / 2
    assert torch.equal(vc[pid, :, at], rv.to(kv))
    assert bool(((kc[pid, :, at].double() - rk).abs() <= bk + half * (rk.abs() + bk)).all())
    kc0[pid, :, at], vc0[pid, :, at] = kc[pid, :, at], vc[pid, :, at]
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)  # and nowhere else


@pytest.mark.parametrize("kv", tp.KV_TYPES)
def test_graph_of_more_than_64_rows(kv):
    """A captured pass of 150 rows (its plan a launch of its own) replayed with other
    rows each time, beside a second graph of the same object, and eager calls."""
    from ai_amd.attn import PagedRopeAttn
    H, KV, HD, page, T = 16, 8, 128, 16, 150
    g = tp._gen(22)
    lens = [900, 40, 333, 2000] + [5 + i for i in range(100)]
    table, n_pages = tp._table(lens, page, g)
    kc, vc = (tp._randn(g, n_pages, KV, page, HD).to(kv) for _ in range(2))
    p = PagedRopeAttn(H, KV, HD, page, kv, tp.EPS)

    def rows(k):
        r = [(0, 800 + j) for j in range(100)] + [(3, 1999 - 3 * j) for j in range(50)] if k == 0 else \
            [(i, lens[i] - 1) for i in range(104)] + [(-1, 0)] * 40 + [(2, j) for j in range(6)] if k == 1 else \
            [(k % 4, j % lens[k % 4]) for j in range(150)]
        return torch.tensor([a for a, _ in r], dtype=torch.int32), torch.tensor([b for _, b in r])
    sides = []
    for _ in range(2):
        q, out = torch.zeros(T, H * HD, device="cuda"), torch.zeros(T, H * HD, device="cuda")
        seq, pos = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int64, device="cuda")
        p.attend(q, seq, pos, table, kc, vc, out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p.attend(q, seq, pos, table, kc, vc, out)
        sides.append((graph, q, seq, pos, out))
    other = torch.cuda.Stream()
    for k in range(5):
        for i, (graph, q, seq, pos, out) in enumerate(sides):
            s, ps = rows((k + i) % 5)
            seq.copy_(s)
            pos.copy_(ps)
            q.copy_(tp._randn(g, T, H * HD))
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        sides[0][0].replay()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            sides[1][0].replay()
        torch.cuda.synchronize()
        for graph, q, seq, pos, out in sides:
            assert torch.equal(tp._check(p, q, seq, pos, table, kc, vc, k), out), k


def test_rules_on_65535_rows():
    """The most rows of the rules: histories, biases, masks and the pick."""
    rng = np.random.default_rng(23)
    T, V = 65535, 37
    x, a = tl._case(rng, T, V, 3, 2, True)
    y, ids, _ = tl._run(x, a)
    pick = [0, 1, 31, 32, 4095, 4096, 32767, 32768, 65533, 65534] + rng.integers(0, T, 3000).tolist()
    ref, bound, ok = tl._ref(x[pick], **{k: v[pick] for k, v in a.items()})
    tl._same(y[pick], ref, bound)
    assert [ids[r] for r in pick] == tl._pick(y[pick], ok)


def test_adapters_on_65536_rows():
    """The most rows of the adapters: runs, mixed tiles, rows without one."""
    from ai_amd.lora import Adapters
    g = torch.Generator(device="cuda").manual_seed(24)
    N, K, R, T = 19, 64, 8, 65536
    A, B, scale = ta._bank(g, 9, R, K, N)
    ad = Adapters(A, B, scale)
    x, y, lnw = ta._inputs(g, T, K, N, 0, True)
    idx = torch.randint(-1, 9, (T,), generator=g, device="cuda", dtype=torch.int32)
    idx[1000:30000] = 4
    out = torch.full_like(y, float("nan"))
    ad.apply(x, y, idx, lnw=lnw, eps=ta.EPS, out=out)
    torch.cuda.synchronize()
    xd = x.double() * (x.double().square().mean(1, keepdim=True) + ta.EPS).rsqrt() * lnw.double()
    own, Ad, Bd = idx.clamp(min=0).long(), A.double(), B.double()
    row = torch.arange(T, device="cuda")

    def through(v, a, b):
        h = torch.stack([v @ m.T for m in a])[own, row]
        return (b[own] * h[:, None, :]).sum(2) * (scale.double()[own] * (idx >= 0))[:, None]
    d = through(xd, Ad, Bd)
    # test_gpu_lora's bound
    rel = (K / 64 + 40 + 16 + 3 * K / 32 + 80 + 3 * R / 32 + 80 + 8) * U
    ta._check(out, y.double() + d, U * y.double().abs() + rel * through(xd.abs(), Ad.abs(), Bd.abs()) + U * d.abs())

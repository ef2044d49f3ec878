"""Low-rank adapters (rv12_lora_apply through ai_amd.lora.Adapters) against
out = y + scale B (A x') in float64.

Tolerance: x' and h in three bf16 parts keep 2^-24 of each value; u = 2^-24.  The
norm's factor is off by at most (K / 64 + 40) u (its sum runs in chains of K / 64
per lane at most, then joins), silu by 16 u; the first product's sum by
(3 K / 32 + 80) u of sum |A x'|, the second's by (3 R / 32 + 80) u, and out has one
rounding of its own.  Bound: all of it against |scale| |B| |A| |x'| + |y|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6


def _ref(x, y, idx, A, B, scale, mode, lnw, ranks=None):
    K = A.shape[2]
    xd = x.double()
    if mode == 2:
        xd = torch.nn.functional.silu(xd[:, :K]) * xd[:, K:]
    if lnw is not None:
        xd = xd * (xd.square().mean(1, keepdim=True) + EPS).rsqrt() * lnw.double()
    out, mag = y.double().clone(), y.double().abs()
    rel = (K / 64 + 40 + 16 + 3 * K / 32 + 80 + 3 * A.shape[1] / 32 + 80 + 8) * U
    bound = U * mag
    for t, a in enumerate(idx.tolist()):
        if not 0 <= a < len(A):
            continue
        r = A.shape[1] if ranks is None else ranks[a]
        Ad, Bd, s = A[a, :r].double(), B[a, :, :r].double(), float(scale[a])
        out[t] += s * (Bd @ (Ad @ xd[t]))
        bound[t] += rel * abs(s) * (Bd.abs() @ (Ad.abs() @ xd[t].abs())) + U * (s * (Bd @ (Ad @ xd[t]))).abs()
    return out, bound


def _bank(g, count, R, K, N):
    A = (torch.randn(count, R, K, device="cuda", generator=g) * K ** -0.5).bfloat16()
    B = (torch.randn(count, N, R, device="cuda", generator=g) * 0.05).bfloat16()
    return A, B, 0.5 + torch.rand(count, device="cuda", generator=g)


def _inputs(g, T, K, N, mode, norm):
    x = torch.randn(T, 2 * K if mode == 2 else K, device="cuda", generator=g)
    x[:, ::97] *= 30
    lnw = (1 + 0.2 * torch.randn(K, device="cuda", generator=g)).bfloat16() if norm else None
    return x, torch.randn(T, N, device="cuda", generator=g), lnw


def _check(out, ref, bound, what=""):
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), (what, float((err - bound).max()))


@pytest.mark.parametrize("N,K", [(1, 32), (17, 64), (1024, 2048), (4099, 1056), (6144, 4096)])
@pytest.mark.parametrize("R", [1, 4, 8, 16, 24, 40, 64, 128])
@pytest.mark.parametrize("mode,norm", [(0, False), (1, True), (2, False)])
def test_matches_float64(N, K, R, mode, norm):
    from ai_amd.lora import Adapters
    g = torch.Generator(device="cuda").manual_seed(N + 31 * K + R)
    A, B, scale = _bank(g, 5, R, K, N)
    ad = Adapters(A, B, scale)
    for T in (1, 2, 16, 17, 37):
        print("case", N, K, R, mode, norm, T, flush=True)
        x, y, lnw = _inputs(g, T, K, N, mode, norm)
        idx = torch.randint(-1, 6, (T,), device="cuda", generator=g, dtype=torch.int32)  # 5: outside, as -1
        ref, bound = _ref(x, y, idx, A, B, scale, mode, lnw)
        out = torch.full_like(y, float("nan"))
        assert ad.apply(x, y, idx, mode=mode, lnw=lnw, eps=EPS, out=out) is out
        torch.cuda.synchronize()
        _check(out, ref, bound, T)
        none = (idx < 0) | (idx > 4)
        assert torch.equal(out[none], y[none])
        y2 = y.clone()
        assert ad.apply(x, y2, idx, mode=mode, lnw=lnw, eps=EPS) is y2
        assert torch.equal(y2, out)


def test_ranks_and_pairs():
    """Adapters of several ranks in one bank; what the bank holds past a rank, NaN
    among it, is not used."""
    from ai_amd.lora import Adapters
    g = torch.Generator(device="cuda").manual_seed(3)
    N, K, R = 96, 256, 37
    A, B, scale = _bank(g, 4, R, K, N)
    ranks = [37, 5, 0, 16]
    for a, r in enumerate(ranks):
        A[a, r:] = float("nan")
        B[a, :, r:] = float("inf")
    ad = Adapters(A, B, scale, ranks)
    x, y, _ = _inputs(g, 20, K, N, 0, False)
    idx = (torch.arange(20, device="cuda") % 5 - 1).int()
    ref, bound = _ref(x, y, idx, A, B, scale, 0, None, ranks)
    out = ad.apply(x, y, idx, out=torch.empty_like(y))
    _check(out, ref, bound)
    pairs = [(A[a, :r].float(), B[a, :, :r], 2.0 * r) for a, r in enumerate(ranks) if r]
    ad2 = Adapters.from_pairs(pairs)
    i2 = torch.tensor([0, 1, 2, 2, -1], dtype=torch.int32, device="cuda")
    two = torch.full((3,), 2.0, device="cuda")
    keep = [0, 1, 3]
    ref, bound = _ref(x[:5], y[:5], i2, A[keep], B[keep], two, 0, None, [ranks[k] for k in keep])
    _check(ad2.apply(x[:5].contiguous(), y[:5].contiguous(), i2), ref, bound)


def test_many_rows_runs_and_slices():
    """A prompt's rows, in runs of one adapter and mixed in one tile of 16; y and
    out slices of a fused projection's output, at addresses of 4 and 16 bytes."""
    from ai_amd.lora import Adapters
    g = torch.Generator(device="cuda").manual_seed(4)
    N, K, R, T = 260, 512, 16, 333
    A, B, scale = _bank(g, 40, R, K, N)
    ad = Adapters(A, B, scale)
    x, _, lnw = _inputs(g, T, K, N, 0, True)
    idx = torch.cat([torch.full((100,), 7), torch.arange(100) % 41 - 1, torch.full((100,), -1), torch.full((33,), 39)]).int().cuda()
    for first, wide in ((0, 512), (4, 512), (3, 700), (1, 261)):
        y = torch.randn(T, wide, device="cuda", generator=g)
        y0 = y.clone()
        ref, bound = _ref(x, y[:, first:first + N], idx, A, B, scale, 0, lnw)
        ad.apply(x, y[:, first:first + N], idx, lnw=lnw, eps=EPS)
        torch.cuda.synchronize()
        _check(y[:, first:first + N], ref, bound, (first, wide))
        y[:, first:first + N] = y0[:, first:first + N]
        assert torch.equal(y, y0)  # nothing beside the slice


def test_row_does_not_depend_on_its_neighbours():
    """A row's output is the same whatever adapters the rows beside it use, and
    NaN or infinity in another row stays there."""
    from ai_amd.lora import Adapters
    g = torch.Generator(device="cuda").manual_seed(5)
    N, K, R, T = 320, 1024, 32, 32
    A, B, scale = _bank(g, 8, R, K, N)
    ad = Adapters(A, B, scale)
    x, y, lnw = _inputs(g, T, K, N, 0, True)
    idx = torch.randint(0, 8, (T,), device="cuda", generator=g, dtype=torch.int32)
    out = ad.apply(x, y, idx, lnw=lnw, out=torch.empty_like(y))
    other = torch.randint(-1, 8, (T,), device="cuda", generator=g, dtype=torch.int32)
    other[5], other[20] = idx[5], idx[20]
    x2 = x.clone()
    x2[6], x2[21, 3] = float("nan"), float("inf")
    o2 = ad.apply(x2, y, other, lnw=lnw, out=torch.empty_like(y))
    assert torch.equal(o2[[5, 20]], out[[5, 20]])
    if int(other[6]) >= 0:
        assert bool(o2[6].isnan().all())


def test_beside_the_linear_in_a_graph():
    """The shared 12-bit linear with its prologue, then the adapters, captured and
    replayed with other rows and adapters, against the sum of both in float64."""
    from ai_amd import wcomp
    from ai_amd.lora import Adapters
    g = torch.Generator(device="cuda").manual_seed(6)
    N, K, R, T = 512, 1024, 16, 9
    W = (torch.randn(N, K, device="cuda", generator=g) * 0.02).bfloat16()
    c = wcomp.compress(W)
    A, B, scale = _bank(g, 3, R, K, N)
    ad = Adapters(A, B, scale)
    x, _, lnw = _inputs(g, T, K, N, 0, True)
    y = torch.zeros(T, N, device="cuda")
    idx = torch.zeros(T, dtype=torch.int32, device="cuda")

    def step():
        wcomp.gemvc_tc(x, c, y, 0, T, lnw=lnw, eps=EPS)
        ad.apply(x, y, idx, lnw=lnw, eps=EPS)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        x.copy_(_inputs(g, T, K, N, 0, True)[0])
        idx.copy_(torch.randint(-1, 3, (T,), device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, y)
        xn = x.double() * (x.double().square().mean(1, keepdim=True) + EPS).rsqrt() * lnw.double()
        ref, bound = _ref(x, (xn @ W.double().T), idx, A, B, scale, 0, lnw)
        _check(y, ref, bound + (3 * K / 32 + 200) * U * (xn.abs() @ W.double().abs().T))


def test_bank_past_32_bits():
    """A bank of more than 2^32 bytes: the last adapters."""
    from ai_amd.lora import Adapters
    N, K, R = 8192, 8192, 128
    count = (1 << 31) // (R * K) + 3
    A = torch.empty(count, R, K, dtype=torch.bfloat16, device="cuda")
    B = torch.empty(count, N, R, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    a, b, s = _bank(g, 2, R, K, N)
    A[-2:], B[-2:] = a, b
    scale = torch.ones(count, device="cuda")
    ad = Adapters(A, B, scale)
    x, y, _ = _inputs(g, 2, K, N, 0, False)
    idx = torch.tensor([count - 1, count - 2], dtype=torch.int32, device="cuda")
    ref, bound = _ref(x, y, torch.tensor([1, 0]), a, b, torch.ones(2), 0, None)
    _check(ad.apply(x, y, idx), ref, bound)


def test_refusals():
    from ai_amd.lora import Adapters
    g = torch.Generator(device="cuda").manual_seed(8)
    N, K, R, T = 64, 64, 8, 3
    A, B, scale = _bank(g, 2, R, K, N)
    for args in ((A.float(), B, scale), (A, B[:1], scale), (A, B[..., :4], scale), (A[..., :40], B, scale), (A.cpu(), B, scale),
                 (A, B, scale.double()), (A, B, scale[:1]), (A[:0], B[:0], scale[:0]), (A, B, scale, [8]),
                 (A, B, scale, [8, 9]), (A, B, scale, [-1, 8]), (A[0], B[0], scale)):
        with pytest.raises(ValueError):
            Adapters(*args)
    big = torch.zeros(1, 129, K, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        Adapters(big, torch.zeros(1, N, 129, dtype=torch.bfloat16, device="cuda"), scale[:1])
    with pytest.raises(ValueError):
        Adapters.from_pairs([])
    with pytest.raises(ValueError):
        Adapters.from_pairs([(A[0], B[0], 1.0), (A[0], B[0, :-1], 1.0)])
    ad = Adapters(A, B, scale)
    x, y, lnw = _inputs(g, T, K, N, 0, True)
    idx = torch.zeros(T, dtype=torch.int32, device="cuda")
    ok = dict(x=x, y=y, idx=idx)
    ad.apply(**ok)
    for bad in (dict(x=x[:2]), dict(x=x.double()), dict(x=x.t().contiguous().t()), dict(mode=2), dict(mode=3), dict(y=y[:, :-1]),
                dict(y=y.bfloat16()), dict(y=y[:1].expand(T, N)), dict(out=y.t()), dict(idx=idx.long()), dict(idx=idx[:2]),
                dict(idx=idx.cpu()), dict(lnw=lnw.float()), dict(lnw=lnw[:-1])):
        with pytest.raises(ValueError):
            ad.apply(**{**ok, **bad})
    x2 = torch.zeros(T, 2 * K, device="cuda")
    with pytest.raises(ValueError):
        ad.apply(x2, y, idx, mode=2, lnw=lnw)
    assert ad.apply(x[:0], y[:0], idx[:0]).shape == (0, N)
    torch.cuda.synchronize()

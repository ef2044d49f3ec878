"""Rules on logits (rv12_logits_adjust through ai_amd.logits.adjust and
Head.pick) against the same rules in float64 numpy.

Tolerance: a logit goes through at most five float32 roundings (the penalty's
product or quotient, frequency times count, plus presence, their subtraction,
the bias): 5 u of the largest magnitude among the terms, u = 2^-24."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _ref(x, tokens=None, length=None, prompt=None, penalties=None, bias_ids=None, bias=None, mask=None):
    """(adjusted, bound, allowed) in float64."""
    y = x.astype(np.float64)
    big = np.abs(y)
    T, V = x.shape
    for r in range(T):
        if tokens is not None:
            past = tokens[r, :min(max(length[r], 0), tokens.shape[1])]
            made = past[max(prompt[r], 0) if prompt is not None else 0:]
            rep, freq, pres = penalties[r].astype(np.float64)
            for n in set(past.tolist()):
                if 0 <= n < V:
                    y[r, n] = y[r, n] / rep if y[r, n] > 0 else y[r, n] * rep
                    c = int((made == n).sum())
                    big[r, n] = max(abs(x[r, n]), abs(y[r, n])) + abs(freq * c) + abs(pres)
                    if c:
                        y[r, n] -= freq * c + pres
        if bias_ids is not None:
            for n, b in dict(zip(bias_ids[r].tolist(), bias[r].astype(np.float64))).items():
                if 0 <= n < V:
                    y[r, n] += b
                    big[r, n] += abs(b)
    ok = np.ones((T, V), bool)
    if mask is not None:
        ok = np.unpackbits(np.ascontiguousarray(mask).view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)
        y[~ok] = -np.inf
    return y, 5 * U * big, ok


def _pick(y, ok):
    out = []
    for r in range(len(y)):
        n = np.flatnonzero(ok[r])
        out.append(int(n[np.argmax(y[r, n])]) if len(n) else -1)  # numpy: the first NaN, else the first largest
    return out


def _case(rng, T, V, L, M, mask, spare=0):
    a = {}
    x = (rng.standard_normal((T, V)) * 3).astype(np.float32)
    if L is not None:
        a["tokens"] = np.where(rng.random((T, L)) < 0.5, rng.integers(0, min(V, 20), (T, L)), rng.integers(0, V, (T, L)))
        a["tokens"][rng.random((T, L)) < 0.02] = -1
        a["tokens"][rng.random((T, L)) < 0.02] = V + 3
        a["length"] = rng.integers(0, L + 1, T).astype(np.int32)
        a["prompt"] = rng.integers(0, L + 1, T).astype(np.int32)
        a["penalties"] = np.stack([rng.uniform(0.8, 1.6, T), rng.uniform(-0.5, 1, T), rng.uniform(-0.5, 1, T)], 1).astype(np.float32)
    if M is not None:
        a["bias_ids"] = rng.integers(-1, V + 1, (T, M))  # ids twice, unused entries and one past the end among them
        a["bias"] = (rng.standard_normal((T, M)) * 4).astype(np.float32)
    if mask:
        words = rng.integers(-2 ** 31, 2 ** 31, (T, -(-V // 32))).astype(np.int32)
        words[:: 3] &= rng.integers(-2 ** 31, 2 ** 31, words[::3].shape).astype(np.int32) & 0x11111111
        a["mask"] = words
    return x, a


def _run(x, a, ids=True, out=None):
    from ai_amd import logits
    T, V = x.shape
    cu = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    xt = torch.from_numpy(x).cuda()
    it = torch.full((T,), -5, dtype=torch.int64, device="cuda") if ids else None
    y = logits.adjust(xt, torch.full((T, V), float("nan"), device="cuda") if out is None else out, ids=it, **cu)
    torch.cuda.synchronize()
    return y.cpu().numpy(), None if it is None else it.tolist(), xt


def _same(y, ref, bound):
    inf = np.isinf(ref) | np.isnan(ref)
    assert np.array_equal(y[inf], ref[inf].astype(np.float32), equal_nan=True)
    err = np.abs(y[~inf].astype(np.float64) - ref[~inf])
    assert (err <= bound[~inf]).all(), float((err - bound[~inf]).max())


@pytest.mark.parametrize("V", [1, 31, 33, 1000, 4096, 4097, 20011, 151936])
@pytest.mark.parametrize("T,L,M,mask", [(1, None, None, False), (1, 1, None, False), (3, 700, 5, True), (2, None, 40, False),
                                        (5, None, None, True), (7, 3000, None, True), (2, 64, 1500, False), (20, 17, 3, True)])
def test_matches_float64(V, T, L, M, mask):
    rng = np.random.default_rng([V, T])
    x, a = _case(rng, T, V, L, M, mask)
    print("case", V, T, L, M, mask, flush=True)
    y, ids, xt = _run(x, a)
    ref, bound, ok = _ref(x, **a)
    _same(y, ref, bound)
    assert ids == _pick(y, ok)
    lead = np.sort(np.where(ok, ref, -np.inf), 1)
    for r in range(T):
        if ok[r].sum() > 1 and lead[r, -1] - lead[r, -2] > 2 * bound[r].max():
            assert ids[r] == _pick(ref[r:r + 1], ok[r:r + 1])[0]
    # in place, and without the pick: the same bits
    y2, _, _ = _run(x, a, ids=False)
    assert np.array_equal(y, y2, equal_nan=True)
    from ai_amd import logits
    got = logits.adjust(xt, **{k: torch.from_numpy(v).cuda() for k, v in a.items()})
    assert got is xt and np.array_equal(got.cpu().numpy(), y, equal_nan=True)


def test_masked_rows_and_special_values():
    """A row whose mask allows nothing, NaN and infinities under the mask and
    beside it, ties, logits of -inf and of the type's lowest value."""
    T, V = 8, 9001
    rng = np.random.default_rng(5)
    x = rng.standard_normal((T, V)).astype(np.float32)
    words = np.full((T, -(-V // 32)), -1, np.int32)

    def forbid(r, n):
        words[r, n >> 5] &= ~np.int32(np.uint32(1 << (n & 31)).astype(np.int32))
    words[0] = 0
    x[0, 7] = np.nan
    x[1, 5000] = np.nan
    forbid(1, 5000)
    x[1, 77] = np.inf
    forbid(1, 77)
    x[2, 6000] = x[2, 8000] = np.nan
    x[3, [10, 4100, 8999]] = 50.0
    forbid(3, 10)
    words[4] = 0
    words[4, 200] = 1 << 3
    x[4, 200 * 32 + 3] = -np.inf
    x[5] = -np.inf
    x[6] = np.finfo(np.float32).min
    words[6, :3] = 0
    x[7, :] = -1.0
    x[7, 4096] = np.inf
    a = {"mask": words, "tokens": np.arange(T * 4).reshape(T, 4) % 50, "length": np.full(T, 4, np.int32),
         "penalties": np.tile(np.float32([1.0, 0.0, 0.0]), (T, 1))}
    y, ids, _ = _run(x, a)
    ref, bound, ok = _ref(x, **a)
    _same(y, ref, bound)
    assert ids == [-1, _pick(y[1:2], ok[1:2])[0], 6000, 4100, 200 * 32 + 3, 0, 96, 4096]


def test_histories_longer_than_the_rows_tokens():
    """length past the tensor, below zero; prompt past the length; a long history
    of one id."""
    V, L = 3001, 9000
    rng = np.random.default_rng(6)
    x = rng.standard_normal((4, V)).astype(np.float32)
    tok = rng.integers(0, V, (4, L))
    tok[3] = 2999
    a = {"tokens": tok, "length": np.array([L + 100, -3, 500, L], np.int32), "prompt": np.array([100, 0, 900, -4], np.int32),
         "penalties": np.tile(np.float32([1.3, 0.25, 0.5]), (4, 1))}
    y, ids, _ = _run(x, a)
    ref, bound, ok = _ref(x, **a)
    _same(y, ref, bound)
    assert ids == _pick(y, ok)


def test_the_largest_counts():
    """2047 biases of one row and a token seen 2^20 - 1 times, generated all or all
    but some; the counts beside the biases of the same ids."""
    V, L, M = 5000, (1 << 20) - 1, 2047
    rng = np.random.default_rng(9)
    x = rng.standard_normal((2, V)).astype(np.float32)
    tok = np.full((2, L), 17)
    tok[1, ::3] = 18
    bias_ids = np.stack([rng.permutation(V)[:M], np.full(M, 17)])
    bias_ids[0, 5] = 17
    a = {"tokens": tok, "length": np.full(2, L, np.int32), "prompt": np.array([0, 1000], np.int32),
         "penalties": np.float32([[1.2, 1e-5, 0.5], [1.2, 1e-5, 0.5]]), "bias_ids": bias_ids,
         "bias": rng.standard_normal((2, M)).astype(np.float32)}
    y, ids, _ = _run(x, a)
    ref, bound, ok = _ref(x, **a)
    _same(y, ref, bound)
    assert ids == _pick(y, ok)


def test_strides_expanded_rows_and_streams():
    """Rows of wider tensors, one history and mask for all rows (stride 0), odd row
    addresses, a side stream, and a captured call replayed with other inputs."""
    from ai_amd import logits
    rng = np.random.default_rng(7)
    T, V, L, M = 6, 5003, 40, 9
    x, a = _case(rng, T, V, L, M, True)
    for k in ("tokens", "mask", "bias_ids", "bias"):
        a[k][:] = a[k][:1]
    ref, bound, ok = _ref(x, **a)
    wide = torch.zeros(T, V + 5, device="cuda")
    wide[:, 3:3 + V] = torch.from_numpy(x).cuda()
    cu = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    for k in ("tokens", "mask", "bias_ids", "bias"):
        cu[k] = cu[k][:1].expand(T, -1)
    ids = torch.zeros(T, dtype=torch.int64, device="cuda")
    out = torch.zeros(T, V + 1, device="cuda")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        logits.adjust(wide[:, 3:3 + V], out[:, 1:], ids=ids, **cu)
    torch.cuda.synchronize()
    y = out[:, 1:].cpu().numpy()
    _same(y, ref, bound)
    assert ids.tolist() == _pick(y, ok) and not bool(out[:, 0].any())
    assert not bool(wide[:, :3].any()) and not bool(wide[:, 3 + V:].any())
    # captured: the replays follow the device's tensors
    xt, o2 = torch.from_numpy(x).cuda(), torch.empty(T, V, device="cuda")
    full = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    logits.adjust(xt, o2, ids=ids, **full)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        logits.adjust(xt, o2, ids=ids, **full)
    for k in range(3):
        x2, a2 = _case(np.random.default_rng(100 + k), T, V, L, M, True)
        xt.copy_(torch.from_numpy(x2))
        for n, v in a2.items():
            full[n].copy_(torch.from_numpy(v))
        g.replay()
        torch.cuda.synchronize()
        y2, ids2, _ = _run(x2, a2)
        assert np.array_equal(o2.cpu().numpy(), y2) and ids.tolist() == ids2


def test_head_pick_with_rules():
    """Head.pick: the rules between the head and the pick, greedy and sampled."""
    from ai_amd.head import Head
    g = torch.Generator(device="cuda").manual_seed(8)
    V, D, T = 5000, 256, 3
    W = (torch.randn(V, D, device="cuda", generator=g) * 0.05).bfloat16()
    h = torch.randn(T, D, device="cuda", generator=g)
    head = Head(W)
    base = head.pick(h, T)
    lg = (h.double() @ W.double().T).cpu().numpy()
    assert base == np.argmax(lg, 1).tolist()
    words = np.full((T, -(-V // 32)), -1, np.int32)
    words[1, base[1] >> 5] &= ~np.int32(np.uint32(1 << (base[1] & 31)).astype(np.int32))
    words[2] = 0
    rules = {"mask": torch.from_numpy(words).cuda(), "bias_ids": torch.tensor([[17], [-1], [3]], device="cuda"),
             "bias": torch.full((T, 1), 100.0, device="cuda")}
    second = int(np.argsort(lg[1])[-2])
    assert head.pick(h, T, rules=rules) == [17, second, -1]
    got = head.pick(h, T, temperature=0.7, top_p=0.9, rng=np.random.default_rng(0), rules=rules)
    assert got[0] == 17 and got[1] != base[1] and got[2] == -1
    # the ids that a mask allows all at -inf: the smallest of them, sampled too
    words[2, 1] = 0b1010
    rules["mask"] = torch.from_numpy(words).cuda()
    rules["bias_ids"] = torch.tensor([[17, 17], [-1, -1], [33, 35]], device="cuda")
    rules["bias"] = torch.tensor([[0.0, 100.0], [0.0, 0.0], [-np.inf, -np.inf]], device="cuda")
    assert head.pick(h, T, rules=rules) == [17, second, 33]
    assert head.pick(h, T, temperature=0.7, rng=np.random.default_rng(1), rules=rules)[2] == 33
    assert head.pick(h, T) == base


def test_head_pick_sampled_beside_infinite_logits():
    """A bias of +inf forces its id (the smallest of several), sampled too, and a
    NaN logit gives its id, as in the greedy pick; the rows beside keep the draws
    that they have alone."""
    from ai_amd.head import Head
    g = torch.Generator(device="cuda").manual_seed(9)
    V, D, T = 3000, 256, 4
    W = (torch.randn(V, D, device="cuda", generator=g) * 0.05).bfloat16()
    h = torch.randn(T, D, device="cuda", generator=g)
    head = Head(W)
    inf = float("inf")
    rules = {"bias_ids": torch.tensor([[2001, 77], [-1, -1], [5, 9], [8, 1500]], device="cuda"),
             "bias": torch.tensor([[inf, inf], [0.0, 0.0], [inf, -inf], [1.0, float("nan")]], device="cuda")}
    greedy = head.pick(h, T, rules=rules)
    base = head.pick(h, T)
    assert greedy == [77, base[1], 5, 1500]
    alone = {k: v[1:2].contiguous() for k, v in rules.items()}
    want = head.pick(h[1:2], 1, temperature=2.0, rng=np.random.default_rng(3), rules=alone)
    got = head.pick(h, T, temperature=2.0, rng=np.random.default_rng(3), rules=rules)
    assert got == [77, want[0], 5, 1500]


def test_refusals():
    from ai_amd import logits
    T, V = 2, 100
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    x = z(T, V)
    tok, ln, pen = z(T, 5, dtype=torch.int64), z(T, dtype=torch.int32), z(T, 3)
    ok = dict(x=x, tokens=tok, length=ln, penalties=pen)
    logits.adjust(**ok)
    for bad in (dict(x=x.cpu()), dict(x=x.double()), dict(x=x[0]), dict(x=x.t()), dict(out=z(T, V + 1)),
                dict(out=z(1, V).expand(T, V)), dict(tokens=tok.int()), dict(tokens=tok[:1]), dict(tokens=tok.cpu()),
                dict(length=None), dict(length=ln.long()), dict(penalties=None), dict(penalties=pen[:, :2]),
                dict(prompt=ln[:1]), dict(tokens=None), dict(bias_ids=tok), dict(bias=pen),
                dict(bias_ids=tok, bias=z(T, 4)), dict(bias_ids=tok, bias=z(T, 6)[:, :5]), dict(mask=z(T, 3, dtype=torch.int32)),
                dict(mask=z(T, 4, dtype=torch.int64)), dict(mask=z(1, 4, dtype=torch.int32)), dict(ids=ln),
                dict(ids=z(T + 1, dtype=torch.int64))):
        with pytest.raises(ValueError):
            logits.adjust(**{**ok, **bad})
    assert logits.adjust(x[:0]).shape == (0, V)
    torch.cuda.synchronize()

"""What the speed of the operators for serving several requests at once is judged on: one call each, on one GPU.

A case is a dict with an "op":

    append   attn.PagedRopeAttn.append: the head norms and the position rotation of T token rows, their keys and values
             into the pages of their sequences
    attend   attn.PagedRopeAttn.attend: the attention of T token rows over the pages of their sequences
    adjust   logits.adjust: repetition, frequency and presence penalties, biases and grammar masks on the logits of T
             rows, and the greedy pick
    adapt    lora.Adapters.apply: the low-rank adapters of T rows' requests added to a shared projection's output

A row is one token of one request.  With own = False every operator is computed in its plain form, from elementary torch
operations in 32 bits; with own = True by the framework.  The cases' head counts and matrix sizes are those of the
Qwen3 configurations of ai_amd/model.py (tiny is its tiny_config()).
"""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e6
VOCAB = 151936
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HEADS = {"0.6b": (16, 8, 128), "8b": (32, 8, 128), "14b": (40, 8, 128), "32b": (64, 8, 128), "tiny": (8, 4, 64)}
MATRICES = {  # (N, K) of fused projections, and what their input goes through: "norm" RMSNorm, "gate" silu(g) * u
    "0.6b-o": (1024, 2048, ""), "0.6b-qkv": (4096, 1024, "norm"), "8b-qkv": (6144, 4096, "norm"),
    "8b-o": (4096, 4096, ""), "8b-gu": (24576, 4096, "norm"), "8b-down": (4096, 12288, "gate"),
    "14b-qkv": (7168, 5120, "norm"), "14b-down": (5120, 17408, "gate"), "32b-o": (5120, 8192, ""),
}


def listed():
    return [
        # the next token of one short chat, Qwen3-0.6B with the default cache type: the smallest call
        dict(name="append-token", op="append", model="0.6b", kv="f32", page=16, seqs=1, tokens=1, lo=130, hi=130, pad=0),
        # one new token of 61 requests in a pass padded to 64 rows, some of them far into a long context
        dict(name="append-batch64", op="append", model="32b", kv="bf16", page=16, seqs=61, tokens=61, lo=40, hi=120000,
             pad=3),
        # the prompts of three requests at once, one of them behind an earlier turn
        dict(name="append-prompts", op="append", model="8b", kv="bf16", page=64, seqs=3, tokens=4099, lo=1, hi=900, pad=0),
        # the next tokens of 8 short chats, Qwen3-0.6B with the default cache type
        dict(name="attend-chats8", op="attend", model="0.6b", kv="f32", page=16, seqs=8, rows=1, lo=60, hi=700, pad=0),
        # one request with a long context
        dict(name="attend-long", op="attend", model="8b", kv="bf16", page=64, seqs=1, rows=1, lo=32771, hi=32771, pad=0),
        # 8 speculated tokens of one request checked behind a long prompt
        dict(name="attend-verify8", op="attend", model="32b", kv="bf16", page=16, seqs=1, rows=8, lo=4104, hi=4104, pad=0),
        # one new token of 64 requests of very different lengths: the largest attention
        dict(name="attend-batch64", op="attend", model="8b", kv="bf16", page=16, seqs=64, rows=1, lo=500, hi=8200, pad=0),
        # the next token of one chat with a repetition penalty
        dict(name="adjust-chat", op="adjust", vocab=VOCAB, rows=1, lo=230, hi=230, bias=0, mask=False, pick=True),
        # the next tokens of 64 requests: long histories, biases, grammars, and the pick
        dict(name="adjust-batch64", op="adjust", vocab=VOCAB, rows=64, lo=20, hi=6000, bias=32, mask=True, pick=True),
        # one token of one request with a small adapter on the attention output of Qwen3-0.6B
        dict(name="adapt-token", op="adapt", matrix="0.6b-o", rows=1, adapters=4, rank=16, runs=1),
        # 16 requests, most with an adapter of their own, beside the fused qkv of Qwen3-8B
        dict(name="adapt-batch16", op="adapt", matrix="8b-qkv", rows=16, adapters=24, rank=32, runs=13),
        # the prompts of three requests beside gate and up of Qwen3-8B: the largest call
        dict(name="adapt-prompts", op="adapt", matrix="8b-gu", rows=2051, adapters=6, rank=64, runs=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "adjust", "adapt"])
    model, kv, page = rng.choice(sorted(HEADS)), rng.choice(sorted(DTYPES)), rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        seqs = _log(rng, 1, 64)
        return dict(op=op, model=model, kv=kv, page=page, seqs=seqs, tokens=max(seqs, _log(rng, 1, 2000)),
                    lo=rng.randint(1, 50), hi=_log(rng, 50, 20000), pad=rng.choice([0, 0, rng.randint(1, 5)]))
    if op == "attend":
        rows = rng.choice([1, 1, 1, rng.randint(2, 16)])
        seqs = _log(rng, 1, 64) if rows == 1 else _log(rng, 1, 6)
        hi = _log(rng, 20, min(32768, 80000 // (seqs * rows)))
        return dict(op=op, model=model, kv=kv, page=page, seqs=seqs, rows=rows, lo=max(rows, _log(rng, 1, hi)),
                    hi=max(rows, hi), pad=rng.choice([0, 0, rng.randint(1, 5)]))
    if op == "adjust":
        hi = _log(rng, 1, 6000)
        return dict(op=op, vocab=_log(rng, 1000, VOCAB), rows=_log(rng, 1, 64), lo=rng.randint(0, hi), hi=hi,
                    bias=rng.choice([0, rng.randint(1, 300)]), mask=rng.random() < 0.6, pick=rng.random() < 0.7)
    rows = _log(rng, 1, 1200)
    return dict(op=op, matrix=rng.choice(sorted(MATRICES)), rows=rows, adapters=rng.randint(1, 24),
                rank=rng.choice([4, 8, 16, 24, 32, 64, 128]), runs=rng.randint(1, min(rows, 24)))


# ------------------------------------------------------------------------------------------------ sizes of a case
def _spread(lo, hi, n):
    """n lengths from lo to hi, evenly over their logarithm."""
    if n == 1:
        return [hi]
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * i / (n - 1)))) - 1 for i in range(n)]


def _shares(total, n):
    """total rows shared out over n sequences, every one at least one and later ones more."""
    extra = total - n
    s = [1 + extra * 2 * i // (n * (n - 1)) if n > 1 else total for i in range(n)]
    s[-1] += total - sum(s)
    return s


def _lengths(case):
    """(cached length after the call, rows of the call) per sequence."""
    if case["op"] == "append":
        new = _shares(case["tokens"], case["seqs"])
        return [(a + b, b) for a, b in zip(_spread(case["lo"], case["hi"], case["seqs"]), new)]
    return [(max(n, case["rows"]), case["rows"]) for n in _spread(case["lo"], case["hi"], case["seqs"])]


def work(case):
    op = case["op"]
    if op in ("append", "attend"):
        H, KV, HD = HEADS[case["model"]]
        eb = 2 if case["kv"] == "bf16" else 4
        lens = _lengths(case)
        T = sum(r for _, r in lens)
        row = T * 12
        if op == "append":
            return {"bytes": row + T * ((H + 2 * KV) * HD * 4 + H * HD * 4 + 2 * KV * HD * eb), "flops": T * (H + KV) * HD * 8}
        kv = sum(n for n, _ in lens) * KV * HD * 2 * eb
        pages = sum(-(-n // case["page"]) * 4 for n, _ in lens)
        seen = sum(r * n - r * (r - 1) // 2 for n, r in lens)
        return {"bytes": row + kv + pages + 2 * T * H * HD * 4, "flops": 4 * seen * H * HD}
    if op == "adjust":
        V, T = case["vocab"], case["rows"]
        hist = sum(_spread(case["lo"], case["hi"], T))
        return {"bytes": T * (8 * V + 12 * case["bias"] + (-(-V // 32) * 4 if case["mask"] else 0) + 20) + hist * 8,
                "flops": 4 * T * V}
    N, K, pro = MATRICES[case["matrix"]]
    T, R = case["rows"], case["rank"]
    used = min(case["runs"], case["adapters"])
    return {"bytes": T * K * 4 * (2 if pro == "gate" else 1) + 2 * T * N * 4 + used * R * (N + K) * 2 + T * 4,
            "flops": 2 * T * R * (N + K)}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    return {"append": _prepare_pages, "attend": _prepare_pages, "adjust": _prepare_adjust,
            "adapt": _prepare_adapt}[case["op"]](case, seed)


def _prepare_pages(case, seed):
    g = _gen(seed)
    H, KV, HD = HEADS[case["model"]]
    page, dt = case["page"], DTYPES[case["kv"]]
    lens = _lengths(case)
    need = [-(-n // page) for n, _ in lens]
    # append: the pages that the call does not write are left out of the pool (their ids are other requests')
    if case["op"] == "append":
        first = [(n - r) // page for n, r in lens]
    else:
        first = [0] * len(lens)
    used = sum(n - f for n, f in zip(need, first))
    n_pages = used + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu().tolist()
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for i, (n, f) in enumerate(zip(need, first)):
        table[i, f:n] = torch.tensor(ids[at:at + n - f], dtype=torch.int32)
        at += n - f
    rows = [(i, n - r + j) for i, (n, r) in enumerate(lens) for j in range(r)]
    seq = torch.tensor([i for i, _ in rows] + [-1] * case["pad"], dtype=torch.int32, device="cuda")
    pos = torch.tensor([p for _, p in rows] + [0] * case["pad"], dtype=torch.int64, device="cuda")
    T = len(rows) + case["pad"]
    # what a cache holds: normed and rotated keys (about 1 each), projected values; old tokens in the unused slots
    pool = (n_pages, KV, page, HD)
    s = SimpleNamespace(op=case["op"], H=H, KV=KV, HD=HD, page=page, seq=seq, pos=pos, table=table.cuda(),
                        kc=_randn(g, *pool).to(dt), vc=_randn(g, *pool).mul_(0.7).to(dt), scale=HD ** -0.5)
    if case["op"] == "append":
        s.qkv = _randn(g, T, (H + 2 * KV) * HD).mul_(1.5)
        s.qn = 1 + 0.2 * _randn(g, HD)
        s.kn = 1 + 0.2 * _randn(g, HD)
        s.inv = (1.0 / (THETA ** (torch.arange(0, HD, 2, dtype=torch.float32) / HD))).cuda()
        s.q = torch.empty(T, H * HD, device="cuda")
    else:
        # queries that follow some positions more than others: scores of a few units
        s.q = _randn(g, T, H * HD).mul_(2.0)
        s.out = torch.empty(T, H * HD, device="cuda")
    if own:
        from ai_amd.attn import PagedRopeAttn
        s.handle = PagedRopeAttn(H, KV, HD, page, dt, EPS)
    return s


def _prepare_adjust(case, seed):
    g = _gen(seed)
    V, T, M = case["vocab"], case["rows"], case["bias"]
    s = SimpleNamespace(op="adjust", V=V, T=T)
    s.x = _randn(g, T, V).mul_(2.5)
    s.out = torch.empty_like(s.x)
    L = max(1, case["hi"])
    # text: few ids often, many seldom
    u = torch.rand(T, L, generator=g, device="cuda")
    s.tokens = (V ** u - 1).long().clamp_(0, V - 1)
    order = torch.randperm(T, generator=g, device="cuda")
    s.length = torch.tensor(_spread(case["lo"], case["hi"], T), dtype=torch.int32, device="cuda")[order]
    s.prompt = (s.length * torch.rand(T, generator=g, device="cuda")).to(torch.int32)
    p = torch.stack([1 + 0.4 * torch.rand(T, generator=g, device="cuda"), 0.5 * torch.rand(T, generator=g, device="cuda"),
                     0.8 * torch.rand(T, generator=g, device="cuda")], 1)
    if T > 1:
        p[::5] = torch.tensor([1.0, 0.0, 0.0], device="cuda")  # requests without penalties
    s.penalties = p.contiguous()
    s.bias_ids = s.bias = s.mask = s.ids = None
    if M:
        # ids of one row all differ; -1 ends a shorter list
        step = V // M
        s.bias_ids = (torch.arange(M, device="cuda") * step)[None, :] + torch.randint(0, step, (T, M), generator=g,
                                                                                     device="cuda")
        s.bias_ids[1::3, M // 2:] = -1
        s.bias = _randn(g, T, M).mul_(3.0)
    if case["mask"]:
        W = -(-V // 32)
        words = torch.zeros(T, W, dtype=torch.int32, device="cuda")
        for r in range(T):
            if r % 3 == 2:
                words[r] = -1  # a request without a grammar
            else:  # a state that allows most tokens, or few
                keep = 0.9 if r % 3 == 0 else 0.002
                bits = torch.rand(W, 32, generator=g, device="cuda") < keep
                words[r] = (bits.long() << torch.arange(32, device="cuda")).sum(1).to(torch.int32)
        s.mask = words
    if case["pick"]:
        s.ids = torch.empty(T, dtype=torch.int64, device="cuda")
    return s


def _prepare_adapt(case, seed):
    g = _gen(seed)
    N, K, pro = MATRICES[case["matrix"]]
    T, L, R = case["rows"], case["adapters"], case["rank"]
    s = SimpleNamespace(op="adapt", T=T, N=N, K=K, L=L)
    chan = torch.where(torch.rand(K, generator=g, device="cuda") < 0.005, 10.0, 1.0)
    if pro == "gate":
        s.x = torch.cat([_randn(g, T, K), _randn(g, T, K) * chan], 1)
    else:
        s.x = _randn(g, T, K) * chan
    s.mode = 2 if pro == "gate" else 0
    s.lnw = (1 + 0.1 * _randn(g, K)).bfloat16() if pro == "norm" else None
    s.A = _randn(g, L, R, K).mul_(K ** -0.5).bfloat16()
    s.B = _randn(g, L, N, R).mul_(0.02).bfloat16()
    s.scale = 0.5 + 2 * torch.rand(L, generator=g, device="cuda")
    # the rows of a request follow each other; of several requests one has no adapter
    which = torch.randperm(max(L, case["runs"]), generator=g, device="cuda")[:case["runs"]] % L
    if case["runs"] > 2:
        which[1] = -1
    s.idx = which.repeat_interleave(torch.tensor(_shares(T, case["runs"]), device="cuda")).to(torch.int32)
    s.y = _randn(g, T, N)
    s.out = torch.empty_like(s.y)
    if own:
        from ai_amd.lora import Adapters
        s.handle = Adapters(s.A, s.B, s.scale)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "attend": _plain_attend, "adjust": _plain_adjust, "adapt": _plain_adapt}[s.op](s)


def _own(s):
    if s.op == "append":
        s.handle.append(s.qkv, s.qn, s.kn, s.inv, s.seq, s.pos, s.table, s.kc, s.vc, s.q)
        return {"q": s.q, "kc": s.kc, "vc": s.vc}
    if s.op == "attend":
        s.handle.attend(s.q, s.seq, s.pos, s.table, s.kc, s.vc, s.out)
        return s.out
    if s.op == "adjust":
        from ai_amd import logits
        logits.adjust(s.x, s.out, tokens=s.tokens, length=s.length, prompt=s.prompt, penalties=s.penalties,
                      bias_ids=s.bias_ids, bias=s.bias, mask=s.mask, ids=s.ids)
        return {"logits": s.out} if s.ids is None else {"logits": s.out, "ids": s.ids}
    s.handle.apply(s.x, s.y, s.idx, mode=s.mode, lnw=s.lnw, eps=EPS, out=s.out)
    return s.out


def _rms(x, w):
    return w * (x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS))


def _plain_append(s):
    H, KV, HD, page = s.H, s.KV, s.HD, s.page
    T = s.qkv.shape[0]
    live = s.seq >= 0
    x = s.qkv.view(T, H + 2 * KV, HD)
    qk = torch.cat([_rms(x[:, :H], s.qn), _rms(x[:, H:H + KV], s.kn)], 1)
    ang = s.pos.double()[:, None] * s.inv.double()[None, :]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    a, b = qk[..., :HD // 2], qk[..., HD // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    torch.mul(qk[:, :H].reshape(T, H * HD), live[:, None], out=s.q)
    n, P = s.table.shape
    # padding rows write nothing: they repeat the first row, which is no padding
    seq = torch.where(live, s.seq, s.seq[0]).long()
    pos = torch.where(live, s.pos, s.pos[0])
    src = torch.where(live, torch.arange(T, device=seq.device), 0)
    pg = s.table.view(-1)[seq * P + pos // page].long()
    s.kc[pg, :, pos % page] = qk[:, H:].to(s.kc.dtype)[src]
    s.vc[pg, :, pos % page] = x[:, H + KV:].to(s.vc.dtype)[src]
    return {"q": s.q, "kc": s.kc, "vc": s.vc}


def _plain_attend(s):
    H, KV, HD, page = s.H, s.KV, s.HD, s.page
    T = s.q.shape[0]
    live = s.seq >= 0
    n, P = s.table.shape
    tab = s.table[s.seq.clamp(min=0).long()]  # [T, P]
    pg = tab.clamp(min=0).long()
    K = s.kc[pg].float().permute(0, 2, 1, 3, 4).reshape(T * KV, P * page, HD)
    q = s.q.view(T * KV, H // KV, HD)
    sc = torch.bmm(q, K.transpose(1, 2).contiguous()).view(T, KV, H // KV, P * page) * s.scale
    del K
    at = torch.arange(P * page, device=pg.device)
    see = (at[None, :] <= s.pos[:, None]) & live[:, None] & (tab >= 0).repeat_interleave(page, 1)
    sc = sc.masked_fill(~see[:, None, None, :], -math.inf)
    m = sc.amax(-1, keepdim=True)
    e = (sc - m.clamp(min=torch.finfo(torch.float32).min)).exp()
    del sc
    V = s.vc[pg].float().permute(0, 2, 1, 3, 4).reshape(T * KV, P * page, HD)
    o = torch.bmm(e.view(T * KV, H // KV, P * page), V).view(T, KV, H // KV, HD)
    den = e.sum(-1, keepdim=True)
    o = o / torch.where(den > 0, den, torch.ones_like(den))
    return torch.mul(o.reshape(T, H * HD), live[:, None], out=s.out)


def _plain_adjust(s):
    V, T = s.V, s.T
    L = s.tokens.shape[1]
    at = torch.arange(L, device="cuda")[None, :]
    in_ctx = at < s.length[:, None]
    gen = in_ctx & (at >= s.prompt[:, None])
    count = torch.zeros(T, V, dtype=torch.int32, device="cuda").scatter_add_(1, s.tokens, gen.int())
    seen = torch.zeros(T, V, dtype=torch.int32, device="cuda").scatter_add_(1, s.tokens, in_ctx.int()) > 0
    r, f, p = (s.penalties[:, i:i + 1] for i in range(3))
    y = torch.where(seen, torch.where(s.x > 0, s.x / r, s.x * r), s.x)
    y = y - (f * count + p * (count > 0))
    if s.bias is not None:
        used = s.bias_ids >= 0
        y = y.scatter_add(1, s.bias_ids.clamp(min=0), torch.where(used, s.bias, torch.zeros_like(s.bias)))
    allowed = None
    if s.mask is not None:
        allowed = ((s.mask[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool()
        allowed = allowed.view(T, -1)[:, :V]
        y = torch.where(allowed, y, torch.full_like(y, -math.inf))
    s.out.copy_(y)
    if s.ids is None:
        return {"logits": s.out}
    top = y.amax(1, keepdim=True)
    ids = torch.arange(V, device="cuda")[None, :]
    hit = (y == top) if allowed is None else (y == top) & allowed
    pick = torch.where(hit, ids, V).amin(1)
    s.ids.copy_(torch.where(pick < V, pick, -1))
    return {"logits": s.out, "ids": s.ids}


def _plain_adapt(s):
    x = s.x
    if s.mode == 2:
        gate, up = x[:, :s.K], x[:, s.K:]
        x = gate / (1 + torch.exp(-gate)) * up
    if s.lnw is not None:
        x = _rms(x, s.lnw.float())
    s.out.copy_(s.y)
    for a in range(s.L):  # every adapter for every row: no row's adapter is known to the host
        mine = (s.idx == a)[:, None]
        h = torch.mm(x, s.A[a].float().t()) * s.scale[a]
        s.out += torch.mm(torch.where(mine, h, torch.zeros_like(h)), s.B[a].float().t())
    return s.out


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "adjust": _exact_adjust, "adapt": _exact_adapt}[s.op](s)


def _exact_append(s):
    H, KV, HD = s.H, s.KV, s.HD
    x = s.qkv.double().view(-1, H + 2 * KV, HD)
    q = torch.zeros(len(x), H * HD, dtype=torch.float64, device="cuda")
    kc, vc = s.kc.double(), s.vc.double()
    norm = x / (x.square().sum(-1, keepdim=True) / HD + EPS).sqrt()
    turn = torch.polar(torch.ones_like(s.inv, dtype=torch.float64)[None, :].expand(len(x), -1),
                       s.pos.double()[:, None] * s.inv.double())[:, None, :]
    rot = lambda h, w: torch.view_as_real(torch.complex(*(h * w.double()).chunk(2, -1)) * turn).transpose(-1, -2).flatten(-2)
    qr, kr = rot(norm[:, :H], s.qn), rot(norm[:, H:H + KV], s.kn)
    rows = (s.seq >= 0).nonzero().squeeze(1)
    q[rows] = qr[rows].flatten(1)
    page = s.table[s.seq[rows].long(), torch.div(s.pos[rows], s.page, rounding_mode="floor")].long()
    slot = s.pos[rows] % s.page
    kc[page, :, slot] = kr[rows]
    vc[page, :, slot] = x[rows, H + KV:]
    return {"q": q, "kc": kc, "vc": vc}


def _exact_attend(s):
    H, KV, HD = s.H, s.KV, s.HD
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for r, (i, p) in enumerate(zip(s.seq.tolist(), s.pos.tolist())):
        if i < 0:
            continue
        pages = s.table[i, :p // s.page + 1].long()
        k, v = (c[pages].double().transpose(0, 1).reshape(KV, -1, HD)[:, :p + 1] for c in (s.kc, s.vc))
        z = (s.q[r].double().view(KV, H // KV, 1, HD) * k[:, None]).sum(-1) * s.scale if p < 64 else \
            torch.matmul(s.q[r].double().view(KV, H // KV, HD), k.transpose(1, 2)) * s.scale
        w = torch.exp(z - z.max(-1, keepdim=True).values)
        out[r] = (torch.matmul(w, v) / w.sum(-1, keepdim=True)).flatten()
    return out


def _exact_adjust(s):
    y = s.x.cpu().numpy().astype(np.float64)
    tok, length, prompt = s.tokens.cpu().numpy(), s.length.cpu().numpy(), s.prompt.cpu().numpy()
    pen = s.penalties.cpu().numpy().astype(np.float64)
    ids = np.empty(s.T, np.int64)
    for r in range(s.T):
        past = tok[r, :length[r]]
        seen = np.unique(past)
        y[r, seen] = np.where(y[r, seen] > 0, y[r, seen] / pen[r, 0], y[r, seen] * pen[r, 0])
        made, times = np.unique(past[prompt[r]:], return_counts=True)
        y[r, made] -= pen[r, 1] * times + pen[r, 2]
        if s.bias is not None:
            b = s.bias_ids[r].cpu().numpy()
            y[r, b[b >= 0]] += s.bias[r].cpu().numpy().astype(np.float64)[b >= 0]
        ok = np.ones(s.V, bool)
        if s.mask is not None:
            ok = np.unpackbits(s.mask[r].cpu().numpy().view(np.uint8), bitorder="little")[:s.V].astype(bool)
            y[r, ~ok] = -np.inf
        cand = np.flatnonzero(ok)
        ids[r] = cand[np.argmax(y[r, cand])] if len(cand) else -1
    y = torch.from_numpy(y)
    return {"logits": y} if s.ids is None else {"logits": y, "ids": torch.from_numpy(ids)}


def _exact_adapt(s):
    out = s.y.double()
    for r0 in range(0, s.T, 256):
        x = s.x[r0:r0 + 256].double()
        if s.mode == 2:
            x = x[:, :s.K] * torch.sigmoid(x[:, :s.K]) * x[:, s.K:]
        if s.lnw is not None:
            x = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * s.lnw.double()
        idx = s.idx[r0:r0 + 256]
        for a in sorted(set(idx.tolist()) - {-1}):
            rows = (idx == a).nonzero().squeeze(1)
            out[r0 + rows] += (x[rows] @ s.A[a].double().T) @ s.B[a].double().T * s.scale[a].double()
    return out

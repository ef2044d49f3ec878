"""Several requests served together: passes of 16 rows that mix prompt chunks, new
tokens and padding, over a paged cache (attn.PagedRopeAttn), with each request's
own adapters beside the shared 12-bit linears (lora.Adapters) and its own rules at
the pick (logits.adjust), captured as one HIP graph, against the float32 oracle of
each request alone (the adapters merged into its weights)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, PAGE = 16, 16


class _Merged:
    """A checkpoint whose layers have one adapter of every matrix added, in float32."""

    def __init__(self, ck, deltas):
        self.__dict__.update(ck.__dict__)
        self.ck, self.deltas = ck, deltas

    def t(self, *a):
        return self.ck.t(*a)

    def head_name(self):
        return self.ck.head_name()

    def layer(self, i, device="cpu"):
        w = self.ck.layer(i, device)
        return {k: v.float() + self.deltas[i][k].to(device) if k in self.deltas[i] else v for k, v in w.items()}


class _Server:
    """The passes' fixed buffers and the model's parts, in a user's own loop."""

    def __init__(self, ck, kv, n_pages):
        from ai_amd import wcomp
        from ai_amd.attn import PagedRopeAttn
        from ai_amd.lora import Adapters
        self.ck = ck
        g = torch.Generator(device="cuda").manual_seed(11)
        z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
        D, H, KV, HD, FF, V = ck.D, ck.H, ck.KV, ck.HD, ck.FF, ck.V
        self.inv = (1.0 / (ck.theta ** (torch.arange(0, HD, 2, dtype=torch.float32) / HD))).cuda()
        self.emb, self.norm = ck.t("model.embed_tokens.weight", "cuda"), ck.t("model.norm.weight", "cuda")
        self.head = wcomp.compress(ck.t(ck.head_name(), "cuda"))
        self.W, self.small, self.ad, self.kc, self.vc, self.deltas = [], [], [], [], [], [[], []]
        for i in range(ck.L):
            w = ck.layer(i, "cuda")
            self.W.append({n: wcomp.compress(w[n]) for n in ("qkv", "o", "gu", "down")})
            self.small.append({k: w[k] for k in ("ln1", "ln2")} | {k: w[k].float() for k in ("qn", "kn")})
            ads = {}
            for n in ("qkv", "o", "down"):
                N, K = w[n].shape
                pairs = [((torch.randn(r, K, device="cuda", generator=g) * K ** -0.5).bfloat16(),
                          (torch.randn(N, r, device="cuda", generator=g) * 0.05).bfloat16(), 2.0 * r) for r in (8, 5)]
                ads[n] = Adapters.from_pairs(pairs)
                for a, (A, B, _) in enumerate(pairs):
                    if len(self.deltas[a]) <= i:
                        self.deltas[a].append({})
                    self.deltas[a][i][n] = (2.0 * B.double() @ A.double()).float().cpu()
            self.ad.append(ads)
            self.kc.append(z(n_pages, KV, PAGE, HD, dtype=kv))
            self.vc.append(z(n_pages, KV, PAGE, HD, dtype=kv))
        self.attn = PagedRopeAttn(H, KV, HD, PAGE, kv, ck.eps)
        self.tok, self.pos = z(ROWS, dtype=torch.int64), z(ROWS, dtype=torch.int64)
        self.seq, self.idx = z(ROWS, dtype=torch.int32), z(ROWS, dtype=torch.int32)
        self.x, self.qkv, self.att, self.gu = z(ROWS, D), z(ROWS, (H + 2 * KV) * HD), z(ROWS, H * HD), z(ROWS, 2 * FF)
        self.lg, self.ids = z(ROWS, V), z(ROWS, dtype=torch.int64)
        self.hist, self.length, self.prompt = z(ROWS, 64, dtype=torch.int64), z(ROWS, dtype=torch.int32), z(ROWS, dtype=torch.int32)
        self.pen, self.mask = z(ROWS, 3), z(ROWS, -(-V // 32), dtype=torch.int32)
        self.bias_ids, self.bias = z(ROWS, 2, dtype=torch.int64), z(ROWS, 2)
        self.raw = z(ROWS, V)
        self.graph = None

    def _pass(self):
        from ai_amd import logits, wcomp
        eps = self.ck.eps
        self.x.copy_(self.emb.index_select(0, self.tok).float())
        for l, W in enumerate(self.W):
            s, ad = self.small[l], self.ad[l]
            wcomp.gemvc_tc(self.x, W["qkv"], self.qkv, 0, ROWS, lnw=s["ln1"], eps=eps)
            ad["qkv"].apply(self.x, self.qkv, self.idx, lnw=s["ln1"], eps=eps)
            self.attn(self.qkv, s["qn"], s["kn"], self.inv, self.seq, self.pos, self.table, self.kc[l], self.vc[l], self.att)
            # (the adapters first: both add to x)
            ad["o"].apply(self.att, self.x, self.idx, mode=1)
            wcomp.gemvc_tc(self.att, W["o"], self.x, 1, ROWS)
            wcomp.gemvc_tc(self.x, W["gu"], self.gu, 0, ROWS, lnw=s["ln2"], eps=eps)
            ad["down"].apply(self.gu, self.x, self.idx, mode=2)
            wcomp.gemvc_tc(self.gu, W["down"], self.x, 2, ROWS)
        wcomp.greedy(self.x, self.head, ROWS, self.ids, lnw=self.norm, eps=eps, logits=self.raw)
        logits.adjust(self.raw, self.lg, tokens=self.hist, length=self.length, prompt=self.prompt, penalties=self.pen,
                      bias_ids=self.bias_ids, bias=self.bias, mask=self.mask, ids=self.ids)

    def run(self):
        if self.graph is None:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                self._pass()
            torch.cuda.current_stream().wait_stream(s)
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self._pass()
        self.graph.replay()
        torch.cuda.synchronize()


@pytest.mark.parametrize("kv", [torch.float32, torch.bfloat16])
def test_requests_together_match_the_oracle_of_each_alone(kv):
    from ai_amd.model import RandomCkpt, tiny_config
    from oracle import qwen3
    ck = RandomCkpt(tiny_config(layers=2, vocab=1003), seed=3)
    s = _Server(ck, kv, n_pages=14)
    rng = np.random.default_rng(5)
    V, new = ck.V, 6
    prompts = [rng.integers(0, V, n).tolist() for n in (5, 37, 17)]
    adapter = [0, -1, 1]
    pen = np.float32([[1.3, 0.2, 0.4], [1.0, 0.0, 0.0], [0.9, -0.1, 0.3]])
    bias = [{7: 2.0, 11: -3.0}, {}, {500: 0.5}]
    allowed = np.ones((3, V), bool)
    allowed[1, rng.permutation(V)[:700]] = False
    words = np.packbits(np.pad(allowed, ((0, 0), (0, -V % 32))), axis=1, bitorder="little").view(np.int32)
    ids = rng.permutation(14).tolist()
    table = np.full((3, 4), -1, np.int32)
    for r, p in enumerate(prompts):
        for j in range(-(-(len(p) + new) // PAGE)):
            table[r, j] = ids.pop()
    s.table = torch.from_numpy(table).cuda()
    fed, text, made = [0, 0, 0], [list(p) for p in prompts], [[], [], []]
    passes = 0
    while any(len(t) - len(p) < new for t, p in zip(text, prompts)):
        rows = []
        for r in rng.permutation(3).tolist():
            if len(text[r]) - len(prompts[r]) >= new:
                continue
            while fed[r] < len(text[r]) and len(rows) < ROWS:
                rows.append((r, fed[r]))
                fed[r] += 1
        last = {r: i for i, (r, p) in enumerate(rows) if p == len(text[r]) - 1}
        pad = ROWS - len(rows)
        cu = lambda a, t: torch.tensor(a, dtype=t.dtype)
        s.tok.copy_(cu([text[r][p] for r, p in rows] + [0] * pad, s.tok))
        s.pos.copy_(cu([p for _, p in rows] + [0] * pad, s.pos))
        s.seq.copy_(cu([r for r, _ in rows] + [-1] * pad, s.seq))
        s.idx.copy_(cu([adapter[r] for r, _ in rows] + [-1] * pad, s.idx))
        s.mask.fill_(-1)
        s.length.zero_()
        s.bias_ids.fill_(-1)
        s.pen.copy_(torch.tensor([[1.0, 0.0, 0.0]] * ROWS))
        for r, i in last.items():
            s.hist[i, :len(text[r])] = torch.tensor(text[r], device="cuda")
            s.length[i], s.prompt[i] = len(text[r]), len(prompts[r])
            s.pen[i] = torch.from_numpy(pen[r]).cuda()
            s.mask[i] = torch.from_numpy(words[r]).cuda()
            for j, (n, b) in enumerate(bias[r].items()):
                s.bias_ids[i, j], s.bias[i, j] = n, b
        s.run()
        passes += 1
        for r, i in last.items():
            made[r].append((s.raw[i].cpu().numpy(), s.lg[i].cpu().numpy(), int(s.ids[i])))
            text[r].append(int(s.ids[i]))
        assert not bool(s.att[len(rows):].any())  # padding rows
    assert passes < 30
    for r in range(3):
        ref = qwen3.logits(_Merged(ck, s.deltas[adapter[r]]) if adapter[r] >= 0 else ck, text[r][:-1], kv_dtype=kv).numpy()
        for k, (raw, lg, pick) in enumerate(made[r]):
            want = ref[len(prompts[r]) - 1 + k]
            # two layers of float32 sums in another order (a bf16 cache: keys that
            # round to the other neighbour, 2^-8 of a key's size in some scores)
            tol = (2e-4 if kv == torch.float32 else 2e-2) * np.abs(want).max()
            assert np.abs(raw - want).max() <= tol, (r, k, np.abs(raw - want).max(), tol)
            past = text[r][:len(prompts[r]) + k]
            y = raw.astype(np.float64)
            for n in set(past):
                y[n] = y[n] / pen[r, 0] if y[n] > 0 else y[n] * pen[r, 0]
                c = past[len(prompts[r]):].count(n)
                if c:
                    y[n] -= pen[r, 1] * c + pen[r, 2]
            for n, b in bias[r].items():
                y[n] += b
            y[~allowed[r]] = -np.inf
            fin = np.isfinite(y)
            assert np.array_equal(np.isfinite(lg), fin) and np.allclose(lg[fin], y[fin], rtol=1e-6, atol=1e-6)
            assert pick == int(np.argmax(lg)) and allowed[r, pick]

"""The operators of many sequences at once as they are used together: a paged cache that is appended to and read, drafted tokens
that are verified and rolled back, and a step that trains the drafting model."""
import math

import numpy as np
import pytest

from test_distill import reference as distill_reference
from test_paged import E4M3, F32, Batch, numpy_of
from test_verify import probabilities, reference as verify_reference

GPU = pytest.mark.gpu
V, H, HKV, DH, PAGE, DRAFTS = 300, 4, 2, 36, 16, 4


class Model:
    """Embeddings straight to queries, keys and values, attention over what there is, an output matrix."""

    def __init__(self, r, bits, B, W, out_std):
        import torch
        from cacti_amd import ops
        self.bits, self.B, self.W, self.T = bits, B, W, 0
        self.table = r.permutation(B * W + 1)[:B * W].reshape(B, W).astype(np.int32)
        self.emb = r.standard_normal((V, (H + 2 * HKV) * DH)).astype(np.float16)
        self.out = (r.standard_normal((H * DH, V)) * out_std).astype(np.float16)
        self.cache = ops.paged_cache(B * W + 1, HKV, PAGE, DH, dtype=torch.float8_e4m3fn if bits == 8 else torch.float16)
        self.cos, self.sin = ops.rope_tables(W * PAGE, DH)
        self.d = {k: torch.from_numpy(np.ascontiguousarray(getattr(self, k))).cuda() for k in ("table", "emb", "out")}
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(self, tok, starts, lens, max_new):
        """Device tensors in, device tensors out: attention [T, H, Dh] and logits [T, V] of the rows."""
        from cacti_amd import ops
        qkv = self.d["emb"][tok]
        q, k, v = qkv[:, :H * DH].view(-1, H, DH), qkv[:, H * DH:(H + HKV) * DH].view(-1, HKV, DH), qkv[:, (H + HKV) * DH:].view(-1, HKV, DH)
        where = (self.d["table"], starts, lens)
        q = ops.paged_append(k, v, self.cache, *where, self.cos, self.sin, q=q, max_new=max_new, status=self.status)
        o = ops.paged_attention(q, self.cache, *where, 1 / math.sqrt(DH), max_new=max_new, status=self.status)
        return q, o, ops.gemm(o.view(-1, H * DH), self.d["out"])

    def run(self, rows, lens):
        """rows: each sequence's new tokens; lens with them."""
        import torch
        n = [len(x) for x in rows]
        dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        tok = torch.tensor(sum(rows, []), device="cuda")
        return self.step(tok, dev([0] + list(np.cumsum(n))), dev(lens), max(n))

    def check(self, q, o, n, lens, kept, growths):
        """The attention of rows of `n` new tokens against 64 bits on what is in the cache, and the cache against the tokens."""
        b = Batch.__new__(Batch)
        b.n, b.lens, b.H, b.Hkv, b.Dh, b.page, b.bits, b.B = n, lens, H, HKV, DH, PAGE, self.bits, self.B
        b.Dp, b.table, b.alpha, b.cos, b.sin = (DH + 15) // 16 * 16, self.table, 1 / math.sqrt(DH), self.cos.cpu().numpy(), self.sin.cpu().numpy()
        b.starts = np.concatenate([[0], np.cumsum(n)])
        cache = [None if x is None else numpy_of(x) for x in self.cache]
        want, tol = b.attend(q.cpu().numpy(), cache)
        off = np.abs(o.cpu().numpy().astype(np.float64) - want) / tol
        assert off.max() <= 1, "attention: %.2f of the bound" % off.max()
        for s in range(self.B):
            K, X = b.dense(s, cache)
            for p, x in enumerate(kept[s][:lens[s]]):
                row = self.emb[x]
                k, v = b.rotated(row[H * DH:(H + HKV) * DH].reshape(HKV, DH), p), row[(H + HKV) * DH:].reshape(HKV, DH).astype(F32)
                for got, true, scale in ((K[p], k, cache[2]), (X[p], v, cache[3])):
                    if self.bits == 16:
                        assert np.array_equal(got, true.astype(np.float16).astype(np.float64))
                    else:
                        # half a step of a code (2^-4 of it), and 2^-10 of the scale for each time that a small one was coded
                        step = scale[self.table[s, p // PAGE]].astype(np.float64)[:, None]
                        assert (np.abs(got - true) <= 2.0 ** -4 * np.abs(true) * (1 + 2.0 ** -20) + growths * 2.0 ** -10 * step).all()


@GPU
@pytest.mark.parametrize("bits,captured", [(16, False), (8, False), (8, True)])
def test_draft_and_verify(bits, captured):
    """Prompts, then rounds of drafted tokens that are kept or not: every round the tokens are those that the reference takes from
    the same logits, the cache holds the tokens that were kept, and the attention is that over them."""
    import torch
    from cacti_amd import ops
    r = np.random.default_rng(40 + bits)
    prompts, rounds, W = [list(r.integers(0, V, n)) for n in (37, 5, 80)], 5, 7
    B = len(prompts)
    target, draft = Model(r, bits, B, W, 0.12), Model(r, bits, B, W, 0.12)
    # the drafting model is near the target model
    draft.emb, draft.d["emb"] = target.emb, target.d["emb"]
    draft.out = (target.out + r.standard_normal(target.out.shape) * 0.02).astype(np.float16)
    draft.d["out"] = torch.from_numpy(draft.out).cuda()
    dev = lambda x, t=torch.int32: torch.tensor(np.asarray(x).tolist(), dtype=t, device="cuda")
    u16 = lambda x: torch.from_numpy(np.asarray(x).astype(np.uint16).view(np.int16)).cuda()
    # the first token behind each prompt: verification of rows without drafted tokens
    kept = [list(p) for p in prompts]
    lens = [len(p) for p in kept]
    q, o, z = target.run(kept, lens)
    target.check(q, o, [len(p) for p in prompts], lens, kept, 1)
    draft.run(kept, lens)
    z0 = z[torch.tensor(np.cumsum(lens) - 1, device="cuda")].contiguous()
    rand = r.random(B).astype(np.float32)
    a, nxt = ops.verify_draft(z0, None, u16([p[-1] for p in kept]), dev(range(B + 1)), dev(np.zeros(B), torch.float32), dev(rand, torch.float32))
    wa, wn = verify_reference(z0.cpu().numpy(), None, np.zeros(B, int), np.arange(B + 1), np.zeros(B, F32), rand, 1.0)
    assert not a.any() and np.array_equal(nxt.cpu().numpy().view(np.uint16), wn)
    for s in range(B):
        kept[s].append(int(wn[s]))
    drafted_upto = list(lens)                                # positions that are in the drafting model's cache
    # a verification step that is captured once and replayed: everything that changes is in these
    T = B * (DRAFTS + 1)
    tok_d, len_d, u_d, r_d = torch.zeros(T, dtype=torch.int64, device="cuda"), dev(lens), torch.zeros(T, device="cuda"), torch.zeros(B, device="cuda")
    draft_d, starts_d = torch.zeros((T, V), dtype=torch.float16, device="cuda"), dev(np.arange(B + 1) * (DRAFTS + 1))

    def verification():
        q, o, z = target.step(tok_d, starts_d, len_d, DRAFTS + 1)
        return q, o, z, *ops.verify_draft(z, draft_d, tok_d.to(torch.int16), starts_d, u_d, r_d)

    graph, outs = None, None
    seen = set()
    for k in range(rounds):
        # drafted tokens, one after another; where all were kept the last one is not in the drafting model's cache yet
        drafts, draft_logits = [[] for _ in range(B)], np.zeros((B, DRAFTS + 1, V), np.float16)
        for i in range(DRAFTS):
            rows = [(kept[s] + drafts[s])[drafted_upto[s]:] for s in range(B)]
            assert all(len(x) in (1, 2) for x in rows)
            ln = [len(kept[s]) + len(drafts[s]) for s in range(B)]
            z = draft.run(rows, ln)[2].cpu().numpy()
            for s in range(B):
                drafted_upto[s] = ln[s]
                draft_logits[s, i] = z[sum(len(x) for x in rows[:s + 1]) - 1]
                drafts[s].append(int(r.choice(V, p=probabilities(draft_logits[s, i], 1.0))))
        tok = np.array([[kept[s][-1]] + drafts[s] for s in range(B)])
        lens = [len(kept[s]) + DRAFTS for s in range(B)]
        u, rr = r.random(T).astype(np.float32), r.random(B).astype(np.float32)
        tok_d.copy_(torch.from_numpy(tok.reshape(-1)))
        len_d.copy_(dev(lens))
        u_d.copy_(torch.from_numpy(u))
        r_d.copy_(torch.from_numpy(rr))
        draft_d.copy_(torch.from_numpy(draft_logits.reshape(T, V)))
        if captured and graph is None:
            outs = verification()                            # (appending the same rows again changes nothing)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = verification()
        if captured:
            graph.replay()
            torch.cuda.synchronize()
        else:
            outs = verification()
        q, o, z, a, nxt = outs
        wa, wn = verify_reference(z.cpu().numpy(), draft_logits.reshape(T, V), tok.reshape(-1), np.arange(B + 1) * (DRAFTS + 1), u, rr, 1.0)
        a, nxt = a.cpu().numpy(), nxt.cpu().numpy().view(np.uint16).reshape(B, -1)
        assert np.array_equal(a, wa) and np.array_equal(nxt.reshape(-1), wn)
        full = [kept[s] + drafts[s] for s in range(B)]
        target.check(q, o, [DRAFTS + 1] * B, lens, full, 2 * k + 4)
        for s in range(B):
            seen.add(int(a[s]))
            kept[s] += [int(x) for x in nxt[s, :a[s] + 1]]
            # the caches go back by their lengths alone
            drafted_upto[s] = min(drafted_upto[s], len(kept[s]) - 1)
    assert int(target.status) == 0 and int(draft.status) == 0
    assert len(seen) > 1, "kept %s drafted tokens everywhere" % seen
    # without any rejected token between: the same tokens appended at once
    if bits == 16:
        fresh = Model(r, bits, B, W, 0.12)
        fresh.emb, fresh.d["emb"], fresh.out, fresh.d["out"] = target.emb, target.d["emb"], target.out, target.d["out"]
        ln = [len(x) for x in kept]
        q, o, z = fresh.run(kept, ln)
        fresh.check(q, o, ln, ln, kept, 1)


@GPU
def test_training_of_the_drafting_model():
    """The gradient of its output matrix for the target model's top logits, through both operators and the product before them."""
    import torch
    from cacti_amd import ops
    r = np.random.default_rng(50)
    B, W, K, temp = 2, 8, 12, 2.0
    target, draft = Model(r, 16, B, W, 0.12), Model(r, 8, B, W, 0.1)
    rows = [list(r.integers(0, V, n)) for n in (70, 113)]
    lens = [len(x) for x in rows]
    N = sum(lens)
    zt = target.run(rows, lens)[2]
    _, x, z = draft.run(rows, lens)
    val, idx = torch.topk(zt, K, dim=1)
    ids = idx.to(torch.int16)
    loss, stats = ops.distill_topk_fwd(z, ids, val, temp)
    scale = torch.full((N,), 1.0 / N, device="cuda")
    dz = ops.distill_topk_bwd(z, ids, val, stats, scale, temp)
    dw = ops.gemm(x.view(N, H * DH), dz, ta=True)
    wl, wg, tl, tg = distill_reference(z.cpu().numpy(), idx.cpu().numpy(), val.cpu().numpy(), scale.cpu().numpy(), temp)
    assert (np.abs(loss.cpu().numpy() - wl) <= tl).all()
    assert (np.abs(dz.cpu().numpy().astype(np.float64) - wg) <= tg).all()
    xx = x.view(N, H * DH).cpu().numpy().astype(np.float64)
    want = xx.T @ wg
    # the rounded gradient's bound through the product, N sums in fp32 and the rounding of the result
    tol = np.abs(xx).T @ tg + 2.0 ** -24 * N * (np.abs(xx).T @ np.abs(wg)) + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    off = np.abs(dw.cpu().numpy().astype(np.float64) - want) / tol
    assert off.max() <= 1, "gradient of the matrix: %.2f of the bound" % off.max()

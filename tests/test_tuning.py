"""Tuning by answers as a program runs it: prompts whose answers share their pages, requests' adapters beside the shared projections, the answers'
log-probabilities, and the losses over them back to the adapters' gradients.

Answers: a cache in which sequences share, hand back and pack pages holds for each of them what a cache of its own would, bit for bit, so
every number of every step has to be equal to that of a run in which each sequence has its own pages and a fork copies them whole.
Gradients: against float64, from the f16 logits that the kernels formed.  dA and dB are sums of products with the loss's gradient; its error (bounded as where the loss
is tested by itself) goes through them by the sums' absolute values, and to that comes the adapters' own bound for the gradient
which they were given."""
import numpy as np
import pytest

from test_adapter import Case, near
from test_answers import dev, gradient64, pairs64, policy64, policy_inputs, rows64

GPU = pytest.mark.gpu
D, H, HKV, DH, V, PAGE, W = 64, 4, 2, 24, 304, 16, 6


class Model:
    def __init__(self, seed, dtype):
        import torch
        from cacti_amd import ops
        r = np.random.default_rng(seed)
        h = lambda *s, std: dev((r.standard_normal(s) * std).astype(np.float16))
        self.embed, self.q, self.k, self.v, self.out = h(V, D, std=1), h(D, H * DH, std=0.2), h(D, HKV * DH, std=0.2), h(D, HKV * DH, std=0.2), h(H * DH, V, std=0.5)
        self.qA, self.qB, self.oA, self.oB = h(3, 8, D, std=0.2), h(3, H * DH, 8, std=0.3), h(3, 16, H * DH, std=0.2), h(3, V, 16, std=0.3)
        self.scale = torch.tensor([1.0, -0.5, 2.0], device="cuda")
        self.cos, self.sin = ops.rope_tables(PAGE * W, DH)
        self.dtype = torch.float16 if dtype == 16 else torch.float8_e4m3fn

    def run(self, cache, table, tok, starts, lens, ids, most, status):
        from cacti_amd import ops
        T = tok.shape[0]
        x = self.embed[tok.long()]
        q = ops.gemm(x, self.q)
        q, _ = ops.adapter_fwd(x, self.qA, self.qB, starts, ids, self.scale, base=q, out=q, max_new=most, status=status)
        k, v = ops.gemm(x, self.k), ops.gemm(x, self.v)
        q = ops.paged_append(k.view(T, HKV, DH), v.view(T, HKV, DH), cache, table, starts, lens, self.cos, self.sin, q=q.view(T, H, DH), max_new=most, status=status)
        o = ops.paged_attention(q, cache, table, starts, lens, DH ** -0.5, max_new=most, status=status).view(T, H * DH)
        z = ops.gemm(o, self.out)
        return ops.adapter_fwd(o, self.oA, self.oB, starts, ids, self.scale, base=z, out=z, max_new=most, status=status)[0]


class Answers:
    """Up to B sequences; shared: their pages come from one pool."""

    def __init__(self, model, B, shared):
        import torch
        from cacti_amd import ops
        self.m, self.B, self.shared = model, B, shared
        P = B * W - 3 if shared else B * W
        self.cache = ops.paged_cache(P, HKV, PAGE, DH, dtype=model.dtype)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.table = i32(B, W) - 1 if shared else torch.arange(B * W, dtype=torch.int32, device="cuda").view(B, W)
        self.refs, self.lens, self.status = i32(P), i32(B), i32(1)

    def fork(self, parent):
        import torch
        from cacti_amd import ops
        if self.shared:
            self.table, self.lens = ops.paged_fork(self.refs, self.table, self.lens, parent, PAGE, status=self.status)
            return
        to = torch.where(parent >= 0, parent, 0).long()
        self.cache = tuple(c if c is None else c.view(torch.uint8).view(self.B, -1)[to].view(c.dtype).view(c.shape) for c in self.cache)
        self.lens = torch.where(parent >= 0, self.lens[to], 0)

    def grow(self, lens):
        """Room for lens positions, behind those that are there; 0: the sequence's pages go back."""
        import torch
        from cacti_amd import ops
        if self.shared:
            moves = ops.paged_fit(self.refs, self.table, torch.minimum(self.lens, lens), lens, PAGE, status=self.status)
            ops.paged_copy([self.cache], *moves)
        self.lens = lens

    def pack(self):
        from cacti_amd import ops
        if self.shared:
            src, dst, used = ops.paged_compact(self.refs, self.table)
            ops.paged_copy([self.cache], src, dst)
            assert int(used) == int((self.refs > 0).sum()) and not bool((self.refs[int(used):] > 0).any())


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def course(bits, shared):
    """All logits and log-probabilities of some prompts, three answers each, a search among them, sequences that end, and others' pages packed."""
    import torch
    from cacti_amd import ops
    r = np.random.default_rng(1)
    a, out = Answers(Model(2, bits), 9, shared), []
    prompts, ids = [5, 16, 37], [0, 0, 0, -1, -1, -1, 2, 2, 2]
    new = [prompts[b // 3] if b % 3 == 0 else 0 for b in range(9)]
    a.grow(ints(new))
    tok = dev(r.integers(0, V, sum(new)))
    starts = np.concatenate([[0], np.cumsum(new)])
    out.append(a.m.run(a.cache, a.table, tok, ints(starts), a.lens, ints(ids), 37, a.status))
    a.fork(ints([0, 0, 0, 3, 3, 3, 6, 6, 6]))
    if shared:
        assert int((a.refs > 0).sum()) == 1 + 1 + 3 and int(a.refs.max()) == 3
    alive = list(range(9))
    tok = dev(r.integers(0, V, 9))
    for step in range(24):
        if step in (6, 13):                    # the best of each three goes on as others
            a.fork(ints([1, 1, 2, 3, 5, 5, 6, 6, 6] if step == 6 else [0, 2, 2, 4, 4, 4, 7, 7, 8]))
        if step == 17:
            alive = [0, 3, 4, 8]
        if step == 18:
            a.pack()
        more = [int(b in alive) for b in range(9)]
        lens = torch.where(ints(more) > 0, a.lens + 1, 0)
        if step < 17 or shared:
            a.grow(lens)
        else:
            a.lens = lens
        starts = ints(np.concatenate([[0], np.cumsum(more)]))
        tok = tok[:len(alive)]
        z = a.m.run(a.cache, a.table, tok, starts, a.lens, ints(ids), 1, a.status)
        drawn = (z.float() + dev(r.gumbel(size=(len(alive), V)).astype(np.float32))).argmax(1).to(torch.int16)
        logp, stats = ops.token_logp_fwd(z, drawn, 0.8)
        out += [z, drawn, logp, stats]
        tok = drawn
    assert int(a.status) == 0
    if shared:
        held = torch.zeros_like(a.refs)
        at = a.table[a.table >= 0].long()
        held.index_add_(0, at, torch.ones_like(at, dtype=torch.int32))
        assert torch.equal(held, a.refs)
    return out


@GPU
@pytest.mark.parametrize("bits", [8, 16])
def test_answers_that_share_pages_are_those_that_do_not(bits):
    import torch
    want, got = course(bits, False), course(bits, True)
    assert len(want) == len(got)
    for i, (x, y) in enumerate(zip(got, want)):
        assert torch.isfinite(x.float()).all() and torch.equal(x, y), i


@GPU
def test_a_step_of_an_answer_captured_and_replayed():
    """Pages, copies, cache, adapters and log-probabilities in one graph, whose lengths, tokens and tables go on from replay to replay; every step
    against the same without a graph."""
    import torch
    from cacti_amd import ops
    m = Model(3, 8)
    prompts, ids = [30, 0, 0, 47, 0], ints([1, 1, 1, -1, -1])
    r = np.random.default_rng(4)
    text, noise = dev(r.integers(0, V, sum(prompts))), dev(r.gumbel(size=(5, V)).astype(np.float32))

    def begin():
        a = Answers(m, 5, True)
        a.grow(ints(prompts))
        m.run(a.cache, a.table, text, ints(np.concatenate([[0], np.cumsum(prompts)])), a.lens, ids, 47, a.status)
        a.fork(ints([0, 0, 0, 3, 3]))
        return a, torch.zeros(5, dtype=torch.int16, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda")

    def step(a, tok, starts):
        lens = a.lens + 1
        moves = ops.paged_fit(a.refs, a.table, a.lens, lens, PAGE, status=a.status)
        ops.paged_copy([a.cache], *moves)
        a.lens.copy_(lens)
        z = m.run(a.cache, a.table, tok, starts, a.lens, ids, 1, a.status)
        tok.copy_((z.float() + noise).argmax(1))
        return [z, *moves, *ops.token_logp_fwd(z, tok)]

    eager, first = begin(), begin()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*begin())
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*first)
    for i in range(20):
        g.replay()
        want = step(*eager)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i
        assert torch.equal(first[0].table, eager[0].table) and torch.equal(first[0].refs, eager[0].refs) and torch.equal(first[1], eager[1])
    assert int(first[0].status) == 0 and int(eager[0].status) == 0


def adapters_within(c, h, dz, tol, got):
    """dx, dA and dB of adapters whose gradient dz (float64) the kernels have to within tol; c.dy is theirs."""
    given = c.adjoint(h, False)                # for theirs: the adapters' own bounds
    dy, c.dy = c.dy, dz
    want = c.adjoint(h, False)
    c.dy = dy
    through = [np.zeros(w.shape) for w, _ in want]
    for a in range(c.n):
        at = c.rows(a)
        x, A, B, s = np.abs(c.x[at].astype(np.float64)), np.abs(c.A[a].astype(np.float64)), np.abs(c.B[a].astype(np.float64)), abs(float(c.scale[a]))
        dh = tol[at] @ B
        through[0][at], through[1][a], through[2][a] = s * dh @ A, s * dh.T @ x, s * tol[at].T @ np.abs(h[at].astype(np.float64))
    used = slice(0, int(c.starts[-1]))
    for g, (w, _), (_, t), more, what in zip(got, want, given, through, ("dx", "dA", "dB")):
        rows = used if what == "dx" else slice(None)
        near(g[rows], w[rows], (t + more)[rows], what)


@GPU
@pytest.mark.parametrize("counts,ids,K,N,R", [([5, 1, 20, 3, 9, 2], [0, 0, 1, 2, -1, 1], 72, 304, 16), ([100, 90, 41, 70], [2, 1, 0, 2], 136, 1000, 8),
                                              ([1] * 8, [0, 1, 2, 0, 1, 2, 0, 1], 64, 40, 64)])
@pytest.mark.parametrize("loss", ["policy", "pairs"])
def test_losses_back_to_adapters(counts, ids, K, N, R, loss):
    """Projection, adapters, loss and back, with a step of the optimiser, and the whole of it captured."""
    import torch
    from cacti_amd import ops
    print(loss, len(counts), K, N, R, flush=True)
    c = Case(K + N, counts, ids, K, N, R, 3)
    r = np.random.default_rng(5)
    x, A, B, starts, ids, scale = c.of("x A B starts ids scale")
    proj = dev((r.standard_normal((K, N)) * K ** -0.5 * 2).astype(np.float16))
    tok = r.integers(0, N, c.T)

    def logits():
        z = ops.gemm(x, proj)
        return ops.adapter_fwd(x, A, B, starts, ids, scale, base=z, out=z, max_new=max(counts))

    z16 = logits()[0].cpu().numpy()
    old, adv, ref, weight = policy_inputs(r, z16, tok, 1.3)
    if loss == "policy":
        args = [dev(v) for v in (tok, old, adv, weight)]

        def back(z):
            return ops.policy_loss(z, *args, ref=dref, beta=0.05, temperature=1.3)
    else:
        weight = weight[:len(counts) // 2]
        dtok, dweight = dev(tok), dev(weight)

        def back(z):
            logp, stats = ops.token_logp_fwd(z, dtok, 1.3)
            l, reward, d = ops.preference_loss(logp, dref, starts, dweight, 0.13, 0.1)
            return l, logp, ops.token_logp_bwd(z, dtok, stats, d, 1.3)
    dref = dev(ref)
    state = [[torch.zeros_like(p, dtype=torch.float32) for p in (A, B)] for _ in range(2)]
    masters, params = [p.float() for p in (A, B)], [A.clone(), B.clone()]
    scalars = ops.adamw32_scalars(1, 1.0, 1e-3, 0.1, 0.1, 0.01, 1e-8)

    def step():
        z, h = logits()
        l, logp, dz = back(z)
        grads = ops.adapter_bwd(x, A, B, starts, ids, scale, h, dz, max_new=max(counts))
        ops.adamw32_step_(list(grads[1:]), *state, masters, params, scalars)
        return [z, h, l, logp, dz, *grads]

    z, h, l, logp, dz, *grads = step()
    assert np.array_equal(z.cpu().numpy(), z16)
    if loss == "policy":
        wl, tl, wp, tp, wz, tz = policy64(z16, tok, old, adv, ref, weight, 0.2, 0.2, 0.05, 1.3)
        near(l, wl, tl, "loss")
        near(logp, wp, tp, "logp")
    else:
        logs, wp, rel, tp = rows64(z16, tok, 1.3)
        near(logp, wp, tp, "logp")
        got = logp.cpu().numpy()
        wl, reward, d = pairs64(got, ref, c.starts, weight, 0.13, 0.1, None, False)
        near(l, wl, 2.0 ** -24 * np.abs(wl) + 1e-12, "loss")
        wz, tz = gradient64(logs, tok, d / 1.3, np.abs(d) / 1.3 * 2.0 ** -22, rel)
    near(dz, wz, tz, "gradient of the logits")
    c.dy = dz.cpu().numpy()
    adapters_within(c, h.cpu().numpy(), wz, tz, grads)
    for p, was, m in zip(params, (A, B), masters):
        assert torch.isfinite(m).all() and torch.equal(p, m.half()) and not torch.equal(p, was)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i in range(4):
        x.copy_(torch.roll(x, 3, 0))
        g.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want)), i


@GPU
def test_two_graphs_and_another_stream():
    """Two captured steps and one on a stream of its own, one after the other and in turn: each has its own workspaces."""
    import torch
    from cacti_amd import ops
    cases = [Case(20 + i, counts, [0, 1, -1, 1], 8640 if i == 1 else 136, 264, 32, 2) for i, counts in enumerate(([5, 9, 2, 1], [40, 1, 7, 3], [300, 2, 90, 11]))]
    r = np.random.default_rng(6)
    steps = []
    for c in cases:
        x, A, B, starts, ids, scale, base = c.of("x A B starts ids scale base")
        tok, old, adv, weight = dev(r.integers(0, 264, c.T)), dev(np.full(c.T, -5, np.float32)), dev(r.standard_normal(c.T).astype(np.float32)), dev(np.ones(c.T, np.float32))

        def step(x=x, A=A, B=B, starts=starts, ids=ids, scale=scale, base=base, tok=tok, old=old, adv=adv, weight=weight, most=max(c.counts)):
            z, h = ops.adapter_fwd(x, A, B, starts, ids, scale, base=base, max_new=most)
            loss, logp, dz = ops.policy_loss(z, tok, old, adv, weight)
            return [z, h, loss, logp, dz, *ops.adapter_bwd(x, A, B, starts, ids, scale, h, dz, max_new=most)]
        steps.append(step)
    want = [[t.clone() for t in step()] for step in steps]
    torch.cuda.synchronize()
    graphs, got = [], []
    for step in steps[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(step())
    side = torch.cuda.Stream()
    for i in range(6):
        with torch.cuda.stream(side):
            third = steps[2]()
        graphs[i % 2].replay()
        graphs[(i + 1) % 2].replay()
        if i % 2:
            for t in got[0] + got[1]:
                t.fill_(3)
            torch.cuda.synchronize()
            graphs[0].replay(), graphs[1].replay()
        torch.cuda.synchronize()
        for g, w in zip(got + [third], want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


@GPU
@pytest.mark.parametrize("bits", [8, 16])
def test_a_step_that_pages_run_out_in_and_the_same_step_again(bits):
    """Three answers to a prompt whose last page is not full, and a single page that is free: one goes on, nothing is written on the page that
    the others share, and with pages free again they go on as answers do that have their own."""
    import torch
    m, ids = Model(4, bits), ints([0, -1, 2])
    r = np.random.default_rng(7)
    text, tok = dev(r.integers(0, V, 20)), dev(r.integers(0, V, 3))
    a, b = Answers(m, 3, True), Answers(m, 3, False)
    for k in (a, b):
        k.grow(ints([20, 0, 0]))
        m.run(k.cache, k.table, text, ints([0, 20, 20, 20]), k.lens, ids, 20, k.status)
        k.fork(ints([0, 0, 0]))
    a.refs[3:] += 1                            # (of somebody else)
    b.grow(ints([21, 21, 21]))
    want = m.run(b.cache, b.table, tok, ints([0, 1, 2, 3]), b.lens, ids, 1, b.status)
    a.grow(ints([21, 21, 21]))
    bits_of = lambda: [x.view(torch.uint8)[1].clone() for x in a.cache if x is not None]
    assert int(a.status) == 3 and a.table[:, 1].tolist() == [-3, 2, -3] and a.refs[:3].tolist() == [3, 2, 1]
    before = bits_of()
    z = m.run(a.cache, a.table, tok, ints([0, 1, 2, 3]), a.lens, ids, 1, a.status)
    assert torch.equal(z[1], want[1]) and all(torch.equal(x, y) for x, y in zip(bits_of(), before))
    a.status.zero_()
    a.lens = ints([20, 21, 20])
    a.refs[3:5] -= 1
    a.grow(ints([21, 21, 21]))
    z = m.run(a.cache, a.table, tok[[0, 2]].contiguous(), ints([0, 1, 1, 2]), a.lens, ids, 1, a.status)
    assert torch.equal(z, want[[0, 2]]) and int(a.status) == 0
    assert a.table[:, 1].tolist() == [1, 2, 3] and a.refs[:5].tolist() == [3, 1, 1, 1, 0]

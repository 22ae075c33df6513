"""Tuning a model by its own answers: the operators as cases that can be timed and compared.

  policy   clipped policy loss with a KL term of sampled tokens, and its gradient (ops.policy_loss)
  prefer   loss over pairs of answers, of which one is preferred, and its gradient (ops.token_logp_fwd, preference_loss,
           token_logp_bwd)
  adapt    low-rank adapters of many requests beside a shared projection (ops.adapter_fwd)
  tune     their gradients (ops.adapter_bwd)
  pages    several answers that share a prompt's pages in the cache, and a cache that is packed (ops.paged_fork, paged_fit,
           paged_copy, paged_compact)

`own` chooses between the framework's operators and their plain form in elementary torch operations.
"""
import math
import random

import torch

own = False

F8 = torch.float8_e4m3fn
F16 = torch.float16
I32 = torch.int32


def listed():
    return [
        # answers of a tiny model, few tokens
        dict(name="policy_tiny", kind="policy", N=192, V=1024, skip=0.25, ref=True, clip=0.2, beta=0.04, temp=1.0),
        # the benchmark's head, a third of the rows prompts
        dict(name="policy_3b", kind="policy", N=2048, V=32000, skip=0.3, ref=True, clip=0.2, beta=0.04, temp=1.0),
        # pairs of short answers, an odd vocabulary, means over the tokens
        dict(name="prefer_odd", kind="prefer", pairs=2, longest=150, V=8191, skip=0.3, mean=True, smoothing=0.1),
        # pairs of answers, the benchmark's vocabulary
        dict(name="prefer_3b", kind="prefer", pairs=2, longest=600, V=32000, skip=0.4, mean=False, smoothing=0.0),
        # a chat's next token, one adapter, the benchmark's width
        dict(name="adapt_one", kind="adapt", S=1, new=1, ragged=False, K=3200, N=3200, R=16, n=4, base=True),
        # a batch of chats with a few drafted tokens each, a dozen adapters
        dict(name="adapt_chats", kind="adapt", S=64, new=5, ragged=True, K=3200, N=3200, R=16, n=12, base=True),
        # prompts through the wide projection, larger adapters
        dict(name="adapt_prompts", kind="adapt", S=4, new=1024, ragged=True, K=3200, N=8640, R=64, n=3, base=True),
        # one adapter of a small model, texts of odd length
        dict(name="tune_small", kind="tune", S=3, new=203, ragged=True, K=1024, N=2816, R=8, n=1),
        # a batch of texts, some adapters in training at once
        dict(name="tune_3b", kind="tune", S=8, new=512, ragged=False, K=3200, N=3200, R=16, n=3),
        # a search over four answers to each of two prompts
        dict(name="pages_search", kind="pages", op="fork", B=8, G=4, lo=300, hi=900, H=32, Dh=100, page=64, bits=8, L=2),
        # eight answers to each prompt of a batch, all go on from the best one
        dict(name="pages_answers", kind="pages", op="fork", B=128, G=8, lo=200, hi=1500, H=8, Dh=128, page=32, bits=8, L=4),
        # a cache with pages all over it, packed so that it can shrink
        dict(name="pages_pack", kind="pages", op="compact", B=40, G=1, lo=200, hi=3000, H=8, Dh=128, page=64, bits=16, L=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_weight(c) for c in listed())
    while True:
        c = _draw(rng)
        if _weight(c) <= most and (c["kind"] != "pages" or _pool(c) * _page_bytes(c) < 2e9):
            return c


def _weight(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


_SIDES = [(256, 256), (256, 688), (1024, 1024), (1024, 2816), (2816, 1024), (2048, 2048), (3200, 3200), (3200, 8640), (8640, 3200)]
_HEADS = [(4, 64), (8, 64), (32, 100), (8, 100), (16, 128), (8, 128), (1, 128), (2, 36)]


def _draw(rng):
    kind = rng.choice(["policy", "prefer", "adapt", "adapt", "tune", "pages"])
    if kind == "policy":
        return dict(kind=kind, N=_log(rng, 1, 2048), V=_log(rng, 500, 60000), skip=rng.choice([0.0, round(rng.uniform(0, 0.9), 2)]),
                    ref=rng.random() < 0.7, clip=round(rng.uniform(0.05, 0.3), 2), beta=round(rng.uniform(0.0, 0.2), 3),
                    temp=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)]))
    if kind == "prefer":
        return dict(kind=kind, pairs=_log(rng, 1, 32), longest=_log(rng, 2, 1000), V=_log(rng, 500, 60000), skip=round(rng.uniform(0, 0.8), 2),
                    mean=rng.random() < 0.3, smoothing=rng.choice([0.0, 0.1]))
    if kind in ("adapt", "tune"):
        K, N = rng.choice(_SIDES)
        c = dict(kind=kind, S=_log(rng, 1, 64), new=rng.choice([1, rng.randint(2, 9), _log(rng, 10, 1200)]), ragged=rng.random() < 0.7, K=K, N=N,
                 R=rng.choice([8, 16, 16, 24, 32, 64, 128]), n=_log(rng, 1, 16))
        return dict(c, base=rng.random() < 0.7) if kind == "adapt" else c
    H, Dh = rng.choice(_HEADS)
    op = rng.choice(["fork", "fork", "compact"])
    G = rng.choice([1, 2, 4, 8]) if op == "fork" else 1
    lo = _log(rng, 2, 1000)
    return dict(kind=kind, op=op, B=G * _log(rng, 1, 24), G=G, lo=lo, hi=lo + _log(rng, 1, 2000), H=H, Dh=Dh, page=rng.choice([16, 32, 64, 128]),
                bits=rng.choice([8, 8, 16]), L=rng.randint(1, 4))


# ---------------------------------------------------------------- sizes that go by the case alone
def _counts(number, most, ragged):
    """Rows of each sequence: all the same, or 1 .. most in a fixed shuffle with the largest among them."""
    if not ragged:
        return [most] * number
    r = random.Random(7 * number + most)
    n = [most] + [r.randint(1, most) for _ in range(number - 1)]
    r.shuffle(n)
    return n


def _texts(case):
    return _counts(2 * case["pairs"], case["longest"], True)


def _masked(n, skip):
    """The first rows of a text that are not the model's own; its last row is."""
    return min(int(n * skip), n - 1)


def _lens(case):
    """Positions of each sequence: those of a group have their prompt in common, and answers of a length each."""
    B, G, lo, hi = (case[x] for x in ("B", "G", "lo", "hi"))
    r = random.Random(13 * B + hi)
    prompts = [int(round(math.exp(r.uniform(math.log(lo), math.log(hi))))) for _ in range(B // G)]
    return prompts, [prompts[b // G] + (r.randint(1, max(1, lo // 2)) if G > 1 else 0) for b in range(B)]


def _winner(case, group):
    return group * case["G"] + random.Random(17 * group + case["hi"]).randrange(case["G"])


NEW = 3                                        # positions that a search goes on by


def _pool(case):
    """Pages of the cache: for a search those of its sequences and as many as they may come to need, for one that is packed 2.5 times
    as many as are held."""
    prompts, lens = _lens(case)
    page, G = case["page"], case["G"]
    held = sum(-(-x // page) for x in lens) - sum(p // page * (G - 1) for p in prompts)
    return held + 2 * case["B"] + 8 if case["op"] == "fork" else int(held / 0.4) + 4


def _page_bytes(case):
    return case["H"] * case["page"] * (-(-case["Dh"] // 16) * 16) * 2 * case["bits"] // 8 * case["L"]


def work(case):
    if case["kind"] == "policy":
        N, V = case["N"], case["V"]
        used = N - _masked(N, case["skip"])
        return dict(bytes=2 * V * (used + N) + 24 * N, flops=8 * used * V)
    if case["kind"] == "prefer":
        n, V = _texts(case), case["V"]
        used = sum(x - _masked(x, case["skip"]) for x in n)
        return dict(bytes=2 * V * (2 * used + sum(n)) + 24 * sum(n), flops=8 * used * V)
    if case["kind"] in ("adapt", "tune"):
        T, K, N, R = sum(_counts(case["S"], case["new"], case["ragged"])), case["K"], case["N"], case["R"]
        weights = min(case["n"], case["S"]) * R * (K + N)
        if case["kind"] == "adapt":
            return dict(bytes=2 * (T * (K + N * (2 if case["base"] else 1)) + weights) + 4 * T * R, flops=2 * T * R * (K + N))
        return dict(bytes=2 * (T * (2 * K + N) + 2 * weights) + 4 * T * R, flops=4 * T * R * (K + N))
    page, at = case["page"], _page_bytes(case) // case["page"]
    prompts, lens = _lens(case)
    held = sum(-(-x // page) for x in lens)
    if case["op"] == "fork":
        slots = sum((lens[_winner(case, g)] % page) * (case["G"] - 1) for g in range(len(prompts)))
        return dict(bytes=2 * slots * at + 12 * held, flops=0)
    moved = held * (1 - 0.4)                   # of the pages that lie all over a pool of which they are 0.4
    return dict(bytes=int(2 * moved * page * at) + 12 * held, flops=0)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=F16).mul_(std)


def _ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def _starts(n):
    s = [0]
    for x in n:
        s.append(s[-1] + x)
    return _ints(s)


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    _PREPARE[case["kind"]](case, g, st)
    return st


def _sampled(g, st, N, V, temp):
    """Logits as a model gives them, tokens that were drawn from its probabilities some steps ago, and log-probabilities of then
    and of the model that it began as."""
    logit = torch.randn((N, V), generator=g, device="cuda").mul_(2.5)
    noise = torch.rand((N, V), generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)
    tok = (logit / temp - torch.log(-torch.log(noise))).argmax(dim=1)
    st["logit"] = logit.to(F16)
    logp = torch.log_softmax(st["logit"].float() / temp, dim=1).gather(1, tok[:, None])[:, 0]
    st["tok"] = tok.to(torch.int16)                                                    # u16 bit patterns
    st["old"] = logp + 0.15 * torch.randn(N, generator=g, device="cuda")
    st["ref"] = logp + 0.4 * torch.randn(N, generator=g, device="cuda")


def _prepare_policy(case, g, st):
    N = case["N"]
    _sampled(g, st, N, case["V"], case["temp"])
    st["adv"] = torch.randn(N, generator=g, device="cuda")
    st["mask"] = torch.arange(N, device="cuda") >= _masked(N, case["skip"])
    st["scale"] = torch.full((N,), 1024.0 / N, device="cuda")
    if not case["ref"]:
        st["ref"] = None


def _prepare_prefer(case, g, st):
    n = _texts(case)
    _sampled(g, st, sum(n), case["V"], 1.0)
    st["starts"] = _starts(n)
    st["mask"] = torch.tensor([i >= _masked(x, case["skip"]) for x in n for i in range(x)], device="cuda")
    st["scale"] = torch.full((case["pairs"],), 1024.0 / case["pairs"], device="cuda")


def _prepare_adapters(case, g, st):
    S, K, N, R, n = (case[x] for x in ("S", "K", "N", "R", "n"))
    counts = _counts(S, case["new"], case["ragged"])
    T = sum(counts)
    st["x"] = _randn(g, T, K)
    st["A"], st["B"] = _randn(g, n, R, K, std=K ** -0.5), _randn(g, n, N, R, std=0.1)
    st["scale"] = 2.0 ** torch.randint(-2, 2, (n,), generator=g, device="cuda").float()
    # (each adapter that there are sequences for has one; in larger batches some sequences have none)
    ids = torch.randint(-1 if S > 4 else 0, n, (S,), generator=g, device="cuda").to(I32)
    st["ids"], st["starts"], st["max_new"] = ids, _starts(counts), case["new"]
    if case["kind"] == "adapt":
        st["base"] = _randn(g, T, N) if case["base"] else None
    else:
        st["dy"] = _randn(g, T, N, std=0.1)
        # what the forward pass leaves: x A^T of each row's adapter
        a = torch.repeat_interleave(ids.long(), torch.tensor(counts, device="cuda"))
        h = torch.matmul(st["x"].float(), st["A"].float().view(n * R, K).t()).view(T, n, R)
        st["h"] = h.gather(1, a.clamp(min=0)[:, None, None].expand(T, 1, R))[:, 0].mul_((a >= 0)[:, None]).contiguous()


def _prepare_pages(case, g, st):
    """A cache whose sequences' pages lie all over it: prompts' whole pages shared by a group, the rest a sequence's own."""
    B, G, H, Dh, page, L = (case[x] for x in ("B", "G", "H", "Dh", "page", "L"))
    prompts, lens = _lens(case)
    r = random.Random(int(torch.randint(1 << 30, (1,), generator=g, device="cuda")))
    W = -(-(max(lens) + NEW) // page) + 1
    P = _pool(case)
    order = r.sample(range(P), P)
    table, refs = [[-1] * W for _ in range(B)], [0] * P
    for b in range(B):
        shared = prompts[b // G] // page if G > 1 else 0
        for j in range(-(-lens[b] // page)):
            table[b][j] = table[b // G * G][j] if j < shared and b % G else order.pop()
            refs[table[b][j]] += 1
    st["table"], st["refs"], st["lens"], st["page"] = _ints(table), _ints(refs), _ints(lens), page
    # every group goes on from one of its sequences; one group in nine is done
    st["parent"] = _ints([_winner(case, b // G) if b // G % 9 != 8 else -1 for b in range(B)])
    Dp = -(-Dh // 16) * 16
    st["caches"] = []
    for _ in range(L):
        k, v = (_randn(g, P, H, page, Dp) for _ in range(2))
        if case["bits"] == 16:
            st["caches"].append((k, v, None, None))
        else:
            ks, vs = (torch.exp2(torch.randint(-7, -4, (P, H), generator=g, device="cuda").float()) for _ in range(2))
            st["caches"].append((k.mul_(48).clamp_(-448, 448).to(F8), v.mul_(48).clamp_(-448, 448).to(F8), ks, vs))


_PREPARE = dict(policy=_prepare_policy, prefer=_prepare_prefer, adapt=_prepare_adapters, tune=_prepare_adapters, pages=_prepare_pages)


# ---------------------------------------------------------------- one pass
def run(st):
    return _RUN[st["case"]["kind"]](st)


def _policy(st):
    case = st["case"]
    if own:
        from cacti_amd import ops
        return ops.policy_loss(st["logit"], st["tok"], st["old"], st["adv"], st["scale"], ref=st["ref"], mask=st["mask"],
                               clip=(case["clip"], case["clip"]), beta=case["beta"], temperature=case["temp"])
    return _plain_policy(st)


BETA = 0.1                                     # of the preference loss


def _prefer(st):
    case = st["case"]
    if own:
        from cacti_amd import ops
        logp, stats = ops.token_logp_fwd(st["logit"], st["tok"], mask=st["mask"])
        loss, reward, dlogp = ops.preference_loss(logp, st["ref"], st["starts"], st["scale"], beta=BETA, smoothing=case["smoothing"],
                                                  mask=st["mask"], mean=case["mean"])
        return logp, loss, reward, ops.token_logp_bwd(st["logit"], st["tok"], stats, dlogp)
    return _plain_prefer(st)


def _adapt(st):
    if own:
        from cacti_amd import ops
        return ops.adapter_fwd(st["x"], st["A"], st["B"], st["starts"], st["ids"], st["scale"], base=st["base"], max_new=st["max_new"])
    return _plain_adapt(st)


def _tune(st):
    if own:
        from cacti_amd import ops
        return ops.adapter_bwd(st["x"], st["A"], st["B"], st["starts"], st["ids"], st["scale"], st["h"], st["dy"], max_new=st["max_new"])
    return _plain_tune(st)


def _pages(st):
    if st["case"]["op"] == "fork":
        return _fork(st)
    refs, table = st["refs"].clone(), st["table"].clone()     # (so that there is something to pack the next time)
    if own:
        from cacti_amd import ops
        src, dst, used = ops.paged_compact(refs, table)
        ops.paged_copy(st["caches"], src, dst)
    else:
        src, dst, used = _plain_compact(refs, table)
        _plain_copy(st["caches"], src, dst, None)
    return refs, table, src, dst, used, st["caches"]


def _fork(st):
    """The sequences go on from their parents, with some positions more; what of their pages would be written by several is copied."""
    page = st["page"]
    if own:
        from cacti_amd import ops
        st["table"], st["lens"] = ops.paged_fork(st["refs"], st["table"], st["lens"], st["parent"], page)
        src, dst, slots = ops.paged_fit(st["refs"], st["table"], st["lens"], st["lens"] + NEW, page)
        ops.paged_copy(st["caches"], src, dst, slots)
    else:
        st["table"], st["lens"] = _plain_fork(st["refs"], st["table"], st["lens"], st["parent"], page)
        src, dst, slots = _plain_fit(st["refs"], st["table"], st["lens"], st["lens"] + NEW, page)
        _plain_copy(st["caches"], src, dst, slots)
    return st["refs"], st["table"], st["lens"], src, dst, slots, st["caches"]


_RUN = dict(policy=_policy, prefer=_prefer, adapt=_adapt, tune=_tune, pages=_pages)


# ---------------------------------------------------------------- plain forms
def _softmax_parts(st, temp):
    """Probabilities, and log-probabilities of the tokens."""
    z = st["logit"].float() / temp
    z -= z.amax(dim=1, keepdim=True)
    tok = st["tok"].long() & 0xffff
    p = z.exp()
    total = p.sum(dim=1, keepdim=True)
    logp = z.gather(1, tok[:, None]) - total.log()
    return p / total, logp[:, 0], tok


def _gradient(p, tok, coefficient):
    """of the log-probabilities of the tokens, times a coefficient."""
    d = p * -coefficient[:, None]
    return d.scatter_add_(1, tok[:, None], coefficient[:, None]).to(F16)


def _plain_policy(st):
    case, mask, adv = st["case"], st["mask"], st["adv"]
    p, logp, tok = _softmax_parts(st, case["temp"])
    ratio = torch.exp(logp - st["old"])
    free, held = ratio * adv, ratio.clamp(1 - case["clip"], 1 + case["clip"]) * adv
    loss = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, 0.0)
    if st["ref"] is not None:
        d = st["ref"].double() - logp.double()
        loss = loss + (case["beta"] * (torch.expm1(d) - d)).float()
        slope = slope - (case["beta"] * torch.expm1(d)).float()
    zero = torch.zeros_like(logp)
    grad = _gradient(p, tok, torch.where(mask, slope * st["scale"] / case["temp"], zero))
    return torch.where(mask, loss, zero), torch.where(mask, logp, zero), grad


def _log_sigmoid(x):
    return torch.minimum(x, torch.zeros_like(x)) - torch.log1p(torch.exp(-x.abs()))


def _plain_prefer(st):
    case, mask = st["case"], st["mask"]
    pairs, eps = case["pairs"], case["smoothing"]
    p, logp, tok = _softmax_parts(st, 1.0)
    logp = torch.where(mask, logp, 0.0)
    at = torch.arange(logp.shape[0], device="cuda", dtype=I32)
    text = torch.searchsorted(st["starts"], at, right=True) - 1
    sums = torch.zeros(2 * pairs, device="cuda", dtype=torch.float64)
    sums.index_add_(0, text, torch.where(mask, logp.double() - st["ref"].double(), 0.0))
    each = torch.ones_like(sums)
    if case["mean"]:
        each = torch.zeros_like(sums).index_add_(0, text, mask.double()).clamp(min=1)
    sums = BETA * sums / each
    h = sums[0::2] - sums[1::2]
    loss = -(1 - eps) * _log_sigmoid(h) - eps * _log_sigmoid(-h)
    slope = st["scale"].double() * (eps / (1 + torch.exp(-h)) - (1 - eps) / (1 + torch.exp(h)))
    both = torch.stack([slope, -slope], 1).view(-1) * BETA / each
    grad = _gradient(p, tok, torch.where(mask, both[text].float(), 0.0))
    return logp, loss.float(), sums.float(), grad


def _own_adapter(st, T, n, R):
    """Which of n R columns are those of a row's adapter, with the adapter's scale: [T, n R]."""
    at = torch.arange(T, device="cuda", dtype=I32)
    a = st["ids"][torch.searchsorted(st["starts"], at, right=True) - 1]
    hot = (a[:, None] == torch.arange(n, device="cuda", dtype=I32)).float()
    return hot, (hot * st["scale"])[:, :, None].expand(T, n, R).reshape(T, n * R)


def _plain_adapt(st):
    x, A, B = st["x"].float(), st["A"].float(), st["B"].float()
    (T, K), (n, N, R) = x.shape, B.shape
    hot, scales = _own_adapter(st, T, n, R)
    h = torch.matmul(x, A.view(n * R, K).t())
    y = torch.matmul(h * scales, B.permute(0, 2, 1).reshape(n * R, N))
    if st["base"] is not None:
        y += st["base"].float()
    return y.to(F16), (h.view(T, n, R) * hot[:, :, None]).sum(dim=1)


def _plain_tune(st):
    x, A, B, dy = st["x"].float(), st["A"].float(), st["B"].float(), st["dy"].float()
    (T, K), (n, N, R) = x.shape, B.shape
    hot, scales = _own_adapter(st, T, n, R)
    dh = torch.matmul(dy, B.permute(0, 2, 1).reshape(n * R, N).t()) * scales
    dx = torch.matmul(dh, A.view(n * R, K))
    dA = torch.matmul(dh.t(), x).view(n, R, K)
    h = (st["h"][:, None] * hot[:, :, None]).view(T, n * R) * scales
    dB = torch.matmul(h.t(), dy).view(n, R, N).permute(0, 2, 1)
    return dx.to(F16), dA.to(F16), dB.contiguous().to(F16)


def _held(table):
    """Where a table's pages are, and 1 for each entry that is one."""
    return table.clamp(min=0).view(-1).long(), (table >= 0).to(I32).view(-1)


def _plain_fork(refs, table, lens, parent, page):
    W = table.shape[1]
    lives, p = parent >= 0, parent.clamp(min=0).long()
    lens = torch.where(lives, lens[p], 0).to(I32)
    j = torch.arange(W, device="cuda")
    new = torch.where(j < ((lens + page - 1) // page)[:, None], table[p], -1)
    at, one = _held(table)
    refs.scatter_add_(0, at, -one)
    at, one = _held(new)
    refs.scatter_add_(0, at, one)
    return new, lens


def _plain_fit(refs, table, first, lens, page):
    B, W = table.shape
    P = refs.shape[0]
    j, b = torch.arange(W, device="cuda")[None], torch.arange(B, device="cuda")[:, None]
    need, begin, writes = ((lens + page - 1) // page)[:, None], (first // page)[:, None], (lens > first)[:, None]
    loose = (table >= 0) & (j >= torch.where(writes, begin, need))                     # entries that are let go, at first
    at = table.clamp(min=0).long()
    refs.scatter_add_(0, at.view(-1), -loose.to(I32).view(-1))
    wanted = writes & (j >= begin) & (j < need)
    mine = wanted & loose & (refs[at] <= 0)                                            # of no one who keeps them
    first_of = torch.full((P,), B, device="cuda", dtype=torch.int64)
    first_of.scatter_reduce_(0, at.view(-1), torch.where(mine, b, B).view(-1), "amin")
    keeps = mine & (first_of[at] == b)
    refs.scatter_reduce_(0, at.view(-1), keeps.to(I32).view(-1), "amax")
    part = wanted & ~keeps & loose & (j == begin) & ((first % page) > 0)[:, None]
    asked = wanted & ~keeps
    free = refs == 0
    pages = torch.argsort((~free).to(torch.int8), stable=True)
    rank = torch.cumsum(asked.view(-1), 0).view(B, W) - 1
    got = asked & (rank < free.sum())
    new = torch.where(got, pages[rank.clamp(0, P - 1)], -1)
    refs.scatter_add_(0, new.clamp(min=0).view(-1), got.to(I32).view(-1))
    copied = part & got
    src = torch.where(copied, table, -1).amax(dim=1).to(I32)
    dst = torch.where(copied, new, -1).amax(dim=1).to(I32)
    slots = torch.where(copied.any(dim=1), first % page, 0).to(I32)
    table.copy_(torch.where(asked, new.to(I32), torch.where(loose & ~keeps, -1, table)))
    return src, dst, slots


def _plain_compact(refs, table):
    P = refs.shape[0]
    at, used = torch.arange(P, device="cuda"), refs > 0
    count = used.sum()
    leaves, holes = used & (at >= count), ~used & (at < count)
    n = torch.arange(P // 2, device="cuda") < leaves.sum()
    src, dst = (torch.where(n, torch.argsort((~x).to(torch.int8), stable=True)[:P // 2], -1).to(I32) for x in (leaves, holes))
    moves = n & (src >= 0)
    to = torch.arange(P + 1, device="cuda", dtype=I32)
    to.scatter_(0, torch.where(moves, src, P).long(), dst)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    moved = torch.cat([refs, refs[:1]]).scatter_(0, torch.where(moves, dst, P).long(), refs[src.clamp(min=0).long()])[:P]
    refs.copy_(torch.where(at < count, moved, 0))
    return src, dst, count.to(I32).view(1)


def _plain_copy(caches, src, dst, slots):
    does = (src >= 0) & (dst >= 0)
    s, d = src[does].long(), dst[does].long()
    for k, v, ks, vs in caches:
        for x in (k, v):
            x = x.view(torch.uint8) if x.dtype is F8 else x
            if slots is None:
                x[d] = x[s]
            else:
                x[d] = torch.where(torch.arange(x.shape[2], device="cuda")[:, None] < slots[does][:, None, None, None], x[s], x[d])
        for x in (ks, vs):
            if x is not None:
                x[d] = x[s]


# ---------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    st = prepare(case, seed)
    return _EXACT[case["kind"]](st)


def _exact_logp(st, temp):
    tok = st["tok"].long() & 0xffff
    logs = torch.log_softmax(st["logit"].double() / temp, dim=1)
    hot = torch.zeros_like(logs).scatter_(1, tok[:, None], 1.0)
    return logs, logs.gather(1, tok[:, None])[:, 0], hot


def _exact_policy(st):
    case = st["case"]
    logs, lp, hot = _exact_logp(st, case["temp"])
    m = st["mask"].double()
    lp = lp.detach().requires_grad_(True)
    r, A = torch.exp(lp - st["old"].double()), st["adv"].double()
    value = torch.min(r * A, torch.clip(r, 1 - case["clip"], 1 + case["clip"]) * A)
    loss = -value
    if st["ref"] is not None:
        q = torch.exp(st["ref"].double() - lp)
        loss = loss + case["beta"] * (q - torch.log(q) - 1)
    slope, = torch.autograd.grad((loss * m * st["scale"].double()).sum(), lp)
    return loss.detach() * m, lp.detach() * m, (hot - logs.exp()) * (slope / case["temp"])[:, None]


def _exact_prefer(st):
    case = st["case"]
    logs, lp, hot = _exact_logp(st, 1.0)
    lp = (lp * st["mask"]).requires_grad_(True)
    n = _texts(case)
    rewards, s = [], 0
    for x in n:
        m = st["mask"][s:s + x].double()
        d = (m * (lp[s:s + x] - st["ref"][s:s + x].double())).sum()
        rewards.append(BETA * (d / m.sum().clamp(min=1) if case["mean"] else d))
        s += x
    losses = []
    for i in range(case["pairs"]):
        h = rewards[2 * i] - rewards[2 * i + 1]
        log_yes, log_no = torch.nn.functional.logsigmoid(h), torch.nn.functional.logsigmoid(-h)
        losses.append(-(1 - case["smoothing"]) * log_yes - case["smoothing"] * log_no)
    losses = torch.stack(losses)
    slope, = torch.autograd.grad((losses * st["scale"].double()).sum(), lp)
    slope = slope * st["mask"]
    return lp.detach(), losses.detach(), torch.stack(rewards).detach(), (hot - logs.exp()) * slope[:, None]


def _by_sequence(st):
    s = 0
    for a, n in zip(st["ids"].tolist(), _counts(st["case"]["S"], st["case"]["new"], st["case"]["ragged"])):
        yield a, slice(s, s + n)
        s += n


def _exact_adapt(st):
    T, N, R = st["x"].shape[0], st["case"]["N"], st["case"]["R"]
    y = torch.zeros((T, N), device="cuda", dtype=torch.float64) if st["base"] is None else st["base"].double()
    hs = torch.zeros((T, R), device="cuda", dtype=torch.float64)
    for a, at in _by_sequence(st):
        if a >= 0:
            hs[at] = st["x"][at].double() @ st["A"][a].double().t().contiguous()
            y[at] += float(st["scale"][a]) * (hs[at] @ st["B"][a].double().t().contiguous())
    return y, hs


def _exact_tune(st):
    dx = torch.zeros(st["x"].shape, device="cuda", dtype=torch.float64)
    dA, dB = (torch.zeros(st[w].shape, device="cuda", dtype=torch.float64) for w in "AB")
    for a, at in _by_sequence(st):
        if a >= 0:
            f, x, dy = float(st["scale"][a]), st["x"][at].double(), st["dy"][at].double()
            dh = f * (dy @ st["B"][a].double())
            dx[at] = dh @ st["A"][a].double()
            dA[a] += dh.t().contiguous() @ x
            dB[a] += f * (dy.t().contiguous() @ st["h"][at].double())
    return dx, dA, dB


def _exact_pages(st):
    """Page by page, as someone with a pencil would."""
    case, page = st["case"], st["page"]
    refs, table, lens = st["refs"].tolist(), st["table"].tolist(), st["lens"].tolist()
    copies = []
    if case["op"] == "compact":
        live = [x for x in range(len(refs)) if refs[x] > 0]
        holes = [x for x in range(len(live)) if refs[x] == 0]
        copies = [(s, d, page) for s, d in zip([x for x in live if x >= len(live)], holes)]
    else:
        parent = st["parent"].tolist()
        rows = [[x for x in table[p][:-(-lens[p] // page)]] if p >= 0 else [] for p in parent]
        for old in table:
            for x in old:
                if x >= 0:
                    refs[x] -= 1
        lens = [lens[p] if p >= 0 else 0 for p in parent]
        for row in rows:
            for x in row:
                refs[x] += 1
        parts = {}                             # pages that sequences are going to write on, and which these are
        for b, row in enumerate(rows):
            if lens[b] % page:
                parts.setdefault(row[-1], []).append(b)
        asked = []
        for b, row in enumerate(rows):
            for j in range(lens[b] // page, -(-(lens[b] + NEW) // page)):
                if j < len(row):
                    of = parts[row[j]]
                    if refs[row[j]] == len(of) and b == of[0]:
                        continue
                    asked.append((row[j], lens[b] % page))
                else:
                    asked.append((None, 0))
        for x, of in parts.items():
            refs[x] = 1 if refs[x] == len(of) else refs[x] - len(of)
        free = [x for x in range(len(refs)) if refs[x] == 0]
        copies = [(s, d, m) for (s, m), d in zip(asked, free) if s is not None]
    caches = []
    for cache in st["caches"]:
        now = [None if x is None else x.to(torch.float64 if x.dtype is torch.float32 else torch.float32) for x in cache]
        for s, d, m in copies:
            for x in now[:2]:
                x[d, :, :m] = x[s, :, :m]
            for x in now[2:]:
                if x is not None:
                    x[d] = x[s]
        caches.append(now)
    return [None] * (5 if case["op"] == "compact" else 6) + [caches]


_EXACT = dict(policy=_exact_policy, prefer=_exact_prefer, adapt=_exact_adapt, tune=_exact_tune, pages=_exact_pages)

"""Serving from a paged cache, checking drafted tokens and training the drafting model: the operators as cases that can be
timed and compared.

  append   new keys and values of a ragged batch into the pages of a cache, rotated on the way, with the queries
           (ops.paged_append)
  attend   attention of the new rows over the pages, in 8 bits with a scale per page and head, or in f16
           (ops.paged_attention)
  verify   which drafted tokens the target model's probabilities keep, and the token after them (ops.verify_draft)
  distill  loss of a student against a teacher's top logits, and its gradient (ops.distill_topk_fwd, distill_topk_bwd)

`own` chooses between the framework's operators and their plain form in elementary torch operations.
"""
import math
import random

import torch

own = False

F8 = torch.float8_e4m3fn
F16 = torch.float16
MAX8 = 448.0                                   # the largest e4m3 value
MIN_EXP, MAX_EXP = -32, 15                     # of a page's scale


def listed():
    return [
        # a chat's next token: one sequence, the benchmark's heads, everything is launch and latency
        dict(name="append_one", kind="append", B=1, new=1, ragged=False, lo=701, hi=701, H=32, Hkv=32, Dh=100, page=64, bits=8),
        # a batch of chats with a few drafted tokens each, queries that share keys four by four, small pages
        dict(name="append_drafts", kind="append", B=96, new=6, ragged=True, lo=40, hi=4000, H=32, Hkv=8, Dh=128, page=16, bits=8),
        # prompts of the benchmark's length and shorter
        dict(name="append_prompts", kind="append", B=4, new=2048, ragged=True, lo=2048, hi=2048, H=32, Hkv=32, Dh=100, page=64, bits=8),
        # a chat's next token over a document
        dict(name="attend_one", kind="attend", B=1, new=1, ragged=False, lo=1540, hi=1540, H=32, Hkv=32, Dh=100, page=64, bits=8),
        # a batch of chats of all lengths, a token each
        dict(name="attend_batch", kind="attend", B=48, new=1, ragged=False, lo=120, hi=8192, H=32, Hkv=32, Dh=100, page=64, bits=8),
        # drafted tokens of a batch, shared keys
        dict(name="attend_drafts", kind="attend", B=24, new=6, ragged=True, lo=100, hi=6000, H=32, Hkv=8, Dh=128, page=32, bits=8),
        # prompts behind what their sequences hold already, f16 pages
        dict(name="attend_prompts", kind="attend", B=3, new=900, ragged=True, lo=1000, hi=4000, H=16, Hkv=16, Dh=128, page=64, bits=16),
        # four drafted tokens of one sequence, the benchmark's vocabulary
        dict(name="verify_one", kind="verify", B=1, new=5, ragged=False, V=32000, temp=1.0, draft=True),
        # a batch with up to seven drafted tokens each
        dict(name="verify_batch", kind="verify", B=64, new=8, ragged=True, V=32000, temp=0.8, draft=True),
        # a tiny student
        dict(name="distill_tiny", kind="distill", N=128, V=1024, K=8, temp=1.0),
        # texts of odd length, an odd vocabulary, softened
        dict(name="distill_odd", kind="distill", N=611, V=8191, K=20, temp=2.0),
        # the benchmark's head
        dict(name="distill_3b", kind="distill", N=2048, V=32000, K=64, temp=1.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_weight(c) for c in listed())
    while True:
        c = _draw(rng)
        if _weight(c) <= most:
            return c


def _weight(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


_HEADS = [(4, 4, 64), (8, 2, 64), (16, 16, 64), (32, 32, 100), (8, 8, 100), (16, 16, 128), (32, 8, 128), (16, 1, 128), (12, 4, 80),
          (14, 2, 36)]


def _draw(rng):
    kind = rng.choice(["append", "attend", "attend", "verify", "distill"])
    if kind in ("append", "attend"):
        H, Hkv, Dh = rng.choice(_HEADS)
        B = _log(rng, 1, 64)
        new = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 1200)])
        lo = new + _log(rng, 1, 2000)
        return dict(kind=kind, B=B, new=new, ragged=rng.random() < 0.7, lo=lo, hi=lo + _log(rng, 1, 6000), H=H, Hkv=Hkv, Dh=Dh,
                    page=rng.choice([16, 32, 64, 128]), bits=rng.choice([8, 8, 16]))
    if kind == "verify":
        return dict(kind=kind, B=_log(rng, 1, 64), new=rng.randint(1, 9), ragged=rng.random() < 0.7, V=_log(rng, 1000, 65000),
                    temp=rng.choice([1.0, 0.7, round(rng.uniform(0.3, 1.6), 2), 0.0]), draft=rng.random() < 0.7)
    return dict(kind=kind, N=_log(rng, 1, 2048), V=_log(rng, 500, 60000), K=_log(rng, 1, 128), temp=round(rng.uniform(0.7, 4.0), 2))


# ---------------------------------------------------------------- sizes of a ragged batch
def _new_of(case):
    """New rows of each sequence: all the same, or 1 .. new in a fixed shuffle with the largest among them."""
    B, new = case["B"], case["new"]
    if not case["ragged"]:
        return [new] * B
    r = random.Random(7 * B + new)
    n = [new] + [r.randint(1, new) for _ in range(B - 1)]
    r.shuffle(n)
    return n


def _lens_of(case):
    """Lengths with the new rows: over lo .. hi in even steps of the logarithm, shuffled."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    r = random.Random(11 * B + hi)
    ls = [int(round(math.exp(math.log(hi) + (math.log(lo) - math.log(hi)) * i / max(1, B - 1)))) for i in range(B)]
    r.shuffle(ls)
    return ls


def work(case):
    if case["kind"] == "append":
        T, Dh, size = sum(_new_of(case)), case["Dh"], case["bits"] // 8
        return dict(bytes=T * (case["H"] * Dh * 4 + case["Hkv"] * Dh * 2 * (2 + size) + Dh * 4),
                    flops=3 * T * Dh * (case["H"] + case["Hkv"]))
    if case["kind"] == "attend":
        n, ls, Dh = _new_of(case), _lens_of(case), case["Dh"]
        seen = sum(m * l - m * (m - 1) // 2 for m, l in zip(n, ls))
        return dict(bytes=sum(ls) * case["Hkv"] * Dh * 2 * (case["bits"] // 8) + sum(n) * case["H"] * Dh * 4,
                    flops=4 * seen * case["H"] * Dh)
    if case["kind"] == "verify":
        n, V = _new_of(case), case["V"]
        return dict(bytes=2 * V * (sum(n) + (sum(n) - case["B"] if case["draft"] and case["temp"] > 0 else 0)), flops=4 * V * sum(n))
    N, V, K = case["N"], case["V"], case["K"]
    return dict(bytes=N * (6 * V + 8 * K + 12), flops=8 * N * V)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=F16).mul_(std)


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _starts(n):
    s = [0]
    for x in n:
        s.append(s[-1] + x)
    return _ints(s)


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    if case["kind"] in ("append", "attend"):
        _prepare_cache(case, g, st)
    elif case["kind"] == "verify":
        _prepare_verify(case, g, st)
    else:
        _prepare_distill(case, g, st)
    return st


def _prepare_cache(case, g, st):
    """A cache with its sequences' pages all over it, filled as earlier tokens left it, and the new rows as the projections
    give them: q, k and v side by side in rows of one matrix."""
    B, H, Hkv, Dh, page = (case[x] for x in ("B", "H", "Hkv", "Dh", "page"))
    n, ls = _new_of(case), _lens_of(case)
    T, W = sum(n), -(-max(ls) // page)
    pages = B * W + 3
    Dp = -(-Dh // 16) * 16
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    st["table"] = order[:B * W].reshape(B, W).contiguous()
    st["starts"], st["lens"] = _starts(n), _ints(ls)
    st["max_new"] = case["new"]
    qkv = _randn(g, T, (H + 2 * Hkv) * Dh)
    st["q"] = qkv[:, :H * Dh].view(T, H, Dh)
    st["k"] = qkv[:, H * Dh:(H + Hkv) * Dh].view(T, Hkv, Dh)
    st["v"] = qkv[:, (H + Hkv) * Dh:].view(T, Hkv, Dh)
    kp, vp = (torch.randn((pages, Hkv, page, Dp), generator=g, device="cuda", dtype=F16) for _ in range(2))
    kp[..., Dh:] = 0
    vp[..., Dh:] = 0
    if case["bits"] == 8:
        # codes up to some 250 of 448 and scales around 2^-6: values of some units
        st["kp"], st["vp"] = (x.mul_(48).clamp_(-MAX8, MAX8).to(F8) for x in (kp, vp))
        st["ks"], st["vs"] = (torch.exp2(torch.randint(-7, -4, (pages, Hkv), generator=g, device="cuda").float()) for _ in range(2))
    else:
        st["kp"], st["vp"], st["ks"], st["vs"] = kp, vp, None, None
    st["cos"], st["sin"] = _rotation(max(ls), Dh)
    st["alpha"] = 1.0 / math.sqrt(Dh)


def _rotation(S, Dh):
    """cos and sin tables of the positions, [S, Dh] f16, two identical halves."""
    inv = torch.pow(10000.0, -torch.arange(0, Dh, 2, device="cuda", dtype=torch.float64) / Dh)
    a = torch.arange(S, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.cos()], 1).to(F16), torch.cat([a.sin(), a.sin()], 1).to(F16)


def _prepare_verify(case, g, st):
    n, V = _new_of(case), case["V"]
    T = sum(n)
    target = torch.randn((T, V), generator=g, device="cuda").mul_(2.5)
    draft = target + torch.randn((T, V), generator=g, device="cuda")
    # tokens as the drafting model took them, from its own probabilities (the first of a sequence is any token); without its
    # probabilities they come from elsewhere and are often what the target model would say
    noise = torch.rand((T, V), generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)
    temp = case["temp"] if case["temp"] > 0 else 0.1
    tok = ((draft if case["draft"] else target * 1.5) / temp - torch.log(-torch.log(noise))).argmax(dim=1)
    st["tok"] = torch.roll(tok, 1).to(torch.int16)                  # u16 bit patterns: row i+1 holds what row i drew
    st["target"], st["draft"] = target.to(F16), draft.to(F16) if case["draft"] else None
    st["starts"] = _starts(n)
    st["u"] = torch.rand(T, generator=g, device="cuda")
    st["r"] = torch.rand(case["B"], generator=g, device="cuda")


def _prepare_distill(case, g, st):
    N, V, K = case["N"], case["V"], case["K"]
    teacher = torch.randn((N, V), generator=g, device="cuda").mul_(3.0)
    top = teacher.topk(K, dim=1)
    st["val"], st["idx"] = top.values.to(F16), top.indices.to(torch.int16)     # u16 bit patterns
    st["logit"] = (teacher * 0.6 + 2.0 * torch.randn((N, V), generator=g, device="cuda")).to(F16)
    st["scale"] = torch.full((N,), 1024.0 / max(1, N - 1), device="cuda")
    if N > 1:
        st["scale"][0] = 0.0                                                   # (as the training example leaves position 0 out)
    st["temp"] = case["temp"]


# ---------------------------------------------------------------- one pass
def run(st):
    return _RUN[st["case"]["kind"]](st)


def _append(st):
    if own:
        from cacti_amd import ops
        cache = (st["kp"], st["vp"], st["ks"], st["vs"])
        q = ops.paged_append(st["k"], st["v"], cache, st["table"], st["starts"], st["lens"], st["cos"], st["sin"], q=st["q"],
                             max_new=st["max_new"])
    else:
        q = _plain_append(st)
    return [q, st["kp"], st["vp"], st["ks"], st["vs"]]


def _attend(st):
    if own:
        from cacti_amd import ops
        cache = (st["kp"], st["vp"], st["ks"], st["vs"])
        return ops.paged_attention(st["q"], cache, st["table"], st["starts"], st["lens"], st["alpha"], max_new=st["max_new"])
    return _plain_attend(st)


def _verify(st):
    if own:
        from cacti_amd import ops
        return ops.verify_draft(st["target"], st["draft"], st["tok"], st["starts"], st["u"], st["r"], temperature=st["case"]["temp"])
    return _plain_verify(st)


def _distill(st):
    if own:
        from cacti_amd import ops
        loss, stats = ops.distill_topk_fwd(st["logit"], st["idx"], st["val"], st["temp"])
        return loss, ops.distill_topk_bwd(st["logit"], st["idx"], st["val"], stats, st["scale"], st["temp"])
    return _plain_distill(st)


_RUN = dict(append=_append, attend=_attend, verify=_verify, distill=_distill)


# ---------------------------------------------------------------- plain forms
def _rows(st, T):
    """Sequence and position of each row."""
    at = torch.arange(T, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(st["starts"], at, right=True) - 1
    pos = st["lens"][b] - (st["starts"][b + 1] - at)
    return b, pos.long()


def _rotated(x, cos, sin, pos):
    """The rotation in fp32: halves (a, b) -> (a cos - b sin, b cos + a sin)."""
    x, c, s = x.float(), cos[pos].float()[:, None], sin[pos].float()[:, None]
    a, b = x.chunk(2, dim=2)
    return x * c + torch.cat([-b, a], 2) * s


def _plain_append(st):
    page = st["case"]["page"]
    T, _, Dh = st["k"].shape
    b, pos = _rows(st, T)
    pid, slot = st["table"][b, pos // page].long(), pos % page
    new_k = _rotated(st["k"], st["cos"], st["sin"], pos)
    first = (st["lens"] - (st["starts"][1:] - st["starts"][:-1])).long()               # of each sequence's new positions
    part = st["table"].gather(1, (first // page)[:, None].clamp(max=st["table"].shape[1] - 1))[:, 0].long()
    older = torch.arange(page, device="cuda")[None, :] < (first % page)[:, None]       # slots of that page that hold older tokens
    for pages, scales, new in ((st["kp"], st["ks"], new_k), (st["vp"], st["vs"], st["v"].float())):
        if scales is None:
            pages[pid, :, slot, :Dh] = new.to(F16)
            continue
        raw = pages.view(torch.uint8)
        need = torch.zeros(scales.shape, device="cuda").index_reduce_(0, pid, new.abs().amax(2), "amax", include_self=True)
        m, e = torch.frexp(need.double() / MAX8)
        need = torch.exp2((e - (m == 0.5).int()).clamp(MIN_EXP, MAX_EXP).float())
        need = torch.where(m == 0, 2.0 ** MIN_EXP, need)
        was = torch.zeros_like(scales)
        was[part] = torch.where((first % page > 0)[:, None], scales[part], 0.0)
        now = torch.maximum(need, was)
        again = (pages[part].float() * (was / now)[part][:, :, None, None]).to(F8).view(torch.uint8)
        raw[part] = torch.where(older[:, None, :, None], again, raw[part])
        scales[pid] = now[pid]
        raw[pid, :, slot, :Dh] = (new / now[pid][:, :, None]).to(F8).view(torch.uint8)
    return _rotated(st["q"], st["cos"], st["sin"], pos).to(F16)


def _plain_attend(st):
    case, q = st["case"], st["q"]
    T, H, Dh = q.shape
    B, Hkv, new = case["B"], case["Hkv"], case["new"]
    G = H // Hkv
    W, page = st["table"].shape[1], case["page"]
    table = st["table"].long()

    def cache(pages, scales):
        x = pages[table][..., :Dh].float()                                             # [B, W, Hkv, page, Dh]
        if scales is not None:
            x *= scales[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, W * page, Dh)

    n = (st["starts"][1:] - st["starts"][:-1]).long()
    b, pos = _rows(st, T)
    i = torch.arange(T, device="cuda") - st["starts"][b].long()
    qp = torch.zeros((B, new, H, Dh), device="cuda")
    qp[b, i] = q.float() * st["alpha"]
    qp = qp.view(B, new, Hkv, G, Dh).permute(0, 2, 1, 3, 4).reshape(B, Hkv, new * G, Dh)
    s = torch.matmul(qp, cache(st["kp"], st["ks"]).transpose(2, 3).contiguous()).view(B, Hkv, new, G, W * page)
    last = st["lens"].long()[:, None] - n[:, None] + torch.arange(new, device="cuda")  # last visible position of each row
    hidden = torch.arange(W * page, device="cuda")[None, None, :] > last[..., None]
    s.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    s -= s.amax(dim=4, keepdim=True)
    s.exp_()
    s /= s.sum(dim=4, keepdim=True)
    o = torch.matmul(s.view(B, Hkv, new * G, W * page), cache(st["vp"], st["vs"]))
    o = o.view(B, Hkv, new, G, Dh).permute(0, 2, 1, 3, 4).reshape(B, new, H, Dh)
    return o[b, i].to(F16)


def _probabilities(logit, temp):
    """In 64 bits: what is drawn goes by where the sums' borders lie."""
    z = logit.double()
    if temp == 0:
        return torch.zeros_like(z).scatter_(1, z.argmax(dim=1, keepdim=True), 1.0)
    z = torch.exp((z - z.amax(dim=1, keepdim=True)) / temp)
    return z / z.sum(dim=1, keepdim=True)


def _plain_verify(st):
    starts, temp = st["starts"].long(), st["case"]["temp"]
    T, V = st["target"].shape
    at = torch.arange(T, device="cuda")
    b = torch.searchsorted(starts, at, right=True) - 1
    final = at == starts[b + 1] - 1                                                    # rows without a drafted token behind them
    x = torch.roll(st["tok"], -1).long() & 0xffff
    p = _probabilities(st["target"], temp)
    if st["draft"] is None or temp == 0:
        q = torch.zeros_like(p).scatter_(1, x[:, None], 1.0)
    else:
        q = _probabilities(st["draft"], temp)
    px, qx = p.gather(1, x[:, None])[:, 0], q.gather(1, x[:, None])[:, 0]
    stop = final | ~(st["u"].double() * qx < px)
    a = torch.full_like(starts[1:], T).index_reduce_(0, b, torch.where(stop, at, T), "amin", include_self=True)
    w = torch.where(final[a][:, None], p[a], (p[a] - q[a]).clamp(min=0))
    w = torch.where(w.sum(dim=1, keepdim=True) > 0, w, p[a])
    c = w.cumsum(dim=1)
    drawn = torch.searchsorted(c, st["r"].double()[:, None] * c[:, -1:], right=True)[:, 0]
    out = torch.where(at < a[b], x, 0)
    out[a] = drawn
    return (a - starts[:-1]).to(torch.int32), out.to(torch.int16)


def _plain_distill(st):
    temp, scale = st["temp"], st["scale"][:, None]
    idx = st["idx"].long() & 0xffff
    z = st["logit"].float() / temp
    z -= z.amax(dim=1, keepdim=True)
    e = z.exp()
    sums = e.sum(dim=1, keepdim=True)
    t = st["val"].float() / temp
    t -= t.amax(dim=1, keepdim=True)
    log_t = t - t.exp().sum(dim=1, keepdim=True).log()
    t = log_t.exp()
    loss = (t * (log_t - z.gather(1, idx) + sums.log())).sum(dim=1)
    grad = (e / sums).scatter_add_(1, idx, -t)
    return loss, (grad * (scale / temp)).to(F16)


# ---------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(st)
    if case["kind"] == "attend":
        return _exact_attend(st)
    if case["kind"] == "distill":
        return _exact_distill(st)
    return None                                # verify's outputs are whole numbers


def _sequences(st):
    n, ls = _new_of(st["case"]), _lens_of(st["case"])
    s = 0
    for b in range(len(n)):
        yield b, s, n[b], ls[b] - n[b]
        s += n[b]


def _exact_append(st):
    case = st["case"]
    Dh, page, bits = case["Dh"], case["page"], case["bits"]
    q, k, v = (st[x].double() for x in "qkv")
    kp, vp = st["kp"].double(), st["vp"].double()
    ks, vs = (None, None) if bits == 16 else (st["ks"].double(), st["vs"].double())
    out_q = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for b, s, n, first in _sequences(st):
        c, sn = (st[x][first:first + n].double()[:, None, :Dh // 2] for x in ("cos", "sin"))

        def turn(x):
            lo, hi = x[..., :Dh // 2], x[..., Dh // 2:]
            return torch.cat([lo * c - hi * sn, hi * c + lo * sn], dim=2)

        out_q[s:s + n] = turn(q[s:s + n])
        for pages, scales, new in ((kp, ks, turn(k[s:s + n])), (vp, vs, v[s:s + n])):
            done = 0
            while done < n:                    # page by page
                slot = (first + done) % page
                m = min(page - slot, n - done)
                pid = int(st["table"][b, (first + done) // page])
                x = new[done:done + m].transpose(0, 1)
                if scales is not None:
                    e = torch.ceil(torch.log2((x.abs().amax(dim=(1, 2)) / MAX8).clamp(min=2.0 ** MIN_EXP)))
                    to = torch.exp2(e)
                    if slot:
                        to = torch.maximum(to, scales[pid])
                        pages[pid, :, :slot] *= (scales[pid] / to)[:, None, None]
                    scales[pid] = to
                    x = x / to[:, None, None]
                pages[pid, :, slot:slot + m, :Dh] = x
                done += m
    return [out_q, kp, vp, ks, vs]


def _exact_attend(st):
    case = st["case"]
    G, Dh = case["H"] // case["Hkv"], case["Dh"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, s, n, first in _sequences(st):
        L = first + n
        ids = st["table"][b, :-(-L // case["page"])].long()
        kk, vv = st["kp"][ids].double()[..., :Dh], st["vp"][ids].double()[..., :Dh]    # [w, Hkv, page, Dh]
        if case["bits"] == 8:
            kk, vv = kk * st["ks"][ids].double()[..., None, None], vv * st["vs"][ids].double()[..., None, None]
        for h in range(case["H"]):
            k1, v1 = kk[:, h // G].reshape(-1, Dh)[:L], vv[:, h // G].reshape(-1, Dh)[:L]
            w = st["alpha"] * (st["q"][s:s + n, h].double() @ k1.t().contiguous())
            w = w + torch.full((n, L), -math.inf, dtype=torch.float64, device="cuda").triu(first + 1)
            out[s:s + n, h] = torch.softmax(w, dim=1) @ v1
    return out


def _exact_distill(st):
    idx = st["idx"].long() & 0xffff
    log_p = torch.log_softmax(st["logit"].double() / st["temp"], dim=1)
    log_t = torch.log_softmax(st["val"].double() / st["temp"], dim=1)
    loss = torch.sum(log_t.exp() * (log_t - log_p.gather(1, idx)), dim=1)
    hot = torch.zeros_like(log_p).scatter_add_(1, idx, log_t.exp())
    return loss, (log_p.exp() - hot) * (st["scale"].double() / st["temp"])[:, None]

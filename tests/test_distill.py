"""Distillation from a teacher's top logits: cacti_hip_distill_topk_{fwd,bwd} against float64.

What the kernels round.  Loss: of the student's side only the sum of V exponentials is fp32, each off by 2^-23 for the
instruction and 2^-23 |z - max| / tau for its argument, a chain of V / 512 additions and some ten more of 2^-24 each; of the
teacher's side the same over K.  So its absolute error is at most
  2^-23 (2 + spread) + 2^-24 (V / 512 + K / 512 + 40), spread = (largest |z - max| with a share of the sum, here all) / tau,
and 2^-21 sum t |log t - log p| for the weights.  Gradient: half a step of f16, 2^-11 |dz| (2^-25 below its normal range), and
scale / tau times the same relative error of p and t, doubled for the quotients; accumulated, one more rounding of each."""
import numpy as np
import pytest

from cacti_amd import ffi

GPU = pytest.mark.gpu
FWD = dict(N=2, V=64, K=4, logit=64, ld=64, idx=64, val=64, temp=1.0, loss=64, stats=64, status=None, stream=None)
BWD = dict(N=2, V=64, K=4, logit=64, ld=64, idx=64, val=64, stats=64, scale=64, temp=1.0, d=64, ldd=64, acc=0, stream=None)
COMMON = [(dict(N=0), "empty"), (dict(V=0), "empty"), (dict(K=0), "empty"), (dict(V=65537, ld=65537, ldd=65537), "65536"), (dict(K=1025), "1024"),
          (dict(N=1 << 23), "2^23"), (dict(ld=63), "pitch"), (dict(logit=None), "null"), (dict(idx=None), "null"), (dict(val=None), "null"),
          (dict(stats=None), "null"), (dict(temp=0.0), "temperature"), (dict(temp=float("nan")), "temperature"), (dict(temp=-2.0), "temperature"),
          (dict(logit=65), "misaligned"), (dict(stats=66), "misaligned")]


@pytest.mark.parametrize("change,why", COMMON + [(dict(loss=None), "null"), (dict(loss=66), "misaligned")])
def test_forward_refuses(change, why):
    L, args = ffi.lib(), {k: v for k, v in dict(FWD, **change).items() if k in FWD}
    assert L.cacti_hip_distill_topk_fwd(*args.values()) < 0
    assert why in L.cacti_hip_last_error().decode()


@pytest.mark.parametrize("change,why", COMMON + [(dict(scale=None), "null"), (dict(d=None), "null"), (dict(ldd=63), "pitch"), (dict(d=65), "misaligned")])
def test_adjoint_refuses(change, why):
    L = ffi.lib()
    assert L.cacti_hip_distill_topk_bwd(*dict(BWD, **change).values()) < 0
    assert why in L.cacti_hip_last_error().decode()


def reference(z, idx, val, scale, temp):
    """loss, gradient before its rounding, error bounds of both."""
    N, V = z.shape
    K = idx.shape[1]
    loss, grad = np.zeros(N), np.zeros((N, V))
    loss_tol, grad_tol = np.zeros(N), np.zeros((N, V))
    for n in range(N):
        v, zz = val[n].astype(np.float64) / temp, z[n].astype(np.float64) / temp
        ok = (idx[n] < V)
        if np.all(val[n] == -np.inf):
            continue
        t = np.exp(v - v.max())
        t /= t.sum()
        log_t = v - v.max() - np.log(np.exp(v - v.max()).sum())
        log_p = zz - zz.max() - np.log(np.exp(zz - zz.max()).sum())
        t, log_t, ids = t[ok], log_t[ok], idx[n][ok]
        use = t > 0
        diff = log_t[use] - log_p[ids[use]]
        loss[n] = (t[use] * diff).sum()
        hot = np.zeros(V)
        np.add.at(hot, ids, t)
        p = np.exp(log_p)
        grad[n] = scale[n] / temp * (p * t.sum() - hot)          # (t of the ids that there are: the loss has no others)
        spread = (zz.max() - zz[np.isfinite(zz)].min()) + (v.max() - v[np.isfinite(v)].min())
        rel = 2.0 ** -23 * (2 + spread) + 2.0 ** -24 * (V / 512 + K / 512 + 40)
        loss_tol[n] = rel + 2.0 ** -21 * (t[use] * np.abs(diff)).sum()
        grad_tol[n] = np.abs(scale[n]) / temp * 2 * (rel + 2.0 ** -21) * (p + hot) + 2.0 ** -11 * np.abs(grad[n]) + 2.0 ** -25
    return loss, grad, loss_tol, grad_tol


def make(seed, N, V, K, temp=1.0, std=3.0):
    r = np.random.default_rng(seed)
    teacher = r.standard_normal((N, V)) * std
    idx = np.argsort(-teacher, 1)[:, :K]
    val = np.take_along_axis(teacher, idx, 1).astype(np.float16)
    z = (teacher * 0.6 + r.standard_normal((N, V)) * 2).astype(np.float16)
    scale = (r.standard_normal(N) * 4).astype(np.float32)
    return z, idx, val, scale, temp


def dev(x):
    import torch
    x = np.ascontiguousarray(x)
    return torch.from_numpy(x.astype(np.uint16).view(np.int16) if x.dtype == np.int64 else x).cuda()


def run(z, idx, val, scale, temp, acc=None):
    from cacti_amd import ops
    dz, di, dv = dev(z), dev(idx), dev(val)
    loss, stats = ops.distill_topk_fwd(dz, di, dv, temp)
    return loss.cpu().numpy(), ops.distill_topk_bwd(dz, di, dv, stats, dev(scale), temp, acc=acc).cpu().numpy()


def check(args):
    loss, grad = run(*args)
    wl, wg, tl, tg = reference(*args)
    assert loss.dtype == np.float32 and np.isfinite(loss).all()
    off = np.abs(loss - wl) / np.maximum(tl, 1e-300)
    assert (np.abs(loss - wl) <= tl).all(), "loss: %.2f of the bound" % off.max()
    over = np.abs(grad.astype(np.float64) - wg) > tg
    assert not over.any(), "gradient: %d of %d beyond the bound" % (over.sum(), over.size)
    return loss, grad


@GPU
@pytest.mark.parametrize("N,V,K,temp", [(1, 1, 1, 1.0), (3, 8, 8, 2.0), (5, 7, 3, 0.7), (2, 1000, 64, 1.0), (4, 1021, 20, 3.0), (3, 8191, 128, 1.5),
                                        (2, 32000, 64, 1.0), (2, 65536, 1000, 2.0), (9, 513, 513, 1.0), (2, 4096, 1024, 1.0)])
def test_distill(N, V, K, temp):
    print("distill_topk", N, V, K, temp, flush=True)
    check(make(V + K, N, V, K, temp))
    check(make(V + K + 1, N, V, K, temp, std=0.1))


@GPU
def test_gradient_against_differences():
    """Central differences of the float64 loss at the kernel's own gradient, in directions of single logits and a random one."""
    z, idx, val, scale, temp = make(3, 2, 50, 6, 1.7)
    _, grad = run(z, idx, val, np.ones(2, np.float32), temp)
    f = lambda x: reference(x, idx, val, scale, temp)[0]
    r = np.random.default_rng(4)
    h = 1e-4
    z64 = z.astype(np.float64)
    for d in [np.eye(50)[j][None] * np.ones((2, 1)) for j in (0, int(idx[0, 0]), int(idx[1, 5]), 49)] + [r.standard_normal((2, 50))]:
        num = (f(z64 + h * d) - f(z64 - h * d)) / (2 * h)
        got = (grad.astype(np.float64) * d).sum(1)
        # differences: h^2 times a third derivative below sum |d|^3; the gradient: half a step of f16 and fp32's share of it
        tol = h * h * (np.abs(d) ** 3).sum(1) + (np.abs(d) * (np.abs(grad) * 2.0 ** -11 + 2.0 ** -18)).sum(1) + 1e-9
        assert (np.abs(num - got) <= tol).all(), (num, got)


@GPU
def test_accumulates():
    from cacti_amd import ops
    args = make(5, 3, 1001, 16, 1.3)
    z, idx, val, scale, temp = args
    old = np.random.default_rng(6).standard_normal(z.shape).astype(np.float16)
    into = dev(old)
    dz, di, dv = dev(z), dev(idx), dev(val)
    _, stats = ops.distill_topk_fwd(dz, di, dv, temp)
    got = ops.distill_topk_bwd(dz, di, dv, stats, dev(scale), temp, acc=into)
    assert got is into
    _, first = run(*args)
    want = (old.astype(np.float32) + first.astype(np.float32)).astype(np.float16)       # the rounded gradient, added in fp32
    assert np.array_equal(got.cpu().numpy(), want)


@GPU
def test_entries_that_are_nothing_or_twice():
    """-inf entries, rows of none but such (also where the student's row is no number), the same id twice, ids beyond the
    vocabulary."""
    import torch
    from cacti_amd import ops
    z, idx, val, scale, temp = make(7, 6, 300, 12)
    val[0, 5:], val[1, :], val[2, 3] = -np.inf, -np.inf, -np.inf
    idx[3, 4], idx[3, 9], idx[3, 11] = idx[3, 0], idx[3, 0], idx[3, 2]
    idx[4, :] = 7
    loss, grad = check((z, idx, val, scale, temp))
    assert loss[1] == 0 and not grad[1].any()
    z[1, :] = np.nan
    loss, grad = run(z, idx, val, scale, temp)
    assert loss[1] == 0 and not grad[1].any() and np.isfinite(grad).all()
    z, idx, val, scale, temp = make(8, 3, 100, 5)
    idx[2, 1], idx[2, 3] = 100, 65535
    loss, grad = check((z, idx, val, scale, temp))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.distill_topk_fwd(dev(z), dev(idx), dev(val), temp, status=status)
    assert int(status) == 3


@GPU
def test_values_that_are_no_numbers_stay_visible():
    """A NaN of the student or of the teacher makes its row NaN, -inf of the student where the teacher has weight an infinite
    loss with a gradient; other rows are as ever."""
    args = make(9, 4, 200, 10)
    z, idx, val, scale, temp = args
    clean = run(*args)
    z, val = z.copy(), val.copy()
    z[0, 3], val[1, 2] = np.nan, np.nan
    z[2, idx[2, 0]] = -np.inf
    loss, grad = run(z, idx, val, scale, temp)
    assert np.isnan(loss[0]) and np.isnan(grad[0]).all() and np.isnan(loss[1])
    assert np.isposinf(loss[2]) and np.isfinite(grad[2]).all()
    assert loss[3] == clean[0][3] and np.array_equal(grad[3], clean[1][3])


@GPU
def test_rows_may_be_strided_and_lie_anywhere():
    import torch
    from cacti_amd import ops
    for V in (1000, 1003):
        z, idx, val, scale, temp = make(10, 5, V, 9)
        wl, wg = run(z, idx, val, scale, temp)
        for ld, off, ldo, offo in ((V, 0, V + 5, 3), (V + 3, 1, V, 0), (V + 8, 8, V + 8, 0), (2 * V, 5, V + 1, 2)):
            big = torch.zeros(5 * ld + 16, dtype=torch.float16, device="cuda")
            rows = big[off:off + 5 * ld].view(5, ld)[:, :V]
            rows.copy_(dev(z))
            loss, stats = ops.distill_topk_fwd(rows, dev(idx), dev(val), temp)
            into = torch.full((5 * ldo + 16,), 7.0, dtype=torch.float16, device="cuda")
            grad = into[offo:offo + 5 * ldo].view(5, ldo)[:, :V]
            grad.zero_()
            ops.distill_topk_bwd(rows, dev(idx), dev(val), stats, dev(scale), temp, acc=grad)
            # (the order in which a row is summed goes by where it begins)
            assert np.abs(loss.cpu().numpy() - wl).max() <= 2e-5
            assert np.abs(grad.cpu().numpy().astype(np.float64) - wg).max() <= 2.0 ** -9 * np.abs(wg).max()
            kept = into.clone()
            kept[offo:offo + 5 * ldo].view(5, ldo)[:, :V] = 7
            assert bool((kept == 7).all())                    # nothing beside the rows


@GPU
def test_arguments_that_do_not_go_together():
    import torch
    from cacti_amd import ops
    z, idx, val, scale, temp = (dev(x) if not isinstance(x, float) else x for x in make(11, 4, 64, 3))
    loss, stats = ops.distill_topk_fwd(z, idx, val, temp)
    for bad in ((z.float(), idx, val), (z, idx.int(), val), (z, idx, val.float()), (z, idx[:2], val[:2]), (z, idx[:, :2], val), (z.cpu(), idx, val),
                (z.t(), idx, val)):
        with pytest.raises(AssertionError):
            ops.distill_topk_fwd(*bad)
    for bad in ((stats[:2], scale), (stats, scale[:1]), (stats.half(), scale), (stats, scale.double())):
        with pytest.raises(AssertionError):
            ops.distill_topk_bwd(z, idx, val, *bad)
    with pytest.raises(AssertionError):
        ops.distill_topk_bwd(z, idx, val, stats, scale, 1.0, acc=z[:2])
    with pytest.raises(ffi.CactiError):
        ops.distill_topk_fwd(z, idx, val, 0.0)
    loss, stats = ops.distill_topk_fwd(z[:0], idx[:0], val[:0])
    assert loss.shape == (0,) and ops.distill_topk_bwd(z[:0], idx[:0], val[:0], stats, scale[:0]).shape == (0, 64)


@GPU
def test_captured_and_replayed():
    import torch
    from cacti_amd import ops
    z, idx, val, scale, temp = (dev(x) if not isinstance(x, float) else x for x in make(12, 33, 2000, 20, 1.5))

    def step():
        loss, stats = ops.distill_topk_fwd(z, idx, val, temp)
        return loss, ops.distill_topk_bwd(z, idx, val, stats, scale, temp)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i in range(4):
        g.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        z.copy_(torch.roll(z, 3, 1))


@pytest.mark.parametrize("change", [dict(d=66), dict(d=64 + 2 * 64), dict(ldd=65), dict(ld=128, ldd=128, d=64 + 2 * 63), dict(d=64 - 2 * 64)])
def test_adjoint_refuses_a_gradient_that_overlaps_the_logits(change):
    L = ffi.lib()
    assert L.cacti_hip_distill_topk_bwd(*dict(BWD, logit=0x1040, **{"d": 0x1000 + change["d"]} if "d" in change else {"d": 0x1040},
                                              **{k: v for k, v in change.items() if k != "d"}).values()) < 0
    assert "place" in L.cacti_hip_last_error().decode()


@GPU
@pytest.mark.parametrize("N,V,ld,off", [(3, 1001, 1001, 0), (2, 32000, 32003, 5), (2, 65536, 65536, 0)])
def test_gradient_in_the_logits_place(N, V, ld, off):
    """Instead of the logits, and added to them."""
    import torch
    from cacti_amd import ops
    z, idx, val, scale, temp = make(8, N, V, 40, 1.2)
    di, dv, ds = dev(idx), dev(val), dev(scale)
    buf = torch.zeros(N * ld + off, dtype=torch.float16, device="cuda")
    rows = buf[off:].view(N, ld)[:, :V]
    for acc in (False, True):
        rows.copy_(dev(z))
        _, stats = ops.distill_topk_fwd(rows, di, dv, temp)
        want = ops.distill_topk_bwd(rows, di, dv, stats, ds, temp, acc=rows.clone() if acc else None)
        if acc:
            ops.distill_topk_bwd(rows, di, dv, stats, ds, temp, acc=rows)
        else:
            assert ffi.lib().cacti_hip_distill_topk_bwd(N, V, 40, rows.data_ptr(), ld, di.data_ptr(), dv.data_ptr(), stats.data_ptr(), ds.data_ptr(),
                                                        temp, rows.data_ptr(), ld, 0, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(rows, want)

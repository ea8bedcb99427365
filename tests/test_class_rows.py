"""Class log probabilities with entropy and alternatives, and distillation from a teacher's kept logits (csrc/class_rows.hip), against
their definitions in 64 bits.

Tolerances (u = 2^-24; half = eps(type) / 2; L = additions in a row's longest chain: K / 64 on a lane and 32 to join lanes and parts):
  log s        s adds at most K terms 2^x, each off by 2 u + |x| u; a chain of L additions: (L + 2 log2 K + 8) u
  log p        (l - m) / T - log s: u (4 |l - m| / T + 2 |log p|) + the error of log s                                     =: tl
  H            log s - t / s: twice the error of log s (once relative to t / s, at most log K, once absolute): (2 + log K) of it
  p            p times (the error of log p + 4 u + |log p| u)
  loss         T^2 sum q (log q - log p): sum_i q_i (tl_i + (8 + nkept + 4 |log q_i|) u) T^2, q_i off by the same relative error
  gradients    products and sums of these with one rounding each; + half |result| (fp16: and its smallest step, 2^-24)
               p below the smallest normal number, 2^-126, comes out of the exponential as 0: 2^-126 times what p is multiplied with
               (|a| + |e| (|log p| + H), up to about 45 at a = 1, e = 1/2 and log p = -88, or T |g|)"""
import ctypes
import math

import pytest
import torch

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def chain(K):
    return (K / 64 + 32 + 2 * math.log2(K + 1) + 8) * U


def log_softmax64(l):
    """log softmax of float64 rows where a row of nothing but -inf is -inf"""
    m = l.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    s = torch.exp(l - m).sum(-1, keepdim=True)
    return torch.where(s == 0, torch.full_like(l, -math.inf), l - m - torch.log(s)), m


def ref_logprobs(l, labels, top, ga=None, ge=None):
    """float64 rows (R,K) -> outputs and tolerances"""
    K = l.shape[1]
    lp, m = log_softmax64(l)
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    h = -plp.sum(1)
    has = labels >= 0
    y = labels.clamp(0, K - 1)
    logp = torch.where(has, lp.gather(1, y[:, None])[:, 0], torch.zeros_like(h))
    finite = torch.where(torch.isfinite(lp), lp.abs(), torch.zeros_like(lp))
    tl = U * (4 * (l - m).nan_to_num(0, 0, 0).abs() + 2 * finite) + chain(K)
    out = {"logp": logp, "entropy": h, "tlogp": tl.gather(1, y[:, None])[:, 0], "tentropy": (2 + math.log(K + 1)) * chain(K) + 4 * U * h}
    key = torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l)
    cls = key.sort(dim=1, descending=True, stable=True)[1][:, :top]
    out.update(top_class=cls, top_logp=lp.gather(1, cls), ttop=tl.gather(1, cls))
    if ga is not None:
        a = torch.where(has, ga, torch.zeros_like(ga))[:, None]
        e = ge[:, None]
        d = -p * a - e * torch.where(p > 0, p * (lp + h[:, None]), torch.zeros_like(p))
        d.scatter_add_(1, y[:, None], a)
        rel = tl + (4 + finite) * U
        spread = a.abs() + e.abs() * (finite + h[:, None])
        tol = 2.0 ** -126 * spread.clamp_max(1e3) + p * spread * (rel + 8 * U) + p * e.abs() * (tl + out["tentropy"][:, None])
        tol.scatter_add_(1, y[:, None], 2 * U * a.abs())
        out.update(dscore=d, tdscore=tol)
    return out


def ref_distill(l, kept, cls, T, g=None):
    K = l.shape[1]
    lp, m = log_softmax64(l / T)
    p = lp.exp()
    has = cls >= 0
    t = torch.where(has, kept / T, torch.full_like(kept, -math.inf))
    logq, _ = log_softmax64(t)
    q = torch.where(torch.isfinite(logq), logq.exp(), torch.zeros_like(logq))
    at = cls.clamp(0, K - 1)
    lc = lp.gather(1, at)
    term = torch.where(q > 0, q * (logq - lc), torch.zeros_like(q))
    finite = torch.where(torch.isfinite(lp), lp.abs(), torch.zeros_like(lp))
    tl = U * (4 * (l / T - m).nan_to_num(0, 0, 0).abs() + 2 * finite) + chain(K)
    tq = (8 + kept.shape[1] + 4 * torch.where(q > 0, logq.abs(), torch.zeros_like(q))) * U
    out = {"loss": T * T * term.sum(1), "tloss": T * T * (q * (tl.gather(1, at) + tq * (2 + (logq - lc).nan_to_num(0, 0, 0).abs()))).sum(1)}
    if g is not None:
        any_ = (q.sum(1, keepdim=True) > 0).double()
        d = (p * any_).scatter_add(1, at, -q)
        tol = (2.0 ** -126 + p * (tl + (12 + finite) * U)).scatter_add(1, at, q * (tq + 8 * U))
        out.update(dscore=T * g[:, None] * d, tdscore=T * g[:, None].abs() * tol)
    return out


def near(got, want, tol, dtype, name):
    got = got.double()
    # a value beyond the largest 32-bit number rounds to infinity (the loss of a row whose student rules out, by the lowest fp32 score, what
    # the teacher keeps: T^2 q 3.4e38 / T)
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want * math.inf, want)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    bound = tol + (torch.finfo(dtype).eps / 2 * want.abs() if dtype else U * want.abs()) + (U if dtype == torch.float16 else 1e-37)
    bad = ~same & ~((got - want).abs() <= bound)
    assert not bad.any(), "%s: %d of %d off, worst %.3g (%.3g allowed there)" % (
        name, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].max()), float(bound[bad].max()))


def lay(rows, how, N=1):
    """(R,K) -> the same rows as the score tensor of a layout, and a function that puts (…) outputs back into row order"""
    R, K = rows.shape
    if how == "rows":
        return rows, lambda t: t
    if how == "wide":                                        # rows of a wider matrix, off 16 bytes
        w = torch.zeros(R, K + 11, dtype=rows.dtype, device=rows.device)
        w[:, 3:3 + K] = rows
        return w[:, 3:3 + K], lambda t: t
    if how == "transposed":
        return rows.t().contiguous().t(), lambda t: t
    if how == "planar":
        return rows.view(N, R // N, K).permute(0, 2, 1).contiguous(), lambda t: t
    if how == "channels_last":
        return rows.view(N, R // N, K).permute(0, 2, 1), lambda t: t
    raise ValueError(how)


def score_rows(t):
    return t if t.dim() == 2 else t.movedim(1, -1).reshape(-1, t.shape[1])


def make(R, K, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = 2 * torch.randn(R, K, device="cuda", generator=g)
    labels = torch.randint(0, K, (R,), device="cuda", generator=g)
    l.scatter_add_(1, labels[:, None], 3 * torch.rand(R, 1, device="cuda", generator=g))
    labels[::7] = -1
    ga, ge = torch.randn(R, device="cuda", generator=g), torch.randn(R, device="cuda", generator=g)
    return l.to(dtype), labels, ga, ge, g


def check_logprobs(l, labels, ga, ge, top, dtype, how="rows", N=1, num=None):
    from sis3d import ops
    score, back = lay(l, how, N)
    shape = (score.shape[0],) if score.dim() == 2 else (score.shape[0],) + tuple(score.shape[2:])
    v = lambda t: t.view(shape)                              # noqa: E731
    logp, h, norm, tl, tc = ops.class_logprobs(score, v(labels), top=top, num=num)
    assert logp.shape == shape and norm.shape == shape + (2,) and tc.shape == shape + (top,) and tl.shape == tc.shape
    d = ops.class_logprobs_backward(score, v(labels), norm, h, v(ga), v(ge), num=num)
    assert d.shape == score.shape and d.dtype == score.dtype
    want = ref_logprobs(l.double(), labels, top, ga.double(), ge.double())
    n = l.shape[0] if num is None else int(num)
    f = lambda t: t.reshape((l.shape[0],) + t.shape[len(shape):])     # noqa: E731
    near(f(logp)[:n], want["logp"][:n], want["tlogp"][:n], None, "logp")
    near(f(h)[:n], want["entropy"][:n], want["tentropy"][:n], None, "entropy")
    assert torch.equal(f(tc)[:n], want["top_class"][:n])
    near(f(tl)[:n], want["top_logp"][:n], want["ttop"][:n], None, "top_logp")
    near(score_rows(d)[:n], want["dscore"][:n], want["tdscore"][:n], dtype, "dscore")
    for t in (f(logp), f(h), f(norm), f(tl), f(tc), score_rows(d)):
        assert (t[n:] == 0).all()
    return logp, h, norm, tl, tc, d


KS = [1, 2, 3, 4, 8, 19, 20, 41, 64, 65, 257, 272, 273, 528, 529, 537, 1000, 1024, 1025, 1203, 4095, 4096, 4097, 8192, 20011, 65536]


@pytest.mark.gpu
@pytest.mark.parametrize("K", KS)
@pytest.mark.parametrize("R", [1, 3, 300, 70001])
@pytest.mark.parametrize("dt", list(DT))
def test_logprobs_match_definition(R, K, dt):
    if R > 1000:
        R = min(R, int(3e6) // K | 1)                           # many rows where rows are short
    l, labels, ga, ge, _ = make(R, K, DT[dt], seed=K + R)
    for top in sorted({0, 1, min(K, 3), min(K, 8), min(K, 32)}):
        check_logprobs(l, labels, ga, ge, top, DT[dt])


@pytest.mark.gpu
@pytest.mark.parametrize("how,R,K,N", [("planar", 300, 2, 1), ("planar", 330, 41, 5), ("planar", 6, 19, 2), ("planar", 60, 1024, 3), ("channels_last", 330, 41, 5),
                                       ("channels_last", 12, 2000, 2), ("transposed", 77, 26, 1), ("wide", 77, 26, 1), ("wide", 9, 2001, 1),
                                       ("wide", 5, 20011, 1), ("planar", 8, 1, 2), ("planar", 3, 19, 3), ("channels_last", 3, 1500, 3)])
@pytest.mark.parametrize("dt", list(DT))
def test_layouts(how, R, K, N, dt):
    l, labels, ga, ge, g = make(R, K, DT[dt], seed=R)
    check_logprobs(l, labels, ga, ge, min(3, K), DT[dt], how, N)
    num = torch.tensor([R // 2], dtype=torch.int32, device="cuda")
    check_logprobs(l, labels, ga, ge, min(3, K), DT[dt], how, N, num)
    check_distill(l, *teacher(l, 5, g), 1.5, DT[dt], how, N, num)


def special_rows(K, device="cuda"):
    """rows that a mask, a tie or a number out of range make special; row -> name"""
    g = torch.Generator(device=device).manual_seed(K)
    base = torch.randn(K, device=device, generator=g)
    inf, low = math.inf, torch.finfo(torch.float32).min
    c = torch.arange(K, device=device)
    rows = [torch.full((K,), -inf), torch.where(c.cpu() == K - 1, 0.5, -inf), torch.full((K,), low), torch.where(c.cpu() % 3 == 1, 1.0, low),
            torch.zeros(K), torch.where(c.cpu() % 2 == 0, 0.0, -0.0), (c.cpu() % 4).float(), -c.cpu().float(), c.cpu().float(),
            torch.where(c.cpu() % 5 == 0, -inf, base.cpu()), base.cpu() * 1e4, base.cpu() * 1e37, base.cpu() * 1e10, base.cpu() + 3e6, base.cpu() - 3e6,
            base.cpu() + 1e9, base.cpu() - 1e9, torch.where(c.cpu() < K - K // 4, -1e30, base.cpu()), torch.where(c.cpu() % 64 < 60, -1e9, base.cpu()),
            # all but every 32nd vector of 4 high: more elements at the alternatives' bound than there is room for
            torch.where((c.cpu() // 4) % 32 == 0, base.cpu() - 50, base.cpu())]
    return torch.stack(rows).to(device)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [2, 19, 64, 300, 530, 1000, 1025, 4096, 5000, 20011])
def test_masked_tied_and_extreme_rows(K):
    l = special_rows(K)
    R = l.shape[0]
    labels = (torch.arange(R, device="cuda") * 7) % K
    labels[1] = K - 1
    ga, ge = torch.ones(R, device="cuda"), torch.full((R,), 0.5, device="cuda")
    check_logprobs(l, labels, ga, ge, min(K, 32), torch.float32)
    check_logprobs(l[:1].repeat(400, 1), labels[:1].repeat(400), ga[:1].repeat(400), ge[:1].repeat(400), min(K, 8), torch.float32)
    check_logprobs(l, labels, ga, ge, 1, torch.float32, "wide")
    for dt in (torch.bfloat16, torch.float16):
        low = torch.full((3, K), torch.finfo(dt).min, dtype=dt, device="cuda")
        low[1, K // 2] = 1.0
        check_logprobs(low, labels[:3], ga[:3], ge[:3], min(K, 3), dt)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [5, 1000, 3000, 20000])
def test_non_finite_rows_and_labels_out_of_range(K):
    """NaN and +inf make their own row NaN and no other; the alternatives stay classes; a label that is no class gives NaN"""
    from sis3d import ops
    l, labels, ga, ge, _ = make(6, K, torch.float32)
    labels[:] = torch.tensor([0, 1, 2, K - 1, K, 1 << 40], device="cuda")
    clean = ops.class_logprobs(l, labels, top=4)
    dclean = ops.class_logprobs_backward(l, labels, clean[2], clean[1], ga, ge)
    assert torch.isnan(clean[0][4:]).all() and torch.isfinite(clean[0][:4]).all()
    assert torch.isnan(dclean[4:]).all() and torch.isfinite(dclean[:4]).all()
    bad = l.clone()
    bad[1, K // 3] = math.nan
    bad[2, K - 1] = math.inf
    logp, h, norm, tl, tc = ops.class_logprobs(bad, labels, top=4)
    d = ops.class_logprobs_backward(bad, labels, norm, h, ga, ge)
    for t in (logp, h, tl, d):
        assert torch.isnan(t[1:3]).all()
    assert ((tc >= 0) & (tc < K)).all()
    assert (tc[1] != K // 3).all() and tc[2, 0] == K - 1                # NaN ranks last, +inf first
    for i in (0, 3):
        assert torch.equal(logp[i], clean[0][i]) and torch.equal(d[i], dclean[i]) and torch.equal(tc[i], clean[4][i])
    allnan = torch.full((300, K), math.nan, device="cuda")
    tc = ops.class_logprobs(allnan, torch.zeros(300, dtype=torch.int64, device="cuda"), top=3)[4]
    assert torch.equal(tc, torch.arange(3, device="cuda").expand(300, 3))


def teacher(l, k, g):
    R, K = l.shape
    k = min(k, K)
    kept, cls = (l.float() + torch.randn(R, K, device=l.device, generator=g)).topk(k, 1)
    return kept.contiguous(), cls


def check_distill(l, kept, cls, T, dtype, how="rows", N=1, num=None, g=None):
    from sis3d import ops
    score, _ = lay(l, how, N)
    R = l.shape[0]
    shape = (R,) if score.dim() == 2 else (score.shape[0],) + tuple(score.shape[2:])
    g = torch.linspace(-2, 3, R, device="cuda") if g is None else g
    kw = dict(temperature=T, num=num)
    kv, cv = kept.view(shape + kept.shape[1:]), cls.view(shape + cls.shape[1:])
    loss, norm = ops.distill_loss(score, kv, cv, **kw)
    d = ops.distill_loss_backward(score, kv, cv, norm, g.view(shape), **kw)
    want = ref_distill(l.double(), kept.double(), cls, T, g.double())
    n = R if num is None else int(num)
    near(loss.reshape(-1)[:n], want["loss"][:n], want["tloss"][:n], None, "loss")
    near(score_rows(d)[:n], want["dscore"][:n], want["tdscore"][:n], dtype, "dscore")
    assert (loss.reshape(-1)[n:] == 0).all() and (score_rows(d)[n:] == 0).all() and d.dtype == score.dtype
    return loss, norm, d


@pytest.mark.gpu
@pytest.mark.parametrize("K", KS)
@pytest.mark.parametrize("R,T", [(1, 1.0), (3, 1.5), (300, 4.0), (70001, 2.0)])
@pytest.mark.parametrize("dt", list(DT))
def test_distillation_matches_definition(R, K, T, dt):
    if R > 1000:
        R = min(R, int(3e6) // K | 1)
    l, _, _, _, g = make(R, K, DT[dt], seed=K)
    for k in sorted({1, min(K, 5), min(K, 128)}):
        kept, cls = teacher(l, k, g)
        check_distill(l, kept, cls, T, DT[dt])
        cls = cls.clone()
        cls[torch.rand(cls.shape, device="cuda", generator=g) < 0.3] = -1       # absent entries; whole rows of them where k is small
        check_distill(l, kept, cls, T, DT[dt])


@pytest.mark.gpu
@pytest.mark.parametrize("K", [3, 19, 1000, 3000, 9000, 20011])
def test_distillation_edges(K):
    from sis3d import ops
    R = 6
    l, _, _, _, g = make(R, K, torch.float32, seed=K)
    l[4] = -math.inf                                                            # a student row that allows nothing
    l[5, 1:] = -math.inf
    kept = torch.randn(R, 6, device="cuda", generator=g)
    cls = torch.randint(0, K, (R, 6), device="cuda", generator=g)
    cls[0] = torch.tensor([2, 0, 2, 2, 1, 0], device="cuda")                    # the same class several times
    cls[1] = -1                                                                 # nothing kept
    kept[2, :5] = -math.inf                                                     # a teacher that allows one class
    kept[3] = -math.inf                                                         # one that allows none
    cls[5] = torch.tensor([0, -1, -1, -1, -1, -1], device="cuda")               # one class for both: loss 0
    loss, norm, d = check_distill(l, kept, cls, 2.0, torch.float32)
    assert loss[1] == 0 and loss[3] == 0 and (d[1] == 0).all() and (d[3] == 0).all()
    assert loss[4] == math.inf and loss[5] == 0
    # a class that is none, and NaN: their own row
    bad_cls, bad_kept = cls.clone(), kept.clone()
    bad_cls[0, 3] = K
    bad_kept[2, 0] = math.nan
    bl, bn = ops.distill_loss(l, bad_kept, bad_cls, 2.0)
    bd = ops.distill_loss_backward(l, bad_kept, bad_cls, bn, torch.ones(R, device="cuda"), 2.0)
    assert torch.isnan(bl[[0, 2]]).all() and torch.isnan(bd[[0, 2]]).all()
    assert torch.equal(bl[[1, 3, 5]], loss[[1, 3, 5]]) and torch.isfinite(bd[[1, 3, 5]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("how,K,k", [("rows", 5, 5), ("rows", 96, 6), ("rows", 97, 16), ("wide", 333, 32), ("rows", 1000, 17), ("rows", 1001, 33), ("rows", 2047, 8),
                                     ("rows", 4100, 6), ("planar", 19, 16), ("planar", 41, 32), ("planar", 200, 70), ("transposed", 130, 9)])
@pytest.mark.parametrize("dt", list(DT))
def test_distillation_of_many_rows_with_edges(how, K, k, dt):
    """more rows than there are lanes to take one each: masked rows, equal classes (and such that are equal modulo 64), absent and bad
    entries beside ordinary rows, live rows that end inside a group of four"""
    from sis3d import ops
    R = 4099
    l, _, _, _, g = make(R, K, DT[dt], seed=K)
    kept = torch.randn(R, k, device="cuda", generator=g)
    cls = torch.randint(0, K, (R, k), device="cuda", generator=g)
    cls[0::11] = cls[0::11] % 64 + 64 * torch.randint(0, max(1, K // 64), (R, k), device="cuda", generator=g)[0::11]
    cls = torch.where(cls < K, cls, 0)
    cls[1::11] = -1                                                             # nothing kept
    cls[2::11] = cls[2::11, :1]                                                 # one class, many times
    cls[3::11, k // 2:] = -1
    kept[4::11, 1:] = -math.inf                                                 # a teacher that allows one class
    kept[5::11] = -math.inf                                                     # one that allows none
    l[6::11] = -math.inf                                                        # a student row that allows nothing
    l[7::11, 1:] = -math.inf
    big = torch.finfo(DT[dt]).max
    l[8::11] = -big                                                             # the type's lowest value throughout
    l[9::11, ::2] = -big
    l = l.contiguous()
    num = torch.tensor([4094], dtype=torch.int32, device="cuda")
    for n in (None, num, num * 0, num * 0 + 3):
        loss, norm, d = check_distill(l, kept, cls, 2.0, DT[dt], how, 1, n)
    loss, norm, d = check_distill(l, kept, cls, 2.0, DT[dt], how)
    bad_cls, bad_kept = cls.clone(), kept.clone()
    bad_cls[10::11, k - 1] = K
    bad_kept[21::11, 0] = math.nan                                              # (some of these entries are absent, and do not count)
    score, _ = lay(l, how)
    one = score.dim() - 2
    bl, bn = ops.distill_loss(score, bad_kept[None] if one else bad_kept, bad_cls[None] if one else bad_cls, 2.0)
    bd = score_rows(ops.distill_loss_backward(score, bad_kept[None] if one else bad_kept, bad_cls[None] if one else bad_cls, bn, torch.linspace(-2, 3, R, device="cuda").view(bl.shape), 2.0))
    bl, loss = bl.reshape(-1), loss.reshape(-1)
    bad = (bad_cls >= K).any(1) | (torch.isnan(bad_kept) & (bad_cls >= 0)).any(1)
    assert bad.any() and torch.isnan(bl[bad]).all() and torch.isnan(bd[bad]).all()
    assert torch.equal(bl[~bad], loss[~bad]) and torch.equal(bd[~bad], score_rows(d)[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("how,K", [("rows", 1), ("rows", 3), ("planar", 2), ("planar", 19), ("rows", 19), ("wide", 300), ("rows", 400), ("rows", 1203), ("rows", 5000), ("rows", 9000)])
@pytest.mark.parametrize("R", [5, 4500])
def test_the_most_entries_that_a_row_may_keep(how, K, R):
    """128 entries, most of them of the same few classes"""
    if R * K > 1e7:
        R = 300
    l, _, _, _, g = make(R, K, torch.float32, seed=K + R)
    kept = torch.randn(R, 128, device="cuda", generator=g)
    cls = torch.randint(0, min(K, 40), (R, 128), device="cuda", generator=g)
    cls[:, ::3] = torch.randint(0, K, (R, 43), device="cuda", generator=g)
    cls[:, 5] = -1
    check_distill(l, kept, cls, 1.5, torch.float32, how)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [19, 300, 2000, 9000])
def test_one_row_of_scores_for_many_labels(K):
    """an expanded tensor: rows that share their memory"""
    from sis3d import ops
    l, _, _, _, g = make(1, K, torch.float32, seed=K)
    R = 4200 if K < 9000 else 200
    labels = torch.randint(0, K, (R,), device="cuda", generator=g)
    ga = torch.randn(R, device="cuda", generator=g)
    kept, cls = torch.randn(R, 4, device="cuda", generator=g), torch.randint(0, K, (R, 4), device="cuda", generator=g)
    for a, b in ((l.expand(R, K), l.expand(R, K).contiguous()),):
        fa, fb = ops.class_logprobs(a, labels, 5), ops.class_logprobs(b, labels, 5)
        assert torch.equal(fa[4], fb[4])
        near(fa[0], fb[0].double(), 8 * U * (1 + fb[0].double().abs()) + chain(K), None, "logp")
        da, db = ops.class_logprobs_backward(a, labels, fa[2], fa[1], ga), ops.class_logprobs_backward(b, labels, fb[2], fb[1], ga)
        near(da, db.double(), ga.double().abs()[:, None] * (32 * U + 2 * chain(K)), None, "dscore")
        (la, na), (lb, nb) = ops.distill_loss(a, kept, cls), ops.distill_loss(b, kept, cls)
        near(la, lb.double(), 32 * U * (1 + lb.double().abs()) + chain(K), None, "loss")
        near(ops.distill_loss_backward(a, kept, cls, na, ga), ops.distill_loss_backward(b, kept, cls, nb, ga).double(),
             ga.double().abs()[:, None] * (64 * U + 2 * chain(K)), None, "dscore")


@pytest.mark.gpu
@pytest.mark.parametrize("K", [300, 1000, 3001, 6000])
@pytest.mark.parametrize("dt", list(DT))
def test_alternatives_of_many_rows(K, dt):
    """every number of alternatives, rows by lanes and waves; among them ascending rows, of which every vector is a new best, and rows of few
    different scores, of which many are at the bound"""
    from sis3d import ops
    R = 4100
    l, labels, _, _, g = make(R, K, DT[dt], seed=K)
    ramp = torch.arange(K, device="cuda", dtype=torch.float32)
    l[0::5] = ramp.to(DT[dt])
    l[1::5] = torch.randint(0, 6, (R, K), device="cuda", generator=g)[1::5].to(DT[dt])
    l[2::5, K // 50:] = -math.inf
    l[3::50] = -ramp.to(DT[dt])
    # the order by (score, class): a stable sort of the scores, largest first
    order = l.float().sort(dim=1, descending=True, stable=True)[1]
    for top in (1, 2, 4, 5, 8, 9, 16, 17, 32):
        logp, _, norm, tl, tc = ops.class_logprobs(l, labels, top)
        assert torch.equal(tc, order[:, :top]), top
        ls = log_softmax64(l.double())[0]
        near(tl, ls.gather(1, tc), 4 * U * torch.where(torch.isfinite(ls), ls.abs(), 0.0).gather(1, tc) + chain(K) + 4 * U * (l.double().amax(1, True) - l.double()).gather(1, tc).nan_to_num(0, 0, 0), None, "top")


@pytest.mark.gpu
def test_streams_graph_and_determinism():
    from sis3d import ops
    for R, K, top in ((200, 19, 3), (64, 3000, 8), (2, 60000, 8), (300, 20011, 32)):
        l, labels, ga, ge, g = make(R, K, torch.bfloat16)
        kept, cls = teacher(l, 4, g)
        num = torch.tensor([R], dtype=torch.int32, device="cuda")

        def step():
            logp, h, norm, tl, tc = ops.class_logprobs(l, labels, top=top, num=num)
            d = ops.class_logprobs_backward(l, labels, norm, h, ga, ge, num=num)
            loss, n2 = ops.distill_loss(l, kept, cls, 2.0, num=num)
            return logp, h, norm, tl, tc, d, loss, n2, ops.distill_loss_backward(l, kept, cls, n2, ga, 2.0, num=num)
        eager = [t.clone() for t in step()]
        assert all(torch.equal(a, c) for a, c in zip(step(), eager))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        side.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(other, eager))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        keep = l.clone()
        for k in range(4):
            l.copy_(keep.roll(k, 0) + k)
            num.fill_(R - k if R > 2 else 1 + k % 2)
            graph.replay()
            torch.cuda.synchronize()
            again = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(held, again)), (R, K, k)


@pytest.mark.gpu
def test_more_than_two_to_the_31_elements():
    from sis3d import ops
    K, R = 32768, (1 << 31) // 32768 + 64
    l = torch.empty(R, K, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for i in range(0, R, 4096):
        l[i:i + 4096].normal_(generator=g)
    labels = torch.randint(0, K, (R,), device="cuda", generator=g)
    logp, h, norm, tl, tc = ops.class_logprobs(l, labels, top=4)
    ga = torch.ones(R, device="cuda")
    d = ops.class_logprobs_backward(l, labels, norm, h, ga)
    for sl in (slice(0, 8), slice(R - 8, R)):
        want = ref_logprobs(l[sl].double(), labels[sl], 4, ga[sl].double(), torch.zeros(8, device="cuda", dtype=torch.float64))
        near(logp[sl], want["logp"], want["tlogp"], None, "logp")
        assert torch.equal(tc[sl], want["top_class"])
        near(d[sl], want["dscore"], want["tdscore"], torch.bfloat16, "dscore")
    # many short rows: V * K past 2^31 in a planar map
    del l, d
    K, V = 41, (1 << 31) // 41 + 1000
    l = torch.empty(1, K, V, dtype=torch.bfloat16, device="cuda")
    for c in range(K):
        l[0, c].normal_(generator=g)
    labels = torch.zeros(1, V, dtype=torch.int64, device="cuda")
    logp, h, norm, tl, tc = ops.class_logprobs(l, labels, top=2)
    rows = l[0, :, V - 100:].t().double()
    want = ref_logprobs(rows, labels[0, :100], 2)
    near(logp[0, V - 100:], want["logp"], want["tlogp"], None, "logp")
    near(h[0, V - 100:], want["entropy"], want["tentropy"], None, "entropy")
    assert torch.equal(tc[0, V - 100:], want["top_class"])


@pytest.mark.gpu
def test_autograd_forms_and_differences():
    from sis3d import ops
    from sis3d.layer_utils.class_losses import ClassLogProbs, DistillLoss
    for K in (19, 1500, 9000):
        l, labels, ga, ge, g = make(12, K, torch.float32, seed=K)
        kept, cls = teacher(l, 6, g)
        s = l.clone().requires_grad_(True)
        logp, h, tl, tc = ClassLogProbs.apply(s, labels, 2, None)
        assert not tl.requires_grad and not tc.requires_grad
        loss = DistillLoss.apply(s, kept, cls, 2.0, None)
        total = (logp * ga).sum() + (h * ge).sum() + (loss * ga).sum()
        total.backward()
        o = ops.class_logprobs(l, labels)
        n2 = ops.distill_loss(l, kept, cls, 2.0)[1]
        d1 = ops.class_logprobs_backward(l, labels, o[2], o[1], ga, ge)
        d2 = ops.distill_loss_backward(l, kept, cls, n2, ga, 2.0)
        assert torch.equal(s.grad, d1 + d2)
        # one of the two gradients alone
        s2 = l.clone().requires_grad_(True)
        ClassLogProbs.apply(s2, labels)[1].sum().backward()
        zero = torch.zeros(12, device="cuda")
        assert torch.equal(s2.grad, ops.class_logprobs_backward(l, labels, o[2], o[1], zero, zero + 1))
        # central differences, step 2^-5: the rounding of 12 rows' values (24 values below 2^4: 24 * 2^4 u) over the step is below 1e-3, the
        # third derivatives' share step^2 / 6 = 1.6e-4 of terms p (1 - p) (1 - 2 p) and their like, each below the first one's size
        for k in range(3):
            v = torch.randn(l.shape, device="cuda", generator=g)
            v /= v.abs().max()
            f = []
            for step in (2.0 ** -5, -2.0 ** -5):
                x = l + step * v
                a = ops.class_logprobs(x, labels)
                f.append(float((a[0] * ga).double().sum() + (a[1] * ge).double().sum() + (ops.distill_loss(x, kept, cls, 2.0)[0] * ga).double().sum()))
            slope, want = (f[0] - f[1]) * 2.0 ** 4, float((s.grad.double() * v.double()).sum())
            assert abs(slope - want) <= 4e-3 + 2e-3 * float((s.grad.double() * v.double()).abs().sum()), (K, slope, want)


@pytest.mark.gpu
def test_cross_entropy_of_the_detector_heads():
    """the classification losses of lib/nets/network.py:319-501 on this package's own score layouts: RPN scores (1,2,X,Y,Z,A) with
    label -1 = ignored, class scores (R,19) of the padded detection rows with the device-side row count"""
    from sis3d import ops
    from sis3d.layer_utils.class_losses import ClassLogProbs
    g = torch.Generator(device="cuda").manual_seed(0)
    rpn = torch.randn(1, 2, 6, 3, 6, 11, device="cuda", generator=g).requires_grad_(True)
    lab = torch.randint(-1, 2, (1, 6, 3, 6, 11), device="cuda", generator=g)
    logp, _, _, _ = ClassLogProbs.apply(rpn, lab)
    (-logp.sum() / (lab >= 0).sum()).backward()
    ref = rpn.detach().double().requires_grad_(True)
    want = torch.nn.functional.cross_entropy(ref, lab, ignore_index=-1)
    want.backward()
    assert abs(float(-logp.detach().sum() / (lab >= 0).sum()) - float(want.detach())) < 1e-5
    assert (rpn.grad - ref.grad).abs().max() < 1e-8                     # gradients of order 1 / 1188, a few u of that
    score = torch.randn(200, 19, device="cuda", generator=g)
    num = torch.tensor([37], dtype=torch.int32, device="cuda")
    labels = torch.randint(0, 19, (200,), device="cuda", generator=g)
    logp, entropy, _, top, cls = ops.class_logprobs(score, labels, top=2, num=num)
    assert torch.equal(cls[:37, 0], score[:37].argmax(1)) and (logp[37:] == 0).all() and (cls[37:] == 0).all()


@pytest.mark.gpu
def test_refusals():
    from sis3d import _lib, ops
    l, labels, ga, ge, g = make(4, 10, torch.float32)
    kept, cls = teacher(l, 3, g)
    _, h, norm, _, _ = ops.class_logprobs(l, labels)
    bad = [lambda: ops.class_logprobs(l.cpu(), labels.cpu()), lambda: ops.class_logprobs(l, labels.int()), lambda: ops.class_logprobs(l, labels[:3]),
           lambda: ops.class_logprobs(l, labels.cpu()), lambda: ops.class_logprobs(l, labels, top=11), lambda: ops.class_logprobs(l, labels, top=-1),
           lambda: ops.class_logprobs(l.repeat(1, 9), labels, top=33), lambda: ops.class_logprobs(l.double(), labels),
           lambda: ops.class_logprobs(l[0], labels), lambda: ops.class_logprobs(l[:, :0], labels),
           lambda: ops.class_logprobs(l, labels, num=torch.tensor([1, 2], dtype=torch.int32, device="cuda")),
           lambda: ops.class_logprobs(l, labels, num=torch.tensor([1], device="cuda")),
           lambda: ops.class_logprobs(torch.zeros(1, 3, 4, 5, 6, device="cuda").permute(0, 1, 4, 2, 3), torch.zeros(1, 6, 4, 5, dtype=torch.int64, device="cuda")),
           lambda: ops.class_logprobs_backward(l, labels, norm, h, ga[:2]), lambda: ops.class_logprobs_backward(l, labels, norm[:, :1], h, ga),
           lambda: ops.class_logprobs_backward(l, labels, norm, h, None), lambda: ops.distill_loss(l, kept, cls, 0.0),
           lambda: ops.distill_loss(l, kept, cls, float("nan")), lambda: ops.distill_loss(l, kept, cls[:, :2]), lambda: ops.distill_loss(l, kept.half(), cls),
           lambda: ops.distill_loss(l, kept[:, :0], cls[:, :0]), lambda: ops.distill_loss(l, kept.repeat(1, 50), cls.repeat(1, 50)),
           lambda: ops.distill_loss_backward(l, kept, cls, norm, ga[:3])]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.Sis3dError):
            f()
            pytest.fail("refusal %d" % i)
    with pytest.raises(ops.Sis3dUnsupported):
        ops.class_logprobs(torch.zeros(1, 1025, 8, device="cuda"), torch.zeros(1, 8, dtype=torch.int64, device="cuda"))
    with pytest.raises(_lib.Sis3dError):
        ops.class_logprobs(l, labels, num=3)
    assert torch.equal(ops.class_logprobs(labels=labels, score=l)[0], ops.class_logprobs(score=l, labels=labels)[0])
    # empty batches give empty outputs
    e = ops.class_logprobs(l[:0], labels[:0], top=2)
    assert e[0].shape == (0,) and e[4].shape == (0, 2)
    assert ops.class_logprobs_backward(l[:0], labels[:0], e[2], e[1], ga[:0]).shape == (0, 10)
    loss, n2 = ops.distill_loss(l[:0], kept[:0], cls[:0])
    assert loss.shape == (0,) and ops.distill_loss_backward(l[:0], kept[:0], cls[:0], n2, ga[:0]).shape == (0, 10)


def test_abi_refuses_bad_arguments_without_a_gpu():
    from sis3d import _lib
    l = _lib.lib()
    p = ctypes.c_void_p(4096)                                                # never dereferenced
    f0 = dict(score=p, dtype=0, N=1, V=4, K=10, sn=0, sv=10, sc=1, labels=p, num=None, top=2, logp=p, entropy=p, norm=p, tl=p, tc=p, ws=None, wsb=0, st=None)

    def fwd(**k):
        return l.sis3d_class_logprobs_forward(*dict(f0, **k).values())
    for k in (dict(dtype=7), dict(N=-1), dict(V=-1), dict(K=0), dict(top=-1), dict(top=11), dict(K=50, top=33), dict(score=None), dict(labels=None),
              dict(logp=None), dict(norm=None), dict(tl=None), dict(tc=None), dict(score=ctypes.c_void_p(4097))):
        assert fwd(**k) == -1, k
    assert fwd(K=1025, sc=4) == -4
    assert fwd(V=0) == 0
    assert fwd(K=65536, sv=65536, wsb=0) == -3 and fwd(K=65536, sv=65536, wsb=1 << 30) == -1
    b0 = dict(score=p, dtype=0, N=1, V=4, K=10, sn=0, sv=10, sc=1, labels=p, num=None, norm=p, h=p, ga=p, ge=None, d=p, dn=0, dv=10, dc=1, st=None)
    for k in (dict(norm=None), dict(h=None), dict(ga=None), dict(d=None), dict(K=-3)):
        assert l.sis3d_class_logprobs_backward(*dict(b0, **k).values()) == -1, k
    assert l.sis3d_class_logprobs_backward(*dict(b0, K=2000, dc=2).values()) == -4
    d0 = dict(score=p, dtype=0, N=1, V=4, K=10, sn=0, sv=10, sc=1, kept=p, cls=p, nk=3, num=None, T=1.0, loss=p, norm=p, ws=None, wsb=0, st=None)
    for k in (dict(nk=0), dict(nk=129), dict(T=0.0), dict(T=-1.0), dict(T=float("nan")), dict(T=1e4), dict(kept=None), dict(cls=None), dict(loss=None)):
        assert l.sis3d_distill_forward(*dict(d0, **k).values()) == -1, k
    e0 = dict(score=p, dtype=0, N=1, V=4, K=10, sn=0, sv=10, sc=1, kept=p, cls=p, nk=3, num=None, T=1.0, norm=p, g=p, d=p, dn=0, dv=10, dc=1, st=None)
    for k in (dict(nk=0), dict(T=0.0), dict(norm=None), dict(g=None), dict(d=None)):
        assert l.sis3d_distill_backward(*dict(e0, **k).values()) == -1, k
    # more rows than a launch has threads for
    many = dict(V=1 << 30, K=5000, sv=5000, top=0)
    assert fwd(**many) == -4 and fwd(**dict(many, K=600)) == -4 and fwd(**dict(many, K=400, top=5)) == -4 and fwd(**dict(many, K=400)) == -4
    many = dict(V=1 << 30, K=5000, sv=5000)
    assert l.sis3d_class_logprobs_backward(*dict(b0, **many).values()) == -4 and l.sis3d_distill_backward(*dict(e0, **many, ).values()) == -4
    assert l.sis3d_distill_backward(*dict(e0, **dict(many, K=400)).values()) == -4
    assert l.sis3d_class_rows_workspace_bytes(200, 19, 1, 3) == 0 and l.sis3d_class_rows_workspace_bytes(2, 65536, 1, 3) > 0


def test_reference_gradients_are_slopes():
    """the oracle of this file: its gradients are autograd's in 64 bits (CPU)"""
    g = torch.Generator().manual_seed(0)
    l = torch.randn(9, 13, generator=g, dtype=torch.float64, requires_grad=True)
    labels = torch.randint(-1, 13, (9,), generator=g)
    ga, ge = torch.randn(9, generator=g, dtype=torch.float64), torch.randn(9, generator=g, dtype=torch.float64)
    lp = torch.log_softmax(l, 1)
    logp = torch.where(labels >= 0, lp.gather(1, labels.clamp_min(0)[:, None])[:, 0], 0.0)
    h = -(lp * lp.exp()).sum(1)
    want, = torch.autograd.grad((logp * ga).sum() + (h * ge).sum(), l)
    got = ref_logprobs(l.detach(), labels, 3, ga, ge)
    assert torch.allclose(got["dscore"], want, atol=1e-13) and torch.allclose(got["logp"], logp.detach()) and torch.allclose(got["entropy"], h.detach())
    kept = torch.randn(9, 4, generator=g, dtype=torch.float64)
    cls = torch.randint(-1, 13, (9, 4), generator=g)
    cls[0, 0] = 3
    T = 1.7
    q = torch.softmax(torch.where(cls >= 0, kept / T, -math.inf), 1).nan_to_num(0.0)
    lt = torch.log_softmax(l / T, 1)
    loss = T * T * torch.where(q > 0, q * (q.clamp_min(1e-300).log() - lt.gather(1, cls.clamp_min(0))), 0.0).sum(1)
    want, = torch.autograd.grad((loss * ga).sum(), l)
    got = ref_distill(l.detach(), kept, cls, T, ga)
    assert torch.allclose(got["loss"], loss.detach()) and torch.allclose(got["dscore"], want, atol=1e-13)


def test_abi_takes_empty_batches_of_any_number_of_classes():
    """no rows: nothing to do, whatever the class list is (the rule that splits few long rows divides by their number)"""
    from sis3d import _lib
    l = _lib.lib()
    p = ctypes.c_void_p(4096)                                                # never dereferenced
    for N, V in ((1, 0), (0, 1), (0, 0), (0, 200)):
        for K in (1, 1000, 1025, 4096, 4097, 20011, 65536):
            rows = [p, 0, N, V, K, K * V, K, 1]
            assert l.sis3d_class_logprobs_forward(*rows, p, None, 1, p, p, p, p, p, None, 0, None) == 0, (N, V, K)
            assert l.sis3d_class_logprobs_backward(*rows, p, None, p, p, p, None, p, K * V, K, 1, None) == 0, (N, V, K)
            assert l.sis3d_distill_forward(*rows, p, p, 3, None, 1.0, p, p, None, 0, None) == 0, (N, V, K)
            assert l.sis3d_distill_backward(*rows, p, p, 3, None, 1.0, p, p, p, K * V, K, 1, None) == 0, (N, V, K)
            assert l.sis3d_class_rows_workspace_bytes(N * V, K, 1, 5) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 10), (0, 4097), (0, 20011), (2, 20011, 0), (0, 20011, 7), (2, 41, 0), (0, 41, 3, 2)])
def test_empty_batches(shape):
    """a scene without detections, against short and long class lists: empty outputs, empty gradients"""
    from sis3d import ops
    rows = shape[:1] + shape[2:]
    n = len(shape)
    score = torch.empty(rows + shape[1:2], device="cuda").permute(0, n - 1, *range(1, n - 1))       # classes last in memory
    assert score.shape == shape
    labels = torch.empty(rows, dtype=torch.int64, device="cuda")
    logp, h, norm, tl, tc = ops.class_logprobs(score, labels, top=3)
    assert logp.shape == rows and h.shape == rows and norm.shape == rows + (2,) and tl.shape == tc.shape == rows + (3,)
    assert ops.class_logprobs_backward(score, labels, norm, h, logp, h).shape == shape
    kept, cls = torch.empty(rows + (4,), device="cuda"), torch.empty(rows + (4,), dtype=torch.int64, device="cuda")
    loss, n2 = ops.distill_loss(score, kept, cls, 2.0)
    assert loss.shape == rows and ops.distill_loss_backward(score, kept, cls, n2, loss, 2.0).shape == shape


# rows whose largest score is a little below the lower end of the range that the fast sums take (l log2(e) / T = -2^22): the largest term is
# still a number there, terms within 2^24 of it are not any more.  How far below, in powers of two; 0 and less: still inside
BELOW = [-3, -0.25, 0.25, 1, 24, 64, 90, 99, 102, 105, 108, 112, 116, 120, 124, 126, 128, 140, 149, 151, 200, 1000]


def rows_below_the_range(K, T):
    """a row for each of BELOW: neighbouring numbers, at most 12 powers of two apart"""
    c2 = 1.4426950408889634 / T
    top = torch.tensor([-(2.0 ** 22 + b) / c2 for b in BELOW], dtype=torch.float64)
    g = torch.Generator().manual_seed(K)
    down = 12 / c2 * torch.rand(len(BELOW), K, generator=g, dtype=torch.float64)
    down[:, K // 2] = 0
    return (top[:, None] - down).float().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [2, 19, 41, 64, 300, 530, 1000, 1025, 4096, 5000, 20011, 65536])
@pytest.mark.parametrize("how", ["rows", "wide", "planar"])
def test_rows_just_below_the_range_of_the_fast_sums(K, how):
    if how == "planar" and K > 1024:
        how = "channels_last"
    R = len(BELOW)
    labels = (torch.arange(R, device="cuda") * 7) % K
    ga, ge = torch.ones(R, device="cuda"), torch.full((R,), 0.5, device="cuda")
    l = rows_below_the_range(K, 1.0)
    for top in (0, min(K, 3)):
        check_logprobs(l, labels, ga, ge, top, torch.float32, how)
    # so many rows that a lane, 16 lanes or a wave has one
    n = max(1, min(200, int(4e6) // (K * R)))
    check_logprobs(l.repeat(n, 1), labels.repeat(n), ga.repeat(n), ge.repeat(n), 1, torch.float32, how)
    for T in (1.0, 1e-3, 2.0 ** -9):
        l = rows_below_the_range(K, T)
        g = torch.Generator(device="cuda").manual_seed(K)
        cls = torch.randint(0, K, (R, 5), device="cuda", generator=g)
        kept = l.gather(1, cls) + 2 * T * torch.randn(R, 5, device="cuda", generator=g)
        check_distill(l, kept, cls, T, torch.float32, how)
        check_distill(l.repeat(n, 1), kept.repeat(n, 1), cls.repeat(n, 1), T, torch.float32, how)

"""Group norm with an activation on channels-last rows (csrc/group_norm.hip) against the formulas in 64 bits.

Tolerances (u = 2^-24, the rounding of a 32-bit operation; half = eps(type) / 2, the rounding of a result):
  h    (x - mu) r with mu and r rounded once: th = 4 u (|mu| r + |h|)
  y    (x - mu) sc + b, sc = r w: ty = 16 u (|mu| r |w| + |h w| + |z| + |b|), which also holds the few roundings of a smooth activation
       (its slope is at most 1.1); + half |y|
  d    dy act'(z): SiLU's slope changes by at most 0.5 a unit of z: td = 0.5 ty |dy|, 0 for the others; te = td |w| for e = d w
  dx   r (e - m1 - h m2): its own roundings, the errors of e, h, m1, m2, and sums of at most L rows a thread in m1 and m2; + half |dx|
  dw   sum d h: a thread's chain of at most L additions, 64 bits behind it: sum (L u |d h| + td |h| + |d| th); db alike: sum (L u |d| + td)
ReLU's slope jumps at 0: dy is 0 where |z| < 1e-3, so that a rounding of z cannot decide it."""
import ctypes

import pytest
import torch

U = 2.0 ** -24
EPS = 1e-5


def reference(x, dy, offsets, groups, w, b, act, eps=EPS):
    """x, dy: (rows, C) float64, offsets: list -> dict of float64 tensors, dy's zeroing near ReLU's corner included"""
    C = x.shape[1]
    c = C // groups
    w = torch.ones(C, dtype=x.dtype, device=x.device) if w is None else w.double()
    b = torch.zeros(C, dtype=x.dtype, device=x.device) if b is None else b.double()
    out = {k: torch.zeros_like(x) for k in ("y", "z", "hw", "dx", "ty", "tdx")}
    out["mean"], out["rstd"] = (torch.zeros(len(offsets) - 1, groups, dtype=x.dtype, device=x.device) for _ in range(2))
    for k in ("dw", "db", "tdw", "tdb"):
        out[k] = torch.zeros(C, dtype=x.dtype, device=x.device)
    for s, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if hi == lo:
            continue
        v = x[lo:hi].reshape(hi - lo, groups, c)
        mu = v.mean((0, 2), keepdim=True)
        r = 1 / torch.sqrt(((v - mu) ** 2).mean((0, 2), keepdim=True) + eps)
        h = (v - mu) * r
        ws, bs = w.view(groups, c), b.view(groups, c)
        z = h * ws + bs
        sig = torch.sigmoid(z)
        y = {"none": z, "relu": z.clamp_min(0), "silu": z * sig}[act]
        slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": sig * (1 + z * (1 - sig))}[act]
        d = dy[lo:hi].reshape(v.shape) * slope
        e = d * ws
        m1, m2 = e.mean((0, 2), keepdim=True), (e * h).mean((0, 2), keepdim=True)
        L = 16 + min(hi - lo, 4096)
        put = lambda k, t: out[k].__setitem__(slice(lo, hi), t.reshape(hi - lo, C))       # noqa: E731
        mean = lambda t: t.mean((0, 2), keepdim=True)                                    # noqa: E731
        th = 4 * U * (mu.abs() * r + h.abs())
        ty = 16 * U * (mu.abs() * r * ws.abs() + (h * ws).abs() + z.abs() + bs.abs())
        td = 0.5 * ty * dy[lo:hi].reshape(v.shape).abs() * (act == "silu")
        te = td * ws.abs()
        put("y", y)
        put("z", z)
        put("dx", r * (e - m1 - h * m2))
        put("ty", ty)
        put("tdx", r * (32 * U * (e.abs() + m1.abs() + (h * m2).abs()) + te + m2.abs() * th + mean(te) + L * U * mean(e.abs())
                        + h.abs() * (mean(te * h.abs() + e.abs() * th) + L * U * mean((e * h).abs()))))
        out["mean"][s], out["rstd"][s] = mu.flatten(), r.flatten()
        out["dw"] += (d * h).sum(0).flatten()
        out["db"] += d.sum(0).flatten()
        out["tdw"] += (L * U * (d * h).abs() + td * h.abs() + d.abs() * th).sum(0).flatten()
        out["tdb"] += (L * U * d.abs() + td).sum(0).flatten()
    return out


def check_close(got, want, tol, name):
    got = got.double()
    bad = (got - want).abs() > tol
    assert torch.isfinite(got).all(), name
    assert not bad.any(), "%s: %d off, worst %.3g of its tolerance" % (name, int(bad.sum()), float(((got - want).abs() / (tol + 1e-30)).max()))


def half_of(dtype):
    return torch.finfo(dtype).eps / 2


def make(shape_rows, C, dtype, seed=0, shift=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)                            # noqa: E731
    x = (n(shape_rows, C) * (0.5 + torch.rand(C, device="cuda", generator=g)) + shift * n(C)).to(dtype)
    return x, n(shape_rows, C).to(dtype), 1 + 0.3 * n(C), 0.3 * n(C)


def away_from_corner(x, dy, offsets, groups, w, b, act):
    z = reference(x.double(), dy.double(), offsets, groups, w, b, act)["z"]
    return torch.where(z.abs() < 1e-3, torch.zeros_like(dy), dy)


def run_rows(x, dy, offsets, groups, w, b, act):
    from sis3d import ops
    off = torch.tensor(offsets, device="cuda")
    y, mean, rstd = ops.group_norm(x, groups, w, b, EPS, act=act, offsets=off, want_stats=True)
    dx, dw, db = ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, act=act, offsets=off)
    return y, mean, rstd, dx, dw, db


def compare_rows(got, want, dtype, has_w=True, has_b=True):
    y, mean, rstd, dx, dw, db = got
    h = half_of(dtype)
    check_close(y, want["y"], want["ty"] + h * want["y"].abs(), "y")
    check_close(dx, want["dx"], want["tdx"] + h * want["dx"].abs() + 1e-7 * (dtype == torch.float16), "dx")     # fp16: its smallest step
    check_close(mean, want["mean"], 4 * U * (want["mean"].abs() + 1 / want["rstd"].clamp_min(1e-30) * (want["rstd"] > 0)), "mean")
    check_close(rstd, want["rstd"], 8 * U * want["rstd"] * 4, "rstd")
    if has_w:
        check_close(dw, want["dw"], want["tdw"], "dw")
    if has_b:
        check_close(db, want["db"], want["tdb"], "db")


CHANNELS = [(128, 32), (128, 1), (64, 8), (32, 32), (24, 8), (20, 4), (19, 19), (6, 3), (5, 1), (2, 1), (1, 1), (256, 2), (514, 2), (1024, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("C,G", CHANNELS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_ragged_rows_match_formula(dtype, C, G, act):
    lens = [0, 1, 700, 0, 3, 129, 0]
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    x, dy, w, b = make(offsets[-1], C, dtype, seed=C * 7 + G)
    dy = away_from_corner(x, dy, offsets, G, w, b, act)
    compare_rows(run_rows(x, dy, offsets, G, w, b, act), reference(x.double(), dy.double(), offsets, G, w, b, act), dtype)


def cl(rows, N, dims):
    """(N*V, C) rows -> (N,C,*dims) in channels-last memory"""
    t = rows.view((N,) + tuple(dims) + (rows.shape[1],))
    n = t.dim()
    return t.permute(0, n - 1, *range(1, n - 1))


def rows_of(t):
    n = t.dim()
    return t.permute(0, *range(2, n), 1).reshape(-1, t.shape[1])


@pytest.mark.gpu
@pytest.mark.parametrize("N,dims,C,G,act", [(1, (12, 6, 12), 128, 16, "relu"), (1, (24, 12, 24), 64, 8, "silu"), (3, (5, 3, 7), 48, 16, "relu"),
                                            (2, (33, 17), 20, 5, "silu"), (4, (), 32, 8, "none"), (1, (1, 1, 1), 64, 8, "relu"),
                                            (2, (1, 1, 1), 8, 8, "silu"), (1, (96, 48, 96), 32, 8, "relu"), (7, (9,), 3, 1, "none")])
@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dense_maps_match_formula(N, dims, C, G, act, affine, dtype):
    from sis3d import ops
    V = 1
    for d in dims:
        V *= d
    offsets = [i * V for i in range(N + 1)]
    x, dy, w, b = make(N * V, C, dtype, seed=V)
    if not affine:
        w = b = None
    dy = away_from_corner(x, dy, offsets, G, w, b, act)
    want = reference(x.double(), dy.double(), offsets, G, w, b, act)
    xm, dm = cl(x, N, dims), cl(dy, N, dims)
    y, mean, rstd = ops.group_norm(xm, G, w, b, EPS, act=act, want_stats=True)
    dx, dw, db = ops.group_norm_backward(dm, xm, mean, rstd, G, w, b, act=act)
    assert y.shape == xm.shape and dx.shape == xm.shape and (dw is None) == (w is None)
    compare_rows((rows_of(y), mean, rstd, rows_of(dx), dw, db), want, dtype, affine, affine)
    assert torch.equal(ops.group_norm(xm, G, w, b, EPS, act=act), y)           # without statistics, and the same bits again


@pytest.mark.gpu
def test_strides_slices_alignment_and_out():
    """a channel range of a wider tensor, a view that starts off 16 bytes, interleaved samples, writing into a range and in place"""
    from sis3d import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(2, 6, 5, 4, 96, device="cuda", generator=g).permute(0, 4, 1, 2, 3)
    dyw = torch.randn(2, 6, 5, 4, 96, device="cuda", generator=g).permute(0, 4, 1, 2, 3)
    for lo, hi, G in ((32, 64, 8), (1, 33, 4), (90, 96, 3)):
        x, dy = wide[:, lo:hi], dyw[:, lo:hi]
        dense = x.permute(0, 2, 3, 4, 1).contiguous()
        n = hi - lo
        w, b = torch.rand(n, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
        want = reference(dense.view(-1, n).double(), dy.permute(0, 2, 3, 4, 1).reshape(-1, n).double(), [0, 120, 240], G, w, b, "silu")
        y, mean, rstd = ops.group_norm(x, G, w, b, act="silu", want_stats=True)
        grads = ops.group_norm_backward(dy, x, mean, rstd, G, w, b, act="silu")
        compare_rows((rows_of(y), mean, rstd, rows_of(grads[0])) + grads[1:], want, torch.float32)
        target = torch.full_like(wide, 7.0)
        before = target.clone()
        assert ops.group_norm(x, G, w, b, act="silu", out=target[:, lo:hi]) .data_ptr() == target[:, lo:hi].data_ptr()
        check_close(rows_of(target[:, lo:hi]), want["y"], want["ty"] + half_of(torch.float32) * want["y"].abs(), "out")
        target[:, lo:hi] = 7.0
        assert torch.equal(target, before)                                     # nothing beside the range
        inplace = x.clone(memory_format=torch.preserve_format)
        inplace = cl(rows_of(inplace).contiguous(), 2, (6, 5, 4))
        ops.group_norm(inplace, G, w, b, act="silu", out=inplace)
        check_close(rows_of(inplace), want["y"], want["ty"] + half_of(torch.float32) * want["y"].abs(), "in place")
    # samples interleaved in memory: (voxels, samples, channels)
    m = torch.randn(50, 3, 16, device="cuda", generator=g)
    x = m.permute(1, 2, 0)
    want = reference(m.permute(1, 0, 2).reshape(-1, 16).double(), torch.zeros(150, 16, device="cuda", dtype=torch.float64), [0, 50, 100, 150], 4, None, None, "none")
    check_close(ops.group_norm(x, 4).permute(0, 2, 1).reshape(-1, 16), want["y"], want["ty"] + half_of(torch.float32) * want["y"].abs(), "interleaved")


@pytest.mark.gpu
def test_rows_behind_the_last_sample_and_empty_batches():
    from sis3d import ops
    x, dy, w, b = make(1000, 32, torch.float32)
    off = torch.tensor([0, 40, 40, 900], device="cuda")
    out = torch.full((1000, 32), 3.0, device="cuda")
    y, mean, rstd = ops.group_norm(x, 8, w, b, offsets=off, out=out, want_stats=True)
    assert (y[900:] == 3.0).all()
    assert (mean[1] == 0).all() and (rstd[1] == 0).all()
    fresh = ops.group_norm(x, 8, w, b, offsets=off)
    assert torch.equal(fresh[:900], y[:900]) and (fresh[900:] == 0).all()
    dirty = dy.clone()
    dirty[900:] = float("nan")
    dx, dw, db = ops.group_norm_backward(dirty, x, mean, rstd, 8, w, b, offsets=off)
    assert (dx[900:] == 0).all() and torch.isfinite(dw).all() and torch.isfinite(dx).all()
    # no samples, no rows
    none = torch.tensor([0], device="cuda")
    assert (ops.group_norm(x, 8, w, b, offsets=none) == 0).all()
    m0 = torch.empty(0, 8, device="cuda")
    dx, dw, db = ops.group_norm_backward(dy, x, m0, m0, 8, w, b, offsets=none)
    assert (dx == 0).all() and (dw == 0).all() and (db == 0).all()
    e = torch.empty(0, 32, device="cuda")
    y, mean, rstd = ops.group_norm(e, 8, w, b, offsets=torch.zeros(3, dtype=torch.int64, device="cuda"), want_stats=True)
    assert y.shape == (0, 32) and (mean == 0).all() and mean.shape == (2, 8)
    dx, dw, db = ops.group_norm_backward(e, e, mean, rstd, 8, w, b, offsets=torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert (dw == 0).all() and (db == 0).all()
    e5 = ops.new_act(32, (0, 4, 4), "cuda")
    y, mean, rstd = ops.group_norm(e5, 8, w, b, want_stats=True)
    assert y.numel() == 0 and (rstd == 0).all()
    # offsets that decrease or leave the buffer are empty / cut samples, never rows outside it
    y = ops.group_norm(x, 8, w, b, offsets=torch.tensor([0, 500, 20, 5000], device="cuda"))
    assert y.shape == (1000, 32)


@pytest.mark.gpu
def test_many_samples_and_one_row_each():
    lens = [(i * 37) % 5 for i in range(5000)]
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    from sis3d import ops
    x, dy, w, b = make(offsets[-1], 16, torch.float32)
    y, mean, rstd = ops.group_norm(x, 4, w, b, offsets=torch.tensor(offsets, device="cuda"), want_stats=True)
    pick = [i for i in range(0, 5000, 97)]
    for s in pick:
        lo, hi = offsets[s], offsets[s + 1]
        want = reference(x[lo:hi].double(), dy[lo:hi].double(), [0, hi - lo], 4, w, b, "none")
        check_close(y[lo:hi], want["y"], want["ty"] * 4 + half_of(torch.float32) * want["y"].abs(), "sample %d" % s)


@pytest.mark.gpu
@pytest.mark.parametrize("C,G", [(256, 32), (96, 32), (20, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_samples_around_a_large_one(dtype, C, G):
    """workgroups with whole rows, offsets that are far from their even places"""
    lens = [(i * 37) % 6 for i in range(300)] + [40000] + [(i * 11) % 5 for i in range(400)] + [0, 0]
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    x, dy, w, b = make(offsets[-1], C, dtype, seed=C)
    compare_rows(run_rows(x, dy, offsets, G, w, b, "silu"), reference(x.double(), dy.double(), offsets, G, w, b, "silu"), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("C,G", [(96, 32), (48, 16), (40, 8), (80, 16), (160, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [(1872, 700, 40, 2028), (600, 171, 510)])
@pytest.mark.parametrize("odd", [0, 1])
def test_last_channels_narrower_than_the_others(dtype, C, G, lens, odd):
    """the groups that are left over have more rows in parallel than the others: all of them count.  odd: rows off 16 bytes"""
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    x, dy, w, b = make(offsets[-1], C, dtype, seed=C)
    if odd:
        wide = torch.zeros(2, offsets[-1], C + 3, dtype=dtype, device="cuda")
        wide[0, :, 1:1 + C], wide[1, :, 1:1 + C] = x, dy
        x, dy = wide[0, :, 1:1 + C], wide[1, :, 1:1 + C]
    compare_rows(run_rows(x, dy, offsets, G, w, b, "silu"), reference(x.double(), dy.double(), offsets, G, w, b, "silu"), dtype)
    from sis3d import ops
    dense = x[:600][None].permute(0, 2, 1)                                      # a dense sample, one launch or two
    y = ops.group_norm(dense, G, w, b, EPS, act="silu")
    want = reference(x[:600].double(), dy[:600].double(), [0, 600], G, w, b, "silu")
    check_close(y[0].t(), want["y"], want["ty"] + half_of(dtype) * want["y"].abs(), "dense y")


@pytest.mark.gpu
@pytest.mark.parametrize("C,G", [(1024, 1024), (2048, 1024), (520, 520)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_groups_than_threads(dtype, C, G):
    lens = [3, 0, 1, 5, 2]
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    x, dy, w, b = make(offsets[-1], C, dtype, seed=C)
    want = reference(x.double(), dy.double(), offsets, G, w, b, "silu")
    compare_rows(run_rows(x, dy, offsets, G, w, b, "silu"), want, dtype)
    from sis3d import ops
    for n, v in ((1, 11), (11, 1)):                                              # dense: one sample of all rows, and one of each
        off = list(range(0, 12, v))
        want = reference(x.double(), dy.double(), off, G, w, b, "silu")
        y, mean, rstd = ops.group_norm(x.view(n, v, C).permute(0, 2, 1), G, w, b, EPS, act="silu", want_stats=True)
        dx, dw, db = ops.group_norm_backward(dy.view(n, v, C).permute(0, 2, 1), x.view(n, v, C).permute(0, 2, 1), mean, rstd, G, w, b, act="silu")
        compare_rows((rows_of(y), mean, rstd, rows_of(dx), dw, db), want, dtype)


@pytest.mark.gpu
def test_large_mean_constant_and_non_finite_inputs():
    from sis3d import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    # deviation 1 around a mean of 4096: the variance must not cancel (u * 4096 is the rounding of the mean itself)
    x = 4096 + torch.randn(5000, 16, device="cuda", generator=g)
    y, mean, rstd = ops.group_norm(x, 2, offsets=torch.tensor([0, 5000], device="cuda"), want_stats=True)
    want = reference(x.double(), torch.zeros_like(x).double(), [0, 5000], 2, None, None, "none")
    assert ((rstd.double() - want["rstd"]).abs() <= 64 * U * want["rstd"]).all()
    check_close(y, want["y"], want["ty"], "y")
    # a constant map has variance 0 exactly: y is the bias
    b = torch.randn(16, device="cuda", generator=g)
    c = torch.full((300, 16), 1.7, device="cuda")
    assert torch.equal(ops.group_norm(c, 4, None, b, offsets=torch.tensor([0, 300], device="cuda")), b.expand(300, 16))
    # a NaN or an infinity stays in its own sample and group
    x = torch.randn(2, 4, 4, 4, 16, device="cuda", generator=g)
    clean = ops.group_norm(x.permute(0, 4, 1, 2, 3), 4, act="relu")
    for v in (float("nan"), float("inf")):
        d = x.clone()
        d[1, 2, 1, 3, 5] = v
        y = ops.group_norm(d.permute(0, 4, 1, 2, 3), 4, act="relu")
        assert torch.isnan(y[1, 4:8]).all()
        y[1, 4:8] = clean[1, 4:8]
        assert torch.equal(y, clean)


@pytest.mark.gpu
def test_streams_graph_and_determinism():
    from sis3d import ops
    x, dy, w, b = make(3456, 64, torch.float32)
    off = torch.tensor([0, 1000, 3456], device="cuda")

    def step():
        y, mean, rstd = ops.group_norm(x, 8, w, b, act="silu", offsets=off, want_stats=True)
        return (y,) + ops.group_norm_backward(dy, x, mean, rstd, 8, w, b, act="silu", offsets=off)
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
    keep = x.clone()
    for k in range(4):
        x.copy_(keep * (1 + k))
        off.copy_(torch.tensor([0, 1000 + k, 3456 - 5 * k]))
        graph.replay()
        torch.cuda.synchronize()
        again = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, again)), k


@pytest.mark.gpu
def test_more_than_two_to_the_31_elements():
    from sis3d import ops
    C, rows = 64, (1 << 31) // 64 + 1000
    x = torch.empty(rows, C, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(0, rows, 1 << 22):
        x[i:i + (1 << 22)].normal_(generator=g)
    off = torch.tensor([0, rows - 700, rows], device="cuda")
    y, mean, rstd = ops.group_norm(x, 8, offsets=off, want_stats=True)
    tail = x[rows - 700:].clone()
    want = reference(tail.double(), torch.zeros_like(tail).double(), [0, 700], 8, None, None, "none")
    check_close(y[rows - 700:], want["y"], want["ty"] + half_of(torch.bfloat16) * want["y"].abs(), "tail")
    # 2^31 standard normal values a sample: mean 0 and deviation 1 to a few parts in 10^4 (2^-14 is one deviation of the mean of 2^28)
    assert float(mean[0].abs().max()) < 6 * 2.0 ** -14 and float((rstd[0] - 1).abs().max()) < 1e-3
    first = x[:512].double().view(512, 8, 8)
    z = (first - mean[0].double().view(8, 1)) * rstd[0].double().view(8, 1)
    check_close(y[:512], z.view(512, 64), half_of(torch.bfloat16) * z.view(512, 64).abs() + 1e-6, "head")
    dx, _, _ = ops.group_norm_backward(x, x, mean, rstd, 8, offsets=off)
    want = reference(tail.double(), tail.double(), [0, 700], 8, None, None, "none")
    check_close(dx[rows - 700:], want["dx"], want["tdx"] + half_of(torch.bfloat16) * want["dx"].abs(), "dx tail")


@pytest.mark.gpu
@pytest.mark.parametrize("dims,C,G", [((10, 9, 11), 32, 8), ((3, 2, 2), 12, 4), ((40, 33, 31), 64, 16)])
def test_relu_passes_a_gradient_exactly_where_it_passes_a_value(dims, C, G):
    """with dy = 1, dbias counts the elements whose gradient passes: whole numbers below 2^24, so no tolerance"""
    from sis3d import ops
    g = torch.Generator(device="cuda").manual_seed(C)
    # few different values: many elements within rounding of 0 after the bias, on both sides
    x = torch.randint(-3, 4, (2,) + dims + (C,), device="cuda", generator=g).float().permute(0, 4, 1, 2, 3)
    w = 1 + torch.rand(C, device="cuda", generator=g)
    b = torch.zeros(C, device="cuda")
    for _ in range(2):
        y, mean, rstd = ops.group_norm(x, G, w, b, act="relu", want_stats=True)
        dx, dw, db = ops.group_norm_backward(torch.ones_like(x), x, mean, rstd, G, w, b, act="relu")
        assert torch.equal(db, (y > 0).sum((0, 2, 3, 4)).float())
        h = (1.0 - mean.view(2, G, 1)) * rstd.view(2, G, 1)                  # of the value 1: a bias that takes it to 0, but for a rounding
        b = -(h.expand(2, G, C // G).reshape(2, C)[0] * w)


@pytest.mark.gpu
def test_autograd_module_and_differences():
    """HipGroupNorm in a training step: autograd's gradients are the operator's, and they are the slope of the loss"""
    from sis3d import ops
    from sis3d.nets.backbones import HipGroupNorm
    g = torch.Generator(device="cuda").manual_seed(5)
    m = HipGroupNorm(4, 32, act="silu").cuda()
    with torch.no_grad():
        m.weight.normal_(1, 0.2, generator=g)
        m.bias.normal_(0, 0.2, generator=g)
    assert set(m.state_dict()) == {"weight", "bias"}
    x = torch.randn(1, 5, 6, 7, 32, device="cuda", generator=g).permute(0, 4, 1, 2, 3).requires_grad_(True)
    t = torch.randn(1, 32, 5, 6, 7, device="cuda", generator=g)              # planar: its gradient arrives planar
    (m(x) * t).sum().backward()
    y, mean, rstd = ops.group_norm(x.detach(), 4, m.weight.detach(), m.bias.detach(), m.eps, act="silu", want_stats=True)
    dx, dw, db = ops.group_norm_backward(t.contiguous(memory_format=torch.channels_last_3d), x.detach(), mean, rstd, 4, m.weight.detach(),
                                         m.bias.detach(), act="silu")
    assert torch.equal(x.grad, dx) and torch.equal(m.weight.grad, dw) and torch.equal(m.bias.grad, db)
    # central differences along random directions, step 2^-6: the rounding of y (u |y| a value, 6720 values, in quadrature) over the step is
    # below 1e-3, the third derivative's share step^2 / 6 times one of order the gradient: both against |grad . v| of order 10..100
    with torch.no_grad():
        for leaf, grad in ((x, dx), (m.weight, dw), (m.bias, db)):
            for k in range(3):
                v = torch.randn(leaf.shape, device="cuda", generator=g)
                keep, step = leaf.detach().clone(), 2.0 ** -6
                f = []
                for s in (step, -step):
                    leaf.copy_(keep + s * v)
                    f.append(float((m(x).double() * t.double()).sum()))
                leaf.copy_(keep)
                slope, want = (f[0] - f[1]) / (2 * step), float((grad.double() * v.double()).sum())
                assert abs(slope - want) <= 1e-3 * float((grad.double() * v.double()).abs().sum()) + 2e-3, (slope, want)


@pytest.mark.gpu
def test_crops_of_the_mask_head():
    """RaggedBatch.group_norm between the convolutions of packed crops: each crop as if it were alone"""
    from sis3d import ops
    windows = [(0, 0, 0, 9, 10, 11), (3, 2, 1, 4, 3, 2), (5, 5, 5, 17, 20, 14)]
    rb = ops.RaggedBatch(windows, torch.device("cuda"))
    g = torch.Generator(device="cuda").manual_seed(2)
    src = torch.randn(rb.voxels, 64, device="cuda", generator=g)
    w, b = torch.rand(64, device="cuda", generator=g), torch.rand(64, device="cuda", generator=g)
    got = rb.group_norm(src, 16, w, b, act="relu")
    for crop, one in zip(rb.views(src), rb.views(got)):
        alone = ops.group_norm(crop, 16, w, b, act="relu")
        # the same formula with other tiles of rows: two results within the tolerance of the formula each
        want = reference(rows_of(crop).double(), torch.zeros_like(rows_of(crop)).double(), [0, crop[0, 0].numel()], 16, w, b, "relu")
        for t in (alone, one):
            check_close(rows_of(t), want["y"], want["ty"] + half_of(torch.float32) * want["y"].abs(), "crop")


@pytest.mark.gpu
def test_refusals():
    from sis3d import _lib, ops
    x = torch.zeros(1, 4, 4, 4, 32, device="cuda").permute(0, 4, 1, 2, 3)
    w = torch.ones(32, device="cuda")
    bad = [lambda: ops.group_norm(x, 5), lambda: ops.group_norm(x, 0), lambda: ops.group_norm(x, 8, act="gelu"),
           lambda: ops.group_norm(x.contiguous(), 8), lambda: ops.group_norm(x.double(), 8), lambda: ops.group_norm(x, 8, w[:16]),
           lambda: ops.group_norm(x, 8, w.half()), lambda: ops.group_norm(x, 8, w.cpu()), lambda: ops.group_norm(x[:, 0, 0, 0, 0], 1),
           lambda: ops.group_norm(x, 8, offsets=torch.tensor([0, 64], device="cuda")),
           lambda: ops.group_norm(rows_of(x), 8, offsets=torch.tensor([0, 64], device="cuda", dtype=torch.int32)),
           lambda: ops.group_norm(rows_of(x), 8, offsets=torch.tensor([0, 64])),
           lambda: ops.group_norm(x, 8, out=torch.zeros(1, 32, 4, 4, 4, device="cuda")),
           lambda: ops.group_norm(x, 8, out=torch.zeros_like(x).half()),
           lambda: ops.group_norm(x.expand(2, -1, -1, -1, -1), 8, out=x.expand(2, -1, -1, -1, -1)),
           lambda: ops.group_norm_backward(x.half(), x, torch.zeros(1, 8, device="cuda"), torch.zeros(1, 8, device="cuda"), 8),
           lambda: ops.group_norm_backward(x, x, torch.zeros(1, 4, device="cuda"), torch.zeros(1, 8, device="cuda"), 8),
           lambda: ops.group_norm(x.cpu(), 8), lambda: ops.group_norm(x, 8, eps=-1.0), lambda: ops.group_norm(x, 8, eps=float("nan"))]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.Sis3dError):
            f()
            pytest.fail("refusal %d" % i)
    with pytest.raises(ops.Sis3dUnsupported):
        ops.group_norm(torch.zeros(1, 4099, 2, device="cuda").permute(0, 2, 1).contiguous().permute(0, 2, 1), 1)
    # keywords throughout; a group count that is a tensor counts by its value
    n = torch.tensor(4)
    y = ops.group_norm(x=x + torch.arange(32., device="cuda").view(1, 32, 1, 1, 1), groups=n)
    n.fill_(32)
    assert float(y.abs().max()) > 1 and float(ops.group_norm(x=x + torch.arange(32., device="cuda").view(1, 32, 1, 1, 1), groups=n).abs().max()) == 0


def test_abi_refuses_bad_arguments_without_a_gpu():
    """every check of the C entry points comes before the first launch: codes, no device needed"""
    from sis3d import _lib
    l = _lib.lib()
    p = ctypes.c_void_p(4096)                                                # never dereferenced
    fwd = dict(x=p, dtype=0, S=1, rows=10 ** 6, off=None, xn=0, xv=32, C=32, G=8, w=None, b=None, eps=1e-5, act=0, y=p, yn=0, yv=32, tail=0, mean=None,
               rstd=None, ws=p, wsb=1 << 30, stream=None)

    def forward(**k):
        return l.sis3d_group_norm_forward(*dict(fwd, **k).values())
    for k in (dict(dtype=3), dict(S=-1), dict(rows=-1), dict(C=0), dict(G=0), dict(G=5), dict(act=3), dict(act=-1), dict(x=None), dict(y=None),
              dict(mean=p), dict(eps=-1.0), dict(eps=float("nan")), dict(ws=None), dict(ws=ctypes.c_void_p(4100))):
        assert forward(**k) == -1, k
    assert forward(wsb=0) == -3
    assert forward(C=4099, G=1, xv=4099, yv=4099) == -4
    assert forward(rows=0) == 0 and forward(S=0) == 0
    bwd = dict(dy=p, dn=0, dv=32, x=p, dtype=0, S=1, rows=10 ** 6, off=None, xn=0, xv=32, C=32, G=8, mean=p, rstd=p, w=None, b=None, act=0, dx=p, gn=0,
               gv=32, dw=None, db=None, ws=p, wsb=1 << 30, stream=None)

    def backward(**k):
        return l.sis3d_group_norm_backward(*dict(bwd, **k).values())
    for k in (dict(dtype=-1), dict(dy=None), dict(dx=None), dict(mean=None), dict(rstd=None), dict(G=3), dict(ws=None)):
        assert backward(**k) == -1, k
    assert backward(wsb=16) == -3 and backward(rows=0) == 0
    # more samples than a launch has workgroups
    assert forward(S=1 << 23, rows=1, wsb=1 << 50) == -4 and backward(S=1 << 23, rows=1, wsb=1 << 50) == -4
    assert l.sis3d_group_norm_workspace_bytes(0, 1, 10, 0, 32, 5, 0) == 0
    for ragged in (0, 1):
        for backward in (0, 1):
            assert l.sis3d_group_norm_workspace_bytes(0, 0, 0, ragged, 32, 8, backward) >= 0        # no rows: an answer, not a division by them
            assert l.sis3d_group_norm_workspace_bytes(2, 3, 0, ragged, 32, 8, backward) >= 0
    # one launch, nothing to keep, where a sample is small; a sum over several samples' gradients takes two
    size = l.sis3d_group_norm_workspace_bytes
    assert size(0, 1, 10 ** 6, 0, 32, 8, 1) > 0 and size(0, 1, 10, 0, 32, 8, 1) == 0 and size(0, 2, 10, 0, 32, 8, 0) == 0 and size(0, 2, 10, 0, 32, 8, 1) > 0


def test_reference_gradients_are_slopes():
    """the oracle of this file: its gradients are autograd's in 64 bits (CPU)"""
    g = torch.Generator().manual_seed(0)
    for act in ("none", "relu", "silu"):
        x = torch.randn(23, 12, generator=g, dtype=torch.float64, requires_grad=True)
        w, b = (torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
        dy = torch.randn(23, 12, generator=g, dtype=torch.float64)
        parts = []
        for lo, hi in ((0, 9), (9, 23)):
            z = torch.nn.functional.group_norm(x[lo:hi].t()[None], 3, w, b, EPS)
            parts.append({"none": z, "relu": z.relu(), "silu": z * z.sigmoid()}[act][0].t())
        y = torch.cat(parts)
        dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
        got = reference(x.detach(), dy, [0, 9, 23], 3, w.detach(), b.detach(), act)
        for k, v in (("y", y.detach()), ("dx", dx), ("dw", dw), ("db", db)):
            assert torch.allclose(got[k], v, rtol=1e-10, atol=1e-12), (act, k)


def stats_of(rows, offsets, G):
    """mean, variance and 1 / sqrt(var + eps) of float64 rows, per sample and group: deviations from the mean itself"""
    C = rows.shape[1]
    mean, rstd = [], []
    for lo, hi in zip(offsets, offsets[1:]):
        v = rows[lo:hi].reshape(hi - lo, G, C // G)
        mu = v[:1, :, :1] + (v - v[:1, :, :1]).mean((0, 2), keepdim=True)
        mean.append(mu.flatten())
        rstd.append(1 / torch.sqrt(((v - mu) ** 2).mean((0, 2)) + EPS))
    return torch.stack(mean), torch.stack(rstd)


@pytest.mark.gpu
@pytest.mark.parametrize("level", [0.0, 1.7, 1e5, 3e5, 1e6, -1.2345e7])
@pytest.mark.parametrize("C,G", [(16, 4), (32, 8), (20, 4), (19, 19), (64, 1), (6, 3), (1024, 4)])
def test_statistics_of_a_large_mean_do_not_cancel(level, C, G):
    """Constant maps and maps of two neighbouring numbers at a level that is far from 0: the variance is 0, or the square of a step.
    rstd: a thread's variance of n rows has a relative error of a few n u at most (differences of neighbours are exact), joined in 64 bits:
    32 u as everywhere here.  The mean, rounded to 32 bits, is off by u |mean| and a few u deviations."""
    from sis3d import ops
    g = torch.Generator(device="cuda").manual_seed(C)
    lens = [13825, 1, 0, 300, 4097]
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    R = offsets[-1]
    live = [i for i, n in enumerate(lens) if n]
    base = torch.full((R, C), level, device="cuda")
    step = torch.nextafter(base[0, 0].cpu(), torch.tensor(float("inf"))).item() - base[0, 0].item()
    one = base + (torch.rand(R, C, device="cuda", generator=g) < 0.3) * step
    ramp = base + torch.randint(0, 16, (R, C), device="cuda", generator=g) * step
    corner = base.clone()                                        # a map that is constant but for the first row
    corner[0] += 64 * step
    cases = [(base, torch.float32), (one, torch.float32), (ramp, torch.float32), (corner, torch.float32)]
    cases += [(base, d) for d in (torch.bfloat16, torch.float16) if abs(level) < torch.finfo(d).max]
    for x, dtype in cases:
        x = x.to(dtype)
        _, mean, rstd = ops.group_norm(x, G, offsets=torch.tensor(offsets, device="cuda"), want_stats=True)
        wm, wr = stats_of(x.double(), [offsets[i] for i in live] + [R], G)
        check_close(rstd[live], wr, 32 * U * wr, "rstd")
        check_close(mean[live], wm, 4 * U * wm.abs() + 4 * U / wr, "mean")
        for lo, n in ((0, 13825), (offsets[3], 300)):            # dense: two launches and one
            _, mean, rstd = ops.group_norm(x[lo:lo + n][None].permute(0, 2, 1), G, want_stats=True)
            wm, wr = stats_of(x[lo:lo + n].double(), [0, n], G)
            check_close(rstd, wr, 32 * U * wr, "dense rstd")
            check_close(mean, wm, 4 * U * wm.abs() + 4 * U / wr, "dense mean")


@pytest.mark.gpu
@pytest.mark.parametrize("C,G,R,dtype", [(511, 1, 60000, torch.float32), (511, 7, 60000, torch.float32), (2048, 1, 20000, torch.float32), (2048, 8, 40000, torch.float16),
                                         (256, 1, 40000, torch.float32), (32, 8, 200000, torch.float32), (19, 19, 40000, torch.bfloat16), (128, 16, 864, torch.float32)])
@pytest.mark.parametrize("level,peak", [(0.1, 10.0), (-0.37, 7.3), (0.1, 1234.567), (100.3, 0.1)])
def test_statistics_of_a_flat_map_with_a_few_peaks(C, G, R, dtype, level, peak):
    """Rows that stand out from a flat map, wherever in a tile they are, the first row of a thread among them: none may spoil the sums of the
    rows behind it.  A thread of n rows joins n / 4 batches, each off by a few u of its squared deviations, to the sum so far, one rounding
    each: (n / 4 + 16) u of the variance and half of it of rstd, with n <= 128 here: 24 u, and a rounding; 32 u as everywhere."""
    from sis3d import ops
    for first in (0, 1, R // 2, R - 1):
        x = torch.full((R, C), level, device="cuda")
        x[first] = peak
        if first == 1:
            x[::3001] = peak
        x = x.to(dtype)
        want = stats_of(x.double(), [0, R], G)
        for off in (None, torch.tensor([0, R], device="cuda")):
            _, mean, rstd = ops.group_norm(x if off is not None else x[None].permute(0, 2, 1), G, offsets=off, want_stats=True)
            check_close(rstd, want[1], 32 * U * want[1], "rstd, row %d" % first)
            check_close(mean, want[0], 4 * U * want[0].abs() + 4 * U / want[1], "mean, row %d" % first)


@pytest.mark.gpu
def test_crops_of_the_mask_head_in_training():
    """RaggedBatch.group_norm is differentiable: gradients of the source, the weight and the bias are the operator's"""
    from sis3d import ops
    windows = [(0, 0, 0, 9, 10, 11), (3, 2, 1, 4, 3, 2), (5, 5, 5, 17, 20, 14)]
    rb = ops.RaggedBatch(windows, torch.device("cuda"))
    g = torch.Generator(device="cuda").manual_seed(2)
    src = torch.randn(rb.voxels, 64, device="cuda", generator=g)
    w, b = torch.rand(64, device="cuda", generator=g), torch.rand(64, device="cuda", generator=g)
    dy = torch.randn(rb.voxels, 64, device="cuda", generator=g)
    y, mean, rstd = ops.group_norm(src, 16, w, b, act="silu", offsets=rb.offsets(), want_stats=True)
    want = ops.group_norm_backward(dy, src, mean, rstd, 16, w, b, act="silu", offsets=rb.offsets())
    for which in ((0, 1, 2), (0,), (1, 2)):                     # a leaf each, and constants beside it
        leaves = [t.clone().requires_grad_(i in which) for i, t in enumerate((src, w, b))]
        got = rb.group_norm(leaves[0], 16, leaves[1], leaves[2], act="silu")
        assert got.requires_grad and torch.equal(got.detach(), y)
        got.backward(dy)
        for i, t in enumerate(leaves):
            assert torch.equal(t.grad, want[i]) if i in which else t.grad is None
    leaf = src.clone().requires_grad_(True)
    rb.group_norm(leaf, 16).backward(dy)                        # no weight, no bias
    y, mean, rstd = ops.group_norm(src, 16, offsets=rb.offsets(), want_stats=True)
    assert torch.equal(leaf.grad, ops.group_norm_backward(dy, src, mean, rstd, 16, offsets=rb.offsets())[0])
    with torch.no_grad():
        got = rb.group_norm(leaf, 16)
    assert not got.requires_grad and torch.equal(got, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("affine", [True, False])
def test_module_in_16_bits(dtype, affine):
    """HipGroupNorm after .bfloat16() / .half(), as nn.GroupNorm: 16-bit parameters, taken at their value, and their gradients in 16 bits"""
    from sis3d import ops
    from sis3d.nets.backbones import HipGroupNorm
    g = torch.Generator(device="cuda").manual_seed(6)
    m = HipGroupNorm(8, 64, act="relu", affine=affine).cuda()
    if affine:
        with torch.no_grad():
            m.weight.normal_(1, 0.2, generator=g)
            m.bias.normal_(0, 0.2, generator=g)
    m = m.to(dtype)
    assert all(p.dtype is dtype for p in m.parameters()) and len(list(m.parameters())) == 2 * affine
    w, b = (m.weight.detach().float(), m.bias.detach().float()) if affine else (None, None)
    rows = torch.randn(700, 64, device="cuda", generator=g).to(dtype)
    dy = torch.randn(700, 64, device="cuda", generator=g).to(dtype)
    off = torch.tensor([0, 300, 700], device="cuda")
    for x, d, offsets in ((rows, dy, off), (rows[None].permute(0, 2, 1), dy[None].permute(0, 2, 1), None)):
        m.zero_grad()
        x = x.detach().requires_grad_(True)
        y = m(x, offsets)
        y.backward(d)
        want, mean, rstd = ops.group_norm(x.detach(), 8, w, b, m.eps, act="relu", offsets=offsets, want_stats=True)
        dx, dw, db = ops.group_norm_backward(d, x.detach(), mean, rstd, 8, w, b, act="relu", offsets=offsets)
        assert y.dtype is dtype and torch.equal(y.detach(), want) and torch.equal(x.grad, dx)
        if affine:
            assert torch.equal(m.weight.grad, dw.to(dtype)) and torch.equal(m.bias.grad, db.to(dtype))
    with torch.no_grad():
        assert torch.equal(m(rows, off), ops.group_norm(rows, 8, w, b, m.eps, act="relu", offsets=off))
    # fp32 maps between 16-bit parameters, and fp32 parameters at 16-bit maps
    assert torch.equal(m(rows.float(), off).detach(), ops.group_norm(rows.float(), 8, w, b, m.eps, act="relu", offsets=off))
    assert torch.equal(m.float()(rows, off).detach(), ops.group_norm(rows, 8, w, b, m.eps, act="relu", offsets=off))


@pytest.mark.gpu
@pytest.mark.parametrize("C,G", [(512, 8), (64, 1), (128, 16), (48, 16), (130, 10)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_mean_of_few_rows_is_rounded_once(C, G, dtype):
    """A thread's only row enters the mean in 64 bits: what comes out is the mean of the group rounded to 32 bits, however much of it cancels
    (u of it, and 2^-40 of the largest value for the additions in 64 bits)."""
    from sis3d import ops
    g = torch.Generator(device="cuda").manual_seed(C)
    x = torch.randn(3, C, device="cuda", generator=g) * 20
    x = (x - x.view(3, G, C // G).mean(2, keepdim=True).expand(-1, -1, C // G).reshape(3, C)).to(dtype)          # means of nearly 0
    for off in ([0, 1, 2, 3], [0, 3], [0, 1, 3]):
        want = stats_of(x.double(), off, G)
        _, mean, rstd = ops.group_norm(x, G, offsets=torch.tensor(off, device="cuda"), want_stats=True)
        check_close(mean, want[0], U * want[0].abs() + 2.0 ** -40 * 100, "mean")
        check_close(rstd, want[1], 32 * U * want[1], "rstd")


@pytest.mark.gpu
@pytest.mark.parametrize("C,G", [(512, 8), (64, 1), (48, 16), (130, 10)])
def test_one_row_whose_squares_are_beyond_32_bits(C, G):
    """a thread's only row needs no square in 32 bits: deviations of 1e25 and more still have their variance (rstd to 32 u)"""
    from sis3d import ops
    g = torch.Generator(device="cuda").manual_seed(C)
    x = torch.randn(2, C, device="cuda", generator=g) * 1e25
    want = stats_of(x.double(), [0, 1, 2], G)
    y, mean, rstd = ops.group_norm(x, G, offsets=torch.tensor([0, 1, 2], device="cuda"), want_stats=True)
    check_close(rstd, want[1], 32 * U * want[1], "rstd")
    check_close(mean, want[0], U * want[0].abs() + 2.0 ** -40 * 1e26, "mean")

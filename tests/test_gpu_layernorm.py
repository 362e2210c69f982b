"""layer_norm of noise_amd (csrc/layernorm.hip) against the formulas in 64 bits, its gradients against differences, and the
calls it refuses."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24            # half a step of fp32, relative


def chain(D):
    """Roundings on the longest path of a row sum: at most 64 values in one lane plus 8 exchange steps, or D / 256 per
    thread in the wide kernels; 8 more for the operations around it."""
    return max(72, D // 256 + 8) + 8


def rand(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def case(rows, D, dtype, wdtype, seed, affine=True):
    g = torch.Generator().manual_seed(seed)
    x = (rand(g, rows, D) * 1.7 + 0.6).to(dtype).to(DEV)
    dy = rand(g, rows, D).to(dtype).to(DEV)
    w = (1 + 0.3 * rand(g, D)).to(wdtype).to(DEV) if affine else None
    b = (0.2 * rand(g, D)).to(wdtype).to(DEV) if affine else None
    return x, dy, w, b


def check_fwd(x, w, b, y, mean, rstd, eps):
    D = x.shape[-1]
    X = x.double()
    m = X.mean(-1, keepdim=True)
    c = X - m
    r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    W = w.double() if w is not None else torch.ones((), device=x.device, dtype=torch.float64)
    Bv = b.double() if b is not None else torch.zeros((), device=x.device, dtype=torch.float64)
    want = c * r * W + Bv
    n = chain(D)
    off = n * U * X.abs().mean(-1, keepdim=True)             # error of the mean
    # the variance's own sum (relative n U), its square root, and what the shifted centre adds to it (second order), then
    # the affine part; one rounding to the output type (none for fp32, where the last operation's is counted in n)
    tol = (off * r + 2 * n * U * (c * r).abs()) * W.abs() + n * U * Bv.abs() + 1e-30
    if y.dtype != torch.float32:
        tol = tol * 1.01 + torch.finfo(y.dtype).eps / 2 * want.abs() + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert ((y.double() - want).abs() <= tol).all(), ((y.double() - want).abs() / tol).max()
    assert ((mean.double() - m[..., 0]).abs() <= off[..., 0] + U * m[..., 0].abs()).all()
    assert ((rstd.double() - r[..., 0]).abs() <= 2 * n * U * r[..., 0] * (1 + X.abs().amax(-1) ** 2 * r[..., 0] ** 2 * n * U)).all()


def check_bwd(dy, x, mean, rstd, w, dx, dw, db):
    rows, D = x.shape
    X, G = x.double(), dy.double()
    m, r = mean.double()[:, None], rstd.double()[:, None]
    W = w.double() if w is not None else torch.ones(D, device=x.device, dtype=torch.float64)
    h, a = (X - m) * r, G * W
    want = r * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
    n = chain(D)
    mag = a.abs() + a.abs().mean(1, keepdim=True) + 2 * (h.abs() + U * (X.abs() + m.abs()) * r) * (a * h).abs().mean(1, keepdim=True)
    # xhat inherits the rounding of x - mean: U |xhat|; the products and both row sums n U of their magnitudes
    tol = n * U * r * mag + 1e-30
    if dx.dtype != torch.float32:
        tol = tol * 1.01 + torch.finfo(dx.dtype).eps / 2 * want.abs() + torch.finfo(dx.dtype).smallest_normal * torch.finfo(dx.dtype).eps
    assert ((dx.double() - want).abs() <= tol).all(), ((dx.double() - want).abs() / tol).max()
    # rows added in one lane: at most rows / 1024 in a 1024-row grid (rows / 64 in the wide kernels) + 1, then 16 groups
    k = rows / 64 + 32
    for got, terms in ((dw, G * h), (db, G)):
        if got is None:
            continue
        # a 16-bit result below the type's smallest normal value is rounded to a multiple of smallest_normal * eps
        # (fp16: 2^-14 * 2^-10 = 2^-24), whatever its size: half of that step, absolute
        fi = torch.finfo(got.dtype)
        tol = k * U * terms.abs().sum(0) + fi.smallest_normal * fi.eps / 2 + (torch.finfo(got.dtype).eps / 2 * terms.sum(0).abs()) * (1.01 if got.dtype != torch.float32 else 1) + 1e-30
        assert ((got.double() - terms.sum(0)).abs() <= tol).all()


SHAPES = [(1, 1), (3, 2), (55, 64), (7, 10), (130, 63), (33, 65), (17, 128), (5, 255), (9, 256), (4, 513), (21, 1000), (6, 1024),
          (3, 2048), (5, 2052), (2, 4096), (3, 5003), (2, 8192), (3, 8200), (1, 16384), (2, 16392), (2, 20001), (2000, 24)]


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                          (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows,D", SHAPES)
def test_forward_and_backward(rows, D, dtype, wdtype):
    import noise_amd as na
    x, dy, w, b = case(rows, D, dtype, wdtype, rows * 131 + D)
    y, mean, rstd = na.layer_norm_fwd(x, w, b, 1e-6)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == torch.float32 and mean.shape == (rows,)
    check_fwd(x, w, b, y, mean, rstd, 1e-6)
    dx, dw, db = na.layer_norm_bwd(dy, x, mean, rstd, w)
    assert dx.dtype == dtype and dw.dtype == db.dtype == wdtype
    check_bwd(dy, x, mean, rstd, w, dx, dw, db)
    again = na.layer_norm_bwd(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))      # no order of summation left to chance


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,wide,at", [(64, 192, 64), (64, 200, 3), (250, 251, 1), (1024, 1032, 8), (2100, 2101, 0)])
def test_strided_rows_are_read_in_place(D, wide, at, dtype):
    import noise_amd as na
    g = torch.Generator().manual_seed(D + at)
    buf = (rand(g, 5, 11, wide) + 0.2).to(dtype).to(DEV)
    gbuf = rand(g, 5, 11, wide).to(dtype).to(DEV)
    w, b = (1 + 0.1 * rand(g, D)).float().to(DEV), rand(g, D).float().to(DEV)
    x, dy = buf[..., at:at + D], gbuf[..., at:at + D]
    y, mean, rstd = na.layer_norm_fwd(x, w, b)
    assert y.shape == x.shape and mean.shape == (5, 11)
    check_fwd(x, w, b, y, mean, rstd, 1e-6)
    dx, dw, db = na.layer_norm_bwd(dy, x, mean, rstd, w)
    check_bwd(dy.reshape(55, D), x.reshape(55, D), mean.view(-1), rstd.view(-1), w, dx.view(55, D), dw, db)
    # every other row, a transposed view (copied), a broadcast gradient
    for xs, ds in ((buf[:, ::2, at:at + D], gbuf[:, ::2, at:at + D]), (buf.transpose(0, 1)[..., at:at + D], gbuf.transpose(0, 1)[..., at:at + D]),
                   (x, dy[:1, :1].expand(5, 11, D))):
        y, mean, rstd = na.layer_norm_fwd(xs, w, b)
        check_fwd(xs, w, b, y, mean, rstd, 1e-6)
        dx, dw, db = na.layer_norm_bwd(ds, xs, mean, rstd, w)
        k = xs.shape[0] * xs.shape[1]
        check_bwd(ds.reshape(k, D), xs.reshape(k, D), mean.reshape(-1), rstd.reshape(-1), w, dx.reshape(k, D), dw, db)


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_without_weight_or_bias(which):
    import noise_amd as na
    x, dy, w, b = case(40, 96, torch.bfloat16, torch.float32, 5)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    y, mean, rstd = na.layer_norm_fwd(x, w, b)
    check_fwd(x, w, b, y, mean, rstd, 1e-6)
    dx, dw, db = na.layer_norm_bwd(dy, x, mean, rstd, w)
    check_bwd(dy, x, mean, rstd, w, dx, dw, db)
    assert na.layer_norm_bwd(dy, x, mean, rstd, w, need_params=False)[1:] == (None, None)


def test_constant_rows_empty_batches_and_poisoned_rows():
    import noise_amd as na
    w, b = torch.full((48,), 2.0, device=DEV), torch.full((48,), 0.5, device=DEV)
    x = torch.full((3, 48), 7.25, device=DEV)
    y, mean, rstd = na.layer_norm_fwd(x, w, b)
    assert (y == 0.5).all() and (mean == 7.25).all() and torch.allclose(rstd, torch.full_like(rstd, 1e3))
    x = torch.randn(4, 48, device=DEV)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    y = na.layer_norm(x, w, b)
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[[0, 3]]).all()
    e = torch.empty(0, 48, device=DEV)
    y, mean, rstd = na.layer_norm_fwd(e, w, b)
    dx, dw, db = na.layer_norm_bwd(e, e, mean, rstd, w)
    assert y.shape == dx.shape == (0, 48) and not dw.any() and not db.any()


def test_large_offset_keeps_the_variance():
    """Rows far from zero: the two-pass variance is what is left after the mean's own rounding."""
    import noise_amd as na
    g = torch.Generator().manual_seed(2)
    x = (rand(g, 30, 512) + 1000.0).float().to(DEV)
    check_fwd(x, None, None, *na.layer_norm_fwd(x), 1e-6)


def test_autograd_against_differences():
    """d/dt of sum(c . layer_norm(x + t u, w + t p, b + t q)) at t = 0 in 64 bits by central differences (step 1e-4: error
    of third order, below 1e-6 of the value's scale) against the gradients: fp32 sums of 24 x 40 products of order one."""
    import noise_amd as na
    g = torch.Generator().manual_seed(9)
    x, u, c = (rand(g, 24, 40) for _ in range(3))
    w, b, p, q = (rand(g, 40) for _ in range(4))

    def f(t):
        X = x + t * u
        m = X.mean(1, keepdim=True)
        r = ((X - m) ** 2).mean(1, keepdim=True).add(1e-6).rsqrt()
        return (c * ((X - m) * r * (w + t * p) + b + t * q)).sum().item()
    want = (f(1e-4) - f(-1e-4)) / 2e-4
    leaves = [t.float().to(DEV).requires_grad_(True) for t in (x, w, b)]
    (na.layer_norm(*leaves) * c.float().to(DEV)).sum().backward()
    got = sum((a.grad.double().cpu() * d).sum().item() for a, d in zip(leaves, (u, p, q)))
    scale = sum((a.grad.double().cpu() * d).abs().sum().item() for a, d in zip(leaves, (u, p, q)))
    assert abs(got - want) <= scale * (chain(40) + 32) * U + 1e-6 * scale
    # only what is asked for; a frozen input skips nothing else
    z = leaves[0].detach()
    w2 = leaves[1].detach().requires_grad_(True)
    na.layer_norm(z, w2, leaves[2].detach()).sum().backward()
    assert w2.grad is not None and z.grad is None


def test_other_stream_and_captured_graph():
    import noise_amd as na
    x, dy, w, b = case(300, 200, torch.bfloat16, torch.float32, 77)
    want = na.layer_norm_fwd(x, w, b)
    wantb = na.layer_norm_bwd(dy, x, want[1], want[2], w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = na.layer_norm_fwd(x, w, b)
        gotb = na.layer_norm_bwd(dy, x, got[1], got[2], w)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want + wantb, got + gotb))
    graph = torch.cuda.CUDAGraph()
    sx, sdy = x.clone(), dy.clone()
    with torch.cuda.graph(graph):
        f = na.layer_norm_fwd(sx, w, b)
        bw = na.layer_norm_bwd(sdy, sx, f[1], f[2], w)
    for k in range(3):
        sx.copy_(x * (k + 1))
        sdy.copy_(dy)
        graph.replay()
        ef = na.layer_norm_fwd(sx, w, b)
        eb = na.layer_norm_bwd(sdy, sx, ef[1], ef[2], w)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ef + eb, f + bw))


# Sizes at which a lane group works on more than one row: forward two rows from 4096 groups on, backward the grid's stride from
# 512 workgroups on (1024 / 256 for rows of a whole workgroup), each with a remainder; every group width, whole 16-byte pieces and
# single values, and rows too wide for registers.  (rows, width, type)
LOOPS = [(65537, 64, torch.float32), (65553, 60, torch.bfloat16), (32777, 128, torch.float32), (32771, 200, torch.bfloat16),
         (16391, 256, torch.float32), (16385, 512, torch.float32), (16387, 1000, torch.float32), (16389, 1016, torch.float16),
         (4099, 2048, torch.float32), (4101, 8192, torch.bfloat16), (4097, 6000, torch.float32), (4100, 16384, torch.float16),
         (65539, 15, torch.bfloat16), (32769, 31, torch.float32), (16389, 63, torch.float16), (16393, 127, torch.float32),
         (16387, 255, torch.bfloat16), (4103, 511, torch.float32), (4099, 1023, torch.float16), (4101, 2047, torch.bfloat16),
         (201, 16392, torch.bfloat16), (333, 2051, torch.float32), (131, 8204, torch.float32)]


@pytest.mark.parametrize("rows,D,dtype", LOOPS)
def test_many_rows_per_group(rows, D, dtype):
    """The sums of a lane run over at most rows / 64 + 32 terms, which check_bwd counts."""
    import noise_amd as na
    x, dy, w, b = case(rows, D, dtype, torch.float32, rows + D)
    y, mean, rstd = na.layer_norm_fwd(x, w, b, 1e-6)
    check_fwd(x, w, b, y, mean, rstd, 1e-6)
    got = na.layer_norm_bwd(dy, x, mean, rstd, w)
    check_bwd(dy, x, mean, rstd, w, *got)
    again = na.layer_norm_bwd(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    # the same rows through views that allow no 16-byte accesses
    wide = torch.zeros(rows, D + 1, device=DEV, dtype=dtype)
    wide[:, 1:] = x
    v = wide[:, 1:]
    y2, mean2, rstd2 = na.layer_norm_fwd(v, w, b, 1e-6)
    check_fwd(v, w, b, y2, mean2, rstd2, 1e-6)
    check_bwd(dy, v, mean, rstd, w, *na.layer_norm_bwd(dy, v, mean, rstd, w))


# Results of 128 MB and more go past the caches, in every group width
@pytest.mark.parametrize("rows,D,dtype", [(524801, 64, torch.float32), (262401, 128, torch.float32), (262147, 256, torch.bfloat16), (65541, 520, torch.float32),
                                          (70001, 1000, torch.bfloat16), (16400, 4096, torch.float16), (8209, 8192, torch.bfloat16),
                                          (4100, 16384, torch.bfloat16)])
def test_results_past_the_caches(rows, D, dtype):
    import noise_amd as na
    assert rows * D * dtype.itemsize >= 1 << 27
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, dy = ((torch.randn(rows, D, generator=g, device=DEV) * 1.7 + 0.6).to(dtype) for _ in range(2))
    w, b = (torch.randn(D, generator=g, device=DEV) for _ in range(2))
    y, mean, rstd = na.layer_norm_fwd(x, w, b, 1e-6)
    check_fwd(x, w, b, y, mean, rstd, 1e-6)
    got = na.layer_norm_bwd(dy, x, mean, rstd, w)
    check_bwd(dy, x, mean, rstd, w, *got)


def test_more_rows_than_one_launch_covers():
    """2^23 rows are one launch's limit."""
    import noise_amd as na
    rows, D = (1 << 23) + 5, 3
    g = torch.Generator(device=DEV).manual_seed(1)
    x, dy = (torch.randn(rows, D, generator=g, device=DEV) for _ in range(2))
    w, b = (torch.randn(D, generator=g, device=DEV) for _ in range(2))
    y, mean, rstd = na.layer_norm_fwd(x, w, b)
    check_fwd(x, w, b, y, mean, rstd, 1e-6)
    check_bwd(dy, x, mean, rstd, w, *na.layer_norm_bwd(dy, x, mean, rstd, w))

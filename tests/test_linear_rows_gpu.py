"""Scores from features and weights on the GPU, through the public entry points, against the definitions in 64 bits.
Bounds are those of linear_reference.py: they count roundings, and were written before the first run."""
import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float32", "bfloat16", "float16")


@pytest.fixture(scope="module")
def gpu():
    import torch
    assert torch.cuda.is_available(), "these tests need a GPU"
    import pcmi355
    import linear_reference
    return torch, pcmi355, linear_reference


def _inputs(torch, dtype, n, k, C, seed, bias="plain", slots=1, scale=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, dtype)
    f = torch.randn(n, k, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(C, k, generator=gen, device="cuda") * scale / k ** 0.5).to(dtype)
    b = None
    if bias:
        b = torch.randn(C, generator=gen, device="cuda")
        if bias == "masked":
            off = torch.rand(C, generator=gen, device="cuda") < 0.3
            off[C // 2] = False
            b.masked_fill_(off, -float("inf"))
        b = b.to(dtype)
        if bias == "lowest":
            off = torch.rand(C, generator=gen, device="cuda") < 0.3
            off[C // 2] = False
            b.masked_fill_(off, torch.finfo(dtype).min)
    g = torch.randint(-1, C, (n, slots), generator=gen, device="cuda")
    gl = -torch.rand(n, slots, generator=gen, device="cuda") / n
    gz = 0.1 * torch.randn(n, generator=gen, device="cuda") / n
    return f, w, b, g, gl, gz


def _check_scores(R, P, f, w, b, g):
    s = R.Scores(f, w, b)
    got = P.linear_scores(f, w, g, bias=b)
    R.within(got.log_sum, s.log_sum, s.log_sum_off, "log_sum")
    if g is not None:
        R.within(got.logp, *s.logp(g), "logp")
    return s, got


def _check_grads(R, P, f, w, b, s, got, g, gl, gz):
    want = R.gradients(f, w, b, s, g, gl, gz)
    d = P.linear_scores_backward(f, w, got.log_sum, g, bias=b, grad_logp=gl, grad_log_sum=gz)
    for name, (v, off) in want.items():
        t = getattr(d, name)
        assert t.dtype == (b.dtype if name == "bias" else f.dtype)
        R.within(t, v, off, name)
    return d


# one entry; few; either side of 32, 64, 128, 256 and of a step's 64 entries; a row of many steps; many categories; few categories
SHAPES = [(1, 1, 1), (1, 64, 2), (3, 5, 7), (31, 63, 33), (32, 64, 128), (33, 65, 129), (64, 128, 256), (65, 200, 257), (127, 64, 1000), (130, 130, 300),
          (256, 192, 512), (300, 1000, 50), (1, 4096, 3001), (17, 33, 20000), (520, 128, 70), (3000, 64, 3), (1000, 3, 1100),
          (201, 700, 300), (512, 515, 130), (48, 130, 40000), (20, 64, 33000), (50, 128, 32770)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_scores_and_gradients_of_every_size(gpu, dtype, shape):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 1, bias="plain" if sum(shape) % 2 else None, slots=1 + sum(shape) % 3)
    s, got = _check_scores(R, P, f, w, b, g)
    _check_grads(R, P, f, w, b, s, got, g, gl, gz)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3400, 64, 3700), (3500, 100, 4000)], ids=lambda s: "x".join(map(str, s)))
def test_large_tiles(gpu, dtype, shape):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 2, bias="masked", slots=2)
    s, got = _check_scores(R, P, f, w, b, g)
    _check_grads(R, P, f, w, b, s, got, g, gl, gz)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_in_pieces_of_the_categories(gpu, dtype):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, 16500, 40, 9100, 3, slots=1)
    s, got = _check_scores(R, P, f, w, b, g)
    _check_grads(R, P, f, w, b, s, got, g, gl, gz)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(16500, 40, 7681), (2, 3, (1 << 20) + 5), (70, 8, (1 << 20) + 3)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_in_pieces_of_unlike_sizes(gpu, dtype, shape):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 31, bias="masked", slots=2)
    g[:, 0] = shape[2] - 1 - torch.arange(shape[0], device="cuda") % 3      # categories of the last piece
    b[-3:] = 0.5
    s, got = _check_scores(R, P, f, w, b, g)
    _check_grads(R, P, f, w, b, s, got, g, gl, gz)


# sums of one and of two steps that are written as they are: gradients of features under few categories, of weights from few rows
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("shape", [(1500, 33, 20), (1024, 64, 64), (2000, 130, 65), (1100, 1001, 128), (64, 515, 1000), (65, 64, 3000), (128, 1000, 257),
                                   (5, 4099, 130)], ids=lambda s: "x".join(map(str, s)))
def test_short_sums(gpu, dtype, shape):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 32, bias="masked", slots=2)
    g[3:5], gz[3:5] = -1, 0.0                                               # rows without derivatives, whatever they hold
    s, got = _check_scores(R, P, f, w, b, g)
    f[3:5] = float("nan")
    clean = f.clone()
    clean[3:5] = 0.0
    s = R.Scores(clean, w, b)
    want = R.gradients(clean, w, b, s, g, gl, gz)
    d = P.linear_scores_backward(f, w, got.log_sum, g, bias=b, grad_logp=gl, grad_log_sum=gz)
    for name, (v, off) in want.items():
        R.within(getattr(d, name), v, off, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", ["masked", "lowest", None])
@pytest.mark.parametrize("slots", [1, 16, 64])
def test_masks_and_many_slots(gpu, dtype, bias, slots):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, 70, 96, 301, 4, bias=bias, slots=slots)
    g[:, slots // 2:] = g[:, :1]                       # the same category again
    g[5] = -1
    g[6] = 300
    if b is not None:
        w[R.masked(b)] = float("nan")                  # what a mask covers
        w[R.masked(b), ::2] = float("inf")
        b[300] = 0.5
        w[300] = 0.25
        masked = R.masked(b)
        clean = w.clone()
        clean[masked] = 0.0
    else:
        clean = w
    s = R.Scores(f, clean, b)
    got = P.linear_scores(f, w, g, bias=b)
    R.within(got.log_sum, s.log_sum, s.log_sum_off, "log_sum")
    R.within(got.logp, *s.logp(g), "logp")
    want = R.gradients(f, clean, b, s, g, gl, gz)
    d = P.linear_scores_backward(f, w, got.log_sum, g, bias=b, grad_logp=gl, grad_log_sum=gz)
    for name, (v, off) in want.items():
        R.within(getattr(d, name), v, off, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(20, 40, 50), (90, 64, 500), (600, 130, 200)], ids=lambda s: "x".join(map(str, s)))
def test_a_padded_batch(gpu, dtype, shape):
    """Rows whose categories are all negative have no part in any gradient, whatever their features hold"""
    torch, P, R = gpu
    f, w, b, g, gl, _ = _inputs(torch, dtype, *shape, 5, slots=2)
    n = shape[0]
    g[n // 2:] = -1
    f[n // 2:] = float("nan")
    f[-1] = float("inf")
    got = P.linear_scores(f, w, g, bias=b)
    assert torch.isnan(got.log_sum[n // 2:]).all() and (got.logp[n // 2:] == 0).all()
    d = P.linear_scores_backward(f, w, got.log_sum, g, bias=b, grad_logp=gl)
    f0, g0, gl0 = f[:n // 2].contiguous(), g[:n // 2].contiguous(), gl[:n // 2].contiguous()
    s, _ = _check_scores(R, P, f0, w, b, g0)
    want = R.gradients(f0, w, b, s, g0, gl0)
    R.within(d.features[:n // 2], *want["features"], "features")
    assert (d.features[n // 2:] == 0).all()
    R.within(d.weight, *want["weight"], "weight")
    R.within(d.bias, *want["bias"], "bias")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [5, 300])
def test_rows_without_a_category_and_rows_of_nan(gpu, dtype, C):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, 40, 70, C, 6)
    none = torch.full_like(b, -float("inf"))
    got = P.linear_scores(f, w, g, bias=none)
    assert (got.log_sum == -float("inf")).all()
    assert torch.equal(got.logp == -float("inf"), g >= 0) and (got.logp[g < 0] == 0).all()
    d = P.linear_scores_backward(f, w, got.log_sum, g, bias=none, grad_logp=gl, grad_log_sum=gz)
    assert all((t == 0).all() for t in d)
    # a row with NaN, one with infinities, one category past the end: NaN there, the others as they were
    want = P.linear_scores(f, w, g, bias=b)
    f2, g2 = f.clone(), g.clamp(min=0)
    f2[3, 5], f2[7] = float("nan"), float("inf")
    g2[9, 0] = C
    got = P.linear_scores(f2, w, g2, bias=b)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 7]] = True
    assert torch.isnan(got.log_sum[bad]).all() and torch.equal(got.log_sum[~bad], want.log_sum[~bad])
    bad[9] = True
    assert torch.equal(torch.isnan(got.logp).any(1), bad)
    gl = gl - 1.0
    d = P.linear_scores_backward(f2, w, got.log_sum, g2, bias=b, grad_logp=gl)
    assert torch.equal(torch.isnan(d.features).any(1), bad) and torch.isnan(d.bias).all() and torch.isnan(d.weight).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [64, 72])
@pytest.mark.parametrize("layout", ["transposed", "sliced", "offset", "every second", "one row for all", "three axes", "axes swapped", "wide rows"])
def test_every_layout(gpu, dtype, k, layout):
    torch, P, R = gpu
    n, C = 60, 90
    f, w, b, g, gl, gz = _inputs(torch, dtype, n, k, C, 7)
    rows = (n,)
    if layout == "transposed":
        f, w = f.t().contiguous().t(), w.t().contiguous().t()
    elif layout in ("sliced", "wide rows"):
        pad = 5 if layout == "sliced" else 64
        f = torch.cat([f, torch.full((n, pad), float("nan"), dtype=f.dtype, device="cuda")], 1)[:, :k]
        w = torch.cat([w, torch.full((C, pad), float("nan"), dtype=f.dtype, device="cuda")], 1)[:, :k]
    elif layout == "offset":
        f = torch.cat([f.reshape(-1)[:1], f.reshape(-1)])[1:].view(n, k)
        w = torch.cat([w.reshape(-1)[:3], w.reshape(-1)])[3:].view(C, k)
    elif layout == "every second":
        f = torch.stack([f, f * float("nan")], 2).view(n, 2 * k)[:, ::2]
        w = torch.stack([w, w * float("nan")], 1).view(2 * C, k)[::2]
    elif layout == "one row for all":
        f = f[:1].expand(n, k)
    elif layout == "three axes":
        f, rows = f.view(12, 5, k), (12, 5)
    elif layout == "axes swapped":
        f, rows = f.view(12, 5, k).transpose(0, 1).contiguous().transpose(0, 1), (12, 5)
    flat = f.reshape(n, k)
    s = R.Scores(flat, w, b)
    given = g.view(*rows, 1).to(torch.int32) if len(rows) == 2 else g.view(n).to(torch.int32)
    shaped = lambda t: t.view(given.shape)
    got = P.linear_scores(f, w, given, bias=b)
    assert got.log_sum.shape == rows and got.logp.shape == given.shape
    R.within(got.log_sum.reshape(-1), s.log_sum, s.log_sum_off, "log_sum")
    R.within(got.logp.reshape(n, 1), *s.logp(g), "logp")
    d = P.linear_scores_backward(f, w, got.log_sum, given, bias=b, grad_logp=shaped(gl), grad_log_sum=gz.view(rows))
    assert d.features.shape == f.shape and d.weight.shape == w.shape
    want = R.gradients(flat, w, b, s, g, gl, gz)
    R.within(d.features.reshape(n, k), *want["features"], "features")
    R.within(d.weight, *want["weight"], "weight")
    R.within(d.bias, *want["bias"], "bias")


@pytest.mark.parametrize("type_", ["uint8", "int32", "int64"])
def test_given_of_every_type(gpu, type_):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, "bfloat16", 50, 64, 200, 8, slots=5)
    g = g.clamp(min=0).to(getattr(torch, type_))
    wide = torch.cat([g, g], 1)
    s = R.Scores(f, w, b)
    got = P.linear_scores(f, w, wide[:, ::2], bias=b)
    R.within(got.logp, *s.logp(wide[:, ::2].long()), "logp")
    got = P.linear_scores(f, w, g[:, :0], bias=b)
    assert got.logp.shape == (50, 0)
    got = P.linear_scores(f, w, bias=b)
    assert got.logp is None
    R.within(got.log_sum, s.log_sum, s.log_sum_off, "log_sum")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [1e-6, 1.0, 60000.0])
def test_losses_of_every_scale(gpu, dtype, scale):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, 90, 64, 400, 9, slots=2)
    rows = torch.logspace(-4, 0, 90, device="cuda")
    gl, gz = gl * scale * rows[:, None], gz * scale * rows
    if dtype == "float16":
        f, w = f / 8, w / 4                            # (results within the type's range)
    s, got = _check_scores(R, P, f, w, b, g)
    _check_grads(R, P, f, w, b, s, got, g, gl, gz)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_far_apart_and_far_from_zero(gpu, dtype):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, 40, 64, 300, 10, scale=60.0)
    b = b.float() + 3000.0
    s, got = _check_scores(R, P, f, w, b, g)
    _check_grads(R, P, f, w, b, s, got, g, gl, gz)
    # one category: certain, whatever its score
    one = P.linear_scores(f, w[:1], torch.zeros(40, dtype=torch.uint8, device="cuda"))
    assert (one.logp == 0).all()
    d = P.linear_scores_backward(f, w[:1], one.log_sum, torch.zeros(40, 1, dtype=torch.uint8, device="cuda"), grad_logp=gl)
    assert float(d.features.abs().max()) <= 1e-6 * float(gl.abs().max() * w[:1].abs().max()) * 64


def test_float_is_as_exact_as_float(gpu):
    """Products of three bfloat16 parts: errors of sums, not of parts.  Rows of one product each, over the whole range of magnitudes"""
    torch, P, R = gpu
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = (1 + torch.rand(400, 1, generator=gen, device="cuda")) * 2.0 ** torch.randint(-12, 12, (400, 1), generator=gen, device="cuda")
    w = -(1 + torch.rand(300, 1, generator=gen, device="cuda"))
    got = P.linear_scores(x, w, torch.zeros(400, dtype=torch.int64, device="cuda"), bias=None)
    one = P.linear_scores(x, w[:1])
    want = (x.double() * w[0].double()).squeeze(1)
    # what the parts leave out: 2^-26 twice or so, and six roundings of the sum
    assert float(((one.log_sum.double() - want) / want).abs().max()) < 2.0 ** -24 + 6 * 2.0 ** -23
    s = R.Scores(x, w)
    R.within(got.logp, s.logp(torch.zeros(400, 1, dtype=torch.int64, device="cuda"))[0].squeeze(1), (s.log_sum_off + s.off[:, 0] + 2.0 ** -22 * s.log_sum.abs() * 2))
    f, w, b, g, gl, gz = _inputs(torch, "float32", 300, 1024, 700, 12)
    s, got = _check_scores(R, P, f, w, b, g)
    d = P.linear_scores_backward(f, w, got.log_sum, g, bias=b, grad_logp=gl, grad_log_sum=gz)
    for name, (v, _) in R.gradients(f, w, b, s, g, gl, gz).items():
        # root mean square: 2^-24 a rounding, of which a sum of 1024 has 6 * 16 steps of the matrix cores and more
        off = (getattr(d, name).double() - v).square().mean().sqrt() / v.square().mean().sqrt()
        assert float(off) < 4e-6, (name, float(off))


def test_gradient_is_the_derivative(gpu):
    """Against differences of linear_scores itself"""
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, "float32", 3, 5, 6, 13, slots=2)
    gl, gz = gl * 3, gz * 3

    def loss(f, w, b):
        s = P.linear_scores(f, w, g, bias=b)
        return float((s.logp.double() * gl.double()).sum() + (s.log_sum.double() * gz.double()).sum())

    d = P.linear_scores_backward(f, w, P.linear_scores(f, w, g, bias=b).log_sum, g, bias=b, grad_logp=gl, grad_log_sum=gz)
    h = 2.0 ** -6
    for i, t in enumerate((f, w, b)):
        for at in range(t.numel()):
            up, down = [u.clone() for u in (f, w, b)], [u.clone() for u in (f, w, b)]
            up[i].view(-1)[at] += h
            down[i].view(-1)[at] -= h
            step = float(up[i].view(-1)[at]) - float(down[i].view(-1)[at])
            # scores of size 10 in float: 1e-6 each, of weight 1 together, over 2 h; and h^2 times third derivatives of order 10
            assert abs((loss(*up) - loss(*down)) / step - float(d[i].view(-1)[at])) < 2e-6 / h + 10 * h * h


@pytest.mark.parametrize("of", ["features", "weight", "bias"])
def test_gradients_one_at_a_time(gpu, of):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, "bfloat16", 100, 64, 300, 14)
    z = P.linear_scores(f, w, bias=b).log_sum
    every = P.linear_scores_backward(f, w, z, g, bias=b, grad_logp=gl, grad_log_sum=gz)
    one = P.linear_scores_backward(f, w, z, g, bias=b, grad_logp=gl, grad_log_sum=gz, of=of)
    for name in ("features", "weight", "bias"):
        assert (getattr(one, name) is not None) == (name == of)
    assert torch.equal(getattr(one, of), getattr(every, of))
    assert P.linear_scores_backward(f, w, z, g, grad_logp=gl).bias is None
    only = P.linear_scores_backward(f, w, z, bias=b, grad_log_sum=gz)
    s = R.Scores(f, w, b)
    R.within(getattr(only, of), *R.gradients(f, w, b, s, None, None, gz)[of], of)
    nothing = P.linear_scores_backward(f, w, z, bias=b)
    assert (getattr(nothing, of) == 0).all()


def test_no_rows(gpu):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, "float16", 4, 64, 30, 15)
    s = P.linear_scores(f[:0], w, g[:0], bias=b)
    assert s.log_sum.shape == (0,) and s.logp.shape == (0, 1)
    d = P.linear_scores_backward(f[:0], w, s.log_sum, g[:0], bias=b, grad_logp=gl[:0])
    assert d.features.shape == (0, 64) and (d.weight == 0).all() and (d.bias == 0).all()
    assert P.rows8(f[:0]).codes.shape == (0, 128)
    assert P.product8(P.rows8(f[:0]), P.rows8(w)).shape == (0, 30)
    assert P.linear_scores(P.rows8(f[:0]), P.rows8(w)).log_sum.shape == (0,)


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_every_time(gpu, dtype):
    torch, P, R = gpu
    for shape in ((40, 100, 3000), (500, 128, 300), (5000, 64, 40)):
        f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 16, slots=3)
        first = None
        for _ in range(3):
            s = P.linear_scores(f, w, g, bias=b)
            d = P.linear_scores_backward(f, w, s.log_sum, g, bias=b, grad_logp=gl, grad_log_sum=gz)
            got = (s.log_sum, s.logp, *d)
            assert first is None or all(torch.equal(x, y) for x, y in zip(first, got))
            first = got


def test_nothing_is_written_behind_the_results(gpu):
    """Through the C entry points: guards around every result and the workspace, and more room than asked for is left alone"""
    torch, P, R = gpu
    from pcmi355._lib import lib, check
    for dtype, n, k, C in (("bfloat16", 37, 64, 131), ("float32", 50, 33, 77), ("float16", 70, 65, 257)):
        f, w, b, g, gl, gz = _inputs(torch, dtype, n, k, C, 17)
        code = {"float32": 0, "bfloat16": 1, "float16": 2}[dtype]
        size = f.element_size()
        factors = (f.data_ptr(), w.data_ptr(), code, k, 0, 1, k, 1, n, 1, k, C)

        def guarded(count):
            buf = torch.full((count + 1024,), 0xA5, dtype=torch.uint8, device="cuda")
            return buf, buf.data_ptr() + 512

        def intact(buf, count):
            return bool((buf[:512] == 0xA5).all() and (buf[512 + count:] == 0xA5).all())

        need = lib.pcm_linear_scores_workspace(*factors)
        work, z, lp = guarded(need), guarded(4 * n), guarded(4 * n)
        check(lib.pcm_linear_scores(*factors, b.data_ptr(), code, g.data_ptr(), 5, 1, 0, 0, 1, lp[1], z[1], work[1], need, None))
        torch.cuda.synchronize()
        assert intact(work[0], need) and intact(z[0], 4 * n) and intact(lp[0], 4 * n)
        back = lib.pcm_linear_scores_backward_workspace(*factors, 7)
        work2, df, dw, db = guarded(back), guarded(size * n * k), guarded(size * C * k), guarded(size * C)
        check(lib.pcm_linear_scores_backward(*factors, b.data_ptr(), code, g.data_ptr(), 5, 1, 0, 0, 1, gl.data_ptr(), gz.data_ptr(), z[1], df[1], dw[1],
                                             db[1], work2[1], back, None))
        torch.cuda.synchronize()
        for buf, count in ((work2[0], back), (df[0], size * n * k), (dw[0], size * C * k), (db[0], size * C), (z[0], 4 * n)):
            assert intact(buf, count)


def test_captured_and_replayed(gpu):
    torch, P, R = gpu
    cases = [_inputs(torch, t, *shape, 18, slots=2) for t, shape in (("float32", (60, 50, 200)), ("bfloat16", (300, 64, 600)), ("float16", (5, 128, 3000)))]

    def step(f, w, b, g, gl, gz):
        s = P.linear_scores(f, w, g, bias=b)
        d = P.linear_scores_backward(f, w, s.log_sum, g, bias=b, grad_logp=gl, grad_log_sum=gz)
        a, c = P.rows8(f), P.rows8(w)
        e = P.linear_scores(a, c, g, bias=b)
        return (s.log_sum, s.logp, *d, P.product8(a, c, bias=b), e.log_sum, e.logp)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cases:
            step(*c)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*c)
        graphs.append((graph, out))
    for turn in range(4):
        for (f, w, b, g, gl, gz) in cases:
            f.copy_(torch.randn(f.shape, generator=torch.Generator().manual_seed(turn)).to(f.dtype))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c, (_, out) in zip(cases, graphs):
            assert all(torch.equal(x, y) for x, y in zip(out, step(*c)))


def test_on_a_stream_of_its_own(gpu):
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, "bfloat16", 400, 128, 3000, 19)
    want = P.linear_scores(f, w, g, bias=b)
    grad = P.linear_scores_backward(f, w, want.log_sum, g, bias=b, grad_logp=gl)
    side = torch.cuda.Stream()
    late = torch.zeros_like(f)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        late.copy_(f)
        got = P.linear_scores(late, w, g, bias=b)
        d = P.linear_scores_backward(late, w, got.log_sum, g, bias=b, grad_logp=gl)
    side.synchronize()
    assert torch.equal(got.log_sum, want.log_sum) and all(torch.equal(x, y) for x, y in zip(d, grad))


def test_offsets_beyond_32_bits(gpu):
    """Weights of more than 2^32 bytes and 2^31 entries; features far into theirs"""
    torch, P, R = gpu
    C, k = 140000, 16384
    w = torch.empty(C, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(20)).mul_(2 / k ** 0.5)
    f = torch.randn(40, k, device="cuda").to(torch.bfloat16)
    g = torch.randint(C - 500, C, (40, 2), device="cuda")
    got = P.linear_scores(f, w, g)
    x = torch.cat([R.product(f, w[i:i + 20000]) for i in range(0, C, 20000)], 1)
    off = R.sum_bound(x.abs().max() * 0 + float(torch.cat([R.product(f.abs(), w[i:i + 20000].abs()) for i in range(0, C, 20000)], 1).max()), k, torch.bfloat16)
    z = torch.logsumexp(x, 1)
    R.within(got.log_sum, z, torch.full_like(z, float(off) + 1e-5), "log_sum")
    R.within(got.logp, x.gather(1, g) - z[:, None], torch.full((40, 2), 2 * float(off) + 1e-5, device="cuda"), "logp")
    gl = -torch.ones(40, 2, device="cuda")
    d = P.linear_scores_backward(f, w, got.log_sum, g, grad_logp=gl)
    dx = torch.zeros_like(x).scatter_add_(1, g, gl.double()) + 2 * (x - z[:, None]).exp()
    for rows in (slice(0, 300), slice(C - 700, C)):
        part = dx[:, rows].t().contiguous()
        v, size = R.product(part, f.t().contiguous()), R.product(part.abs(), f.abs().t().contiguous())
        R.within(d.weight[rows], v, (2.0 ** -8 * 1.1 + 48 * 2.0 ** -23 + 2.01 * float(off)) * size + 2.0 ** -8 * v.abs() + 1e-30, "weight")


# ---- 8 bits ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (4, 127), (5, 128), (6, 129), (300, 1000), (2, 131071), (17, 4096)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["plain", "odd values", "small", "every second"])
def test_rows_in_eight_bits(gpu, dtype, shape, kind):
    torch, P, R = gpu
    gen = torch.Generator(device="cuda").manual_seed(21)
    x = torch.randn(*shape, generator=gen, device="cuda").to(getattr(torch, dtype))
    if kind == "odd values":                           # zeros, NaN, infinities, ties at half a step, a lone value
        x[0] = 0.0
        x[-1, -1] = float("nan")
        if shape[0] > 2:
            x[1, 0] = -float("inf")
            x[2] = 0.5
            x[2, 0] = -1.0
    elif kind == "small":
        x = (x.float() * 1e-37).to(x.dtype)
    elif kind == "every second":
        x = torch.stack([x, x], 2).view(shape[0], -1)[:, ::2]
    got = P.rows8(x)
    codes, scales = R.codes_of(x)
    pad = got.codes.shape[1] - shape[1]
    assert pad >= 0 and got.codes.shape[1] % 128 == 0 and (got.codes[:, shape[1]:] == 0).all()
    assert torch.equal(got.codes[:, :shape[1]], codes)
    assert torch.equal(got.scales.nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))


def _eight(torch, dtype, n, k, C, seed):
    f, w, b, g, gl, gz = _inputs(torch, dtype, n, k, C, seed)
    return f, w, b, g


def _exact_product(torch, R, a, c, k):
    """The whole-number sums"""
    return R.product(a.codes[:, :k].float(), c.codes[:, :k].float())


SHAPES8 = [(1, 1, 1), (1, 4096, 3001), (3, 5, 7), (31, 127, 33), (32, 128, 128), (33, 129, 130), (64, 1000, 256), (65, 200, 257), (300, 4000, 50), (2, 131071, 3),
           (520, 128, 70), (3600, 100, 4000), (17, 33, 20000), (4096, 8192, 64), (20, 200, 33000), (50, 129, 32800)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES8, ids=lambda s: "x".join(map(str, s)))
def test_products_of_eight_bits(gpu, dtype, shape):
    torch, P, R = gpu
    n, k, C = shape
    f, w, b, _ = _eight(torch, dtype, n, k, C, 22)
    a, c = P.rows8(f), P.rows8(w)
    whole = _exact_product(torch, R, a, c, k)
    assert float(whole.abs().max()) < 2 ** 31
    for bias in (None, b):
        v = whole * a.scales.double()[:, None] * c.scales.double()
        size = v.abs()
        if bias is not None:
            v = v + bias.double()
        got = P.product8(a, c, bias=bias)
        assert got.dtype == f.dtype and got.shape == (n, C)
        # the sum as a float, two products and a sum: four roundings; then the type's
        R.within(got, v, 4 * 2.0 ** -24 * (size + v.abs()) + R.half_step(f.dtype) * v.abs() * 1.001 + R.LEAST[f.dtype], "product")
    if n * C < 1 << 20:
        exact = P.product8(a, c, dtype=torch.float32)
        # in the plain order, the same bits
        assert torch.equal(exact, whole.float() * a.scales[:, None] * c.scales)


@pytest.mark.parametrize("shape", [(3, 130, 50), (70, 8192, 20)], ids=lambda s: "x".join(map(str, s)))
def test_largest_codes_and_rows_of_nan(gpu, shape):
    torch, P, R = gpu
    n, k, C = shape
    pitch = -(-k // 128) * 128
    make = lambda n, v: P.Rows8(torch.nn.functional.pad(torch.full((n, k), v, dtype=torch.int8, device="cuda"), (0, pitch - k)),
                                torch.ones(n, device="cuda"), (n, k), torch.float32)
    for u, v in ((-128, -128), (-128, 127), (127, 127)):
        assert (P.product8(make(n, u), make(C, v)) == u * v * k).all()
    a, c = make(n, 3), make(C, 5)
    a.scales[1] = float("nan")
    got = P.product8(a, c)
    assert torch.isnan(got[1]).all() and (got[0] == 15 * k).all()


def test_longest_rows(gpu):
    torch, P, R = gpu
    k = 131071
    codes = torch.nn.functional.pad(torch.full((2, k), -128, dtype=torch.int8, device="cuda"), (0, 1))
    a = P.Rows8(codes, torch.ones(2, device="cuda"), (2, k), torch.float32)
    assert (P.product8(a, a).double() == torch.tensor(float(16384 * k), dtype=torch.float32).double().item()).all()


def test_products_into_what_is_given(gpu):
    torch, P, R = gpu
    f, w, b, _ = _eight(torch, "bfloat16", 6, 64, 40, 23)
    a, c = P.rows8(f), P.rows8(w)
    want = P.product8(a, c, bias=b)
    out = torch.empty(6, 40, dtype=torch.bfloat16, device="cuda")
    assert P.product8(a, c, bias=b, out=out) is out and torch.equal(out, want)
    shaped = P.rows8(f.view(2, 3, 64))
    assert P.product8(shaped, c, bias=b).shape == (2, 3, 40) and torch.equal(P.product8(shaped, c, bias=b).view(6, 40), want)
    odd = torch.empty(6 * 41 + 1, dtype=torch.float32, device="cuda")[1:].view(6, 41)
    assert torch.equal(P.product8(a, P.rows8(torch.cat([w, w[:1]])), out=odd)[:, :40], P.product8(a, c, dtype=torch.float32))
    for bad in (out[:, :39], out.float().double(), out.t(), torch.empty(6, 80, dtype=torch.bfloat16, device="cuda")[:, ::2]):
        with pytest.raises(ValueError, match="out|float32"):
            P.product8(a, c, out=bad)
    over = torch.empty(6 * 40, dtype=torch.float32, device="cuda")
    clash = P.Rows8(over.view(torch.int8)[:6 * 128].view(6, 128), a.scales, (6, 64), torch.float32)
    with pytest.raises(ValueError, match="overlaps"):
        P.product8(clash, c, out=over.view(6, 40))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 64, 3), (1, 4096, 3001), (40, 200, 500), (300, 129, 1000), (3600, 128, 4000), (20, 200, 33000), (50, 129, 32800), (200, 600, 700)], ids=lambda s: "x".join(map(str, s)))
def test_scores_of_eight_bits(gpu, dtype, shape):
    torch, P, R = gpu
    n, k, C = shape
    f, w, b, g, _, _ = _inputs(torch, dtype, n, k, C, 24, bias="masked" if n > 1 else "plain", slots=3)
    a, c = P.rows8(f), P.rows8(w)
    x = _exact_product(torch, R, a, c, k) * a.scales.double()[:, None] * c.scales.double()
    off = 4 * 2.0 ** -24 * x.abs()
    x = x + b.double()
    off = off + 2.0 ** -24 * x.abs().nan_to_num(posinf=0.0)
    x[:, R.masked(b)] = -float("inf")
    z = torch.logsumexp(x, 1)
    got = P.linear_scores(a, c, g, bias=b)
    most = off.max(1).values + 2.0 ** -24 * (160 + 4 * z.abs())
    R.within(got.log_sum, z, most, "log_sum")
    at = g.clamp(min=0)
    lp = torch.where(g < 0, 0.0, x.gather(1, at) - z[:, None])
    R.within(got.logp, lp, 2 * most[:, None] + 2.0 ** -22 * lp.abs().nan_to_num(posinf=0.0), "logp")


# ---- together ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
def test_scores_agree_with_scores_in_memory(gpu, dtype):
    """linear_scores beside category_scores of the product, and its gradient beside that of category_scores_backward"""
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, 12 * 8, 64, 130, 25, bias="masked")
    x = (R.product(f, w) + b.double()).float().view(12, 8, 130)
    given = g.view(12, 8)
    kept = P.category_scores(x, given)
    s = R.Scores(f, w, b)
    got = P.linear_scores(f.view(12, 8, 64), w, given, bias=b)
    R.within(got.log_sum.view(-1), kept.log_sum.view(-1), s.log_sum_off * 2 + 2.0 ** -20, "log_sum")
    R.within(got.logp.view(-1, 1), kept.logp.view(-1, 1), s.logp(g)[1] * 2 + 2.0 ** -20, "logp")
    dx = P.category_scores_backward(x, kept.log_sum, given, grad_logp=gl.view(12, 8)).view(-1, 130)
    d = P.linear_scores_backward(f.view(12, 8, 64), w, got.log_sum, given, bias=b, grad_logp=gl.view(12, 8))
    want = R.gradients(f, w, b, s, g, gl)
    seen = w.clone()
    seen[R.masked(b)] = 0.0                            # (a masked category, also a given one, has no part in the features' gradient)
    R.within(d.features.view(-1, 64).double(), R.product(dx, seen.t().contiguous()), want["features"][1] * 3, "features")
    R.within(d.weight.double(), R.product(dx.t().contiguous(), f.t().contiguous()), want["weight"][1] * 3, "weight")


def test_a_network_taught_the_clusters_of_a_circuit(gpu):
    """A head's training steps on the cluster ids that a multi-head circuit finds likeliest, then in 8 bits: the gradients drive
    the loss that linear_scores reports, and 8-bit scores follow those of the head"""
    torch, P, R = gpu
    import numpy as np
    rng = np.random.default_rng(26)
    V, K, C, H, N = 12, 16, 16, 8, 256
    parent = np.arange(-1, V - 1).astype(np.int32)
    body = P.multihead_hclt_from_clt(parent, C, K, H)
    data = torch.from_numpy(rng.integers(0, C, (N, V)).astype(np.uint8)).cuda()
    clusters = P.head_scores(body, data, top=1).top.view(-1)
    f = torch.nn.functional.one_hot(data.long(), C).float().view(N, -1)
    w, b = torch.zeros(H, V * C, device="cuda"), torch.zeros(H, device="cuda")
    by = torch.full((N,), -1.0 / N, device="cuda")
    for _ in range(3):
        s = P.linear_scores(f, w, clusters, bias=b)
        d = P.linear_scores_backward(f, w, s.log_sum, clusters, bias=b, grad_logp=by)
        ref = R.gradients(f, w, b, R.Scores(f, w, b), clusters.long().view(-1, 1), by.view(-1, 1))
        for name, (v, off) in ref.items():
            R.within(getattr(d, name), v, off, name)
        w, b = w - 0.5 * d.weight, b - 0.5 * d.bias
    a, c = P.rows8(f), P.rows8(w)
    x = P.product8(a, c, bias=b, dtype=torch.float32)
    kept = P.category_scores(x, clusters, top=2)
    direct = P.linear_scores(a, c, clusters, bias=b)
    assert float((kept.log_sum - direct.log_sum).abs().max()) < 1e-5 and float((kept.logp - direct.logp).abs().max()) < 1e-5
    # each weight off by half a step: at most V of them in a score
    exact = P.linear_scores(f, w, clusters, bias=b)
    step = float((w.abs().max(1).values / 127).max())
    assert float((exact.log_sum - direct.log_sum).abs().max()) <= V * step / 2 * 1.01 + 1e-5


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_no_rows_through_the_c_entry(gpu, dtype):
    """Weights' and bias's gradients are sums of nothing; no workspace, no features, no log-sums"""
    torch, P, R = gpu
    from pcmi355._lib import lib, check
    code = {"float32": 0, "bfloat16": 1, "float16": 2}[dtype]
    k, C = 70, 301
    w = torch.ones(C, k, dtype=getattr(torch, dtype), device="cuda")
    dw, db = torch.full((C + 1, k), 7.0, dtype=w.dtype, device="cuda"), torch.full((C + 1,), 7.0, device="cuda")
    check(lib.pcm_linear_scores_backward(None, w.data_ptr(), code, k, 0, 1, k, 1, 0, 1, k, C, None, 0, None, 5, 0, 0, 0, 0, None, None, None, None,
                                         dw.data_ptr(), db.data_ptr(), None, 0, None))
    torch.cuda.synchronize()
    assert (dw[:C] == 0).all() and (db[:C] == 0).all() and (dw[C] == 7).all() and db[C] == 7


@pytest.mark.parametrize("dtype", TYPES)
def test_more_categories_than_a_launch_has_threads_for(gpu, dtype):
    """2^28 categories in tiles of 32, a workgroup of 512 threads each, pass 2^32 threads; those behind weigh most"""
    torch, P, R = gpu
    C = (1 << 28) + 133
    w = torch.empty(C, 1, dtype=getattr(torch, dtype), device="cuda").uniform_(-1, 0, generator=torch.Generator(device="cuda").manual_seed(41))
    last = 300
    w[C - last:] = torch.linspace(24, 30, last, device="cuda")[:, None].to(w.dtype)
    f = torch.tensor([[1.0], [0.5], [-1.0]], device="cuda").to(w.dtype)
    g = torch.tensor([[C - 1, C - 150], [C - last, 0], [1 << 28, C]], device="cuda")
    got = P.linear_scores(f, w, g)
    tail, z, chunk = w[C - last:], [], 1 << 24
    for v in f:
        part = [torch.logsumexp(w[i:i + chunk, 0].double() * v.double(), 0) for i in range(0, C, chunk)]
        z.append(torch.logsumexp(torch.stack(part), 0))
    z = torch.stack(z)
    # of the sum: a lane adds (2^23 + 5) / 256 parts one after the other, and 32 exponentials of 2^-22 and some joins before and after
    off = 2.0 ** -24 * ((1 << 15) + 200 + 4 * z.abs())
    R.within(got.log_sum, z, off, "log_sum")
    x = torch.cat([w[g.clamp(max=C - 1).reshape(-1), 0]]).double().view(3, 2) * f.double()
    want = x - z[:, None]
    want[2, 1] = float("nan")
    R.within(got.logp, want, off[:, None] + 2.0 ** -22 * (x.abs() + z.abs()[:, None]), "logp")
    assert float(torch.logsumexp(tail[:, 0].double(), 0) - z[0]) > -0.01     # (row 0: without them it would be another number)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_more_tiles_than_a_launch_has_threads_for(gpu, dtype):
    """2^13 + 2 rows of tiles by 2^11 tiles of 256 threads: 64 rows of features again and again, every repetition the same"""
    torch, P, R = gpu
    n, k, C = (1 << 20) + 130, 64 if dtype == "bfloat16" else 8, 1 << 18
    few, w, b, g, _, _ = _inputs(torch, dtype, 64, k, C, 42)
    f = few.repeat(-(-n // 64), 1)[:n].contiguous()
    given = g.repeat(-(-n // 64), 1)[:n].contiguous()
    got = P.linear_scores(f, w, given, bias=b)
    x = R.product(few, w) + b.double()
    z = torch.logsumexp(x, 1)
    size = R.product(few.abs(), w.abs()) + b.double().abs()
    most = R.sum_bound(size, k, few.dtype).max(1).values + 2.0 ** -24 * (160 + 2048 / 16 + 4 * z.abs())
    R.within(got.log_sum[:64], z, most, "log_sum")
    lp = torch.where(g < 0, 0.0, x.gather(1, g.clamp(min=0)) - z[:, None])
    R.within(got.logp[:64], lp, 2 * most[:, None] + 2.0 ** -22 * (lp.abs() + z.abs()[:, None]), "logp")
    again = torch.arange(n, device="cuda") % 64
    assert torch.equal(got.log_sum, got.log_sum[:64][again]) and torch.equal(got.logp, got.logp[:64][again])


@pytest.mark.parametrize("n", [3, 200])
def test_floats_beyond_the_largest_of_16_bits(gpu, n):
    """float32's finite entries past bfloat16's largest (3.39e38) are as good as any other: in scores, and in both gradients' sums"""
    torch, P, R = gpu
    big = torch.tensor([torch.finfo(torch.float32).max, 3.396e38, -3.4e38, 3.3895314e38, 1e38], device="cuda")
    f = big.repeat(n)[:n, None] if n < 5 else big.repeat(n // 5)[:, None]
    small = torch.tensor([[2.0 ** -100], [-1.7 * 2.0 ** -110], [1.3 * 2.0 ** -120]], device="cuda")
    for w in small:                                    # one category: its score is the log-sum
        for x, y in ((f, w[None]), (w[None].expand(n, 1), f[:1])):
            got = P.linear_scores(x, y).log_sum.double()
            want = x.double()[:, 0] * y.double()[0, 0]
            # (and the small factor's third part ends at bfloat16's least number, 2^-133: up to half of it is left out, 2^-134 / |w| of the product)
            assert float(((got - want) / want).abs().max()) < 2.0 ** -24 + 6 * 2.0 ** -23 + 2.0 ** -134 / float(w.abs())
    # two categories of equal scores: dx is +-gl / 2
    given, by = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.full((n,), 2.0 ** -12, device="cuda")
    zero, w = torch.zeros(n, 5, device="cuda"), torch.stack([big, big.flip(0)])
    s = P.linear_scores(zero, w, given)
    d = P.linear_scores_backward(zero, w, s.log_sum, given, grad_logp=by, of="features").features.double()
    want = 2.0 ** -13 * (w[0].double() - w[1].double())
    size = 2.0 ** -13 * w.double().abs().sum(0)
    assert (((d - want).abs() - size * (2.0 ** -20 + 14 * 2.0 ** -23)) <= 0).all()     # (p: 2^-20 of it)
    f, w = big.expand(n, 5).contiguous(), torch.zeros(2, 5, device="cuda")
    s = P.linear_scores(f, w, given)
    d = P.linear_scores_backward(f, w, s.log_sum, given, grad_logp=by / n, of="weight").weight.double()
    want = 2.0 ** -13 * big.double()
    size = want.abs() * (2.0 ** -20 + (6 * n + 8) * 2.0 ** -23)
    assert ((d[0] - want).abs() <= size).all() and ((d[1] + want).abs() <= size).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,v", [((140001, 24, 4200), 1), ((140001, 40, 4097), 3), ((262200, 8, 2100), 1)], ids=lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else str(s))
def test_gradients_in_parts_of_the_rows(gpu, dtype, shape, v):
    """So many rows that a piece's derivatives are taken in parts: 2^29 of them and what is left, or whole examples"""
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 43, bias="masked", slots=2)
    n = shape[0]
    g[n - 40:], gz[n - 40:] = -1, 0.0                                       # a padded end, in the last part
    g[131000:131150, 0] = shape[2] - 1                                      # the same category on both sides of a border
    b[-1] = 0.5
    s = R.Scores(f, w, b)
    rows = (n // v, v) if v > 1 else (n,)
    if v > 1:
        f = f.view(n // v, v, -1).transpose(0, 1).contiguous().transpose(0, 1)
    shaped = lambda t: t.view(*rows, 2)
    got = P.linear_scores(f, w, shaped(g).to(torch.int32), bias=b)
    R.within(got.log_sum.reshape(-1), s.log_sum, s.log_sum_off, "log_sum")
    flat = f.reshape(n, -1).clone()
    f[-1] = float("nan")                                                    # (rows of the padded end)
    d = P.linear_scores_backward(f, w, got.log_sum, shaped(g).to(torch.int32), bias=b, grad_logp=shaped(gl), grad_log_sum=gz.view(rows))
    want = R.gradients(flat, w, b, s, g, gl, gz)
    R.within(d.features.reshape(n, -1), *want["features"], "features")
    R.within(d.weight, *want["weight"], "weight")
    R.within(d.bias, *want["bias"], "bias")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_gradients_in_pieces_of_long_weights(gpu, dtype):
    """Few rows, and weights of more than 2^30 entries: pieces of the categories"""
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, 3, 8200, 131100, 44, bias="masked", slots=2)
    g[:, 0] = 131099 - torch.arange(3, device="cuda")
    b[-3:] = 0.5
    s, got = _check_scores(R, P, f, w, b, g)
    _check_grads(R, P, f, w, b, s, got, g, gl, gz)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("at", range(5))
def test_tiles_of_256(gpu, dtype, at):
    """Sizes that the host test of the rule holds to be cut into tiles of 256 x 256: odd borders, masks, several slots, padded rows"""
    torch, P, R = gpu
    assert len(R.WIDE) == 5
    shape = R.WIDE[at][0]
    f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 45, bias="masked", slots=2)
    g[:, 0] = shape[2] - 1 - torch.arange(shape[0], device="cuda") % 7      # categories of the last tile
    b[-7:] = 0.5
    g[-20:], gz[-20:] = -1, 0.0
    s, got = _check_scores(R, P, f, w, b, g)
    _check_grads(R, P, f, w, b, s, got, g, gl, gz)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", range(2))
def test_tiles_of_256_of_eight_bits(gpu, dtype, at):
    torch, P, R = gpu
    assert len(R.WIDE8) == 2
    n, k, C = R.WIDE8[at]
    f, w, b, g, _, _ = _inputs(torch, dtype, n, k, C, 46, bias="masked", slots=3)
    a, c = P.rows8(f), P.rows8(w)
    whole = _exact_product(torch, R, a, c, k)
    x = whole * a.scales.double()[:, None] * c.scales.double()
    seen = torch.where(R.masked(b), torch.zeros_like(b), b)
    v = x + seen.double()
    R.within(P.product8(a, c, bias=seen), v, 4 * 2.0 ** -24 * (x.abs() + v.abs()) + R.half_step(f.dtype) * v.abs() * 1.001 + R.LEAST[f.dtype], "product")
    assert torch.equal(P.product8(a, c, dtype=torch.float32), whole.float() * a.scales[:, None] * c.scales)
    off = 4 * 2.0 ** -24 * x.abs() + 2.0 ** -24 * v.abs()
    v[:, R.masked(b)] = -float("inf")
    off[:, R.masked(b)] = 0.0
    z = torch.logsumexp(v, 1)
    most = off.max(1).values + 2.0 ** -24 * (160 + 4 * z.abs())
    got = P.linear_scores(a, c, g, bias=b)
    R.within(got.log_sum, z, most, "log_sum")
    lp = torch.where(g < 0, 0.0, v.gather(1, g.clamp(min=0)) - z[:, None])
    R.within(got.logp, lp, 2 * most[:, None] + 2.0 ** -22 * lp.abs().nan_to_num(posinf=0.0), "logp")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,cut", [((50, 96, 301), 100), ((1100, 64, 700), 256)], ids=["few", "many"])
def test_shards_of_the_categories(gpu, dtype, shape, cut):
    """Two shards' log-sums join by their log-sum, log-probabilities are the scores less the joined one, and each shard's gradients come from it: a slot
    whose category the other shard has is negative, its derivative goes from grad_log_sum"""
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 47, bias="masked", slots=3)
    s = R.Scores(f, w, b)
    parts = ((0, cut), (cut, shape[2]))
    own = [torch.where((g >= lo) & (g < hi), g - lo, -1) for lo, hi in parts]
    each = [P.linear_scores(f, w[lo:hi], o, bias=b[lo:hi]) for (lo, hi), o in zip(parts, own)]
    z = torch.logsumexp(torch.stack([e.log_sum.double() for e in each]), 0).float()
    s.log_sum_off = s.log_sum_off + 2.0 ** -24 * s.log_sum.abs()            # (the joined one is rounded once more)
    R.within(z, s.log_sum, s.log_sum_off, "log_sum")
    lp = sum(torch.where(o < 0, 0.0, (e.logp.double() + e.log_sum.double()[:, None] - z.double()[:, None])) for o, e in zip(own, each))
    v, off = s.logp(g)
    R.within(lp, v, off + sum(e.log_sum.abs().double()[:, None] for e in each) * 2.0 ** -22, "logp")
    want = R.gradients(f, w, b, s, g, gl, gz)
    dx = R.dx_of(s, g, gl, gz)[0]
    got, sizes = [], torch.zeros(shape[0], shape[1], dtype=torch.float64, device="cuda")
    for (lo, hi), o in zip(parts, own):
        other = torch.where((g >= 0) & (o < 0), gl, 0.0).sum(1)
        got.append(P.linear_scores_backward(f, w[lo:hi], z, o, bias=b[lo:hi], grad_logp=gl, grad_log_sum=gz - other))
        seen = torch.where(R.masked(b[lo:hi])[:, None], torch.zeros_like(w[lo:hi]), w[lo:hi])
        sizes += R.product(dx[:, lo:hi], seen.t().contiguous()).abs()
    # (gz less a slot's derivative is rounded once: 2^-24 of the row's size, of which p is a part at most)
    R.within(sum(d.features.double() for d in got), want["features"][0], want["features"][1] * 1.01 + R.half_step(f.dtype) * sizes + R.LEAST[f.dtype], "features")
    R.within(torch.cat([d.weight for d in got]), *want["weight"], "weight")
    R.within(torch.cat([d.bias for d in got]), *want["bias"], "bias")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(7, 70, 40), (300, 64, 200), (1100, 100, 300)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_with_large_factors(gpu, dtype, shape):
    """Finite gradients where factors are as large as their types (float32, bfloat16) have them: weights against features of 0 and the other way round"""
    torch, P, R = gpu
    f, w, b, g, gl, gz = _inputs(torch, dtype, *shape, 48, slots=2)
    n, k, C = shape
    f[:, 0], f[:, 1], w[:, 0], w[:, 1] = 0.0, 0.0, 0.0, 0.0
    w[g[0].clamp(min=0), 0] = 2.0 ** 120                                   # (one or two categories; derivatives are 1 / n at most)
    f[1, 1] = 2.0 ** 120
    s, got = _check_scores(R, P, f, w, b, g)
    d = _check_grads(R, P, f, w, b, s, got, g, gl, gz)
    assert torch.isfinite(d.features).all() and torch.isfinite(d.weight).all()
    assert float(d.features[:, 0].float().abs().max()) > 2.0 ** 100 and float(d.weight[:, 1].float().abs().max()) > 2.0 ** 100

"""The operators on rows of category scores on the GPU, through the public entry points, against the definitions in 64 bits.
Bounds are those of category_reference.py: they count roundings, and were written before the first run."""
import numpy as np
import pytest

import category_reference as R

pytestmark = pytest.mark.gpu

TYPES = ("float32", "bfloat16", "float16")


@pytest.fixture(scope="module")
def gpu():
    import torch
    assert torch.cuda.is_available(), "these tests need a GPU"
    import pcmi355
    return torch, pcmi355


def _scores(torch, dtype, shape, seed, kind="plain"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * 3.0 - 1.0
    C = shape[-1]
    if kind == "masked":                              # a third of the categories, and every fifth row altogether
        x.masked_fill_(torch.rand(C, generator=g) < 0.33, -float("inf"))
        x.view(-1, C)[::5] = -float("inf")
    elif kind == "lowest":                            # masks of the type's lowest value, a row of nothing else
        x.masked_fill_(torch.rand(C, generator=g) < 0.33, torch.finfo(getattr(torch, dtype)).min)
        x.view(-1, C)[::5] = torch.finfo(getattr(torch, dtype)).min
    elif kind == "ties":                              # three values, and a row of one
        x = torch.randint(0, 3, shape, generator=g).float() * torch.tensor([0.5])
        x.view(-1, C)[-1] = -0.0
    elif kind == "rising":                            # every entry is the likeliest so far
        x = torch.arange(C).float().expand(shape) * (8.0 / C) + torch.zeros(shape)
    elif kind == "falling":
        x = -torch.arange(C).float().expand(shape) * (8.0 / C) + torch.zeros(shape)
    elif kind == "nan":
        x.view(-1, C)[0, C // 2] = float("nan")
        x.view(-1, C)[-1, C - 1] = float("inf")
    elif kind == "peaked":
        x.view(-1, C)[:, C // 3] += 40.0
    elif kind == "wide":                              # far from zero, far apart
        x = x * 100.0 - 5000.0
    return x.to(getattr(torch, dtype))


def _numbers(t):
    return t.double().cpu().numpy().reshape(-1, t.shape[-1])


def _near(got, want, bound, what):
    got, want = got.double().cpu().numpy().reshape(want.shape), want
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad), what
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), what
    ok = ~bad & ~inf
    off = np.abs(got[ok] - want[ok])
    past = off - np.broadcast_to(bound, want.shape)[ok]
    assert off.size == 0 or past.max() <= 0, (what, float(off.max()), float(past.max()))


def _check(torch, P, x, dtype, given, top, entropy=True, checkpoint=False):
    s = P.category_scores(x, given, top=top, entropy=entropy, checkpoint=checkpoint)
    rows, C = x.shape[:-1], x.shape[-1]
    raw = _numbers(x)
    y = R.seen(raw, dtype)
    z, h = R.statistics(y)
    near = R.log_bound(y, z, C)
    assert s.log_sum.shape == rows and s.log_sum.dtype == torch.float32
    _near(s.log_sum, z, near, "log_sum")
    if entropy:
        _near(s.entropy, h, R.entropy_bound(y, z, C), "entropy")
    else:
        assert s.entropy is None
    if given is not None:
        g = given.cpu().numpy().astype(np.int64).reshape(len(y), -1)
        assert s.logp.shape == given.shape
        _near(s.logp, R.logp_of(y, g), near[:, None], "logp")
    if top:
        index, logp = R.likeliest(y, top)
        assert s.top.shape == (*rows, top) and s.top.dtype == torch.int32
        assert np.array_equal(s.top.cpu().numpy().reshape(index.shape), index), "top"
        _near(s.top_logp, logp, near[:, None], "top_logp")
    if checkpoint:
        back = s.checkpoint.restore(torch.float32)
        assert np.array_equal(_numbers(back), R.rounded(raw, dtype), equal_nan=True), "checkpoint"
        assert (s.checkpoint.codes[:, C:] == 255).all()
    return s


SHAPES = [(1, 1), (3, 2), (70, 3), (5, 7), (130, 16), (9, 31), (65, 33), (4, 63), (4, 64), (7, 65), (33, 100), (8, 128), (3, 250), (21, 256),
          (6, 257), (5, 300), (4, 511), (3, 512), (3, 513), (9, 1000), (2, 1024), (3, 1025), (5, 2047), (2, 2048), (3, 2049), (2, 4100),
          (3, 10007), (2, 16384), (1, 50021), (2, 131072)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_scores_of_every_length(gpu, dtype, shape):
    torch, P = gpu
    g = torch.Generator().manual_seed(shape[1])
    x = _scores(torch, dtype, shape, 100 + shape[1]).cuda()
    given = torch.randint(0, shape[1], (shape[0],), generator=g).cuda()
    _check(torch, P, x, dtype, given, 0, checkpoint=True)
    _check(torch, P, x, dtype, None, min(8, shape[1] + 1), entropy=False)
    _check(torch, P, x, dtype, given.int()[:, None].repeat(1, 3), 20 if shape[1] > 300 else 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["masked", "lowest", "ties", "rising", "falling", "nan", "peaked", "wide"])
@pytest.mark.parametrize("shape", [(11, 5), (12, 30), (11, 130), (11, 256), (6, 700), (6, 3001), (6, 20000)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_scores_of_every_kind(gpu, dtype, kind, shape):
    torch, P = gpu
    x = _scores(torch, dtype, shape, 7, kind).cuda()
    given = torch.randint(-2, shape[1] + 2, (shape[0], 5), generator=torch.Generator().manual_seed(8)).cuda()
    _check(torch, P, x, dtype, given, 10, checkpoint=True)
    _check(torch, P, x, dtype, given[:, 0], 64)
    _check(torch, P, x, dtype, given[:, 0], 1, entropy=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [4, 17, 128, 400, 5000])
@pytest.mark.parametrize("layout", ["examples last", "sliced", "every second", "spread", "one row for all", "offset", "variables first"])
def test_scores_of_every_layout(gpu, dtype, C, layout):
    torch, P = gpu
    n, v = 70, 3
    if layout == "examples last":                     # what a forest's forward pass leaves: [variable][category][example]
        x = _scores(torch, dtype, (v, C, n), 1).cuda().permute(2, 0, 1)
    elif layout == "variables first":
        x = _scores(torch, dtype, (v, n, C), 2).cuda().transpose(0, 1)
    elif layout == "sliced":
        x = _scores(torch, dtype, (n, v, C + 3), 3).cuda()[:, :, 1:C + 1]
    elif layout == "every second":
        x = _scores(torch, dtype, (n, v, 2 * C), 4).cuda()[:, :, ::2]
    elif layout == "spread":
        x = _scores(torch, dtype, (C, n, v), 5).cuda().permute(1, 2, 0)
    elif layout == "one row for all":
        x = _scores(torch, dtype, (1, v, C), 6).cuda().expand(n, v, C)
    else:
        x = _scores(torch, dtype, (n * v * C + 1,), 7).cuda()[1:].view(n, v, C)
    given = torch.randint(0, C, (v, n), generator=torch.Generator().manual_seed(9), dtype=torch.uint8 if C <= 256 else torch.int64)
    given = given.cuda().t()                          # strides of its own
    s = _check(torch, P, x, dtype, given, 5, checkpoint=True)
    _check(torch, P, x[:, 1], dtype, given[:, 1], 20)
    flat = P.category_scores(x.contiguous(), given.contiguous(), top=5, entropy=True)
    assert torch.equal(s.top, flat.top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(24, 5), (24, 30), (24, 200), (24, 700), (24, 20000), (65544, 40)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_scores_far_from_zero(gpu, dtype, shape):
    """Rows of any level up to the largest number of the type: their log-probabilities and entropies depend on differences only"""
    torch, P = gpu
    n, C = shape
    levels = [0.0, -5000.0, 3e4, -3e4] if dtype == "float16" else \
        [5e3, -5e3, 1e6, -1e6, 2e9, -2e9, 2.0 ** 30, -2.0 ** 30, 2.0 ** 30 - 64, 64 - 2.0 ** 30, 7e12, -7e12, 1e20, -1e20, 1.5e38, -1.5e38, 3.3e38]
    g = torch.Generator().manual_seed(C)
    x = torch.randint(-3, 3, shape, generator=g).double() * 0.75 + torch.tensor(levels).double()[torch.arange(n) % len(levels), None]
    x[:, C // 2:] -= x[:, C // 2:].abs() * 2.0 ** -6    # some far below, at the end
    x[-1, C - 1] = x[-1, 0] + 40.0                      # and a largest one late
    x = x.to(getattr(torch, dtype)).cuda()
    given = torch.randint(0, C, (n, 3), generator=g).cuda()
    few = slice(-24, None)
    raw = _numbers(x[few])
    want, (index, best) = R.logp_of(raw, given[few].cpu().numpy()), R.likeliest(raw, 9)
    # as R.sum_bound, whose arguments are now off by the rounding of up to 64 more, and the roundings of a difference and of two logarithms
    slack = R.sum_bound(C) + 128 * R.EPS
    bound = lambda lp: slack + 8 * R.EPS * (np.abs(np.where(np.isfinite(lp), lp, 0.0)) + 84.0)
    for entropy, top in ((True, 9), (False, 0), (True, 1)):
        s = P.category_scores(x, given, top=top, entropy=entropy)
        _near(s.log_sum[few], R.statistics(raw)[0], R.log_bound(raw, R.statistics(raw)[0], C), "log_sum")
        _near(s.logp[few], want, bound(want), "logp")
        if entropy:
            _near(s.entropy[few], R.statistics(raw)[1], R.entropy_bound(raw, 0.0, C) + 256 * R.EPS * (2.0 + np.log(C)), "entropy")
        if top:
            assert np.array_equal(s.top[few].cpu().numpy(), index[:, :top])
            _near(s.top_logp[few], best[:, :top], bound(best[:, :top]), "top_logp")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(40, 2), (40, 30), (40, 250), (40, 900), (3, 90000), (65600, 20), (6200, 50)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_rows_of_one_category_are_certain(gpu, dtype, shape):
    """All but one category masked: its log-probability and the entropy are 0, not nearly, and the gradient vanishes"""
    torch, P = gpu
    n, C = shape
    g = torch.randint(0, C, (n,), generator=torch.Generator().manual_seed(C))
    x = torch.full(shape, -float("inf"))
    x[torch.arange(n), g] = torch.randn(n) * 9.0 - 2.0
    x = x.to(getattr(torch, dtype)).cuda()
    for y in (x, x.t().contiguous().t()):
        for top in (0, 1, 3):
            s = P.category_scores(y, g.cuda(), top=top, entropy=True)
            assert (s.logp == 0).all() and (s.entropy == 0).all()
            assert torch.equal(s.log_sum, x.float().amax(1))
            if top:
                assert torch.equal(s.top[:, 0].cpu().long(), g) and (s.top_logp[:, 0] == 0).all() and (s.top[:, 1:] == -1).all()
        d = P.category_scores_backward(y, s.log_sum, g.cuda(), grad_logp=torch.ones(n, device="cuda"), entropy=s.entropy, grad_entropy=torch.ones(n, device="cuda"))
        assert (d == 0).all()


@pytest.mark.parametrize("type_", ["uint8", "int32", "int64"])
def test_given_of_every_type_and_number(gpu, type_):
    torch, P = gpu
    x = _scores(torch, "float32", (40, 300), 11).cuda()
    for slots in (1, 2, 16, 63, 64):
        g = torch.randint(0, 250, (40, slots), generator=torch.Generator().manual_seed(slots)).to(getattr(torch, type_)).cuda()
        _check(torch, P, x, "float32", g, 0)
    if type_ == "int64":                              # not wrapped to 32 bits
        g = torch.full((40,), (1 << 32) + 3, device="cuda")
        assert torch.isnan(P.category_scores(x, g).logp).all()
        assert (P.category_scores(x, -g).logp == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(65537, 17), (65600, 33), (65536, 130), (32769, 257), (32800, 511), (32768, 1100)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_scores_of_many_short_rows(gpu, dtype, shape):
    """A lane a row: the last rows of a wave, of a workgroup, and rows whose list keeps changing"""
    torch, P = gpu
    n, C = shape
    kinds = ("plain", "masked", "ties", "rising", "falling", "nan", "lowest")
    x = torch.cat([_scores(torch, dtype, (n // 7 + 1, C), 61 + k, kind) for k, kind in enumerate(kinds)])[:n].cuda()
    x = x[torch.randperm(n, generator=torch.Generator().manual_seed(1)).cuda()]      # kinds side by side
    given = torch.randint(0, C, (n,), generator=torch.Generator().manual_seed(2)).cuda()
    for top in (0, 1, 4, 7, 16):
        s = P.category_scores(x, given, top=top, entropy=True)
        few = slice(None) if top == 4 else slice(n - 300, n)                          # all of them once, the last ones always
        t = P.category_scores(x[few][:300], given[few][:300], top=top, entropy=True)
        _check(torch, P, x[few][-300:], dtype, given[few][-300:], top)
        for a, b in zip(s[:5], t[:5]):
            if a is not None:
                a = a[few][:300]
                if a.dtype == torch.int32:
                    assert torch.equal(a, b)
                else:                                                                 # another order of the same sums
                    assert torch.equal(torch.isfinite(a), torch.isfinite(b))
                    assert (torch.nan_to_num(a, 0, 0, 0) - torch.nan_to_num(b, 0, 0, 0)).abs().max() < 5e-5
    if C == 130:
        v = x.view(256, 256, C)
        g = given.view(256, 256).t().contiguous().t()                                # given of other strides than the rows
        s = P.category_scores(v, g, top=3)
        t = P.category_scores(x, given, top=3)
        assert torch.equal(s.top.view(-1, 3), t.top) and torch.equal(torch.nan_to_num(s.logp.reshape(-1), 7), torch.nan_to_num(t.logp, 7))


def _within(torch, got, want, bound, what):
    """_near on the device: NaN where NaN is wanted, the same infinities, the rest within the bound"""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), what
    past = torch.where(torch.isfinite(want), (got - want).abs() - bound, 0.0)
    assert past.max() <= 0, (what, float(past.max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(65537, 17), (65600, 33), (65536, 130), (32769, 257), (32800, 511), (32768, 1100)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_every_one_of_many_short_rows(gpu, dtype, shape):
    """A lane a row: each row of every kind against its definition in 64 bits, here on the device"""
    torch, P = gpu
    n, C = shape
    kinds = ("plain", "masked", "ties", "rising", "falling", "nan", "lowest")
    x = torch.cat([_scores(torch, dtype, (n // 7 + 1, C), 101 + k, kind) for k, kind in enumerate(kinds)])[:n].cuda()
    x = x[torch.randperm(n, generator=torch.Generator().manual_seed(1)).cuda()]
    given = torch.randint(-1, C + 1, (n, 2), generator=torch.Generator().manual_seed(2)).cuda()
    y = x.double()
    y = torch.where(y <= R.LOWEST[dtype] / 2, -np.inf, y)
    bad = (torch.isnan(y) | (y == np.inf)).any(1)
    none = ~bad & (y == -np.inf).all(1)
    nan, inf = torch.full((), np.nan, dtype=torch.float64, device="cuda"), torch.full((), np.inf, dtype=torch.float64, device="cuda")
    m = torch.where(bad | none, 0.0, y.amax(1))
    d = y - m[:, None]
    q = torch.log(d.exp().sum(1))
    lp = d - q[:, None]
    z = torch.where(bad, nan, torch.where(none, -inf, m + q))
    h = torch.where(bad | none, nan, -torch.where(lp > -np.inf, lp.exp() * lp, 0.0).sum(1))
    lp = torch.where(bad[:, None], nan, torch.where(none[:, None], -inf, lp))
    want = lp.gather(1, given.clamp(0, C - 1))
    want = torch.where(given < 0, 0.0, torch.where(given >= C, nan, want))
    value, index = torch.sort(torch.where(bad[:, None], -inf, y), dim=1, descending=True, stable=True)
    index = torch.where(value > -np.inf, index, -1)[:, :16]
    best = torch.where(bad[:, None], nan, torch.where(index >= 0, lp.gather(1, index.clamp(min=0)), -inf))
    # the sums of R.sum_bound, but added up by one lane: 16 entries one after the other, then C / 16 groups, then up to four parts
    chain = (2 * 104 + 4 + C / 16 + 16 + 4) * R.EPS
    near = chain + 4 * R.EPS * (torch.where(torch.isfinite(y), y.abs(), 0.0).amax(1) + torch.nan_to_num(z.abs(), 0.0, 0.0) + 20.0)
    for top in (0, 1, 4, 7, 16):
        s = P.category_scores(x, given, top=top, entropy=True)
        _within(torch, s.log_sum, z, near, "log_sum")
        _within(torch, s.entropy, h, (chain + 8 * R.EPS) * (2.0 + 2.0 * np.log(C + 1.0)), "entropy")
        _within(torch, s.logp, want, near[:, None], "logp")
        if top:
            assert torch.equal(s.top.long(), index[:, :top])
            _within(torch, s.top_logp, best[:, :top], near[:, None], "top_logp")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [3, 20, 128, 256, 300, 2100])
@pytest.mark.parametrize("last", ["examples", "variables"])
def test_scores_of_many_rows_side_by_side(gpu, dtype, C, last):
    """As many as go a lane each, and a few less"""
    torch, P = gpu
    kinds = ("plain", "masked", "ties", "rising", "falling", "nan", "lowest")
    for rows in ((6147, 6141) if C <= 256 else (2049, 2046)):
        v = 3
        n = rows // v
        y = torch.cat([_scores(torch, dtype, (rows // 7 + 1, C), 81 + k, kind) for k, kind in enumerate(kinds)])[:rows].cuda()
        y = y[torch.randperm(rows, generator=torch.Generator().manual_seed(1)).cuda()].view(n, v, C)
        x = y.permute(1, 2, 0).contiguous().permute(2, 0, 1) if last == "examples" else y.transpose(1, 2).contiguous().transpose(1, 2)
        given = torch.randint(-1, C + 1, (n, v), generator=torch.Generator().manual_seed(2)).cuda()
        for top in (0, 2, 8, 15):
            s = P.category_scores(x, given, top=top, entropy=True)
            t = P.category_scores(y, given, top=top, entropy=True)
            if top:
                assert torch.equal(s.top, t.top)
            few = slice(n - 60, n)
            _check(torch, P, x[few], dtype, given[few], top)
            raw = _numbers(x[few])
            z, h = R.statistics(R.seen(raw, dtype))
            _near(s.log_sum[few], z, R.log_bound(R.seen(raw, dtype), z, C), "log_sum")
            _near(s.entropy[few], h, R.entropy_bound(R.seen(raw, dtype), z, C), "entropy")
            want = R.logp_of(R.seen(raw, dtype), given[few].cpu().numpy().reshape(-1, 1))
            _near(s.logp[few].reshape(-1, 1), want, R.log_bound(R.seen(raw, dtype), z, C)[:, None], "logp")


def test_no_rows(gpu):
    torch, P = gpu
    x = torch.zeros((0, 10), device="cuda")
    s = P.category_scores(x, torch.zeros(0, dtype=torch.int64, device="cuda"), top=3, entropy=True, checkpoint=True)
    assert s.logp.shape == (0,) and s.top.shape == (0, 3) and s.checkpoint.restore().shape == (0, 10)
    assert P.category_scores_backward(x, s.log_sum).shape == (0, 10)
    assert P.category_scores(torch.zeros((4, 0, 10), device="cuda"), top=2).top.shape == (4, 0, 2)


# ---- gradients ----------------------------------------------------------------------------------------------------

def _slots(torch, rows, C, k, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-1, C, (*rows, k), generator=g).cuda(), torch.randn((*rows, k), generator=g).cuda()


def _check_grad(torch, P, x, dtype, k=2, top=0, gh=True, kept=False, out=None, seed=5):
    rows, C = tuple(x.shape[:-1]), x.shape[-1]
    s = P.category_scores(x, top=top, entropy=True, checkpoint=kept)
    kw, slots = {}, []
    given = None
    if k:
        given, kw["grad_logp"] = _slots(torch, rows, C, k, seed)
        slots.append((given.cpu().numpy().reshape(-1, k), _numbers(kw["grad_logp"])))
    if top:
        kw["top"], kw["grad_top"] = s.top, _slots(torch, rows, C, top, seed + 1)[1]
        slots.append((s.top.cpu().numpy().reshape(-1, top), _numbers(kw["grad_top"])))
    w = None
    if gh:
        kw["entropy"], kw["grad_entropy"] = s.entropy, torch.randn(rows, generator=torch.Generator().manual_seed(seed + 2)).cuda()
        w = kw["grad_entropy"].double().cpu().numpy().reshape(-1)
    y = _numbers(x)
    z, h = (t.double().cpu().numpy().reshape(-1) for t in (s.log_sum, s.entropy))
    want, size, under = R.gradient(R.rounded(y, dtype) if kept else R.seen(y, dtype), z, h, slots, w)
    got = P.category_scores_backward(s.checkpoint if kept else x, s.log_sum, given, out=out, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype and (out is None or got is out)
    # the terms' sizes carry the roundings in 32 bits: a dozen operations, one addition per slot; then one to the type,
    # the smallest normal number, and underflow
    bound = size * ((16 + k + top) * R.EPS) + np.abs(np.nan_to_num(want)) * R.HALF[dtype] + R.TINY[dtype] + 2.0 ** -126 + under
    _near(got, want.reshape(-1, C), bound, "gradient")
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kept", [False, True], ids=["scores", "8 bits"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_gradient_of_every_length(gpu, dtype, kept, shape):
    torch, P = gpu
    x = _scores(torch, dtype, shape, 200 + shape[1]).cuda()
    _check_grad(torch, P, x, dtype, k=1, gh=False, kept=kept)
    _check_grad(torch, P, x, dtype, k=7, top=min(5, shape[1]), kept=kept)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kept", [False, True], ids=["scores", "8 bits"])
@pytest.mark.parametrize("kind", ["masked", "lowest", "ties", "nan", "peaked", "wide"])
@pytest.mark.parametrize("shape", [(12, 30), (11, 256), (6, 700), (6, 9000)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_gradient_of_every_kind(gpu, dtype, kept, kind, shape):
    torch, P = gpu
    x = _scores(torch, dtype, shape, 17, kind).cuda()
    _check_grad(torch, P, x, dtype, k=3, top=4, kept=kept)
    _check_grad(torch, P, x, dtype, k=0, kept=kept)
    _check_grad(torch, P, x, dtype, k=64, top=64, gh=False, kept=kept)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kept", [False, True], ids=["scores", "8 bits"])
@pytest.mark.parametrize("C", [4, 128, 5000])
def test_gradient_into_every_layout(gpu, dtype, kept, C):
    torch, P = gpu
    n, v = 70, 3
    t = getattr(torch, dtype)
    heads = _scores(torch, dtype, (v, C, n), 1).cuda().permute(2, 0, 1)
    assert _check_grad(torch, P, heads, dtype, kept=False).stride() == heads.stride()
    for x in (heads, heads.contiguous(), _scores(torch, dtype, (n, v, C + 3), 3).cuda()[:, :, 1:C + 1]):
        _check_grad(torch, P, x, dtype, kept=kept)
        around = torch.full((n, v, C + 5), 7.0, dtype=t, device="cuda")
        _check_grad(torch, P, x, dtype, kept=kept, out=around[:, :, 2:C + 2])
        assert (around[:, :, :2] == 7).all() and (around[:, :, C + 2:] == 7).all()      # nothing beside the rows is touched
        _check_grad(torch, P, x, dtype, kept=kept, out=torch.empty((v, C, n), dtype=t, device="cuda").permute(2, 0, 1))
        _check_grad(torch, P, x, dtype, kept=kept, out=torch.empty((n, v, 2 * C), dtype=t, device="cuda")[:, :, 1::2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [5, 100, 256, 1001, 20000])
def test_gradient_in_place_of_the_scores(gpu, dtype, C):
    torch, P = gpu
    x = _scores(torch, dtype, (9, C), 23).cuda()
    g, w = _slots(torch, (9,), C, 6, 1)
    s = P.category_scores(x, g, top=min(C, 8), entropy=True)
    kw = dict(grad_logp=w, entropy=s.entropy, grad_entropy=torch.ones(9, device="cuda"), top=s.top, grad_top=torch.ones(s.top.shape, device="cuda"))
    want = P.category_scores_backward(x, s.log_sum, g, **kw)
    assert P.category_scores_backward(x, s.log_sum, g, out=x, **kw) is x and torch.equal(x, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [3, 70, 300, 5000])
@pytest.mark.parametrize("slots", [1, 9])
def test_gradient_of_rows_of_nothing_but_masks(gpu, dtype, C, slots):
    """Zeros, whatever their slots: missing, within the row or past it; a row beside them with a slot past its end is NaN"""
    torch, P = gpu
    n = 70
    for mask in (-float("inf"), R.LOWEST[dtype]):
        x = _scores(torch, dtype, (n, C), 29)
        x[::2] = mask
        g = torch.full((n, slots), C, dtype=torch.int64)
        g[::4] = C - 1
        g[2::8, 0] = -1
        x, g, one = x.cuda(), g.cuda(), torch.ones(n, device="cuda")
        s = P.category_scores(x, entropy=True, checkpoint=True)
        for source in (x, s.checkpoint):
            for kw in (dict(), dict(entropy=s.entropy, grad_entropy=one)):
                for out in (torch.empty((n, C), dtype=x.dtype, device="cuda"), torch.empty((C, n), dtype=x.dtype, device="cuda").t()):
                    d = P.category_scores_backward(source, s.log_sum, g, grad_logp=one[:, None].expand(n, slots), out=out, **kw)
                    assert (d[::2] == 0).all() and torch.isnan(d[1::2]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [40, 128, 300, 500, 900])
@pytest.mark.parametrize("kept", [False, True], ids=["scores", "8 bits"])
def test_gradient_of_many_slots_in_few_categories(gpu, dtype, kept, C):
    """Slots that share categories, in every layout of the gradient: the same bits every time (the order of a row's total differs
    between layouts)"""
    torch, P = gpu
    n, k = 301, 20
    x = _scores(torch, dtype, (n, C), 27, "masked").cuda()
    gen = torch.Generator().manual_seed(C)
    g, w = torch.randint(-1, 4, (n, k), generator=gen).cuda() * (C // 4), torch.randn((n, k), generator=gen).cuda()
    g[7, 3] = C
    s = P.category_scores(x, g, entropy=True, checkpoint=True)
    source = s.checkpoint if kept else x
    for kw in (dict(), dict(entropy=s.entropy, grad_entropy=w[:, 0].contiguous())):
        want = P.category_scores_backward(source, s.log_sum, g, grad_logp=w, **kw)
        raw = _numbers(x)
        z, h = s.log_sum.double().cpu().numpy(), s.entropy.double().cpu().numpy()
        exact, size, under = R.gradient(R.rounded(raw, dtype) if kept else R.seen(raw, dtype), z, h, [(g.cpu().numpy(), _numbers(w))],
                                        _numbers(w)[:, 0] if kw else None)
        bound = size * ((16 + k) * R.EPS) + np.abs(np.nan_to_num(exact)) * R.HALF[dtype] + R.TINY[dtype] + 2.0 ** -126 + under
        _near(want, exact, bound, "gradient")
        for out in (torch.empty((C, n), dtype=x.dtype, device="cuda").t(), torch.empty((n, 2 * C), dtype=x.dtype, device="cuda")[:, ::2], torch.empty_like(x)):
            got = P.category_scores_backward(source, s.log_sum, g, grad_logp=w, out=out, **kw)
            _near(got, exact, bound, "gradient")
            first = torch.nan_to_num(got.double(), 1e300)
            again = P.category_scores_backward(source, s.log_sum, g, grad_logp=w, out=out.zero_(), **kw)
            assert torch.equal(torch.nan_to_num(again.double(), 1e300), first)


def test_results_refuse_to_overlap_what_is_read(gpu):
    torch, P = gpu
    x = torch.randn((8, 64), device="cuda")
    g = torch.zeros(8, dtype=torch.int64, device="cuda")
    s = P.category_scores(x, g, checkpoint=True)
    buf = torch.zeros(8 * 64 + 8, device="cuda")
    for k in (0, 500):
        w = buf[k:k + 8]
        with pytest.raises(ValueError, match="overlaps"):
            P.category_scores_backward(x, s.log_sum, g, grad_logp=w, out=buf[:512].view(8, 64))
        with pytest.raises(ValueError, match="overlaps"):
            P.category_scores_backward(x, w, out=buf[:512].view(8, 64))
    P.category_scores_backward(x, s.log_sum, g, grad_logp=buf[512:], out=buf[:512].view(8, 64))
    bytes_ = torch.zeros(8 * 64 * 5, dtype=torch.uint8, device="cuda")
    kept = P.Checkpoint8(bytes_[:512].view(8, 64), s.checkpoint.scales, (8, 64), torch.float32)
    out = bytes_[496:496 + 2048].view(torch.float32).view(8, 64)
    with pytest.raises(ValueError, match="overlaps"):
        kept.restore(out=out)
    with pytest.raises(ValueError, match="overlaps"):
        P.category_scores_backward(kept, s.log_sum, out=out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [20, 129, 1000])
def test_results_beside_what_is_read(gpu, dtype, C):
    """A gradient into the other columns, or the other rows, of the buffer that holds the scores; rows back beside their source"""
    torch, P = gpu
    n, t = 150, getattr(torch, dtype)
    buf, side = torch.empty((2 * n, 2 * C + 3), dtype=t, device="cuda"), torch.empty((2 * C, n), dtype=t, device="cuda")
    for x, out in ((buf[:n, :C], buf[:n, C + 3:]), (buf[::2, :C], buf[1::2, :C]), (buf[:n, :2 * C:2], buf[:n, 1:2 * C:2]),
                   (side[::2].t(), side[1::2].t())):
        x.copy_(_scores(torch, dtype, (n, C), 71).cuda())
        before = x.clone()
        kept = P.checkpoint_rows(x)
        _check_grad(torch, P, x, dtype, k=3, out=out)
        assert torch.equal(x, before)
        _check_grad(torch, P, x, dtype, k=3, kept=True, out=out)
        assert kept.restore(out=out) is out and torch.equal(out, kept.restore()) and torch.equal(x, before)


def test_gradient_refuses_overlapping_results(gpu):
    torch, P = gpu
    buf = torch.zeros(200, device="cuda")
    x = buf[:80].view(8, 10)
    z = P.category_scores(x).log_sum
    for out in (buf[5:85].view(8, 10), buf[:10].expand(8, 10), torch.zeros((8, 10)), torch.zeros((8, 9), device="cuda"),
                torch.zeros((8, 10), device="cuda", dtype=torch.float16)):
        with pytest.raises(ValueError):
            P.category_scores_backward(x, z, out=out)
    with pytest.raises(ValueError):
        P.category_scores(x, torch.zeros(8, dtype=torch.int64))                          # given on the host
    with pytest.raises(ValueError):
        P.category_scores_backward(x, z.cpu())


def test_gradient_is_the_derivative(gpu):
    """Central differences of the forward pass itself: its values are off by about 1e-6, the step is 1e-2, third derivatives
    are of order one: 2 x 1e-6 / 2e-2 + 1e-4 / 6 for each of the four summands"""
    torch, P = gpu
    C = 40
    x = _scores(torch, "float32", (1, C), 31).cuda()
    g, w = torch.tensor([[3, 17, 3]]).cuda(), torch.tensor([[0.5, -1.0, 0.25]]).cuda()
    s = P.category_scores(x, g, entropy=True)
    grad = P.category_scores_backward(x, s.log_sum, g, grad_logp=w, entropy=s.entropy, grad_entropy=torch.tensor([0.7]).cuda())[0]
    step = 1e-2
    moved = x + torch.cat([torch.eye(C), -torch.eye(C)]).cuda() * step
    t = P.category_scores(moved, g.expand(2 * C, 3), entropy=True)
    loss = (t.logp.double() * w.double()).sum(1) + 0.7 * t.entropy.double()
    diff = (loss[:C] - loss[C:]) / (2 * step)
    assert (diff - grad.double()).abs().max() < 4 * (1e-4 + 2e-5)


# ---- 8 bits -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["plain", "masked", "lowest", "ties", "rising", "nan", "wide"])
@pytest.mark.parametrize("shape", [(5, 1), (3, 15), (7, 64), (4, 65), (3, 128), (9, 1000), (2, 10007), (1, 70001)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_rows_in_eight_bits(gpu, dtype, kind, shape):
    torch, P = gpu
    x = _scores(torch, dtype, shape, 41, kind).cuda()
    kept = P.checkpoint_rows(x)
    want = R.rounded(_numbers(x), dtype)
    back = kept.restore(torch.float32)
    assert np.array_equal(_numbers(back), want, equal_nan=True)
    own = kept.restore()
    top = torch.finfo(x.dtype).max
    assert own.dtype == x.dtype and torch.equal(torch.nan_to_num(own, 1e3), torch.nan_to_num(back.clamp(max=top).to(x.dtype), 1e3))
    assert kept.codes.shape == (shape[0], -(-shape[1] // 16) * 16) and (kept.codes[:, shape[1]:] == 255).all()


@pytest.mark.parametrize("C", [64, 200, 1000])
def test_gradient_from_eight_bits_far_from_zero(gpu, C):
    """Likelihoods of whole images lie thousands below zero: what 8 bits may cost their probabilities there, and that scores less
    their log-sum pay for their range alone"""
    torch, P = gpu
    n = 300
    g, w = _slots(torch, (n,), C, 1, 3)
    slots = [(g.cpu().numpy(), _numbers(w))]
    for level in (0.0, -600.0, -3000.0, -8000.0, -20000.0):
        x = (torch.randn((n, C), generator=torch.Generator().manual_seed(C)) * 2.5 + level).cuda()
        z = P.category_scores(x).log_sum
        for y, far in ((x, True), (x - z[:, None], False)):
            s = P.category_scores(y, checkpoint=True)
            raw = _numbers(y)
            half = np.zeros(n)
            for b in range(0, C, 64):
                part = raw[:, b:b + 64]
                # a block of few entries may span less than the level alone asks for: of a row less its log-sum |x| is below 64
                half = np.maximum(half, np.maximum(np.ptp(part, axis=1) / 253, np.abs(part).max(1) / 2.0 ** 14))
            assert far or half.max() <= max(np.ptp(raw, axis=1).max() / 253, 64 / 2.0 ** 14)
            want, size, under = R.gradient(raw, s.log_sum.double().cpu().numpy(), None, slots)
            got = P.category_scores_backward(s.checkpoint, s.log_sum, g, grad_logp=w)
            # p |w| times what half a step makes of p, and roundings in 32 bits of the larger p
            p = np.exp(raw - s.log_sum.double().cpu().numpy()[:, None]) * np.abs(_numbers(w)) * (g.cpu().numpy() >= 0)
            bound = p * np.expm1(half)[:, None] + size * np.exp(half)[:, None] * 17 * R.EPS + 2.0 ** -126 + under
            _near(got, want, bound, "gradient")


def test_extreme_rows_in_eight_bits(gpu):
    torch, P = gpu
    lo, hi = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max
    rows = [[hi, -hi / 2.1, 1.0, 0.0], [lo, lo / 8, -lo, 0.0], [0.0, -0.0, 0.0, 0.0], [hi, hi, hi, hi], [-hi, -float("inf"), -hi, -hi],
            [1e-3, 1.0, 253.0 / 256, 254.0 / 256], [5.0, 5.0 + 2.0 ** -20, 5.0, 5.0], [-1.6e38, 3.4e38, 0.0, -hi]]
    x = torch.tensor(rows).cuda()
    assert np.array_equal(_numbers(P.checkpoint_rows(x).restore()), R.rounded(_numbers(x), "float32"))
    for t, name in ((torch.float16, "float16"), (torch.bfloat16, "bfloat16")):
        m = torch.finfo(t).max
        y = torch.tensor([[m, -m / 3, 0.5, 1.0], [m, m, m, m], [torch.finfo(t).tiny, 0.0, -torch.finfo(t).tiny, 0.0]], dtype=t).cuda()
        kept = P.checkpoint_rows(y)
        assert np.array_equal(_numbers(kept.restore(torch.float32)), R.rounded(_numbers(y), name))
        assert torch.isfinite(kept.restore()).all()


def test_eight_bits_of_every_layout(gpu):
    torch, P = gpu
    for dtype in TYPES:
        for x in (_scores(torch, dtype, (300, 70), 1).cuda().t(), _scores(torch, dtype, (9, 210), 2).cuda()[:, 3:203],
                  _scores(torch, dtype, (9, 200), 2).cuda()[:, ::2], _scores(torch, dtype, (3, 100, 5), 3).cuda().permute(2, 0, 1),
                  _scores(torch, dtype, (1, 200), 4).cuda().expand(6, 200)):
            kept = P.checkpoint_rows(x)
            want = R.rounded(_numbers(x), dtype)
            assert np.array_equal(_numbers(kept.restore(torch.float32)), want)
            around = torch.full((*x.shape[:-1], x.shape[-1] + 4), 3.0, device="cuda")
            out = around[..., 1:-3]
            assert kept.restore(out=out) is out and np.array_equal(_numbers(out.contiguous()), want)
            assert (around[..., 0] == 3).all() and (around[..., -3:] == 3).all()
            out = torch.zeros(x.shape[::-1], device="cuda").permute(*reversed(range(x.dim())))
            kept.restore(out=out)
            assert np.array_equal(_numbers(out.contiguous()), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [1, 15, 17, 64, 70, 128, 200, 321])
def test_eight_bits_of_many_rows_of_any_strides(gpu, dtype, C):
    """The same codes whatever the strides, rows back into any strides, and gradients from codes and in place"""
    torch, P = gpu
    n, v = 47, 3
    kinds = ("plain", "masked", "lowest", "ties", "rising", "nan", "wide")
    rows = n * v
    y = torch.cat([_scores(torch, dtype, (rows // 7 + 1, C), 91 + k, kind) for k, kind in enumerate(kinds)])[:rows].cuda()
    y = y[torch.randperm(rows, generator=torch.Generator().manual_seed(1)).cuda()].view(n, v, C)
    want = P.checkpoint_rows(y)
    plain, wide = want.restore(), want.restore(torch.float32)
    g, w = _slots(torch, (n, v), C, 6, 3)
    s = P.category_scores(y, g, entropy=True)
    kw = dict(grad_logp=w, entropy=s.entropy, grad_entropy=w[..., 0].contiguous())
    from_codes, from_scores = P.category_scores_backward(want, s.log_sum, g, **kw), P.category_scores_backward(y, s.log_sum, g, **kw)
    same = lambda a, b: torch.equal(torch.nan_to_num(a.double(), 1e300), torch.nan_to_num(b.double(), 1e300))
    layouts = ((lambda t: torch.empty((v, C, n), dtype=t, device="cuda").permute(2, 0, 1)), (lambda t: torch.empty((n, C, v), dtype=t, device="cuda").transpose(1, 2)),
               (lambda t: torch.empty((C, n, v), dtype=t, device="cuda").permute(1, 2, 0)), (lambda t: torch.empty((n, v, 3 * C), dtype=t, device="cuda")[..., 1::3]),
               (lambda t: torch.empty((n, v, C + 1), dtype=t, device="cuda")[..., 1:]))
    for layout in layouts:
        x = layout(y.dtype)
        x.copy_(y)
        kept = P.checkpoint_rows(x)
        assert torch.equal(kept.codes, want.codes) and torch.equal(kept.scales, want.scales)
        kept = P.category_scores(x, checkpoint=True).checkpoint
        assert torch.equal(kept.codes, want.codes) and torch.equal(kept.scales, want.scales)
        assert same(want.restore(out=layout(y.dtype)), plain) and same(want.restore(out=layout(torch.float32)), wide)
        assert same(P.category_scores_backward(want, s.log_sum, g, out=layout(y.dtype), **kw), from_codes)
        assert same(P.category_scores_backward(x, s.log_sum, g, out=layout(y.dtype), **kw), from_scores)
        assert same(P.category_scores_backward(y, s.log_sum, g, out=layout(y.dtype), **kw), from_scores)
        assert same(P.category_scores_backward(x, s.log_sum, g, out=x, **kw), from_scores)


# ---- as they are used ---------------------------------------------------------------------------------------------

def test_same_bits_every_time(gpu):
    torch, P = gpu
    for shape, dtype in (((2, 131072), "bfloat16"), ((700, 256), "float32"), ((5, 20000), "float16")):
        x = _scores(torch, dtype, shape, 51, "ties" if dtype == "bfloat16" else "plain").cuda()
        g, w = _slots(torch, shape[:1], shape[1], 64, 1)
        first = None
        for _ in range(3):
            s = P.category_scores(x, g, top=20, entropy=True)
            d = P.category_scores_backward(x, s.log_sum, g, grad_logp=w, entropy=s.entropy, grad_entropy=w[:, 0])
            got = (*s[:5], d)
            if first is None:
                first = got
            assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_captured_and_replayed(gpu):
    """A training step over 8-bit scores in a graph, replayed on new scores between eager calls on other streams"""
    torch, P = gpu
    for shape, dtype in (((3, 70001), torch.bfloat16), ((50, 256), torch.float32), ((64, 6), torch.float32)):
        C = shape[1]
        x = torch.randn(shape, device="cuda").to(dtype)
        g = torch.randint(0, C, shape[:1], device="cuda")
        w = torch.randn(shape[:1], device="cuda")

        def step(x, g, w):
            s = P.category_scores(x, g, top=4, entropy=True, checkpoint=True)
            d = P.category_scores_backward(s.checkpoint, s.log_sum, g, grad_logp=w, entropy=s.entropy, grad_entropy=w, top=s.top,
                                           grad_top=s.top_logp)
            return s.logp, s.log_sum, s.entropy, s.top, s.top_logp, d, P.category_scores_backward(x, s.log_sum, g, grad_logp=w)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, g, w)
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for _ in range(2):                            # two graphs of the same call, replayed one after the other
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                graphs.append((graph, None))
                out = step(x, g, w)
            graphs[-1] = (graph, out)
        for k in range(4):
            x.copy_(torch.randn(shape, device="cuda"))
            g.copy_(torch.randint(0, C, shape[:1], device="cuda"))
            for graph, _ in graphs:
                graph.replay()
            want = step(x, g, w)
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(out, want)), (shape, k)


def test_on_a_stream_of_its_own(gpu):
    torch, P = gpu
    side = torch.cuda.Stream()
    for shape in ((4, 131072), (3000, 128)):
        host = torch.randn(shape)
        x = torch.empty(shape, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)             # the scores arrive late, on the stream that the call is made on
            x.copy_(host)
            s = P.category_scores(x, top=3, entropy=True, checkpoint=True)
            d = P.category_scores_backward(x, s.log_sum, entropy=s.entropy, grad_entropy=torch.ones(shape[0], device="cuda"))
        side.synchronize()
        t = P.category_scores(x, top=3, entropy=True, checkpoint=True)
        assert torch.equal(s.top, t.top) and torch.equal(s.log_sum, t.log_sum) and torch.equal(s.checkpoint.codes, t.checkpoint.codes)
        assert torch.equal(d, P.category_scores_backward(x, t.log_sum, entropy=t.entropy, grad_entropy=torch.ones(shape[0], device="cuda")))


def test_offsets_beyond_32_bits(gpu):
    """Rows behind 2^31 elements and 2^32 bytes, and categories that lie further apart than that"""
    torch, P = gpu
    buf = torch.zeros((1 << 31) + (1 << 20), dtype=torch.float16, device="cuda")
    far = buf[-(1 << 19):].view(4, -1)
    far.copy_(torch.randn(far.shape, device="cuda"))
    x = buf.as_strided((2, 1 << 17), (buf.numel() - (1 << 17), 1))
    assert x[1].data_ptr() == far[3].data_ptr()
    g = torch.tensor([5, 6], device="cuda")
    w = torch.ones(2, device="cuda")
    s = _check(torch, P, x, "float16", g, 5, checkpoint=True)
    near = x.contiguous()
    want = P.category_scores_backward(near, s.log_sum, g, grad_logp=w)
    assert torch.equal(P.category_scores_backward(x, s.log_sum, g, grad_logp=w, out=x), want) and torch.equal(x, want)
    y = buf.as_strided((1, 2), (1, buf.numel() - 1))
    y.copy_(torch.tensor([[1.0, 2.0]]))
    _check(torch, P, y, "float16", None, 2, checkpoint=True)
    del buf, far, x, y
    torch.cuda.empty_cache()


def test_many_rows(gpu):
    """More rows than a launch has workgroups for"""
    torch, P = gpu
    n = (1 << 21) + 3
    x = torch.randn((n, 3), device="cuda")
    g = torch.randint(0, 3, (n,), device="cuda", dtype=torch.uint8)
    s = P.category_scores(x, g, top=1, entropy=True, checkpoint=True)
    want = torch.log_softmax(x.double(), 1)
    assert (s.logp - want.gather(1, g.long()[:, None])[:, 0]).abs().max() < 2e-6
    assert torch.equal(s.top[:, 0].long(), x.argmax(1))
    d = P.category_scores_backward(x, s.log_sum, g, grad_logp=torch.ones(n, device="cuda"))
    assert (d - (torch.nn.functional.one_hot(g.long(), 3) - want.exp())).abs().max() < 2e-6
    back = s.checkpoint.restore()
    assert (back - x).abs().max() <= (x.amax(1) - x.amin(1)).max() / 126.5 / 2 + 1e-6


# A launch has at most 2^22 workgroups (gradients, tiles of checkpoints and of rows back) or 2^20 (all others); rows
# beyond go to the same workgroups in further turns, which use the LDS and the registers of the turns before.  Rows that overlap in
# memory keep the scores small.  All rows at once, and in parts that a launch takes in one turn: the same bits.

def _whole_and_in_parts(torch, n, parts, call):
    """call(first, end) gives the results of those rows, tensors with a row axis at 0"""
    whole, step = call(0, n), n // parts + 1
    for a in range(0, n, step):
        for w, p in zip(whole, call(a, min(a + step, n))):
            w = w[a:a + step]
            assert w.shape == p.shape and (torch.equal(w, p) if w.dtype in (torch.int32, torch.uint8) else bool((w == p).all()))


@pytest.mark.parametrize("kind, C, per, top, checkpoint, strides", [
    ("a lane a row", 2, 256, 0, False, (1, 1)),
    ("a lane a row by way of LDS", 17, 256, 0, False, (1, 1)),
    ("a lane a row, side by side", 17, 256, 1, False, (1, 3)),
    ("sixteen lanes a row", 40, 16, 3, True, (1, 1)),
    ("a wave a row with a list", 300, 1, 20, False, (1, 1)),
    ("a wave a row with a checkpoint", 300, 1, 0, True, (1, 1)),
    ("a wave a row of any strides", 300, 1, 20, False, (2, 2)),
], ids=lambda v: v.replace(" ", "_") if isinstance(v, str) else None)
def test_scores_of_more_rows_than_workgroups(gpu, kind, C, per, top, checkpoint, strides):
    torch, P = gpu
    most = (1 << 20) * per
    n = most + 5 * per + 3
    buf = torch.randn(strides[0] * n + strides[1] * C, device="cuda").to(torch.float16)
    x = buf.as_strided((n, C), strides)
    given = torch.randint(-1, C, (n,), device="cuda", dtype=torch.int32)

    def call(a, b):
        s = P.category_scores(x[a:b], given[a:b], top=top, entropy=not checkpoint, checkpoint=checkpoint)
        return [t for t in s[:5] if t is not None] + ([s.checkpoint.codes, s.checkpoint.scales] if checkpoint else [])

    _whole_and_in_parts(torch, n, 2, call)
    z = P.category_scores(x, None).log_sum[-300:]
    y = _numbers(x[-300:])
    _near(z, R.statistics(y)[0], R.log_bound(y, R.statistics(y)[0], C), "log_sum")
    del buf, x, given
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind, dtype, C, per, slots, side", [
    ("slots of short rows in LDS", "float16", 2, 256, 1, False),
    ("gradients of short rows in LDS", "float32", 65, 32, 7, False),
    ("side by side", "float16", 2, 256, 1, True),
], ids=lambda v: v.replace(" ", "_") if isinstance(v, str) and " " in v else None)
def test_gradient_of_more_rows_than_workgroups(gpu, kind, dtype, C, per, slots, side):
    torch, P = gpu
    most = (1 << 22) * per
    n, t = most + 5 * per + 3, getattr(torch, dtype)
    x = torch.randn(n + 3 * C, device="cuda", dtype=t).as_strided((n, C), (1, 3) if side else (1, 1))
    z = P.category_scores(x).log_sum
    given = torch.randint(0, C, (n, slots), device="cuda", dtype=torch.uint8)
    w = torch.randn((n, slots), device="cuda")

    def call(a, b):
        out = torch.empty((C, b - a), dtype=t, device="cuda").t() if side else torch.empty((b - a, C), dtype=t, device="cuda")
        return (P.category_scores_backward(x[a:b], z[a:b], given[a:b], grad_logp=w[a:b], out=out),)

    _whole_and_in_parts(torch, n, 4, call)
    want, size, under = R.gradient(_numbers(x[-300:]), z[-300:].double().cpu().numpy(), None, [(given[-300:].cpu().numpy(), _numbers(w[-300:]))])
    got = call(n - 300, n)[0]
    _near(got, want, size * ((16 + slots) * R.EPS) + np.abs(want) * R.HALF[dtype] + R.TINY[dtype] + 2.0 ** -126 + under, "gradient")
    del x, z, given, w, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind, dtype, C, log2_rows, strides", [
    ("tiles", "float32", 2, 26, (1, 1)),
    ("side by side", "float16", 2, 28, (1, 3)),
    ("any strides", "float16", 2, 22, (2, 3)),
], ids=lambda v: v.replace(" ", "_") if isinstance(v, str) and v != "float32" and v != "float16" else None)
def test_checkpoints_of_more_rows_than_workgroups(gpu, kind, dtype, C, log2_rows, strides):
    torch, P = gpu
    n = (1 << log2_rows) + 700
    x = torch.randn(strides[0] * n + strides[1] * C, device="cuda").to(getattr(torch, dtype)).as_strided((n, C), strides)

    def call(a, b):
        kept = P.checkpoint_rows(x[a:b])
        return kept.codes, kept.scales

    _whole_and_in_parts(torch, n, 2, call)
    assert np.array_equal(_numbers(P.checkpoint_rows(x[-300:]).restore(torch.float32)), R.rounded(_numbers(x[-300:]), dtype))
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind, log2_rows", [("tiles", 30), ("side by side", 28), ("any strides", 27)], ids=lambda v: v.replace(" ", "_") if isinstance(v, str) else None)
def test_rows_back_of_more_rows_than_workgroups(gpu, kind, log2_rows):
    torch, P = gpu
    n, C = (1 << log2_rows) + 700, 2
    few = P.checkpoint_rows(torch.randn((1 << 16, C), device="cuda").to(torch.float16))
    turns = n // (1 << 16) + 1
    codes, scales = few.codes.repeat(turns, 1)[:n].contiguous(), few.scales.repeat(turns, 1)[:n].contiguous()
    out = torch.empty((C, n), dtype=torch.float16, device="cuda").t() if kind == "side by side" else torch.empty((n, 2 * C), dtype=torch.float16, device="cuda")[:, ::2] \
        if kind == "any strides" else torch.empty((n, C), dtype=torch.float16, device="cuda")
    want = few.restore()
    P.Checkpoint8(codes, scales, (n, C), torch.float16).restore(out=out)
    for a in range(0, n, 1 << 26):
        part = out[a:a + (1 << 26)]
        assert bool((part == want.repeat(-(-len(part) // (1 << 16)), 1)[:len(part)]).all())
    del codes, scales, out
    torch.cuda.empty_cache()


def test_posterior_of_heads(gpu):
    """A multi-head circuit and a forest: log-posterior of the examples' clusters from the per-head likelihoods"""
    torch, P = gpu
    from pcmi355 import workloads as W
    rng = np.random.default_rng(3)
    V, K, C, H, n = 24, 16, 8, 5, 37
    data = rng.integers(0, C, (n, V)).astype(np.uint8)
    par = W.chow_liu_parent(rng.integers(0, C, (200, V)).astype(np.uint8))
    d = torch.from_numpy(data).cuda()
    for forest in (False, True):
        if forest:
            parent = np.concatenate([par, np.where(par < 0, -1, par + V)]).astype(np.int32)
            c = P.hclt_forest_from_clts(parent, C, K, H)
            x = d.repeat(1, 2)
        else:
            c, x = P.multihead_hclt_from_clt(par, C, K, H), d
        c.set_params(*W.init_params(np.zeros(x.shape[1]), K, C, 4, kind="dirichlet"))
        trees = 2 if forest else 1
        heads = np.log(rng.dirichlet(np.ones(K), (trees, H))).astype(np.float32)
        c.set_heads(heads)
        if forest:
            ll = P.forest_loglikelihoods(c, x).permute(2, 0, 1)
            given = torch.randint(0, H, (n, trees), device="cuda", dtype=torch.uint8)
        else:
            ll = P.loglikelihoods(c, x)
            given = torch.randint(0, H, (n,), device="cuda", dtype=torch.uint8)
        s = P.head_scores(c, x, given, top=2)
        want = torch.log_softmax(ll.double(), -1)
        pick = want.gather(-1, given.long().unsqueeze(-1)).squeeze(-1)
        # a likelihood near -60 has steps of 4e-6; the log-sum is stored at that size, differences are not
        assert (s.logp - pick).abs().max() < 4e-6
        assert torch.equal(s.top.long(), torch.sort(ll, dim=-1, descending=True, stable=True).indices[..., :2])
        assert (s.entropy + (want.exp() * want).sum(-1)).abs().max() < 4e-6
        ids = torch.tensor([5, 0, 30], device="cuda")
        sub = P.head_scores(c, x, given[ids], top=2, example_ids=ids)
        assert torch.equal(sub.top, s.top[ids]) and (sub.logp - s.logp[ids]).abs().max() < 1e-5
        if not forest:
            mix = P.multihead_loglikelihoods(c, x, torch.ones((n, H), device="cuda"))
            assert (s.log_sum - np.log(H) - mix).abs().max() < 2e-5
            part = P.head_scores(c, x, given, top=2, batch_size=10)
            assert torch.equal(part.top, s.top)
    with pytest.raises(ValueError, match="heads"):
        P.head_scores(P.hclt_from_clt(par, C, K), d)


def test_variational_step_from_eight_bits(gpu):
    """KL and relaxed samples whose parameter rows wait for the reverse pass in 8 bits: the gradients are those at the rounded
    rows, bit for bit; forward results are untouched"""
    torch, P = gpu
    from pcmi355 import workloads as W
    prealloc = P.prealloc
    rng = np.random.default_rng(5)
    V, K, C, rows = 12, 16, 12, 6
    par = W.chow_liu_parent(rng.integers(0, C, (200, V)).astype(np.uint8))
    c = P.hclt_from_clt(par, C, K)
    n = c.num_parameters()
    p1, p2 = (np.log(rng.uniform(0.05, 1.0, (rows, n))).astype(np.float32) for _ in range(2))
    p2 = p2[:1]
    r1, r2 = (P.checkpoint_rows(torch.from_numpy(p).cuda()).restore().cpu().numpy() for p in (p1, p2))
    assert np.abs(r1 - p1).max() <= 3.0 / 126 / 2 + 1e-6 and np.abs(r1 - p1).max() > 0
    prealloc.kld_preallocation(c, num_examples=rows)
    want = prealloc.kld_with_prealloc(c, p1, p2)
    prealloc.kld_with_prealloc(c, r1, r2)
    grads = prealloc.kld_backward_with_prealloc(c)
    prealloc.kld_preallocation(c, num_examples=rows, checkpoint=True)
    assert np.array_equal(prealloc.kld_with_prealloc(c, p1, p2), want)
    kept = prealloc._state["kld"]["rows"]
    assert kept[0].nbytes < 4 * rows * n * 0.28
    for a, b in zip(prealloc.kld_backward_with_prealloc(c), grads):
        assert np.array_equal(a, b)
    prealloc.kld_free_mem()

    og = rng.normal(size=(rows, V, C)).astype(np.float32)
    found = []
    for params, checkpoint in ((r1, False), (p1, True)):
        prealloc.gumbel_sample_preallocation(c, num_examples=rows, num_vars=V, par_buffer_size=C, allocate_for_grad=True,
                                             checkpoint=checkpoint)
        gen = torch.Generator(device="cuda").manual_seed(9)
        prealloc.gumbel_sample_with_prealloc(c, params, temperature=0.8, generator=gen)
        found.append(prealloc.gumbel_sample_backward_with_prealloc(c, og, temperature=0.8))
        prealloc.gumbel_sample_free_mem()
    assert np.array_equal(*found)

"""Scores from features and weights on the CPU: the reference against closed forms and differences, and what the entry points refuse."""
import ctypes

import pytest
import torch

import linear_reference as R


def _inputs(seed, n, k, C, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, k, generator=g, dtype=torch.float64).to(dtype), torch.randn(C, k, generator=g, dtype=torch.float64).to(dtype),
            torch.randn(C, generator=g, dtype=torch.float64).to(dtype))


def test_reference_scores():
    f, w, b = _inputs(1, 5, 7, 11, torch.float32)
    s = R.Scores(f, w, b)
    x = torch.nn.functional.linear(f.double(), w.double(), b.double())
    assert torch.allclose(s.x, x, rtol=1e-14, atol=1e-14)
    assert torch.allclose(s.log_sum, torch.log(x.exp().sum(1)), rtol=1e-13)
    b[2] = torch.finfo(torch.float32).min
    w[2] = float("nan")
    s = R.Scores(f, w, b)
    assert torch.isinf(s.x[:, 2]).all() and torch.isfinite(s.log_sum).all()
    lp, _ = s.logp(torch.tensor([[0, -1, 11]]).expand(5, 3))
    assert torch.allclose(lp[:, 0], torch.log_softmax(s.x, 1)[:, 0]) and (lp[:, 1] == 0).all() and torch.isnan(lp[:, 2]).all()
    s = R.Scores(f, w, torch.full_like(b, -float("inf")))
    assert (s.log_sum == -float("inf")).all()


@pytest.mark.parametrize("what", ["features", "weight", "bias"])
def test_reference_gradient_is_the_derivative(what):
    n, k, C = 3, 4, 5
    f, w, b = (t.float() for t in _inputs(2, n, k, C))
    g = torch.tensor([[0, 0, -1], [4, 2, 1], [3, -1, -1]])
    gl, gz = torch.randn(3, 3, generator=torch.Generator().manual_seed(3)), torch.tensor([0.3, -0.2, 0.5])
    # a derivative of the sum by autograd in 64 bits, and by differences
    t = {"features": f.double(), "weight": w.double(), "bias": b.double()}

    def loss(t):
        x = t["features"] @ t["weight"].t() + t["bias"]
        z = torch.logsumexp(x, 1)
        lp = torch.where(g < 0, 0.0, x.gather(1, g.clamp(min=0)) - z[:, None])
        return (lp * gl.double()).sum() + (gz.double() * z).sum()

    got = R.gradients(f, w, b, R.Scores(f, w, b), g, gl, gz)[what][0].reshape(-1)
    h = 1e-6
    for i in range(got.numel()):
        up, down = dict(t), dict(t)
        up[what], down[what] = t[what].clone(), t[what].clone()
        up[what].view(-1)[i] += h
        down[what].view(-1)[i] -= h
        # third derivatives of order 10: h^2 10 / 6, and 1e-15 / 1e-6 of rounding
        assert abs(float((loss(up) - loss(down)) / (2 * h)) - float(got[i])) < 1e-8


def test_reference_codes():
    x = torch.tensor([[1.0, -0.5, 0.25, 0.0], [0.0, 0.0, 0.0, 0.0], [1e-38, 0.0, 0.0, 0.0], [float("nan"), 1.0, 0.0, 0.0],
                      [float("inf"), 1.0, 0.0, 0.0]])
    q, s = R.codes_of(x)
    assert q.tolist() == [[127, -64, 32, 0], [0] * 4, [0] * 4, [0] * 4, [0] * 4]
    assert s[0] == torch.tensor(1.0) / torch.tensor(127.0) and (s[1:3] == 0).all() and torch.isnan(s[3:]).all()


def _cpu():
    import pcmi355 as P
    return P, torch.zeros(4, 8), torch.zeros(10, 8)


def test_arguments_are_checked():
    P, f, w = _cpu()
    given = torch.zeros(4, dtype=torch.int64)
    for call in (lambda *a, **k: P.linear_scores(*a, **k), lambda f, w, *a, **k: P.linear_scores_backward(f, w, torch.zeros(f.shape[:-1]), *a, **k)):
        with pytest.raises(ValueError, match="GPU"):
            call(f, w)
        for bad in (f[0], f.double(), f.int(), f.view(1, 1, 4, 8)):
            with pytest.raises(ValueError, match="features"):
                call(bad, w)
        for bad in (w[0], w.half(), torch.zeros(10, 7), torch.zeros(0, 8), w.view(1, 10, 8)):
            with pytest.raises(ValueError, match="weight"):
                call(f, bad)
        with pytest.raises(ValueError, match="weight"):
            call(torch.zeros(4, 0), torch.zeros(10, 0))
        for bad in (torch.zeros(9), torch.zeros(10, 1), torch.zeros(10, dtype=torch.float64), [0.0] * 10):
            with pytest.raises(ValueError, match="bias"):
                call(f, w, bias=bad)
        with pytest.raises(ValueError, match="2.22 rows"):
            call(torch.zeros(1, 8).expand((1 << 22) + 1, 8), w)
        with pytest.raises(ValueError, match="length"):
            call(torch.zeros(1, 1).expand(4, (1 << 20) + 1), torch.zeros(1, 1).expand(10, (1 << 20) + 1))
    with pytest.raises(ValueError, match="given"):
        P.linear_scores(f, w, given[:3])
    with pytest.raises(ValueError, match="given"):
        P.linear_scores(f, w, given.float())
    with pytest.raises(ValueError, match="64"):
        P.linear_scores(f, w, torch.zeros(4, 65, dtype=torch.int64))
    z = torch.zeros(4)
    with pytest.raises(ValueError, match="together"):
        P.linear_scores_backward(f, w, z, given)
    with pytest.raises(ValueError, match="together"):
        P.linear_scores_backward(f, w, z, grad_logp=z)
    with pytest.raises(ValueError, match="log_sum"):
        P.linear_scores_backward(f, w, torch.zeros(3))
    with pytest.raises(ValueError, match="grad_log_sum"):
        P.linear_scores_backward(f, w, z, grad_log_sum=torch.zeros(3))
    with pytest.raises(ValueError, match="grad_logp"):
        P.linear_scores_backward(f, w, z, given, grad_logp=torch.zeros(4, 1))
    for of in ((), ("weights",), "logits"):
        with pytest.raises(ValueError, match="of must"):
            P.linear_scores_backward(f, w, z, of=of)


def test_eight_bit_arguments_are_checked():
    P, f, w = _cpu()
    for bad in (f[0], f.double(), f.view(1, 1, 4, 8), None):
        with pytest.raises(ValueError, match="rows must"):
            P.rows8(bad)
    with pytest.raises(ValueError, match="131071"):
        P.rows8(torch.zeros(1, 1).expand(2, 131072))
    with pytest.raises(ValueError, match="entries"):
        P.rows8(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="GPU"):
        P.rows8(f)
    eight = lambda n, k: P.Rows8(torch.zeros(n, -(-k // 128) * 128, dtype=torch.int8), torch.zeros(n), (n, k), torch.float32)
    a, b = eight(4, 200), eight(10, 200)
    assert a.nbytes == 4 * 256 + 16
    for codes, scales, shape in ((torch.zeros(4, 200, dtype=torch.int8), torch.zeros(4), (4, 200)), (a.codes.to(torch.uint8), a.scales, (4, 200)),
                                 (a.codes, a.scales[:3], (4, 200)), (a.codes, a.scales.double(), (4, 200)), (a.codes, a.scales, (4, 300)),
                                 (a.codes.t().contiguous().t(), a.scales, (4, 200))):
        with pytest.raises(ValueError, match="no 8-bit rows"):
            P.Rows8(codes, scales, shape, torch.float32)
    with pytest.raises(ValueError, match="rows8 returned"):
        P.product8(f, b)
    with pytest.raises(ValueError, match="channels"):
        P.product8(a, eight(10, 201))
    with pytest.raises(ValueError, match="bias"):
        P.product8(a, b, bias=torch.zeros(4))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        P.product8(a, b, dtype=torch.float64)
    with pytest.raises(ValueError, match="GPU"):
        P.product8(a, b)
    with pytest.raises(ValueError, match="both"):
        P.linear_scores(a, w)
    with pytest.raises(ValueError, match="both"):
        P.linear_scores(f, b)
    with pytest.raises(ValueError, match="gradient"):
        P.linear_scores_backward(a, b, torch.zeros(4))
    with pytest.raises(ValueError, match="GPU"):
        P.linear_scores(a, b)


def test_entry_points_refuse_without_a_gpu():
    from pcmi355._lib import lib
    big = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(big) + 255) & ~255
    much = 1 << 40

    def scores(f=p, w=p, type=0, n=4, v=1, k=8, c=10, bias=None, btype=0, given=None, gtype=5, slots=0, logp=None, work=p, size=much):
        return lib.pcm_linear_scores(f, w, type, k, 0, 1, k, 1, n, v, k, c, bias, btype, given, gtype, 1, 0, 0, slots, logp, None, work, size, None)

    def back(f=p, w=p, type=0, n=4, v=1, k=8, c=10, bias=None, btype=0, given=None, gtype=5, slots=0, gl=None, z=p, work=p, size=much):
        return lib.pcm_linear_scores_backward(f, w, type, k, 0, 1, k, 1, n, v, k, c, bias, btype, given, gtype, 1, 0, 0, slots, gl, None, z, p, p, p,
                                              work, size, None)

    def eight(f=p, w=p, fs=p, ws=p, n=4, v=1, k=8, c=10, bias=None, btype=0, given=None, gtype=5, slots=0, logp=None, work=p, size=much):
        return lib.pcm_linear_scores8(f, fs, w, ws, n, v, k, c, bias, btype, given, gtype, 1, 0, 0, slots, logp, None, work, size, None)

    def code(x=p, type=0, n=4, v=1, k=8, codes=p, scales=p):
        return lib.pcm_rows8(x, type, k, 0, 1, n, v, k, codes, scales, None)

    def product(a=p, sa=p, n=4, b=p, sb=p, c=10, k=8, bias=None, btype=0, out=p, type=0, pitch=10, work=p, size=much):
        return lib.pcm_product8(a, sa, n, b, sb, c, k, bias, btype, out, type, pitch, work, size, None)

    for f in (scores, back):
        assert f(type=3) == -1 and f(type=-1) == -1 and b"type" in lib.pcm_last_error()
    for f in (scores, back, eight):
        assert f(btype=3) == -1 and f(btype=-1) == -1
        assert f(n=-1) == -2 and f(v=0) == -2 and f(k=0) == -2 and f(c=0) == -2
        assert f(n=(1 << 22) + 1) == -3 and f(n=1 << 21, v=3) == -3 and f(c=(1 << 30) + 1) == -3 and f(k=(1 << 20) + 1) == -3
        assert f(slots=65, given=p) == -3 and f(slots=-1) == -3 and f(slots=1) == -1 and f(slots=1, given=p, gtype=0) == -1
        assert f(f=None) == -1 and f(w=None) == -1 and f(slots=1, given=p) == -1
        assert f(work=None) == -1 and b"workspace" in lib.pcm_last_error() and f(size=0) == -1
        assert f(work=p + 8) == -1 and b"aligned" in lib.pcm_last_error()
    assert back(z=None) == -1
    assert scores(n=0) == 0 and eight(n=0) == 0                         # nothing to do: nothing is touched
    assert eight(k=131072) == -3 and eight(fs=None) == -1 and eight(ws=None) == -1 and eight(f=p + 8) == -1 and eight(w=p + 1) == -1
    assert code(type=3) == -1 and code(n=-1) == -2 and code(v=0) == -2 and code(k=0) == -2 and code(k=131072) == -3 and code(n=1 << 31) == -3
    assert code(n=1 << 30, v=2) == -3 and code(x=None) == -1 and code(codes=None) == -1 and code(scales=None) == -1 and code(codes=p + 8) == -1
    assert code(n=0) == 0 and product(n=0) == 0
    assert product(type=3) == -1 and product(bias=p, btype=3) == -1 and product(n=-1) == -2 and product(c=0) == -2 and product(k=0) == -2
    assert product(pitch=9) == -2 and product(k=131072) == -3 and product(n=1 << 31) == -3 and product(c=1 << 31, pitch=1 << 31) == -3
    for missing in ("a", "sa", "b", "sb", "out"):
        assert product(**{missing: None}) == -1
    assert product(a=p + 8) == -1 and product(b=p + 4) == -1


def test_workspaces_follow_the_arguments():
    from pcmi355._lib import lib
    p = 1 << 20

    def scores(type=1, k=64, at=p, stride=None, inner=1, n=100, c=1000):
        return lib.pcm_linear_scores_workspace(at, p, type, stride or k, 0, inner, k, 1, n, 1, k, c)

    least = scores()
    assert least > 0 and scores(k=128) == least                          # nothing laid out
    assert scores(type=0, k=65, inner=2, stride=130, at=p + 4) == scores(type=0)   # float is read whatever its strides
    for other in (scores(k=65), scores(at=p + 2), scores(stride=65), scores(inner=2, stride=128)):
        assert other > least
    assert scores(n=0) == 0 and scores(k=0) == 0 and scores(c=0) == 0 and scores(n=(1 << 22) + 1) == 0
    back = lambda of, n=100: lib.pcm_linear_scores_backward_workspace(p, p, 1, 64, 0, 1, 64, 1, n, 1, 64, 1000, of)
    assert 0 < back(4) < back(1) < back(7) and back(2) < back(7) and back(7, 0) == 0
    assert lib.pcm_product8_workspace(0, 10, 100) == 0 and lib.pcm_product8_workspace(10, 10, 131072) == 0
    assert lib.pcm_linear_scores8_workspace(0, 1, 10, 10) == 0 and lib.pcm_linear_scores8_workspace(5, 1, 10, 10) > 0


@pytest.mark.parametrize("type_", [0, 1, 2])
def test_a_gradient_of_no_rows_needs_nothing(type_):
    from pcmi355._lib import lib
    p = 4096                                                             # (nothing is read there)
    assert lib.pcm_linear_scores_backward_workspace(p, p, type_, 8, 0, 1, 8, 1, 0, 1, 8, 10, 7) == 0
    for at in (p, None):
        assert lib.pcm_linear_scores_backward(at, at, type_, 8, 0, 1, 8, 1, 0, 1, 8, 10, None, 0, None, 5, 0, 0, 0, 0, None, None, None, None, None,
                                              None, None, 0, None) == 0
    assert lib.pcm_linear_scores_backward(p, p, type_, 8, 0, 1, 8, 1, 0, 1, 0, 10, None, 0, None, 5, 0, 0, 0, 0, None, None, None, None, None, None,
                                          None, 0, None) == -2           # (what is refused with rows is refused without)


@pytest.mark.parametrize("type_", [0, 1, 2])
def test_the_gradients_workspace_has_a_bound(type_):
    """5 GiB beside the features turned and summed, whatever the number of categories, of rows and of entries"""
    from pcmi355._lib import lib
    p = 1 << 20
    for n in (1, 2, 40, 64, 65, 1000, 1023, 1024, 4096, 16500, 65536, 65537, 100000, 1 << 18, 1 << 20, 1 << 22):
        for k in (1, 3, 64, 65, 768, 4096, 8192, 16384, 100000, 1 << 20):
            for c in (2, 300, 4096, 4097, 50304, 140000, 1 << 20, 1 << 24, 1 << 30):
                for inner in (1, 2):                                     # (2: both are laid out)
                    for v in (1, 32) if n % 32 == 0 else (1,):
                        need = lib.pcm_linear_scores_backward_workspace(p, p, type_, k * inner * v, k * inner, inner, k * inner, inner, n // v, v, k, c, 7)
                        assert 0 < need <= (5 << 30) + n * (8 * (k + 63) + 264) + 4 * c, (n, k, c, inner, v, need)

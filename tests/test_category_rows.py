"""Rows of category scores on the CPU: the reference against closed forms and differences, and what the entry points refuse."""
import ctypes

import numpy as np
import pytest
import torch

import category_reference as R


def _rows(seed, n, C, spread=3.0):
    return np.random.default_rng(seed).normal(size=(n, C)) * spread


def test_reference_statistics():
    from scipy.special import logsumexp, softmax
    from scipy.stats import entropy
    x = _rows(1, 5, 37)
    z, h = R.statistics(x)
    np.testing.assert_allclose(z, logsumexp(x, 1), rtol=1e-13)
    np.testing.assert_allclose(h, entropy(softmax(x, 1), axis=1), rtol=1e-12)
    x[1, 3:] = -np.inf
    x[2] = -np.inf
    x[3, 5] = np.nan
    x[4, 5] = np.inf
    z, h = R.statistics(x)
    assert z[2] == -np.inf and np.isnan(h[2]) and np.isnan(z[3:]).all() and np.isnan(h[3:]).all() and np.isfinite(z[1])
    i, lp = R.likeliest(np.array([[1.0, 2.0, 2.0, -np.inf]]), 5)
    assert i.tolist() == [[1, 2, 0, -1, -1]] and lp[0, 3] == -np.inf


def test_reference_gradient_is_the_derivative():
    n, C = 3, 11
    x = _rows(2, n, C)
    rng = np.random.default_rng(3)
    g = rng.integers(-1, C, (n, 4))
    g[0] = [2, 2, -1, 5]
    w, gh = rng.normal(size=(n, 4)), rng.normal(size=n)

    def loss(y):
        z, h = R.statistics(y)
        return (R.logp_of(y, g) * w).sum() + (gh * h).sum()

    z, h = R.statistics(x)
    got = R.gradient(x, z, h, [(g, w)], gh)[0]
    for r in range(n):
        for c in range(C):
            y = x.copy()
            y[r, c] += 1e-6
            u = x.copy()
            u[r, c] -= 1e-6
            # a central difference of a function with third derivatives of order one: 1e-12, and 1e-16 / 1e-6 of rounding
            assert abs((loss(y) - loss(u)) / 2e-6 - got[r, c]) < 1e-8


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_reference_rounding_is_off_by_half_a_step(dtype):
    x = torch.from_numpy(_rows(4, 6, 150, 9.0)).to(getattr(torch, dtype)).double().numpy()
    x[1, 7] = -np.inf
    x[2, 70] = R.LOWEST[dtype]
    x[3, 130] = np.nan
    x[4] = -5000.0 + np.arange(150) / 128.0
    y = R.rounded(x, dtype)
    assert y[1, 7] == -np.inf and y[2, 70] == -np.inf and np.isnan(y[3, 128:]).all() and np.isfinite(y[3, :128]).all()
    for s in range(0, 150, 64):
        b, c = x[[0, 4, 5], s:s + 64], y[[0, 4, 5], s:s + 64]
        span, size = b.max(1) - b.min(1), np.abs(b).max(1)
        assert (np.abs(c - b).max(1) <= np.maximum(span / 126.5, size * 2.0 ** -12) / 2).all()


def test_reference_rounding_follows_the_level():
    """Half a step is at most 1/253 of the range of 64 neighbours or 2^-14 of the largest |x|, whichever is more; far from zero it is
    the latter, and the former alone would not hold"""
    for level in (0.0, -600.0, -3000.0, -8000.0, -20000.0):
        x = (level + _rows(6, 500, 64, 2.5)).astype(np.float32).astype(np.float64)
        off, span, size = np.abs(R.rounded(x, "float32") - x).max(1), np.ptp(x, axis=1), np.abs(x).max(1)
        assert (off <= np.maximum(span / 253, size / 2.0 ** 14)).all()
        assert (off > span / 253).any() == (level <= -3000.0)
        shifted = (x - R.statistics(x)[0][:, None]).astype(np.float32).astype(np.float64)
        assert (np.abs(R.rounded(shifted, "float32") - shifted).max(1) <= np.ptp(shifted, axis=1) / 253).all()


# ---- refusals -----------------------------------------------------------------------------------------------------

def test_python_refuses_what_it_cannot_do():
    import pcmi355 as P
    x = torch.zeros((4, 10))
    for bad, what in ((torch.zeros(10), "tensor"), (torch.zeros((4, 10), dtype=torch.float64), "float"), (torch.zeros((4, 0)), "category"),
                      (np.zeros((4, 10)), "tensor")):
        for f in (P.category_scores, P.checkpoint_rows):
            with pytest.raises(ValueError, match=what):
                f(bad)
    for given in (torch.zeros(4), torch.zeros(3, dtype=torch.int64), torch.zeros((4, 65), dtype=torch.int32),
                  torch.zeros((4, 2, 2), dtype=torch.int32), [0, 1, 2, 3]):
        with pytest.raises(ValueError, match="given"):
            P.category_scores(x, given)
    for top in (-1, 65):
        with pytest.raises(ValueError, match="top"):
            P.category_scores(x, top=top)
    for f in (P.category_scores, P.checkpoint_rows):
        with pytest.raises(ValueError, match="GPU"):
            f(x)
    z, g, w = torch.zeros(4), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    back = P.category_scores_backward
    for call in (lambda: back(x, z, g), lambda: back(x, z, grad_logp=w), lambda: back(x, z, top=g), lambda: back(x, z, grad_entropy=w),
                 lambda: back(x, torch.zeros(3), g, grad_logp=w), lambda: back(x, z, g, grad_logp=torch.zeros(5)),
                 lambda: back(x, z, top=torch.zeros((4, 2)), grad_top=torch.zeros((4, 2))),
                 lambda: back(x, z, top=torch.zeros((4, 2), dtype=torch.int32), grad_top=torch.zeros((4, 3))),
                 lambda: back(x, z, entropy=torch.zeros(2), grad_entropy=w),
                 lambda: P.restore_rows(x)):
        with pytest.raises(ValueError):
            call()
    kept = P.Checkpoint8(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.int32), (4, 10), torch.bfloat16)
    assert kept.nbytes == 4 * 16 + 16
    with pytest.raises(ValueError, match="come back"):
        kept.restore(torch.float16)
    with pytest.raises(ValueError, match="out must be"):
        kept.restore(out=torch.zeros((4, 9), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="GPU"):
        kept.restore()


def test_sizes_beyond_32_bits_are_refused():
    """Sizes reach the library in 32 bits: 2^32 + 5 categories are not 5, 2^32 + 1 rows not one"""
    import pcmi355 as P
    one = torch.zeros(1, dtype=torch.float16)
    for shape in ((1, (1 << 32) + 5), (2, 3, (1 << 31) + 7), (1, (1 << 30) + 1), ((1 << 32) + 1, 4), (1, (1 << 32) + 1, 4), (1 << 16, 1 << 15, 2)):
        x = one.expand(shape)
        for f in (P.category_scores, P.checkpoint_rows, lambda y: P.category_scores_backward(y, one)):
            with pytest.raises(ValueError, match="at most 2.30 categories"):
                f(x)
        rows = shape[0] if len(shape) == 2 else shape[0] * shape[1]
        codes = torch.zeros(1, dtype=torch.uint8, device="meta").expand(rows, -(-shape[-1] // 16) * 16)
        with pytest.raises(ValueError, match="at most 2.30 categories"):
            P.Checkpoint8(codes, torch.zeros(1, dtype=torch.int32, device="meta").expand(rows, -(-shape[-1] // 64)), shape, torch.float16)
    with pytest.raises(ValueError, match="GPU"):                        # the largest that the library takes
        P.checkpoint_rows(one.expand(1, 1 << 30))


def test_a_checkpoint_is_of_its_shape():
    import pcmi355 as P
    codes, scales = torch.zeros((6, 80), dtype=torch.uint8), torch.zeros((6, 2), dtype=torch.int32)
    P.Checkpoint8(codes, scales, (2, 3, 70), torch.float32)
    for c, s, shape, dtype in ((codes, scales, (6, 64), torch.float32), (codes, scales, (5, 70), torch.float32), (codes.int(), scales, (6, 70), torch.float32),
                               (codes, scales.long(), (6, 70), torch.float32), (codes, scales[:, :1], (6, 70), torch.float32),
                               (codes[:, :79], scales, (6, 70), torch.float32), (torch.zeros((80, 6), dtype=torch.uint8).t(), scales, (6, 70), torch.float32),
                               (codes, torch.zeros((2, 6), dtype=torch.int32).t(), (6, 70), torch.float32), (codes, scales, (6, 70), torch.float64),
                               (codes, scales.to("meta"), (6, 70), torch.float32), (codes, scales, (420,), torch.float32)):
        with pytest.raises(ValueError):
            P.Checkpoint8(c, s, shape, dtype)


def test_workspaces_are_asked_for_and_checked():
    from pcmi355._lib import lib
    big = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(big) + 15) & ~15
    need = lib.pcm_category_scores_workspace(1, 1, 131072, 8)
    assert need > 0 and lib.pcm_category_scores_workspace(100000, 1, 131072, 8) == 0
    call = lambda work, size: lib.pcm_category_scores(p, 0, 131072, 0, 1, 1, 1, 131072, None, 3, 0, 0, 0, 0, 8, None, None, None, p, p, None, None,
                                                      work, size, None)
    assert call(None, need) == -1 and call(p, need - 1) == -1 and b"workspace" in lib.pcm_last_error()
    assert call(p + 8, need) == -1 and b"aligned" in lib.pcm_last_error()
    for n, v, c in ((1, 1, (1 << 31) - 1), (1 << 40, 1, 10), (1 << 30, 4, 10)):
        assert lib.pcm_category_scores_workspace(n, v, c, 8) == 0      # such rows are refused


def test_where_results_may_go():
    from pcmi355 import category_rows as M
    t = torch.zeros((6, 8))
    assert M._no_overlap(t) and M._no_overlap(t.t()) and M._no_overlap(t[:, ::2]) and M._no_overlap(t[2:5, 3:])
    assert M._no_overlap(torch.zeros((2, 3, 4)).permute(2, 0, 1)) and M._no_overlap(t[:1].expand(1, 8))
    assert not M._no_overlap(t[:1].expand(6, 8)) and not M._no_overlap(t.as_strided((4, 8), (1, 1)))
    assert not M._no_overlap(t.as_strided((3, 3), (2, 1)))
    assert M._apart(t[:3], t[3:]) and not M._apart(t[:4], t[3:])
    assert M._apart(t[:3], None, t[3:4], t[:0], t[4:]) and not M._apart(t[:3], None, t[4:], t[2]) and M._apart(t[:0], t)


def test_results_may_lie_between_what_is_read():
    """Tensors whose extents cross are refused only where an element may be shared: counted byte by byte"""
    from pcmi355 import category_rows as M
    t = torch.zeros((6, 20))
    for a, b in ((t[:, :10], t[:, 10:]), (t[:, ::2], t[:, 1::2]), (t[:, 4:9], t[:, 12:13]), (t[::2], t[1::2]), (t[:, :10].t(), t[:, 10:]),
                 (t[:, 3], t[:, 5:9]), (t[:, :18:2], t[:, 1:18:2]), (t.view(-1)[:114].view(6, 19)[:, :18:2], t.view(-1)[:114].view(6, 19)[:, 1:18:2]),
                 (t.view(6, 4, 5)[:, :2], t.view(6, 4, 5)[:, 2:]), (t.view(6, 4, 5)[..., :3], t.view(6, 4, 5)[..., 3:])):
        assert M._apart(a, b) and M._apart(b, a)
    for a, b in ((t[:, :10], t[:, 9:]), (t[:, ::2], t[:, ::2]), (t[:, ::2], t[:, 1::3]), (t[::2], t[::3]), (t[:, :10].t(), t), (t[:, 3], t[:, 3:9]),
                 (t.view(6, 4, 5)[:, :2], t.view(6, 4, 5)[:, 1]), (t.view(6, 4, 5)[..., :3], t.view(6, 4, 5)[:, 2, 2:])):
        assert not M._apart(a, b) and not M._apart(b, a)
    # any two views of a buffer: never called apart where a byte is shared
    rng = np.random.default_rng(1)
    buf = torch.zeros(400, dtype=torch.uint8)

    def view():
        dtype = (torch.uint8, torch.float16, torch.float32)[rng.integers(3)]
        whole = buf.view(dtype)
        size, stride = rng.integers(1, 5, 3).tolist(), rng.integers(0, 12, 3).tolist()
        reach = sum(s * (n - 1) for s, n in zip(stride, size))
        return whole.as_strided(size, stride, int(rng.integers(0, max(1, len(whole) - reach)))) if reach < len(whole) else whole[:3]

    def bytes_of(v):
        at = torch.zeros(v.shape, dtype=torch.int64) + (v.data_ptr() - buf.data_ptr())
        for d, (s, n) in enumerate(zip(v.stride(), v.shape)):
            at = at + (torch.arange(n) * s * v.element_size()).view([-1 if i == d else 1 for i in range(v.dim())])
        return {int(x) + k for x in at.reshape(-1) for k in range(v.element_size())}

    between = 0
    for _ in range(3000):
        a, b = view(), view()
        shared = bool(bytes_of(a) & bytes_of(b))
        assert not (shared and M._apart(a, b))
        between += M._apart(a, b) and not (M._extent(a)[1] <= M._extent(b)[0] or M._extent(b)[1] <= M._extent(a)[0])
    assert between                                    # (some of them lie between each other)


def test_entry_points_refuse_without_a_gpu():
    from pcmi355._lib import lib
    big = ctypes.create_string_buffer(64)
    p = ctypes.addressof(big)

    def scores(x=p, type=0, n=4, v=1, c=10, given=None, gtype=3, slots=0, top=0, logp=None, best=None, codes=None, scales=None, work=None,
               size=0):
        return lib.pcm_category_scores(x, type, c, 0, 1, n, v, c, given, gtype, 1, 0, 0, slots, top, logp, None, None, best, best, codes,
                                       scales, work, size, None)

    def back(x=p, type=0, n=4, v=1, c=10, codes=None, scales=None, given=None, gtype=3, slots=0, gl=None, top=0, best=None, gt=None, z=p,
             h=None, gh=None, out=p):
        return lib.pcm_category_scores_backward(x, type, c, 0, 1, n, v, c, codes, scales, given, gtype, 1, 0, 0, slots, gl, top, best, gt, z,
                                                h, gh, out, c, 0, 1, None)

    def keep(x=p, type=0, n=4, v=1, c=10, codes=p, scales=p):
        return lib.pcm_checkpoint_rows(x, type, c, 0, 1, n, v, c, codes, scales, None)

    def restore(codes=p, scales=p, n=4, v=1, c=10, out=p, type=0):
        return lib.pcm_restore_rows(codes, scales, n, v, c, out, type, c, 0, 1, None)

    for f in (scores, back, keep, restore):
        assert f(type=3) == -1 and f(type=-1) == -1 and b"type" in lib.pcm_last_error()
        assert f(c=0) == -2 and f(v=0) == -2 and f(n=-1) == -2
        assert f(n=1 << 40) == -3 and f(n=1 << 30, v=4) == -3 and f(c=(1 << 30) + 1) == -3
        assert f(n=0) == 0                                              # nothing to do: nothing is touched
    for f in (scores, back):
        assert f(slots=65, given=p) == -3 and f(top=65) == -3 and f(slots=-1) == -3 and f(top=-1) == -3
        assert f(slots=1) == -1                                         # no categories
        assert f(slots=1, given=p, gtype=0) == -1
        assert f(codes=p) == -1 and f(scales=p) == -1
    assert scores(x=None) == -1 and scores(slots=1, given=p) == -1 and scores(top=2) == -1
    assert back(x=None) == -1 and back(codes=p, scales=p) == -1         # neither scores nor checkpoint, or both
    assert back(slots=1, given=p) == -1 and back(top=1) == -1 and back(gh=p) == -1 and back(z=None) == -1 and back(out=None) == -1
    assert keep(x=None) == -1 and keep(codes=None) == -1 and restore(out=None) == -1 and restore(scales=None) == -1
    assert lib.pcm_category_scores_workspace(0, 1, 10, 3) == 0 and lib.pcm_category_scores_workspace(-1, 0, 0, 99) == 0

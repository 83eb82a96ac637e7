"""Scores that are products of features and weights, their gradients and 8-bit rows by their definitions in 64 bits, with bounds on how far
32-bit sums and one rounding of dx may lie from them.  Bounds count roundings: a sum of K products, however it is ordered and whether its
steps round or cut off, is off by K 2^-23 of the sum of the products' sizes; float taken as three bfloat16 leaves out 2^-24 of them
at most and sums six times as many."""
import torch

# (rows, length, categories) at which products of 16-bit types go by tiles of 256 x 256, and which do: scores and dx, the features' gradient and the
# weights' (with pieces of the categories: of how many); fewer than 1024 rows have dx in two parts
WIDE = [((3501, 800, 4001), ("scores",), 1), ((3501, 3590, 4001), ("scores", "features", "weight"), 1), ((16500, 770, 9100), ("scores", "features"), 3),
        ((1001, 12500, 800), ("features", "weight"), 1), ((1001, 800, 12500), ("scores",), 1)]
WIDE8 = [(3601, 1601, 4001), (3584, 1664, 4096)]      # of 8-bit rows

LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def masked(bias):
    return bias <= torch.finfo(bias.dtype).min / 2


def product(a, b):
    """a @ b.T in 64 bits"""
    return torch.mm(a.double(), b.double().t().contiguous())


def sum_bound(sizes, k, dtype):
    """of a 32-bit sum of k products whose sizes add up to `sizes`"""
    return sizes * ((6 * k if dtype == torch.float32 else k) + 8) * 2.0 ** -23


class Scores:
    """x [rows, cats], log_sum [rows] and their bounds"""

    def __init__(self, f, w, bias=None):
        k = f.shape[1]
        self.x = product(f, w)
        sizes = product(f.abs(), w.abs())
        if bias is not None:
            self.x = self.x + bias.double()
            sizes = sizes + bias.double().abs().nan_to_num(posinf=0.0, neginf=0.0)
        self.off = sum_bound(sizes, k, f.dtype)
        if bias is not None:
            self.x[:, masked(bias)] = -float("inf")
            self.off[:, masked(bias)] = 0.0
        self.log_sum = torch.logsumexp(self.x, 1)
        # a factor of exp(off) in every term; then at most 64 terms one after the other and a tree, exponentials of 2^-22, and Z itself
        most = self.off.max(1).values
        self.log_sum_off = most + 2.0 ** -24 * (160 + 4 * self.log_sum.abs().nan_to_num(posinf=0.0))

    def logp(self, g):
        """(values, bounds) for g [rows, slots]"""
        C = self.x.shape[1]
        at = g.clamp(0, C - 1)
        v = self.x.gather(1, at)
        z = self.log_sum[:, None]
        lp = torch.where(z == -float("inf"), z, v - z)
        lp = torch.where(g < 0, 0.0, torch.where(g >= C, float("nan"), lp))
        off = self.off.gather(1, at) + self.log_sum_off[:, None] + 2.0 ** -22 * (v.abs() + z.abs()).nan_to_num(posinf=0.0)
        return lp, off


def dx_of(s, g=None, gl=None, gz=None):
    """dx [rows, cats] from its formula, rows without derivatives and without categories zero, with the rows' size sum |gl| + |weight of p|"""
    n, C = s.x.shape
    total = torch.zeros(n, dtype=torch.float64, device=s.x.device)
    size = torch.zeros_like(total)
    dx = torch.zeros_like(s.x)
    past = torch.zeros(n, dtype=torch.bool, device=s.x.device)
    if g is not None:
        by = torch.where(g < 0, 0.0, gl.double())
        total, size, past = by.sum(1), by.abs().sum(1), (g >= C).any(1)
        for j in range(g.shape[1]):
            dx.scatter_add_(1, g[:, j:j + 1].clamp(0, C - 1), by[:, j:j + 1])
    if gz is not None:
        total = total - gz.double()
    size = size + total.abs()
    p = (s.x - s.log_sum[:, None]).exp()
    dx = dx - total[:, None] * p
    dx[past] = float("nan")
    dead = (size == 0) & ~past | (s.log_sum == -float("inf"))
    dx[dead] = 0.0
    return dx, torch.where(dead, 0.0, size), p


def gradients(f, w, bias, s, g=None, gl=None, gz=None):
    """{name: (values, bounds)}"""
    dtype, u = f.dtype, half_step(f.dtype)
    dx, size, p = dx_of(s, g, gl, gz)
    dead = size == 0
    # p: a factor of exp(off of x and Z); sums of up to 64 derivatives; then dx in three parts or rounded once, of half no finer than 2^-25
    # beside 2^15, which stands for 4 times the row's size at most
    offp = p * (torch.expm1(s.off.nan_to_num(nan=0.0) + s.log_sum_off[:, None].nan_to_num(nan=0.0)) + 2.0 ** -21)
    offx = size[:, None] * (offp + 2.0 ** -17 * p)
    offx = offx + (u if dtype != torch.float32 else 2.0 ** -24) * (dx.abs() + offx) + size[:, None] * 2.0 ** (-38 if dtype == torch.float16 else -60)
    offx[dead] = 0.0
    fd, wd = f.double().clone(), w.double().clone()
    fd[dead] = 0.0
    if bias is not None:
        wd[masked(bias)] = 0.0
    out = {}
    v = product(dx, wd.t().contiguous())
    off = product(offx, wd.abs().t().contiguous()) + sum_bound(product(dx.abs(), wd.abs().t().contiguous()), dx.shape[1], dtype)
    out["features"] = v, off * 1.01 + u * v.abs() + LEAST[dtype]
    v = product(dx.t().contiguous(), fd.t().contiguous())
    off = product(offx.t().contiguous(), fd.abs().t().contiguous()) + sum_bound(product(dx.abs().t().contiguous(), fd.abs().t().contiguous()), dx.shape[0], dtype)
    if dtype == torch.float16:      # features scaled by powers of two down to 2^-25 of the row of the largest derivatives
        off = off + 2.0 ** -22 * size.max() * (dx.abs() / size[:, None]).nan_to_num(nan=0.0).sum(0)[:, None]
    out["weight"] = v, off * 1.01 + u * v.abs() + LEAST[dtype]
    if bias is not None:
        v = dx.sum(0)
        off = offx.sum(0) + (dx.shape[0] + 8) * 2.0 ** -24 * dx.abs().sum(0)
        out["bias"] = v, off * 1.01 + half_step(bias.dtype) * v.abs() + LEAST[bias.dtype]
    return out


def codes_of(x):
    """8-bit codes and scales of rows, quotient and product rounded to 32 bits as the format says"""
    y = x.double()
    a = y.abs().amax(-1, keepdim=True)
    bad, none = ~(a < float("inf")), a < 2.0 ** -119
    by = torch.where(bad | none, 0.0, (127.0 / a).float().double())
    code = torch.round((y * by).float()).nan_to_num(nan=0.0)
    code = torch.where(bad, torch.zeros_like(code), code)
    return code.to(torch.int8), torch.where(bad, float("nan"), torch.where(none, 0.0, (a / 127.0).float())).float().squeeze(-1)


def within(got, want, bound, what=""):
    """got as near to want as the bound says; NaN and infinities where want has them"""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    bad = torch.isnan(want)
    assert torch.equal(torch.isnan(got), bad), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities"
    ok = ~bad & ~inf
    past = ((got - want).abs() - bound)[ok]
    assert not past.numel() or float(past.max()) <= 0, \
        f"{what}: off by {float((got - want).abs()[ok][past.argmax()])}, allowed {float(bound.expand_as(want)[ok][past.argmax()])}"

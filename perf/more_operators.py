"""The operators between features and category scores, as cases that can be timed and compared: log-probabilities of given
categories under scores that are products of features and weights, without keeping the scores; their gradient with respect to
features, weights and bias; matrix products in 8-bit integers with a scale for each row of both factors, and log-probabilities
from such rows.

Where `own` is false `run` computes them in elementary torch operations; where it is true through the package's public
entry points.  `exact` has the definitions once more, in 64 bits and a few rows at a time.

Definitions, for features f[r] and weights w[c] of n entries each, and a bias b[c] (0 where there is none):
  scores           x[r, c] = sum_k f[r, k] w[c, k] + b[c];  -inf where b[c] is -inf, whatever the product
  log-sum          Z[r] = log sum_c exp x[r, c]
  log-probability  x[r, g] - Z[r] of a given category g; 0 for g < 0 (not observed)
  gradient, of a loss with the derivatives gl[r, j] by the log-probabilities of g[r, j] and gz[r] by the log-sums
                   dx[r, c] = sum_j gl[r, j] [c = g[r, j]] - (sum_j gl[r, j] - gz[r]) p[r, c],  p = exp(x - Z), slots with
                   g < 0 left out of all sums;  features: dx w;  weights: dx^T f;  bias: sum_r dx
  8-bit rows       code = rint(x * (127 / a)), a the row's largest |x|, quotient and product rounded to 32 bits; scale a / 127;
                   a row of zeros has codes and scale 0
  8-bit product    y[r, c] = (sum_k codes[r, k] codes[c, k]) scale[r] scale[c] + b[c], the sum in whole numbers
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
# operations of a drawn case at most, by kind: those of the largest listed case of that kind, f32 an eighth of it
MOST = {"score": 8.8e12, "step": 6.7e12, "score8": 2.2e12, "product": 1.1e12}


# ---- cases ------------------------------------------------------------------------------------------------------

def _case(kind, rows, n, c, dtype, v=0, given=1, bias=False, masked=0.0, log_sum=False, name=None):
    case = dict(kind=kind, rows=rows, v=v, n=n, c=c, dtype=dtype, given=given, bias=bias, masked=masked, log_sum=log_sum)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one served request: how likely the token was that it was answered with
        _case("score", 1, 4096, 131072, "bf16", name="score_token"),
        # the live hypotheses of a search over an odd vocabulary, some of its entries forbidden; features of odd width
        _case("score", 48, 1001, 50021, "f16", bias=True, masked=0.1, name="score_beam"),
        # 64 patches of each of 512 images scored against their cluster ids: which soft evidence a top-level circuit gets
        _case("score", 512, 768, 128, "f32", v=64, bias=True, name="score_patches"),
        # the largest: a long batch's tokens over a large vocabulary
        _case("score", 8192, 4096, 131072, "bf16", name="score_vocabulary"),
        # a few rows of odd sizes
        _case("step", 37, 509, 1009, "f32", bias=True, given=3, name="step_few"),
        # a network that is taught cluster ids: a training step's loss and gradients over the patches of 512 images
        _case("step", 512, 768, 128, "f16", v=64, bias=True, name="step_patches"),
        # a student taught the 16 alternatives that its teacher offers, in 32 bits
        _case("step", 2048, 1024, 32003, "f32", given=16, name="step_teacher"),
        # a training step over a vocabulary, with a term that holds the log-sums near 0
        _case("step", 4096, 4096, 50304, "bf16", log_sum=True, name="step_vocabulary"),
        # one token through a layer held in 8 bits
        _case("product", 1, 4096, 16384, "bf16", name="product_token"),
        # some hypotheses, odd sizes
        _case("product", 48, 1001, 50021, "f16", bias=True, name="product_beam"),
        # a batch's tokens through a layer held in 8 bits
        _case("product", 8192, 4096, 16384, "bf16", name="product_batch"),
        # evaluation: log-probabilities of a text's tokens under a model held in 8 bits
        _case("score8", 2048, 4096, 131072, "bf16", name="score8_vocabulary"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("score", "step", "step", "product", "score8"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    n = _between(rng, 16, 8192)
    if rng.random() < 0.5:
        n = -(-n // 64) * 64
    c = _between(rng, 2, 131072)
    most = MOST[kind] / (8.0 if dtype == "f32" and kind in ("score", "step") else 1.0) / (8.0 if kind == "step" else 2.0)
    top = max(1, int(min(8192 if kind == "step" else 32768, most / (n * c), 2**30 / c)))
    rows, v = _between(rng, 1, top), 0
    if rows >= 128 and rng.random() < 0.3:
        v = _between(rng, 2, 64)
        rows //= v
    given = rng.choice((1, 1, 1, 2, 16))
    return _case(kind, rows, n, c, dtype, v=v, given=given, bias=rng.random() < 0.5, masked=rng.choice((0.0, 0.0, 0.1)),
                 log_sum=kind == "step" and rng.random() < 0.4)


# ---- inputs -----------------------------------------------------------------------------------------------------

def _rows(case):
    return (case["rows"], case["v"]) if case["v"] else (case["rows"],)


def prepare(case, seed, keep_weight=False):
    """Features as a normalised last layer gives them, weights for scores of standard deviation 2, a bias that falls with the
    category's rank, categories of which some are not observed and, in a batch of some length, the last rows not at all"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, n, c, dtype = _rows(case), case["n"], case["c"], TYPES[case["dtype"]]
    normal = lambda *shape: torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    state = dict(case=case, features=normal(*rows, n), weight=normal(c, n).mul_(2.0 / math.sqrt(n)), bias=None)
    if case["bias"]:
        rank = torch.randperm(c, device="cuda", generator=gen)
        b = -0.5 * torch.log(rank + 1.0)
        if case["masked"] and case["kind"] != "product":
            off = torch.rand(c, device="cuda", generator=gen) < case["masked"]
            off[int(torch.randint(c, (1,), device="cuda", generator=gen))] = False
            b.masked_fill_(off, -math.inf)
        state["bias"] = b.to(dtype)
    if case["kind"] in ("product", "score8") and not keep_weight:      # the layer in 8 bits, laid out once
        if own:
            state["weight8"] = _package().rows8(state.pop("weight"))
        else:
            state["codes"], state["scales"] = _codes(state.pop("weight"))
    if case["kind"] == "product":
        return state
    shape = rows if case["given"] == 1 else (*rows, case["given"])
    g = torch.randint(c, shape, device="cuda", generator=gen)
    if state["bias"] is not None:                  # a forbidden category is not given
        g.masked_fill_((state["bias"] == -math.inf)[g], -1)
    g.masked_fill_(torch.rand(shape, device="cuda", generator=gen) < 0.02, -1)
    if rows[0] >= 32:
        g[rows[0] - rows[0] // 20:] = -1
    state["given"] = g.to(torch.int32) if case["given"] > 1 else g
    if case["kind"] == "step":
        # the derivative of a mean over rows; in f16, whose range is 6e-8 to 65504, of the loss scaled up
        each = min(16.0, 32768.0 / math.prod(rows)) if case["dtype"] == "f16" else 1.0 / math.prod(rows)
        state["grad_logp"] = -each * torch.rand(shape, device="cuda", generator=gen)
        if case["log_sum"]:
            state["grad_log_sum"] = 0.01 * each * torch.randn(rows, device="cuda", generator=gen)
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------

def _codes(x):
    """8-bit codes (int8) and scales of rows"""
    x = x.float()
    a = x.abs().amax(-1, keepdim=True)
    most = torch.full_like(a, 127.0)               # (a quotient by a number would be a product with its rounded reciprocal)
    inv = torch.where(a > 0, most / a, 0.0)
    return torch.round(x * inv).to(torch.int8), (a / most).squeeze(-1)


def _whole(a, b):
    """Product of rows of codes as whole numbers: pieces of 1024 entries are exact in 32-bit floats"""
    out = torch.zeros((a.shape[0], b.shape[0]), dtype=torch.int32, device=a.device)
    for s in range(0, a.shape[1], 1024):
        out += (a[:, s:s + 1024].float() @ b[:, s:s + 1024].float().t()).int()
    return out


def _add_bias(x, bias):
    if bias is None:
        return x
    b = bias.float()
    return (x + b).masked_fill_(b == -math.inf, -math.inf)


def _plain(state):
    case = state["case"]
    rows, c = _rows(case), case["c"]
    f = state["features"].reshape(-1, case["n"])
    if case["kind"] in ("product", "score8"):
        codes, scales = _codes(f)
        x = _whole(codes, state["codes"]).float() * scales.unsqueeze(-1) * state["scales"]
        if case["kind"] == "product":
            return _add_bias(x, state["bias"]).to(f.dtype).view(*rows, c)
        x = _add_bias(x, state["bias"])
    else:
        f, w = f.float(), state["weight"].float()
        x = _add_bias(f @ w.t(), state["bias"])
    m = x.amax(-1, keepdim=True)
    z = (x - m).exp_().sum(-1, keepdim=True).log_().add_(m)
    g = state["given"].reshape(x.shape[0], -1).long()
    seen = g >= 0
    g = g.clamp(min=0)
    out = dict(log_sum=z.view(rows), logp=torch.where(seen, x.gather(1, g) - z, 0.0).view(state["given"].shape))
    if case["kind"] == "step":
        gl = torch.where(seen, state["grad_logp"].reshape(g.shape), 0.0)
        total = gl.sum(-1, keepdim=True)
        if case["log_sum"]:
            total = total - state["grad_log_sum"].reshape(-1, 1)
        dx = x.sub_(z).exp_().mul_(-total).scatter_add_(1, g, gl)
        dtype = state["features"].dtype
        out["grad_features"] = (dx @ w).to(dtype).view(*rows, -1)
        out["grad_weight"] = (dx.t() @ f).to(dtype)
        if case["bias"]:
            out["grad_bias"] = dx.sum(0).to(dtype)
    return out


# ---- the package's own ------------------------------------------------------------------------------------------

def _package():
    where = os.path.join(os.getcwd(), "lvd-pg_amd")
    if where not in sys.path:
        sys.path.insert(0, where)
    import pcmi355
    return pcmi355


def _call(state):
    P, case, f, bias = _package(), state["case"], state["features"], state["bias"]
    if case["kind"] == "product":
        return P.product8(P.rows8(f), state["weight8"], bias=bias)
    if case["kind"] == "score8":
        s = P.linear_scores(P.rows8(f), state["weight8"], state["given"], bias=bias)
        return dict(log_sum=s.log_sum, logp=s.logp)
    w, given = state["weight"], state["given"]
    s = P.linear_scores(f, w, given, bias=bias)
    out = dict(log_sum=s.log_sum, logp=s.logp)
    if case["kind"] == "step":
        d = P.linear_scores_backward(f, w, s.log_sum, given, bias=bias, grad_logp=state["grad_logp"],
                                     grad_log_sum=state.get("grad_log_sum"))
        out["grad_features"], out["grad_weight"] = d.features, d.weight
        if bias is not None:
            out["grad_bias"] = d.bias
    return out


def run(state):
    if own:
        return _call(state)
    return _plain(state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _eight(x):
    """Rows as codes (whole numbers in 64 bits) and scales; quotient and product are rounded to 32 bits by their definition"""
    y = x.double()
    largest = y.abs().max(-1, keepdim=True).values
    step = (largest / 127).float().double()
    times = torch.where(largest > 0, (127 / largest).float().double(), 0.0)
    return torch.round((y * times).float()).double(), step


def exact(case, seed):
    state = prepare(case, seed, keep_weight=True)
    rows, n, c, kind = _rows(case), case["n"], case["c"], case["kind"]
    f = state["features"].reshape(-1, n)
    total = f.shape[0]
    if kind in ("product", "score8"):
        w, wide = _eight(state["weight"])
        f, high = _eight(f)
    else:
        w, wide, f, high = state["weight"].double(), None, f.double(), None
    bias = None if state["bias"] is None else state["bias"].double()
    chunk = max(1, (1 << 28) // c)
    found = dict(log_sum=[], logp=[], grad_features=[], y=[])
    dw = torch.zeros((c, n), dtype=torch.float64, device=f.device) if kind == "step" else None
    db = torch.zeros(c, dtype=torch.float64, device=f.device)
    for s in range(0, total, chunk):
        x = torch.mm(f[s:s + chunk], w.t())
        if high is not None:
            x = x * high[s:s + chunk] * wide.t()
        if bias is not None:
            x = torch.where(bias > -math.inf, x + bias, bias)
        if kind == "product":
            found["y"].append(x)
            continue
        z = torch.logsumexp(x, 1)
        found["log_sum"].append(z)
        x = x - z[:, None]
        g = state["given"].reshape(total, -1)[s:s + chunk].long()
        found["logp"].append(torch.where(g < 0, 0.0, x.gather(1, g.clamp(min=0))))
        if kind == "step":
            by = state["grad_logp"].reshape(total, -1)[s:s + chunk].double()
            weight_of_p = torch.zeros_like(z)
            if case["log_sum"]:
                weight_of_p += state["grad_log_sum"].reshape(-1)[s:s + chunk].double()
            dx = torch.zeros_like(x)
            for j in range(g.shape[1]):
                each = torch.where(g[:, j] < 0, 0.0, by[:, j])
                weight_of_p -= each
                dx.scatter_add_(1, g[:, j:j + 1].clamp(min=0), each[:, None])
            dx += weight_of_p[:, None] * x.exp()
            found["grad_features"].append(torch.mm(dx, w))
            dw += torch.mm(dx.t().contiguous(), f[s:s + chunk])
            db += dx.sum(0)
    if kind == "product":
        return torch.cat(found["y"]).view(*rows, c)
    out = dict(log_sum=torch.cat(found["log_sum"]).view(rows), logp=torch.cat(found["logp"]).view(state["given"].shape))
    if kind == "step":
        out["grad_features"] = torch.cat(found["grad_features"]).view(*rows, n)
        out["grad_weight"] = dw
        if case["bias"]:
            out["grad_bias"] = db
    return out


def work(case):
    """Bytes: features, weights and what comes with them in once, results out once; a step reads features and weights in both of its
    passes.  Operations: a product of features and weights, and for a step three more (the scores, which are not kept, once
    again, and one each for the gradients of features and weights); four an entry for the exponential sum, as many for dx."""
    rows, n, c, size = math.prod(_rows(case)), case["n"], case["c"], SIZE[case["dtype"]]
    pairs, bias = rows * c, c * size if case["bias"] else 0
    if case["kind"] == "product":
        return dict(bytes=rows * n * size + c * (n + 4) + bias + pairs * size, flops=2 * pairs * n)
    index = rows * case["given"] * (4 if case["given"] > 1 else 8)
    out = 4 * rows * (1 + case["given"])
    if case["kind"] == "score8":
        return dict(bytes=rows * n * size + c * (n + 4) + bias + index + out, flops=2 * pairs * n + 4 * pairs)
    factors = (rows + c) * n * size
    if case["kind"] == "score":
        return dict(bytes=factors + bias + index + out, flops=2 * pairs * n + 4 * pairs)
    return dict(bytes=3 * factors + 3 * bias + 2 * index + 3 * out, flops=8 * pairs * n + 8 * pairs)

"""The operators on rows of category scores, as cases that can be timed and compared: log-probabilities of given categories
with the row's entropy and its likeliest categories, their gradient with respect to the scores, checkpoints of rows in
8 bits, and the training step whose backward pass reads such a checkpoint.

Where `own` is false `run` computes them in elementary torch operations; where it is true through the package's public
entry points.  `exact` has the definitions once more, in 64 bits and a few rows at a time.

Definitions, for one row x[0..C) with Z = sum_c exp x[c]:
  log-probability of category g   x[g] - log Z; 0 for g < 0 (not observed), NaN for g >= C
  entropy                         -sum_c p[c] log p[c], p = exp(x - log Z), nothing added where p = 0
  likeliest categories            by falling x, equal ones by rising index; entries of -inf are never offered: index -1 and
                                  log-probability -inf stand where a row has no more categories
  a row of -inf alone             log Z = -inf, log-probability -inf, entropy 0, gradient 0
  a row with NaN or +inf          NaN in all of its numbers, no categories offered
  gradient, of a loss with the derivatives gl[j] by the given log-probabilities, gt[i] by the likeliest ones, gh by the entropy
                                  sum_j gl[j] ([c = g_j] - p[c]) + sum_i gt[i] ([c = top_i] - p[c]) - gh p[c] (log p[c] + H)
  8 bits                          per 64 neighbours of a row with largest and smallest entries M, m: a step of 2^e, the smallest
                                  power of two that covers M - m in 254 steps and M in 2^14; an entry stands for the nearest
                                  multiple of the step.  Entries at or below half of the type's lowest value are masked (-inf).
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MOST = {"score": 1 << 29, "gradient": 1 << 28, "checkpoint": 1 << 28, "step": 1 << 28}   # entries of a drawn case
BLOCK = 64


# ---- cases ------------------------------------------------------------------------------------------------------

def _case(kind, n, c, dtype, v=0, given=0, top=0, entropy=True, layout="rows", masked=0.0, name=None):
    case = dict(kind=kind, n=n, v=v, c=c, dtype=dtype, given=given, top=top, entropy=entropy, layout=layout, masked=masked)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one served request: the next token's row, the log-probability of the one that was taken and 20 alternatives
        _case("score", 1, 131072, "bf16", given=1, top=20, name="score_token"),
        # the live hypotheses of a search over an odd vocabulary, some of its entries forbidden
        _case("score", 48, 50021, "f16", given=1, top=5, entropy=False, masked=0.1, name="score_beam"),
        # cluster posteriors of a batch of 64-patch images straight from a forest's likelihoods (tree, head, example)
        _case("score", 512, 128, "f32", v=64, given=1, top=4, layout="heads", name="score_clusters"),
        # the soft evidence that a top-level circuit is trained on, scored against the patches' cluster ids
        _case("score", 8192, 128, "f32", v=64, given=1, top=4, name="score_patches"),
        # a student's log-probabilities of the 16 alternatives that its teacher offers, and its own 16
        _case("score", 2048, 32003, "f32", given=16, top=16, name="score_teacher"),
        # the largest: a long batch's tokens over a large vocabulary
        _case("score", 4096, 131072, "bf16", given=1, top=8, name="score_vocabulary"),
        # a loss on a few rows of odd length
        _case("gradient", 16, 1009, "f32", given=3, top=2, name="gradient_few"),
        # 28 x 28 images whose every pixel has 256 scores: likelihood with an entropy bonus
        _case("gradient", 512, 256, "f16", v=784, given=1, name="gradient_pixels"),
        # a variational model's parameter rows (100 rows of the 16 x 16 x 3 circuit), kept in 8 bits and read back
        _case("checkpoint", 100, 3342336, "f32", name="checkpoint_rows"),
        # activations of odd width
        _case("checkpoint", 333, 10007, "bf16", name="checkpoint_odd"),
        # a training step over pixels: scores and 8-bit checkpoint forward, gradient from the checkpoint backward
        _case("step", 64, 256, "f32", v=784, given=1, name="step_pixels"),
        # the same over a vocabulary
        _case("step", 4096, 50304, "bf16", given=1, entropy=False, name="step_vocabulary"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("score", "score", "gradient", "checkpoint", "step"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    most = MOST[kind] * 2 // SIZE[dtype]
    if kind == "checkpoint":
        c = _between(rng, 5, 1 << 22)
        return _case(kind, _between(rng, 1, max(1, min(1 << 18, most // c))), c, dtype, entropy=False)
    c = _between(rng, 2, 131072)
    # rows by the thousand where they are short, down to a few where they are long; never so few entries in all that a
    # pass is nothing but launches
    least = max(1, min(1 << 12, (1 << 16) // c))
    n, v, layout = _between(rng, least, max(least, min(1 << 19, most // c))), 0, "rows"
    if c <= 512 and n >= 64 and rng.random() < 0.6:
        v = _between(rng, 2, min(800, n // 16))
        n = n // v
        layout = rng.choice(("rows", "heads")) if dtype == "f32" else "rows"
    given = rng.choice((0, 1, 1, 1, 4, 16))
    top = min(c, rng.choice((0, 0, 1, 5, 8, 20)))
    if kind == "step":
        given, top = max(given, 1), 0
    if kind == "gradient" and given + top == 0:
        given = 1
    return _case(kind, n, c, dtype, v=v, given=given, top=top, entropy=rng.random() < 0.6, layout=layout,
                 masked=rng.choice((0.0, 0.0, 0.1, 0.9)))


# ---- inputs -----------------------------------------------------------------------------------------------------

def _rows(case):
    return (case["n"], case["v"]) if case["v"] else (case["n"],)


def _logits(case, gen):
    """Scores as a model gives them: a common level that falls with the category's rank, noise on top, and with `masked`
    that share of the categories at -inf and a few rows masked altogether (the padding of a batch)"""
    c, dtype = case["c"], TYPES[case["dtype"]]
    if case["layout"] == "heads":                # log-likelihoods of heads: (variable, category, example) in memory
        x = torch.empty((case["v"], c, case["n"]), dtype=dtype, device="cuda").normal_(generator=gen).mul_(6.0)
        x = x.add_(-600.0).permute(2, 0, 1)
    else:
        x = torch.empty((*_rows(case), c), dtype=dtype, device="cuda").normal_(generator=gen).mul_(2.5)
        rank = torch.randperm(c, device="cuda", generator=gen)
        x += (-0.5 * torch.log(rank + 1.0)).to(dtype)
    if case["masked"]:
        off = torch.rand(c, device="cuda", generator=gen) < case["masked"]
        off[int(torch.randint(c, (1,), device="cuda", generator=gen))] = False
        x.masked_fill_(off, -math.inf)
        x.masked_fill_((torch.rand(_rows(case), device="cuda", generator=gen) < 0.02).unsqueeze(-1), -math.inf)
    return x


def _parameters(case, gen):
    """Rows of log-probabilities in groups of 256 (leaf tables), Dirichlet(1)"""
    n, c = case["n"], case["c"]
    x = torch.empty((n, c), device="cuda").exponential_(generator=gen)
    for part in x.split(max(1, (1 << 26) // c)):
        whole = part[:, :c // 256 * 256].view(part.shape[0], -1, 256)
        whole /= whole.sum(-1, keepdim=True)
        part[:, c // 256 * 256:] /= 256.0
        part.clamp_(min=1e-9).log_()
    return x.to(TYPES[case["dtype"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "checkpoint":
        return dict(case=case, x=_parameters(case, gen))
    x, rows, c = _logits(case, gen), _rows(case), case["c"]
    state = dict(case=case, x=x, given=None)
    if case["given"]:
        shape = rows if case["given"] == 1 else (*rows, case["given"])
        g = torch.randint(c, shape, device="cuda", generator=gen)
        if c > 256:                                # token ids: some positions carry none; pixels and clusters are bytes
            g.masked_fill_(torch.rand(shape, device="cuda", generator=gen) < 0.01, -1)
        state["given"] = g.to(torch.uint8) if c <= 256 else g.to(torch.int32) if case["given"] > 1 else g
    if case["kind"] in ("gradient", "step"):
        # the derivative of a mean over rows; in f16, whose range ends at 6e-8, of the loss scaled up
        each = 16.0 if case["dtype"] == "f16" else 1.0 / math.prod(rows)
        if case["given"]:
            state["grad_logp"] = -each * torch.rand(state["given"].shape, device="cuda", generator=gen)
        if case["entropy"]:
            state["grad_entropy"] = 0.1 * each * torch.randn(rows, device="cuda", generator=gen)
        if case["top"]:
            state["grad_top"] = each * torch.randn((*rows, case["top"]), device="cuda", generator=gen)
    if case["kind"] == "gradient":                 # what the forward pass left
        state["log_sum"], state["entropy"] = _statistics(x.float())
        if case["top"]:
            state["top"] = _likeliest(x.float(), state["log_sum"], case["top"])[0]
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------

def _statistics(x):
    """log Z and entropy of rows in 32 bits"""
    m = x.amax(-1, keepdim=True)
    m = m.masked_fill(m == -math.inf, 0.0)
    z = (x - m).exp_().sum(-1, keepdim=True).log_().add_(m)
    d = x - z
    p = d.exp()
    return z.squeeze(-1), -(p * d.masked_fill_(p == 0, 0.0)).sum(-1)


def _likeliest(x, log_sum, top):
    """Indices and log-probabilities of the `top` largest entries, equal ones by rising index: the order of whole numbers
    that hold the entry's bits above the index counted from behind"""
    c = x.shape[-1]
    bits = (x + 0.0).contiguous().view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    key = (bits << 32).add_(torch.arange(c - 1, -1, -1, device=x.device))
    index = c - 1 - (key.topk(top, -1).values & 0xffffffff)
    value = x.gather(-1, index)
    z = log_sum.unsqueeze(-1)
    offered = (value > -math.inf) & ~torch.isnan(z)
    logp = torch.where(offered, value - z, torch.where(torch.isnan(z), math.nan, -math.inf))
    return torch.where(offered, index, -1).int(), logp


def _of_given(x, log_sum, given):
    """Log-probabilities of the given categories"""
    g = given.long() if given.dim() == x.dim() else given.long().unsqueeze(-1)
    c = x.shape[-1]
    z = log_sum.unsqueeze(-1)
    value = x.gather(-1, g.clamp(0, c - 1))
    logp = torch.where(z == -math.inf, z, value - z)
    logp = torch.where(g < 0, 0.0, torch.where(g >= c, math.nan, logp))
    return logp.reshape(given.shape)


def _scatter(x, index, grad):
    """x[index] += grad along the last axis, nothing where index < 0"""
    i = index.long() if index.dim() == x.dim() else index.long().unsqueeze(-1)
    g = torch.where(i < 0, 0.0, grad.reshape(i.shape))
    x.scatter_add_(-1, i.clamp(min=0), g)
    return g.sum(-1, keepdim=True)


def _gradient(x, log_sum, dtype, given=None, grad_logp=None, entropy=None, grad_entropy=None, top=None, grad_top=None):
    z = log_sum.unsqueeze(-1)
    d = x - z
    p = d.exp()
    out, total = torch.zeros_like(p), 0.0
    if given is not None:
        total = total + _scatter(out, given, grad_logp)
    if top is not None:
        total = total + _scatter(out, top, grad_top)
    out -= p * total
    if grad_entropy is not None:
        out -= grad_entropy.unsqueeze(-1) * p * (d + entropy.unsqueeze(-1)).masked_fill_(p == 0, 0.0)
    return out.masked_fill_(z == -math.inf, 0.0).to(dtype)


def _rounded(x, dtype):
    """The values that rows stand for in 8 bits, in 32 bits"""
    n, c = x.shape
    lowest = torch.finfo(dtype).min / 2
    pad = -c % BLOCK
    b = torch.nn.functional.pad(x, (0, pad), value=-math.inf).view(n, -1, BLOCK)
    bad = (torch.isnan(b) | (b == math.inf)).any(-1, keepdim=True)
    off = b <= lowest
    hi = b.masked_fill(off, -math.inf).amax(-1, keepdim=True)
    lo = b.masked_fill(off, math.inf).amin(-1, keepdim=True)
    none = hi == -math.inf
    hi, lo = hi.masked_fill(none, 0.0), lo.masked_fill(none, 0.0)
    f, q = torch.frexp(0.5 * hi - 0.5 * lo)
    e = torch.where(f > 0, q + torch.where(f > 253.0 / 256.0, -6, -7), -126)
    a = torch.maximum(hi.abs(), lo.abs())
    e = torch.maximum(e, torch.where(a > 0, torch.frexp(a)[1] - 14, -126)).clamp_(min=-126).int()
    step, steps = ((127 + k) << 23 for k in (e, -e))                    # the bits of 2^e and 2^-e
    v = torch.round(b * steps.view(torch.float32)) * step.view(torch.float32)
    v = v.clamp(max=torch.finfo(torch.float32).max).masked_fill(off, -math.inf).masked_fill(bad, math.nan)
    return v.view(n, -1)[:, :c]


def _plain(state):
    case, x = state["case"], state["x"]
    kind, dtype = case["kind"], x.dtype
    if kind == "checkpoint":
        return _rounded(x.float(), dtype)
    f = x.float()
    grads = {k: state[k] for k in ("given", "grad_logp", "grad_entropy", "top", "grad_top") if state.get(k) is not None}
    if kind == "gradient":
        return _gradient(f, state["log_sum"], dtype, entropy=state["entropy"], **grads)
    log_sum, entropy = _statistics(f)
    out = dict(log_sum=log_sum)
    if state["given"] is not None:
        out["logp"] = _of_given(f, log_sum, state["given"])
    if case["entropy"]:
        out["entropy"] = entropy
    if case["top"]:
        out["top"], out["top_logp"] = _likeliest(f, log_sum, case["top"])
    if kind == "step":
        kept = _rounded(f.reshape(-1, case["c"]), dtype).view(f.shape)
        out["grad"] = _gradient(kept, log_sum, dtype, entropy=entropy, **grads)
    return out


# ---- the package's own ------------------------------------------------------------------------------------------

def _package():
    where = os.path.join(os.getcwd(), "lvd-pg_amd")
    if where not in sys.path:
        sys.path.insert(0, where)
    import pcmi355
    return pcmi355


def _call(state):
    P, case, x = _package(), state["case"], state["x"]
    if case["kind"] == "checkpoint":
        return P.checkpoint_rows(x).restore(torch.float32)
    grads = {k: state[k] for k in ("grad_logp", "grad_entropy", "top", "grad_top") if state.get(k) is not None}
    if case["kind"] == "gradient":
        if case["entropy"]:
            grads["entropy"] = state["entropy"]
        return P.category_scores_backward(x, state["log_sum"], state["given"], **grads)
    s = P.category_scores(x, state["given"], top=case["top"], entropy=case["entropy"], checkpoint=case["kind"] == "step")
    out = dict(log_sum=s.log_sum)
    if state["given"] is not None:
        out["logp"] = s.logp
    if case["entropy"]:
        out["entropy"] = s.entropy
        grads["entropy"] = s.entropy
    if case["top"]:
        out["top"], out["top_logp"] = s.top, s.top_logp
    if case["kind"] == "step":
        out["grad"] = P.category_scores_backward(s.checkpoint, s.log_sum, state["given"], **grads)
    return out


def run(state):
    if own:
        return _call(state)
    return _plain(state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _grid64(x, dtype):
    """Rows (64 bits, holding values of `dtype`) as 8 bits hold them: block by block along the row"""
    out = torch.empty_like(x)
    limit = float(torch.finfo(dtype).min) / 2
    for s in range(0, x.shape[1], BLOCK << 14):
        part = x[:, s:s + (BLOCK << 14)]
        width = part.shape[1]
        blocks = -(-width // BLOCK)
        b = torch.full((x.shape[0], blocks * BLOCK), -math.inf, dtype=torch.float64, device=x.device)
        b[:, :width] = part
        b = b.view(-1, BLOCK)
        kept = b > limit
        high = torch.where(kept, b, -math.inf).max(1).values
        low = torch.where(kept, b, math.inf).min(1).values
        some = kept.any(1)
        high, low = torch.where(some, high, 0.0), torch.where(some, low, 0.0)
        spread = (high - low).float().double()     # the format takes the difference in 32 bits
        # smallest power of two that has 253 steps over the spread where the mantissa allows, 2^14 over the largest entry
        e = torch.full_like(spread, -126, dtype=torch.int64)
        f, q = torch.frexp(spread)
        e = torch.where(spread > 0, torch.maximum(e, q - 7 - (256 * f <= 253).long()), e)
        size = torch.maximum(high.abs(), low.abs())
        e = torch.where(size > 0, torch.maximum(e, torch.frexp(size)[1] - 14), e)
        unit = ((1023 + e) << 52).view(torch.float64)[:, None]
        v = torch.where(kept, torch.round(b / unit) * unit, -math.inf)
        v = torch.where((torch.isnan(b) | (b == math.inf)).any(1, keepdim=True), math.nan, v)
        out[:, s:s + width] = v.view(x.shape[0], -1)[:, :width]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind, c, rows = case["kind"], case["c"], _rows(case)
    x = state["x"].reshape(-1, c)
    total, dtype = x.shape[0], x.dtype
    chunk = max(1, (1 << 25) // c)
    flat = {k: state[k].reshape(total, -1) for k in ("given", "grad_logp", "grad_entropy", "top", "grad_top", "log_sum", "entropy")
            if state.get(k) is not None}
    found = {}
    for s in range(0, total, chunk):
        y = x[s:s + chunk].double()
        part = {k: t[s:s + chunk] for k, t in flat.items()}
        if kind == "checkpoint":
            found.setdefault("out", []).append(_grid64(y, dtype))
            continue
        if kind == "gradient":
            z, h = part["log_sum"].double(), part["entropy"].double()
        else:
            z = torch.logsumexp(y, 1, keepdim=True)
            d = y - z
            h = -torch.where(y > -math.inf, d.exp() * d, 0.0).sum(1, keepdim=True)
            found.setdefault("log_sum", []).append(z)
            found.setdefault("entropy", []).append(h)
            if "given" in part:
                g = part["given"].long()
                lp = torch.where(z == -math.inf, z, y.gather(1, g.clamp(min=0)) - z)
                found.setdefault("logp", []).append(torch.where(g < 0, 0.0, lp))
            if case["top"]:
                order = torch.sort(y, dim=1, descending=True, stable=True)
                value, index = order.values[:, :case["top"]], order.indices[:, :case["top"]]
                found.setdefault("top", []).append(torch.where(value > -math.inf, index, -1).int())
                found.setdefault("top_logp", []).append(torch.where(value > -math.inf, value - z, -math.inf))
                del order
        if kind in ("gradient", "step"):
            if kind == "step":
                y = _grid64(y, dtype)
            alive = z > -math.inf
            d = torch.where(alive & (y > -math.inf), y - z, 0.0)
            p = torch.where(alive & (y > -math.inf), d.exp(), 0.0)
            grad = torch.zeros_like(p)
            for index, by in (("given", "grad_logp"), ("top", "grad_top")):
                for j in range(part[index].shape[1] if by in part else 0):
                    g, w = part[index][:, j:j + 1].long(), part[by][:, j:j + 1].double()
                    w = torch.where(g < 0, 0.0, w)
                    grad -= p * w
                    grad.scatter_add_(1, g.clamp(min=0), w)
            if "grad_entropy" in part:
                grad -= part["grad_entropy"].double() * p * (d + h)
            found.setdefault("grad", []).append(torch.where(alive, grad, 0.0))
    found = {k: torch.cat(v) for k, v in found.items()}
    if kind == "checkpoint":
        return found["out"]
    if kind == "gradient":
        return found["grad"].view(*rows, c)
    out = dict(log_sum=found["log_sum"].view(rows))
    if "logp" in found:
        out["logp"] = found["logp"].view(state["given"].shape)
    if case["entropy"]:
        out["entropy"] = found["entropy"].view(rows)
    if case["top"]:
        out["top"], out["top_logp"] = (found[k].view(*rows, case["top"]) for k in ("top", "top_logp"))
    if kind == "step":
        out["grad"] = found["grad"].view(*rows, c)
    return out


def work(case):
    """Bytes: scores in once, results out once (a step also writes and reads its checkpoint: an entry a byte, four bytes per 64).
    Flops: difference, exponential, sum and the entropy's product per entry, about as many again for a gradient."""
    rows, c, size = math.prod(_rows(case)), case["c"], SIZE[case["dtype"]]
    entries = rows * c
    kept = entries + 4 * rows * -(-c // BLOCK)
    if case["kind"] == "checkpoint":
        return dict(bytes=entries * (size + 4) + 2 * kept, flops=6 * entries)
    index = 1 if c <= 256 else 4 if case["given"] > 1 else 8
    given, top, h = case["given"] * rows, case["top"] * rows, rows if case["entropy"] else 0
    if case["kind"] == "gradient":
        return dict(bytes=2 * entries * size + given * (index + 4) + 8 * top + 8 * h + 4 * rows, flops=6 * entries)
    forward = entries * size + given * (index + 4) + 8 * top + 4 * h + 4 * rows
    if case["kind"] == "score":
        return dict(bytes=forward, flops=5 * entries)
    return dict(bytes=forward + 2 * kept + entries * size + given * (index + 4) + 8 * h, flops=16 * entries)

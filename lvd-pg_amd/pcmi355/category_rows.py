"""Rows of category scores: log-probabilities of given categories, entropy and likeliest categories, their gradient, and
rows kept in 8 bits between a forward and a backward pass.

The rows are whatever has a score per category: soft evidence [examples, variables, categories], the per-head
log-likelihoods of a multi-head circuit or a forest (`head_scores`), the logits of the network that a circuit is distilled
from, matrices of parameter rows.  The reference leaves this to its Python programs; there is nothing to cite.

Everything runs on torch's current stream of the tensors' device, waits for nothing, and can be captured into a graph; nothing
here records for torch.autograd: a backward pass is a call, as `kld_backward` is."""
import math
from typing import NamedTuple, Optional

import torch

from ._lib import lib, check
from . import queries
from .circuits import HcltForest

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INDEX_TYPES = {torch.uint8: 3, torch.int32: 4, torch.int64: 5}
_MAX_SLOTS = 64      # most given, and most likeliest, categories of a row
_BLOCK = 64          # neighbours of a row that share a scale
_MAX_CATS, _MAX_ROWS = 1 << 30, (1 << 31) - 1


class Checkpoint8:
    """Rows in 8 bits (`checkpoint_rows`): `codes` uint8 [rows, categories rounded up to 16], `scales` int32 [rows, blocks of
    64], with the `shape` and `dtype` of the rows they stand for."""
    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        n, v, c = _sizes(shape)
        _check_sizes(shape, "a checkpoint of rows")
        if codes.dtype != torch.uint8 or codes.shape != (n * v, -(-c // 16) * 16) or not codes.is_contiguous() \
                or scales.dtype != torch.int32 or scales.shape != (n * v, -(-c // _BLOCK)) or not scales.is_contiguous() \
                or scales.device != codes.device or dtype not in _TYPES:
            raise ValueError(f"no checkpoint of rows {tuple(shape)} of {dtype}: codes {codes.dtype} {tuple(codes.shape)}, scales "
                             f"{scales.dtype} {tuple(scales.shape)}")
        self.codes, self.scales, self.shape, self.dtype = codes, scales, tuple(shape), dtype

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + 4 * self.scales.numel()

    def restore(self, dtype=None, out=None):
        """The rows that the codes stand for, see `restore_rows`."""
        return restore_rows(self, dtype, out)


class CategoryScores(NamedTuple):
    """What `category_scores` returns; None for what was not asked for."""
    logp: Optional[torch.Tensor]         # shaped like `given`
    log_sum: torch.Tensor                # [rows...]
    entropy: Optional[torch.Tensor]      # [rows...]
    top: Optional[torch.Tensor]          # [rows..., top] int32
    top_logp: Optional[torch.Tensor]     # [rows..., top]
    checkpoint: Optional[Checkpoint8]


def _check_rows(x, what):
    if not isinstance(x, torch.Tensor) or x.dim() not in (2, 3) or x.dtype not in _TYPES:
        raise ValueError(f"{what} must be a float32, bfloat16 or float16 tensor [rows, categories] or "
                         "[examples, variables, categories]")
    if x.shape[-1] < 1:
        raise ValueError(f"{what} need at least one category")
    if x.numel() >> 30:                                      # (fewer entries: none of the sizes is past its limit)
        _check_sizes(x.shape, what)


def _check_sizes(shape, what):
    """The entry points take sizes in 32 bits: what does not fit is refused here, it would arrive cut off"""
    if shape[-1] > _MAX_CATS or math.prod(shape[:-1]) > _MAX_ROWS:
        raise ValueError(f"{what} of shape {tuple(shape)}: at most 2^30 categories and 2^31 - 1 rows")


def _on_gpu(*tensors):
    first = tensors[0]
    index = first.get_device() if first.is_cuda else -1
    if index < 0:
        raise ValueError("the rows must be on the GPU")
    for t in tensors[1:]:
        if t is not None and t.get_device() != index:
            raise ValueError(f"a tensor is on {t.device}, the rows on {first.device}")


def _sizes(shape):
    return (shape[0], 1, shape[1]) if len(shape) == 2 else tuple(shape)


def _strides(x):
    s = x.stride()
    return (s[0], 0, s[1]) if len(s) == 2 else s


def _check_given(given, rows):
    """Given categories: a tensor shaped like the rows, or with a last axis of slots.  Returns (pointer, type, strides, slots)."""
    if given is None:
        return None, 3, 0, 0, 0, 0
    if not isinstance(given, torch.Tensor) or given.dtype not in _INDEX_TYPES:
        raise ValueError("given categories must be a uint8, int32 or int64 tensor")
    k = len(rows)
    if given.shape[:k] != rows or given.dim() not in (k, k + 1):
        raise ValueError(f"given categories are {tuple(given.shape)}, the rows {rows}: one per row, or [rows, slots]")
    slots = 1 if given.dim() == k else given.shape[k]
    if slots > _MAX_SLOTS:
        raise ValueError(f"at most {_MAX_SLOTS} given categories a row, got {slots}")
    s = given.stride()
    slot = s[k] if given.dim() > k else 0
    return given.data_ptr(), _INDEX_TYPES[given.dtype], s[0], s[1] if k == 2 else 0, slot, slots


def _f32(t, shape, what):
    if not isinstance(t, torch.Tensor) or t.shape != shape:
        raise ValueError(f"{what} must be a tensor of shape {tuple(shape)}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _no_overlap(t):
    """Whether no two elements of a tensor are one (sufficient: every stride passes the extent of the smaller ones)"""
    reach = 0
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s <= reach:
            return False
        reach += s * (n - 1)
    return True


def _extent(t):
    return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape)))


def _check_out(out, shape, dtype, device):
    if not isinstance(out, torch.Tensor) or tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != device:
        raise ValueError(f"out must be a {dtype} tensor of shape {tuple(shape)} on {device}")
    if not _no_overlap(out):
        raise ValueError("out has elements that share memory")


def _may_meet(ahead, a, b):
    """Whether two sets of bytes may share one (False: they do not).  A set is (bytes of an element, [(stride, number), ...]), the
    second one's first byte lies `ahead` of the first one's.  Strides that are multiples of a period drop out modulo that
    period, and what is left of the sets can only meet as it lies or one period back."""
    if ahead >= a[0] + sum(s * (n - 1) for s, n in a[1]) or -ahead >= b[0] + sum(s * (n - 1) for s, n in b[1]):
        return False
    for period in {s for s, _ in a[1] + b[1]}:
        rest = [(e, [(s, n) for s, n in parts if s % period]) for e, parts in (a, b)]
        if all(e + sum(s * (n - 1) for s, n in parts) <= period for e, parts in rest) \
                and not any(_may_meet(ahead % period - back, *rest) for back in (0, period)):
            return False
    return True


def _bytes(t):
    return t.element_size(), [(s * t.element_size(), n) for s, n in zip(t.stride(), t.shape) if s and n > 1]


def _apart(out, *others):
    """out shares no memory with other tensors"""
    (a, b), rest = _extent(out), ((t, *_extent(t)) for t in others if t is not None and t.numel())
    return not out.numel() or all(b <= c or d <= a or not _may_meet(c - a, _bytes(out), _bytes(t)) for t, c, d in rest)


# the stream without an object around it, where torch has it: 0.1 us instead of 2.9
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _on_device_of(t, call):
    """call(stream) with a tensor's device as the current one"""
    index = t.device.index
    if index == torch.cuda.current_device():
        check(call(_raw_stream(index)))
    else:
        with torch.cuda.device(index):
            check(call(_raw_stream(index)))


def _new_checkpoint(x, shape):
    n, v, c = _sizes(shape)
    kept = Checkpoint8.__new__(Checkpoint8)                  # (its parts fit by construction)
    kept.codes = torch.empty(n * v, -(-c // 16) * 16, dtype=torch.uint8, device=x.device)
    kept.scales = torch.empty(n * v, -(-c // _BLOCK), dtype=torch.int32, device=x.device)
    kept.shape, kept.dtype = shape, x.dtype
    return kept


def category_scores(scores, given=None, *, top=0, entropy=False, checkpoint=False):
    """Log-probabilities of `given` categories under rows of scores, with the rows' log-sum, entropy and `top` likeliest
    categories, in one pass over the scores (a checkpoint of rows whose categories are not neighbours takes a second one).

    scores: float32, bfloat16 or float16 GPU tensor [rows, categories] or [examples, variables, categories], any strides.
    given: uint8, int32 or int64, one category per row or [rows..., slots] with up to 64; a negative one was not observed and has
    log-probability 0, one past the categories NaN.  top: 0 to 64; equal scores by rising category, masked categories
    never among them (-1 and -inf where a row has no more).  A score at or below half of the type's lowest value is a mask and
    counts as -inf; a row of nothing else has log-sum and log-probabilities -inf and, being no distribution, entropy NaN
    (leave such rows out of a mean over a padded batch); a row with NaN or +inf has NaN and -1.  checkpoint: also the scores in 8 bits (`checkpoint_rows`), for
    `category_scores_backward`, which see for scores far from zero.  Returns `CategoryScores`, numbers in float32."""
    _check_rows(scores, "scores")
    shape = tuple(scores.shape)
    rows = shape[:-1]
    if not 0 <= top <= _MAX_SLOTS:
        raise ValueError(f"top must lie in 0..{_MAX_SLOTS}, got {top}")
    where = _check_given(given, rows)
    _on_gpu(scores, given)
    new, dev = torch.empty, scores.device
    f32 = torch.float32
    log_sum = new(*rows, dtype=f32, device=dev)              # (sizes one by one: 1.3 us of the host, 1.7 as a tuple, 2.2 as a Size)
    logp = None if given is None else new(*given.shape, dtype=f32, device=dev)
    ent = new(*rows, dtype=f32, device=dev) if entropy else None
    best = new(*rows, top, dtype=torch.int32, device=dev) if top else None
    best_logp = new(*rows, top, dtype=f32, device=dev) if top else None
    kept = _new_checkpoint(scores, shape) if checkpoint else None
    if log_sum.numel():
        n, v, c = _sizes(shape)
        size = lib.pcm_category_scores_workspace(n, v, c, top)
        work = new(size, dtype=torch.uint8, device=dev) if size else None
        _on_device_of(scores, lambda stream: lib.pcm_category_scores(
            scores.data_ptr(), _TYPES[scores.dtype], *_strides(scores), n, v, c, *where, top,
            None if logp is None else logp.data_ptr(), log_sum.data_ptr(), None if ent is None else ent.data_ptr(),
            None if best is None else best_logp.data_ptr(), None if best is None else best.data_ptr(),
            None if kept is None else kept.codes.data_ptr(), None if kept is None else kept.scales.data_ptr(),
            None if work is None else work.data_ptr(), size, stream))
    return CategoryScores(logp, log_sum, ent, best, best_logp, kept)


def category_scores_backward(scores, log_sum, given=None, *, grad_logp=None, entropy=None, grad_entropy=None, top=None,
                             grad_top=None, out=None):
    """Gradient with respect to the scores of a loss with the derivatives `grad_logp` by the log-probabilities of `given`,
    `grad_top` by those of the `top` categories and `grad_entropy` by the entropy (each may be left out); `log_sum`,
    `entropy` and `top` as `category_scores` returned them.

    `scores`: the scores, or their `Checkpoint8`: the backward pass then reads a byte per score,
    and its probabilities are off by a factor of exp(half a step) at most, 1 + 1/253 of the range of 64 neighbours for small ones.
    Steps grow with the level of a row, |x| / 2^13 at most: the factor may be 1.13 for scores near -3000, 1.3 near -8000, e near
    -20000.  Nothing but differences within a row counts here, so keep such scores less their `log_sum` (`category_scores` of
    `scores - s.log_sum[..., None]`): the level is gone, and steps follow the range alone.  Returns a tensor of the scores'
    shape and type; `out`: where it goes, also the scores themselves, which are then overwritten.  The same category in several
    slots adds up, a negative one adds nothing, one past the categories makes its row NaN."""
    kept = scores if isinstance(scores, Checkpoint8) else None
    if kept is None:
        _check_rows(scores, "scores")
    shape, dtype, dev = tuple(scores.shape), scores.dtype, scores.device
    rows = shape[:-1]
    if (given is None) != (grad_logp is None) or (top is None) != (grad_top is None):
        raise ValueError("given and grad_logp, top and grad_top go together")
    if grad_entropy is not None and entropy is None:
        raise ValueError("grad_entropy needs the entropy")
    where = _check_given(given, rows)
    log_sum = _f32(log_sum, rows, "log_sum")
    if given is not None:
        grad_logp = _f32(grad_logp, given.shape, "grad_logp")
    slots = 0
    if top is not None:
        if not isinstance(top, torch.Tensor) or top.dtype != torch.int32 or top.shape[:-1] != rows or top.dim() != len(shape) \
                or top.shape[-1] > _MAX_SLOTS:
            raise ValueError(f"top must be int32 {(*rows, 'up to 64')}, as category_scores returns it")
        top, slots = top.contiguous(), top.shape[-1]
        grad_top = _f32(grad_top, top.shape, "grad_top")
    if grad_entropy is not None:
        entropy, grad_entropy = _f32(entropy, rows, "entropy"), _f32(grad_entropy, rows, "grad_entropy")
    else:
        entropy = None
    _on_gpu(kept.codes if kept is not None else scores, log_sum, given, grad_logp, entropy, grad_entropy, top, grad_top)
    if out is None:
        out = torch.empty(*shape, dtype=dtype, device=dev) if kept is not None else torch.empty_like(scores)
    else:
        _check_out(out, shape, dtype, dev)
        if kept is None and not (out.data_ptr() == scores.data_ptr() and out.stride() == scores.stride()) and not _apart(out, scores):
            raise ValueError("out overlaps the scores without being them")
        if not _apart(out, log_sum, given, grad_logp, entropy, grad_entropy, top, grad_top, *((kept.codes, kept.scales) if kept else ())):
            raise ValueError("out overlaps another argument")
    if log_sum.numel():
        n, v, c = _sizes(shape)
        ptr = queries._dev_ptr
        _on_device_of(out, lambda stream: lib.pcm_category_scores_backward(
            None if kept is not None else scores.data_ptr(), _TYPES[dtype], *((0, 0, 0) if kept is not None else _strides(scores)),
            n, v, c, None if kept is None else kept.codes.data_ptr(), None if kept is None else kept.scales.data_ptr(), *where,
            ptr(grad_logp), slots, ptr(top), ptr(grad_top), log_sum.data_ptr(), ptr(entropy), ptr(grad_entropy), out.data_ptr(),
            *_strides(out), stream))
    return out


def checkpoint_rows(rows):
    """Rows (float32, bfloat16 or float16, [rows, n] or [examples, variables, n], any strides) in 8 bits, for what a forward pass
    keeps for its backward pass: 64 neighbours of a row share a power-of-two step, the smallest that covers their range in at
    most 253 steps and the largest |x| among them in 2^14, and every entry becomes the nearest multiple of it.  It is off by half a
    step at most: 1/253 of the range, or |x| / 2^14 where that is more, as in rows that lie far from zero.  Entries
    at or below half of the type's lowest value (masks) come back as -inf, a block with NaN or +inf as NaN.  Returns a
    `Checkpoint8`, 1.06 bytes an entry."""
    _check_rows(rows, "rows")
    _on_gpu(rows)
    kept = _new_checkpoint(rows, tuple(rows.shape))
    if kept.codes.numel():
        n, v, c = _sizes(rows.shape)
        _on_device_of(rows, lambda stream: lib.pcm_checkpoint_rows(
            rows.data_ptr(), _TYPES[rows.dtype], *_strides(rows), n, v, c, kept.codes.data_ptr(), kept.scales.data_ptr(), stream))
    return kept


def restore_rows(checkpoint, dtype=None, out=None):
    """The rows that a `Checkpoint8` stands for, in the type they had or in float32 (where every value is exact), into `out`
    (any strides) if given."""
    if not isinstance(checkpoint, Checkpoint8):
        raise ValueError("restore_rows takes what checkpoint_rows returned")
    dtype = (checkpoint.dtype if out is None else out.dtype) if dtype is None else dtype
    if dtype not in (checkpoint.dtype, torch.float32):
        raise ValueError(f"rows of {checkpoint.dtype} come back as such or as float32, not as {dtype}")
    if out is None:
        out = torch.empty(*checkpoint.shape, dtype=dtype, device=checkpoint.device)
    else:
        _check_out(out, checkpoint.shape, dtype, checkpoint.device)
        if not _apart(out, checkpoint.codes, checkpoint.scales):
            raise ValueError("out overlaps the checkpoint")
    _on_gpu(out)
    if out.numel():
        n, v, c = _sizes(checkpoint.shape)
        _on_device_of(out, lambda stream: lib.pcm_restore_rows(
            checkpoint.codes.data_ptr(), checkpoint.scales.data_ptr(), n, v, c, out.data_ptr(), _TYPES[dtype], *_strides(out), stream))
    return out


def head_scores(mhbpc, data, given=None, *, top=0, entropy=True, batch_size=None, example_ids=None):
    """The posterior of the heads (clusters) of a multi-head circuit, or of every tree of a forest, for each example, all heads
    equally likely beforehand: `category_scores` of the per-head log-likelihoods (src-jl/multi_head_pc/likelihood.jl:37-71)
    where the forward pass left them.  `given`: cluster ids [examples] (forest: [examples, trees]), their log-probabilities come
    back; `log_sum` minus log(heads) is the log-likelihood of the mixture.  `batch_size` as for `loglikelihoods` (a forest
    takes its examples as one batch)."""
    if not getattr(mhbpc, "num_heads", 0):
        raise ValueError("the circuit has no heads")
    if isinstance(mhbpc, HcltForest):
        scores = queries.forest_loglikelihoods(mhbpc, data, example_ids=example_ids).permute(2, 0, 1)
    else:
        scores = queries._head_values(mhbpc, data, batch_size, example_ids).t()
    return category_scores(scores, given, top=top, entropy=entropy)

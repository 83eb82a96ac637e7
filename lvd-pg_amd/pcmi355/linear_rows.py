"""Category scores that are products of features and weights: log-probabilities without keeping the scores, their gradient, and
products of rows in 8-bit integers.

This is the head of a network that is taught what a circuit is distilled with (cluster ids, soft evidence) or from (tokens): `category_scores`
takes scores that are in memory, `linear_scores` the two matrices they are products of.  The reference leaves this to its Python
programs; there is nothing to cite.

Everything runs on torch's current stream of the tensors' device, waits for nothing, and can be captured into a graph; nothing
here records for torch.autograd: a backward pass is a call, as `category_scores_backward` is."""
import math
from typing import NamedTuple, Optional

import torch

from ._lib import lib
from .category_rows import _TYPES, _apart, _check_given, _check_out, _f32, _on_device_of, _on_gpu, _sizes, _strides

_MAX_ROWS, _MAX_CATS, _MAX_LENGTH = 1 << 22, 1 << 30, 1 << 20
_MAX_ROWS8, _MAX_LENGTH8 = (1 << 31) - 1, 131071       # (so many products of -128 and -128 stay within 32 bits)
_STEP8 = 128                                           # 8-bit rows are laid out in multiples of so many codes


class Rows8:
    """Rows in 8-bit integers (`rows8`): `codes` int8 [rows, length rounded up to 128] with zeros behind a row's end, `scales`
    float32 [rows], with the `shape` and `dtype` of the rows they stand for, codes times scale."""
    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        _check_rows8(shape)
        rows, length = math.prod(shape[:-1]), shape[-1]
        if codes.dtype != torch.int8 or codes.shape != (rows, -(-length // _STEP8) * _STEP8) or not codes.is_contiguous() \
                or codes.data_ptr() % 16 or scales.dtype != torch.float32 or scales.shape != (rows,) or not scales.is_contiguous() \
                or scales.device != codes.device or dtype not in _TYPES:
            raise ValueError(f"no 8-bit rows {tuple(shape)} of {dtype}: codes {codes.dtype} {tuple(codes.shape)}, scales "
                             f"{scales.dtype} {tuple(scales.shape)}")
        self.codes, self.scales, self.shape, self.dtype = codes, scales, tuple(shape), dtype

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + 4 * self.scales.numel()


class LinearScores(NamedTuple):
    """What `linear_scores` returns; `logp` is None where no categories are given."""
    logp: Optional[torch.Tensor]         # shaped like `given`
    log_sum: torch.Tensor                # [rows...]


class LinearGradients(NamedTuple):
    """What `linear_scores_backward` returns; None for what was not asked for."""
    features: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]


def _check_rows8(shape):
    if len(shape) not in (2, 3) or shape[-1] < 1 or shape[-1] > _MAX_LENGTH8 or math.prod(shape[:-1]) > _MAX_ROWS8:
        raise ValueError(f"8-bit rows of shape {tuple(shape)}: [rows, length] or [examples, variables, length], at most 2^31 - 1 rows "
                         f"of 1 to {_MAX_LENGTH8} entries")


def _check_factors(features, weight):
    """Features and weights that fit each other; whether they are rows in 8 bits"""
    eight = isinstance(features, Rows8)
    if eight != isinstance(weight, Rows8):
        raise ValueError("features and weight must both be tensors, or both rows in 8 bits")
    if not eight:
        if not isinstance(features, torch.Tensor) or features.dim() not in (2, 3) or features.dtype not in _TYPES:
            raise ValueError("features must be a float32, bfloat16 or float16 tensor [rows, length] or [examples, variables, length]")
        if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.dtype != features.dtype:
            raise ValueError(f"weight must be a {features.dtype} tensor [categories, length]")
    if len(weight.shape) != 2 or weight.shape[1] != features.shape[-1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [categories, {features.shape[-1]}], one category and one entry at least, got {tuple(weight.shape)}")
    if math.prod(features.shape[:-1]) > _MAX_ROWS or weight.shape[0] > _MAX_CATS or weight.shape[1] > _MAX_LENGTH:
        raise ValueError(f"features {tuple(features.shape)} and weight {tuple(weight.shape)}: at most 2^22 rows, 2^30 categories, length 2^20")
    return eight


def _check_bias(bias, count):
    """Returns (pointer, type, the tensor)"""
    if bias is None:
        return None, 0, None
    if not isinstance(bias, torch.Tensor) or bias.dtype not in _TYPES or bias.shape != (count,):
        raise ValueError(f"bias must be a float32, bfloat16 or float16 tensor [{count}]")
    bias = bias.contiguous()
    return bias.data_ptr(), _TYPES[bias.dtype], bias


def _work(size, device):
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    return work, None if work is None else work.data_ptr()


def _factors(features, weight):
    n, v, k = _sizes(features.shape)
    return (features.data_ptr(), weight.data_ptr(), _TYPES[features.dtype], *_strides(features), *weight.stride(), n, v, k, weight.shape[0])


def linear_scores(features, weight, given=None, *, bias=None):
    """Log-probabilities of `given` categories under the scores `features @ weight.T + bias`, with the rows' log-sums, without
    keeping the scores: `category_scores(features @ weight.T + bias, given)` in one pass over features and weights.

    features: float32, bfloat16 or float16 GPU tensor [rows, length] or [examples, variables, length]; weight: the same type,
    [categories, length]; any strides.  Both are read where they are, but for 16-bit types in some layouts (with more than 64 rows: lengths that
    are no multiple of 64, rows not at multiples of 16 bytes; entries that are not neighbours), which are laid out in a workspace in each
    call.  Or both as `rows8` returned them.
    given: uint8, int32 or int64, one category per row or [rows..., slots] with up to 64; a negative one was not observed and has
    log-probability 0, one past the categories NaN.  bias: [categories], any of the three types; at or below half of its type's lowest
    value it masks its category, whatever the weights hold.  A row of nothing but masks has log-sum and log-probabilities -inf, one with NaN or +inf
    NaN (float32: with any infinity among its factors, or products past the type's range).  float32 is taken as three bfloat16 parts whose six largest
    products are summed, which leaves out less than 2^-24 of a product, and what lies below 2^-134 of a factor; all sums are held in 32 bits.  Returns `LinearScores`, numbers in float32."""
    eight = _check_factors(features, weight)
    rows = tuple(features.shape[:-1])
    where = _check_given(given, rows)
    bias_at, bias_type, bias = _check_bias(bias, weight.shape[0])
    first = features.codes if eight else features
    _on_gpu(first, weight.codes if eight else weight, given, bias)
    dev = first.device
    log_sum = torch.empty(*rows, dtype=torch.float32, device=dev)
    logp = None if given is None else torch.empty(*given.shape, dtype=torch.float32, device=dev)
    if log_sum.numel():
        logp_at = None if logp is None or not logp.numel() else logp.data_ptr()
        if eight:
            n, v, k = _sizes(features.shape)
            size = lib.pcm_linear_scores8_workspace(n, v, k, weight.shape[0])
            work, work_at = _work(size, dev)
            _on_device_of(first, lambda stream: lib.pcm_linear_scores8(
                first.data_ptr(), features.scales.data_ptr(), weight.codes.data_ptr(), weight.scales.data_ptr(), n, v, k, weight.shape[0],
                bias_at, bias_type, *where, logp_at, log_sum.data_ptr(), work_at, size, stream))
        else:
            factors = _factors(features, weight)
            size = lib.pcm_linear_scores_workspace(*factors)
            work, work_at = _work(size, dev)
            _on_device_of(first, lambda stream: lib.pcm_linear_scores(
                *factors, bias_at, bias_type, *where, logp_at, log_sum.data_ptr(), work_at, size, stream))
    return LinearScores(logp, log_sum)


def linear_scores_backward(features, weight, log_sum, given=None, *, bias=None, grad_logp=None, grad_log_sum=None,
                           of=("features", "weight", "bias")):
    """Gradients with respect to features, weight and bias (those named in `of`; the bias's only if there is one) of a loss with the
    derivatives `grad_logp` by the log-probabilities of `given` and `grad_log_sum` by the log-sums (each may be left out);
    arguments and `log_sum` as for and from `linear_scores`, 8-bit rows excepted.

    The scores are computed once more, in pieces of the categories; their derivatives are rounded to the features' type, float16's
    relative to a power of two a row, which no scale of the loss overflows (float32: three bfloat16 parts; fewer than 1024 rows of 16 bits: two parts;
    rounded once, they are off by as much again as rounding the results is: bfloat16 gradients 2.3e-3 of their norm instead of 1.7e-3, float16 2.8e-4 instead of 2.1e-4).
    float16 features count in the weights' gradient down to 2^-25 of the largest derivative of any row.  The same category in several slots adds up, a negative one
    adds nothing, one past the categories makes its row's derivatives NaN.  A row whose derivatives are all 0 (a batch's padding,
    whose categories are all negative) has no part in any gradient, whatever its features hold; nor have a masked category's weights in the features' gradient.
    Returns `LinearGradients`: tensors of the shapes and types of features, weight and bias; the same bits every time."""
    if _check_factors(features, weight):
        raise ValueError("rows in 8 bits have no gradient")
    of = (of,) if isinstance(of, str) else tuple(of)
    if not of or set(of) - {"features", "weight", "bias"}:
        raise ValueError(f'of must name some of "features", "weight", "bias", got {of}')
    rows = tuple(features.shape[:-1])
    if (given is None) != (grad_logp is None):
        raise ValueError("given and grad_logp go together")
    where = _check_given(given, rows)
    bias_at, bias_type, bias = _check_bias(bias, weight.shape[0])
    log_sum = _f32(log_sum, rows, "log_sum")
    if given is not None:
        grad_logp = _f32(grad_logp, given.shape, "grad_logp")
    if grad_log_sum is not None:
        grad_log_sum = _f32(grad_log_sum, rows, "grad_log_sum")
    _on_gpu(features, weight, log_sum, given, bias, grad_logp, grad_log_sum)
    dev, dtype = features.device, features.dtype
    out = [None, None, None]
    if "features" in of:
        out[0] = torch.empty(*features.shape, dtype=dtype, device=dev)
    if "weight" in of:
        out[1] = torch.empty(*weight.shape, dtype=dtype, device=dev)
    if "bias" in of and bias is not None:
        out[2] = torch.empty(*bias.shape, dtype=bias.dtype, device=dev)
    if not log_sum.numel():
        return LinearGradients(*(None if t is None else t.zero_() for t in out))
    if any(t is not None for t in out):
        factors = _factors(features, weight)
        size = lib.pcm_linear_scores_backward_workspace(*factors, sum(1 << i for i, t in enumerate(out) if t is not None))
        work, work_at = _work(size, dev)
        _on_device_of(features, lambda stream: lib.pcm_linear_scores_backward(
            *factors, bias_at, bias_type, *where, None if grad_logp is None or not grad_logp.numel() else grad_logp.data_ptr(),
            None if grad_log_sum is None else grad_log_sum.data_ptr(), log_sum.data_ptr(), *(None if t is None else t.data_ptr() for t in out),
            work_at, size, stream))
    return LinearGradients(*out)


def rows8(rows):
    """Rows (float32, bfloat16 or float16, [rows, length] or [examples, variables, length], any strides) in 8-bit integers with a scale
    each: weights once, features in each call.  Code rint(x (127 / a)), scale a / 127, a the row's largest |x|: off by half a scale at most
    (and 2^-23 of |x|).  A row whose a lies below 2^-119 is one of zeros; one with NaN or an infinity has scale NaN, and so have its products.  Returns `Rows8`."""
    if not isinstance(rows, torch.Tensor) or rows.dtype not in _TYPES or rows.dim() not in (2, 3):
        raise ValueError("rows must be a float32, bfloat16 or float16 tensor [rows, length] or [examples, variables, length]")
    _check_rows8(rows.shape)
    _on_gpu(rows)
    n, v, k = _sizes(rows.shape)
    out = Rows8.__new__(Rows8)                               # (its parts fit by construction)
    out.codes = torch.empty(n * v, -(-k // _STEP8) * _STEP8, dtype=torch.int8, device=rows.device)
    out.scales = torch.empty(n * v, dtype=torch.float32, device=rows.device)
    out.shape, out.dtype = tuple(rows.shape), rows.dtype
    if out.scales.numel():
        _on_device_of(rows, lambda stream: lib.pcm_rows8(
            rows.data_ptr(), _TYPES[rows.dtype], *_strides(rows), n, v, k, out.codes.data_ptr(), out.scales.data_ptr(), stream))
    return out


def product8(rows, channels, *, bias=None, dtype=None, out=None):
    """The product rows @ channels.T + bias of rows in 8 bits: [rows..., channels] of `dtype` (the type that `rows` had, if not given),
    each entry the exact sum of the products of codes, times the row's and the channel's scale, plus the bias, in float32, rounded
    once.  rows, channels: `Rows8` of the same length, channels [channels, length].  bias: [channels], any of the three types.
    out: where the result goes, a tensor of that shape whose rows are neighbours [rows..., channels] in memory."""
    if not isinstance(rows, Rows8) or not isinstance(channels, Rows8):
        raise ValueError("product8 takes what rows8 returned")
    if len(channels.shape) != 2 or channels.shape[1] != rows.shape[-1] or channels.shape[0] < 1:
        raise ValueError(f"channels must be [channels, {rows.shape[-1]}], one at least, got {channels.shape}")
    count, length = channels.shape
    dtype = (rows.dtype if out is None else out.dtype) if dtype is None else dtype
    if dtype not in _TYPES:
        raise ValueError(f"a product is float32, bfloat16 or float16, not {dtype}")
    bias_at, bias_type, bias = _check_bias(bias, count)
    _on_gpu(rows.codes, channels.codes, bias)
    shape = (*rows.shape[:-1], count)
    if out is None:
        out = torch.empty(*shape, dtype=dtype, device=rows.device)
    else:
        _check_out(out, shape, dtype, rows.device)
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
        if not _apart(out, rows.codes, rows.scales, channels.codes, channels.scales, bias):
            raise ValueError("out overlaps another argument")
    if out.numel():
        n = rows.scales.numel()
        size = lib.pcm_product8_workspace(n, count, length)
        work, work_at = _work(size, out.device)
        _on_device_of(out, lambda stream: lib.pcm_product8(
            rows.codes.data_ptr(), rows.scales.data_ptr(), n, channels.codes.data_ptr(), channels.scales.data_ptr(), count, length, bias_at,
            bias_type, out.data_ptr(), _TYPES[dtype], count, work_at, size, stream))
    return out

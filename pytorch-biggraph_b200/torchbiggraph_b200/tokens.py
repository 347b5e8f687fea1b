"""Token operators on CUDA tensors: rows of a table by id, log probabilities over rows of scores, and their gradients.

They stand on either side of what this package trains: a table of embeddings, and answers that are rows of a table.  The
reference has no counterpart (it gathers with F.embedding and takes its losses over sampled negatives).  As everywhere
here the arithmetic runs in libpbg_b200.so and gradients are functions of their own: nothing is recorded for autograd, and a tensor
that requires a gradient is refused while gradients are being recorded -- detach it, or call under torch.no_grad() -- as is one
that carries a forward-mode tangent.  A tensor given as `out` counts as modified: what autograd has saved of it is not used any more.

All calls are queued on PyTorch's current stream of the tensors' device and return at once; workspaces come from PyTorch's allocator.
No call synchronises, so all of them can be captured into a CUDA graph.  Ids and targets are int64.  One outside of its range
cannot raise: a looked-up row and a log probability of it are NaN and a rank of it 0 (a row's lse and entropy, which do not depend on the
target, are as they are), its part of a gradient is left out, and 1 is set in `errors`, an int32 tensor of one element, where
one is given (`check_errors` reads it and raises).  Results of a kernel whose bounded wait ran out are NaN, and 2 is set.

Types: float32, bfloat16, float16; sums and statistics are float32 and results rounded once."""
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib

IGNORE_INDEX = -100
MAX_TOP = 32


class _TokenLogprobs(NamedTuple):
    logprob: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    rank: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


class TokenLogprobs(_TokenLogprobs):
    """Per row: log probability of the target, entropy, log of the sum of exponentials (float32), rank of the target (1 = best; 0
    for padding); with top > 0 the best log probabilities [n, top] and their ids.  Beside these six stands the attribute lse_rest: what float32
    cannot hold of lse, for token_logprobs_grad."""
    lse_rest: Optional[torch.Tensor] = None


# A call is tens of microseconds of host work or it is not: the checks below ask each tensor for as little as they can.
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}                    # pbg_dtype
_entry_points = {}


def _matrix(name, t, dtype=None, device=None):
    """The pbg_dtype of a matrix whose rows can be read."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.requires_grad or forward_ad._current_level >= 0:
        _no_grad(name, t)
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}: the token operators work on CUDA tensors only (no CPU fallback)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    code = _DTYPES.get(t.dtype)
    if code is None or (dtype is not None and t.dtype is not dtype):
        raise TypeError(f"{name} has type {t.dtype}" + (f", not {dtype}" if dtype is not None else "; float32, bfloat16 and float16 are supported"))
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions")
    width = t.shape[1]
    if width < 1:
        raise ValueError(f"{name} has rows without elements")
    if width > 1 and t.stride(1) != 1:
        raise ValueError(f"the elements of a row of {name} must lie next to each other")
    return code


def _no_grad(name, t):
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, which the token operators do not record: detach it or call under torch.no_grad()")
    if forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} carries a forward-mode tangent, which the token operators do not propagate: take its primal")


def _vector(name, t, dtype, n, device):
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype:
        raise TypeError(f"{name} must be a tensor of {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must have one dimension of {n} elements")
    if t.requires_grad or forward_ad._current_level >= 0:
        _no_grad(name, t)
    return t if t.is_contiguous() else t.contiguous()


def _ids(ids, device):
    if not isinstance(ids, torch.Tensor) or ids.dtype is not torch.long:
        raise TypeError("ids must be an int64 tensor")
    if ids.device != device:
        raise ValueError(f"ids is on {ids.device}, not on {device}")
    if ids.dim() != 1:
        ids = ids.reshape(-1)
    return ids if ids.is_contiguous() else ids.contiguous()


def _scale(scale, positive):
    scale = float(scale)
    if not math.isfinite(scale) or (positive and not 1e-20 <= scale <= 1e20):
        raise ValueError("scale must lie between 1e-20 and 1e20" if positive else "scale must be finite")
    return scale


def _error_word(errors, device):
    if errors is None:
        return None
    if not isinstance(errors, torch.Tensor) or errors.dtype != torch.int32 or errors.numel() != 1:
        raise TypeError("errors must be an int32 tensor of one element")
    if errors.device != device:
        raise ValueError(f"errors is on {errors.device}, not on {device}")
    return errors.data_ptr()


def _row_stride(t):
    """Elements from row to row (a single row's stride says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _overlap(a, b):
    """Whether the address ranges of two strided matrices meet."""
    def span(t):
        first = t.data_ptr()
        return first, first + (sum((s - 1) * abs(k) for s, k in zip(t.shape, t.stride())) + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _call(name, device, *args):
    """The entry point `name` on the current stream of `device`."""
    fn = _entry_points.get(name)
    if fn is None:
        fn = _entry_points[name] = getattr(_lib.lib(), name)
    index = device.index
    if torch.cuda.current_device() == index:
        status = fn(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _current_stream(index))
    if status:
        _lib.check(status)


def _workspace(name, device, *sizes):
    """Device memory of the size that the function `name` gives, and that size.  (Under the tensors' device: it may depend on it.)"""
    fn = _entry_points.get(name)
    if fn is None:
        fn = _entry_points[name] = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == device.index:
        size = fn(*sizes)
    else:
        with torch.cuda.device(device.index):
            size = fn(*sizes)
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None, size


def check_errors(errors: torch.Tensor) -> None:
    """Raises what the calls that were given `errors` have found so far, and clears it.  Waits for them."""
    found = int(errors.item())
    if found:
        errors.zero_()
    if found & 2:
        raise _lib.PbgError(_lib.PBG_ERR_TIMEOUT, "a bounded device-side wait ran out")
    if found & 1:
        raise IndexError("an id or target lies outside of its range")
    if found & 4:
        raise ValueError("the lse of a row lies beyond 1e6: the gradient needs the lse_rest of the forward call")


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0, errors: Optional[torch.Tensor] = None) -> torch.Tensor:
    """scale * table[ids]: a tensor of the table's type and of shape ids.shape + (dim,).  The table's rows may lie apart (a
    view of some columns); ids of any shape.  An id outside of the table gives a row of NaN."""
    code, device = _matrix("table", table), table.device
    flat = _ids(ids, device)
    (rows, dim), n = table.shape, flat.shape[0]
    if rows == 0 and n > 0:
        raise ValueError("table has no rows")
    out = table.new_empty((n, dim))
    _call("pbg_embedding_lookup", device, table.data_ptr(), _row_stride(table), rows, dim, code, flat.data_ptr(), n, _scale(scale, False),
          out.data_ptr(), _error_word(errors, device))
    return out if ids.dim() == 1 else out.view(*ids.shape, dim)


def embedding_lookup_grad(grad: torch.Tensor, ids: torch.Tensor, num_rows: int, *, scale: float = 1.0, out: Optional[torch.Tensor] = None,
                          accumulate: bool = False, errors: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of embedding_lookup with respect to the table: [num_rows, dim] of grad's type, out[v] = scale * (sum of the
    rows of `grad` whose id is v).  grad: ids.shape + (dim,), or one row per id.  The rows of an id are added in their
    order, in float32: the same input gives the same bits.  With `out` the result goes there; accumulate=True adds the sums to what `out` holds
    and leaves its other rows alone (a table that also serves as the output layer).  An id outside of the table is skipped."""
    if isinstance(grad, torch.Tensor) and grad.dim() != 2 and isinstance(ids, torch.Tensor) and tuple(grad.shape[:-1]) == tuple(ids.shape):
        grad = grad.reshape(-1, grad.shape[-1])
    code, device = _matrix("grad", grad), grad.device
    flat = _ids(ids, device)
    n, dim = grad.shape
    if flat.shape[0] != n:
        raise ValueError(f"{flat.shape[0]} ids for {n} rows of grad")
    num_rows = int(num_rows)
    if num_rows < 1:
        raise ValueError("num_rows must be positive")
    if accumulate and out is None:
        raise ValueError("accumulate=True adds to `out`, which is missing")
    if out is None:
        out = grad.new_empty((num_rows, dim))
    else:
        _matrix("out", out, grad.dtype, device)
        if tuple(out.shape) != (num_rows, dim):
            raise ValueError(f"out has shape {tuple(out.shape)}, not {(num_rows, dim)}")
        if num_rows > 1 and out.stride(0) < dim:
            raise ValueError("the rows of out overlap")
        if _overlap(out, grad):
            raise ValueError("out and grad share memory")
        torch.autograd.graph.increment_version(out)
    ws, size = _workspace("pbg_embedding_lookup_grad_workspace", device, n, num_rows, dim)
    _call("pbg_embedding_lookup_grad", device, grad.data_ptr(), _row_stride(grad), flat.data_ptr(), n, num_rows, dim, code, _scale(scale, False),
          out.data_ptr(), _row_stride(out), int(bool(accumulate)), _ptr(ws), size, _error_word(errors, device))
    return out


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, scale: float = 1.0, top: int = 0, ignore_index: int = IGNORE_INDEX,
                   errors: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """Log probabilities of `targets` [n] under softmax(scale * logits) of rows [n, vocab], with each row's entropy, log of the sum,
    the target's rank (scores in front of it: larger ones, and equal ones with a smaller id; 1 = best) and, with top > 0
    (at most 32), the best alternatives in order.  scale is the inverse temperature.  Rows may lie apart (a padded vocabulary).

    A row whose target is ignore_index is padding: it is not read, its results are 0 (top_ids -1).  A row of -inf alone has log
    probabilities -inf and entropy 0; NaN or +inf in a row makes its log probabilities NaN; in the order of `top` NaN counts as -inf."""
    code, device = _matrix("logits", logits), logits.device
    n, vocab = logits.shape
    targets = _vector("targets", targets, torch.long, n, device)
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must lie between 0 and {min(MAX_TOP, vocab)}")
    logprob, entropy, lse, lse_rest = torch.empty((4, n), dtype=torch.float32, device=device).unbind(0)
    rank = torch.empty(n, dtype=torch.long, device=device)
    best = torch.empty((n, top), dtype=torch.float32, device=device) if top else None
    best_ids = torch.empty((n, top), dtype=torch.long, device=device) if top else None
    _call("pbg_token_logprobs_wide", device, logits.data_ptr(), _row_stride(logits), n, vocab, code, targets.data_ptr(), int(ignore_index),
          _scale(scale, True), top, logprob.data_ptr(), entropy.data_ptr(), lse.data_ptr(), lse_rest.data_ptr(), rank.data_ptr(), _ptr(best),
          _ptr(best_ids), _error_word(errors, device))
    result = TokenLogprobs(logprob, entropy, lse, rank, best, best_ids)
    result.lse_rest = lse_rest
    return result


def _row_grads(n, device, lse, entropy, grad_logprob, grad_entropy):
    """The statistics and gradients of a forward call's rows, checked."""
    if grad_logprob is None and grad_entropy is None:
        raise ValueError("neither grad_logprob nor grad_entropy is given")
    lse = _vector("lse", lse, torch.float32, n, device)
    if grad_entropy is not None:
        if entropy is None:
            raise ValueError("the gradient of the entropy needs the entropy")
        grad_entropy = _vector("grad_entropy", grad_entropy, torch.float32, n, device)
        entropy = _vector("entropy", entropy, torch.float32, n, device)
    if grad_logprob is not None:
        grad_logprob = _vector("grad_logprob", grad_logprob, torch.float32, n, device)
    return lse, entropy, grad_logprob, grad_entropy


def _ptr(t):
    return None if t is None else t.data_ptr()


def token_logprobs_grad(logits: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, entropy: Optional[torch.Tensor],
                        grad_logprob: Optional[torch.Tensor], grad_entropy: Optional[torch.Tensor] = None, *, scale: float = 1.0,
                        ignore_index: int = IGNORE_INDEX, out: Optional[torch.Tensor] = None, errors: Optional[torch.Tensor] = None,
                        lse_rest: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient with respect to the logits of sum(grad_logprob * logprob + grad_entropy * entropy), from the lse and the entropy that
    token_logprobs returned (the entropy only where grad_entropy is given).  `out` may be `logits` itself: the gradient then takes the scores'
    place.  Rows of padding, rows whose target is out of range and rows of -inf alone (an lse of -inf) get zeros.

    Probabilities are e^(z - lse - lse_rest).  With the lse_rest of the forward call they are exact wherever the scores lie; without it they
    are off by half a step of lse, relatively (4e-6 for an lse of 64, 2e-3 for 65,000), and cannot be had where lse is beyond 1e6: such
    a row sets 4 in `errors` and gets zeros below -1e6 (a mask of -1e9 that has left nothing) and NaN above 1e6."""
    code, device = _matrix("logits", logits), logits.device
    n, vocab = logits.shape
    targets = _vector("targets", targets, torch.long, n, device)
    lse, entropy, grad_logprob, grad_entropy = _row_grads(n, device, lse, entropy, grad_logprob, grad_entropy)
    if lse_rest is not None:
        lse_rest = _vector("lse_rest", lse_rest, torch.float32, n, device)
    if out is None:
        # rows as far apart as those of the scores, so that both lie alike against 16 bytes
        stride = max(_row_stride(logits), vocab)
        out = torch.empty_strided((n, vocab), (stride if stride < vocab + 4096 else vocab, 1), dtype=logits.dtype, device=device)
    else:
        _matrix("out", out, logits.dtype, device)
        if out.shape != logits.shape:
            raise ValueError(f"out has shape {tuple(out.shape)}, not {tuple(logits.shape)}")
        if n > 1 and out.stride(0) < vocab:
            raise ValueError("the rows of out overlap")
        if _overlap(out, logits) and (out.data_ptr() != logits.data_ptr() or _row_stride(out) != _row_stride(logits)):
            raise ValueError("out shares memory with logits without being them")
        torch.autograd.graph.increment_version(out)
    _call("pbg_token_logprobs_grad_wide", device, logits.data_ptr(), _row_stride(logits), n, vocab, code, targets.data_ptr(), int(ignore_index),
          _scale(scale, True), lse.data_ptr(), _ptr(lse_rest), _ptr(entropy), _ptr(grad_logprob), _ptr(grad_entropy), out.data_ptr(), _row_stride(out),
          _error_word(errors, device))
    return out


class TableLogprobs(NamedTuple):
    """Per query: log probability of its target, entropy, log of the sum of exponentials (float32)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor


def _queries_and_table(queries, table, targets):
    code = _matrix("queries", queries)
    _matrix("table", table, queries.dtype, queries.device)
    if queries.shape[1] != table.shape[1]:
        raise ValueError(f"queries have {queries.shape[1]} elements, the table's rows {table.shape[1]}")
    if table.shape[0] == 0:
        raise ValueError("table has no rows")
    n, dim = queries.shape
    return code, n, table.shape[0], dim, _vector("targets", targets, torch.long, n, queries.device)


def table_logprobs(queries: torch.Tensor, table: torch.Tensor, targets: torch.Tensor, *, scale: float = 1.0, ignore_index: int = IGNORE_INDEX,
                   errors: Optional[torch.Tensor] = None) -> TableLogprobs:
    """Log probabilities of rows `targets` [n] of the table under softmax(scale * queries . table^T), with the entropies and logs of the
    sums; the n x rows scores are never stored.  What token_logprobs(queries @ table.T, targets) gives, at the accuracy of
    float32 sums over the operands as they are (float32 operands are multiplied at 22 bits and more where they reach 2^-17 of the largest
    element of their own row; what other rows hold does not matter).  Queries whose target is ignore_index
    are padding: 0.  NaN or +inf among a query's scores makes its results NaN, -inf is a probability of 0; no other query's results change.
    (An infinite element of more than sixteen float32 queries, or of a row of their table, makes NaN of its scores.)  Scores are float32
    sums: of differences between scores beyond 1e7 nothing is left.  No log probability is above 0."""
    code, n, rows, dim, targets = _queries_and_table(queries, table, targets)
    device = queries.device
    r = TableLogprobs(*torch.empty((3, n), dtype=torch.float32, device=device).unbind(0))
    ws, size = _workspace("pbg_table_logprobs_workspace", device, n, rows, dim, code, 0)
    _call("pbg_table_logprobs", device, queries.data_ptr(), _row_stride(queries), n, table.data_ptr(), _row_stride(table), rows, dim, code, targets.data_ptr(),
          int(ignore_index), _scale(scale, True), r.logprob.data_ptr(), r.entropy.data_ptr(), r.lse.data_ptr(), _ptr(ws), size, _error_word(errors, device))
    return r


def table_logprobs_grad(queries: torch.Tensor, table: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, entropy: Optional[torch.Tensor],
                        grad_logprob: Optional[torch.Tensor], grad_entropy: Optional[torch.Tensor] = None, *, scale: float = 1.0,
                        ignore_index: int = IGNORE_INDEX, errors: Optional[torch.Tensor] = None, rounded: bool = False):
    """Gradients (of the queries, of the table) of sum(grad_logprob * logprob + grad_entropy * entropy), from the lse and the entropy that
    table_logprobs returned (the entropy only where grad_entropy is given).  Queries that are padding, and those whose
    target is out of range, get zeros and add nothing to the table's gradient, whatever they hold -- unless the table holds NaN or
    infinities, which reach all gradients of the queries.

    16-bit operands: the gradient of the scores keeps 16 bits or more on its way into the two products.  rounded=True rounds it to the
    operands' type above 128 queries, as training in 16 bits commonly does: a third less time, bf16 results 2.3e-3 off instead of the 1.7e-3
    of their own rounding (more where all rows of the table have much in common)."""
    code, n, rows, dim, targets = _queries_and_table(queries, table, targets)
    device = queries.device
    lse, entropy, grad_logprob, grad_entropy = _row_grads(n, device, lse, entropy, grad_logprob, grad_entropy)
    dq = torch.empty((n, dim), dtype=queries.dtype, device=device)
    dt = torch.empty((rows, dim), dtype=table.dtype, device=device)
    ws, size = _workspace("pbg_table_logprobs_workspace", device, n, rows, dim, code, 2 if rounded else 1)
    _call("pbg_table_logprobs_grad_rounded" if rounded else "pbg_table_logprobs_grad", device, queries.data_ptr(), _row_stride(queries), n,
          table.data_ptr(), _row_stride(table), rows, dim, code, targets.data_ptr(), int(ignore_index), _scale(scale, True),
          lse.data_ptr(), _ptr(entropy), _ptr(grad_logprob), _ptr(grad_entropy), dq.data_ptr(), dt.data_ptr(),
          _ptr(ws), size, _error_word(errors, device))
    return dq, dt

"""The loss that an encoder is trained with against every row: softmax cross entropy whose scores are not kept, and its gradient.

``log_probs`` and ``log_probs_backward`` work on scores that are there: of candidate lists, or of a matrix of every row.  Of thousands of queries against a million
rows that matrix would be gigabytes; here it is made piece by piece and used up at once, forward and backward.

    result = culsh.cross_entropy(Q, X, targets, temperature=0.05)          # Q: [m, d], X: [n, d], targets: [m] rows of X
    loss = result.losses.mean()
    grad_Q, grad_X = culsh.cross_entropy_backward(Q, X, targets, result, torch.full_like(result.losses, 1 / m), temperature=0.05)

Results are torch tensors on the device of the queries; calls run on torch's current stream and return when their work is queued.  They are not part of autograd's
graph.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._culsh_core import get_handle
from .ranking import _SCORE_TYPES, _TYPES, _floats, _matrix, _pitch, _stream, _targets, _temperature

MAX_FEATURES = 1 << 16


class CrossEntropy(NamedTuple):
    """What ``cross_entropy`` returns, float32; an entry is a query."""
    losses: torch.Tensor   # [m] lse - score of the target: 0 where the target is not one of the rows, inf where it is masked
    lse: torch.Tensor      # [m] log of the sum of exp(scores); -inf where the bias leaves no row
    lse_low: torch.Tensor  # [m] what lse leaves behind its last bit

    def check(self) -> None:
        """Waits for the current stream; raises if a product of this thread's losses or gradients had to give up a wait (what it should have made is NaN)."""
        h = get_handle(self.losses.device.index)
        _lib.check(h.lib.culsh_mx_product_check(h.ptr, _stream(self.losses.device)))


def _sides(Q, X, bias):
    Q = _matrix(Q)
    X = _matrix(X, Q.device)
    if Q.dtype not in _SCORE_TYPES:
        raise TypeError(f"Unsupported dtype: {Q.dtype}. Supported dtypes are float32, float16, bfloat16.")
    if X.dtype != Q.dtype:
        raise TypeError(f"queries are {Q.dtype}, rows {X.dtype}")
    if X.shape[1] != Q.shape[1]:
        raise ValueError(f"Query features ({Q.shape[1]}) != row features ({X.shape[1]})")
    if not 0 < Q.shape[1] <= MAX_FEATURES:
        raise ValueError(f"features must be between 1 and {MAX_FEATURES}")
    if X.shape[0] == 0:
        raise ValueError("there are no rows")
    return Q, X, None if bias is None else _floats(bias, "bias", (X.shape[0],), Q.device)


@functools.lru_cache(maxsize=256)
def _workspace_size(device, q_at, q_pitch, x_at, x_pitch, dtype, m, n, d, has_bias, gradients):
    """A workspace's size goes by sizes and alignments alone: the addresses are what they leave by 16, and 16."""
    h, need = get_handle(device), C.c_uint64()
    _lib.check(h.lib.culsh_cross_entropy_workspace(h.ptr, q_at + 16, q_pitch, x_at + 16, x_pitch, _TYPES[dtype], m, n, d, has_bias, gradients, C.byref(need)))
    return need.value


def _workspace(Q, X, m, n, d, bias, gradients):
    device = Q.device
    size = _workspace_size(device.index, Q.data_ptr() & 15, _pitch(Q), X.data_ptr() & 15, _pitch(X), Q.dtype, m, n, d, bias is not None, gradients)
    return torch.empty(size, dtype=torch.uint8, device=device), size


def cross_entropy(Q, X, targets, bias=None, temperature: float = 1.0) -> CrossEntropy:
    """Softmax cross entropy of queries over every row: with scores z[i, j] = Q[i] . X[j] / temperature + bias[j], losses logsumexp(z[i]) - z[i, targets[i]].

    ``Q``: [m, d], ``X``: [n, d], both float32, float16 or bfloat16.  ``targets``: [m] int64 or int32; one that is not in 0 .. n - 1 has no loss.  ``bias``: [n] float32, e.g.
    the log of how often a row is drawn, taken off; -inf takes a row out."""
    _temperature(temperature)
    Q, X, bias = _sides(Q, X, bias)
    m, device = int(Q.shape[0]), Q.device
    targets = _targets(targets, None, m, device)
    if targets is None:
        raise ValueError("losses need targets")
    out = torch.empty((3, m), dtype=torch.float32, device=device)
    result = CrossEntropy(*out.unbind())
    if m:
        h = get_handle(device.index)
        work, size = _workspace(Q, X, m, int(X.shape[0]), int(Q.shape[1]), bias, 0)
        at = out.data_ptr()
        _lib.check(h.lib.culsh_cross_entropy(h.ptr, Q.data_ptr(), _pitch(Q), X.data_ptr(), _pitch(X), _TYPES[Q.dtype], m, X.shape[0], Q.shape[1], targets.data_ptr(),
                                             None if bias is None else bias.data_ptr(), float(temperature), at, at + 4 * m, at + 8 * m, work.data_ptr(), size,
                                             _stream(device)))
    return result


def cross_entropy_backward(Q, X, targets, result: CrossEntropy, grad_losses=None, grad_lse=None, bias=None, temperature: float = 1.0, queries: bool = True,
                           rows: bool = True) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients with respect to Q and X, in their type, from those of the losses and of lse (e.g. of a penalty on its square), [m] float32, and the result of
    ``cross_entropy`` for the same arguments.  None in the place of one that is not wanted (``queries``, ``rows``).  A target that is not in 0 .. n - 1, or is masked, has no
    loss to go by.  The bias is taken as a constant: one that is learned is a column of X beside a column of ones in Q.  In half precision, gradients below 6e-8 are 0: scale the
    losses' up, as is usual."""
    _temperature(temperature)
    Q, X, bias = _sides(Q, X, bias)
    m, n, d, device = int(Q.shape[0]), int(X.shape[0]), int(Q.shape[1]), Q.device
    targets = _targets(targets, None, m, device)
    if targets is None and grad_losses is not None:
        raise ValueError("the gradient of losses needs their targets")
    losses, lse, low = (_floats(x, name, (m,), device) for x, name in zip(result, ("losses", "lse", "lse_low")))
    g = None if grad_losses is None else _floats(grad_losses, "grad_losses", (m,), device)
    e = None if grad_lse is None else _floats(grad_lse, "grad_lse", (m,), device)
    grad_Q = torch.empty((m, d), dtype=Q.dtype, device=device) if queries else None
    grad_X = torch.empty((n, d), dtype=Q.dtype, device=device) if rows else None
    if m == 0:
        return grad_Q, None if grad_X is None else grad_X.zero_()
    if queries or rows:
        h = get_handle(device.index)
        work, size = _workspace(Q, X, m, n, d, bias, bool(queries) + 2 * bool(rows))
        _lib.check(h.lib.culsh_cross_entropy_backward(
            h.ptr, Q.data_ptr(), _pitch(Q), X.data_ptr(), _pitch(X), _TYPES[Q.dtype], m, n, d, None if targets is None else targets.data_ptr(),
            None if bias is None else bias.data_ptr(), float(temperature), losses.data_ptr(), lse.data_ptr(), low.data_ptr(), None if g is None else g.data_ptr(),
            None if e is None else e.data_ptr(), grad_Q.data_ptr() if queries else None, d, grad_X.data_ptr() if rows else None, d, work.data_ptr(), size,
            _stream(device)))
    return grad_Q, grad_X

"""Ranking of candidates: rows held in 4 bits, their scores against queries, and log probabilities over scores.

``query`` answers with the ids of candidate rows, not ranked.  Here the rows are kept in microscaled 4-bit floating point
(``MXRows``: 17 bytes for 32 values), queries are scored against their candidates (``MXRows.score``) or against every
row (``MXRows.product``), and ``log_probs`` turns scores into what an answer needs: the most likely rows, their log
probabilities, and the entropy of the distribution; ``log_probs_backward`` is its gradient, for training an encoder on candidate lists.

    rows = culsh.MXRows(X)
    candidates = model.query(Q)
    best = culsh.rank(rows, Q, candidates, top_k=10, metric="cosine", temperature=0.05)
    best.top_ids, best.top_log_probs, best.entropy

Results are torch tensors on the device of the rows.  Unlike the index's calls these run on torch's current stream and
return when their work is queued.  In a graph, keep the Candidates that it reads.  Results are not part of autograd's graph: gradients come
from ``log_probs_backward``.  Pairs (ids, offsets) have offsets from 0 to the number of ids.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple, Union

import numpy as np
import torch

from . import _lib
from ._culsh_core import Candidates, get_handle

METRICS = {"dot": 0, "cosine": 1, "euclidean": 2}
_TYPES = {torch.float32: 0, torch.float64: 1, torch.float16: 2, torch.bfloat16: 3}
_SCORE_TYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_TOP_K = 128


def _on_device(x, device=None) -> torch.Tensor:
    """A CUDA tensor of a torch, CuPy or NumPy array, without a copy where it is on a device already."""
    if not isinstance(x, torch.Tensor):
        x = torch.as_tensor(x, device="cuda") if hasattr(x, "__cuda_array_interface__") else torch.from_numpy(np.ascontiguousarray(x))
    if not x.is_cuda:
        return x.to("cuda" if device is None else device)
    if device is not None and x.device != device:
        raise ValueError(f"arrays are on {x.device} and {device}")
    return x


def _matrix(x, device=None) -> torch.Tensor:
    """A 2-D CUDA tensor whose rows have no gaps inside and do not overlap."""
    if not (isinstance(x, torch.Tensor) and x.is_cuda and (device is None or x.device == device)):
        x = _on_device(x, device)
    if x.ndim != 2:
        raise ValueError(f"Expected 2D array, got {x.ndim}D")
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x


def _pitch(x: torch.Tensor) -> int:
    return int(x.stride(0)) if x.shape[0] > 1 else max(int(x.shape[1]), 1)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # without a Stream object, whose making costs as much as an allocation


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device.index)


def _metric(name: str) -> int:
    if name not in METRICS:
        raise ValueError(f"metric must be one of {tuple(METRICS)}")
    return METRICS[name]


def _floats(x, name, shape, device) -> torch.Tensor:
    if not (isinstance(x, torch.Tensor) and x.device == device):
        x = _on_device(x, device)
    if x.shape != shape:
        raise ValueError(f"{name} must have the shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {x.dtype}")
    return x if x.is_contiguous() else x.contiguous()


class _Lists:
    """Candidate lists as device addresses: a Candidates object, or a pair (ids, offsets)."""

    def __init__(self, lists, device, need_ids=True):
        self.result, self.device = None, device
        if isinstance(lists, Candidates):
            if lists._h.device != device.index:
                raise ValueError(f"candidates are on cuda:{lists._h.device}, not on {device}")
            self.n, self.total = lists.n_queries, 0 if lists.empty() else lists.n_total_candidates
            if not lists.empty():
                self.result = lists
                self.ids, _, self.offsets = lists.device_pointers()
            else:
                self.keep = torch.zeros(self.n + 1, dtype=torch.int64, device=device)
                self.ids, self.offsets = 0, self.keep.data_ptr()
        else:
            ids, offsets = lists
            offsets = _on_device(offsets, device)
            if offsets.dtype not in (torch.int64, torch.uint64) or offsets.ndim != 1 or offsets.shape[0] < 1:
                raise TypeError("offsets must be a 1D int64 or uint64 array with one entry more than there are lists")
            offsets = offsets.contiguous()
            if ids is None:
                if need_ids:
                    raise ValueError("lists need ids")
                self.total = None
            else:
                ids = _on_device(ids, device)
                if ids.dtype != torch.int32 or ids.ndim != 1:
                    raise TypeError("ids must be a 1D int32 array")
                ids = ids.contiguous()
                self.total = int(ids.shape[0])
            self.n = int(offsets.shape[0]) - 1
            self.ids, self.offsets = 0 if ids is None else ids.data_ptr(), offsets.data_ptr()
            self.keep = (ids, offsets)
        if not self.ids and (self.result is not None or self.total == 0):
            self.ids = self.offsets  # no list has an entry: nothing is read through it

    def done(self, handle, stream):
        """The device arrays of a Candidates object may go as soon as it does: its handle waits for what has been queued (not for a graph that is being
        captured, whose candidates have to stay as long as it does)."""
        if self.result is not None:
            _lib.check(handle.lib.culsh_candidates_after(handle.ptr, self.result._ptr, stream))
            if getattr(self.result, "_keepalive", None) is not None:  # a receive buffer that other processes write
                torch.cuda.current_stream(self.device).synchronize()


class MXRows:
    """Rows in microscaled 4-bit floating point: blocks of 32 values share a power of two, a value is one of
    +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times it.

    ``X``: 2-D, float32, float64, float16 or bfloat16.  A block with a NaN or an infinity becomes NaN."""

    def __init__(self, X):
        X = _matrix(X)
        if X.dtype not in _TYPES:
            raise TypeError(f"Unsupported dtype: {X.dtype}. Supported dtypes are float32, float64, float16, bfloat16.")
        n, d = int(X.shape[0]), int(X.shape[1])
        if d == 0:
            raise ValueError("rows have no features")
        self._n, self._d, self._h = n, d, get_handle(X.device.index)
        groups = -(-d // 128)
        # codes and scales in one allocation; the tensors that show them are made when they are asked for
        self._codes = self._scales = None
        self._held = torch.empty(64 * groups * n + 512 * groups * -(-n // 128), dtype=torch.uint8, device=X.device)
        self.norms = torch.empty(n, dtype=torch.float32, device=X.device)
        at = self._held.data_ptr()
        self._at = (at, at + 64 * groups * n, self.norms.data_ptr())
        if n:
            h = self._h
            _lib.check(h.lib.culsh_mx_quantize(h.ptr, X.data_ptr(), _TYPES[X.dtype], n, d, _pitch(X), *self._at, _stream(X.device)))

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scales: torch.Tensor, norms: torch.Tensor, n_features: int) -> "MXRows":
        """Rows from the arrays of another MXRows, e.g. loaded from a file: ``codes`` [n, 64 G] (two to a byte, the first in the
        low half, zeros behind the row's end) with G = ceil(n_features / 128), ``scales`` [ceil(n / 128), G, 32, 4, 4] (127 + exponent of block 4 g + b
        of row 128 t + 32 j + i at [t, g, i, j, b]), ``norms`` [n] float32 (squared lengths, 0 for rows of zeros alone)."""
        d = int(n_features)
        if d <= 0:
            raise ValueError("n_features must be positive")
        if codes.ndim != 2 or codes.dtype != torch.uint8 or codes.shape[1] != 64 * -(-d // 128):
            raise ValueError(f"codes must be uint8 of the shape [n, {64 * -(-d // 128)}]")
        n = int(codes.shape[0])
        if scales.dtype != torch.uint8 or tuple(scales.shape) != (-(-n // 128), -(-d // 128), 32, 4, 4):
            raise ValueError(f"scales must be uint8 of the shape {(-(-n // 128), -(-d // 128), 32, 4, 4)}")
        if norms.dtype != torch.float32 or tuple(norms.shape) != (n,):
            raise ValueError(f"norms must be float32 of the shape {(n,)}")
        if not (codes.is_cuda and codes.device == scales.device == norms.device):
            raise ValueError("codes, scales and norms must be on one CUDA device")
        self = cls.__new__(cls)
        self._n, self._d, self._h = n, d, get_handle(codes.device.index)
        self._codes, self._scales, self.norms = codes.contiguous(), scales.contiguous(), norms.contiguous()
        self._at = (self._codes.data_ptr(), self._scales.data_ptr(), self.norms.data_ptr())
        return self

    n_rows = property(lambda self: self._n)
    n_features = property(lambda self: self._d)
    device = property(lambda self: self.norms.device)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._held[:64 * -(-self._d // 128) * self._n].view(self._n, -1) if self._n else self._held.view(0, 64 * -(-self._d // 128))
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            groups = -(-self._d // 128)
            self._scales = self._held[64 * groups * self._n:].view(-(-self._n // 128), groups, 32, 4, 4)
        return self._scales

    def size_bytes(self) -> int:
        return self.codes.numel() + self.scales.numel() + 4 * self.norms.numel()

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that are held, [n_rows, n_features]."""
        if dtype not in _TYPES:
            raise TypeError(f"Unsupported dtype: {dtype}. Supported dtypes are float32, float64, float16, bfloat16.")
        out = torch.empty((self._n, self._d), dtype=dtype, device=self.device)
        if self._n:
            _lib.check(self._h.lib.culsh_mx_dequantize(self._h.ptr, self._at[0], self._at[1], self._n, self._d, out.data_ptr(), _TYPES[dtype],
                                                       _stream(self.device)))
        return out

    def product(self, Q, metric: str = "dot", dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Scores [n_queries, n_rows] of queries against every row: dot products, cosines or negative squared
        distances ("euclidean").  Cosines with a row of zeros are 0, with lengths outside of 1.1e-19 to 1.8e19 NaN.  ``Q``: MXRows, or an array that is held in 4 bits for the call.  Rows of many scores begin at multiples of
        128 bytes, so that the result of an odd number of rows is not contiguous."""
        m = _metric(metric)
        if dtype not in _SCORE_TYPES:
            raise TypeError(f"Unsupported dtype: {dtype}. Supported dtypes are float32, float16, bfloat16.")
        device = self.device
        held = isinstance(Q, MXRows)
        if held:
            if Q.device != device:
                raise ValueError(f"queries are on {Q.device}, rows on {device}")
            nq, d = Q._n, Q._d
        else:
            Q = _matrix(Q, device)
            if Q.dtype not in _TYPES:
                raise TypeError(f"Unsupported dtype: {Q.dtype}. Supported dtypes are float32, float64, float16, bfloat16.")
            nq, d = Q.shape
        if d != self._d:
            raise ValueError(f"Query features ({d}) != row features ({self._d})")
        n = self._n
        # rows that share their first and last 32 bytes with others take the memory twice as long (1,000 x 999,999 float32 scores 2,036 us against 792)
        line = 128 // dtype.itemsize
        pitch = n if n < 8 * line else -(-n // line) * line
        out = torch.empty((nq, pitch), dtype=dtype, device=device)
        if pitch != n:
            out = out[:, :n]
        if n and nq:
            h, stream = self._h, _stream(device)
            if held:
                _lib.check(h.lib.culsh_mx_product(h.ptr, *Q._at, nq, *self._at, n, d, m, out.data_ptr(), _TYPES[dtype], pitch, stream))
            else:
                groups = -(-d // 128)
                need = 64 * groups * nq + 512 * groups * -(-nq // 128) + 4 * nq
                work = torch.empty(need, dtype=torch.uint8, device=device)
                _lib.check(h.lib.culsh_mx_product_dense(h.ptr, Q.data_ptr(), _TYPES[Q.dtype], nq, _pitch(Q), *self._at, n, d, m, out.data_ptr(),
                                                        _TYPES[dtype], pitch, work.data_ptr(), need, stream))
        return out

    def check(self) -> None:
        """Waits for the current stream; raises if a product or scores had to give up a wait (and are NaN in part)."""
        _lib.check(self._h.lib.culsh_mx_product_check(self._h.ptr, _stream(self.device)))

    def score(self, Q, candidates: Union[Candidates, Tuple], metric: str = "dot") -> torch.Tensor:
        """Scores of queries against their candidates, float32, in the order of the candidates' ids.  ``Q`` (float32,
        float64, float16 or bfloat16) is taken in 32 bits, not in 4.  ``candidates``: what ``query`` returned for Q, or a pair (ids, offsets) of int32 and int64.
        A candidate that is no row gets NaN, and so do all of a query that has an infinity or a NaN, and scores whose sums pass float32; cosines as in
        ``product``."""
        m = _metric(metric)
        Q = _matrix(Q, self.device)
        if Q.dtype not in _TYPES:
            raise TypeError(f"Unsupported dtype: {Q.dtype}. Supported dtypes are float32, float64, float16, bfloat16.")
        if Q.shape[1] != self._d:
            raise ValueError(f"Query features ({Q.shape[1]}) != row features ({self._d})")
        lists = _Lists(candidates, self.device)
        if lists.n != Q.shape[0]:
            raise ValueError(f"{Q.shape[0]} queries, but {lists.n} lists")
        out = torch.empty(lists.total, dtype=torch.float32, device=self.device)
        if lists.total:
            if not self._n:
                return out.fill_(float("nan"))
            h, stream = self._h, _stream(self.device)
            need = C.c_uint64()
            _lib.check(h.lib.culsh_mx_score_workspace(h.ptr, lists.n, self._d, lists.total, C.byref(need)))
            work = torch.empty(need.value, dtype=torch.uint8, device=self.device) if need.value else None
            _lib.check(h.lib.culsh_mx_score(
                h.ptr, Q.data_ptr(), _TYPES[Q.dtype], lists.n, _pitch(Q), *self._at, self._n, self._d, m, lists.ids, lists.offsets, lists.total,
                out.data_ptr(), work.data_ptr() if need.value else None, need.value, stream))
            lists.done(h, stream)
        return out


class LogProbs(NamedTuple):
    """What ``log_probs`` returns; a row is a query.  ``log_probs`` is None without targets, the last two without ``top_k``."""
    log_probs: Optional[torch.Tensor]      # [m] of the given entry; -inf where the row has none such
    entropy: torch.Tensor                  # [m] in nats
    lse: torch.Tensor                      # [m] log of the sum of exp(scores / temperature)
    top_log_probs: Optional[torch.Tensor]  # [m, k], the largest first; -inf behind the last one
    top_ids: Optional[torch.Tensor]        # [m, k] int32 columns, or ids of the lists; -1 behind the last one


def _scores(scores, lists):
    """(scores, lists, rows, columns, pitch) of a matrix, or of lists."""
    if lists is None:
        scores = _matrix(scores)
        m, cols, pitch = int(scores.shape[0]), int(scores.shape[1]), _pitch(scores)
    else:
        scores = _on_device(scores)
        if scores.ndim != 1:
            raise ValueError(f"scores of lists are 1D, got {scores.ndim}D")
        scores = scores.contiguous()
        lists = _Lists(lists, scores.device, need_ids=False)
        if lists.total is None:
            lists.total = int(scores.shape[0])
        if lists.total != scores.shape[0]:
            raise ValueError(f"{scores.shape[0]} scores, but {lists.total} candidates")
        m, cols, pitch = lists.n, 0, 0
    if scores.dtype not in _SCORE_TYPES:
        raise TypeError(f"Unsupported dtype: {scores.dtype}. Supported dtypes are float32, float16, bfloat16.")
    return scores, lists, m, cols, pitch


def _targets(targets, lists, m, device):
    if targets is None:
        return None
    if not (isinstance(targets, torch.Tensor) and targets.device == device):
        targets = _on_device(targets, device)
    if targets.shape != (m,) or targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets must be int64 or int32 of the shape {(m,)}, got {targets.dtype} {tuple(targets.shape)}")
    if lists is not None and not lists.ids:
        raise ValueError("targets of lists need the lists' ids")
    return targets if targets.dtype == torch.int64 and targets.is_contiguous() else targets.to(torch.int64).contiguous()


def _temperature(temperature):
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError("temperature must be positive")
    if temperature < 4.3e-39:  # below, log2(e) by it is no float
        raise ValueError("temperature is too small")


def log_probs(scores, targets=None, lists: Union[Candidates, Tuple, None] = None, top_k: int = 0, temperature: float = 1.0) -> LogProbs:
    """Log probabilities under softmax(scores / temperature): of given entries, with the entropy and the most likely ones.

    ``scores``: [m, n] (``MXRows.product``), or the scores of candidate lists (``MXRows.score``) with ``lists`` the Candidates or a pair
    (ids or None, offsets); float32, float16 or bfloat16; -inf takes an entry out.
    ``targets``: [m] columns, or ids of the lists, each of which may stand in any order and holds an id once.  ``top_k``: at most 128; of equal scores the first one goes first."""
    top_k = int(top_k)
    if not 0 <= top_k <= MAX_TOP_K:
        raise ValueError(f"top_k must be between 0 and {MAX_TOP_K}")
    _temperature(temperature)
    scores, lists, m, cols, pitch = _scores(scores, lists)
    device = scores.device
    targets = _targets(targets, lists, m, device)
    few = torch.empty((3, m), dtype=torch.float32, device=device)
    top, ids = None, None
    if top_k:
        top = torch.empty((m, top_k), dtype=torch.float32, device=device)
        ids = torch.empty((m, top_k), dtype=torch.int32, device=device)
    log_p, entropy, lse = few.unbind()
    result = LogProbs(log_p if targets is not None else None, entropy, lse, top, ids)
    if m == 0:
        return result
    if lists is None and cols == 0:  # rows of nothing
        few.fill_(-float("inf"))
        few[1].zero_()
        if top_k:
            top.fill_(-float("inf"))
            ids.fill_(-1)
        return result
    h, stream = get_handle(device.index), _stream(device)
    total = 0 if lists is None else lists.total
    need, work = C.c_uint64(), None
    if max(cols, total // m) > 16384:  # rows that are shorter on average need none
        _lib.check(h.lib.culsh_log_probs_workspace(h.ptr, _TYPES[scores.dtype], m, cols, lists is not None, total, C.byref(need)))
        if need.value:
            work = torch.empty(need.value, dtype=torch.uint8, device=device)
    at = few.data_ptr()
    _lib.check(h.lib.culsh_log_probs(
        h.ptr, scores.data_ptr(), _TYPES[scores.dtype], m, cols, pitch, lists.offsets if lists else None, (lists.ids or None) if lists else None,
        total, float(temperature), targets.data_ptr() if targets is not None else None, top_k, at, at + 4 * m, at + 8 * m,
        top.data_ptr() if top_k else None, ids.data_ptr() if top_k else None, work.data_ptr() if work is not None else None, need.value, stream))
    if lists is not None:
        lists.done(h, stream)
    return result


def log_probs_backward(scores, targets, lse, entropy, grad_log_probs=None, grad_entropy=None, lists: Union[Candidates, Tuple, None] = None,
                       temperature: float = 1.0) -> torch.Tensor:
    """Gradient with respect to ``scores``, in their type, from the gradients of the log probabilities and of the entropies of
    ``log_probs(scores, targets, lists, temperature=temperature)``, whose ``lse`` and ``entropy`` it takes.  A target that is not in
    its row, or is masked with -inf, has no gradient."""
    _temperature(temperature)
    scores, lists, m, cols, pitch = _scores(scores, lists)
    device = scores.device
    if grad_log_probs is not None and targets is None:
        raise ValueError("the gradient of log probabilities needs their targets")
    targets = _targets(targets, lists, m, device)
    lse, entropy = _floats(lse, "lse", (m,), device), _floats(entropy, "entropy", (m,), device)
    g = None if grad_log_probs is None else _floats(grad_log_probs, "grad_log_probs", (m,), device)
    e = None if grad_entropy is None else _floats(grad_entropy, "grad_entropy", (m,), device)
    out = torch.empty(scores.shape, dtype=scores.dtype, device=device)
    if out.numel() == 0:
        return out
    h, stream = get_handle(device.index), _stream(device)
    _lib.check(h.lib.culsh_log_probs_backward(
        h.ptr, scores.data_ptr(), _TYPES[scores.dtype], m, cols, pitch, lists.offsets if lists else None, (lists.ids or None) if lists else None,
        lists.total if lists else 0, float(temperature), targets.data_ptr() if targets is not None else None, lse.data_ptr(), entropy.data_ptr(),
        g.data_ptr() if g is not None else None, e.data_ptr() if e is not None else None, out.data_ptr(), cols, stream))
    if lists is not None:
        lists.done(h, stream)
    return out


def rank(rows: MXRows, Q, candidates: Union[Candidates, Tuple, None] = None, top_k: int = 10, metric: str = "dot", temperature: float = 1.0,
         targets=None) -> LogProbs:
    """The ``top_k`` best rows of each query with their log probabilities: among its candidates, or among all rows without any."""
    if candidates is None:
        return log_probs(rows.product(Q, metric=metric), targets, top_k=top_k, temperature=temperature)
    return log_probs(rows.score(Q, candidates, metric=metric), targets, candidates, top_k=top_k, temperature=temperature)

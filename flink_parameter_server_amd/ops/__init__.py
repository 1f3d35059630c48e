"""Device-op dispatch.

CPU tensors -> plain-PyTorch fp32 reference (``ops.reference``), which is
also the semantics oracle for the kernels.
CUDA (= ROCm/MI355X) tensors -> hand-written HIP/CDNA4 kernels from the
in-tree extension; a missing extension raises (never a silent fallback).
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional, Sequence, Tuple

import torch

from . import reference
from . import hip

__all__ = [
    "gather", "apply_add", "apply_adagrad", "hash_init",
    "mf_sgd_step", "pa_step", "pa_multiclass_step", "lr_step", "sgns_step",
    "record_bytes", "row_cache", "cache_write", "cache_read",
    "MUON_COEFFS", "orthogonalize", "apply_muon",
    "reference", "hip",
]


def _cuda(t: torch.Tensor) -> bool:
    return t.is_cuda


def gather(table: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
    if _cuda(table):
        return hip.ext().gather(table, rows)
    return reference.gather(table, rows)


def apply_add(table: torch.Tensor, rows: torch.Tensor,
              deltas: torch.Tensor, unique: bool = False) -> None:
    if _cuda(table):
        hip.ext().apply_add(table, rows, deltas, unique)
        return
    reference.apply_add(table, rows, deltas, unique)


def apply_adagrad(table: torch.Tensor, accum: torch.Tensor,
                  rows: torch.Tensor, grads: torch.Tensor,
                  lr: float, eps: float = 1e-8,
                  sorted_unique: bool = False) -> None:
    """``sorted_unique``: the caller guarantees ``rows`` ascending with no
    duplicates (our model logics push per sorted unique pulled id), so
    the pre-sort is skipped."""
    if _cuda(table):
        # K2 contract: duplicates pre-aggregated, one RMW per distinct
        # row.  Sort the batch (device radix sort) and let segment
        # leaders aggregate in-kernel.
        if sorted_unique:
            hip.ext().apply_adagrad_sorted(table, accum,
                                           rows.contiguous(),
                                           grads.contiguous(), lr, eps)
            return
        srows, order = torch.sort(rows)
        hip.ext().apply_adagrad_sorted(table, accum, srows.contiguous(),
                                       grads.index_select(0, order)
                                       .contiguous(), lr, eps)
        return
    reference.apply_adagrad(table, accum, rows, grads, lr, eps)


def hash_init(ids: torch.Tensor, dim: int, lo: float, hi: float,
              seed: int = 0) -> torch.Tensor:
    if _cuda(ids):
        return hip.ext().hash_init(ids, dim, lo, hi, seed)
    return reference.hash_init(ids, dim, lo, hi, seed)


def hash_init_rows(out: torch.Tensor, first_id: int, stride: int,
                   lo: float, hi: float, seed: int = 0) -> None:
    """Initialize a whole dense shard slab in place: row r of ``out`` is the
    deterministic init vector of global id ``first_id + r * stride``.
    Device path runs one kernel over the slab; CPU path materializes ids.
    """
    if _cuda(out):
        hip.ext().hash_init_rows(out, first_id, stride, lo, hi, seed)
        return
    ids = torch.arange(out.shape[0], dtype=torch.int64) * stride + first_id
    out.copy_(reference.hash_init(ids, out.shape[1], lo, hi, seed))


def mf_sgd_step(user_table: torch.Tensor, user_rows: torch.Tensor,
                item_vecs: torch.Tensor, item_slots: torch.Tensor,
                ratings: torch.Tensor, lr: float, reg: float = 0.0,
                reuse_tag: int = 0,
                mean_users: bool = False) -> torch.Tensor:
    """``reuse_tag != 0`` promises that whenever the same (tag,
    user_rows buffer, item_slots buffer) recur, their CONTENT is
    unchanged (epoch resweeps over resident batches) — the HIP path then
    reuses the cached sort positions instead of re-sorting, and caches
    both sorted record arrays outright (zero per-visit scatter rebuilds)
    when additionally the SAME ratings buffer recurs with unchanged
    content; a different ratings buffer safely re-scatters only the
    first-pass records."""
    if _cuda(user_table):
        return hip.ext().mf_sgd_step(user_table, user_rows, item_vecs,
                                     item_slots, ratings, lr, reg,
                                     reuse_tag, mean_users)
    # torch index ops need int64; the HIP path takes int32 directly
    return reference.mf_sgd_step(user_table, user_rows.long(), item_vecs,
                                 item_slots.long(), ratings, lr, reg,
                                 mean_users=mean_users)


def pa_step(indptr: torch.Tensor, feat_slots: torch.Tensor,
            x_vals: torch.Tensor, labels: torch.Tensor,
            weights: torch.Tensor, variant: str = "PA-I", C: float = 1.0
            ) -> Tuple[torch.Tensor, torch.Tensor]:
    if _cuda(weights):
        return hip.ext().pa_step(indptr, feat_slots, x_vals, labels,
                                 weights, variant, C)
    return reference.pa_step(indptr, feat_slots, x_vals, labels, weights,
                             variant, C)


def pa_multiclass_step(indptr: torch.Tensor, feat_slots: torch.Tensor,
                       x_vals: torch.Tensor, labels: torch.Tensor,
                       weights: torch.Tensor, variant: str = "PA-I",
                       C: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    if _cuda(weights):
        return hip.ext().pa_multiclass_step(indptr, feat_slots, x_vals,
                                            labels, weights, variant, C)
    return reference.pa_multiclass_step(indptr, feat_slots, x_vals, labels,
                                        weights, variant, C)


def lr_step(indptr: torch.Tensor, feat_slots: torch.Tensor,
            x_vals: torch.Tensor, labels: torch.Tensor,
            weights: torch.Tensor, reuse_tag: int = 0
            ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``reuse_tag != 0`` promises the same (tag, feat_slots buffer,
    x_vals buffer) recur with unchanged content (epoch resweeps); the
    HIP path then runs the slot-sorted record walk with the records and
    per-instance norms cached per batch — the per-element gather/
    scatter form (random 4-B line traffic) leaves the steady round."""
    if _cuda(weights):
        return hip.ext().lr_step(indptr, feat_slots, x_vals, labels,
                                 weights, reuse_tag)
    return reference.lr_step(indptr, feat_slots.long(), x_vals, labels,
                             weights)


def sgns_step(vecs: torch.Tensor, center_slots: torch.Tensor,
              ctx_slots: torch.Tensor, labels: torch.Tensor, lr: float
              ) -> torch.Tensor:
    """Fused SGNS step over one shared row buffer (center and context
    slots index disjoint rows); returns the combined deltas buffer."""
    if _cuda(vecs):
        return hip.ext().sgns_step(vecs, center_slots, ctx_slots, labels,
                                   lr)
    return reference.sgns_step(vecs, center_slots.long(),
                               ctx_slots.long(), labels, lr)


# ---------------------------------------------------------------------------
# 8-bit row records
# ---------------------------------------------------------------------------

_VALUE_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def record_bytes(dim: int) -> int:
    """Bytes of one record of a row of ``dim`` values: the codes, zeros to a
    multiple of 4, the f32 scale."""
    return (int(dim) + 3) // 4 * 4 + 4


def row_cache(rows: int, dim: int,
              device: Optional[torch.device] = None) -> torch.Tensor:
    """An empty cache of ``rows`` records (uint8, ``(rows,
    record_bytes(dim))``); a record that nothing was written to reads back
    as zeros."""
    if int(rows) < 0 or int(dim) < 1:
        raise ValueError(f"row_cache: rows >= 0 and dim >= 1, got "
                         f"{rows} and {dim}")
    return torch.zeros(int(rows), record_bytes(dim), dtype=torch.uint8,
                       device=device)


def cache_write(cache: torch.Tensor, values: torch.Tensor,
                slots: Optional[torch.Tensor] = None, fmt: str = "int8",
                unique: bool = False) -> None:
    """Quantise the rows of ``values`` (n, dim; f32, bf16 or f16) into
    records of ``cache`` in place: row j goes to ``slots[j]``, or to record j
    without ``slots`` (then n is the cache's length).

    ``fmt="int8"``: scale = amax / 127, equal steps; ``"fp8"``: e4m3 under a
    power-of-two scale, a relative error of at most 2^-4 a value down to
    1 / 14336 of the row's largest (for rows whose largest is 2^-118 or
    more; smaller ones have a scale of 2^-126).  A row with an infinity or NaN reads back as
    NaN throughout.  Slots outside the cache are padding and not written.
    Of several rows for one slot the last one is kept; ``unique=True``
    asserts that there are none and saves the pass that finds out, which
    takes 4 bytes a record of the cache (64 rows into 10^7 records: 15 us,
    5 without)."""
    if _cuda(cache):
        hip.ext().cache_write(cache, values, slots, fmt, unique)
        return
    reference.cache_write(cache, values, slots, fmt, unique)


def cache_read(cache: torch.Tensor, dim: int,
               slots: Optional[torch.Tensor] = None, fmt: str = "int8",
               dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values (n, ``dim``) of the records at ``slots``, or of all of them
    in order; ``dim`` and ``fmt`` as written.  A slot outside the cache is
    padding and reads as zeros."""
    if _cuda(cache):
        return hip.ext().cache_read(cache, dim, slots, fmt, dtype)
    return reference.cache_read(cache, dim, slots, fmt, dtype)


# ---------------------------------------------------------------------------
# Muon
# ---------------------------------------------------------------------------

#: the quintic of the Muon optimiser: steep at zero, values near one after
#: five steps (0.7 to 1.2)
MUON_COEFFS = (3.4445, -4.7750, 2.0315)


def _check_chain(name: str, steps: int, coeffs: Sequence[float],
                 eps: float) -> Tuple[float, float, float]:
    if not 1 <= int(steps) <= 100:
        raise ValueError(f"{name}: steps must be 1 to 100, got {steps}")
    if len(coeffs) != 3:
        raise ValueError(f"{name}: coeffs are (a, b, c), got {coeffs!r}")
    if not 0 < eps < float("inf"):
        raise ValueError(f"{name}: eps must be positive, got {eps}")
    a, b, c = (float(v) for v in coeffs)
    if not _bounded(a, b, c, int(steps)):
        raise ValueError(f"{name}: with coeffs {coeffs!r} singular values "
                         f"grow beyond 3.9 in {steps} steps")
    if abs(a) ** int(steps) < 2.0 ** -12:
        raise ValueError(f"{name}: with coeffs {coeffs!r} singular values "
                         f"near zero shrink to less than 2^-12 of what they "
                         f"were in {steps} steps")
    return a, b, c


@lru_cache(maxsize=64)
def _bounded(a: float, b: float, c: float, steps: int) -> bool:
    """Whether singular values from [0, 1] stay within 3.9, and what a step
    multiplies them by within 15.9: the kernels hold values in f16 planes
    scaled by 2^12."""
    x = torch.linspace(0.0, 1.0, 4097, dtype=torch.float64)
    for _ in range(steps):
        q = a + b * x ** 2 + c * x ** 4
        x = q * x
        if not (bool((x.abs() <= 3.9).all()) and
                bool((q.abs() <= 15.9).all())):
            return False
    return True


def orthogonalize(x: torch.Tensor, steps: int = 5,
                  coeffs: Sequence[float] = MUON_COEFFS,
                  eps: float = 1e-7) -> torch.Tensor:
    """The nearest (semi-)orthogonal matrices to those of ``x`` (..., m, n;
    f32, bf16 or f16), approximately: X = x / (|x|_F + eps), then ``steps``
    times X <- a X + (b G + c G^2) X with G = X X^T.  Singular values near
    zero stay there, the others come near one.

    Computed in f32, on the device with products of 22 to 24 bits, whatever
    the type, and rounded once at the end: before that, off by a few 1e-6 of
    the result's norm where singular values are alike, and by up to 4e-4
    where all but a few are near zero, whose roundings the steps multiply.
    In last places a result may depend on how many matrices there are, not
    on what the others hold.  The result is new and contiguous.  A matrix that holds an infinity or NaN
    gives NaN throughout, a matrix of zeros gives zeros.  Has no gradient."""
    if x.dim() < 2 or x.dtype not in _VALUE_TYPES:
        raise ValueError("orthogonalize: x must be matrices of float32, "
                         f"bfloat16 or float16, got {x.dtype} of "
                         f"{tuple(x.shape)}")
    a, b, c = _check_chain("orthogonalize", steps, coeffs, eps)
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("orthogonalize has no gradient: pass x.detach()")
    reference.check_no_tangent("orthogonalize", x)
    if not x.numel():
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    batch = x.detach().reshape(-1, *x.shape[-2:]).contiguous()
    if _cuda(x):
        out = hip.ext().orthogonalize(batch, int(steps), a, b, c, float(eps))
    else:
        out = reference.orthogonalize(batch, int(steps), (a, b, c),
                                      float(eps))
    return out.view(x.shape)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether contiguous tensors share memory."""
    return a.data_ptr() < b.data_ptr() + b.nbytes \
        and b.data_ptr() < a.data_ptr() + a.nbytes


def apply_muon(table: torch.Tensor, momentum: torch.Tensor,
               rows: torch.Tensor, grads: torch.Tensor, lr: float,
               mu: float = 0.95, nesterov: bool = True,
               weight_decay: float = 0.0, steps: int = 5,
               matrix_rows: Optional[int] = None,
               sorted_unique: bool = False,
               coeffs: Sequence[float] = MUON_COEFFS,
               eps: float = 1e-7) -> None:
    """Muon apply: ``table`` (f32) is a stack of matrices of ``matrix_rows``
    rows each (one matrix by default).  For every matrix W that ``rows``
    names a row of, with g the sum of its rows of ``grads`` (zero where none
    was given) and M its part of ``momentum``:

        M <- mu M + g;  U = g + mu M (``nesterov``) or M
        W <- (1 - lr weight_decay) W - lr sqrt(max(1, m / n)) O(U)

    with O as :func:`orthogonalize`.  The other matrices keep W and M.  Rows
    outside the table are left out.  Repeated rows are summed in the order
    that they come in.  ``sorted_unique``: the caller guarantees ``rows``
    ascending with no duplicates, so the pre-sort is skipped.  Of other
    pushes, those of up to 16384 rows can be captured into a graph, for
    tables of up to 2^20 windows (256 rows of a matrix, or what is left of
    one)."""
    a, b, c = _check_chain("apply_muon", steps, coeffs, eps)
    if table.dim() != 2 or table.dtype != torch.float32 \
            or momentum.shape != table.shape \
            or momentum.dtype != torch.float32:
        raise ValueError("apply_muon: table and momentum must be float32 of "
                         f"one 2-D shape, got {table.dtype} of "
                         f"{tuple(table.shape)} and {momentum.dtype} of "
                         f"{tuple(momentum.shape)}")
    if not table.is_contiguous() or not momentum.is_contiguous():
        raise ValueError("apply_muon: table and momentum must be contiguous")
    if _overlap(table, momentum):
        raise ValueError("apply_muon: table and momentum are the same memory")
    if rows.dim() != 1 or rows.dtype not in (torch.int64, torch.int32) \
            or grads.dtype != torch.float32 \
            or grads.shape != (rows.numel(), table.shape[1]):
        raise ValueError("apply_muon: rows must be 1-D int64 or int32 and "
                         "grads float32 with one row for each, got "
                         f"{rows.dtype} of {tuple(rows.shape)} and "
                         f"{grads.dtype} of {tuple(grads.shape)}")
    if not table.device == momentum.device == rows.device == grads.device:
        raise ValueError("apply_muon: operands on several devices")
    reference.check_no_tangent("apply_muon", table, momentum, grads)
    m = table.shape[0] if matrix_rows is None else int(matrix_rows)
    if table.shape[0] and (m < 1 or table.shape[0] % m):
        raise ValueError(f"apply_muon: a table of {table.shape[0]} rows is "
                         f"not a whole number of matrices of {m}")
    if not rows.numel() or not table.numel():
        return
    rows, grads = rows.long().contiguous(), grads.detach().contiguous()
    if _overlap(grads, momentum) or _overlap(grads, table):
        grads = grads.clone()
    args = (lr, mu, nesterov, weight_decay, int(steps), m)
    if _cuda(table):
        hip.ext().apply_muon(table, momentum, rows, bool(sorted_unique), grads,
                             *args, a, b, c, float(eps))
        return
    if not sorted_unique:
        rows, order = torch.sort(rows, stable=True)
        grads = grads[order]
    reference.apply_muon(table, momentum, rows, grads, *args, (a, b, c),
                         float(eps))

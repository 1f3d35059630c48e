"""HBM-resident sharded parameter table.

This is the MI355X-native replacement for the reference's
``server/SimplePSLogic.scala`` ``mutable.HashMap[Int, P]`` (SURVEY.md
§2.1/§2.3 K1–K3): each shard keeps its parameter partition as one dense
f32 slab in HBM (288 GB per GPU fits every BASELINE config dense — e.g.
1e9 features x 2 f32 = 8 GB over 8 shards), initialized eagerly with the
deterministic per-id hash init (semantically identical to the reference's
lazy ``getOrElseUpdate(id, paramInit(id))`` because init is a pure function
of the id), updated by HIP scatter-apply kernels.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import ops
from .parallel.partitioner import Partitioner


class ShardedTable:
    """One shard (this rank's partition) of the global parameter table.

    optimizer:
      "add"     — W[id] += delta           (reference paramUpdate = vectorSum /
                                            '+'; the worker scales by lr)
      "adagrad" — G += g^2; W -= lr*g/sqrt(G+eps)   (new capability)
      "muon"    — for tables of weight matrices, ``matrix_rows``
                  consecutive ids each (default: the whole table is one):
                  M = momentum*M + g; W = (1-lr*weight_decay)*W -
                  lr*sqrt(max(1, m/n))*O, O the orthogonalised g +
                  momentum*M (``nesterov``) or M (ops.apply_muon).  Every
                  ``apply`` is one step of the matrices that it names a
                  row of; TableServerLogic makes one of all the pushes
                  that a round brings, whose gradients are summed (those of
                  another round are another step).  A matrix has to lie
                  on one shard: with several shards use a RangePartitioner
                  whose blocks hold whole matrices.  M is checkpointed as
                  the accumulator.
    """

    def __init__(self, part: Partitioner, shard: int, dim: int,
                 device: torch.device,
                 init: Tuple[float, float] = (0.0, 0.0),
                 optimizer: str = "add", lr: float = 0.0,
                 eps: float = 1e-8, seed: int = 0,
                 momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0,
                 matrix_rows: Optional[int] = None):
        if optimizer not in ("add", "adagrad", "muon"):
            raise ValueError(f"unknown optimizer {optimizer!r}")
        if optimizer == "muon":
            matrix_rows = self._whole_matrices(part, shard, matrix_rows)
        self.momentum = float(momentum)
        self.nesterov = bool(nesterov)
        self.weight_decay = float(weight_decay)
        self.matrix_rows = matrix_rows
        self.part = part
        self.shard = shard
        self._full_ids: "torch.Tensor | None" = None
        self.dim = int(dim)
        self.device = torch.device(device)
        self.optimizer = optimizer
        self.lr = float(lr)
        self.eps = float(eps)
        rows = part.shard_rows(shard)
        self.rows = rows
        self.data = torch.empty(rows, dim, dtype=torch.float32,
                                device=self.device)
        lo, hi = init
        if lo == 0.0 and hi == 0.0:
            self.data.zero_()
        else:
            # Deterministic per-global-id init: row r holds global id
            # part.global_id(shard, r).  For ModPartitioner that is
            # first_id=shard, stride=n_shards; for RangePartitioner
            # first_id=shard*block, stride=1.
            first = int(self.part.global_id(
                self.shard, torch.zeros(1, dtype=torch.int64)).item()) if rows else 0
            if rows >= 2:
                second = int(self.part.global_id(
                    self.shard, torch.ones(1, dtype=torch.int64)).item())
                stride = second - first
            else:
                stride = 1
            if rows:
                ops.hash_init_rows(self.data, first, stride, lo, hi, seed)
        if optimizer in ("adagrad", "muon"):
            self.accum = torch.zeros(rows, dim, dtype=torch.float32,
                                     device=self.device)
        else:
            self.accum = None

    @staticmethod
    def _whole_matrices(part: Partitioner, shard: int,
                        matrix_rows: Optional[int]) -> int:
        """``matrix_rows``, checked: the shard's rows are whole matrices of
        consecutive ids."""
        rows = part.shard_rows(shard)
        if matrix_rows is None:
            if part.n_shards > 1:
                raise ValueError(
                    "optimizer 'muon' over several shards needs matrix_rows "
                    "(consecutive ids of one matrix)")
            return max(1, rows)
        m = int(matrix_rows)
        if m < 1:
            raise ValueError(f"matrix_rows must be at least 1, got {m}")
        if rows:
            ends = part.global_id(shard, torch.tensor([0, rows - 1])).tolist()
            if ends[1] - ends[0] != rows - 1 or ends[0] % m or rows % m:
                raise ValueError(
                    f"shard {shard} does not hold whole matrices of {m} "
                    "consecutive ids: use a RangePartitioner whose blocks "
                    "are multiples of matrix_rows")
        return m

    # -- server-side ops (K3 gather / K1 sgd apply / K2 adagrad apply) ----

    def gather(self, ids: torch.Tensor) -> torch.Tensor:
        if self._is_full_range(ids):
            # dense pull of the whole shard: the "gather" is the slab
            # itself.  Answer values alias the live table; the engine's
            # round order (worker consumes answers BEFORE this round's
            # pushes apply) makes that observationally identical to a
            # copy taken at answer time under fresh/merged schedules.
            # Under "pipelined" a self-addressed alias is consumed one
            # round later, after one more local push-apply — the worker
            # then sees FRESHER values than gather time, which the
            # async pull contract allows (answers carry no freshness
            # guarantee; remote segments are real copies either way).
            return self.data
        rows = self.part.local_row(ids)
        return ops.gather(self.data, rows)

    def _is_full_range(self, ids: torch.Tensor) -> bool:
        """ids == every row of this shard in local-row order?  Verified
        with one tensor compare on first sight, then recognized by
        buffer IDENTITY (dense-pull workers re-send one cached tensor).
        The verified tensor itself is retained in the cache entry — as
        runtime._shard_counts and the HIP position cache do — so its
        storage stays alive and a recycled allocation of the same
        pointer (e.g. a fresh multi-GPU recv buffer each round) can
        never be misclassified as the cached full-range pull."""
        if ids.numel() != self.rows or self.rows == 0:
            return False
        cached = self._full_ids
        if cached is not None and ids is cached:
            return True
        rows = self.part.local_row(ids)
        expect = torch.arange(self.rows, dtype=rows.dtype,
                              device=rows.device)
        if bool(torch.equal(rows, expect)):
            self._full_ids = ids
            return True
        return False

    def apply(self, ids: torch.Tensor, deltas: torch.Tensor,
              unique: bool = False) -> None:
        rows = self.part.local_row(ids)
        if self.optimizer == "add":
            ops.apply_add(self.data, rows, deltas, unique)
        elif self.optimizer == "muon":
            ops.apply_muon(self.data, self.accum, rows.to(self.device),
                           deltas, self.lr, mu=self.momentum,
                           nesterov=self.nesterov,
                           weight_decay=self.weight_decay,
                           matrix_rows=self.matrix_rows,
                           sorted_unique=unique)
        else:
            # `unique` batches arrive as sorted unique pulled ids, and
            # both partitioners are monotone per shard, so the local
            # rows are already sorted — the adagrad pre-sort is skipped.
            ops.apply_adagrad(self.data, self.accum, rows, deltas,
                              self.lr, self.eps, sorted_unique=unique)

    def dump(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """(global_ids, values) of every row of the shard — the reference's
        ``ParameterServerLogic.close`` model dump (unordered contract;
        ours happens to be local-row order)."""
        rows = torch.arange(self.rows, dtype=torch.int64)
        gids = self.part.global_id(self.shard, rows)
        return gids, self.data

    def load(self, ids: torch.Tensor, values: torch.Tensor) -> None:
        """Warm start (``transformWithModelLoad``): overwrite rows by id."""
        rows = self.part.local_row(ids).to(self.device)
        self.data.index_copy_(0, rows, values.to(self.device,
                                                 self.data.dtype))


class TableServerLogic:
    """ServerLogic over a ShardedTable — the production default server.

    Semantics parity: ``SimplePSLogic(paramInit, paramUpdate)`` with
    paramInit = deterministic ranged-random init and paramUpdate = '+'
    (or the Adagrad rule).
    """

    #: answers every pull batch in full, in received order, same round —
    #: lets the engine elide answer ids from the feedback edge.
    answers_in_order = True

    # the push at hand is that of several workers, whose ids repeat
    _joined = False

    def __init__(self, table: ShardedTable, dump_on_close: bool = True,
                 pushes_unique: bool = False):
        """``pushes_unique=True``: the application guarantees every push
        batch carries SORTED distinct ids (all bundled model logics do —
        they push pre-aggregated deltas per sorted unique pulled id, one
        push per round), enabling the non-atomic add fast path and the
        sort-free adagrad path.  Leave False when pushes may repeat or
        interleave ids (e.g. under a count/time flush strategy that
        coalesces several logical pushes into one round)."""
        self.table = table
        self.dump_on_close = dump_on_close
        self.pushes_unique = pushes_unique

    @property
    def whole_steps(self) -> bool:
        """Whether an apply is a step of all the rows of what it touches, and
        not a sum that may come in parts (Muon: of whole matrices)."""
        return getattr(self.table, "optimizer", None) == "muon"

    def on_pull_recv(self, ids: torch.Tensor, worker: int, ps) -> None:
        ps.answer_pull(ids, self.table.gather(ids), worker)

    def on_push_recv(self, ids: torch.Tensor, deltas: torch.Tensor,
                     ps) -> None:
        self.table.apply(ids, deltas,
                         unique=self.pushes_unique and not self._joined)

    def on_pushes_recv(self, pushes: List[Tuple[torch.Tensor, torch.Tensor]],
                       ps) -> None:
        """A round's pushes one after the other, or, where an apply is a
        whole step, as one push: a step of each would move a matrix as often
        as there are workers, however small their shares of the gradient
        are."""
        if len(pushes) == 1 or not self.whole_steps:
            for ids, deltas in pushes:
                self.on_push_recv(ids, deltas, ps)
            return
        self._joined = True
        try:
            self.on_push_recv(torch.cat([i for i, _ in pushes]),
                              torch.cat([d for _, d in pushes]), ps)
        finally:
            self._joined = False

    def close(self, ps) -> None:
        if self.dump_on_close:
            ps.output(self.table.dump())

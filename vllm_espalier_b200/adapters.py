"""Low-rank adapters of many requests at once, beside one shared (coded) projection.

A batch's rows share the projection's coded weights; each row may add the product of its own request's adapter:

    out[t] = y[t] + scale[a] (x[t] A[a, s]^T) B[a, s]^T     with a = ids[t], for every matrix s of the layer

y is the projection's output (dense.Dense of the same matrices, side by side), x its input. Rows may come in any order
and any mix of adapters, rows without one (id -1) keep y; a row's bits depend on its own id, x and y only. The kernel is
esp_adapt (csrc/adapters.cu).
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import DTYPE, esp_adapters_t, launch, lib

MAX_RANK, MAX_MATS, MAX_SLOTS = 128, 4, 4096
NONE = -1                     # the id of a row without an adapter
MAX_ROWS = 1 << 26            # of one call
MAX_COLUMNS = 1 << 30         # k, and the sum of the widths
NO_PLAN = 64                  # rows up to which the kernel takes no workspace


class Adapters:
    """The adapters of one layer, in `slots` places that load() fills and clear() empties.

    a: [slots, matrices, rank, k], b: [slots, sum(widths), rank], fp16 or bf16 and contiguous; rank is the capacity, a
    multiple of 8 up to 128, k and the widths are multiples of 8. ranks int32 [slots] (None: all of the full rank): a
    slot of rank q uses the rows of a and the columns of b below q rounded up to 8, which from q on must hold zeros.
    scales fp32 [slots] (None: ones). All are kept, not copied."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, widths, ranks: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None):
        widths = [int(w) for w in widths]
        if a.dim() != 4 or b.dim() != 3:
            raise ValueError(f"a must be [slots, matrices, rank, k] and b [slots, columns, rank], got "
                             f"{tuple(a.shape)} and {tuple(b.shape)}")
        slots, mats, rank, k = a.shape
        if len(widths) != mats or not 1 <= mats <= MAX_MATS or b.shape != (slots, sum(widths), rank) or \
                not 1 <= slots <= MAX_SLOTS:
            raise ValueError(f"widths {widths} do not fit a {tuple(a.shape)} and b {tuple(b.shape)} (at most "
                             f"{MAX_MATS} matrices and {MAX_SLOTS} slots)")
        if rank % 8 or not 8 <= rank <= MAX_RANK or k % 8 or k < 8 or any(w % 8 or w < 8 for w in widths):
            raise ValueError(f"rank {rank} (8..{MAX_RANK}), k {k} and widths {widths} must be multiples of 8")
        if k > MAX_COLUMNS or sum(widths) > MAX_COLUMNS:
            raise ValueError(f"k {k} and {sum(widths)} columns must be {MAX_COLUMNS} at most")
        if not a.is_cuda or a.dtype not in (torch.float16, torch.bfloat16) or b.dtype != a.dtype:
            raise ValueError(f"a and b must be CUDA tensors, both fp16 or both bf16, got {a.dtype} and {b.dtype}")
        for name, t, dtype in (("b", b, a.dtype), ("ranks", ranks, torch.int32), ("scales", scales, torch.float32)):
            if t is not None and (t.device != a.device or t.dtype != dtype):
                raise ValueError(f"{name} must be {dtype} on {a.device}, got {t.dtype} on {t.device}")
        for name, t in (("ranks", ranks), ("scales", scales)):
            if t is not None and t.shape != (slots,):
                raise ValueError(f"{name} must be [{slots}], got {tuple(t.shape)}")
        if not all(t is None or t.is_contiguous() for t in (a, b, ranks, scales)):
            raise ValueError("a, b, ranks and scales must be contiguous")
        self.a, self.b, self.ranks, self.scales = a, b, ranks, scales
        self.slots, self.rank, self.k, self.widths, self.n = slots, rank, k, widths, sum(widths)
        self.dtype, self.device = a.dtype, a.device
        self._c = esp_adapters_t(a.data_ptr(), b.data_ptr(), None if ranks is None else ranks.data_ptr(),
                                 None if scales is None else scales.data_ptr(), DTYPE[a.dtype], slots, rank, k, mats,
                                 (C.c_int * 4)(*widths))
        self._ref = C.addressof(self._c)

    @classmethod
    def empty(cls, k: int, widths, slots: int, rank: int, dtype=torch.bfloat16, device="cuda") -> "Adapters":
        """`slots` empty places (rank 0: rows that name them keep y)."""
        widths = list(widths)
        return cls(torch.zeros((slots, len(widths), rank, k), dtype=dtype, device=device),
                   torch.zeros((slots, sum(widths), rank), dtype=dtype, device=device), widths,
                   torch.zeros(slots, dtype=torch.int32, device=device),
                   torch.ones(slots, dtype=torch.float32, device=device))

    def load(self, slot: int, a, b, scale: float = 1.0):
        """Put one adapter into a slot: a [q, k] and b [width, q] of each matrix (None for a matrix without one), any
        rank q up to the capacity, the same for all of them."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} outside 0..{self.slots - 1}")
        if self.ranks is None or self.scales is None:
            raise ValueError("these adapters were made without ranks and scales: write a and b instead")
        a, b = list(a), list(b)
        given = [x.shape[0] for x in a if x is not None]
        if len(a) != len(self.widths) or len(b) != len(self.widths) or not given:
            raise ValueError(f"one a and one b for each of {len(self.widths)} matrices, at least one of them given")
        q = given[0]
        if not 1 <= q <= self.rank:
            raise ValueError(f"rank {q} outside 1..{self.rank}")
        for x, w, width in zip(a, b, self.widths):
            if (x is None) != (w is None):
                raise ValueError("a matrix has both a and b or neither")
            if x is not None and (x.shape != (q, self.k) or w.shape != (width, q)):
                raise ValueError(f"a must be [{q}, {self.k}] and b [{width}, {q}], got {tuple(x.shape)} and "
                                 f"{tuple(w.shape)}")
        self.clear(slot)
        col = 0
        for m, (x, w, width) in enumerate(zip(a, b, self.widths)):
            if x is not None:
                self.a[slot, m, :q].copy_(x)
                self.b[slot, col:col + width, :q].copy_(w)
            col += width
        self.scales[slot] = scale
        self.ranks[slot] = q

    def clear(self, slot: int):
        """Empty a slot: rows that name it keep y."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} outside 0..{self.slots - 1}")
        if self.ranks is not None:
            self.ranks[slot] = 0
        self.a[slot].zero_()
        self.b[slot].zero_()

    def _rows(self, t: torch.Tensor, name: str, columns: int) -> tuple[int, bool]:
        """(row stride, whether the kernel takes the rows as they are: unit columns, 16-byte aligned)."""
        if t.dtype != self.dtype or t.dim() != 2 or t.shape[1] != columns or t.device != self.device:
            raise ValueError(f"{name} must be {self.dtype} [rows, {columns}] on {self.device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        stride, step = t.stride()
        return stride, step == 1 and not stride & 7 and not t.data_ptr() & 15

    def forward(self, x: torch.Tensor, y: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None):
        """x [rows, k], y [rows, sum(widths)] in the adapters' dtype, ids int32 [rows] (outside [0, slots): no adapter).
        Returns out (a new tensor, or the one given: y itself adds in place)."""
        (x_stride, x_fits), (y_stride, y_fits) = self._rows(x, "x", self.k), self._rows(y, "y", self.n)
        rows = x.shape[0]
        if y.shape[0] != rows or ids.dim() != 1 or ids.numel() != rows:
            raise ValueError(f"x has {rows} rows, y {y.shape[0]}, ids {tuple(ids.shape)}")
        if rows > MAX_ROWS:
            raise ValueError(f"{rows} rows are more than {MAX_ROWS}")
        if ids.dtype != torch.int32 or ids.device != self.device or not ids.is_contiguous():
            raise ValueError(f"ids must be contiguous int32 on {self.device}, got {ids.dtype} on {ids.device}")
        if out is None:
            out, out_stride = y.new_empty((rows, self.n)), self.n
        else:
            out_stride, fits = self._rows(out, "out", self.n)
            if out.shape[0] != rows or (rows and not fits):
                raise ValueError(f"out must be [{rows}, {self.n}] with 16-byte aligned rows and unit column stride")
        if not rows:
            return out
        if not x_fits:
            x, x_stride = x.clone(memory_format=torch.contiguous_format), self.k
        if not y_fits:
            y, y_stride = y.clone(memory_format=torch.contiguous_format), self.n
        need = ws = 0
        if rows > NO_PLAN:
            need = lib().esp_adapt_ws_bytes(rows, self.slots)
            scratch = ids.new_empty((need + 3) // 4)
            ws = scratch.data_ptr()
        launch(self.device, lib().esp_adapt, self._ref, x.data_ptr(), x_stride, y.data_ptr(), y_stride, ids.data_ptr(), rows,
               out.data_ptr(), out_stride, ws, need)
        return out

    __call__ = forward

"""A batch whose rows belong to several requests: which rows are whose, and the adapters they use.

One `RequestRows` is made per batch, on the host, and handed to every layer of the step (the shared int8 projections with
one low-rank adapter per request, the gated residual update with one modulation per request).  `stack_adapters` lays the
factors of a layer's adapters out as the bank that the projections read.
"""
from __future__ import annotations

import ctypes
from collections.abc import Sequence

import numpy as np
import torch
from torch import Tensor

from . import _native as nat

CHUNK_ROWS = 4      # rows of one adapter that a small work item of the kernels takes together


class RequestRows:
    """The rows of a batch: `lengths[i]` consecutive rows belong to request i (0 is allowed), which uses entry `adapters[i]`
    of the bank of adapters, or none (-1, also without `adapters`).  Rows that pad a batch are a request without an adapter.

    The tables are copied to `device` here (the host waits for the copy, so they may be used on any stream afterwards);
    make the plan outside a graph capture.  A captured call keeps the plan that it was captured with, which has to outlive
    the graph.
    """

    def __init__(self, lengths: Sequence[int], adapters: Sequence[int] | None = None,
                 device: torch.device | str = "cuda"):
        n = np.asarray(lengths, dtype=np.int64).reshape(-1)
        a = np.full(n.shape, -1, dtype=np.int64) if adapters is None else np.asarray(adapters, dtype=np.int64).reshape(-1)
        if n.size == 0 or (n < 0).any():
            raise ValueError("lengths must be one or more row counts, none of them negative")
        if a.shape != n.shape:
            raise ValueError(f"{n.size} requests, but {a.size} adapters")
        if (a < -1).any() or int(n.sum()) >= 1 << 31 or (a >= 1 << 20).any():
            raise ValueError("an adapter is an index into the bank or -1 for none")
        self.lengths = tuple(int(v) for v in n)
        self.adapters = tuple(int(v) for v in a)
        self.requests = int(n.size)
        self.total = int(n.sum())
        used = a[n > 0]
        self.max_adapter = int(used.max()) if used.size else -1
        row_adapter = np.repeat(a, n)
        row_request = np.repeat(np.arange(n.size), n)
        chunks = self._chunks(row_adapter)
        parts = [row_adapter, row_request, chunks.reshape(-1)]
        offsets = np.cumsum([0] + [-(-p.size // 4) * 4 for p in parts])      # 16-byte aligned tables in one buffer
        packed = np.zeros(max(int(offsets[-1]), 4), dtype=np.int32)
        for o, p in zip(offsets, parts):
            packed[o:o + p.size] = p
        self._tables = torch.from_numpy(packed).to(device)
        self.device = self._tables.device
        base = self._tables.data_ptr()
        self.native = nat.RequestRowsStruct(rows=self.total, row_adapter=base + 4 * int(offsets[0]),
                                            row_request=base + 4 * int(offsets[1]), chunks=base + 4 * int(offsets[2]),
                                            n_chunks=chunks.shape[0], max_adapter=self.max_adapter)
        self.native_ptr = ctypes.byref(self.native)

    @staticmethod
    def _chunks(row_adapter: np.ndarray) -> np.ndarray:
        """[n, 4] first row, row count, adapter, 0: runs of rows with one adapter, cut into pieces of CHUNK_ROWS."""
        if row_adapter.size == 0:
            return np.zeros((0, 4), dtype=np.int64)
        starts = np.concatenate([[0], np.flatnonzero(np.diff(row_adapter)) + 1])
        ends = np.concatenate([starts[1:], [row_adapter.size]])
        pieces = -(-(ends - starts) // CHUNK_ROWS)
        run = np.repeat(np.arange(starts.size), pieces)
        first = starts[run] + CHUNK_ROWS * (np.arange(run.size) - np.repeat(np.cumsum(pieces) - pieces, pieces))
        count = np.minimum(CHUNK_ROWS, ends[run] - first)
        return np.stack([first, count, row_adapter[first], np.zeros_like(first)], axis=1)


def stack_adapters(factors: Sequence[tuple[Tensor, Tensor] | tuple[Tensor, Tensor, float]], dtype: torch.dtype,
                   device: torch.device | str) -> tuple[Tensor, Tensor]:
    """The adapters of one layer as a bank: `factors` holds (down [r_i, K], up [N, r_i]) or (down, up, scale) of each.

    Returns (lora_a [n, r, K], lora_b [n, N, r]) in `dtype`, r the largest rank rounded up to a multiple of 8 (16-byte
    rows); smaller ranks are filled with zeros, the scale is multiplied into `down` in fp32.
    """
    if not factors:
        raise ValueError("a bank needs at least one adapter")
    downs = [f[0].flatten(1) for f in factors]
    ups = [f[1].flatten(1) for f in factors]
    K, N = downs[0].shape[1], ups[0].shape[0]
    for d, u in zip(downs, ups):
        if d.shape[1] != K or u.shape[0] != N or d.shape[0] != u.shape[1]:
            raise ValueError(f"factors {tuple(d.shape)} and {tuple(u.shape)} do not fit a layer [{N}, {K}]")
    r = max(8, -(-max(d.shape[0] for d in downs) // 8) * 8)
    lora_a = torch.zeros((len(factors), r, K), dtype=dtype, device=device)
    lora_b = torch.zeros((len(factors), N, r), dtype=dtype, device=device)
    for i, (f, d, u) in enumerate(zip(factors, downs, ups)):
        scale = float(f[2]) if len(f) > 2 else 1.0
        lora_a[i, :d.shape[0]] = (d.to(device).float() * scale).to(dtype) if scale != 1.0 else d.to(device=device, dtype=dtype)
        lora_b[i, :, :u.shape[1]] = u.to(device=device, dtype=dtype)
    return lora_a, lora_b

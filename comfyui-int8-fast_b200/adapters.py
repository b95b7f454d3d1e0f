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

TILE_ROWS = 256     # rows of a tile of the projection
TILE_SLOTS = 8      # adapters with more than a few rows that a tile may have to be run on the tensor cores
TILE_ADAPTERS = 16  # adapters in all that it may have (an up-projection MMA each; the few rows' down projection is chunked)
DENSE_ROWS = 256    # batches of fewer rows are chunked throughout
FEW_ROWS = 8        # rows of a tile up to which an adapter's down projection is left to chunks where the tile has others
MAX_RANK = 1024     # ranks of an adapter that the projections take
CHUNK_ROWS = 4      # rows of one adapter that a small work item of the kernels takes together


class RequestRows:
    """The rows of a batch: `lengths[i]` consecutive rows belong to request i (0 is allowed), which uses entry `adapters[i]`
    of the bank of adapters, or none (-1, also without `adapters`).  Rows that pad a batch are a request without an adapter.

    The tables are copied to `device` here (the host waits for the copy, so they may be used on any stream afterwards, and the
    plan may be dropped while calls with it are under way); make the plan outside a graph capture.  A captured call keeps
    the tables that it was captured with: the plan has to outlive the graph.
    """

    def __init__(self, lengths: Sequence[int], adapters: Sequence[int] | None = None,
                 device: torch.device | str = "cuda"):
        device = torch.device(device)
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a row plan is made outside of a graph capture: its tables are copied from the host")
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
        tiles, slots, chunks, addend_rows = self._plan(row_adapter, self.lengths, self.adapters)
        parts = [row_adapter, row_request, tiles.reshape(-1), slots.reshape(-1), chunks.reshape(-1)]
        offsets = np.cumsum([0] + [-(-p.size // 4) * 4 for p in parts])      # 16-byte aligned tables in one buffer
        packed = np.zeros(max(int(offsets[-1]), 4), dtype=np.int32)
        for o, p in zip(offsets, parts):
            packed[o:o + p.size] = p
        self._tables = torch.from_numpy(packed).to(device)
        self.device = self._tables.device
        at = [self._tables.data_ptr() + 4 * int(o) for o in offsets]
        self.native = nat.RequestRowsStruct(rows=self.total, row_adapter=at[0], row_request=at[1], tiles=at[2], slots=at[3], chunks=at[4],
                                            n_dense=int((tiles[:, 2] < 0).sum()), n_chunks=chunks.shape[0], addend_rows=addend_rows,
                                            max_adapter=self.max_adapter)
        # streams whose calls the allocator waits for before it hands the tables' memory on
        self.streams = {nat.stream_handle(self.device)} if self.device.type == "cuda" else set()
        self.native_ptr = ctypes.byref(self.native)
        self.row_request_ptr = at[1]
        self.workspace_bytes: dict = {}      # sizes the library asks for, by layer shape

    def use_on(self, stream: int) -> None:
        """A call on `stream` (the handle of the device's current one, not in `streams` yet) is about to read the tables."""
        if not torch.cuda.is_current_stream_capturing():
            self._tables.record_stream(torch.cuda.current_stream(self.device))
            self.streams.add(stream)

    @staticmethod
    def _plan(row_adapter: np.ndarray, lengths: Sequence[int], adapters: Sequence[int]):
        """tiles [n, 4], slots [n, 12], chunks [n, 4] and the rows of the addend, as i8f_request_rows describes them."""
        rows = row_adapter.size
        n_tiles = -(-rows // TILE_ROWS)
        dense = np.zeros(n_tiles, dtype=bool)
        tiles = np.zeros((n_tiles, 4), dtype=np.int64)
        slots = np.zeros((0, 12), dtype=np.int32)
        if rows >= DENSE_ROWS:
            # per tile and adapter the rows that use it, as the bits of an integer
            masks: list[dict] = [{} for _ in range(n_tiles)]
            first = 0
            for n, a in zip(lengths, adapters):
                last = first + n
                if a >= 0:
                    for i in range(first // TILE_ROWS, -(-last // TILE_ROWS) if n else 0):
                        lo, hi = max(first - i * TILE_ROWS, 0), min(last - i * TILE_ROWS, TILE_ROWS)
                        masks[i][a] = masks[i].get(a, 0) | (((1 << (hi - lo)) - 1) << lo)
                first = last
            per_tile = np.array([len(m) for m in masks])
            many = np.array([sum(mask.bit_count() > FEW_ROWS for mask in m.values()) for m in masks])
            dense = (per_tile <= TILE_ADAPTERS) & (many <= TILE_SLOTS)
            # an MMA costs a tile the same for one row as for all: an adapter's few rows beside others are cheaper as chunks there
            table = [(a, int(len(m) > 1 and mask.bit_count() <= FEW_ROWS), mask) for m, d in zip(masks, dense) if d for a, mask in m.items()]
            slots = np.zeros((len(table), 12), dtype=np.int32)
            if table:
                slots[:, 0] = [a for a, _, _ in table]
                slots[:, 1] = [few for _, few, _ in table]
                slots[:, 4:] = np.frombuffer(b"".join(mask.to_bytes(TILE_ROWS // 8, "little") for _, _, mask in table), dtype="<i4").reshape(-1, 8)
            tiles[:, 1] = np.where(dense, per_tile, 0)
            tiles[:, 0] = np.cumsum(tiles[:, 1]) - tiles[:, 1]
        tiles[:, 2] = np.where(dense, -1, (np.cumsum(~dense) - 1) * TILE_ROWS)
        last = max(0, n_tiles * TILE_ROWS - rows) if n_tiles and not dense[-1] else 0
        addend_rows = int((~dense).sum()) * TILE_ROWS - last
        few = np.zeros((n_tiles, TILE_ROWS), dtype=bool)      # rows of dense tiles that are chunked all the same
        if slots[:, 1].any():
            slot_tile = np.repeat(np.arange(n_tiles), tiles[:, 1])
            bits = np.unpackbits(np.ascontiguousarray(slots[:, 4:]).view(np.uint8), axis=1, bitorder="little").astype(bool)
            np.logical_or.at(few, slot_tile[slots[:, 1] > 0], bits[slots[:, 1] > 0])
        elif dense.all():
            return tiles, slots, np.zeros((0, 4), dtype=np.int64), addend_rows
        tile_of = np.arange(rows) // TILE_ROWS
        # runs of rows with one adapter among the chunked rows, cut into pieces of CHUNK_ROWS
        left = np.flatnonzero(~dense[tile_of] | few.reshape(-1)[:rows])
        cut = (np.diff(left) != 1) | (np.diff(row_adapter[left]) != 0) | (np.diff(tile_of[left]) != 0)
        starts = np.concatenate([[0], np.flatnonzero(cut) + 1])
        ends = np.concatenate([starts[1:], [left.size]])
        pieces = -(-(ends - starts) // CHUNK_ROWS)
        run = np.repeat(np.arange(starts.size), pieces)
        first = starts[run] + CHUNK_ROWS * (np.arange(run.size) - np.repeat(np.cumsum(pieces) - pieces, pieces))
        count = np.minimum(CHUNK_ROWS, ends[run] - first)
        row = left[first]
        addend = np.where(dense[tile_of[row]], -1, tiles[tile_of[row], 2] + row % TILE_ROWS)
        return tiles, slots, np.stack([row, count, row_adapter[row], addend], axis=1), addend_rows


class RequestLoras:
    """The adapters of one quantised layer for a batch whose samples belong to several requests, as the Linear holds them.

    `entries[i]` is the bank entry of request i (-1: none), `plans` a dict that the layers of a model share, so that a batch
    shape is planned once.  Sample j of a batch belongs to request j modulo the number of requests (a batch that repeats its
    samples, for guidance say, repeats the requests with them).
    """

    def __init__(self, lora_a: Tensor, lora_b: Tensor, entries: Sequence[int], plans: dict | None = None):
        if lora_a.dim() != 3 or lora_b.dim() != 3 or lora_a.shape[0] != lora_b.shape[0] or lora_a.shape[1] != lora_b.shape[2]:
            raise ValueError(f"{tuple(lora_a.shape)} and {tuple(lora_b.shape)} are no bank [n, r, K], [n, N, r]")
        if not len(entries) or any(not -1 <= e < lora_a.shape[0] for e in entries):
            raise ValueError(f"entries {tuple(entries)} do not index a bank of {lora_a.shape[0]}")
        self.lora_a, self.lora_b = lora_a, lora_b
        self.entries = tuple(int(e) for e in entries)
        self._plans = {} if plans is None else plans
        self._converted = None
        self._streams: set = set()      # those that have waited for the conversion
        self._ready = None

    @property
    def samples(self) -> int | None:
        """Samples of the model's current batch, where the model's hook has left word and could see it."""
        return self._plans.get("samples")

    def bank(self, device: torch.device, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
        """The bank in the compute type on the compute device, converted once: another stream than the first waits for that, and
        the allocator for it.  Within a graph capture nothing is kept, since the conversion only runs with the graph."""
        held = self._converted
        fits = held is not None and held[0].device == device and held[0].dtype == dtype
        if not fits:
            held = (self.lora_a.to(device=device, dtype=dtype).contiguous(), self.lora_b.to(device=device, dtype=dtype).contiguous())
        if device.type == "cuda":
            handle = nat.stream_handle(device)
            if (fits and handle in self._streams) or torch.cuda.is_current_stream_capturing():
                return held
            stream = torch.cuda.current_stream(device)
            if fits:
                stream.wait_event(self._ready)
            else:
                self._ready = stream.record_event()
                self._streams = set()
            self._streams.add(handle)
            for t in held:
                t.record_stream(stream)
        self._converted = held
        return held

    def plan(self, rows: int, leading: int | None, device: torch.device) -> RequestRows:
        """The plan of an input of `rows` rows, equal runs of them one per sample of the batch.  `leading` is the first of the
        input's three or more dimensions, None for fewer.

        Where the requests differ, the samples are as many as the model's batch has where its hook has said so: the input's
        leading dimension has to be that many, or 1 with the rows of all samples behind it (rows that the samples share have no
        adapter of their own).  Another leading dimension is refused, since it does not say whether it repeats the batch or cuts
        every sample in pieces.  Where the hook could not see the batch `leading` counts and an input of two dimensions is
        refused; where no hook speaks for the model such an input is one run of rows per request.  Rows that are not equal
        runs for every request are refused."""
        known, n = self.samples, len(self.entries)
        if not rows:
            samples = n
        elif len(set(self.entries)) == 1:      # one composition for all: nothing to tell apart
            return self._planned([rows], self.entries[:1], device)
        elif known is not None:
            if leading not in (None, 1, known):
                raise ValueError(f"a leading dimension of {leading} for a batch of {known} samples: which rows are whose cannot be known "
                                 "(an input of two dimensions holds the samples' rows one sample after the other)")
            samples = known
        elif leading is not None:
            samples = leading
        elif "samples" in self._plans:
            raise ValueError(f"the batch of the model's call is not known (its first argument is no tensor), {rows} rows in two "
                             "dimensions cannot be told apart by request")
        else:
            samples = n
        if not samples or rows % samples:
            raise ValueError(f"{rows} rows are not {samples} samples of equal length")
        return self.rows(samples, rows // samples, device)

    def rows(self, samples: int, rows_per_sample: int, device: torch.device) -> RequestRows:
        n = len(self.entries)
        if samples % n:
            raise ValueError(f"a batch of {samples} samples for {n} requests")
        return self._planned([rows_per_sample] * samples, self.entries * (samples // n), device)

    def _planned(self, lengths: list[int], entries: tuple[int, ...], device: torch.device) -> RequestRows:
        key = (entries, len(lengths), lengths[0] if lengths else 0, device)
        plan = self._plans.get(key)
        if plan is None:
            plan = self._plans[key] = RequestRows(lengths, entries, device)
        return plan


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

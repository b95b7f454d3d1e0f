"""The operators of a batch of requests against plain 64-bit forms, on a B200.

Tolerances are worst cases of the roundings named beside them: u = eps / 2 of the output type per rounding, 2^-24 per fp32
operation.  They are evaluated element by element in 64 bits next to the reference.
"""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64
E32 = 2.0 ** -24
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}   # half a denormal step, or below


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(autouse=True)
def _status_clean(cuda_pkg):
    yield
    torch.cuda.synchronize()
    assert cuda_pkg._native.device_status() == 0, "a bounded device-side wait ran out"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def check(got, want, tol):
    assert got.shape == want.shape
    off = (got.to(F64) - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.3g} of its tolerance"


# ------------------------------------------------------------------ adapters
def layer(K, N, r, n, dtype, seed, per_channel=True, bias=True):
    g = gen(seed)
    w = torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    ws = torch.rand(N, 1, generator=g, device=DEV) * 4e-4 + 1e-4 if per_channel else torch.full((1,), 3e-4, device=DEV)
    b = torch.randn(N, generator=g, device=DEV).to(dtype) if bias else None
    la = (torch.randn(n, r, K, generator=g, device=DEV) / K ** 0.5).to(dtype)
    lb = (torch.randn(n, N, r, generator=g, device=DEV) * 0.3).to(dtype)
    return w, ws, b, la, lb


def adapter_rows(rows):
    return torch.tensor([a for n, a in zip(rows.lengths, rows.adapters) for _ in range(n)], device=DEV, dtype=torch.long)


def low_rank(x, la, lb, at, dtype):
    """The low-rank term in 64 bits and how far the kernels' may be from it: t in any order of fp32 sums (K 2^-23 of the sum
    of magnitudes), rounded to dtype (u), then r products summed in fp32."""
    N, r, K = lb.shape[1], la.shape[1], la.shape[2]
    want = torch.zeros(x.shape[0], N, dtype=F64, device=DEV)
    tol = torch.zeros_like(want)
    for a in sorted(set(at.tolist()) - {-1}):
        m = (at == a).nonzero().flatten()
        A, B = la[a].to(F64), lb[a].to(F64)
        xa = x[m].to(F64)
        t = xa @ A.T
        t_off = K * 2 * E32 * (xa.abs() @ A.abs().T)
        t_off = t_off + u_of(dtype) * (t.abs() + t_off) + TINY[dtype]
        want[m] = t @ B.T
        tol[m] = t_off @ B.abs().T + 2 * r * E32 * ((t.abs() + t_off) @ B.abs().T)
    return want, tol


def base_quantised(q, qs, w, ws, b):
    """The dequantised product in 64 bits from the quantised rows (exact int32 sums in the kernels: four fp32 roundings)."""
    y = (q.to(F64) @ w.to(F64).T) * qs.to(F64) * ws.to(F64).reshape(1, -1)
    mag = y.abs()
    if b is not None:
        y = y + b.to(F64)
        mag = mag + b.to(F64).abs()
    return y, 4 * E32 * mag


LINEAR = [
    # lengths, adapters, K, N, r, dtype
    ([17], [0], 64, 64, 8, torch.bfloat16),
    ([1] * 40, [i % 5 - 1 for i in range(40)], 256, 200, 16, torch.bfloat16),
    ([100, 0, 29, 1, 1, 3], [1, 0, -1, 2, 1, 1], 512, 328, 24, torch.float16),
    ([130], [-1], 128, 96, 8, torch.bfloat16),
    ([300, 211, 1, 1, 257], [0, 1, 2, 3, 0], 1024, 1000, 64, torch.bfloat16),
    ([255, 1, 256, 3, 800], [2, 1, 0, -1, 2], 272, 513, 40, torch.float16),
    ([700, 1348], [1, 0], 512, 1536, 128, torch.bfloat16),
    ([1] * 64, list(range(64)), 4096, 512, 16, torch.bfloat16),
    ([5, 900, 400, 1] + [1] * 30 + [1000], [0, 1, -1, 2] + [i % 3 for i in range(30)] + [1], 384, 640, 16, torch.bfloat16),
    ([2600, 0, 2008], [0, 1, 1], 256, 4104, 32, torch.float16),
    ([33, 44], [0, 0], 64, 40, 1024, torch.bfloat16),
    # 256-wide tiles: dense and chunked ones side by side, ranks of several slabs, a batch of chunks only, the shortest rows
    ([1] * 300 + [900], [i % 20 for i in range(300)] + [3], 256, 4096, 24, torch.bfloat16),
    ([300, 5, 295], [1, -1, 0], 192, 4104, 264, torch.float16),
    ([100, 60, 40], [0, -1, 1], 64, 24576, 16, torch.bfloat16),
    ([2000, 1, 559], [0, 1, 0], 16, 2049, 8, torch.bfloat16),
    ([256], [0], 4224, 64, 128, torch.bfloat16),
    # sixteen adapters in a tile, some with a few rows: on wide tiles, on narrow ones, without a full tile of rows
    ([1] * 10 + [240, 3, 8, 9, 700], [*range(10), 10, 11, 12, 13, 14], 512, 12288, 72, torch.bfloat16),
    ([20] * 8 + [8] * 8 + [40], [*range(16), -1], 320, 336, 16, torch.float16),
    ([9, 8] * 8 + [1300], [*range(16), 3], 256, 4104, 136, torch.float16),
]


@pytest.mark.parametrize("case", range(len(LINEAR)))
@pytest.mark.parametrize("per_channel,bias", [(True, True), (False, False)])
def test_linear_lora_requests(cuda_pkg, case, per_channel, bias):
    F, nat = cuda_pkg.functional, cuda_pkg._native
    lengths, adapters, K, N, r, dtype = LINEAR[case]
    rows = cuda_pkg.adapters.RequestRows(lengths, adapters, DEV)
    w, ws, b, la, lb = layer(K, N, r, max(adapters) + 1 or 1, dtype, 100 + case, per_channel, bias)
    x = torch.randn(rows.total, K, generator=gen(case), device=DEV).to(dtype)
    at = adapter_rows(rows)
    y = F.linear_lora_requests(x, w, ws, b, la, lb, rows, dtype)
    q, qs = F.quantize_rowwise(x)
    base, base_tol = base_quantised(q, qs, w, ws, b)
    term, term_tol = low_rank(x, la, lb, at, dtype)
    # the term is accumulated onto the base, sixteen ranks at a time: r / 16 fp32 additions (one more for a part of sixteen), each
    # off by at most a unit in the last place (2 E32) of what has been added up
    steps = r // 16 + 1
    want, off = base + term, base_tol + term_tol + 2 * steps * E32 * (base.abs() + term.abs())
    check(y, want, off + u_of(dtype) * (want.abs() + off) + TINY[dtype])
    # the parts: t of the rows without an adapter is zero; pitched activations give the same bits
    t = F.lora_down_requests(x, la, rows)
    assert not t[at < 0].any()
    assert torch.equal(F.linear_w8a8_lora_requests(q, qs, w, ws, b, t, lb, rows, dtype), y)
    wide = torch.full((rows.total, K + 24), float("nan"), dtype=dtype, device=DEV)
    wide[:, 8:8 + K] = x
    assert torch.equal(F.linear_lora_requests(wide[:, 8:8 + K], w, ws, b, la, lb, rows, dtype), y)
    # the reference's roundings: of the base, of the bias sum, of the low-rank term, of their sum
    y2 = F.linear_lora_requests(x, w, ws, b, la, lb, rows, dtype, order=nat.EPI_PYTORCH)
    u = u_of(dtype)
    mag = (base.abs() + (b.to(F64).abs() * 2 if b is not None else 0) + base_tol) * (2 * u + u * u) + (term.abs() + term_tol) * u
    check(y2, want, off + mag + u * (want.abs() + off + mag) + 4 * TINY[dtype])


@pytest.mark.parametrize("lengths,N", [([40, 600, 1, 7], 768), ([40, 900, 300, 7], 4096), ([3, 20, 1, 7], 520)])
def test_rows_without_adapter_are_the_plain_linear(cuda_pkg, lengths, N):
    F, nat = cuda_pkg.functional, cuda_pkg._native
    adapters = [-1, 0, -1, 1]
    rows = cuda_pkg.adapters.RequestRows(lengths, adapters, DEV)
    w, ws, b, la, lb = layer(512, N, 16, 2, torch.bfloat16, 7)
    x = torch.randn(rows.total, 512, generator=gen(8), device=DEV).bfloat16()
    none = adapter_rows(rows) < 0
    for order in (nat.EPI_SINGLE, nat.EPI_PYTORCH):
        y = F.linear_lora_requests(x, w, ws, b, la, lb, rows, torch.bfloat16, order=order)
        assert torch.equal(y[none], F.linear_forward(x, w, ws, b, torch.bfloat16, order=order)[none])


@pytest.mark.parametrize("lengths,N", [([1, 3, 40, 300, 1, 200], 320), ([1, 3, 2, 5, 1, 4], 320), ([1, 300, 40, 600, 1, 400], 4096),
                                       ([1, 3, 40, 3, 1, 20], 320)])
def test_nothing_leaks_between_requests(cuda_pkg, lengths, N):
    """An adapter of infinities and NaN, and non-finite activations, reach the rows of their own request only."""
    F = cuda_pkg.functional
    adapters = [0, 1, -1, 2, 0, 1]
    rows = cuda_pkg.adapters.RequestRows(lengths, adapters, DEV)
    w, ws, b, la, lb = layer(256, N, 16, 3, torch.bfloat16, 17)
    x = torch.randn(rows.total, 256, generator=gen(18), device=DEV).bfloat16()
    call = F.linear_small_batch_lora_requests if rows.total <= 16 else (lambda *a: F.linear_lora_requests(*a, torch.bfloat16))
    clean = call(x, w, ws, b, la, lb, rows)
    la2, lb2 = la.clone(), lb.clone()
    la2[1, 3] = float("inf")
    lb2[1, :, 5] = float("nan")
    y = call(x, w, ws, b, la2, lb2, rows)
    at = adapter_rows(rows)
    assert torch.equal(y[at != 1], clean[at != 1])
    assert y[at == 1].isnan().all()
    x2 = x.clone()
    x2[0, 7] = float("inf")          # the first request's only row
    y = call(x2, w, ws, b, la, lb, rows)
    assert torch.equal(y[1:], clean[1:]) and not y[0].isfinite().any()


@pytest.mark.parametrize("lengths,N,hadamard,rotated", [
    ([3, 1, 40, 9], 320, False, True), ([300, 5, 40, 200], 320, False, True), ([300, 500, 40, 900], 4096, False, True),
    ([3, 1, 40, 9], 320, True, True), ([3, 1, 40, 9], 320, True, False), ([300, 5, 40, 200], 320, True, True),
    ([300, 500, 40, 900], 4096, True, True), ([300, 500, 40, 900], 4096, True, False),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_nan_activations_stay_nan(cuda_pkg, lengths, N, hadamard, rotated, dtype):
    """A NaN in a row's activations makes that row NaN, with an adapter and without one, and no other."""
    F, nat = cuda_pkg.functional, cuda_pkg._native
    rows = cuda_pkg.adapters.RequestRows(lengths, [-1, 0, 1, -1], DEV)
    w, ws, b, la, lb = layer(256, N, 16, 2, dtype, 57)
    x = torch.randn(rows.total, 256, generator=gen(58), device=DEV).to(dtype)
    bad = torch.zeros(rows.total, dtype=torch.bool, device=DEV)
    x2 = x.clone()
    for m, k in ((1, 7), (lengths[0] + lengths[1] + 3, 255), (rows.total - 1, 128)):
        x2[m, k] = float("nan")
        bad[m] = True
    for order in (nat.EPI_SINGLE, nat.EPI_PYTORCH):
        clean, y = (F.linear_lora_requests(v, w, ws, b, la, lb, rows, dtype, hadamard=hadamard, rotated_lora_input=rotated, order=order)
                    for v in (x, x2))
        assert y[bad].isnan().all()
        assert torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("rotated", [True, False])
def test_linear_lora_requests_rotated(cuda_pkg, rotated):
    F = cuda_pkg.functional
    rows = cuda_pkg.adapters.RequestRows([30, 1, 400], [1, 0, 1], DEV)
    w, ws, b, la, lb = layer(512, 264, 16, 2, torch.bfloat16, 27)
    x = torch.randn(rows.total, 512, generator=gen(28), device=DEV).bfloat16()
    q, qs, xr = F.quantize_rowwise(x, hadamard=True, return_rotated=True)
    y = F.linear_lora_requests(x, w, ws, b, la, lb, rows, torch.bfloat16, hadamard=True, rotated_lora_input=rotated)
    t = F.lora_down_requests(xr if rotated else x, la, rows)
    assert torch.equal(y, F.linear_w8a8_lora_requests(q, qs, w, ws, b, t, lb, rows, torch.bfloat16))


@pytest.mark.parametrize("lengths,adapters", [([9, 8], [0, 1]), ([1] * 30 + [70, 100], [i % 3 - 1 for i in range(30)] + [0, 2]), ([255], [1])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_lora_requests_plain_adapter_input_beside_rotated_rows(cuda_pkg, lengths, adapters, dtype):
    """17 to 255 rows whose quantiser rotates while the adapters see the activations as they came."""
    F = cuda_pkg.functional
    rows = cuda_pkg.adapters.RequestRows(lengths, adapters, DEV)
    w, ws, b, la, lb = layer(640, 328, 24, 3, dtype, 29)
    x = torch.randn(rows.total, 640, generator=gen(30), device=DEV).to(dtype)
    y = F.linear_lora_requests(x, w, ws, b, la, lb, rows, dtype, hadamard=True, rotated_lora_input=False)
    q, qs = F.quantize_rowwise(x, hadamard=True)
    assert torch.equal(y, F.linear_w8a8_lora_requests(q, qs, w, ws, b, F.lora_down_requests(x, la, rows), lb, rows, dtype))
    base, base_tol = base_quantised(q, qs, w, ws, b)
    term, term_tol = low_rank(x, la, lb, adapter_rows(rows), dtype)
    want, off = base + term, base_tol + term_tol + 2 * 3 * E32 * (base.abs() + term.abs())      # two additions of sixteen ranks, one more
    check(y, want, off + u_of(dtype) * (want.abs() + off) + TINY[dtype])


SMALL = [
    ([1], [0], 64, 16, 8, torch.bfloat16), ([1], [-1], 64, 24, 8, torch.bfloat16), ([16], [1], 1040, 333, 24, torch.float16),
    ([1] * 16, [i % 7 - 1 for i in range(16)], 4096, 1000, 32, torch.bfloat16), ([3, 0, 5, 1], [0, 1, -1, 2], 256, 77, 128, torch.float16),
    ([8], [0], 80, 2064, 16, torch.bfloat16), ([9, 2], [3, 0], 128, 40, 64, torch.bfloat16), ([5], [0], 4096, 4096, 1024, torch.float16),
]


@pytest.mark.parametrize("case", range(len(SMALL)))
@pytest.mark.parametrize("per_channel,bias", [(True, True), (False, False)])
def test_linear_small_batch_lora_requests(cuda_pkg, case, per_channel, bias):
    F = cuda_pkg.functional
    lengths, adapters, K, N, r, dtype = SMALL[case]
    rows = cuda_pkg.adapters.RequestRows(lengths, adapters, DEV)
    w, ws, b, la, lb = layer(K, N, r, max(adapters) + 1 or 1, dtype, 200 + case, per_channel, bias)
    x = torch.randn(rows.total, K, generator=gen(case), device=DEV).to(dtype)
    y = F.linear_small_batch_lora_requests(x, w, ws, b, la, lb, rows)
    s = ws.to(F64).reshape(1, -1)
    base = (x.to(F64) @ w.to(F64).T) * s
    off = (2 * K + 4) * E32 * (x.to(F64).abs() @ w.to(F64).abs().T) * s      # fp32 sums of exact products, in any order
    if b is not None:
        base = base + b.to(F64)
        off = off + E32 * base.abs()
    term, term_tol = low_rank(x, la, lb, adapter_rows(rows), dtype)
    want, off = base + term, off + term_tol + 2 * E32 * (base.abs() + term.abs())
    check(y, want, off + u_of(dtype) * (want.abs() + off) + TINY[dtype])
    wide = torch.full((rows.total, K + 8), float("nan"), dtype=dtype, device=DEV)
    wide[:, :K] = x
    assert torch.equal(F.linear_small_batch_lora_requests(wide[:, :K], w, ws, b, la, lb, rows), y)


def test_adapter_calls_refuse(cuda_pkg):
    F, E = cuda_pkg.functional, cuda_pkg._native.NativeLibraryError
    Rows = cuda_pkg.adapters.RequestRows
    rows = Rows([20, 4], [0, 1], DEV)
    w, ws, b, la, lb = layer(128, 64, 16, 2, torch.bfloat16, 3)
    x = torch.zeros(24, 128, dtype=torch.bfloat16, device=DEV)
    ok = dict(x=x, w=w, w_scale=ws, bias=b, lora_a=la, lora_b=lb, rows=rows, out_dtype=torch.bfloat16)
    assert F.linear_lora_requests(**ok).shape == (24, 64)
    for bad in (dict(x=x[:23]), dict(rows=Rows([20, 3], [0, 1], DEV)), dict(rows=Rows([20, 4], [0, 2], DEV)), dict(rows=Rows([24], [0], "cpu")),
                dict(out_dtype=torch.float16), dict(x=x.half(), out_dtype=torch.float16), dict(lora_a=la[:1]), dict(lora_a=la.half()),
                dict(lora_b=lb[:, :63]), dict(lora_b=lb.transpose(1, 2)), dict(lora_a=la[:, :, ::2]), dict(lora_a=la[0]),
                dict(lora_b=lb.cpu()), dict(bias=b[:5]), dict(w_scale=ws[:5]), dict(w=w.cpu()), dict(w=w[:, :64])):
        with pytest.raises((ValueError, E)):
            F.linear_lora_requests(**{**ok, **bad})
    odd = layer(128, 64, 12, 2, torch.bfloat16, 3)
    with pytest.raises(E, match="multiple of 8"):
        F.linear_lora_requests(**{**ok, "lora_a": odd[3], "lora_b": odd[4]})
    with pytest.raises(E, match="16 rows"):
        F.linear_small_batch_lora_requests(x, w, ws, b, la, lb, rows)
    assert F.linear_lora_requests(**{**ok, "x": x[:0], "rows": Rows([0], [0], DEV)}).shape == (0, 64)
    assert F.linear_small_batch_lora_requests(x[:0], w, ws, b, la, lb, Rows([0, 0], [1, 0], DEV)).shape == (0, 64)


# ------------------------------------------------------------------ gated residual update between two norms
def ref_norm(v, off, kind, weight, eps):
    """The norm in 64 bits and its error from an input that is `off` wrong: fp32 row sums of at most 64 additions in a chain
    (32 elements per thread, five shuffles, sixteen warps) plus a handful of operations."""
    if kind is None:
        return v, off
    n = 80 * E32
    if kind == "layer":
        mean = v.mean(1, keepdim=True)
        off = off + off.mean(1, keepdim=True) + n * v.abs().mean(1, keepdim=True) + 2 * E32 * v.abs()
        v = v - mean
    ms = (v * v).mean(1, keepdim=True)
    ms_off = (2 * v.abs() * off + off * off).mean(1, keepdim=True) + n * ms
    root = torch.sqrt(ms + eps)
    r = 1 / root
    r_off = r * (ms_off / (ms + eps) + 6 * E32)
    out, off = v * r, off * (r + r_off) + v.abs() * r_off + 2 * E32 * v.abs() * r
    if weight is not None:
        w = weight.to(F64)
        out, off = out * w, off * w.abs() + E32 * (out * w).abs()
    return out, off


def ref_update(x, y, gate, scale, shift, at, gate_tanh, residual_scale, post, post_weight, norm, weight, eps):
    zero = torch.zeros_like(x, dtype=F64)
    p, p_off = ref_norm(y.to(F64), zero, post, post_weight if post else None, eps)
    g = torch.ones_like(zero) if gate is None else gate.to(F64)[at]
    g_off = 0.0
    if gate_tanh:
        g = torch.tanh(g)
        g_off = 4 * E32 * g.abs()          # CUDA's tanhf: at most two units in the last place
    c = float(torch.tensor(residual_scale, dtype=torch.float32))
    xn = c * x.to(F64) + g * p
    x_off = g.abs() * p_off + g_off * (p.abs() + p_off) + 2 * E32 * ((c * x.to(F64)).abs() + (g * p).abs() + xn.abs())
    h, h_off = ref_norm(xn, x_off, norm, weight, eps)
    s = 1 + (0 if scale is None else scale.to(F64)[at])
    t = 0 if shift is None else shift.to(F64)[at]
    out = h * s + t
    return xn, x_off, out, h_off * abs(s) + 3 * E32 * ((h * s).abs() + out.abs())


NORM = [
    # lengths, K, y dtype, x dtype, post, norm, tanh, weights, scale, shift, gate, residual_scale
    ([1], 8, torch.bfloat16, torch.bfloat16, "rms", "rms", True, True, True, False, True, 1.0),
    ([1], 1, torch.float16, torch.float16, "rms", "rms", False, True, True, True, True, 0.5),
    ([3, 0, 2], 4096, torch.bfloat16, torch.bfloat16, None, "layer", False, False, True, True, True, 1.0),
    ([70, 1, 30], 2305, torch.float16, torch.float16, "layer", "layer", False, True, True, True, True, 0.7),
    ([5, 6], 16384, torch.bfloat16, torch.float32, "rms", "layer", True, True, True, True, True, 1.0),
    ([4, 1], 16383, torch.bfloat16, torch.float32, "layer", "rms", False, True, False, True, True, -2.0),
    ([9], 12, torch.float16, torch.float32, "layer", "rms", False, False, False, False, False, 1.0),
    ([2] * 50, 1152, torch.bfloat16, torch.bfloat16, "rms", "rms", True, True, True, False, True, 1.0),
    ([600, 500, 1], 520, torch.float16, torch.float16, "rms", "layer", False, True, True, True, True, 0.0),
    ([257, 1024], 6144, torch.bfloat16, torch.bfloat16, "rms", "rms", True, False, True, True, True, 1.0),
    ([33], 8200, torch.bfloat16, torch.bfloat16, None, "rms", False, True, True, False, True, 1.0),
    ([2000, 1, 999, 1700], 4096, torch.bfloat16, torch.bfloat16, "rms", "rms", True, True, True, False, True, 1.0),
    # many rows whose length eight does not divide: they start anywhere between two 16-byte boundaries
    ([300, 0, 477], 2305, torch.float16, torch.float16, "layer", "layer", False, True, True, True, True, 0.5),
    ([1000, 3], 1027, torch.bfloat16, torch.float32, "rms", "layer", True, True, True, True, True, 1.0),
    ([1, 400], 4094, torch.bfloat16, torch.bfloat16, None, "rms", False, False, True, False, True, 1.0),
    ([700], 4101, torch.float16, torch.float32, "layer", "rms", True, True, False, True, False, 1.0),
    ([300], 9001, torch.bfloat16, torch.bfloat16, "rms", "rms", True, True, True, True, True, 1.0),
    ([260], 12287, torch.float16, torch.float16, "rms", "layer", False, True, True, True, True, 1.0),
    # many rows of other lengths: a warp each, a group each, one row of the ring at a time
    ([500, 800], 64, torch.bfloat16, torch.float32, "rms", "layer", True, True, True, True, True, 1.0),
    ([999], 1016, torch.float16, torch.float16, "layer", "rms", False, True, True, True, True, 1.0),
    ([400, 111], 251, torch.bfloat16, torch.bfloat16, "layer", "layer", False, True, True, True, True, 1.0),
    ([256], 8192, torch.bfloat16, torch.float32, "layer", "layer", False, True, True, True, True, 1.0),
    ([310], 12288, torch.bfloat16, torch.bfloat16, "rms", "rms", True, True, True, True, True, 1.0),
    ([280], 16384, torch.float16, torch.float16, "rms", "layer", False, True, True, True, True, 1.0),
    ([1] * 600, 2048, torch.bfloat16, torch.bfloat16, "rms", "rms", True, True, True, False, True, 1.0),
]


def norm_inputs(case, seed):
    lengths, K, dt, xdt, post, norm, tanh, weights, scale, shift, gate, c = NORM[case]
    g = gen(seed)
    M, R = sum(lengths), len(lengths)
    x = (torch.randn(M, K, generator=g, device=DEV) * 3 + 0.5).to(xdt)
    y = (torch.randn(M, K, generator=g, device=DEV) + 0.25).to(dt)
    mod = (torch.randn(R, 3 * K, generator=g, device=DEV) * 0.5).to(dt)     # pitched slices, as a modulation layer gives them
    kw = dict(gate_tanh=tanh, residual_scale=c, post_norm=post, norm=norm, eps=1e-5,
              post_weight=(torch.randn(K, generator=g, device=DEV) + 1).to(dt) if weights and post else None,
              weight=(torch.randn(K, generator=g, device=DEV) + 1).to(dt) if weights else None,
              scale=mod[:, :K] if scale else None, shift=mod[:, K:2 * K] if shift else None)
    return lengths, x, y, mod[:, 2 * K:] if gate else None, kw


@pytest.mark.parametrize("case", range(len(NORM)))
def test_gated_residual_norm(cuda_pkg, case):
    F = cuda_pkg.functional
    lengths, x, y, gate, kw = norm_inputs(case, 300 + case)
    rows = cuda_pkg.adapters.RequestRows(lengths, None, DEV)
    at = torch.tensor([i for i, n in enumerate(lengths) for _ in range(n)], device=DEV)
    xn, xn_off, hn, hn_off = ref_update(x, y, gate, kw["scale"], kw["shift"], at, kw["gate_tanh"], kw["residual_scale"], kw["post_norm"],
                                        kw["post_weight"], kw["norm"], kw["weight"], kw["eps"])
    x0 = x.clone()
    x_new, h = F.gated_residual_norm(x, y, gate, rows=rows, **kw)
    assert torch.equal(x, x0) and x_new.dtype == x.dtype and h.dtype == y.dtype
    check(x_new, xn, xn_off + u_of(x.dtype) * (xn.abs() + xn_off) + TINY[x.dtype])
    check(h, hn, hn_off + u_of(h.dtype) * (hn.abs() + hn_off) + TINY[h.dtype])
    # int8: half a step, the error of h, three fp32 roundings of a value of up to 127.5 steps
    x_q, q, qs, h_q = F.quantize_rowwise_gated_residual_norm(x, y, gate, rows=rows, return_h=True, **kw)
    assert torch.equal(x_q, x_new) and torch.equal(h_q, h)
    step = qs.to(F64)
    amax, amax_off = hn.abs().amax(1, keepdim=True), hn_off.amax(1, keepdim=True)
    check(step, (amax / 127).clamp_min(1e-30), amax_off / 127 + 2 * E32 * amax / 127 + 1e-37)
    check(q.to(F64) * step, hn, step / 2 + hn_off + 128 * 4 * E32 * step + 127 * amax_off / 127)
    x_q2, q2, qs2 = F.quantize_rowwise_gated_residual_norm(x, y, gate, rows=rows, **kw)
    assert torch.equal(x_q2, x_new) and torch.equal(q2, q) and torch.equal(qs2, qs)
    # in place, and with the rows of a wider buffer: the same bits, nothing written beside them
    wide = torch.full((x.shape[0], x.shape[1] + 16), 7.0, dtype=x.dtype, device=DEV)
    view = wide[:, 8:8 + x.shape[1]]
    view.copy_(x)
    out, h2 = F.gated_residual_norm(view, y, gate, rows=rows, x_out=view, **kw)
    assert out is view and torch.equal(view, x_new) and torch.equal(h2, h)
    assert (wide[:, :8] == 7).all() and (wide[:, 8 + x.shape[1]:] == 7).all()


def test_gated_residual_norm_shared_vectors(cuda_pkg):
    """One vector for all rows, given as [K], as [1, K], or repeated per request: the same bits."""
    F = cuda_pkg.functional
    g = gen(5)
    x, y = (torch.randn(50, 264, generator=g, device=DEV).bfloat16() for _ in range(2))
    gate, scale = (torch.randn(264, generator=g, device=DEV).bfloat16() for _ in range(2))
    rows = cuda_pkg.adapters.RequestRows([20, 30], None, DEV)
    want = F.gated_residual_norm(x, y, gate, scale=scale, norm="layer")
    for got in (F.gated_residual_norm(x, y, gate[None], scale=scale[None], norm="layer", rows=rows),
                F.gated_residual_norm(x, y, gate.repeat(2, 1), scale=scale, norm="layer", rows=rows),
                F.gated_residual_norm(x, y, gate.repeat(2, 1), scale=scale.expand(2, 264), norm="layer", rows=rows)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("M,K,dt,xdt", [(6, 512, torch.bfloat16, torch.bfloat16), (5, 2305, torch.float16, torch.float32), (300, 256, torch.bfloat16, torch.float32),
                                        (300, 4096, torch.bfloat16, torch.bfloat16), (300, 2305, torch.float16, torch.float16),
                                        (260, 16384, torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("with_gate", [True, False])
def test_gated_residual_norm_weight_without_post_norm(cuda_pkg, M, K, dt, xdt, with_gate):
    """A weight behind the branch that no norm precedes (a layer scale): x' = c x + g y w, by every kernel."""
    F = cuda_pkg.functional
    g = gen(K)
    x, y = (torch.randn(M, K, generator=g, device=DEV) * 3).to(xdt), torch.randn(M, K, generator=g, device=DEV).to(dt)
    w, weight = ((torch.randn(K, generator=g, device=DEV) + 1).to(dt) for _ in range(2))
    lengths = [M // 2, M - M // 2]
    rows = cuda_pkg.adapters.RequestRows(lengths, None, DEV)
    gate = torch.randn(2, K, generator=g, device=DEV).to(dt) if with_gate else None
    x_new, h = F.gated_residual_norm(x, y, gate, rows=rows, residual_scale=0.5, post_weight=w, norm="layer", weight=weight, eps=1e-5)
    at = torch.repeat_interleave(torch.arange(2, device=DEV), torch.tensor(lengths, device=DEV))
    term = y.to(F64) * w.to(F64) * (gate.to(F64)[at] if with_gate else 1.0)
    xn = 0.5 * x.to(F64) + term
    xn_off = E32 * (2 * term.abs() + xn.abs())          # two products (0.5 x is exact) and their sum, in fp32
    check(x_new, xn, xn_off + u_of(xdt) * (xn.abs() + xn_off) + TINY[xdt])
    hn, hn_off = ref_norm(xn, xn_off, "layer", weight, 1e-5)
    check(h, hn, hn_off + u_of(dt) * (hn.abs() + hn_off) + TINY[dt])
    x_q, q, qs = F.quantize_rowwise_gated_residual_norm(x, y, gate, rows=rows, residual_scale=0.5, post_weight=w, norm="layer", weight=weight,
                                                        eps=1e-5)
    assert torch.equal(x_q, x_new)


@pytest.mark.parametrize("M,K,dt", [(40, 512, torch.bfloat16), (40, 509, torch.float16), (600, 256, torch.float16), (600, 4096, torch.bfloat16),
                                    (600, 2305, torch.bfloat16)])
def test_int8_rows_of_the_residual_norm_are_the_quantisers(cuda_pkg, M, K, dt):
    """A scale of -1 leaves h = shift, exactly: its int8 form has the bits that the quantiser gives the same rows, a step of
    absmax / 127 rounded once."""
    F = cuda_pkg.functional
    g = gen(K + M)
    x, y, shift = (torch.randn(M, K, generator=g, device=DEV).to(dt) for _ in range(3))
    rows = cuda_pkg.adapters.RequestRows([1] * M, None, DEV)
    shared = cuda_pkg.adapters.RequestRows([M // 4] * 4, None, DEV)
    one = torch.full((K,), -1.0, dtype=dt, device=DEV)
    for plan, t, at in ((rows, shift, torch.arange(M, device=DEV)), (shared, shift[:4], torch.arange(M, device=DEV) // (M // 4))):
        _, q, qs, h = F.quantize_rowwise_gated_residual_norm(x, y, rows=plan, scale=one, shift=t, return_h=True)
        assert torch.equal(h, t[at])
        amax = h.float().abs().amax(1, keepdim=True)
        step = torch.div(amax, torch.full_like(amax, 127.0))       # by a tensor: a division, not a product with 1 / 127
        assert torch.equal(qs, step)
        assert torch.equal(q, torch.round(h.float() * torch.div(torch.ones_like(step), step)).to(torch.int8))
        if K % 16 == 0:
            want_q, want_s = F.quantize_rowwise(h)
            assert torch.equal(q, want_q) and torch.equal(qs, want_s)


def test_gated_residual_norm_special_rows(cuda_pkg):
    """Constant and zero rows are what eps makes of them; a NaN or an infinity stays in its row and shows in its scale."""
    F = cuda_pkg.functional
    x = torch.zeros(6, 512, dtype=torch.bfloat16, device=DEV)
    y = torch.zeros_like(x)
    x[1] = 3.0
    x[2, 9] = float("nan")
    y[3, 100] = float("inf")
    x[4] = torch.randn(512, generator=gen(1), device=DEV).bfloat16()
    for norm in ("rms", "layer"):
        x_new, q, qs, h = F.quantize_rowwise_gated_residual_norm(x, y, post_norm="rms", norm=norm, return_h=True)
        assert not h[0].any() and not q[0].any() and float(qs[0]) == float(torch.tensor(1e-30))
        if norm == "layer":
            assert not h[1].any()
        else:
            check(h[1].to(F64), torch.ones(512, dtype=F64, device=DEV), 2.0 ** -8)
        assert h[2].isnan().all() and qs[2].isnan().all() and x_new[2].isnan().sum() == 1
        assert not h[3].isfinite().any() and not qs[3].isfinite().any()
        assert h[4:].isfinite().all() and qs[4:].isfinite().all() and not h[5].any()


@pytest.mark.parametrize("K,xdt", [(4096, torch.float32), (4096, torch.bfloat16), (2305, torch.bfloat16), (8192, torch.bfloat16)])
def test_gated_residual_norm_many_launches(cuda_pkg, K, xdt):
    """Rows arrive in any order and every launch gives the same bits (the fixture checks that no wait ran out)."""
    F = cuda_pkg.functional
    g = gen(13)
    x, y = torch.randn(9000, K, generator=g, device=DEV).to(xdt), torch.randn(9000, K, generator=g, device=DEV).bfloat16()
    mod = torch.randn(3, K, generator=g, device=DEV).bfloat16()
    rows = cuda_pkg.adapters.RequestRows([4000, 1, 4999], None, DEV)
    want = F.gated_residual_norm(x, y, mod, rows=rows, post_norm="rms", norm="layer")
    wrong = torch.zeros((), dtype=torch.int64, device=DEV)
    for _ in range(400):
        got = F.gated_residual_norm(x, y, mod, rows=rows, post_norm="rms", norm="layer")
        wrong += (got[0] != want[0]).any() | (got[1] != want[1]).any()
    assert int(wrong) == 0


def test_gated_residual_norm_refuses(cuda_pkg):
    F, E = cuda_pkg.functional, cuda_pkg._native.NativeLibraryError
    Rows = cuda_pkg.adapters.RequestRows
    x = torch.zeros(6, 64, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(64, dtype=torch.bfloat16, device=DEV)
    rows = Rows([2, 4], None, DEV)
    for args, kw in (((x, x[:5]), {}), ((x.half(), x), {}), ((x, x.float()), {}), ((x[0], x[0]), {}), ((x, x.cpu()), {}),
                     ((x, x, v[:63]), {}), ((x, x, v.repeat(3, 1)), dict(rows=rows)), ((x, x, v.repeat(2, 1)), {}),
                     ((x, x), dict(norm=None)), ((x, x), dict(norm="group")), ((x, x), dict(post_norm="batch")), ((x, x), dict(weight=v[:5])),
                     ((x, x), dict(rows=Rows([5], None, DEV))), ((x, x), dict(rows=Rows([6], None, "cpu"))),
                     ((x, x), dict(x_out=x[:5])), ((x, x), dict(x_out=x.float())), ((x, x), dict(x_out=x.t().contiguous().t())),
                     ((x, x), dict(x_out=v.expand(6, 64))), ((x, x), dict(eps=-1.0)),
                     ((x.new_zeros(2, 16392), x.new_zeros(2, 16392)), {})):
        with pytest.raises((ValueError, E)):
            F.gated_residual_norm(*args, **kw)
    for M, K in ((0, 64), (4, 0)):
        e = x.new_zeros(M, K)
        x_new, h = F.gated_residual_norm(e, e)
        assert x_new.shape == h.shape == (M, K)


def test_gated_residual_norm_into_shared_memory(cuda_pkg):
    """x_out as y, as another view of x, as the columns beside x: the bits of a call into memory of its own.  Rows that overlap
    otherwise are refused."""
    F = cuda_pkg.functional
    for M, K in ((9, 264), (700, 2048), (700, 1001)):
        g = gen(M + K)
        x, y = (torch.randn(M, K, generator=g, device=DEV).bfloat16() for _ in range(2))
        want = F.gated_residual_norm(x, y, post_norm="rms")
        y2 = y.clone()
        got = F.gated_residual_norm(x, y2, post_norm="rms", x_out=y2)
        assert torch.equal(y2, want[0]) and torch.equal(got[1], want[1])
        wide = torch.zeros(M + 1, 2 * K, dtype=torch.bfloat16, device=DEV)
        left, right = wide[:M, :K], wide[:M, K:]
        left.copy_(x)
        # the same rows at the same places: rows that lie otherwise to one another may be another kernel's, with sums in another order
        want = F.gated_residual_norm(left, y, post_norm="rms")
        got = F.gated_residual_norm(left, y, post_norm="rms", x_out=right)
        assert torch.equal(right, want[0]) and torch.equal(got[1], want[1]) and torch.equal(left, x)
        got = F.gated_residual_norm(left, y, post_norm="rms", x_out=wide[:M, :K])
        assert torch.equal(left, want[0]) and torch.equal(got[1], want[1])
        for out in (wide[1:, :K], wide[:M, 1:K + 1]):
            with pytest.raises(ValueError, match="share memory"):
                F.gated_residual_norm(left, y, x_out=out)
            with pytest.raises(ValueError, match="share memory"):
                F.gated_residual_norm(x, left, x_out=out)


# ------------------------------------------------------------------ together, streams, graphs, long offsets
def block_step(pkg, s):
    """A residual update with its int8 output and the quantised projection with adapters that follows it, as a block runs them."""
    F = pkg.functional
    x, q, qs, h = F.quantize_rowwise_gated_residual_norm(s["x"], s["y"], s["gate"], rows=s["rows"], post_norm="rms", norm="layer",
                                                         scale=s["scale"], shift=s["shift"], return_h=True)
    t = F.lora_down_requests(h, s["la"], s["rows"])
    return x, F.linear_w8a8_lora_requests(q, qs, s["w"], s["ws"], s["b"], t, s["lb"], s["rows"], torch.bfloat16)


def block_state(pkg, lengths, adapters, K, N, r, seed):
    g = gen(seed)
    M, R = sum(lengths), len(lengths)
    w, ws, b, la, lb = layer(K, N, r, max(adapters) + 1, torch.bfloat16, seed)
    mod = (torch.randn(R, 3 * K, generator=g, device=DEV) * 0.3).bfloat16()
    return dict(x=torch.randn(M, K, generator=g, device=DEV).bfloat16(), y=torch.randn(M, K, generator=g, device=DEV).bfloat16(),
                gate=mod[:, :K], scale=mod[:, K:2 * K], shift=mod[:, 2 * K:], w=w, ws=ws, b=b, la=la, lb=lb,
                rows=pkg.adapters.RequestRows(lengths, adapters, DEV))


BLOCKS = [([40, 1, 1, 1, 86], [0, 1, -1, 2, 1]), ([700, 1, 1, 1400], [1, 0, 2, 2]), ([1] * 40 + [1500], [i % 9 for i in range(40)] + [8])]


@pytest.mark.parametrize("lengths,adapters", BLOCKS)
def test_block_of_operators(cuda_pkg, lengths, adapters):
    s = block_state(cuda_pkg, lengths, adapters, 1024, 1536, 16, 61)
    x, y = block_step(cuda_pkg, s)
    at = torch.tensor([i for i, n in enumerate(lengths) for _ in range(n)], device=DEV)
    xn, xn_off, hn, hn_off = ref_update(s["x"], s["y"], s["gate"], s["scale"], s["shift"], at, False, 1.0, "rms", None, "layer", None, 1e-6)
    check(x, xn, xn_off + u_of(x.dtype) * (xn.abs() + xn_off))
    u = u_of(torch.bfloat16)
    w = s["w"].to(F64) * s["ws"].to(F64)
    step = (hn.abs() + hn_off).amax(1, keepdim=True) / 127
    q_off = step * 0.51 + 2 * hn_off.amax(1, keepdim=True)
    term, term_tol = low_rank(hn, s["la"], s["lb"], adapter_rows(s["rows"]), torch.bfloat16)
    h_off = hn_off + u * (hn.abs() + hn_off)
    for a in range(max(adapters) + 1):        # h is rounded to 16 bits before the adapters
        m = adapter_rows(s["rows"]) == a
        term_tol[m] += 1.01 * (h_off[m] @ s["la"][a].to(F64).abs().T) @ s["lb"][a].to(F64).abs().T
    want = hn @ w.T + s["b"].to(F64) + term
    off = (q_off @ torch.ones(1, w.shape[1], dtype=F64, device=DEV)) @ w.abs().T + term_tol + 8 * E32 * (hn.abs() @ w.abs().T)
    check(y, want, off + u * (want.abs() + off))


def test_two_graphs_and_a_side_stream(cuda_pkg):
    states = [block_state(cuda_pkg, *BLOCKS[i], 512, 640, 24, 70 + i) for i in range(2)]
    want = [block_step(cuda_pkg, s) for s in states]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [block_step(cuda_pkg, s) for s in states]
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block_step(cuda_pkg, s))
        graphs.append(g)
    side.synchronize()
    for w, o in zip(want, got):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])
    for order in ((0, 1), (1, 0, 0)):
        for i in order:
            graphs[i].replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])
    # new values in the captured inputs
    states[0]["x"].add_(1.0)
    graphs[0].replay()
    again = block_step(cuda_pkg, states[0])
    assert torch.equal(again[0], outs[0][0]) and torch.equal(again[1], outs[0][1]) and not torch.equal(again[0], want[0][0])


def test_two_calls_at_once_on_two_streams(cuda_pkg):
    states = [block_state(cuda_pkg, [600, 1, 900], [0, 1, 2], 1024, 2048, 32, 80 + i) for i in range(2)]
    want = [block_step(cuda_pkg, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(block_step(cuda_pkg, states[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o[0], want[i][0]) and torch.equal(o[1], want[i][1]) for o in outs[i])


CHAINS = [
    # rows, K = N, rank, whether the form for at most 16 rows
    ([1] * 9, [0, 1, 2, -1, 0, 1, 2, 0, 1], 512, 24, True),
    ([1] * 40 + [20], [i % 3 for i in range(40)] + [2], 512, 16, False),
    ([200, 30, 100], [0, -1, 1], 512, 64, False),
    ([600, 1, 3, 900], [0, 1, 2, 2], 2048, 32, False),
]


@pytest.mark.parametrize("case", range(len(CHAINS)))
@pytest.mark.parametrize("hadamard,rotated", [(False, True), (True, True), (True, False)])
def test_whole_forwards_behind_one_another(cuda_pkg, case, hadamard, rotated):
    """The whole-forward calls overlap their kernels' tails: chained layers, each behind the kernel that makes its input and in the
    workspace of the one before, on two streams at once and as two captured graphs, give the bits of calls that wait for all else."""
    F = cuda_pkg.functional
    lengths, adapters, K, r, small = CHAINS[case]
    if small and hadamard:
        pytest.skip("the form for at most 16 rows takes rotated activations as they come")
    rows = cuda_pkg.adapters.RequestRows(lengths, adapters, DEV)

    def chain(state, wait):
        x = state["x"]
        for i, (w, ws, b, la, lb) in enumerate(state["layers"]):
            if i % 2 == 0:
                x = torch.nn.functional.rms_norm(x, (K,))
            if wait:
                torch.cuda.synchronize()
            if small:
                x = F.linear_small_batch_lora_requests(x, w, ws, b, la, lb, rows)
            else:
                x = F.linear_lora_requests(x, w, ws, b, la, lb, rows, x.dtype, hadamard=hadamard, rotated_lora_input=rotated)
        return x

    states = [dict(x=torch.randn(rows.total, K, generator=gen(900 + i), device=DEV).bfloat16(),
                   layers=[layer(K, K, r, 3, torch.bfloat16, 910 + 10 * i + j) for j in range(6)]) for i in range(2)]
    want = [chain(s, True) for s in states]
    assert all(w.isfinite().all() for w in want) and not torch.equal(*want)
    torch.cuda.synchronize()
    for s, w in zip(states, want):
        assert torch.equal(chain(s, False), w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(chain(states[i], False))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    graphs, captured = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured.append(chain(s, False))
        graphs.append(g)
    for i in (0, 1, 1, 0):
        graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(c, w) for c, w in zip(captured, want))


def test_plan_within_a_capture_leaves_the_capture_whole(cuda_pkg):
    """A plan is refused before anything reaches the device, so the capture goes on."""
    x = torch.ones(4, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="outside of a graph capture"):
            cuda_pkg.adapters.RequestRows([4], [0], DEV)
        y = x + 1
    graph.replay()
    assert (y == 2).all()


def test_plan_dropped_while_another_stream_reads_it(cuda_pkg):
    """The tables' memory is not handed on before the calls on other streams are done, whichever entry point made them."""
    F = cuda_pkg.functional
    Rows = cuda_pkg.adapters.RequestRows
    w, ws, b, la, lb = layer(512, 640, 16, 3, torch.bfloat16, 95)
    x = torch.randn(600, 512, generator=gen(96), device=DEV).bfloat16()
    y = torch.randn(600, 512, generator=gen(97), device=DEV).bfloat16()
    gate = torch.randn(3, 512, generator=gen(98), device=DEV).bfloat16()
    q, qs = F.quantize_rowwise(x)
    t = F.lora_down_requests(x, la, Rows([300, 100, 200], [0, -1, 2], DEV))
    calls = [lambda p: F.linear_lora_requests(x, w, ws, b, la, lb, p, x.dtype), lambda p: F.lora_down_requests(x, la, p),
             lambda p: F.linear_w8a8_lora_requests(q, qs, w, ws, b, t, lb, p, x.dtype),
             lambda p: F.gated_residual_norm(x, y, gate, rows=p)[1],
             lambda p: F.linear_small_batch_lora_requests(x[:9], w, ws, b, la, lb, p)]
    side = torch.cuda.Stream()
    for i, call in enumerate(calls):
        plan = Rows([3, 1, 5] if i == 4 else [300, 100, 200], [0, -1, 2], DEV)
        want = call(plan)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)        # some 30 ms
            got = call(plan)
        at, n = plan._tables.data_ptr(), plan._tables.numel()
        assert not side.query()
        del plan
        later = [torch.full((n,), 1 << 20, dtype=torch.int32, device=DEV) for _ in range(8)]
        assert all(v.data_ptr() != at for v in later)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del later


def test_offsets_past_32_bits(cuda_pkg):
    """Rows that lie further apart than 32 bits can count: 20 rows with a pitch of 2^27 elements."""
    F = cuda_pkg.functional
    M, K, pitch = 20, 256, 1 << 27
    buf = torch.empty((M - 1) * pitch + K, dtype=torch.bfloat16, device=DEV)
    far = buf.as_strided((M, K), (pitch, 1))
    x = torch.randn(M, K, generator=gen(9), device=DEV).bfloat16()
    far.copy_(x)
    rows = cuda_pkg.adapters.RequestRows([12, 8], [0, 1], DEV)
    w, ws, b, la, lb = layer(K, 64, 8, 2, torch.bfloat16, 91)
    assert torch.equal(F.linear_lora_requests(far, w, ws, b, la, lb, rows, torch.bfloat16),
                       F.linear_lora_requests(x, w, ws, b, la, lb, rows, torch.bfloat16))
    y = torch.randn(M, K, generator=gen(10), device=DEV).bfloat16()
    want = F.gated_residual_norm(x, y, post_norm="rms")
    got = F.gated_residual_norm(far, y, post_norm="rms", x_out=far)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_draws_of_row_plans(cuda_pkg):
    """Random plans, small and large, against the 64-bit forms."""
    F = cuda_pkg.functional
    rng = random.Random(11)
    for _ in range(12):
        M = rng.choice([17, 60, 256, 257, 700, 1300, 3000])
        n = rng.randint(1, min(M, 40))
        cuts = sorted(rng.randint(0, M) for _ in range(n - 1))
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [M])]
        bank = rng.randint(1, 6)
        adapters = [rng.randint(-1, bank - 1) for _ in lengths]
        K, N, r = 16 * rng.randint(1, 60), rng.randint(1, 1100), 8 * rng.randint(1, 12)
        dtype = rng.choice([torch.bfloat16, torch.float16])
        rows = cuda_pkg.adapters.RequestRows(lengths, adapters, DEV)
        w, ws, b, la, lb = layer(K, N, r, bank, dtype, rng.randint(1, 1000))
        x = torch.randn(M, K, generator=gen(M), device=DEV).to(dtype)
        y = F.linear_lora_requests(x, w, ws, b, la, lb, rows, dtype)
        base, base_tol = base_quantised(*F.quantize_rowwise(x), w, ws, b)
        term, term_tol = low_rank(x, la, lb, adapter_rows(rows), dtype)
        want, off = base + term, base_tol + term_tol + 2 * (r // 16 + 1) * E32 * (base.abs() + term.abs())
        check(y, want, off + u_of(dtype) * (want.abs() + off) + TINY[dtype])


# ------------------------------------------------------------------ the layers and the model that use them
@pytest.mark.parametrize("tokens", [1, 4, 5, 200])
@pytest.mark.parametrize("quarot", [False, True])
def test_linear_module_with_request_loras(cuda_pkg, tokens, quarot):
    """The Linear of a batch of requests gives every sample what it gives that sample's LoRA alone."""
    F, nat = cuda_pkg.functional, cuda_pkg._native
    K, N, r = 256, 320, 16
    w, ws, b, la, lb = layer(K, N, r, 3, torch.bfloat16, 41)
    lin = cuda_pkg.ops.StandaloneInt8Ops.Linear(K, N, bias=True, device="meta")
    lin._load_from_state_dict({"weight": w, "weight_scale": ws, "bias": b}, "", {}, True, [], [], [])
    lin._use_quarot = quarot
    x = torch.randn(8, tokens, K, generator=gen(42), device=DEV).bfloat16()
    lin.request_loras = cuda_pkg.adapters.RequestLoras(la, lb, [1, -1, 2, 1])
    y = lin(x)
    assert y.shape == (8, tokens, N)
    xr = cuda_pkg.quarot.rotate_activation(x.reshape(-1, K), None, 128).reshape(x.shape) if quarot else x
    u = u_of(torch.bfloat16)
    for j in range(8):
        e = (1, -1, 2, 1)[j % 4]
        at = torch.full((tokens,), e, device=DEV)
        if 8 * tokens > 16:
            base, off = base_quantised(*F.quantize_rowwise(x[j], hadamard=quarot), w, ws, b)
        else:
            base = (xr[j].to(F64) @ w.to(F64).T) * ws.to(F64).T + b.to(F64)
            off = (2 * K + 8) * E32 * ((xr[j].to(F64).abs() @ w.to(F64).abs().T) * ws.to(F64).T + b.to(F64).abs())
        term, term_tol = low_rank(xr[j], la, lb, at, torch.bfloat16)
        want, off = base + term, off + term_tol + 4 * E32 * (base.abs() + term.abs())
        check(y[j], want, off + u * (want.abs() + off))
    with pytest.raises(ValueError):
        lin(x[:6])
    lin.request_loras = cuda_pkg.adapters.RequestLoras(la, lb, [1, -1, 2, 1] * 2)
    assert torch.equal(lin(x.reshape(-1, K)).reshape(y.shape), y)      # two dimensions: as many runs of rows as requests
    lin.request_loras = cuda_pkg.adapters.RequestLoras(la, lb, [1, -1, 2, 1], {"samples": 8})
    assert torch.equal(lin(x.reshape(-1, K)).reshape(y.shape), y)      # or as the model's batch has samples
    assert torch.equal(lin(x.reshape(1, -1, K)).reshape(y.shape), y)


def test_linear_module_on_two_streams_and_captured_first(cuda_pkg):
    """A bank of another type than the activations is converted by the first call: a second stream waits for that, and a first call
    within a graph capture leaves nothing that later calls would take for converted."""
    K, N = 256, 320
    w, ws, b, la, lb = layer(K, N, 16, 3, torch.bfloat16, 45)
    lin = cuda_pkg.ops.StandaloneInt8Ops.Linear(K, N, bias=True, device="meta")
    lin._load_from_state_dict({"weight": w, "weight_scale": ws, "bias": b}, "", {}, True, [], [], [])
    x = torch.randn(4, 50, K, generator=gen(46), device=DEV).bfloat16()
    wide = la.float(), lb.float()
    plans: dict = {}

    def loras():
        return cuda_pkg.adapters.RequestLoras(*wide, [1, -1], plans)

    lin.request_loras = loras()
    want = lin(x)
    torch.cuda.synchronize()
    lin.request_loras = loras()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        first = lin(x)
    second = lin(x)                        # the conversion is still to come, on the other stream
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)
    lin.request_loras = loras()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = lin(x)
    assert torch.equal(lin(x), want)       # before the graph has run
    graph.replay()
    assert torch.equal(captured, want)


@pytest.mark.parametrize("tokens", [2, 50])
def test_compiled_linear_with_request_loras(cuda_pkg, tokens):
    """A compiled layer runs the adapters outside of its graph, with the same bits, and follows the adapters that it is given."""
    w, ws, b, la, lb = layer(256, 320, 16, 3, torch.bfloat16, 47)
    lin = cuda_pkg.ops.StandaloneInt8Ops.Linear(256, 320, bias=True, device="meta")
    lin._load_from_state_dict({"weight": w, "weight_scale": ws, "bias": b}, "", {}, True, [], [], [])
    x = torch.randn(4, tokens, 256, generator=gen(48), device=DEV).bfloat16()
    compiled = torch.compile(lin, backend="eager")
    for loras in (None, cuda_pkg.adapters.RequestLoras(la, lb, [1, -1]), cuda_pkg.adapters.RequestLoras(la, lb, [2, 0, 1, 1]), None):
        lin.request_loras = loras
        assert torch.equal(compiled(x), lin(x))


def test_dit_batch_of_samples_fused(cuda_pkg):
    """A batch of samples through the fused block code against the same model in element-wise steps: the differences are 16-bit
    roundings that the fused pass leaves out, and the int8 steps they move."""
    import importlib
    dit = importlib.import_module(cuda_pkg.__name__ + ".dit")
    cfg = dit.DiTConfig(hidden=512, heads=4, mlp_ratio=3, double_blocks=2, single_blocks=2, img_tokens=96, txt_tokens=40, txt_dim=256)
    model = dit.SyntheticDiT(cfg, seed=3, fused_batch=True)
    g = gen(44)
    img = torch.randn(3, 96, cfg.in_channels, generator=g, device=DEV).bfloat16()
    txt = torch.randn(3, 40, cfg.txt_dim, generator=g, device=DEV).bfloat16()
    t = torch.tensor([0.9, 0.4, 0.1], device=DEV)
    got = model(img, txt, t)
    model.fused_batch = False
    want = model(img, txt, t)
    assert got.shape == want.shape
    rel = float((got.float() - want.float()).norm() / want.float().norm())
    assert rel < 0.05, rel
    # every sample has its own modulation: the first sample's result does not depend on the others' time steps
    model.fused_batch = True
    again = model(img, txt, torch.tensor([0.9, 0.7, 0.8], device=DEV))
    assert torch.equal(again[0], got[0]) and not torch.equal(again[1], got[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = model(img, txt, t)
    graph.replay()
    assert torch.equal(captured, got)

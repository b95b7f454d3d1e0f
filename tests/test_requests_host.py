"""The host side of a batch of requests: the row plan, the bank of adapters, and what the entry points refuse (no GPU)."""
import ctypes

import numpy as np
import pytest
import torch


def tables(rows):
    """The tables of a plan made on the CPU, read back through the struct that the library gets."""
    n = rows.native

    def at(ptr, *shape):
        count = int(np.prod(shape))
        if not count:
            return np.zeros(shape, np.int32)
        assert ptr % 16 == 0
        return np.ctypeslib.as_array(ctypes.cast(ptr, ctypes.POINTER(ctypes.c_int32)), (count,)).copy().reshape(shape)

    tiles = at(n.tiles, -(-n.rows // 256), 4)
    return (at(n.row_adapter, n.rows), at(n.row_request, n.rows), tiles, at(n.slots, int(tiles[:, 1].sum()), 12), at(n.chunks, n.n_chunks, 4))


@pytest.mark.parametrize("lengths,adapters", [
    ([1], None), ([1], [3]), ([0, 5, 0], [0, 1, 2]), ([1] * 9, [0, 0, 0, 0, 0, 1, -1, -1, 1]), ([257, 3, 0, 255], [2, -1, 5, 2]),
    ([4, 4, 1, 300], [1, 1, 1, 0]), ([0, 0], [0, 0]), ([1000], [-1]), ([1] * 400, [i % 9 for i in range(400)]), ([255], [0]), ([256], [0]),
    ([1] * 300 + [500] + [1] * 100, [i % 20 for i in range(401)]), ([600] + [1] * 50, [0] * 51),
    ([1] * 14 + [400], [*range(15)]), ([1] * 15 + [400], [*range(16)]), ([1] * 16 + [400], [*range(17)]),
    ([20] * 8 + [8] * 8 + [300], [*range(16)] + [-1]), ([20] * 9 + [300], [*range(9)] + [-1]), ([130, 2, 700], [1048575, -1, 7]),
])
def test_row_plan_describes_every_row_once(pkg, lengths, adapters):
    rows = pkg.adapters.RequestRows(lengths, adapters, device="cpu")
    M = sum(lengths)
    want_adapter = [a for n, a in zip(lengths, adapters or [-1] * len(lengths)) for _ in range(n)]
    want_request = [i for i, n in enumerate(lengths) for _ in range(n)]
    row_adapter, row_request, tiles, slots, chunks = tables(rows)
    assert rows.total == rows.native.rows == M and rows.requests == len(lengths)
    assert row_adapter.tolist() == want_adapter and row_request.tolist() == want_request
    assert rows.native.max_adapter == max(want_adapter, default=-1)
    assert rows.native.n_dense == (tiles[:, 2] < 0).sum() and (M > 16 or rows.native.n_dense == 0)
    # dense tiles: one slot for each adapter, its rows and no others; few rows beside other adapters are chunked as well
    next_slot = 0
    addend_at, few = {}, {}
    for i, (begin, count, addend, _) in enumerate(tiles.tolist()):
        tile_rows = range(256 * i, min(M, 256 * i + 256))
        if addend >= 0:
            assert count == 0
            addend_at.update({m: addend + m - 256 * i for m in tile_rows})
            continue
        assert addend == -1 and 0 <= count <= 16 and begin == next_slot
        next_slot += count
        mine = slots[begin:begin + count]
        assert (mine[:, 1] == 0).sum() <= 8
        assert sorted(mine[:, 0].tolist()) == sorted({want_adapter[m] for m in tile_rows} - {-1})
        for slot in mine:
            bits = np.unpackbits(slot[4:].view(np.uint8), bitorder="little")
            mine_rows = [m for m in tile_rows if want_adapter[m] == slot[0]]
            assert (256 * i + np.flatnonzero(bits)).tolist() == mine_rows and slot[1] == (count > 1 and len(mine_rows) <= 8)
            if slot[1]:
                few.update(dict.fromkeys(mine_rows, -1))
    # chunked tiles: every row in one chunk, with a place of its own in the addend
    covered = {}
    for first, count, adapter, addend in chunks.tolist():
        assert 1 <= count <= 4
        for j in range(count):
            assert first + j not in covered and want_adapter[first + j] == adapter
            covered[first + j] = addend + j if addend >= 0 else -1
    assert covered == {**addend_at, **few}
    assert rows.native.addend_rows == len(addend_at) and sorted(addend_at.values()) == list(range(len(addend_at)))


@pytest.mark.parametrize("lengths,adapters", [([], None), ([-1], None), ([2, 3], [0]), ([2], [-2]), ([2], [1 << 20]), ([1 << 30, 1 << 30], None)])
def test_row_plan_refuses(pkg, lengths, adapters):
    with pytest.raises(ValueError):
        pkg.adapters.RequestRows(lengths, adapters, device="cpu")


def test_stack_adapters_pads_ranks_and_scales(pkg):
    g = torch.Generator().manual_seed(1)
    factors = [(torch.randn(r, 32, generator=g), torch.randn(24, r, generator=g), s) for r, s in ((3, 0.5), (8, 1.0), (11, 2.0))]
    a, b = pkg.adapters.stack_adapters(factors + [(factors[0][0], factors[0][1])], torch.float32, "cpu")
    assert a.shape == (4, 16, 32) and b.shape == (4, 24, 16) and a.is_contiguous() and b.is_contiguous()
    for i, (down, up, s) in enumerate(factors):
        torch.testing.assert_close(b[i] @ a[i], up @ down * s, rtol=0, atol=11 * 2 ** -22 * float((up.abs() @ down.abs()).max()) * s)
        assert not a[i, down.shape[0]:].any() and not b[i, :, down.shape[0]:].any()
    assert torch.equal(a[3, :3], factors[0][0])
    with pytest.raises(ValueError):
        pkg.adapters.stack_adapters([], torch.float32, "cpu")
    with pytest.raises(ValueError):
        pkg.adapters.stack_adapters([factors[0][:2], (torch.zeros(4, 31), torch.zeros(24, 4))], torch.float32, "cpu")
    with pytest.raises(ValueError):
        pkg.adapters.stack_adapters([(torch.zeros(4, 32), torch.zeros(24, 5))], torch.float32, "cpu")


def test_cpu_tensors_are_rejected(pkg):
    rows = pkg.adapters.RequestRows([4], [0], device="cpu")
    F, E = pkg.functional, pkg._native.NativeLibraryError
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.int8)
    a, b = torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 32, 8, dtype=torch.bfloat16)
    for call in (lambda: F.linear_lora_requests(x, w, 1.0, None, a, b, rows, torch.bfloat16),
                 lambda: F.linear_small_batch_lora_requests(x, w, 1.0, None, a, b, rows),
                 lambda: F.lora_down_requests(x, a, rows),
                 lambda: F.gated_residual_norm(x, x), lambda: F.quantize_rowwise_gated_residual_norm(x, x)):
        with pytest.raises(E, match="CUDA"):
            call()


P = ctypes.c_void_p(4096)        # an aligned address that no refused call ever reads
ODD = ctypes.c_void_p(4098)


def native_rows(pkg, rows=8, max_adapter=1, **kw):
    s = pkg._native.RequestRowsStruct(rows=rows, row_adapter=4096, row_request=4096, tiles=4096, slots=4096, chunks=4096, n_dense=0, n_chunks=2,
                                      addend_rows=rows, max_adapter=max_adapter)
    for k, v in kw.items():
        setattr(s, k, v)
    return ctypes.byref(s)


def test_abi_refuses_bad_adapter_calls(pkg):
    nat = pkg._native
    lib = nat.load()

    def down(x=P, ldx=64, bank=P, adapters=2, r=16, rows=None, t=P, ldt=16, dt=nat.I8F_BF16, M=8, K=64):
        return lib.i8f_lora_down_requests(x, ldx, bank, adapters, r, rows or native_rows(pkg), t, ldt, dt, M, K, None)

    for want, kw in ((-1, dict(M=9)), (-1, dict(rows=native_rows(pkg, chunks=None))), (-1, dict(rows=native_rows(pkg, n_chunks=0))),
                     (-3, dict(dt=nat.I8F_F32)), (-1, dict(adapters=1)), (-1, dict(bank=None)), (-3, dict(r=12)), (-3, dict(r=0)),
                     (-3, dict(r=1032, ldt=1032)), (-2, dict(bank=ODD)), (-1, dict(x=None)), (-1, dict(t=None)), (-1, dict(ldx=56)),
                     (-1, dict(ldt=8)), (-2, dict(x=ODD)), (-2, dict(t=ODD)), (-2, dict(K=60)), (-2, dict(ldx=68)), (-2, dict(ldt=20))):
        assert down(**kw) == want, kw
        assert nat.last_error()
    assert down(M=0, rows=native_rows(pkg, rows=0)) == 0

    def gemm(t=P, ldt=16, bank=P, adapters=2, r=16, rows=None, dt=nat.I8F_BF16, M=8, N=64, K=64, order=1, ws=P, ws_bytes=1 << 20, a=P):
        return lib.i8f_linear_w8a8_lora_requests(a, K, P, P, K, P, 0, None, 0, t, ldt, bank, adapters, r, rows or native_rows(pkg), P, dt, N,
                                                 M, N, K, order, ws, ws_bytes, None)

    for want, kw in ((-1, dict(M=9)), (-3, dict(dt=nat.I8F_F32)), (-1, dict(adapters=1)), (-3, dict(r=20)), (-1, dict(t=None)), (-1, dict(ldt=8)),
                     (-2, dict(t=ODD)), (-2, dict(bank=ODD)), (-6, dict(ws=None)), (-6, dict(ws_bytes=64)), (-2, dict(ws=ODD))):
        assert gemm(**kw) == want, kw
        assert nat.last_error()
    for rows in (dict(n_chunks=0), dict(n_chunks=-1, n_dense=2), dict(n_dense=1, slots=None), dict(addend_rows=0), dict(addend_rows=-1, n_dense=1),
                 dict(row_adapter=None)):
        assert gemm(rows=native_rows(pkg, **rows)) == -1, rows
    assert gemm(M=0, rows=native_rows(pkg, rows=0)) == 0
    assert gemm(N=0) == 0

    def whole(x=P, dt=nat.I8F_BF16, ldx=64, had=0, rot=0, w=P, ws=P, wsb=1 << 20, bank_a=P, bank_b=P, adapters=2, r=16, rows=None, M=8, N=64,
              K=64, order=1, ldo=64):
        return lib.i8f_linear_lora_requests(x, dt, ldx, had, rot, w, K, P, 0, None, 0, bank_a, bank_b, adapters, r,
                                            rows or native_rows(pkg, rows=M), P, ldo, M, N, K, order, ws, wsb, None)

    for want, kw in ((-1, dict(rows=native_rows(pkg, rows=7))), (-3, dict(dt=nat.I8F_F32)), (-2, dict(K=72, ldx=72)), (-1, dict(adapters=1)),
                     (-1, dict(bank_a=None)), (-1, dict(bank_b=None)), (-3, dict(r=12)), (-1, dict(x=None)), (-1, dict(w=None)),
                     (-1, dict(ldx=56)), (-2, dict(x=ODD)), (-2, dict(w=ODD)), (-1, dict(ldo=63)), (-1, dict(order=2)),
                     (-6, dict(ws=None)), (-6, dict(wsb=64)), (-2, dict(ws=ODD)), (-3, dict(had=1, rot=1, K=128, ldx=136))):
        assert whole(**kw) == want, kw
        assert nat.last_error()
    assert whole(M=0, rows=native_rows(pkg, rows=0)) == 0 and whole(N=0) == 0

    def small(x=P, dt=nat.I8F_BF16, ldx=64, bank_a=P, bank_b=P, adapters=2, r=16, rows=None, M=8, N=64, K=64, ws=P, ws_bytes=1 << 20):
        return lib.i8f_linear_w8a16_small_lora_requests(x, dt, ldx, P, K, P, 0, None, 0, bank_a, bank_b, adapters, r,
                                                        rows or native_rows(pkg, rows=M), P, N, M, N, K, ws, ws_bytes, None)

    for want, kw in ((-1, dict(rows=native_rows(pkg, rows=7))), (-3, dict(M=17)), (-3, dict(dt=nat.I8F_F32)), (-1, dict(adapters=1)), (-3, dict(r=4)),
                     (-1, dict(bank_a=None)), (-2, dict(bank_b=ODD)), (-2, dict(K=72, ldx=72)), (-6, dict(ws=None)), (-6, dict(ws_bytes=64)),
                     (-1, dict(x=None)), (-1, dict(rows=native_rows(pkg, n_dense=1)))):
        assert small(**kw) == want, kw
        assert nat.last_error()


def test_abi_refuses_bad_norm_calls(pkg):
    nat = pkg._native
    lib = nat.load()

    def call(x=P, xdt=nat.I8F_BF16, ldx=64, y=P, ydt=nat.I8F_BF16, ldy=64, M=8, K=64, gate=P, ldg=64, post=1, norm=1, scale=None, lds=0,
             shift=None, ldt=0, eps=1e-6, xo=P, ldxo=64, h=P, ldh=64, q=None, ldq=0, rs=None, req=1):
        return lib.i8f_gated_residual_norm(x, xdt, ldx, y, ydt, ldy, M, K, None, req, gate, ldg, 0, 1.0, post, None, norm, None, scale, lds, shift,
                                           ldt, eps, xo, ldxo, h, ldh, q, ldq, rs, None)

    for want, kw in ((-3, dict(ydt=nat.I8F_F32)), (-3, dict(xdt=nat.I8F_F16)), (-1, dict(M=-1)), (-1, dict(K=-8)),
                     (-3, dict(K=16392, ldx=16392, ldy=16392, ldg=16392, ldxo=16392, ldh=16392)), (-1, dict(post=3)), (-1, dict(norm=0)),
                     (-1, dict(eps=-1.0)), (-1, dict(req=0)), (-1, dict(x=None)), (-1, dict(y=None)), (-1, dict(xo=None)), (-1, dict(h=None)),
                     (-1, dict(h=None, q=P, ldq=64)), (-1, dict(ldx=63)), (-1, dict(ldy=63)), (-1, dict(ldxo=63)), (-1, dict(ldh=63)),
                     (-1, dict(q=P, ldq=63, rs=P)), (-1, dict(ldg=63)), (-1, dict(scale=P, lds=63)), (-1, dict(shift=P, ldt=63))):
        assert call(**kw) == want, kw
        assert nat.last_error()
    assert call(M=0) == 0 and call(K=0) == 0


class _Adapter:
    def __init__(self, up, down, alpha=None, mid=None):
        self.weights = (up, down, alpha, mid, None, None)


class _Layer(torch.nn.Module):
    def __init__(self, n, k):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.zeros(n, k), requires_grad=False)
        self.lora_A = self.lora_B = self.lora_alpha = self.request_loras = None


def test_hook_gives_each_request_its_composition(pkg):
    g = torch.Generator().manual_seed(2)
    model = torch.nn.ModuleDict({"a": _Layer(24, 32), "b": _Layer(16, 32), "c": _Layer(8, 8)})

    def entry(strength, **layers):
        return {"patches": {f"diffusion_model.{k}.weight": _Adapter(torch.randn(n, r, generator=g), torch.randn(r, 32, generator=g), 4.0)
                            for k, (n, r) in layers.items()}, "strength": strength}

    one, two, shared = entry(0.5, a=(24, 3), b=(16, 5)), entry(1.0, a=(24, 9)), entry(2.0, b=(16, 2))
    hook = pkg.ops.DynamicLoRAHook()
    opts = {"request_loras": [[one], [], [one, two], [one]]}
    hook.pre_forward(model, (), {"transformer_options": opts})

    def delta(layer, i):
        e = model[layer].request_loras.entries[i]
        bank = model[layer].request_loras
        return torch.zeros(bank.lora_b.shape[1], 32) if e < 0 else bank.lora_b[e] @ bank.lora_a[e]

    def want(layer, *entries):
        total = torch.zeros(model[layer].weight.shape)
        for d in entries:
            ad = d["patches"].get(f"diffusion_model.{layer}.weight")
            if ad is not None:
                up, down, alpha = ad.weights[:3]
                total = total + (alpha / down.shape[0] * d["strength"]) * (up @ down)
        return total

    def check(per_request):
        for layer in "ab":
            for i, entries in enumerate(per_request):
                # at most 14 products of magnitudes that add up to less than 200, each rounded to fp32 a few times
                torch.testing.assert_close(delta(layer, i), want(layer, *entries), rtol=0, atol=14 * 4 * 2 ** -24 * 200)

    check([[one], [], [one, two], [one]])
    assert model["a"].request_loras.entries == (0, -1, 1, 0) and model["a"].request_loras.lora_a.shape == (2, 16, 32)
    assert model["c"].request_loras is None and model["a"].lora_A is None
    before = model["a"].request_loras
    hook.pre_forward(model, (), {"transformer_options": opts})
    assert model["a"].request_loras is before                    # the same requests: nothing is rebuilt
    hook.pre_forward(model, (), {"transformer_options": {**opts, "dynamic_loras": [shared]}})
    check([[shared, one], [shared], [shared, one, two], [shared, one]])
    # plans are shared by the layers, repeated samples repeat the requests
    plan = model["a"].request_loras.rows(8, 5, torch.device("cpu"))
    assert plan is model["b"].request_loras.rows(8, 5, torch.device("cpu"))
    assert plan.lengths == (5,) * 8 and plan.adapters == model["a"].request_loras.entries * 2
    with pytest.raises(ValueError):
        model["a"].request_loras.rows(6, 5, torch.device("cpu"))
    # the batch of the call tells the layers how many samples they see
    hook.pre_forward(model, (torch.zeros(8, 3),), {"transformer_options": {**opts, "dynamic_loras": [shared]}})
    assert model["a"].request_loras.samples == model["b"].request_loras.samples == 8
    # the patches are held for as long as the hook goes by their ids
    assert [id(p) for p in hook._held] == [id(d["patches"]) for d in (shared, one, one, two, one)]
    # back to one composition for all, then to none
    hook.pre_forward(model, (), {"transformer_options": {"dynamic_loras": [one]}})
    assert model["a"].request_loras is None and model["a"].lora_A.shape == (3, 32)
    hook.pre_forward(model, (), {"transformer_options": {}})
    assert model["a"].request_loras is None and model["a"].lora_A is None


def test_request_loras_refuse(pkg):
    A = pkg.adapters.RequestLoras
    a, b = torch.zeros(2, 8, 32), torch.zeros(2, 24, 8)
    assert A(a, b, [0, -1, 1]).entries == (0, -1, 1)
    for args in ((a[0], b, [0]), (a, b[:1], [0]), (a, b[:, :, :4], [0]), (a, b, []), (a, b, [2]), (a, b, [-2])):
        with pytest.raises(ValueError):
            A(*args)


def linear_plan(pkg, monkeypatch, loras, shape):
    """Lengths and adapters of the rows that the Linear's forward hands to the kernels for an input of this shape."""
    seen = []

    def take(x, weight, w_scale, bias, lora_a, lora_b, rows, *args, **kw):
        seen.append(rows)
        return x

    monkeypatch.setattr(pkg.ops.F, "linear_lora_requests", take)
    monkeypatch.setattr(pkg.ops.F, "linear_small_batch_lora_requests", take)
    x = torch.zeros(shape)
    pkg.ops._request_forward(loras, x.reshape(-1, shape[-1]), shape[0] if len(shape) > 2 else None, None, None, None, x.dtype, False, True)
    return [a for n, a in zip(seen[0].lengths, seen[0].adapters) for _ in range(n)]


class _Model(torch.nn.Module):
    def __init__(self, forward):
        super().__init__()
        self.layer = _Layer(24, 32)
        self._run = forward

    def forward(self, latent, t=None, transformer_options={}):
        return self._run(latent)


def two_requests(pkg, *input_args, **input_kwargs):
    """The first layer's RequestLoras and the hook's model after a call of two requests with one LoRA each."""
    model = _Model(lambda latent: latent)
    one, two = ({"patches": {"layer.weight": _Adapter(torch.ones(24, 4), torch.ones(4, 32))}, "strength": 1.0} for _ in range(2))
    pkg.ops.DynamicLoRAHook.register(model)
    model(*input_args, transformer_options={"request_loras": [[one], [two]]}, **input_kwargs)
    return model.layer.request_loras


def test_hook_sees_a_batch_that_is_passed_by_keyword(pkg, monkeypatch):
    """Two requests under guidance, four samples: row j of a two-dimensional input is request j modulo 2, however the batch is
    passed; where the hook cannot see the batch, such an input is refused, never cut by guess."""
    for loras in (two_requests(pkg, torch.zeros(4, 3)), two_requests(pkg, latent=torch.zeros(4, 3))):
        assert loras.samples == 4
        assert linear_plan(pkg, monkeypatch, loras, (4, 32)) == [0, 1, 0, 1]
        assert linear_plan(pkg, monkeypatch, loras, (4, 2, 32)) == [0, 0, 1, 1, 0, 0, 1, 1]
    unseen = two_requests(pkg, [torch.zeros(4, 3)])
    assert unseen.samples is None
    with pytest.raises(ValueError, match="batch"):
        linear_plan(pkg, monkeypatch, unseen, (4, 32))
    assert linear_plan(pkg, monkeypatch, unseen, (4, 1, 32)) == [0, 1, 0, 1]       # the leading dimension says it
    # a layer whose model has no hook: two dimensions are one run of rows per request, as it is told
    alone = pkg.adapters.RequestLoras(unseen.lora_a, unseen.lora_b, [0, 1])
    assert linear_plan(pkg, monkeypatch, alone, (4, 32)) == [0, 0, 1, 1]
    for shape in ((0, 32), (0, 5, 32), (2, 0, 32)):
        assert linear_plan(pkg, monkeypatch, alone, shape) == linear_plan(pkg, monkeypatch, unseen, shape) == []


def test_batch_that_is_no_multiple_of_the_requests_is_refused(pkg, monkeypatch):
    loras = two_requests(pkg, torch.zeros(3, 3))
    for shape in ((6, 32), (2, 32), (3, 2, 32), (6, 2, 32)):
        with pytest.raises(ValueError):
            linear_plan(pkg, monkeypatch, loras, shape)
    loras = two_requests(pkg, torch.zeros(4, 3))
    for shape in ((6, 32), (2, 32)):               # rows that are not four samples, in two dimensions
        with pytest.raises(ValueError):
            linear_plan(pkg, monkeypatch, loras, shape)
    # where all requests have one composition there is nothing to tell apart
    for entries, known in (([0], 3), ([1, 1], 3), ([-1, -1, -1], 4), ([0], None)):
        same = pkg.adapters.RequestLoras(loras.lora_a, loras.lora_b, entries, {"samples": known})
        for shape in ((6, 32), (7, 32), (1, 5, 32), (5, 3, 32)):
            assert linear_plan(pkg, monkeypatch, same, shape) == [entries[0]] * int(np.prod(shape[:-1]))


def test_leading_dimension_that_is_not_the_batch_is_refused(pkg, monkeypatch):
    """[2 B, T, K] may be the batch twice (0, 1, 0, 1) or two pieces of every sample (0, 0, 1, 1)."""
    for batch in (2, 4):
        loras = two_requests(pkg, torch.zeros(batch, 3))
        assert loras.samples == batch
        for leading in (2 * batch, 3 * batch, batch + 1, 6 - batch):
            with pytest.raises(ValueError, match="leading"):
                linear_plan(pkg, monkeypatch, loras, (leading, 12, 32))
        want = [j % 2 for j in range(batch) for _ in range(12)]
        for shape in ((batch, 12, 32), (batch, 3, 4, 32), (1, 12 * batch, 32), (12 * batch, 32)):
            assert linear_plan(pkg, monkeypatch, loras, shape) == want
        with pytest.raises(ValueError):
            linear_plan(pkg, monkeypatch, loras, (1, 12 * batch + 1, 32))


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16), (torch.float16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16)])
def test_bank_holds_every_requests_factors_in_full(pkg, types):
    """LoRAs of several types in one batch, in either order: each entry of the bank has its own LoRA's values to the bit."""
    g = torch.Generator().manual_seed(5)
    factors = {t: (torch.randn(24, 4, generator=g) * 1e5 if t is not torch.float16 else torch.randn(24, 4, generator=g),
                   torch.randn(4, 32, generator=g) * 1e-9 if t is not torch.float16 else torch.randn(4, 32, generator=g)) for t in set(types)}
    for order in (types, types[::-1]):
        model = _Model(lambda latent: latent)
        pkg.ops.DynamicLoRAHook.register(model)
        entries = [{"patches": {"layer.weight": _Adapter(*(f.to(t) for f in factors[t]), alpha=4.0)}, "strength": 1.0} for t in order]
        model(torch.zeros(2, 3), transformer_options={"request_loras": [[e] for e in entries]})
        bank = model.layer.request_loras
        for i, t in enumerate(order):
            up, down = (f.to(t) for f in factors[t])
            assert torch.equal(bank.lora_a[bank.entries[i], :4].float(), down.float())
            assert torch.equal(bank.lora_b[bank.entries[i], :, :4].float(), up.float())
    assert types[0] is not types[1] or bank.lora_a.dtype is types[0]


def test_refused_composition_does_not_pass_for_the_one_before(pkg):
    """A composition that does not fit a layer raises; the next call sets every layer up again, whatever it asks for."""
    model = torch.nn.ModuleDict({"a": _Layer(24, 32), "b": _Layer(16, 32)})
    hook = pkg.ops.DynamicLoRAHook()

    def entry(n_b):
        return {"patches": {"a.weight": _Adapter(torch.ones(24, 4), torch.ones(4, 32)), "b.weight": _Adapter(torch.ones(n_b, 4), torch.ones(5, 32))},
                "strength": 1.0}

    good = {"patches": {k + ".weight": _Adapter(torch.ones(n, 4), torch.ones(4, 32)) for k, n in (("a", 24), ("b", 16))}, "strength": 1.0}
    for opts in ({"request_loras": [[good], []]}, {"dynamic_loras": [good]}, {}):
        hook.pre_forward(model, (), {"transformer_options": opts})
        want = [(m.request_loras is not None, m.lora_A is not None) for m in model.values()]
        with pytest.raises(ValueError):
            hook.pre_forward(model, (), {"transformer_options": {"request_loras": [[entry(16)]]}})
        hook.pre_forward(model, (), {"transformer_options": opts})
        assert [(m.request_loras is not None, m.lora_A is not None) for m in model.values()] == want


def test_hook_refuses_ranks_that_the_layers_would(pkg):
    """A request's LoRAs add up to more ranks than the projections take: refused by name when the banks are made."""
    model = torch.nn.ModuleDict({"a": _Layer(24, 32)})
    hook = pkg.ops.DynamicLoRAHook()

    def entry(r):
        return {"patches": {"a.weight": _Adapter(torch.zeros(24, r), torch.zeros(r, 32))}, "strength": 1.0}

    hook.pre_forward(model, (), {"transformer_options": {"request_loras": [[entry(1000), entry(24)], [entry(8)]]}})
    assert model["a"].request_loras.lora_a.shape == (2, 1024, 32)
    with pytest.raises(ValueError, match="^a: .* 1025 ranks"):
        hook.pre_forward(model, (), {"transformer_options": {"request_loras": [[entry(8)], [entry(1000), entry(25)]]}})
    assert pkg.adapters.MAX_RANK == 1024      # what the library refuses beyond (test_abi_refuses_bad_adapter_calls)


def test_plan_is_held_for_the_streams_that_read_it(pkg, monkeypatch):
    """Every entry point that hands the tables to the library reports its stream; the first report of a stream is recorded with the
    allocator, but not within a graph capture, whose plan the caller holds."""
    rows = pkg.adapters.RequestRows([3, 2], [0, -1], device="cpu")
    recorded, capturing = [], [False]

    class Tables:
        def record_stream(self, stream):
            recorded.append(stream)

    rows._tables = Tables()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: ("stream", handle[0]))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    handle = [5]
    monkeypatch.setattr(pkg.functional.nat, "stream_handle", lambda device: handle[0])
    stream_for = pkg.functional._stream_for
    assert rows.streams == set()
    for h in (5, 5, 7, 5):
        handle[0] = h
        assert stream_for(rows, rows.device) == h
    assert recorded == [("stream", 5), ("stream", 7)]
    capturing[0], handle[0] = True, 9
    assert stream_for(rows, rows.device) == 9 and len(recorded) == 2
    capturing[0] = False
    assert stream_for(rows, rows.device) == 9 and recorded[2:] == [("stream", 9)]


class _FakeTensor:
    """A factor bank on a pretended device, which notes the streams that it is recorded for."""

    def __init__(self, shape, device, dtype, made):
        self.shape, self.device, self.dtype, self.made, self.streams = shape, device, dtype, made, []
        made.append(self)

    def dim(self):
        return len(self.shape)

    def to(self, device, dtype):
        return _FakeTensor(self.shape, device, dtype, self.made)

    def contiguous(self):
        return self

    def record_stream(self, stream):
        self.streams.append(stream.name)


def test_converted_bank_on_other_streams_and_in_captures(pkg, monkeypatch):
    """A second stream waits for the conversion that the first one made, and holds its memory; a conversion within a capture is not
    kept for calls outside of it."""
    log, state = [], dict(stream="a", capturing=False)

    class Stream:
        name = property(lambda self: state["stream"])

        def record_event(self):
            log.append(("record", self.name))
            return "event of " + self.name

        def wait_event(self, event):
            log.append(("wait", self.name, event))

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(pkg.adapters.nat, "stream_handle", lambda device: state["stream"])
    made, device = [], torch.device("cuda", 0)
    loras = pkg.adapters.RequestLoras(_FakeTensor((2, 8, 32), device, torch.float32, made), _FakeTensor((2, 24, 8), device, torch.float32, made), [0, 1])
    state["capturing"] = True
    captured = loras.bank(device, torch.bfloat16)
    state["capturing"] = False
    first = loras.bank(device, torch.bfloat16)
    assert first[0] is not captured[0] and log == [("record", "a")]
    assert loras.bank(device, torch.bfloat16) is first and len(log) == 1
    state["stream"] = "b"
    assert loras.bank(device, torch.bfloat16) is first and loras.bank(device, torch.bfloat16) is first
    assert log[1:] == [("wait", "b", "event of a")] and [t.streams for t in first] == [["a", "b"]] * 2
    state["capturing"], state["stream"] = True, "c"
    assert loras.bank(device, torch.bfloat16) is first and len(log) == 2
    state["capturing"] = False
    other = loras.bank(device, torch.float16)              # another type: converted anew, on the stream that asks
    assert other is not first and log[2:] == [("record", "c")] and [t.streams for t in other] == [["c"]] * 2
    assert len(made) == 2 + 2 * 3


def test_workspace_of_the_whole_forward(pkg):
    """The fp32 addend is asked for only where the product reads it: chunked rows on 256-wide tiles (gemm_plan)."""
    lib = pkg._native.load()

    def padded(n):
        return -(-n // 256) * 256

    for lengths, N, K, r in (([1] * 64, 4096, 4096, 16), ([77], 4096, 4096, 64), ([1] * 400, 512, 1024, 8), ([1] * 5000, 12288, 4096, 16),
                             ([1] * 300 + [5000], 12288, 4096, 16), ([5000], 12288, 4096, 16)):
        rows = pkg.adapters.RequestRows(lengths, [i % 40 for i in range(len(lengths))], device="cpu")
        M = rows.total
        wide = pkg.functional.gemm_plan(M, N, K)["tile"][1] == 256
        base = padded(M * K) + padded(4 * M) + padded(2 * M * r)
        for rotated in (0, 1):
            want = base + rotated * padded(2 * M * K) + (rows.native.addend_rows * N * 4 if wide else 0)
            assert lib.i8f_linear_lora_requests_workspace_bytes(rows.native_ptr, N, K, r, rotated, rotated) == want


def test_plan_within_a_capture_is_refused(pkg, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="outside of a graph capture"):
        pkg.adapters.RequestRows([4], [0], device="cuda")
    assert pkg.adapters.RequestRows([4], [0], device="cpu").total == 4


def test_output_rows_that_overlap_the_input_are_seen(pkg):
    """The rows of x_out may be those of x, or lie beside them in one buffer; anything else that shares memory would be read and
    written at once."""
    overlap = pkg.functional._rows_overlap
    buf = torch.zeros(4000)
    wide = buf[:3000].view(30, 100)
    x = wide[2:12, 8:40]
    for other in (x, x[:], wide[2:12, 40:72], wide[2:12, 68:100], wide[12:22, 8:40], torch.zeros(10, 32), buf[3000:3320].view(10, 32)):
        assert not overlap(x, other) and not overlap(other, x)
    assert not overlap(x[:, :24], wide[1:11, 76:]) and not overlap(x[:1], buf[208:240].view(1, 32))
    for other in (wide[3:13, 8:40], wide[1:11, 8:40], wide[2:12, 9:41], wide[2:12, 0:32], wide[3:13, 39:71], wide[1:11, 68:100].as_strided((10, 32), (100, 1), 180),
                  buf[208:528].view(10, 32), buf[:2000].view(10, 200)[:, :32]):
        assert overlap(x, other) and overlap(other, x)
    half = buf.view(torch.bfloat16)
    assert overlap(x, half[416:416 + 320].view(10, 32)) and overlap(half.view(40, 200)[2:12, 16:48], x)
    assert not overlap(half.view(40, 200)[2:12, 80:112], x) and not overlap(x[:0], x[:0])

"""Timing cases of the operators for a batch of requests: the shared int8 projection with one low-rank adapter per
request, and the gated residual update between two norms with one modulation per request.

`run` computes a case in elementary torch operations, or, with the module flag `own` set, through the package's entry
points.  `exact` is the definition in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one sampled token (or one pooled vector) of one request: latency
        dict(name="adapters_1_token", op="small", rows=1, requests=1, spread="even", K=4096, N=4096, rank=16, bank=4,
             dtype="bf16", bias=True, per_channel=True, none_every=0),
        # sixteen requests, a token each, every one with an adapter of its own
        dict(name="adapters_16_tokens", op="small", rows=16, requests=16, spread="even", K=4096, N=12288, rank=32, bank=16,
             dtype="f16", bias=False, per_channel=False, none_every=0),
        # a decode step of 64 requests, every eighth without an adapter
        dict(name="adapters_64_tokens", op="linear", rows=64, requests=64, spread="even", K=4096, N=4096, rank=16, bank=48,
             dtype="bf16", bias=True, per_channel=True, none_every=8),
        # prompts of odd lengths and single tokens in one batch, one request empty
        dict(name="adapters_mixed", op="linear", rows=1531, requests=30, spread="mixed", K=4096, N=4096, rank=64, bank=12,
             dtype="bf16", bias=True, per_channel=True, none_every=7),
        # nine text streams of 512 tokens into the MLP
        dict(name="adapters_prompts", op="linear", rows=4608, requests=9, spread="even", K=4096, N=12288, rank=64, bank=9,
             dtype="f16", bias=False, per_channel=False, none_every=0),
        # four samples of 4096 image and 512 text tokens each: the largest
        dict(name="adapters_images", op="linear", rows=18432, requests=4, spread="even", K=4096, N=12288, rank=32, bank=4,
             dtype="bf16", bias=True, per_channel=True, none_every=0),
        # one token through the residual update
        dict(name="norm_1_row", op="norm", rows=1, requests=1, spread="even", H=4096, post="rms", pre="rms", tanh=True,
             weights=True, shift=False, residual_scale=1.0, dtype="bf16", residual="bf16", int8=False),
        # a text encoder's ragged batch, a row length that no vector width divides
        dict(name="norm_ragged_text", op="norm", rows=777, requests=11, spread="ragged", H=2305, post="layer", pre="layer",
             tanh=False, weights=True, shift=True, residual_scale=0.5, dtype="f16", residual="f16", int8=False),
        # norm after the branch, tanh gate, norm before the next: 4 samples
        dict(name="norm_images", op="norm", rows=4608, requests=4, spread="ragged", H=4096, post="rms", pre="rms", tanh=True,
             weights=True, shift=False, residual_scale=1.0, dtype="bf16", residual="bf16", int8=False),
        # plain gate, LayerNorm with scale and shift, int8 rows for the quantised linear that follows
        dict(name="norm_images_int8", op="norm", rows=4608, requests=4, spread="even", H=4096, post="none", pre="layer",
             tanh=False, weights=False, shift=True, residual_scale=1.0, dtype="bf16", residual="bf16", int8=True),
        # eight samples, the residual stream kept in fp32
        dict(name="norm_batch_f32", op="norm", rows=18432, requests=8, spread="even", H=4096, post="rms", pre="layer",
             tanh=False, weights=True, shift=True, residual_scale=1.0, dtype="bf16", residual="f32", int8=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["small", "linear", "linear", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm":
        int8 = rng.random() < 0.3
        H = _log(rng, 64, 12288)
        if int8 or rng.random() < 0.6:
            H = (H + 7) // 8 * 8
        rows = max(1, min(_log(rng, 1, 18432), 18432 * 4096 // H))
        return dict(op=op, rows=rows, requests=min(rows, _log(rng, 1, 64)), spread=rng.choice(["even", "ragged", "mixed"]), H=H,
                    post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["rms", "layer"]), tanh=rng.random() < 0.5,
                    weights=rng.random() < 0.6, shift=rng.random() < 0.6, residual_scale=rng.choice([1.0, 0.5, 0.7071]),
                    dtype=dtype, residual=rng.choice([dtype, dtype, "f32"]), int8=int8)
    K = 16 * _log(rng, 16, 768)
    N = _log(rng, 64, 12288)
    if rng.random() < 0.7:
        N = (N + 7) // 8 * 8
    rank = 8 * rng.choice([1, 2, 2, 4, 4, 8, 8, 16])
    rows = rng.randint(1, 16) if op == "small" else _log(rng, 17, 9216)
    requests = min(rows, _log(rng, 1, 64))
    return dict(op=op, rows=rows, requests=requests, spread=rng.choice(["even", "ragged", "mixed"]), K=K, N=N, rank=rank,
                bank=rng.randint(1, min(requests, 24)), dtype=dtype, bias=rng.random() < 0.5, per_channel=rng.random() < 0.6,
                none_every=rng.choice([0, 0, 5]))


def _lengths(case):
    """Rows of each request, from the case alone: even, ragged, or mixed (single tokens, ragged prompts and an empty one)."""
    rows, n = case["rows"], case["requests"]
    rng = random.Random("%d/%d/%s" % (rows, n, case["spread"]))
    if case["spread"] == "even" or n == 1:
        return [rows // n + (1 if i < rows % n else 0) for i in range(n)]
    singles = (2 * n) // 3 if case["spread"] == "mixed" else 0
    rest = n - singles
    cuts = sorted(rng.randint(0, rows - singles) for _ in range(rest - 1))
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [rows - singles])] + [1] * singles
    if case["spread"] == "mixed" and rest > 1:
        lengths[1], lengths[0] = lengths[0] + lengths[1], 0
    rng.shuffle(lengths)
    return lengths


def _adapters(case):
    """Bank entry of each request; -1: none."""
    every = case["none_every"]
    return [-1 if every and i % every == every - 1 else (5 * i + 1) % case["bank"] for i in range(case["requests"])]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    lengths = _lengths(case)
    counts = torch.tensor(lengths, device=DEV)
    s = dict(case=case, request=torch.repeat_interleave(torch.arange(len(lengths), device=DEV), counts))

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if case["op"] == "norm":
        H, n, M = case["H"], case["requests"], case["rows"]
        s["x"] = (randn(M, H) * 4.0).to(DTYPES[case["residual"]])
        s["y"] = randn(M, H).to(dt)
        # what a modulation linear gives: one row per request, cut into gate | scale | shift
        mod = (randn(n, 3 * H) * 0.3).to(dt)
        s["gate"], s["scale"], s["shift"] = (mod[:, i * H:(i + 1) * H] for i in range(3))
        if not case["shift"]:
            s["shift"] = None
        s["post_weight"] = (1.0 + 0.1 * randn(H)).to(dt) if case["weights"] and case["post"] != "none" else None
        s["weight"] = (1.0 + 0.1 * randn(H)).to(dt) if case["weights"] else None
        adapters = None
    else:
        K, N, r, bank, M = case["K"], case["N"], case["rank"], case["bank"], case["rows"]
        x = randn(M, K)
        x[:, torch.randperm(K, device=DEV, generator=g)[: max(1, K // 100)]] *= 20.0     # outlier channels
        s["x"] = x.to(dt)
        s["w"] = torch.randint(-127, 128, (N, K), device=DEV, generator=g, dtype=torch.int8)
        s["w_scale"] = (0.02 / 73 * (0.5 + torch.rand(N, 1, device=DEV, generator=g))) if case["per_channel"] else torch.full(
            (1,), 0.02 / 73, device=DEV)
        s["bias"] = (randn(N) * 0.01).to(dt) if case["bias"] else None
        s["lora_a"] = (randn(bank, r, K) / math.sqrt(K)).to(dt)
        s["lora_b"] = (randn(bank, N, r) * (0.3 / math.sqrt(r))).to(dt)
        adapters = _adapters(case)
        s["adapter"] = torch.repeat_interleave(torch.tensor(adapters, device=DEV), counts)
    if own:   # the batch's row plan, which a program makes once per batch and hands to every layer of the step
        s["rows"] = _package().adapters.RequestRows(lengths, adapters, device=torch.device("cuda", torch.cuda.current_device()))
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        return _plain_norm(state, case) if case["op"] == "norm" else _plain_linear(state, case)


def _run_own(s, case):
    F = _package().functional
    if case["op"] == "small":
        return F.linear_small_batch_lora_requests(s["x"], s["w"], s["w_scale"], s["bias"], s["lora_a"], s["lora_b"], s["rows"])
    if case["op"] == "linear":
        return F.linear_lora_requests(s["x"], s["w"], s["w_scale"], s["bias"], s["lora_a"], s["lora_b"], s["rows"], s["x"].dtype)
    more = dict(rows=s["rows"], gate_tanh=case["tanh"], residual_scale=case["residual_scale"],
                post_norm=None if case["post"] == "none" else case["post"], post_weight=s["post_weight"], norm=case["pre"],
                weight=s["weight"], scale=s["scale"], shift=s["shift"], eps=1e-6)
    if case["int8"]:
        x, q, q_scale = F.quantize_rowwise_gated_residual_norm(s["x"], s["y"], s["gate"], **more)
        h = torch.empty(q.shape, dtype=s["y"].dtype, device=q.device)
        return x, torch.mul(q, q_scale, out=h)       # the values that the int8 rows stand for
    return F.gated_residual_norm(s["x"], s["y"], s["gate"], **more)


def _lora_term(x, lora_a, lora_b, adapter):
    """(x A_a^T) B_a^T with the adapter a of each row: all adapters' columns, those of other adapters dropped."""
    bank, r, K = lora_a.shape
    t = x @ lora_a.reshape(bank * r, K).T
    mine = torch.arange(bank, device=x.device).repeat_interleave(r)[None, :] == adapter[:, None]
    return torch.where(mine, t, 0.0) @ lora_b.transpose(1, 2).reshape(bank * r, -1)


def _plain_linear(s, case):
    x = s["x"].float()
    if case["op"] == "small":
        y = x @ (s["w"].float() * s["w_scale"]).T
    else:
        xs = (x.abs().amax(1, keepdim=True) / 127.0).clamp_min(1e-30)
        q = torch.clamp(torch.round(x * (1.0 / xs)), -128, 127)
        y = (q @ s["w"].float().T) * xs * s["w_scale"].reshape(1, -1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = y + _lora_term(x, s["lora_a"].float(), s["lora_b"].float(), s["adapter"])
    return y.to(s["x"].dtype)


def _plain_normed(v, kind, weight, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    return v if weight is None else v * weight.float()


def _plain_norm(s, case):
    at = s["request"]
    gate = s["gate"].float()
    if case["tanh"]:
        gate = torch.tanh(gate)
    x = case["residual_scale"] * s["x"].float() + gate[at] * _plain_normed(s["y"].float(), case["post"], s["post_weight"], 1e-6)
    h = _plain_normed(x, case["pre"], s["weight"], 1e-6) * (1.0 + s["scale"].float()[at])
    if s["shift"] is not None:
        h = h + s["shift"].float()[at]
    if case["int8"]:
        hs = (h.abs().amax(1, keepdim=True) / 127.0).clamp_min(1e-30)
        h = torch.clamp(torch.round(h * (1.0 / hs)), -128, 127) * hs
    return x.to(s["x"].dtype), h.to(s["y"].dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    M = case["rows"]
    if case["op"] == "norm":
        H = case["H"]
        residual = 4 if case["residual"] == "f32" else 2
        vectors = (2 + (1 if case["shift"] else 0)) * case["requests"] + (2 if case["weights"] else 0)
        return {"bytes": M * H * (2 * residual + 2 + (1 if case["int8"] else 2)) + 2 * H * vectors, "flops": 16 * M * H}
    K, N, r = case["K"], case["N"], case["rank"]
    used, with_adapter = set(), 0
    for length, a in zip(_lengths(case), _adapters(case)):
        if length and a >= 0:
            used.add(a)
            with_adapter += length
    return {"bytes": 2 * M * K + N * K + 2 * M * N + 2 * len(used) * r * (K + N) + (4 * N if case["per_channel"] else 4) +
            (2 * N if case["bias"] else 0),
            "flops": 2 * M * N * K + 2 * with_adapter * r * (K + N)}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "norm":
        def unit(v, kind, weight):
            if kind == "none":
                return v
            if kind == "layer":
                var, mean = torch.var_mean(v, dim=1, correction=0, keepdim=True)
                v = (v - mean) * torch.rsqrt(var + 1e-6)
            else:
                v = v * torch.rsqrt(v.square().sum(1, keepdim=True) / v.shape[1] + 1e-6)
            return v if weight is None else v * weight.to(f64)

        x, h = [], []
        first = 0
        for i, length in enumerate(_lengths(case)):       # request by request
            rows = slice(first, first + length)
            first += length
            g = s["gate"][i].to(f64)
            g = torch.tanh(g) if case["tanh"] else g
            xi = s["x"][rows].to(f64) * case["residual_scale"] + unit(s["y"][rows].to(f64), case["post"], s["post_weight"]) * g
            hi = unit(xi, case["pre"], s["weight"])
            hi = hi + hi * s["scale"][i].to(f64)
            if s["shift"] is not None:
                hi = hi + s["shift"][i].to(f64)
            x.append(xi)
            h.append(hi)
        x, h = torch.cat(x), torch.cat(h)
        if case["int8"]:
            step = h.abs().amax(dim=1, keepdim=True).div(127).clamp(min=1e-30)
            h = h.div(step).round().clamp(-128, 127).mul(step)
        return x, h
    x, w, ws = s["x"].to(f64), s["w"].to(f64), s["w_scale"].to(f64).flatten()
    if case["op"] == "linear":
        step = x.abs().amax(dim=1, keepdim=True).div(127).clamp(min=1e-30)
        xq = x.div(step).round().clamp(-128, 127).mul(step)
    else:
        xq = x
    y = torch.mm(xq, w.t()).mul_(ws)
    if s["bias"] is not None:
        y += s["bias"].to(f64)
    first = 0
    for length, a in zip(_lengths(case), _adapters(case)):
        if length and a >= 0:
            rows = slice(first, first + length)
            y[rows] += torch.mm(torch.mm(x[rows], s["lora_a"][a].to(f64).t()), s["lora_b"][a].to(f64).t())
        first += length
    return y

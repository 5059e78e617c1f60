"""Eight-bit floating point beside the quantized matmuls, as an inference engine calls it in a layer.

Operators that belong together: what produces a product's activations in 8 bits (e4m3) with a scale for each 128 of a
row -- the RMS norm with the residual's addition, SiLU(gate) * up, plain rows -- and the products themselves, of such
activations with weights in 8 bits that have a scale for each block of 128 x 128: one matrix, or a stack of them whose
rows are grouped by expert. Sizes are those of this repository's configurations (a layer of hidden 4096 with an FFN of
14336, one of hidden 2048 with 128 experts of 768) or generic; ``draw`` spreads them.
"""
import math

import torch

own = False
DEV = "cuda:0"
BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -120
F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # a decode step of a small batch, in the engine's own f32: latency is all there is
        {"name": "norm decode 32", "kind": "norm", "rows": 32, "k": 4096, "x": "f32"},
        # the norm before a prompt's projections
        {"name": "norm prefill 4096", "kind": "norm", "rows": 4096, "k": 4096, "x": "bf16"},
        # decode of a batch of 32 through 8 experts of 768 each
        {"name": "silu decode 256", "kind": "silu", "rows": 256, "k": 768, "x": "f32"},
        # a prompt's FFN: gate and up lie side by side, as one product wrote them
        {"name": "silu prefill 4096", "kind": "silu", "rows": 4096, "k": 14336, "x": "bf16"},
        # one token's attention result, before the output projection
        {"name": "quantize decode 1", "kind": "quantize", "rows": 1, "k": 4096, "x": "bf16"},
        # odd sizes: the last group of a row is short, no row starts at a multiple of 16 bytes
        {"name": "quantize ragged", "kind": "quantize", "rows": 777, "k": 1235, "x": "f16"},
        # decode of one token: the gate projection
        {"name": "gemm decode 1", "kind": "gemm", "rows": 1, "k": 4096, "n": 14336, "y": "f32"},
        # prefill of an ordinary prompt: the down projection
        {"name": "gemm prefill 512", "kind": "gemm", "rows": 512, "k": 14336, "n": 4096, "y": "bf16"},
        # prefill of a long prompt: the gate projection (the largest case)
        {"name": "gemm prefill 4096", "kind": "gemm", "rows": 4096, "k": 4096, "n": 14336, "y": "bf16"},
        # odd sizes throughout: short last groups and blocks, rows at any byte
        {"name": "gemm ragged", "kind": "gemm", "rows": 333, "k": 1235, "n": 1531, "y": "f32"},
        # decode of a batch: the down projection of its experts, back into the pairs' order
        {"name": "experts decode 32", "kind": "experts", "side": "down", "tokens": 32, "experts": 128, "top_k": 8,
         "k": 768, "n": 2048, "y": "f32"},
        # prefill of a long prompt: the gate projection, about 256 rows an expert
        {"name": "experts prefill 4096", "kind": "experts", "side": "gate", "tokens": 4096, "experts": 128, "top_k": 8,
         "k": 2048, "n": 768, "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: mostly a multiple of 128, at times of 16, at times odd."""
    v, how = _log(rng, lo, hi), rng.random()
    return max(128, v // 128 * 128) if how < 0.6 else max(16, v // 16 * 16) if how < 0.85 else v | 1


def draw(rng):
    kind = rng.choice(["norm", "silu", "quantize", "gemm", "gemm", "gemm", "experts", "experts"])
    x = rng.choice(["f32", "f16", "bf16"])
    if kind in ("norm", "silu", "quantize"):
        k = _size(rng, 64, 14336)
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(8192, 58_000_000 // k))), "k": k, "x": x}
    if kind == "gemm":
        k, n = _size(rng, 64, 14336), _size(rng, 64, 14336)
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(4096, 240_000_000_000 // (k * n)))), "k": k, "n": n, "y": x}
    experts = _log(rng, 2, 160)
    top_k = rng.randint(1, min(8, experts))
    k = _size(rng, 64, 8192)
    n = _size(rng, 64, max(65, min(8192, 400_000_000 // (experts * k))))
    return {"kind": kind, "side": rng.choice(["gate", "down"]), "experts": experts, "top_k": top_k, "k": k, "n": n, "y": x,
            "tokens": _log(rng, 1, max(1, min(4096, 120_000_000_000 // (k * n * top_k))))}


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _acts(gen, rows, k):
    """Normal activations of rows of different sizes, one channel in 256 eight times as large."""
    big = torch.ones(k, device=DEV)
    big[torch.randperm(k, device=DEV, generator=gen)[: max(1, k // 256)]] = 8.0
    return _normal(gen, rows, k) * big * torch.exp(0.5 * _normal(gen, rows, 1))


def _groups(k):
    return -(-k // BLOCK)


def _to_f8(v):
    """[rows, k] values (of any float type) as e4m3 with a scale for each 128 of a row."""
    rows, k = v.shape
    padded = torch.nn.functional.pad(v, (0, _groups(k) * BLOCK - k)).view(rows, _groups(k), BLOCK)
    scales = padded.abs().amax(2).clamp(min=TOP * LEAST) / TOP
    return (padded / scales.unsqueeze(2)).to(F8).view(rows, -1)[:, :k].contiguous(), scales


def _weights(gen, count, n, k):
    """[count, n, k] weights of standard deviation near 0.02 as e4m3, a scale for each block of 128 x 128, as a
    checkpoint holds them."""
    codes = torch.empty(count, n, k, dtype=F8, device=DEV)
    scales = torch.empty(count, _groups(n), _groups(k), device=DEV)
    for e in range(count):
        w = _normal(gen, n, k).mul_(0.02)
        p = torch.nn.functional.pad(w, (0, _groups(k) * BLOCK - k, 0, _groups(n) * BLOCK - n))
        p = p.view(_groups(n), BLOCK, _groups(k), BLOCK)
        scales[e] = p.abs().amax((1, 3)) / TOP
        codes[e] = (p / scales[e].view(_groups(n), 1, _groups(k), 1)).to(F8).view(_groups(n) * BLOCK, -1)[:n, :k]
    return codes, scales


def _grouped(ids, groups):
    """(offsets, order) of ids: order lists the rows of group 0, then of group 1, ..."""
    keys, order = torch.sort(ids, stable=True)
    offsets = torch.searchsorted(keys, torch.arange(groups + 1, dtype=keys.dtype, device=DEV))
    return offsets.to(torch.int32), order.to(torch.int32)


def prepare(case, seed):
    gen = _gen(seed)
    s = {"case": case}
    kind, k = case["kind"], case["k"]
    if kind in ("norm", "silu", "quantize"):
        rows, dtype = case["rows"], TYPES[case["x"]]
        if kind == "norm":
            s["x"], s["residual"] = _acts(gen, rows, k).to(dtype), (3.0 * _acts(gen, rows, k)).to(dtype)
            s["weight"] = 1.0 + 0.2 * _normal(gen, k)
            s["sum"] = torch.empty_like(s["x"])
        elif kind == "silu":
            both = torch.cat([_acts(gen, rows, k), _acts(gen, rows, k)], 1).to(dtype)
            s["gate"], s["up"] = both[:, :k], both[:, k:]
        else:
            s["x"] = _acts(gen, rows, k).to(dtype)
        s["codes"] = torch.empty(rows, k, dtype=F8, device=DEV)
        s["scales"] = torch.empty(rows, _groups(k), device=DEV)
        if own:
            import reflex_amd as rq

            s["out"] = rq.F8Rows(s["codes"], s["scales"])
        return s
    n = case["n"]
    if kind == "gemm":
        count, xrows, yrows = 1, case["rows"], case["rows"]
    else:
        count, yrows = case["experts"], case["tokens"] * case["top_k"]
        xrows = case["tokens"] if case["side"] == "gate" else yrows
        logits = _normal(gen, 1, count) * 0.7 + _normal(gen, case["tokens"], count)
        ids = logits.topk(case["top_k"], dim=1).indices.to(torch.int32).reshape(-1)
        s["offsets"], s["order"] = _grouped(ids, count)
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # the plain form's padding
    s["x"], s["xs"] = _to_f8(_acts(gen, xrows, k))
    s["w"], s["ws"] = _weights(gen, count, n, k)
    s["y"] = torch.empty(yrows, n, dtype=TYPES[case["y"]], device=DEV)
    if kind == "gemm":
        s["w"], s["ws"] = s["w"][0], s["ws"][0]
    if own:
        import reflex_amd as rq

        s["rows"], s["weight"] = rq.F8Rows(s["x"], s["xs"]), rq.F8Weight(s["w"], s["ws"])
    return s


# ---------------------------------------------------------------- one pass

def _wide(codes, scales):
    """e4m3 rows with a scale for each 128 of a row, as f32."""
    k = codes.shape[-1]
    return codes.float() * scales.repeat_interleave(BLOCK, -1)[..., :k]


def _wide_weight(codes, scales):
    """e4m3 weights with a scale for each block of 128 x 128, as f32."""
    return _wide(codes, scales.repeat_interleave(BLOCK, -2)[..., : codes.shape[-2], :])


def _plain_rows(s):
    case = s["case"]
    if case["kind"] == "norm":
        v = s["x"].float() + s["residual"].float()
        s["sum"].copy_(v)
        v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * s["weight"]
    elif case["kind"] == "silu":
        gate = s["gate"].float()
        v = gate / (1.0 + torch.exp(-gate)) * s["up"].float()
    else:
        v = s["x"].float()
    codes, scales = _to_f8(v)
    s["codes"].copy_(codes)
    s["scales"].copy_(scales)
    return (s["codes"], s["scales"], s["sum"]) if case["kind"] == "norm" else (s["codes"], s["scales"])


def _plain_experts(s):
    case, order = s["case"], s["order"].long()
    rows = order.numel()
    x = _wide(s["x"], s["xs"])
    if case["side"] == "gate":
        x = x[order // case["top_k"]]
    at = torch.arange(rows, device=DEV)
    group = torch.searchsorted(s["offsets"], at.to(torch.int32), right=True) - 1
    number = at - s["offsets"][group].long()
    if rows <= case["experts"]:  # few rows: each takes its own matrix
        y = torch.bmm(_wide_weight(s["w"][group], s["ws"][group]), x.unsqueeze(2)).squeeze(2)
    else:  # each group padded to the largest
        padded = torch.zeros(case["experts"], s["most"], case["k"], device=DEV)
        padded[group, number] = x
        y = torch.bmm(padded, _wide_weight(s["w"], s["ws"]).transpose(1, 2).contiguous())[group, number]
    y = y.to(s["y"].dtype)
    if case["side"] == "down":
        s["y"][order] = y
    else:
        s["y"].copy_(y)
    return s["y"]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        import reflex_amd as rq

        if kind == "norm":
            rq.add_rmsnorm_f8(s["x"], s["residual"], s["weight"], EPS, sum_out=s["sum"], out=s["out"])
            return s["codes"], s["scales"], s["sum"]
        if kind == "silu":
            rq.silu_and_mul_f8(s["gate"], s["up"], out=s["out"])
            return s["codes"], s["scales"]
        if kind == "quantize":
            rq.quantize_f8(s["x"], out=s["out"])
            return s["codes"], s["scales"]
        if kind == "gemm":
            return rq.gemm_f8(s["rows"], s["weight"], out=s["y"])
        rows = s["order"].numel()
        if case["side"] == "gate":
            return rq.grouped_gemm_f8(s["rows"], s["weight"], s["offsets"], rows, x_index=s["order"],
                                      x_div=case["top_k"], out=s["y"])
        return rq.grouped_gemm_f8(s["rows"], s["weight"], s["offsets"], rows, y_index=s["order"], out=s["y"])
    if kind in ("norm", "silu", "quantize"):
        return _plain_rows(s)
    if kind == "gemm":
        s["y"].copy_(_wide(s["x"], s["xs"]) @ _wide_weight(s["w"], s["ws"]).t())
        return s["y"]
    return _plain_experts(s)


# ---------------------------------------------------------------- what a pass cannot do without

def _bytes(name):
    return 4 if name == "f32" else 2


def work(case):
    k = case["k"]
    if case["kind"] in ("norm", "silu", "quantize"):
        rows, e = case["rows"], _bytes(case["x"])
        out = rows * (k + 4 * _groups(k))
        if case["kind"] == "norm":
            return {"bytes": 3 * rows * k * e + 4 * k + out, "flops": 8 * rows * k}
        return {"bytes": (2 if case["kind"] == "silu" else 1) * rows * k * e + out, "flops": 3 * rows * k}
    n = case["n"]
    if case["kind"] == "gemm":
        used, xrows, yrows = 1, case["rows"], case["rows"]
    else:
        e, t, top_k = case["experts"], case["tokens"], case["top_k"]
        used = e * (1.0 - (1.0 - top_k / e) ** t)  # experts that get a row, on average
        yrows = t * top_k
        xrows = t if case["side"] == "gate" else yrows
    return {"bytes": used * (n * k + 4 * _groups(n) * _groups(k)) + xrows * (k + 4 * _groups(k)) + yrows * n * _bytes(case["y"]),
            "flops": 2 * yrows * n * k}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_rows(s):
    """What the 8 bits stand for before they are rounded, in units of the scales; the scales; the residual's sum."""
    case = s["case"]
    kind, k = case["kind"], case["k"]
    if kind == "norm":
        total = s["x"].double() + s["residual"].double()
        v = s["weight"].double() * total / (total.pow(2).sum(1, keepdim=True) / k + EPS).sqrt()
    elif kind == "silu":
        v = s["gate"].double() * torch.sigmoid(s["gate"].double()) * s["up"].double()
    else:
        v = s["x"].double()
    scales = torch.empty(case["rows"], _groups(k), dtype=torch.float64, device=DEV)
    codes = torch.empty_like(v)
    for g in range(_groups(k)):
        part = v[:, g * BLOCK:(g + 1) * BLOCK]
        scales[:, g] = part.abs().max(1).values.clamp(min=TOP * LEAST) / TOP
        codes[:, g * BLOCK:(g + 1) * BLOCK] = part / scales[:, g:g + 1]
    return (codes, scales, total) if kind == "norm" else (codes, scales)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "silu", "quantize"):
        return _exact_rows(s)
    k, n = case["k"], case["n"]
    x = s["x"].double()
    for g in range(_groups(k)):
        x[:, g * BLOCK:(g + 1) * BLOCK] *= s["xs"][:, g:g + 1].double()

    def matrix(codes, scales):
        w = codes.double()
        for g in range(_groups(n)):
            for h in range(_groups(k)):
                w[g * BLOCK:(g + 1) * BLOCK, h * BLOCK:(h + 1) * BLOCK] *= scales[g, h].double()
        return w

    if case["kind"] == "gemm":
        return x @ matrix(s["w"], s["ws"]).t()
    offsets, order = s["offsets"].tolist(), s["order"].long()
    y = torch.zeros(order.numel(), n, dtype=torch.float64, device=DEV)
    for e in range(case["experts"]):
        at = torch.arange(offsets[e], offsets[e + 1], device=DEV)
        if at.numel():
            src, dst = (order[at] // case["top_k"], at) if case["side"] == "gate" else (at, order[at])
            y[dst] = x[src] @ matrix(s["w"][e], s["ws"][e]).t()
    return y

"""Products with half-typed weight stacks, as an inference engine calls them beside its quantized matmuls.

Three operators that belong together: rows are grouped by an id (the expert a router chose, the adapter a request
asked for), a mixture-of-experts layer whose stacked expert tensors are F16 or BF16 multiplies each group with its own
matrix, and low-rank adapters of many requests are added to a projection that all rows share. Sizes are those of this
repository's configurations (a layer of hidden 2048 with 128 experts of 768, one of hidden 4096 with an FFN of 14336)
or generic; ``draw`` spreads them.
"""
import math

import torch

own = False
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # grouping the routed pairs of a small decode batch: latency is all there is
        {"name": "group decode 32x8", "kind": "group", "tokens": 32, "groups": 128, "top_k": 8},
        # grouping the routed pairs of a long prompt
        {"name": "group prefill 16384x8", "kind": "group", "tokens": 16384, "groups": 128, "top_k": 8},
        # grouping the rows of a batch by the adapter that each request asked for, some for none
        {"name": "group adapters 2050", "kind": "group", "tokens": 2050, "groups": 37, "top_k": 1},
        # decode of one token: the gate projection of its eight experts
        {"name": "experts decode 1", "kind": "experts", "side": "gate", "tokens": 1, "experts": 128, "top_k": 8,
         "k": 2048, "n": 768, "x": "bf16", "w": "bf16"},
        # decode of a batch in the engine's own f32 activations: the down projection, back into the pairs' order
        {"name": "experts decode 32 f32", "kind": "experts", "side": "down", "tokens": 32, "experts": 128, "top_k": 8,
         "k": 768, "n": 2048, "x": "f32", "w": "f16"},
        # prefill of an ordinary prompt: gate projection, about 32 rows an expert
        {"name": "experts prefill 512", "kind": "experts", "side": "gate", "tokens": 512, "experts": 128, "top_k": 8,
         "k": 2048, "n": 768, "x": "bf16", "w": "bf16"},
        # prefill of a long prompt through few, large experts (the largest case)
        {"name": "experts prefill 4096", "kind": "experts", "side": "gate", "tokens": 4096, "experts": 8, "top_k": 2,
         "k": 4096, "n": 14336, "x": "f16", "w": "f16"},
        # odd sizes: no row starts at a multiple of 16 bytes, f32 activations
        {"name": "experts ragged f32", "kind": "experts", "side": "down", "tokens": 777, "experts": 11, "top_k": 3,
         "k": 1235, "n": 1531, "x": "f32", "w": "bf16"},
        # a decode step of 16 requests with an adapter each, in the engine's f32 activations
        {"name": "lora decode 16", "kind": "lora", "rows": 16, "adapters": 16, "rank": 16, "k": 4096, "n": 4096,
         "x": "f32", "w": "f16"},
        # a decode step of a large batch over many adapters of mixed ranks
        {"name": "lora decode 256", "kind": "lora", "rows": 256, "adapters": 64, "rank": 64, "k": 4096, "n": 14336,
         "x": "bf16", "w": "bf16"},
        # prefill of several long prompts, an adapter each, f32 activations
        {"name": "lora prefill 4096", "kind": "lora", "rows": 4096, "adapters": 6, "rank": 64, "k": 4096, "n": 4096,
         "x": "f32", "w": "f16"},
        # odd sizes throughout
        {"name": "lora ragged", "kind": "lora", "rows": 1037, "adapters": 9, "rank": 13, "k": 1235, "n": 1531,
         "x": "f16", "w": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: mostly a multiple of 64, at times of 8, at times odd."""
    v, how = _log(rng, lo, hi), rng.random()
    return max(64, v // 64 * 64) if how < 0.6 else max(8, v // 8 * 8) if how < 0.85 else v | 1


def draw(rng):
    kind = rng.choice(["group", "experts", "experts", "experts", "lora", "lora"])
    w = rng.choice(["f16", "bf16"])
    x = rng.choice([w, w, "f32"])
    if kind == "group":
        groups = _log(rng, 2, 512)
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "groups": groups, "top_k": rng.randint(1, min(8, groups))}
    if kind == "experts":
        experts = _log(rng, 2, 160)
        top_k = rng.randint(1, min(8, experts))
        k = _size(rng, 64, 8192)
        n = _size(rng, 64, min(14336, 400_000_000 // (experts * k)))
        tokens = _log(rng, 1, max(1, min(4096, 400_000_000_000 // (2 * k * n * top_k))))
        return {"kind": kind, "side": rng.choice(["gate", "down"]), "tokens": tokens, "experts": experts,
                "top_k": top_k, "k": k, "n": n, "x": x, "w": w}
    return {"kind": kind, "rows": _log(rng, 1, 4096), "adapters": _log(rng, 1, 64), "rank": _log(rng, 1, 128),
            "k": _size(rng, 256, 8192), "n": _size(rng, 256, 14336), "x": x, "w": w}


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _acts(gen, rows, k, dtype):
    """Normal activations, one channel in 256 eight times as large."""
    big = torch.ones(k, device=DEV)
    big[torch.randperm(k, device=DEV, generator=gen)[: max(1, k // 256)]] = 8.0
    return (_normal(gen, rows, k) * big).to(dtype)


def _stack(gen, count, n, k, dtype):
    """[count][n][k] weights of standard deviation near 0.02, made one matrix at a time."""
    w = torch.empty(count, n, k, dtype=dtype, device=DEV)
    for e in range(count):
        w[e].copy_(_normal(gen, n, k).mul_(0.02))
    return w


def _routed(gen, tokens, experts, top_k):
    """[tokens * top_k] expert ids, a token's distinct, some experts asked for more often."""
    logits = _normal(gen, 1, experts) * 0.7 + _normal(gen, tokens, experts)
    return logits.topk(top_k, dim=1).indices.to(torch.int32).reshape(-1)


def _grouped(ids, groups):
    """(offsets, order) of ids: order lists the rows of group 0, then of group 1, ...; rows in no group come last."""
    key = torch.where((ids >= 0) & (ids < groups), ids, groups)
    keys, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(keys, torch.arange(groups + 1, dtype=keys.dtype, device=DEV))
    return offsets.to(torch.int32), order.to(torch.int32)


def prepare(case, seed):
    gen = _gen(seed)
    s = {"case": case}
    if case["kind"] == "group":
        ids = _routed(gen, case["tokens"], case["groups"], case["top_k"])
        if case["top_k"] == 1:  # rows that ask for no adapter
            ids[torch.rand(ids.numel(), device=DEV, generator=gen) < 0.1] = -1
        s["ids"] = ids
    elif case["kind"] == "experts":
        pairs = case["tokens"] * case["top_k"]
        ids = _routed(gen, case["tokens"], case["experts"], case["top_k"])
        s["offsets"], s["order"] = _grouped(ids, case["experts"])
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # the plain form's padding
        s["w"] = _stack(gen, case["experts"], case["n"], case["k"], TYPES[case["w"]])
        s["x"] = _acts(gen, case["tokens"] if case["side"] == "gate" else pairs, case["k"], TYPES[case["x"]])
        s["y"] = torch.empty(pairs, case["n"], dtype=TYPES[case["x"]], device=DEV)
        if own:
            import reflex_amd as rq

            s["weight"] = rq.Weight.from_tensor(s["w"])
    else:
        rows, count, rank = case["rows"], case["adapters"], case["rank"]
        if rows <= 512:  # a decode step: any row may ask for any adapter
            ids = torch.randint(0, count, (rows,), device=DEV, generator=gen, dtype=torch.int32)
        else:  # prompts one after another
            ends = torch.randint(0, rows, (count - 1,), device=DEV, generator=gen).sort().values
            ids = torch.searchsorted(ends, torch.arange(rows, device=DEV), right=True).to(torch.int32)
        if count > 1:  # the last one's rows have asked for none
            ids[ids == count - 1] = -1
        s["offsets"], s["order"] = _grouped(ids, count)
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        # a pool of adapters, each in the first rows (a) and columns (b) of its place, the others hold old values
        s["a"] = _stack(gen, count, rank, case["k"], TYPES[case["w"]])
        s["b"] = _stack(gen, count, case["n"], rank, TYPES[case["w"]])
        part = torch.randint(0, 3, (count,), device=DEV, generator=gen)
        s["ranks"] = torch.clamp(rank >> part, min=1).to(torch.int32)
        s["scales"] = 32.0 / s["ranks"].float()
        s["x"] = _acts(gen, rows, case["k"], TYPES[case["x"]])
        s["y"] = _normal(gen, rows, case["n"]).to(TYPES[case["x"]])  # what the shared projection gave
        s["out"] = torch.empty_like(s["y"])
        if own:
            import reflex_amd as rq

            s["weights"] = (rq.Weight.from_tensor(s["a"]), rq.Weight.from_tensor(s["b"]))
            s["groups"] = rq.RowGroups(s["offsets"], s["order"])
    return s


# ---------------------------------------------------------------- one pass

def _places(offsets, rows):
    """Of each place in the grouped order: its group and its number in the group."""
    at = torch.arange(rows, device=DEV)
    group = torch.searchsorted(offsets, at.to(offsets.dtype), right=True) - 1
    return group, at - offsets[group].long()


def _plain_experts(s):
    case, order = s["case"], s["order"].long()
    rows = order.numel()
    x = s["x"][order // case["top_k"]] if case["side"] == "gate" else s["x"]
    group, number = _places(s["offsets"], rows)
    if rows <= case["experts"]:  # few rows: each takes its own matrix
        y = torch.bmm(s["w"][group].float(), x.float().unsqueeze(2)).squeeze(2)
    else:  # each group padded to the largest
        padded = torch.zeros(case["experts"], s["most"], case["k"], device=DEV)
        padded[group, number] = x.float()
        y = torch.bmm(padded, s["w"].float().transpose(1, 2).contiguous())[group, number]
    y = y.to(s["y"].dtype)
    if case["side"] == "down":
        s["y"][order] = y
    else:
        s["y"].copy_(y)
    return s["y"]


def _plain_lora(s):
    case, order = s["case"], s["order"].long()
    count, rank = case["adapters"], case["rank"]
    group, number = _places(s["offsets"], order.numel())
    group = torch.where(group < count, group, count)  # rows without an adapter go to a place of their own
    keep = torch.arange(rank, device=DEV) < s["ranks"].unsqueeze(1)
    a = torch.where(keep.unsqueeze(2), s["a"].float(), 0.0)
    b = torch.where(keep.unsqueeze(1), s["b"].float(), 0.0)
    padded = torch.zeros(count + 1, s["most"] + 1, case["k"], device=DEV)
    number = torch.where(group < count, number, s["most"])
    padded[group, number] = s["x"][order].float()
    low = torch.bmm(padded[:count], a.transpose(1, 2).contiguous()) * s["scales"].view(-1, 1, 1)
    delta = torch.zeros(count + 1, padded.shape[1], case["n"], device=DEV)
    delta[:count] = torch.bmm(low, b.transpose(1, 2).contiguous())
    y = s["y"][order].float() + delta[group, number]
    s["out"][order] = y.to(s["out"].dtype)
    return s["out"]


def run(s):
    case = s["case"]
    if case["kind"] == "group":
        if own:
            import reflex_amd as rq

            g = rq.group_rows(s["ids"], case["groups"])
            return g.offsets, g.order
        return _grouped(s["ids"], case["groups"])
    if case["kind"] == "experts":
        if own:
            import reflex_amd as rq

            rows = s["order"].numel()
            if case["side"] == "gate":
                return rq.grouped_gemm(s["x"], s["weight"], s["offsets"], rows, x_index=s["order"],
                                       x_div=case["top_k"], out=s["y"])
            return rq.grouped_gemm(s["x"], s["weight"], s["offsets"], rows, y_index=s["order"], out=s["y"])
        return _plain_experts(s)
    if own:
        import reflex_amd as rq

        return rq.lora_add(s["x"], *s["weights"], s["groups"], s["y"], ranks=s["ranks"], scales=s["scales"],
                           out=s["out"])
    return _plain_lora(s)


# ---------------------------------------------------------------- what a pass cannot do without

def _bytes(name):
    return 4 if name == "f32" else 2


def work(case):
    if case["kind"] == "group":
        n = case["tokens"] * case["top_k"]
        return {"bytes": 8 * n + 4 * (case["groups"] + 1), "flops": 0}
    if case["kind"] == "experts":
        e, t, top_k = case["experts"], case["tokens"], case["top_k"]
        used = e * (1.0 - (1.0 - top_k / e) ** t)  # experts that get a row, on average
        xrows = t if case["side"] == "gate" else t * top_k
        return {"bytes": used * case["n"] * case["k"] * _bytes(case["w"])
                + _bytes(case["x"]) * (xrows * case["k"] + t * top_k * case["n"]),
                "flops": 2 * t * top_k * case["k"] * case["n"]}
    rows, count = case["rows"], case["adapters"]
    used = count * (1.0 - (1.0 - 1.0 / count) ** rows)
    rank = max(1.0, case["rank"] * 7 / 12)  # a third each of the whole, half and a quarter
    return {"bytes": used * rank * (case["k"] + case["n"]) * _bytes(case["w"])
            + _bytes(case["x"]) * rows * (case["k"] + 2 * case["n"]),
            "flops": 2 * rows * rank * (case["k"] + case["n"])}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "group":
        return None
    offsets, order = s["offsets"].tolist(), s["order"].long()
    if case["kind"] == "experts":
        y = torch.empty(order.numel(), case["n"], dtype=torch.float64, device=DEV)
        for e in range(case["experts"]):
            at = torch.arange(offsets[e], offsets[e + 1], device=DEV)
            if at.numel():
                src, dst = (order[at] // case["top_k"], at) if case["side"] == "gate" else (at, order[at])
                y[dst] = s["x"][src].double() @ s["w"][e].double().t()
        return y
    y = s["y"].double()
    for e, r in enumerate(s["ranks"].tolist()):
        rows = order[offsets[e]:offsets[e + 1]]
        if rows.numel():
            low = s["x"][rows].double() @ s["a"][e, :r].double().t()
            y[rows] += s["scales"][e].double() * (low @ s["b"][e, :, :r].double().t())
    return y

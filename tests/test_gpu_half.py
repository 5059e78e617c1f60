"""Grouped rows, products with F16 / BF16 stacks and low-rank adapters (rfxq_group_rows,
rfxq_grouped_gemm, rfxq_lora_add) against their definitions in 64 bits on the CPU.

Bounds, per result: a half-typed output is off by half a step, eps / 2 of its value; a sum of K products
held in f32 by at most 2^-23 of the sum of the products' sizes per addition, with K / 32 + 32 additions in
a row (the matrix instructions add 32 products, or 4 of f32 operands, to the sum at once; parts of a sum that are
added later are counted in). f32 activations beside f16 weights are split into two f16 pieces, which leave
2^-22 of a value (half a step of the second piece, 2^-11 of 2^-11) and 2^-39 of the largest of its row or of
its step of the row (half a step of f16's smallest number, 2^-25, at a largest of 2^14 or more); beside bf16
weights three pieces are exact but for what is below f32's range. A value below f32's or f16's normal range keeps an absolute step."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}


def _say(*what):
    print(*what, flush=True)


# ------------------------------------------------------------------ group_rows

def _grouped(ids, groups):
    key = np.where((ids >= 0) & (ids < groups), ids, groups)
    order = np.argsort(key, kind="stable").astype(np.int32)
    offsets = np.searchsorted(key[order], np.arange(groups + 1)).astype(np.int32)
    return offsets, order


def _ids(n, groups, how, seed=0):
    r = np.random.default_rng(seed + n + groups)
    if how == "any":  # some in no group, on either side
        return r.integers(-1, groups + 1, n).astype(np.int32)
    if how == "one":
        return np.full(n, groups - 1, np.int32)
    if how == "none":
        return np.where(r.random(n) < 0.5, -(1 << 31), (1 << 31) - 1).astype(np.int32)
    if how == "rising":
        return np.sort(r.integers(0, groups, n)).astype(np.int32)
    return r.integers(0, groups, n).astype(np.int32)


@pytest.mark.parametrize("how", ["any", "one", "none", "rising", "all"])
@pytest.mark.parametrize("n,groups", [(0, 5), (1, 1), (2, 3), (63, 2), (64, 128), (65, 1024), (300, 37), (1000, 128),
                                      (1024, 7), (1025, 1023), (4096, 128), (32768, 3), (32769, 256), (65536, 64),
                                      (65537, 1024), (131072, 257), (131073, 900),
                                      (131077, 129), (270001, 256), (300007, 1000)])
def test_group_rows(rq, n, groups, how):
    _say("group_rows", n, groups, how)
    ids = _ids(n, groups, how)
    guard = 77
    offsets = torch.full((groups + 1 + 8,), guard, dtype=torch.int32, device=DEV)
    order = torch.full((n + 8,), guard, dtype=torch.int32, device=DEV)
    g = rq.group_rows(torch.from_numpy(ids).to(DEV), groups, out=rq.RowGroups(offsets, order))
    want_offsets, want_order = _grouped(ids, groups)
    assert np.array_equal(g.offsets.cpu().numpy()[:groups + 1], want_offsets)
    assert np.array_equal(g.order.cpu().numpy()[:n], want_order)
    assert (offsets[groups + 1:] == guard).all() and (order[n:] == guard).all()


def test_group_rows_unaligned_ids_and_new_outputs(rq):
    ids = _ids(5001, 37, "any")
    t = torch.from_numpy(np.concatenate([ids[:1], ids])).to(DEV)[1:]  # starts 4 bytes into its memory
    g = rq.group_rows(t, 37)
    want_offsets, want_order = _grouped(ids, 37)
    assert np.array_equal(g.offsets.cpu().numpy(), want_offsets) and np.array_equal(g.order.cpu().numpy(), want_order)


def test_group_rows_own_workspace(rq):
    n, groups = 100_001, 200
    ids = _ids(n, groups, "any")
    t = torch.from_numpy(ids).to(DEV)
    size = rq.group_rows_workspace_size(n, groups)
    ws = torch.full((size + 64,), 7, dtype=torch.uint8, device=DEV)
    g = rq.group_rows(t, groups, workspace=ws[:size])
    want_offsets, want_order = _grouped(ids, groups)
    assert np.array_equal(g.offsets.cpu().numpy(), want_offsets) and np.array_equal(g.order.cpu().numpy(), want_order)
    assert (ws[size:] == 7).all()
    with pytest.raises(rq.InvalidInputError, match="needs"):
        rq.group_rows(t, groups, workspace=ws[:size - 1])
    with pytest.raises(rq.ReflexError, match="16-byte aligned"):
        rq.group_rows(t, groups, workspace=ws[8:])
    assert rq.group_rows_workspace_size(1000, groups) == 0


# ------------------------------------------------------------------ grouped_gemm

def _strided(values, stride, shift, pad):
    """`values` [rows, cols] on the GPU as a view of rows `stride` apart, `shift` elements into memory that
    holds `pad` elsewhere."""
    rows, cols = values.shape
    memory = torch.full((shift + max(rows, 1) * stride + 8,), pad, dtype=values.dtype, device=DEV)
    view = memory[shift:shift + rows * stride].view(rows, stride)[:, :cols]
    view.copy_(values)
    return view, memory


def _product_bound(x, w, y64, x_type, w_type, y_type, pieces=None):
    """Largest allowed |error| per result of x @ w.T (64-bit arrays)."""
    k = x.shape[1]
    size = np.abs(x) @ np.abs(w).T
    count = {F32: 2 if w_type == F16 else 3}.get(x_type, 1)
    b = (count * (k / 32) + 32) * 2.0 ** -23 * size
    if x_type == F32:
        b = b + 2.0 ** -22 * size + 2.0 ** -39 * np.abs(x).max(1, keepdims=True, initial=0) * np.abs(w).sum(1)
    return b + torch.finfo(y_type).eps / 2 * (np.abs(y64) + b) + TINY[y_type]


def _case(rows, groups, k, n, x_type, w_type, seed, x_rows=None):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(x_rows or rows, k, generator=gen)
    if k > 1:
        x[:, k // 2] *= 8
    w = (torch.randn(groups, n, k, generator=gen) * 0.05).to(w_type)
    return x.to(x_type), w


def _run_grouped(rq, x, w, offsets, rows, x_index, x_div, y_index, y_type, y_rows, xs=(0, 0), ys=(0, 0), ws=0):
    """grouped_gemm on strided and shifted copies: (y, what lies around y unchanged)."""
    k, n = x.shape[1], w.shape[1]
    xv, _ = _strided(x.to(DEV), k + xs[0], xs[1], float("nan"))
    yv, ymem = _strided(torch.full((y_rows, n), 123.0, dtype=y_type, device=DEV), n + ys[0], ys[1], 99.0)
    wmem = torch.full((w.numel() + ws + 8,), float("nan"), dtype=w.dtype, device=DEV)
    wmem[ws:ws + w.numel()] = w.reshape(-1).to(DEV)
    weight = rq.Weight.from_tensor(wmem[ws:ws + w.numel()].view(w.shape))
    dev = lambda v: None if v is None else torch.from_numpy(np.asarray(v, np.int32)).to(DEV)  # noqa: E731
    rq.grouped_gemm(xv, weight, dev(offsets), rows, x_index=dev(x_index), x_div=x_div, y_index=dev(y_index), out=yv)
    torch.cuda.synchronize()
    around = ymem.clone()
    around[ys[1]:ys[1] + y_rows * (n + ys[0])].view(y_rows, -1)[:, :n] = 99.0
    return yv.cpu(), bool((around == 99.0).all())


def _check_grouped(x, w, offsets, x_index, x_div, y_index, y):
    """Every row of y: its product's within the bound, or what it was."""
    want = np.full(y.shape, 123.0)
    bound = np.zeros(y.shape)
    x64, w64 = x.double().numpy(), w.double().numpy()
    for g in range(w.shape[0]):
        p = np.arange(offsets[g], offsets[g + 1])
        src = p if x_index is None else np.where(np.asarray(x_index)[p] < 0, -1, np.asarray(x_index)[p] // x_div)
        dst = p if y_index is None else np.asarray(y_index)[p]
        fine = (src >= 0) & (src < x.shape[0]) & (dst >= 0) & (dst < y.shape[0])
        src, dst = src[fine], dst[fine]
        want[dst] = x64[src] @ w64[g].T
        bound[dst] = _product_bound(x64[src], w64[g], want[dst], x.dtype, w.dtype, y.dtype)
    off = np.abs(y.double().numpy() - want)
    assert np.isfinite(off).all()
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert (off <= bound).all(), (worst, off[worst], bound[worst])
    rel = np.linalg.norm(off) / np.linalg.norm(want)
    # rounding errors of either sign: well under a half step of y, and for f32 under 2^-19 (a lost piece
    # of the activations would leave 2^-13)
    assert rel <= (torch.finfo(y.dtype).eps / 2 if y.dtype != F32 else 2.0 ** -19), rel


TYPES = [(F16, F16, F16), (BF16, BF16, BF16), (F32, F16, F32), (F32, BF16, F32), (F16, F16, F32), (F32, BF16, BF16)]


@pytest.mark.parametrize("x_type,w_type,y_type", TYPES)
@pytest.mark.parametrize("rows,groups,k,n", [
    (1, 1, 1, 1), (1, 8, 64, 128), (2, 3, 7, 15), (8, 128, 256, 96), (17, 4, 72, 64), (33, 2, 128, 129), (64, 5, 8, 16),
    (65, 3, 200, 300), (130, 7, 1235, 153), (300, 1, 576, 257), (513, 40, 320, 128), (700, 6, 2056, 384)])
def test_grouped_gemm(rq, rows, groups, k, n, x_type, w_type, y_type):
    _say("grouped_gemm", rows, groups, k, n, x_type, w_type, y_type)
    x, w = _case(rows, groups, k, n, x_type, w_type, rows + k)
    ids = _ids(rows, groups, "all")
    offsets, _ = _grouped(ids, groups)
    y, kept = _run_grouped(rq, x, w, offsets, rows, None, 1, None, y_type, rows)
    _check_grouped(x, w, offsets, None, 1, None, y)
    assert kept


# sizes at which each kernel is chosen, whole and ragged: few tiles, few rows over short K with many columns
# (half types, then f32), quarters of K (f32) or tiles copied ahead, tiles through registers, large tiles
@pytest.mark.parametrize("x_type,w_type,y_type", TYPES)
@pytest.mark.parametrize("rows,groups,k,n", [
    (150, 128, 128, 520), (70, 64, 1160, 200), (40, 9, 1152, 48), (64, 3, 640, 1032), (20, 1, 264, 24),
    (400, 4, 200, 136), (1000, 3, 328, 520), (1030, 4, 64, 272), (1500, 2, 136, 264), (1200, 1, 8, 256),
    (128, 64, 520, 1024), (512, 256, 72, 768), (300, 4, 200, 700), (300, 4, 201, 700), (260, 20, 1000, 640),
    (2000, 4, 72, 2104), (2000, 2, 136, 5200), (1999, 2, 72, 5121)])
def test_grouped_gemm_each_kernel(rq, rows, groups, k, n, x_type, w_type, y_type):
    _say("grouped_gemm kernels", rows, groups, k, n, x_type, w_type, y_type)
    x, w = _case(rows, groups, k, n, x_type, w_type, rows + k)
    offsets, order = _grouped(_ids(rows, groups, "all"), groups)
    y, kept = _run_grouped(rq, x, w, offsets, rows, order, 1, order, y_type, rows, (8, 8), (8, 0), 8)
    _check_grouped(x, w, offsets, order, 1, order, y)
    assert kept


@pytest.mark.parametrize("rows", [3, 300, 6000])
def test_grouped_gemm_rows_past_4_gib(rq, rows):
    """Rows of x, y and matrices of a stack whose bytes lie past 32-bit offsets."""
    _say("grouped_gemm past 4 GiB", rows)
    k, n, far, count = 1024, 2200, 2_200_000, 1000
    x, w = _case(rows, 2, k, n, F16, F16, 1)
    xd = torch.empty(far, k, dtype=F16, device=DEV)
    at = torch.arange(far - rows, far, device=DEV)
    xd[at] = x.to(DEV)
    yd = torch.empty(far, n, dtype=F16, device=DEV)
    stack = torch.empty(count, n, k, dtype=F16, device=DEV)
    stack[-2:] = w.to(DEV)
    idx = at.to(torch.int32)
    offsets = torch.zeros(count + 1, dtype=torch.int32, device=DEV)
    offsets[-2], offsets[-1] = rows // 2, rows
    rq.grouped_gemm(xd, rq.Weight.from_tensor(stack), offsets, rows, x_index=idx, y_index=idx, out=yd)
    _check_grouped(x, w, [0, rows // 2, rows], None, 1, None, yd[at].cpu())


@pytest.mark.parametrize("x_type,w_type,y_type", TYPES[:4])
@pytest.mark.parametrize("xs,ys,ws", [((8, 0), (8, 0), 0), ((3, 1), (5, 3), 1), ((0, 2), (0, 0), 0), ((0, 0), (1, 0), 2),
                                      ((16, 8), (16, 8), 8)])
def test_grouped_gemm_strides(rq, xs, ys, ws, x_type, w_type, y_type):
    """Rows with space behind them (NaN in it), and memory that starts anywhere."""
    _say("grouped_gemm strides", xs, ys, ws, x_type, w_type, y_type)
    rows, groups, k, n = 90, 4, 136, 144
    x, w = _case(rows, groups, k, n, x_type, w_type, 5)
    offsets, _ = _grouped(_ids(rows, groups, "all"), groups)
    y, kept = _run_grouped(rq, x, w, offsets, rows, None, 1, None, y_type, rows, xs, ys, ws)
    _check_grouped(x, w, offsets, None, 1, None, y)
    assert kept


@pytest.mark.parametrize("x_type,w_type,y_type", TYPES[:4])
@pytest.mark.parametrize("tokens,top_k", [(1, 1), (1, 8), (5, 3), (40, 4), (200, 6)])
def test_grouped_gemm_indexes(rq, tokens, top_k, x_type, w_type, y_type):
    """A router's pairs: gathered into groups, and scattered back; pairs that ask for no expert."""
    _say("grouped_gemm indexes", tokens, top_k, x_type, w_type, y_type)
    groups, k, n, pairs = 12, 96, 80, tokens * top_k
    ids = _ids(pairs, groups, "any")
    offsets, order = _grouped(ids, groups)
    x, w = _case(pairs, groups, k, n, x_type, w_type, tokens, x_rows=tokens)
    y, kept = _run_grouped(rq, x, w, offsets, pairs, order, top_k, None, y_type, pairs)
    _check_grouped(x, w, offsets, order, top_k, None, y)
    assert kept
    x, w = _case(pairs, groups, k, n, x_type, w_type, tokens)
    y, kept = _run_grouped(rq, x, w, offsets, pairs, None, 1, order, y_type, pairs)
    _check_grouped(x, w, offsets, None, 1, order, y)
    assert kept


@pytest.mark.parametrize("x_type,w_type,y_type", TYPES[:4])
def test_grouped_gemm_indexes_out_of_range(rq, x_type, w_type, y_type):
    rows, groups, k, n = 70, 3, 64, 72
    x, w = _case(rows, groups, k, n, x_type, w_type, 3)
    offsets = np.array([0, 30, 30, 66], np.int32)
    r = np.random.default_rng(4)
    xi, yi = np.arange(rows) * 2, r.permutation(rows)
    xi[[0, 5, 31, 65]] = [-1, 2 * rows, -(1 << 31), (1 << 31) - 1]
    yi[[1, 7, 40]] = [rows, -5, (1 << 31) - 1]
    y, kept = _run_grouped(rq, x, w, offsets, rows, xi, 2, yi, y_type, rows)
    _check_grouped(x, w, offsets, xi, 2, yi, y)
    assert kept


@pytest.mark.parametrize("offsets", [[5, 9, 9, 20], [0, 40, 10, 50], [-7, 3, 1 << 30, 50], [0, 0, 0, 0], [50, 50, 0, 0]])
def test_grouped_gemm_odd_offsets(rq, offsets):
    """Offsets that do not rise from 0 to the rows stay inside the arrays: rows of no group are left alone."""
    x, w = _case(50, 3, 64, 64, F16, F16, 9)
    y, kept = _run_grouped(rq, x, w, offsets, 50, None, 1, None, F16, 50)
    assert kept and bool(torch.isfinite(y).all())
    inside = np.zeros(50, bool)
    for b, e in zip(offsets, offsets[1:]):
        inside[max(b, 0):max(min(e, 50), 0)] = True
    assert bool((y[~inside] == 123.0).all())


@pytest.mark.parametrize("w_type", [F16, BF16])
@pytest.mark.parametrize("k", [64, 203])
def test_grouped_gemm_not_finite_rows(rq, w_type, k):
    """Infinities and NaN stay in their own rows; f32 values at the ends of their range."""
    rows, n = 40, 64
    x, w = _case(rows, 2, k, n, F32, w_type, 11)
    x[3, 5], x[8, 0], x[20] = float("inf"), float("nan"), 0.0
    x[21] *= 1e37
    x[22] *= 1e-37
    x[23], x[23, 1] = 0.0, 3e38
    offsets = np.array([0, 17, rows], np.int32)
    y, _ = _run_grouped(rq, x, w, offsets, rows, None, 1, None, F32, rows)
    x64, w64 = x.double().numpy(), w.double().numpy()
    with np.errstate(invalid="ignore"):
        want = np.concatenate([x64[:17] @ w64[0].T, x64[17:] @ w64[1].T])
    assert torch.isinf(y[3]).all() and np.array_equal(np.sign(y[3].numpy()), np.sign(want[3]))
    assert torch.isnan(y[8]).all() and (y[20] == 0).all()
    fine = [r for r in range(rows) if r not in (3, 8)]
    g = np.array([0] * 17 + [1] * (rows - 17))
    for r in fine:
        b = _product_bound(x64[r:r + 1], w64[g[r]], want[r:r + 1], F32, w_type, F32)[0]
        # pieces below f32's range are lost: k products of 2^-149 and a weight
        b = b + k * 2.0 ** -149 * (1 + np.abs(w64[g[r]]).max())
        assert (np.abs(y[r].double().numpy() - want[r]) <= b).all(), r


# quarters of K (whole and ragged), few rows over short K, tiles through registers
@pytest.mark.parametrize("w_type", [F16, BF16])
@pytest.mark.parametrize("rows,groups,k,n", [(300, 4, 136, 700), (300, 4, 203, 700), (512, 256, 72, 768), (2000, 4, 72, 1000),
                                              (2000, 4, 75, 1000)])
def test_grouped_gemm_not_finite_rows_each_kernel(rq, rows, groups, k, n, w_type):
    _say("grouped_gemm not finite", rows, groups, k, n, w_type)
    x, w = _case(rows, groups, k, n, F32, w_type, 12)
    at = np.arange(0, 240, 30)
    x[at[0], 5], x[at[1], 0], x[at[2]] = float("inf"), float("nan"), 0.0
    x[at[3]] *= 1e37
    x[at[4]] *= 1e-37
    x[at[5]], x[at[5], 1] = 0.0, 3e38
    x[at[6], k - 1], x[at[7], k - 1] = float("-inf"), float("nan")
    offsets, _ = _grouped(_ids(rows, groups, "all"), groups)
    y, _ = _run_grouped(rq, x, w, offsets, rows, None, 1, None, F32, rows)
    x64, w64 = x.double().numpy(), w.double().numpy()
    lost = at[[0, 1, 6, 7]]
    assert not torch.isfinite(y[lost]).any() and torch.isnan(y[at[[1, 7]]]).all() and (y[at[2]] == 0).all()
    got = y.double().numpy()
    for g in range(groups):
        r = np.array([p for p in range(offsets[g], offsets[g + 1]) if p not in lost], int)
        if r.size == 0:
            continue
        want = x64[r] @ w64[g].T
        b = _product_bound(x64[r], w64[g], want, F32, w_type, F32) + k * 2.0 ** -149 * (1 + np.abs(w64[g]).max())
        assert (np.abs(got[r] - want) <= b).all(), g


def test_grouped_gemm_2d_weight_and_new_output(rq):
    x, w = _case(50, 1, 100, 40, F32, F16, 2)
    weight = rq.Weight.from_tensor(w[0].contiguous().to(DEV))
    offsets = torch.tensor([0, 47], dtype=torch.int32, device=DEV)
    y = rq.grouped_gemm(x.to(DEV), weight, offsets, 50).cpu()
    assert (y[47:] == 0).all()
    y[47:] = 123.0
    _check_grouped(x, w, [0, 47], None, 1, None, y)


# ------------------------------------------------------------------ lora_add

def _run_lora(rq, x, a, b, ids, ranks, scales, y, in_place, xs=(0, 0), ys=(0, 0), shift=0):
    count = a.shape[0]
    k, n = x.shape[1], y.shape[1]
    xv, _ = _strided(x.to(DEV), k + xs[0], xs[1], float("nan"))
    yv, ymem = _strided(y.to(DEV), n + ys[0], ys[1], 99.0)
    wa, wb = (torch.full((w.numel() + shift + 8,), float("nan"), dtype=w.dtype, device=DEV) for w in (a, b))
    for m, w in ((wa, a), (wb, b)):
        m[shift:shift + w.numel()] = w.reshape(-1).to(DEV)
    wa, wb = (rq.Weight.from_tensor(m[shift:shift + w.numel()].view(w.shape)) for m, w in ((wa, a), (wb, b)))
    groups = rq.group_rows(torch.from_numpy(ids).to(DEV), count)
    out = None
    if not in_place:
        out = torch.full(y.shape, 123.0, dtype=y.dtype, device=DEV)
    dev = lambda v, t: None if v is None else torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    got = rq.lora_add(xv, wa, wb, groups, yv, ranks=dev(ranks, torch.int32), scales=dev(scales, F32), out=out)
    torch.cuda.synchronize()
    if not in_place:
        assert torch.equal(yv.cpu(), y)
    around = ymem.clone()
    around[ys[1]:ys[1] + y.shape[0] * (n + ys[0])].view(y.shape[0], -1)[:, :n] = 99.0
    assert bool((around == 99.0).all())
    return got.cpu()


def _check_lora(x, a, b, ids, ranks, scales, y, got):
    count, rank, k = a.shape
    x64, y64 = x.double().numpy(), y.double().numpy()
    want, bound = y64.copy(), np.zeros(y64.shape)
    for g in range(count):
        r = rank if ranks is None else min(max(ranks[g], 0), rank)
        s = 1.0 if scales is None else np.float64(np.float32(scales[g]))
        rows = np.flatnonzero(ids == g)
        if not len(rows) or not r:
            continue
        a64, b64 = a[g, :r].double().numpy(), b[g, :, :r].double().numpy()
        low, low_size = x64[rows] @ a64.T, np.abs(x64[rows]) @ np.abs(a64).T
        # v is off by its own sum's error (x's pieces as in the grouped products, where it is split), which B carries on
        low_bound = ((k / 4 + 64) * 2.0 ** -23 + 2.0 ** -22) * low_size
        low_bound += 2.0 ** -39 * np.abs(x64[rows]).max(1, keepdims=True) * np.abs(a64).sum(1)
        delta = s * (low @ b64.T)
        size = np.abs(s) * (np.abs(low) @ np.abs(b64).T)
        e = np.abs(s) * (low_bound @ np.abs(b64).T) + (r / 4 + 40) * 2.0 ** -23 * size
        e += 2.0 ** -15 * size if x.dtype == BF16 else 2.0 ** -21 * size if x.dtype == F16 else 2.0 ** -22 * size
        want[rows] = y64[rows] + delta
        e += 2.0 ** -23 * (np.abs(y64[rows]) + np.abs(delta))
        bound[rows] = e + torch.finfo(y.dtype).eps / 2 * (np.abs(want[rows]) + e) + TINY[y.dtype]
    off = np.abs(got.double().numpy() - want)
    assert np.isfinite(off).all()
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert (off <= bound).all(), (worst, off[worst], bound[worst])


def _lora_case(rows, count, rank, k, n, x_type, w_type, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=gen).to(x_type)
    a = (torch.randn(count, rank, k, generator=gen) * 0.05).to(w_type)
    b = (torch.randn(count, n, rank, generator=gen) * 0.05).to(w_type)
    y = torch.randn(rows, n, generator=gen).to(x_type)
    r = np.random.default_rng(seed)
    ids = r.integers(-1, count + 1, rows).astype(np.int32)
    ranks = r.integers(0, rank + 1, count).tolist()
    scales = r.uniform(-2, 4, count).tolist()
    for g in range(count):  # what lies past an adapter's rank is not used
        a[g, ranks[g]:] = float("nan")
        b[g, :, ranks[g]:] = float("inf")
    return x, a, b, ids, ranks, scales, y


LORA_TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("x_type,w_type", LORA_TYPES)
@pytest.mark.parametrize("rows,count,rank,k,n", [
    (1, 1, 1, 1, 1), (1, 3, 16, 64, 256), (2, 2, 8, 40, 17), (16, 16, 16, 512, 300), (17, 1, 13, 1235, 153),
    (40, 5, 64, 128, 257), (129, 4, 130, 264, 512), (300, 9, 32, 2048, 80), (700, 3, 24, 136, 264), (65, 70, 33, 72, 40)])
def test_lora_add(rq, rows, count, rank, k, n, x_type, w_type):
    _say("lora_add", rows, count, rank, k, n, x_type, w_type)
    c = _lora_case(rows, count, rank, k, n, x_type, w_type, rows + k)
    for in_place in (False, True):
        _check_lora(*c, _run_lora(rq, *c, in_place))


@pytest.mark.parametrize("x_type,w_type", LORA_TYPES)
@pytest.mark.parametrize("xs,ys,shift", [((8, 0), (8, 0), 0), ((3, 1), (5, 3), 1), ((0, 2), (0, 0), 0), ((16, 8), (16, 8), 8)])
def test_lora_add_strides(rq, xs, ys, shift, x_type, w_type):
    _say("lora_add strides", xs, ys, shift, x_type, w_type)
    c = _lora_case(50, 4, 24, 136, 144, x_type, w_type, 3)
    for in_place in (False, True):
        _check_lora(*c, _run_lora(rq, *c, in_place, xs, ys, shift))


def test_lora_add_whole_ranks_and_one_scale(rq):
    x, a, b, ids, _, _, y = _lora_case(40, 3, 16, 96, 64, F32, F16, 8)
    a, b = (torch.where(torch.isfinite(t), t, 0.25) for t in (a, b))
    _check_lora(x, a, b, ids, None, None, y, _run_lora(rq, x, a, b, ids, None, None, y, True))
    # ranks out of range are taken as the nearest that is not
    ranks = [-3, 99, 16]
    _check_lora(x, a, b, ids, ranks, None, y, _run_lora(rq, x, a, b, ids, ranks, None, y, False))


def test_lora_add_no_row_in_a_group(rq):
    c = list(_lora_case(20, 3, 16, 96, 64, F16, F16, 8))
    c[3] = np.full(20, -1, np.int32)
    for in_place in (False, True):
        assert torch.equal(_run_lora(rq, *c, in_place), c[6])


@pytest.mark.parametrize("x_type,w_type", LORA_TYPES)
@pytest.mark.parametrize("rows,count,rank,k,n", [(20, 2, 512, 64, 40), (33, 1, 256, 96, 64), (90, 2, 264, 40, 136),
                                                  (50, 3, 300, 33, 12), (200, 1, 8, 8200, 4)])
def test_lora_add_long_ranks_and_rows(rq, rows, count, rank, k, n, x_type, w_type):
    _say("lora_add long", rows, count, rank, k, n, x_type, w_type)
    c = _lora_case(rows, count, rank, k, n, x_type, w_type, rows)
    _check_lora(*c, _run_lora(rq, *c, False))


@pytest.mark.parametrize("w_type", [F16, BF16])
def test_lora_add_values_at_the_ends_of_f32(rq, w_type):
    """Steps of large and of small values, of both in one row, and of infinities: finite rows keep the bound
    (of v's own steps: values below 2^-39 of a step's largest may be lost), the others do not come out finite."""
    rows, k, n, rank = 12, 96, 32, 16
    x, a, b, _, _, _, y = _lora_case(rows, 1, rank, k, n, F32, w_type, 6)
    a, b = (torch.where(torch.isfinite(t), t, 0.25) for t in (a, b))
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3, :32] *= 1e25
    x[4, 40] = 1e-38
    x[5] = 0.0
    x[6, 3], x[7, 90] = float("inf"), float("nan")
    y[1:4] = 0.0
    ids = np.zeros(rows, np.int32)
    got = _run_lora(rq, x, a, b, ids, None, None, y, False)
    assert not torch.isfinite(got[6]).any() and torch.isnan(got[7]).all() and torch.equal(got[5], y[5])
    fine = [r for r in range(rows) if r not in (6, 7)]
    _check_lora(x[fine], a, b, ids[fine], None, None, y[fine], got[fine])


def test_lora_add_own_workspace(rq):
    x, a, b, ids, ranks, scales, y = _lora_case(30, 3, 16, 4096, 64, F32, F16, 4)
    wa, wb = rq.Weight.from_tensor(a.to(DEV)), rq.Weight.from_tensor(b.to(DEV))
    g = rq.group_rows(torch.from_numpy(ids).to(DEV), 3)
    size = rq.lora_add_workspace_size(wa, 30)
    ws = torch.full((size + 64,), 7, dtype=torch.uint8, device=DEV)
    yd, rd, sd = y.to(DEV), torch.tensor(ranks, dtype=torch.int32, device=DEV), torch.tensor(scales, device=DEV)
    rq.lora_add(x.to(DEV), wa, wb, g, yd, ranks=rd, scales=sd, workspace=ws[:size])
    _check_lora(x, a, b, ids, ranks, scales, y, yd.cpu())
    assert (ws[size:] == 7).all()
    with pytest.raises(rq.InvalidInputError, match="needs"):
        rq.lora_add(x.to(DEV), wa, wb, g, yd, workspace=ws[:16])
    with pytest.raises(rq.ReflexError, match="16-byte aligned"):
        rq.lora_add(x.to(DEV), wa, wb, g, yd, workspace=ws[8:])


def test_python_counts_do_not_wrap(rq):
    x = torch.zeros(4, 8, dtype=F16, device=DEV)
    w = rq.Weight.from_tensor(torch.zeros(2, 8, 8, dtype=F16, device=DEV))
    offsets = torch.zeros(3, dtype=torch.int32, device=DEV)
    out = torch.zeros(4, 8, dtype=F16, device=DEV)
    for n in (-1, 1 << 31, (1 << 32) + 4):
        with pytest.raises(rq.InvalidInputError, match="rows="):
            rq.grouped_gemm(x, w, offsets, n, out=out)
        with pytest.raises(rq.InvalidInputError, match="x_div="):
            rq.grouped_gemm(x, w, offsets, 2, x_index=offsets, x_div=n, out=out)
        with pytest.raises(rq.InvalidInputError, match="groups="):
            rq.group_rows(offsets, n)


def test_stacks_from_a_file(rq, tmp_path):
    """F16 and BF16 expert tensors of a GGUF file, uploaded and multiplied."""
    from test_gguf import write_gguf

    k, n, groups, rows = 72, 40, 3, 30
    stacks = {}
    tensors = []
    for name, t, ty in (("a", F16, 1), ("b", BF16, 30)):
        x, w = _case(rows, groups, k, n, t, t, ty)
        stacks[name] = (x, w)
        tensors.append((name, [k, n, groups], ty, w.view(torch.int16).numpy().tobytes()))
    write_gguf(tmp_path / "f.gguf", [], tensors)
    weights = rq.GgufFile(tmp_path / "f.gguf").upload(["a", "b"], device=DEV)
    offsets, _ = _grouped(_ids(rows, groups, "all"), groups)
    for name, (x, w) in stacks.items():
        assert weights[name].shape == [k, n, groups]
        y = rq.grouped_gemm(x.to(DEV), weights[name], torch.from_numpy(offsets).to(DEV), rows)
        _check_grouped(x, w, offsets, None, 1, None, y.cpu())


# ------------------------------------------------------------------ together, captured, on other streams

def _expert_layer(rq, x, logits, weights, top_k):
    """Routed experts of half-typed stacks in the library's own f32 activations."""
    tokens, groups = logits.shape
    ids, share = rq.moe_route_device(logits.reshape(-1), tokens, groups, top_k, True)
    g = rq.group_rows(ids.reshape(-1), groups)
    pairs = tokens * top_k
    gate, up = (rq.grouped_gemm(x, w, g.offsets, pairs, x_index=g.order, x_div=top_k) for w in weights[:2])
    inner = rq.silu_and_mul(gate, up)
    down = rq.grouped_gemm(inner, weights[2], g.offsets, pairs, y_index=g.order)
    return (down.view(tokens, top_k, -1) * share.unsqueeze(2)).sum(1), ids, share


def _layer_inputs(tokens, groups, hidden, ffn, w_type, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=gen)
    logits = torch.randn(tokens, groups, generator=gen)
    w = [(torch.randn(groups, *s, generator=gen) * 0.05).to(w_type) for s in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
    return x, logits, w


def _layer_64(x, ids, share, w):
    x, w = x.double(), [t.double() for t in w]
    out = torch.zeros_like(x)
    for t in range(x.shape[0]):
        for e, s in zip(ids[t].tolist(), share[t].tolist()):
            gate, up = w[0][e] @ x[t], w[1][e] @ x[t]
            out[t] += s * (w[2][e] @ (gate / (1 + torch.exp(-gate)) * up))
    return out


@pytest.mark.parametrize("w_type", [F16, BF16])
@pytest.mark.parametrize("tokens", [1, 7, 90])
def test_expert_layer_and_adapters(rq, tokens, w_type):
    """Route, group, three grouped products; then adapters beside a quantized projection of the result.
    Each product is f32 through and through, so the layer is within 2^-17 of 64 bits in norm (three products
    of 2^-19 each and SiLU's few steps)."""
    from reflex_amd import synth

    hidden, ffn, groups, top_k = 256, 192, 16, 4
    x, logits, w = _layer_inputs(tokens, groups, hidden, ffn, w_type, tokens)
    weights = [rq.Weight.from_tensor(t.to(DEV)) for t in w]
    out, ids, share = _expert_layer(rq, x.to(DEV), logits.to(DEV), weights, top_k)
    want = _layer_64(x, ids.cpu(), share.cpu(), w)
    assert (out.cpu().double() - want).norm() <= 2.0 ** -17 * want.norm()

    n, rank, count = 320, 8, 3
    q = rq.Weight.from_blocks(12, synth.weights(12, n, hidden, 5), hidden, n, device=DEV)
    y = rq.gemm(out.reshape(-1), q, tokens).view(tokens, n)
    base = y.cpu()
    _, a, b, _, _, scales, _ = _lora_case(1, count, rank, hidden, n, F32, w_type, 4)
    a, b = (torch.where(torch.isfinite(t), t, 0.25) for t in (a, b))
    adapter = (np.arange(tokens) % (count + 1)).astype(np.int32)
    g = rq.group_rows(torch.from_numpy(adapter).to(DEV), count)
    wa, wb = rq.Weight.from_tensor(a.to(DEV)), rq.Weight.from_tensor(b.to(DEV))
    rq.lora_add(out, wa, wb, g, y, scales=torch.tensor(scales, device=DEV))
    _check_lora(out.cpu(), a, b, adapter, None, scales, base, y.cpu())


@pytest.mark.parametrize("gate_type,down_type", [(F16, F16), (BF16, BF16), (F16, BF16)])
@pytest.mark.parametrize("tokens,groups,hidden,ffn,top_k", [(1, 8, 128, 96, 2), (5, 3, 100, 77, 3), (64, 16, 256, 192, 4),
                                                            (300, 12, 264, 160, 5)])
def test_moe_ffn_grouped_half_stacks(rq, tokens, groups, hidden, ffn, top_k, gate_type, down_type):
    """The library's own expert layer over F16 / BF16 stacks, routed on the device and on the host.
    Within 2^-17 of 64 bits in norm (see test_expert_layer_and_adapters)."""
    _say("moe_ffn_grouped half", tokens, groups, hidden, ffn, top_k, gate_type, down_type)
    x, logits, w = _layer_inputs(tokens, groups, hidden, ffn, gate_type, tokens)
    w[2] = w[2].to(down_type)
    weights = [rq.Weight.from_tensor(t.to(DEV)) for t in w]
    xd, ld = x.to(DEV).reshape(-1), logits.to(DEV).reshape(-1)
    ids, share = rq.moe_route_device(ld, tokens, groups, top_k, True, 1.5)
    want = _layer_64(x, ids.cpu(), share.cpu(), w)
    out = torch.full((tokens * hidden,), float("nan"), device=DEV)
    rq.moe_ffn_grouped_device(xd, tokens, hidden, ld, groups, top_k, True, 1.5, *weights, out)
    first = out.cpu()
    assert (first.view(tokens, hidden).double() - want).norm() <= 2.0 ** -17 * want.norm()
    out.fill_(float("nan"))
    rq.moe_ffn_grouped_device(xd, tokens, hidden, ld, groups, top_k, True, 1.5, *weights, out)
    assert torch.equal(out.cpu(), first)
    out.fill_(float("nan"))
    rq.moe_ffn_grouped(xd, tokens, hidden, logits.numpy(), groups, top_k, True, 1.5, *weights, out)
    assert (out.cpu().view(tokens, hidden).double() - want).norm() <= 2.0 ** -17 * want.norm()


def test_moe_ffn_grouped_half_refusals(rq):
    x, logits, w = _layer_inputs(4, 4, 64, 48, F16, 1)
    g, u, d = (rq.Weight.from_tensor(t.to(DEV)) for t in w)
    q = rq.Weight.from_blocks(12, np.zeros(4 * 256 * 144, np.uint8), 256, 256, expert_count=4, device=DEV)
    xd, ld, out = x.to(DEV), logits.to(DEV), torch.empty(4 * 64, device=DEV)
    run = lambda *a, k=2, o=out: rq.moe_ffn_grouped_device(xd, 4, 64, ld, 4, k, True, 1.0, *a, o)  # noqa: E731
    with pytest.raises(rq.ReflexError, match="shapes"):
        run(g, u, u)
    with pytest.raises(rq.ReflexError, match="k \\(5\\)"):
        run(g, u, d, k=5)
    with pytest.raises(rq.InvalidInputError, match="overlap"):
        run(g, u, d, o=xd)
    with pytest.raises(rq.ReflexError):  # half-typed and quantized stacks in one layer
        run(g, u, q)


def test_moe_ffn_grouped_half_captured(rq):
    tokens, hidden, ffn, groups, top_k = 40, 128, 96, 8, 2
    x, logits, w = _layer_inputs(tokens, groups, hidden, ffn, BF16, 3)
    weights = [rq.Weight.from_tensor(t.to(DEV)) for t in w]
    xd, ld = x.to(DEV), logits.to(DEV)
    out = torch.empty(tokens * hidden, device=DEV)
    step = lambda: rq.moe_ffn_grouped_device(xd, tokens, hidden, ld, groups, top_k, True, 1.0, *weights, out)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for r in range(3):
        xd.copy_(torch.randn(tokens, hidden))
        ld.copy_(torch.randn(tokens, groups))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out), f"replay {r}"


def test_captured_and_replayed(rq):
    """The whole run in one graph, replayed on new inputs, with eager work between."""
    tokens, hidden, ffn, groups, top_k = 33, 128, 96, 8, 2
    x, logits, w = _layer_inputs(tokens, groups, hidden, ffn, F16, 1)
    weights = [rq.Weight.from_tensor(t.to(DEV)) for t in w]
    pairs = tokens * top_k
    xd, ld, ids = x.to(DEV), logits.to(DEV), torch.empty(pairs, dtype=torch.int32, device=DEV)
    g = rq.RowGroups(torch.empty(groups + 1, dtype=torch.int32, device=DEV), torch.empty_like(ids))
    gate, y = (torch.empty(pairs, m, device=DEV) for m in (ffn, hidden))
    a = rq.Weight.from_tensor((torch.randn(groups, 5, ffn) * 0.1).half().to(DEV))
    b = rq.Weight.from_tensor((torch.randn(groups, hidden, 5) * 0.1).half().to(DEV))
    lws = torch.empty(rq.lora_add_workspace_size(a, pairs), dtype=torch.uint8, device=DEV)

    def step():
        ids.copy_(ld.topk(top_k, dim=1).indices.reshape(-1))
        rq.group_rows(ids, groups, out=g)
        rq.grouped_gemm(xd, weights[0], g.offsets, pairs, x_index=g.order, x_div=top_k, out=gate)
        rq.grouped_gemm(gate, weights[2], g.offsets, pairs, y_index=g.order, out=y)
        rq.lora_add(gate, a, b, g, y, workspace=lws)
        return y

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for r in range(4):
        xd.copy_(torch.randn(tokens, hidden))
        ld.copy_(torch.randn(tokens, groups))
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        want = step().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {r}"


def test_other_stream(rq):
    """Calls go to the current stream, behind the work that makes their inputs there."""
    x, w = _case(200, 5, 256, 128, F16, F16, 6)
    offsets, _ = _grouped(_ids(200, 5, "all"), 5)
    weight, od = rq.Weight.from_tensor(w.to(DEV)), torch.from_numpy(offsets).to(DEV)
    s = torch.cuda.Stream()
    xd = torch.zeros(200, 256, dtype=F16, device=DEV)
    src = x.to(DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        big = torch.randn(2048, 2048, device=DEV)
        for _ in range(20):
            big = big @ big * 1e-3
        xd.copy_(src)
        y = rq.grouped_gemm(xd, weight, od, 200)
    s.synchronize()
    _check_grouped(x, w, offsets, None, 1, None, y.cpu())


def test_same_results_every_time(rq):
    x, a, b, ids, ranks, scales, y = _lora_case(37, 4, 16, 4096, 512, F32, F16, 2)
    first = _run_lora(rq, x, a, b, ids, ranks, scales, y, False)
    for _ in range(3):
        assert torch.equal(_run_lora(rq, x, a, b, ids, ranks, scales, y, False), first)


# ------------------------------------------------------------------ v = A x to its last bit

def _whole_v(rows, count, rank, k, n, x_type, w_type):
    """A case in which every sum is exact in f32, whatever its order. v is 1.something times a power of two a row,
    of all the bits that are kept: 24 (F32 adapters: in one value of A; BF16: in three), 22 (F16: in two). Each
    value of A that counts lies in 32 of K of its own, and a row of B has a single power of two. y is the
    adapter's part rounded to 8 bits and negated: what is left of their sum is the lower bits of v alone."""
    gen = torch.Generator().manual_seed(rows + rank)
    pieces, bits = {F32: (1, 24), F16: (2, 11), BF16: (3, 8)}[w_type]
    a = torch.randn(count, rank, k, generator=gen).to(w_type)
    x = torch.zeros(rows, k)
    sign = torch.where(torch.arange(rows) % 3 == 1, -1.0, 1.0) * 2.0 ** (torch.arange(rows) % 7 - 3)
    for p in range(pieces):
        a[:, :, 37 * p + 5] = (1 + 0.9 * torch.rand(count, rank, generator=gen)).to(w_type)
        x[:, 37 * p + 5] = sign * 2.0 ** (-bits * p)
    b = torch.zeros(count, n, rank)
    b[:, torch.arange(n), torch.arange(n) % rank] = 2.0 ** (torch.arange(n) % 3)
    ids = (torch.arange(rows) * 7 % count).to(torch.int32)
    v = torch.stack([a[g].double() @ x[r].double() for r, g in enumerate(ids.tolist())])
    assert torch.equal(v.float().double(), v) and (v.abs() >= 2.0 ** -3).all()
    delta = 2.0 * v @ b[0].double().t()
    y = -delta.to(BF16).to(x_type)
    want = (delta + y.double()).to(x_type)
    return x.to(x_type), a, b.to(w_type), ids.numpy(), y, want


@pytest.mark.parametrize("x_type,w_type", LORA_TYPES)
@pytest.mark.parametrize("rows,count,rank,n", [(3, 2, 16, 48), (40, 2, 40, 52), (9, 3, 13, 51), (20, 2, 264, 300)])
def test_lora_add_keeps_v(rq, rows, count, rank, n, x_type, w_type):
    """A x is kept to 22 bits beside F16 adapters and to all of f32's 24 beside the others: where y and the
    adapter cancel, only the result's own rounding is left."""
    _say("lora_add keeps v", rows, count, rank, n, x_type, w_type)
    x, a, b, ids, y, want = _whole_v(rows, count, rank, 128, n, x_type, w_type)
    got = _run_lora(rq, x, a, b, ids, None, [2.0] * count, y, False)
    assert torch.equal(got, want), (got.double() - want.double()).abs().max()


def test_moe_ffn_grouped_half_one_rule_for_both_entries(rq):
    """Gate and up of two half types, x at any element, stacks in memory that is longer than they are: layers that
    the device-routed entry runs, the host-routed one runs too. Bound: see test_expert_layer_and_adapters."""
    tokens, groups, hidden, ffn, top_k = 6, 5, 72, 40, 2
    x, logits, w = _layer_inputs(tokens, groups, hidden, ffn, F16, 9)
    w[1] = w[1].to(BF16)
    weights = []
    for t in w:
        memory = torch.cat([t.reshape(-1), torch.full((3,), float("nan"), dtype=t.dtype)]).to(DEV)
        weights.append(rq.Weight(rq.GgmlType.F16 if t.dtype == F16 else rq.GgmlType.BF16, memory,
                                 list(reversed(t.shape)), len=memory.numel() * 2))
    memory = torch.full((1 + tokens * hidden,), float("nan"), device=DEV)
    xd = memory[1:]
    xd.copy_(x.reshape(-1))
    ld = logits.to(DEV).reshape(-1)
    ids, share = rq.moe_route_device(ld, tokens, groups, top_k, True, 1.0)
    want = _layer_64(x, ids.cpu(), share.cpu(), w)
    for entry, lg in ((rq.moe_ffn_grouped_device, ld), (rq.moe_ffn_grouped, logits.numpy())):
        _say("moe_ffn_grouped", entry.__name__)
        out = torch.full((tokens * hidden,), float("nan"), device=DEV)
        entry(xd, tokens, hidden, lg, groups, top_k, True, 1.0, *weights, out)
        assert (out.cpu().view(tokens, hidden).double() - want).norm() <= 2.0 ** -17 * want.norm()


FEW4, FEW, QUARTERS, LARGE, COPIED, TILES = range(6)  # rfxq_grouped_policy.kernel


# (kernel of half-typed, of f32 activations): ten steps of 64 of K and more, so that every buffer is filled
# again several times; odd and even numbers of steps, whole and with a tail
@pytest.mark.parametrize("x_type,w_type,y_type", TYPES)
@pytest.mark.parametrize("rows,groups,k,n,shift,half_kernel,f32_kernel", [
    (1500, 2, 704, 7168, 0, LARGE, TILES), (1500, 2, 776, 7161, 0, LARGE, TILES), (1536, 2, 640, 7168, 0, LARGE, TILES),
    (1000, 3, 704, 520, 0, COPIED, QUARTERS), (1000, 3, 776, 520, 0, COPIED, QUARTERS), (999, 3, 648, 513, 0, COPIED, QUARTERS),
    (2000, 4, 704, 2104, 0, TILES, TILES), (2000, 4, 776, 2104, 0, TILES, TILES), (2000, 4, 649, 2103, 1, TILES, TILES),
    (600, 4, 771, 1400, 3, TILES, QUARTERS), (400, 4, 2888, 1000, 0, COPIED, QUARTERS), (400, 4, 2891, 1001, 1, TILES, QUARTERS),
    (150, 40, 1160, 1032, 0, FEW4, FEW), (60, 32, 1992, 1024, 0, FEW4, FEW), (40, 9, 1355, 48, 1, FEW4, FEW4),
    (70, 64, 904, 1032, 0, FEW, FEW)])
def test_grouped_gemm_many_steps(rq, rows, groups, k, n, shift, half_kernel, f32_kernel, x_type, w_type, y_type):
    import ctypes

    want = f32_kernel if x_type == F32 else half_kernel
    _say("grouped_gemm many steps", rows, groups, k, n, shift, x_type, w_type, y_type)
    x, w = _case(rows, groups, k, n, x_type, w_type, rows + k)
    p = rq.RfxqGroupedPolicy()
    xr = rq.RfxqRows(1 << 20 | x.element_size() * shift, {F32: 0, F16: 1, BF16: 30}[x_type], rows, k + 8 - k % 8)
    wt = rq.Weight.from_tensor(w)
    rq.lib().rfxq_grouped_gemm_policy(ctypes.byref(xr), wt.cref(), rows, ctypes.byref(p))
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert p.kernel == want
    offsets, order = _grouped(_ids(rows, groups, "all"), groups)
    y, kept = _run_grouped(rq, x, w, offsets, rows, order, 1, order, y_type, rows, (8 - k % 8, shift), (8, 0), 8 * (shift == 0))
    _check_grouped(x, w, offsets, order, 1, order, y)
    assert kept


# ------------------------------------------------------------------ adapters: orders and offsets of any values

def _lora_ordered(rq, c, offsets, order):
    """lora_add on given offsets and order (out apart from y): the result, what lies around it unchanged."""
    x, a, b, _, ranks, scales, y = c
    dev = lambda v, t=torch.int32: None if v is None else torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    out, memory = _strided(torch.full(y.shape, 123.0, dtype=y.dtype), y.shape[1] + 8, 8, 99.0)
    rq.lora_add(x.to(DEV), *(rq.Weight.from_tensor(t.to(DEV)) for t in (a, b)), rq.RowGroups(dev(offsets), dev(order)),
                y.to(DEV), ranks=dev(ranks), scales=dev(scales, F32), out=out)
    torch.cuda.synchronize()
    got, around = out.cpu(), memory.clone()
    around[8:8 + y.shape[0] * (y.shape[1] + 8)].view(y.shape[0], -1)[:, :y.shape[1]] = 99.0
    assert bool((around == 99.0).all())
    return got


@pytest.mark.parametrize("x_type,w_type", LORA_TYPES)
@pytest.mark.parametrize("rows,count,rank,k,n", [(1, 1, 8, 40, 16), (50, 4, 24, 136, 144), (200, 3, 13, 72, 33)])
def test_lora_add_without_an_order(rq, rows, count, rank, k, n, x_type, w_type):
    """order = None: the rows themselves are grouped; rows behind the last group are copied."""
    _say("lora_add without an order", rows, count, rank, k, n, x_type, w_type)
    c = _lora_case(rows, count, rank, k, n, x_type, w_type, rows)
    ids = np.sort(np.where((c[3] < 0) | (c[3] >= count), count, c[3])).astype(np.int32)
    offsets, _ = _grouped(ids, count)
    got = _lora_ordered(rq, c, offsets.tolist(), None)
    _check_lora(*c[:3], ids, *c[4:], got)


@pytest.mark.parametrize("x_type,w_type", LORA_TYPES)
@pytest.mark.parametrize("rows,count,rank,k,n", [(70, 3, 16, 64, 72), (140, 3, 11, 200, 45)])
def test_lora_add_order_out_of_range(rq, rows, count, rank, k, n, x_type, w_type):
    """Places that name no row compute nothing; a row that the order does not list keeps what out held."""
    _say("lora_add order out of range", rows, count, rank, k, n, x_type, w_type)
    c = _lora_case(rows, count, rank, k, n, x_type, w_type, rows)
    offsets, order = _grouped(c[3], count)
    at = [0, 5, 31, rows - 1]
    left = order[at].copy()
    order[at] = [-1, rows, -(1 << 31), (1 << 31) - 1]
    got = _lora_ordered(rq, c, offsets.tolist(), order.tolist())
    assert bool((got[left] == 123.0).all())
    keep = np.setdiff1d(np.arange(rows), left)
    _check_lora(c[0][keep], *c[1:3], c[3][keep], *c[4:6], c[6][keep], got[keep])


@pytest.mark.parametrize("rank,n", [(16, 72), (11, 45)])
@pytest.mark.parametrize("offsets", [[5, 9, 9, 20], [0, 40, 10, 50], [-7, 3, 1 << 30, 50], [50, 50, 0, 0],
                                     [0, -(1 << 31), (1 << 31) - 1, -5], [0, 0, 0, 1 << 30]])
def test_lora_add_odd_offsets(rq, offsets, rank, n):
    """Offsets that do not rise from 0 to the rows stay inside the arrays: every row is what it was, or y's, with
    or without an adapter's part."""
    _say("lora_add odd offsets", offsets, rank, n)
    x, a, b, _, _, _, y = _lora_case(50, 3, rank, 64, n, F16, F16, 9)
    a, b = (torch.where(torch.isfinite(t), t, 0.25) for t in (a, b))
    got = _lora_ordered(rq, (x, a, b, None, None, None, y), offsets, list(range(50)))
    one = [_run_lora(rq, x, a, b, np.full(50, g, np.int32), None, None, y, False) for g in range(3)]
    for r in range(50):
        assert any(torch.equal(got[r], t[r]) for t in [torch.full_like(y, 123.0), y] + one) or \
            sum(b <= r < e for b, e in zip(offsets, offsets[1:])) + (r >= offsets[-1]) > 1, r


# ------------------------------------------------------------------ weights that are not finite

@pytest.mark.parametrize("x_type,w_type,y_type", TYPES[:4])
@pytest.mark.parametrize("rows,groups,k,n", [(30, 3, 72, 40), (1000, 3, 136, 520), (2000, 4, 72, 2104)])
def test_grouped_gemm_weights_not_finite(rq, rows, groups, k, n, x_type, w_type, y_type):
    """An infinite or NaN weight leaves its own column of its own group without a finite result, and no other."""
    _say("grouped_gemm weights not finite", rows, groups, k, n, x_type, w_type)
    x, w = _case(rows, groups, k, n, x_type, w_type, 21)
    offsets, _ = _grouped(_ids(rows, groups, "all"), groups)
    lost = {(0, 3): float("inf"), (1, n - 1): float("-inf"), (2, 17): float("nan")}
    clean = w.clone()
    for i, ((g, c), v) in enumerate(lost.items()):
        w[g, c, (5 + 30 * i) % k] = v
    y, kept = _run_grouped(rq, x, w, offsets, rows, None, 1, None, y_type, rows)
    assert kept
    for g, c in lost:
        part = y[offsets[g]:offsets[g + 1], c]
        assert part.numel() and not torch.isfinite(part).any()
        # the column's own results are checked above; the others against the weights without it
        x64 = x[offsets[g]:offsets[g + 1]].double().numpy()
        y[offsets[g]:offsets[g + 1], c] = torch.from_numpy(x64 @ clean[g, c].double().numpy()).to(y_type)
    _check_grouped(x, clean, offsets, None, 1, None, y)


@pytest.mark.parametrize("x_type,w_type", LORA_TYPES)
@pytest.mark.parametrize("rows,count,rank,k,n", [(20, 2, 16, 72, 40), (90, 2, 24, 136, 144), (33, 2, 13, 75, 51)])
def test_lora_add_weights_not_finite(rq, rows, count, rank, k, n, x_type, w_type):
    """An infinite value of B leaves its column of its adapter's rows without a finite result, one of A all of them;
    the other adapter's rows keep theirs."""
    _say("lora_add weights not finite", rows, count, rank, k, n, x_type, w_type)
    x, a, b, _, _, scales, y = _lora_case(rows, count, rank, k, n, x_type, w_type, 5)
    a, b = (torch.where(torch.isfinite(t), t, 0.25) for t in (a, b))
    ids = (np.arange(rows) % 2).astype(np.int32)
    bad = b.clone()
    bad[0, n // 2, rank - 2] = float("inf")
    got = _run_lora(rq, x, a, bad, ids, None, scales, y, False)
    assert not torch.isfinite(got[0::2, n // 2]).any()
    keep = [c for c in range(n) if c != n // 2]
    _check_lora(x, a, b[:, keep], ids, None, scales, y[:, keep], got[:, keep])
    bad = a.clone()
    bad[0, rank - 2, k // 3] = float("-inf")
    got = _run_lora(rq, x, bad, b, ids, None, scales, y, False)
    assert not torch.isfinite(got[0::2]).any()
    _check_lora(x[1::2], a, b, ids[1::2], None, scales, y[1::2], got[1::2])


# ------------------------------------------------------------------ the largest calls, and calls side by side

@pytest.mark.parametrize("groups", [1, 300, 1024])
def test_group_rows_of_the_most_rows(rq, groups):
    n = 1 << 24
    _say("group_rows", n, groups)
    ids = _ids(n, groups, "any")
    g = rq.group_rows(torch.from_numpy(ids).to(DEV), groups)
    want_offsets, want_order = _grouped(ids, groups)
    assert np.array_equal(g.offsets.cpu().numpy(), want_offsets) and np.array_equal(g.order.cpu().numpy(), want_order)


def test_lora_add_rows_past_4_gib(rq):
    """Rows of x, y and out whose bytes lie past 32-bit offsets; the first, some and the last are looked at."""
    _say("lora_add past 4 GiB")
    rows, count, rank, k, n = 2_200_001, 3, 8, 1024, 1024
    gen = torch.Generator(device=DEV).manual_seed(3)
    x, y = (torch.empty(rows, m, dtype=F16, device=DEV) for m in (k, n))
    for t in (x, y):
        for b in range(0, rows, 1 << 18):
            t[b:b + (1 << 18)].normal_(generator=gen)
    a, b = ((torch.randn(*s, generator=torch.Generator().manual_seed(4)) * 0.05).half() for s in ((count, rank, k), (count, n, rank)))
    ids = (torch.arange(rows, dtype=torch.int32, device=DEV) * 7 % (count + 1))
    out = torch.full((rows, n), 123.0, dtype=F16, device=DEV)
    rq.lora_add(x, rq.Weight.from_tensor(a.to(DEV)), rq.Weight.from_tensor(b.to(DEV)), rq.group_rows(ids, count), y, out=out)
    at = torch.cat([torch.arange(0, 40), torch.arange(rows // 2, rows // 2 + 40), torch.arange(rows - 200, rows)])
    d = at.to(DEV)
    _check_lora(x[d].cpu(), a, b, ids[d].cpu().numpy(), None, None, y[d].cpu(), out[d].cpu())
    none = ids == count
    assert torch.equal(out[none], y[none]) and not bool((out[~none] == 123.0).all(1).any())


def test_lora_add_stacks_past_4_gib(rq):
    """Adapters whose bytes lie past 32-bit offsets in their stacks."""
    _say("lora_add stacks past 4 GiB")
    rows, count, rank, k, n = 70, 1000, 256, 8256, 8320
    a, b = (torch.zeros(count, *s, dtype=F16, device=DEV) for s in ((rank, k), (n, rank)))
    c = _lora_case(rows, 2, rank, k, n, F16, F16, 8)
    a[-2:], b[-2:] = c[1].to(DEV), c[2].to(DEV)
    far = torch.from_numpy(np.where((c[3] == 0) | (c[3] == 1), c[3] + count - 2, -1).astype(np.int32)).to(DEV)
    full = lambda v, t: torch.cat([torch.zeros(count - 2, dtype=t), torch.tensor(v, dtype=t)]).to(DEV)  # noqa: E731
    got = rq.lora_add(c[0].to(DEV), rq.Weight.from_tensor(a), rq.Weight.from_tensor(b), rq.group_rows(far, count), c[6].to(DEV),
                      ranks=full(c[4], torch.int32), scales=full(c[5], F32))
    _check_lora(*c, got.cpu())


def test_two_streams_at_once(rq):
    """Calls on two streams that overlap, each with its own workspace."""
    cases = [_lora_case(300, 5, 40, 4096, 264, F32, BF16, s) for s in (1, 2)]
    ids = [torch.from_numpy(_ids(70_001, 300, "any", s)).to(DEV) for s in (1, 2)]
    want = [rq.group_rows(i, 300) for i in ids]
    dev = [(x.to(DEV), rq.Weight.from_tensor(a.to(DEV)), rq.Weight.from_tensor(b.to(DEV)),
            rq.group_rows(torch.from_numpy(i).to(DEV), 5), torch.tensor(r, dtype=torch.int32, device=DEV),
            torch.tensor(s, device=DEV), y.to(DEV)) for x, a, b, i, r, s, y in cases]
    lws = [torch.empty(rq.lora_add_workspace_size(d[1], 300), dtype=torch.uint8, device=DEV) for d in dev]
    gws = [torch.empty(rq.group_rows_workspace_size(70_001, 300), dtype=torch.uint8, device=DEV) for _ in dev]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs, groups = [[], []], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, a, b, g, r, sc, y = dev[i]
                outs[i].append(rq.lora_add(x, a, b, g, y, ranks=r, scales=sc, out=torch.empty_like(y), workspace=lws[i]))
                groups[i].append(rq.group_rows(ids[i], 300, workspace=gws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        _check_lora(*cases[i], outs[i][0].cpu())
        assert all(torch.equal(o, outs[i][0]) for o in outs[i])
        assert all(torch.equal(g.order, want[i].order) and torch.equal(g.offsets, want[i].offsets) for g in groups[i])


def test_moe_ffn_grouped_half_host_routing_is_not_captured(rq):
    """The host-routed layer copies its routing up, which a graph would not repeat: refused while capturing, and
    the graph of what came before it is whole."""
    x, logits, w = _layer_inputs(4, 4, 64, 48, F16, 1)
    weights = [rq.Weight.from_tensor(t.to(DEV)) for t in w]
    xd, out, seen = x.to(DEV), torch.full((4 * 64,), 5.0, device=DEV), torch.zeros(8, device=DEV)
    run = lambda: rq.moe_ffn_grouped(xd, 4, 64, logits.numpy(), 4, 2, True, 1.0, *weights, out)  # noqa: E731
    run()
    torch.cuda.synchronize()
    out.fill_(5.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seen.add_(1.0)
        with pytest.raises(rq.InvalidInputError, match="captured"):
            run()
    for r in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert bool((seen == r + 1.0).all()) and bool((out == 5.0).all())

"""Refusals and workspace sizes of the entry points on grouped rows (rfxq_group_rows,
rfxq_grouped_gemm, rfxq_lora_add): all of them are decided on the host, before any launch, so
they run without a GPU (addresses that are never read)."""
import ctypes

import pytest
import torch

P = 1 << 20  # a plausible device address
F32, F16, BF16, Q4K = 0, 1, 30, 12


@pytest.fixture(scope="module")
def L():
    import reflex_amd

    return reflex_amd.lib()


def _weight(ty=F16, k=64, n=32, e=4, data=P, length=None):
    import reflex_amd as rq

    size = {F32: 4, F16: 2, BF16: 2}.get(ty, 2)
    return rq.RfxqWeight(ty, k, n, e, data, k * n * max(e, 1) * size if length is None else length)


def _rows(ty=F16, rows=8, stride=64, data=2 * P):
    import reflex_amd as rq

    return rq.RfxqRows(data, ty, rows, stride)


def _expect(L, rc, code, text):
    assert rc == code and text in L.rfxq_last_error().decode(), (rc, L.rfxq_last_error())


@pytest.mark.parametrize("change,code,text", [
    ({"groups": 0}, 12, "groups=0"),
    ({"groups": 1025}, 12, "groups=1025"),
    ({"n": (1 << 24) + 1}, 12, "at most"),
    ({"ids": None}, 11, "NULL"),
    ({"offsets": None}, 11, "NULL"),
    ({"order": None}, 11, "NULL"),
    ({"ids": P + 2}, 12, "4-byte aligned"),
    ({"order": P}, 11, "overlap"),
    ({"order": P + 4}, 11, "overlap"),
    ({"offsets": 3 * P + 8}, 11, "overlap"),
])
def test_group_rows_refusals(L, change, code, text):
    a = {"ids": P, "n": 100, "groups": 8, "offsets": 2 * P, "order": 3 * P, **change}
    _expect(L, L.rfxq_group_rows(a["ids"], a["n"], a["groups"], a["offsets"], a["order"], None, 0, None), code, text)


def _grouped(L, x=None, w=None, offsets=5 * P, rows=8, x_index=None, x_div=1, y_index=None, y=None):
    ref = lambda v: None if v is None else ctypes.byref(v)  # noqa: E731
    return L.rfxq_grouped_gemm(ref(x), ref(w), offsets, rows, x_index, x_div, y_index, ref(y), None)


@pytest.mark.parametrize("change,code,text", [
    ({"w": None}, 11, "weight is NULL"),
    ({"w": {"ty": Q4K}}, 1, "F16 or BF16"),
    ({"w": {"ty": F32}}, 1, "F16 or BF16"),
    ({"w": {"k": 0}}, 12, "shape"),
    ({"w": {"n": 0}}, 12, "shape"),
    ({"w": {"e": 1025}}, 12, "expert_count=1025"),
    ({"w": {"length": 64 * 32 * 4 * 2 - 1}}, 12, "needs"),
    ({"w": {"k": 0xFFFFFFFF, "n": 0xFFFFFFFF, "length": 1 << 40}}, 12, "needs"),
    ({"w": {"data": None}}, 11, "data is NULL"),
    ({"w": {"data": P + 1}}, 12, "aligned"),
    ({"x": None}, 11, "x is NULL"),
    ({"x": {"ty": Q4K}}, 1, "of type 12"),
    ({"x": {"ty": BF16}}, 11, "x of type 30"),
    ({"x": {"stride": 63}}, 12, "stride=63"),
    ({"x": {"data": None}}, 11, "x data is NULL"),
    ({"x": {"data": P + 1}}, 12, "aligned"),
    ({"y": None}, 11, "y is NULL"),
    ({"y": {"ty": BF16}}, 11, "y of type 30"),
    ({"y": {"stride": 31}}, 12, "stride=31"),
    ({"y": {"data": 2 * P + 64}}, 11, "overlap"),
    ({"rows": 1 << 31}, 12, "rows="),
    ({"w": {"k": 1 << 31, "n": 1, "length": 1 << 40}}, 12, "shape"),
    ({"w": {"k": 1, "n": 1 << 31, "length": 1 << 40}}, 12, "shape"),
    ({"x": {"rows": 1 << 30, "stride": 1 << 40}}, 12, "rows of x"),
    ({"y": {"rows": 1 << 30, "stride": 1 << 20}}, 12, "rows of y"),
    ({"x_div": 0}, 11, "x_div=0"),
    ({"x_div": 2}, 11, "without x_index"),
    ({"offsets": None}, 11, "offsets is NULL"),
])
def test_grouped_gemm_refusals(L, change, code, text):
    a = {"x": {}, "w": {}, "y": {}, **change}
    for m, make in (("x", _rows), ("w", _weight), ("y", lambda **c: _rows(**{"stride": 32, "data": 4 * P, **c}))):
        if a[m] is not None:
            a[m] = make(**a[m])
    _expect(L, _grouped(L, **a), code, text)


@pytest.mark.parametrize("empty", ["rows", "x", "y"])
def test_grouped_gemm_of_nothing(L, empty):
    a = {"x": _rows(), "w": _weight(), "y": _rows(stride=32, data=4 * P)}
    if empty == "rows":
        a["rows"] = 0
    else:
        a[empty].rows = 0
    assert _grouped(L, **a) == 0


FEW4, FEW, QUARTERS, LARGE, COPIED, TILES = range(6)


@pytest.mark.parametrize("rows,groups,k,n,f32,shift,kernel", [
    # few tiles, of either kind; rows that do not start at 16 bytes up to a lower limit
    (20, 1, 264, 24, True, 0, FEW4), (48, 3, 640, 4096, False, 0, FEW4), (48, 3, 640, 4112, False, 0, COPIED),
    (32, 2, 640, 4096, False, 2, FEW4), (32, 2, 640, 4112, False, 2, TILES),
    # few rows a group
    (256, 128, 768, 2048, True, 0, FEW), (512, 256, 72, 768, False, 0, FEW), (768, 256, 72, 768, False, 0, TILES),
    (512, 128, 1024, 2048, False, 0, FEW4), (640, 128, 1024, 2048, False, 0, TILES),
    (60, 32, 1992, 1024, True, 0, FEW), (60, 32, 1992, 1016, True, 0, FEW), (60, 32, 1992, 896, True, 0, QUARTERS),
    # f32 in quarters of K: long K, or few tiles
    (4096, 128, 2048, 768, True, 0, QUARTERS), (4224, 128, 2048, 768, True, 0, TILES), (512, 8, 4096, 1024, True, 0, QUARTERS),
    (1000, 4, 203, 700, True, 1, QUARTERS), (2000, 4, 72, 2104, True, 0, TILES),
    # large tiles, tiles copied ahead, tiles through registers
    (1500, 2, 704, 7168, False, 0, LARGE), (1500, 2, 704, 6400, False, 0, TILES), (1500, 2, 704, 7168, False, 2, TILES),
    (1500, 2, 708, 7168, False, 0, TILES), (1000, 3, 704, 520, False, 0, COPIED), (2000, 4, 776, 2104, False, 0, TILES),
])
def test_grouped_gemm_kernel(L, rows, groups, k, n, f32, shift, kernel):
    """The kernel that the rule takes for 256 compute units."""
    import reflex_amd as rq

    if torch.cuda.is_available():
        pytest.skip("the rule for the device's own compute units")
    p = rq.RfxqGroupedPolicy()
    x = _rows(F32 if f32 else F16, rows, k + 8 - k % 8, 2 * P + (4 if f32 else 1) * shift)
    w = _weight(F16, k, n, groups)
    assert L.rfxq_grouped_gemm_policy(ctypes.byref(x), ctypes.byref(w), rows, ctypes.byref(p)) == 0
    tile = {FEW4: (16, 16), FEW: (16, 128), QUARTERS: (32, 64), LARGE: (256, 256)}.get(kernel, (64, 128))
    assert (p.kernel, (p.tile_m, p.tile_n)) == (kernel, tile)


def test_grouped_gemm_kernel_refusals(L):
    import reflex_amd as rq

    p, x, w = rq.RfxqGroupedPolicy(), _rows(), _weight()
    ask = lambda x, w, rows, out: L.rfxq_grouped_gemm_policy(  # noqa: E731
        *(None if v is None else ctypes.byref(v) for v in (x, w)), rows, None if out is None else ctypes.byref(out))
    _expect(L, ask(x, w, 8, None), 11, "NULL output")
    _expect(L, ask(None, w, 8, p), 11, "x is NULL")
    _expect(L, ask(x, None, 8, p), 11, "weight is NULL")
    _expect(L, ask(x, w, 0, p), 11, "rows=0")
    _expect(L, ask(_rows(rows=0), w, 8, p), 11, "of 0")
    _expect(L, ask(x, _weight(ty=Q4K), 8, p), 1, "F16 or BF16")


def _lora(L, x=None, a=None, b=None, y=None, out=None, offsets=9 * P, ws=None, ws_bytes=0):
    ref = lambda v: None if v is None else ctypes.byref(v)  # noqa: E731
    return L.rfxq_lora_add(ref(x), ref(a), ref(b), None, None, offsets, None, ref(y), ref(out), ws, ws_bytes, None)


@pytest.mark.parametrize("change,code,text", [
    ({"a": None}, 11, "a: weight is NULL"),
    ({"b": None}, 11, "b: weight is NULL"),
    ({"a": {"ty": Q4K}}, 1, "F32, F16 or BF16"),
    ({"b": {"ty": BF16}}, 12, "of type 30"),
    ({"b": {"k": 7}}, 12, "lora_add: a"),
    ({"b": {"e": 3}}, 12, "lora_add: a"),
    ({"x": {"rows": 9}}, 12, "9 rows of x"),
    ({"out": {"rows": 9}}, 12, "9 of out"),
    ({"x": {"ty": F32}}, 11, "x of type 0"),
    ({"x": {"ty": BF16}, "y": {"ty": BF16}, "out": {"ty": BF16}}, 11, "x of type 30"),
    ({"y": {"stride": 47}}, 12, "stride=47"),
    ({"offsets": None}, 11, "offsets is NULL"),
    ({"out": {"data": 2 * P}}, 11, "x and out overlap"),
    ({"out": {"data": 6 * P + 96}}, 11, "y and out overlap"),
    ({"out": {"data": 6 * P, "stride": 50}}, 11, "y and out overlap"),
])
def test_lora_add_refusals(L, change, code, text):
    base = {"x": dict(data=2 * P), "a": dict(n=6), "b": dict(k=6, n=48, data=4 * P), "y": dict(stride=48, data=6 * P),
            "out": dict(stride=48, data=8 * P)}
    a = {}
    for m, c in base.items():
        if m in change and change[m] is None:
            a[m] = None
        else:
            a[m] = (_weight if m in "ab" else _rows)(**{**c, **change.get(m, {})})
    if "offsets" in change:
        a["offsets"] = change["offsets"]
    _expect(L, _lora(L, **a), code, text)


def _layer(L, entry, rows=4, experts=16, top_k=2, logits=None, x=2 * P, out=8 * P, gate=None, up=None, down=None):
    logits = logits or (ctypes.c_float * (rows * experts))()
    w = [_weight(**{"k": 32, "n": 48, "e": experts, **(gate or {})}), _weight(**{"k": 32, "n": 48, "e": experts, **(up or {})}),
         _weight(**{"k": 48, "n": 32, "e": experts, **(down or {})})]
    return getattr(L, entry)(x, rows, 32, logits, experts, top_k, 1, 1.0, *map(ctypes.byref, w), out, None)


@pytest.mark.parametrize("entry", ["rfxq_moe_ffn_grouped", "rfxq_moe_ffn_grouped_device"])
@pytest.mark.parametrize("change,code,text", [
    ({"rows": 1 << 21, "top_k": 16, "logits": 3 * P}, 12, "33554432 routed pairs"),  # before any logit is read
    ({"top_k": 17}, 12, "route_top_k: k (17)"),
    ({"experts": 128, "top_k": 65}, 12, "route_top_k: k (65)"),
    ({"experts": 1025, "logits": 3 * P}, 12, "expert_count=1025"),
    ({"up": {"k": 31}}, 12, "shapes"),
    ({"up": {"e": 15}}, 12, "expert_count=16"),
    ({"down": {"length": 100}}, 12, "weight of 100 bytes"),
    ({"gate": {"data": P + 1}}, 12, "aligned"),
    ({"out": 2 * P + 64}, 11, "overlap"),
    ({"x": 2 * P + 2}, 12, "4-byte aligned"),
    ({"x": None}, 11, "NULL"),
])
def test_half_layer_refusals(L, entry, change, code, text):
    """Both entry points refuse the same layers of F16 / BF16 stacks, before any routing."""
    _expect(L, _layer(L, entry, **change), code, text)


@pytest.mark.parametrize("entry", ["rfxq_moe_ffn_grouped", "rfxq_moe_ffn_grouped_device"])
@pytest.mark.parametrize("change", [{"up": {"ty": BF16}}, {"x": 2 * P + 4}, {"down": {"length": 48 * 32 * 16 * 2 + 2}}])
def test_half_layers_of_any_half_types_and_alignment(L, entry, change):
    """What the device-routed entry takes, the host-routed one takes too: no refusal of the layer itself (none at
    rows = 0; with rows, on a machine without a GPU, the missing device is what fails)."""
    if not torch.cuda.is_available():
        rc = _layer(L, entry, **change)
        assert rc not in (0, 1, 11, 12), L.rfxq_last_error()
    assert _layer(L, entry, **{**change, "rows": 0}) == 0


def test_workspace_sizes(L):
    # a buffer for the most rows holds any fewer rows' needs
    a = _weight(k=4096, n=64, e=64)
    sizes = [L.rfxq_lora_add_workspace_size(ctypes.byref(a), r) for r in range(1, 9000, 7)]
    assert sizes == sorted(sizes) and sizes[0] > 0


def test_python_checks():
    import reflex_amd as rq

    w = rq.Weight.from_tensor(torch.zeros(3, 16, 8, dtype=torch.float16))
    assert (w.ty, w.shape, w._c.len) == (rq.GgmlType.F16, [8, 16, 3], 3 * 16 * 8 * 2)
    for bad in (torch.zeros(4, 4, dtype=torch.int32), torch.zeros(4), torch.zeros(4, 6).t()):
        with pytest.raises(rq.InvalidInputError):
            rq.Weight.from_tensor(bad)
    x, ids = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(rq.InvalidInputError, match="ids on cpu"):
        rq.group_rows(ids, 3)
    with pytest.raises(rq.InvalidInputError, match="x on cpu"):
        rq.grouped_gemm(x, w, ids, 4)
    with pytest.raises(rq.InvalidInputError, match="x on cpu"):
        rq.lora_add(x, w, w, rq.RowGroups(ids, ids), x)


def test_python_counts_do_not_wrap():
    import reflex_amd as rq

    for n in (-1, 1 << 31, 1 << 32):
        with pytest.raises(rq.InvalidInputError, match="group_rows: n="):
            rq.group_rows_workspace_size(n, 4)
        with pytest.raises(rq.InvalidInputError, match="groups="):
            rq.group_rows_workspace_size(4, n)
        with pytest.raises(rq.InvalidInputError, match="rows="):
            rq.lora_add_workspace_size(rq.Weight.from_tensor(torch.zeros(4, 8)), n)


def test_matrix_results_are_not_read_too_early(tmp_path):
    """The kernels' listing: on no path is a matrix instruction's result read before the wait states that the
    compiler itself keeps in straight code (10 behind v_mfma_f32_16x16x4_f32, 8 behind the 16x16x32 ones). It
    has left them out where the reading instruction is the first behind a branch."""
    import os
    import re
    import subprocess

    from reflex_amd import build

    listing = tmp_path / "half.s"
    flags = [f for f in build.DEVICE_FLAGS if f != "--no-gpu-bundle-output"]
    subprocess.run([os.path.join(build.ROCM, "bin", "hipcc"), *flags, "-S", os.path.join(build.CSRC, "half.hip"), "-o",
                    str(listing)], check=True, capture_output=True)
    code, labels, kernel = [], {}, None
    for line in listing.read_text().split("\n"):
        m = re.match(r"^([\w.$]+):", line)
        if m:
            labels[m.group(1)] = len(code)
            kernel = m.group(1) if m.group(1).startswith("rfxq") else kernel
            continue
        text = line.split(";")[0].strip()
        if text and not text.startswith("."):
            code.append((text, kernel))

    def registers(operand):
        found = set()
        for m in re.finditer(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)", operand):
            lo, hi = (m.group(2), m.group(3)) if m.group(2) else (m.group(4), m.group(4))
            found |= {(m.group(1), i) for i in range(int(lo), int(hi) + 1)}
        return found

    early, products = [], 0
    for i, (text, kernel) in enumerate(code):
        if not text.startswith("v_mfma"):
            continue
        products += 1
        need = 10 if "x4_f32" in text else 8
        paths, seen = [(i + 1, 0, frozenset(registers(text.split(None, 1)[1].split(", ")[0])))], set()
        while paths:
            at, waited, live = state = paths.pop()
            if waited >= need or not live or at >= len(code) or state in seen:
                continue
            seen.add(state)
            name, _, rest = code[at][0].partition(" ")
            operands = rest.split(", ")
            if name == "s_endpgm":
                continue
            if name == "s_nop":
                paths.append((at + 1, waited + int(rest, 0) + 1, live))
                continue
            if name.startswith(("s_branch", "s_cbranch")):
                paths.append((labels[rest.strip()], waited + 1, live))
                if name == "s_branch":
                    continue
            elif name.startswith(("v_", "ds_", "global_", "buffer_", "flat_")):
                writes = set() if "store" in name or "ds_write" in name else registers(operands[0])
                reads = set().union(*map(registers, operands[1:] if writes else operands))
                if name.startswith("v_mfma"):  # the next product may add to the same result
                    reads = registers(operands[1]) | registers(operands[2])
                if reads & live:
                    early.append((kernel, text, code[at][0], waited))
                live = frozenset(live - writes)
            paths.append((at + 1, waited + 1, live))
    assert products > 500 and not early, early[:5]

"""Refusals of the entry points in 8-bit floating point (rfxq_quantize_f8, rfxq_silu_and_mul_f8,
rfxq_add_rmsnorm_f8, rfxq_gemm_f8, rfxq_grouped_gemm_f8): all of them are decided on the host, before
any launch, so they run without a GPU (addresses that are never read)."""
import ctypes

import pytest
import torch

P = 1 << 20  # a plausible device address
F32, F16, BF16, Q4K = 0, 1, 30, 12
INF = float("inf")


@pytest.fixture(scope="module")
def L():
    import reflex_amd

    return reflex_amd.lib()


def _rows(ty=F16, rows=8, stride=300, data=2 * P):
    import reflex_amd as rq

    return rq.RfxqRows(data, ty, rows, stride)


def _f8(rows=8, stride=300, scale_stride=3, data=4 * P, scales=5 * P):
    import reflex_amd as rq

    return rq.RfxqF8Rows(data, scales, rows, stride, scale_stride)


def _weight(k=300, n=200, e=0, data=6 * P, scales=7 * P, length=None, scales_len=None):
    import reflex_amd as rq

    c = max(e, 1)
    return rq.RfxqF8Weight(k, n, e, data, scales, c * k * n if length is None else length,
                           4 * c * ((k + 127) // 128) * ((n + 127) // 128) if scales_len is None else scales_len)


def _ref(make, v):
    return None if v is None else ctypes.byref(make(**v))


def _expect(L, rc, code, text):
    assert rc == code and text in L.rfxq_last_error().decode(), (rc, L.rfxq_last_error())


ROWS = [
    ({"x": None}, 11, "x is NULL"),
    ({"x": {"ty": Q4K}}, 1, "of type 12"),
    ({"x": {"data": None}}, 11, "x data is NULL"),
    ({"x": {"data": 2 * P + 1}}, 12, "aligned"),
    ({"x": {"stride": 299}}, 12, "stride=299"),
    ({"x": {"rows": 7}}, 12, "7"),
    ({"x": {"rows": 1 << 31}}, 12, "rows"),
    ({"out": None}, 11, "out is NULL"),
    ({"out": {"data": None}}, 11, "data or scales is NULL"),
    ({"out": {"scales": None}}, 11, "data or scales is NULL"),
    ({"out": {"scales": 5 * P + 2}}, 12, "4-byte aligned"),
    ({"out": {"stride": 299}}, 12, "stride=299"),
    ({"out": {"scale_stride": 2}}, 12, "scale_stride=2"),
    ({"out": {"stride": 1 << 46}}, 12, "stride="),
    ({"out": {"rows": 9}}, 12, "9"),
    ({"out": {"data": 2 * P + 100}}, 11, "overlap"),
    ({"out": {"scales": 2 * P + 100}}, 11, "overlap"),
    ({"out": {"scales": 4 * P + 2000}}, 11, "overlap"),
    ({"k": 0}, 12, "k=0"),
    ({"k": 1 << 31}, 12, "k="),
]


@pytest.mark.parametrize("change,code,text", ROWS)
def test_quantize_refusals(L, change, code, text):
    a = {"x": {}, "out": {}, "k": 300, **change}
    _expect(L, L.rfxq_quantize_f8(_ref(_rows, a["x"]), a["k"], _ref(_f8, a["out"]), None), code, text)


@pytest.mark.parametrize("change,code,text", [(c, code, "gate is NULL" if text == "x is NULL" else
                                               "gate data is NULL" if text == "x data is NULL" else text)
                                              for c, code, text in ROWS] + [
    ({"up": None}, 11, "up is NULL"),
    ({"up": {"ty": F32}}, 11, "gate of type 1, up 0"),
    ({"up": {"rows": 9}}, 12, "9 of up"),
    ({"up": {"stride": 200}}, 12, "stride=200"),
    ({"up": {"data": 4 * P}}, 11, "overlap"),
])
def test_silu_refusals(L, change, code, text):
    a = {"x": {}, "up": {"data": 3 * P}, "out": {}, "k": 300, **change}
    if a["up"] is not None:
        a["up"] = {"data": 3 * P, **a["up"]}
    _expect(L, L.rfxq_silu_and_mul_f8(_ref(_rows, a["x"]), _ref(_rows, a["up"]), a["k"], _ref(_f8, a["out"]), None), code,
            text)


@pytest.mark.parametrize("change,code,text", ROWS + [
    ({"residual": {"ty": F32}}, 11, "types 1 and 0"),
    ({"residual": {"rows": 5}}, 12, "8 and 5 rows"),
    ({"residual": {"data": 4 * P}}, 11, "overlap"),
    ({"sum": {"ty": BF16}}, 11, "types 1 and 30"),
    ({"sum": {"stride": 1}}, 12, "stride=1"),
    ({"sum": {"data": 2 * P + 64}}, 11, "x and sum overlap"),
    ({"sum": {"data": 2 * P, "stride": 400}}, 11, "x and sum overlap"),
    ({"sum": {"data": 3 * P + 2}}, 11, "residual and sum overlap"),
    ({"sum": {"data": 4 * P}}, 11, "out and sum overlap"),
    ({"sum": {"data": 10 * P}}, 11, "weight and sum overlap"),
    ({"y": {"data": 2 * P}}, 11, "x and y overlap"),
    ({"y": {"data": 9 * P}}, 11, "sum and y overlap"),
    ({"y": {"ty": F32}}, 11, "types 1 and 0"),
    ({"weight": None}, 11, "weight is NULL"),
    ({"weight": 10 * P + 2}, 11, "weight is NULL or not 4-byte aligned"),
    ({"eps": -1e-6}, 11, "eps="),
    ({"eps": INF}, 11, "eps="),
    ({"eps": float("nan")}, 11, "eps="),
])
def test_norm_refusals(L, change, code, text):
    a = {"x": {}, "residual": {}, "sum": {}, "y": None, "out": {}, "k": 300, "weight": 10 * P, "eps": 1e-6, **change}
    a["residual"] = {"data": 3 * P, **a["residual"]}
    a["sum"] = {"data": 9 * P, **a["sum"]}
    _expect(L, L.rfxq_add_rmsnorm_f8(_ref(_rows, a["x"]), _ref(_rows, a["residual"]), a["weight"], a["k"], a["eps"],
                                     _ref(_rows, a["sum"]), _ref(_f8, a["out"]), _ref(_rows, a["y"]), None), code, text)


PRODUCT = [
    ({"w": None}, 11, "weight is NULL"),
    ({"w": {"k": 0}}, 12, "shape"),
    ({"w": {"n": 0}}, 12, "shape"),
    ({"w": {"n": 1 << 31, "length": 1 << 62}}, 12, "shape"),
    ({"w": {"length": 300 * 200 - 1}}, 12, "needs"),
    ({"w": {"scales_len": 4 * 6 - 1}}, 12, "needs"),
    ({"w": {"data": None}}, 11, "data or scales is NULL"),
    ({"w": {"scales": None}}, 11, "data or scales is NULL"),
    ({"w": {"scales": 7 * P + 1}}, 12, "aligned"),
    ({"w": {"e": 1025}}, 12, "expert_count=1025"),
    ({"x": None}, 11, "x is NULL"),
    ({"x": {"data": None}}, 11, "NULL"),
    ({"x": {"scales": None}}, 11, "NULL"),
    ({"x": {"stride": 299}}, 12, "stride=299"),
    ({"x": {"scale_stride": 2}}, 12, "scale_stride=2"),
    ({"x": {"scales": 5 * P + 1}}, 12, "aligned"),
    ({"y": None}, 11, "y is NULL"),
    ({"y": {"ty": Q4K}}, 1, "of type 12"),
    ({"y": {"stride": 199}}, 12, "stride=199"),
    ({"y": {"data": 2 * P + 1}}, 12, "aligned"),
    ({"y": {"data": 4 * P + 128}}, 11, "x and y overlap"),
    ({"y": {"data": 5 * P + 8}}, 11, "x's scales and y overlap"),
    ({"y": {"data": 6 * P + 16}}, 11, "weight and y overlap"),
    ({"y": {"data": 7 * P - 16}}, 11, "weight's scales and y overlap"),
]


@pytest.mark.parametrize("change,code,text", PRODUCT + [
    ({"w": {"e": 2}}, 12, "stack of 2"),
    ({"y": {"rows": 9}}, 12, "8 rows of x, 9 of y"),
])
def test_gemm_refusals(L, change, code, text):
    a = {"x": {}, "w": {}, "y": {}, **change}
    _expect(L, L.rfxq_gemm_f8(_ref(_f8, a["x"]), _ref(_weight, a["w"]), _ref(_rows, a["y"]), None), code, text)


def _grouped(L, x={}, w={}, offsets=8 * P, rows=8, x_index=None, x_div=1, y_index=None, y={}):
    return L.rfxq_grouped_gemm_f8(_ref(_f8, x), _ref(_weight, w), offsets, rows, x_index, x_div, y_index, _ref(_rows, y), None)


@pytest.mark.parametrize("change,code,text", PRODUCT + [
    ({"rows": 1 << 31}, 12, "rows="),
    ({"x_div": 0}, 11, "x_div=0"),
    ({"x_div": 2}, 11, "x_div=2 without x_index"),
    ({"offsets": None}, 11, "offsets is NULL"),
])
def test_grouped_refusals(L, change, code, text):
    if isinstance(change.get("w"), dict) and "e" not in change["w"] and change["w"].get("length") is None:
        change = {**change, "w": {"e": 1, **change["w"]}}
    _expect(L, _grouped(L, **change), code, text)


@pytest.mark.parametrize("change,code,text", PRODUCT + [({"w": {"e": 2}}, 12, "stack of 2"), ({"y": {"rows": 9}}, 12, "9 of y")])
def test_exact_refusals(L, change, code, text):
    """The exact forms refuse what the others do."""
    a = {"x": {}, "w": {}, "y": {}, **change}
    _expect(L, L.rfxq_gemm_f8_exact(_ref(_f8, a["x"]), _ref(_weight, a["w"]), _ref(_rows, a["y"]), None), code, text)
    assert L.rfxq_last_error().decode().startswith("gemm_f8_exact: ")
    if "e" in (a["w"] or {}) or "rows" in (a["y"] or {}):
        return
    rc = L.rfxq_grouped_gemm_f8_exact(_ref(_f8, a["x"]), _ref(_weight, a["w"]), 8 * P, 8, None, 1, None, _ref(_rows, a["y"]), None)
    _expect(L, rc, code, text)
    assert L.rfxq_last_error().decode().startswith("grouped_gemm_f8_exact: ")


@pytest.mark.parametrize("empty", [{"rows": 0}, {"x": {"rows": 0, "data": None, "scales": None}},
                                   {"y": {"rows": 0, "data": None}}])
def test_products_of_nothing(L, empty):
    assert _grouped(L, **empty) == 0
    if "rows" not in empty:
        both = {"x": {"rows": 0, "data": None}, "y": {"rows": 0, "data": None}}
        assert L.rfxq_gemm_f8(_ref(_f8, both["x"]), _ref(_weight, {}), _ref(_rows, both["y"]), None) == 0


def test_rows_of_nothing(L):
    x, out = _ref(_rows, {"rows": 0, "data": None}), _ref(_f8, {"rows": 0, "data": None})
    assert L.rfxq_quantize_f8(x, 300, out, None) == 0
    assert L.rfxq_silu_and_mul_f8(x, x, 300, out, None) == 0
    assert L.rfxq_add_rmsnorm_f8(x, None, None, 300, 1e-6, None, out, None, None) == 0


def test_policy_refusals(L):
    import reflex_amd as rq

    p = rq.RfxqF8Policy()
    x, w = _ref(_f8, {}), _ref(_weight, {})
    _expect(L, L.rfxq_gemm_f8_policy(x, w, 8, 0, F32, None), 11, "NULL output")
    _expect(L, L.rfxq_gemm_f8_policy(x, None, 8, 0, F32, ctypes.byref(p)), 11, "weight is NULL")
    _expect(L, L.rfxq_gemm_f8_policy(None, w, 8, 0, F32, ctypes.byref(p)), 11, "x is NULL")
    _expect(L, L.rfxq_gemm_f8_policy(x, w, 0, 0, F32, ctypes.byref(p)), 11, "rows=0")
    _expect(L, L.rfxq_gemm_f8_policy(x, w, 8, 0, Q4K, ctypes.byref(p)), 1, "of type 12")
    assert L.rfxq_gemm_f8_policy(x, w, 8, 1, F16, ctypes.byref(p)) == 0


ANY, FEW, STREAM, COPIED, LARGE = range(5)


@pytest.mark.parametrize("rows,experts,k,n,ty,shift,kernel", [
    (1, 0, 4096, 1024, F32, 0, (STREAM, 16, 16)),
    (1, 0, 4096, 14336, BF16, 0, (STREAM, 16, 32)),
    (32, 0, 4096, 4096, F32, 0, (STREAM, 16, 32)),
    (64, 0, 14336, 4096, F16, 0, (STREAM, 32, 32)),
    (256, 128, 768, 2048, F32, 0, (STREAM, 16, 64)),
    (512, 0, 14336, 4096, BF16, 0, (COPIED, 64, 128)),
    (512, 0, 14336, 4096, F32, 0, (COPIED, 64, 128)),
    (1000, 0, 4096, 4096, F16, 0, (COPIED, 128, 128)),
    (4096, 0, 4096, 14336, F32, 0, (COPIED, 128, 128)),
    (2048, 0, 4096, 4096, BF16, 0, (LARGE, 128, 256)),
    (4096, 0, 4096, 14336, BF16, 0, (LARGE, 256, 256)),
    (4096, 0, 4096, 14336, BF16, 8, (ANY, 64, 128)),      # rows at 8 bytes
    (4096, 0, 4104, 14336, F32, 0, (ANY, 64, 128)),       # K not a multiple of 16
    (1, 0, 4096, 4096, F32, 1, (FEW, 16, 16)),
    (333, 0, 1235, 1531, F32, 0, (ANY, 32, 64)),
    (333, 0, 4099, 4099, F32, 0, (ANY, 64, 128)),
    (16, 0, 4099, 14336, BF16, 0, (ANY, 32, 64)),
    (1200, 128, 200, 512, F16, 0, (ANY, 64, 128)),
    (128, 128, 1235, 1000, F32, 0, (ANY, 32, 64)),
    (4, 0, 65536, 65536, BF16, 0, (ANY, 64, 128)),        # a matrix of 4 GiB
    (1, 0, 65520, 65552, BF16, 0, (STREAM, 16, 32)),      # a little less
])
def test_product_kernel(L, rows, experts, k, n, ty, shift, kernel):
    import reflex_amd as rq

    x = rq.RfxqF8Rows(4 * P + shift, 64 * P, rows, (k + 15) // 16 * 16, (k + 127) // 128)
    w = _weight(k, n, experts, data=1 << 30, scales=1 << 40)
    p = rq.RfxqF8Policy()
    assert L.rfxq_gemm_f8_policy(ctypes.byref(x), ctypes.byref(w), rows, 1 if experts else 0, ty, ctypes.byref(p)) == 0
    assert (p.kernel, p.tile_m, p.tile_n) == kernel


@pytest.mark.parametrize("rows,experts,k,n,ty", [
    (4096, 0, 4096, 14336, BF16), (32768, 128, 2048, 768, BF16), (1 << 26, 0, 17, 5, F32), ((1 << 27) + 12345, 0, 17, 5, F16),
    (1 << 28, 0, 16, 16, F32), ((1 << 31) - 1, 0, 1, 1, F32), (1, 0, 17, (1 << 27) + 77, F32), (1, 0, 1, (1 << 31) - 1, BF16),
    ((1 << 27) + 999, 3, 17, 5, F16), (1 << 26, 0, 16, 1 << 20, BF16), (1 << 30, 1000, 3, 1 << 20, F32)])
def test_launches_have_fewer_than_2_32_threads(L, rows, experts, k, n, ty):
    """Products of any sizes are as many launches as that takes: one where it can be, few more than the threads need
    (each launch at least a quarter full, tiles of 8 XCDs' blocks left empty at the ends)."""
    import reflex_amd as rq

    x = rq.RfxqF8Rows(1 << 44, 1 << 45, rows, k, -(-k // 128))
    w = _weight(k, n, experts, data=1 << 43, scales=1 << 42)
    p, how = rq.RfxqF8Policy(), rq.RfxqF8Launch()
    args = ctypes.byref(x), ctypes.byref(w), rows, 1 if experts else 0, ty
    assert L.rfxq_gemm_f8_policy(*args, ctypes.byref(p)) == 0 and L.rfxq_gemm_f8_launch(*args, ctypes.byref(how)) == 0
    assert how.threads in (256, 512)
    threads = -(-rows // p.tile_m) * -(-n // p.tile_n) * how.threads
    if threads < 1 << 31:
        assert how.launches == 1
    assert threads / ((1 << 32) - 1) <= how.launches <= max(1, threads / (1 << 29))
    _expect(L, L.rfxq_gemm_f8_launch(*args, None), 11, "NULL output")
    _expect(L, L.rfxq_gemm_f8_launch(args[0], args[1], 0, args[3], ty, ctypes.byref(how)), 11, "rows=0")


def test_python_checks():
    import reflex_amd as rq

    f8 = torch.float8_e4m3fn
    codes, scales = torch.zeros(4, 300, dtype=f8), torch.zeros(4, 3)
    bad = rq.InvalidInputError
    with pytest.raises(bad, match="codes"):
        rq.F8Weight(torch.zeros(4, 300), scales)
    with pytest.raises(bad, match="codes"):
        rq.F8Weight(codes[:, ::2], scales)
    with pytest.raises(bad, match="codes"):
        rq.F8Weight(codes[0], scales)
    with pytest.raises(bad, match="scales"):
        rq.F8Weight(codes, scales)
    with pytest.raises(bad, match="scales"):
        rq.F8Weight(codes, torch.zeros(1, 3, dtype=torch.float16))
    with pytest.raises(bad, match="shape=0"):
        rq.F8Weight(torch.zeros(0, 300, dtype=f8), torch.zeros(0, 3))
    with pytest.raises(bad, match="count=0"):
        rq.F8Weight(torch.zeros(0, 4, 300, dtype=f8), torch.zeros(0, 1, 3))
    w = rq.F8Weight(codes, torch.zeros(1, 3))
    assert (w.in_features, w.out_features, w.count) == (300, 4, 0)
    assert rq.F8Weight(torch.zeros(2, 4, 300, dtype=torch.uint8), torch.zeros(2, 1, 3)).count == 2
    # rows on the CPU
    for call in (lambda: rq.quantize_f8(torch.zeros(4, 300)), lambda: rq.silu_and_mul_f8(torch.zeros(4, 3), torch.zeros(4, 3)),
                 lambda: rq.add_rmsnorm_f8(torch.zeros(4, 3), None, torch.zeros(3), 1e-6),
                 lambda: rq.gemm_f8(rq.F8Rows(codes, scales), w),
                 lambda: rq.grouped_gemm_f8(rq.F8Rows(codes, scales), w, torch.zeros(2, dtype=torch.int32), 4)):
        with pytest.raises(bad, match="on cpu"):
            call()
    for args, text in (((torch.zeros(4, 300), scales), "codes"), ((codes[0], scales), "codes"), ((codes[:, :0], scales), "codes"),
                       ((codes, scales[:3]), "scales"), ((codes, scales.double()), "scales"), ((codes, scales[:, :2]), "scales"),
                       ((codes.t(), torch.zeros(300, 1)), "strides"), ((codes[:1].expand(4, 300), scales), "strides")):
        with pytest.raises(bad, match=text):
            rq.F8Rows(*args)
    rows = rq.F8Rows(codes, scales)
    with pytest.raises(AttributeError):
        rows.codes = codes
    empty = rq.F8Rows.empty(3, 129, "cpu")
    assert empty.codes.shape == (3, 129) and empty.scales.shape == (3, 2)


def test_weights_keep_what_they_were_made_of():
    """Calls read the memory that a weight was made with: another tensor put in its place would not be read."""
    import reflex_amd as rq

    codes, scales = torch.zeros(2, 4, 300, dtype=torch.uint8), torch.zeros(2, 1, 3)
    w = rq.F8Weight(codes, scales)
    assert w.codes is codes and w.scales is scales
    for name, value in (("codes", codes.clone()), ("scales", scales.clone()), ("count", 1), ("out_features", 2),
                        ("in_features", 2), ("anything", 0)):
        with pytest.raises(AttributeError):
            setattr(w, name, value)
    assert (w._c.data, w._c.scales) == (codes.data_ptr(), scales.data_ptr())
    assert (w.count, w.out_features, w.in_features) == (2, 4, 300)


def test_matrix_results_are_not_read_too_early(tmp_path):
    """The kernels' listing: on no path is a matrix instruction's result read before the wait states that the
    compiler itself keeps in straight code (12 behind the 16x16x128 ones on e4m3, 8 behind the 16x16x32 ones). It
    has left them out where the reading instruction is the first behind a branch."""
    import os
    import re
    import subprocess

    from reflex_amd import build

    listing = tmp_path / "f8.s"
    flags = [f for f in build.DEVICE_FLAGS if f != "--no-gpu-bundle-output"]
    subprocess.run([os.path.join(build.ROCM, "bin", "hipcc"), *flags, "-S", os.path.join(build.CSRC, "f8.hip"), "-o",
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

    early, products = [], {"f8f6f4": 0, "32_f16": 0}
    for i, (text, kernel) in enumerate(code):
        if not text.startswith("v_mfma"):
            continue
        kind = "f8f6f4" if "16x16x128_f8f6f4" in text else "32_f16" if "16x16x32_f16" in text else None
        assert kind, text
        products[kind] += 1
        need = 12 if kind == "f8f6f4" else 8
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
            elif name.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")):
                writes = set() if "store" in name or "ds_write" in name else registers(operands[0])
                reads = set().union(*map(registers, operands[1:] if writes else operands))
                if name.startswith("v_mfma"):  # the next product may add to the same result
                    reads = registers(operands[1]) | registers(operands[2])
                if reads & live:
                    early.append((kernel, text, code[at][0], waited))
                live = frozenset(live - writes)
            paths.append((at + 1, waited + 1, live))
    assert products["f8f6f4"] > 500 and products["32_f16"] > 200 and not early, (products, early[:5])
    # copies that the compiler does not count: nothing that it does count may be spilled beside them
    assert "Folded" not in listing.read_text()


def test_registers_that_inline_assembly_writes_are_declared():
    """The compiler may keep a copy's LDS address in m0 across inline assembly that does not say that it writes there."""
    import glob
    import os
    import re

    from reflex_amd import build

    found = 0
    for path in sorted(glob.glob(os.path.join(build.CSRC, "*.h*"))):
        for text in re.findall(r"asm volatile\((.*?)\);", open(path).read(), re.S):
            if re.search(r"s_mov_b32 (m0|vcc|exec)", text):
                found += 1
                register = re.search(r"s_mov_b32 (m0|vcc|exec)", text).group(1)
                assert f'"{register}"' in text.rsplit(":", 1)[1], (path, text)
    assert found

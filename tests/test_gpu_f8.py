"""8-bit floating point (rfxq_quantize_f8, rfxq_silu_and_mul_f8, rfxq_add_rmsnorm_f8, rfxq_gemm_f8,
rfxq_grouped_gemm_f8) against their definitions in 64 bits on the CPU.

Bounds. A code is its quotient rounded to e4m3: off by at most half a step, 2^-4 of the power of two below it, 2^-10
below 2^-6. The quotient is a f32 value times 1 / scale, each within 2^-22; a scale is amax / 448 within 2^-22. The
values themselves: SiLU's five f32 operations within 2^-20; the norm's squares are added in chains of at most
K / 128 + 64, each addition within 2^-24 of the sum, half of that in the square root, and a few roundings more:
(K / 128 + 80) 2^-24. A product: each block's sum and the sum over blocks in f32, at most K / 128 + 32 additions in a
row, each within 2^-23 of the sum of the products' sizes (scales included); the result rounded once, eps / 2 of its
value. Where the result is f16 or bf16 the matrix instructions may add eight neighbouring products cut to multiples of
2^-13 2^e, e the largest sum of two codes' exponents there (at least -6 each): eight products, 2^-10 2^e, and e is at
most the sum of the largest exponents of either side."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
F8 = torch.float8_e4m3fn
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}
LEAST = 2.0 ** -120


def _say(*what):
    print(*what, flush=True)


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _strided(values, stride, shift, fill):
    """values [rows, columns] on the GPU with rows `stride` elements apart, `shift` elements into a buffer of `fill`;
    and that buffer."""
    rows, columns = values.shape
    buf = torch.empty(shift + max(rows, 1) * stride + 64, dtype=values.dtype, device=DEV)
    buf.view(torch.uint8).fill_(fill)
    view = buf[shift:shift + rows * stride].view(rows, stride)[:, :columns]
    view.copy_(values.to(DEV))
    return view, buf


# ------------------------------------------------------------------ rows in 8 bits

def _blocks(k):
    return (k + 127) // 128


def _check_codes(codes, scales, v, rel):
    """Codes and scales [rows, ..] of values v (64 bits, CPU), each of which is known within rel of its size."""
    codes, scales = codes.cpu().float().double(), scales.cpu().double()
    rows, k = v.shape
    for b in range(_blocks(k)):
        part, s = v[:, 128 * b:128 * b + 128], scales[:, b]
        c = codes[:, 128 * b:128 * b + 128]
        fine = torch.isfinite(part).all(1)
        assert torch.isnan(s[~fine]).all()
        part, s, c = part[fine], s[fine], c[fine]
        if not part.numel():
            continue
        want = part.abs().amax(1).clamp(min=448.0 * LEAST) / 448.0
        assert ((s - want).abs() <= want * (2.0 ** -22 + rel)).all(), (b, s, want)
        quotient = part / s[:, None]
        e = torch.floor(torch.log2(quotient.abs().clamp(min=2.0 ** -30)))
        half = torch.exp2(e.clamp(min=-6.0) - 4.0)
        off = (c - quotient).abs()
        assert (off <= half * (1 + 2.0 ** -20) + quotient.abs() * (rel + 2.0 ** -21)).all(), (b, off.max())


def _values(rows, k, dtype, seed, spread=2.0):
    g = _gen(seed)
    v = torch.randn(rows, k, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
    v[torch.rand(rows, k, generator=g) < 0.05] = 0.0
    return v.to(dtype)


SIZES = [(1, 1), (1, 128), (2, 7), (3, 127), (5, 129), (1, 4096), (33, 256), (64, 1000), (7, 2048), (130, 768), (9, 1235),
         (2, 8200), (3, 14336), (300, 511), (1, 40000), (2, 33000)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k", SIZES)
def test_quantize(rq, rows, k, dtype):
    _say("quantize", rows, k, dtype)
    x = _values(rows, k, dtype, rows + k)
    got = rq.quantize_f8(x.to(DEV))
    assert got.codes.dtype == F8 and got.codes.shape == (rows, k) and got.scales.shape == (rows, _blocks(k))
    _check_codes(got.codes, got.scales, x.double(), 0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k", SIZES)
def test_silu(rq, rows, k, dtype):
    _say("silu", rows, k, dtype)
    gate, up = _values(rows, k, dtype, rows + k, 1.0), _values(rows, k, dtype, rows + k + 1, 1.0)
    both = torch.cat([gate, up], 1).to(DEV)
    got = rq.silu_and_mul_f8(both[:, :k], both[:, k:])
    g = gate.double()
    _check_codes(got.codes, got.scales, g * torch.sigmoid(g) * up.double(), 2.0 ** -20)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,k", SIZES)
def test_norm(rq, rows, k, residual, dtype):
    _say("norm", rows, k, residual, dtype)
    x = _values(rows, k, dtype, rows + k)
    r = _values(rows, k, dtype, rows + k + 1) if residual else None
    w = 1.0 + 0.3 * torch.randn(k, generator=_gen(k))
    out, total, y = rq.add_rmsnorm_f8(x.to(DEV), r.to(DEV) if residual else None, w.to(DEV), 1e-5, want_y=True)
    assert (total is None) == (not residual)
    _check_norm(x, r, w, 1e-5, out, total, y)


def _check_norm(x, r, w, eps, out, total, y):
    k, dtype = x.shape[1], x.dtype
    t = x.double() + (0 if r is None else r.double())
    if total is not None:
        half = torch.finfo(dtype).eps / 2
        assert ((total.cpu().double() - t).abs() <= t.abs() * (half + 2.0 ** -24) + TINY[dtype]).all()
    v = t / torch.sqrt(t.square().mean(1, keepdim=True) + eps) * w.double()
    rel = (k / 128 + 80) * 2.0 ** -24
    _check_codes(out.codes, out.scales, v, rel)
    if y is not None:
        assert ((y.cpu().double() - v).abs() <= v.abs() * (torch.finfo(dtype).eps / 2 + rel) + TINY[dtype]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 1), (3, 5), (8, 64), (0, 3)])
@pytest.mark.parametrize("k", [128, 333, 1024, 33001])
def test_rows_of_any_stride(rq, k, shift, pad, dtype):
    """Strides, alignment, and that nothing else is written."""
    _say("strides", k, shift, pad, dtype)
    rows = 5
    x, r = _values(rows, k, dtype, k), _values(rows, k, dtype, k + 1)
    w = torch.rand(k, generator=_gen(1)) + 0.5
    xd, _ = _strided(x, k + pad, shift, 0x7F)
    rd, _ = _strided(r, k + 2 * pad, shift + 1, 0x7F)

    def outputs():
        codes, cbuf = _strided(torch.zeros(rows, k, dtype=torch.uint8), k + pad, shift, 0xA5)
        scales, sbuf = _strided(torch.zeros(rows, _blocks(k)), _blocks(k) + pad, shift, 0xA5)
        return rq.F8Rows(codes, scales), cbuf, sbuf

    def untouched(view, buf):
        buf = buf.clone()
        n, step = view.shape[0], view.stride(0)
        off = view.storage_offset()
        buf[off:off + n * step].view(n, step)[:, :view.shape[1]].view(torch.uint8 if buf.dtype == torch.uint8 else buf.dtype).fill_(0)
        raw = torch.empty_like(buf)
        raw.view(torch.uint8).fill_(0xA5)
        raw[off:off + n * step].view(n, step)[:, :view.shape[1]].fill_(0)
        assert torch.equal(buf.view(torch.uint8), raw.view(torch.uint8))

    def check(o, cbuf, sbuf, v, rel):
        _check_codes(o.codes.view(F8) if o.codes.is_contiguous() else o.codes.contiguous().view(F8), o.scales, v, rel)
        untouched(o.codes, cbuf)
        untouched(o.scales, sbuf)

    o, cbuf, sbuf = outputs()
    rq.quantize_f8(xd, out=o)
    check(o, cbuf, sbuf, x.double(), 0.0)
    o, cbuf, sbuf = outputs()
    rq.silu_and_mul_f8(xd, rd, out=o)
    check(o, cbuf, sbuf, x.double() * torch.sigmoid(x.double()) * r.double(), 2.0 ** -20)
    o, cbuf, sbuf = outputs()
    total, tbuf = _strided(torch.zeros(rows, k, dtype=dtype), k + pad, shift, 0xA5)
    _, same, _ = rq.add_rmsnorm_f8(xd, rd, w.to(DEV), 1e-6, sum_out=total, out=o)
    assert same is total
    total = total.clone()
    _check_norm(x, r, w, 1e-6, rq.F8Rows(o.codes.contiguous().view(F8), o.scales), total, None)
    untouched(o.codes, cbuf)
    untouched(o.scales, sbuf)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("k", [100, 1024, 9000, 40000])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_norm_in_place(rq, k, into, dtype):
    x, r = _values(6, k, dtype, k), _values(6, k, dtype, k + 1)
    w = torch.rand(k, generator=_gen(1)) + 0.5
    xd, rd = x.to(DEV), r.to(DEV)
    out, total, _ = rq.add_rmsnorm_f8(xd, rd, w.to(DEV), 1e-6, sum_out=xd if into == "x" else rd)
    _check_norm(x, r, w, 1e-6, out, total, None)
    kept, had = (rd, r) if into == "x" else (xd, x)
    assert torch.equal(kept.cpu(), had)


def test_groups_of_every_size(rq):
    """Zeros, the smallest and the largest values, and what is not finite: each group by itself."""
    inf, nan, top = float("inf"), float("nan"), torch.finfo(F32).max
    rows = [torch.zeros(128), torch.full((128,), -0.0), torch.full((128,), 2.0 ** -149), torch.full((128,), 448 * LEAST),
            torch.full((128,), 447 * LEAST), torch.linspace(-1, 1, 128) * 2.0 ** -126, torch.linspace(-top, top, 128),
            torch.linspace(-3, 5, 128)]
    for bad in (inf, -inf, nan):
        for at in (0, 77, 127):
            v = torch.linspace(-1, 1, 128)
            v[at] = bad
            rows.append(v)
    rows.append(torch.full((128,), nan))
    # one long row of all groups, so that each has neighbours of the others
    x = torch.stack(rows)
    for shape in (x, x.reshape(1, -1), torch.nn.functional.pad(x, (0, 1))):
        got = rq.quantize_f8(shape.to(DEV))
        _check_codes(got.codes, got.scales, shape.double(), 0.0)
    got = rq.quantize_f8(x.to(DEV))
    assert (got.scales[:5].cpu().double() == LEAST).all() or (got.scales[:5].cpu().double() <= LEAST * (1 + 2.0 ** -22)).all()
    assert (got.codes[:3].cpu().float() == 0).all()


def _quantized(x):
    """Codes and scales of [rows, k] values by f32's 1 / 448 and f32 divisions, on the CPU; scale NaN where a group is not
    finite."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, _blocks(k) * 128 - k)).view(rows, _blocks(k), 128).numpy()
    with np.errstate(invalid="ignore"):
        scales = np.maximum(np.abs(v).max(2) * (np.float32(1) / np.float32(448)), np.float32(LEAST))
        codes = torch.from_numpy(v / scales[:, :, None]).to(F8).view(torch.uint8).view(rows, -1)[:, :k]
    return codes, torch.from_numpy(np.where(np.isfinite(scales), scales, np.float32("nan")))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k", [(1, 4096), (777, 1235), (400, 2048), (3, 129)])
def test_quantize_by_division(rq, rows, k, dtype):
    """Scales and codes to the last bit, ties included (8-bit values meet many): what torch makes of the same formula."""
    _say("by division", rows, k, dtype)
    g = _gen(rows + k)
    whole = torch.randint(-448, 449, (rows, k), generator=g).float() * torch.exp2(torch.randint(-5, 3, (rows, 1), generator=g))
    for x in (_values(rows, k, dtype, rows, 1.0), whole.to(dtype)):
        codes, scales = _quantized(x)
        got = rq.quantize_f8(x.to(DEV))
        assert torch.equal(got.scales.cpu(), scales)
        assert torch.equal(got.codes.view(torch.uint8).cpu(), codes)
        v = torch.nn.functional.pad(x.to(DEV).float(), (0, _blocks(k) * 128 - k)).view(rows, -1, 128)
        scales = v.abs().amax(2).clamp(min=448.0 * LEAST) / 448.0
        assert torch.equal(got.scales, scales)
        assert torch.equal(got.codes.float(), (v / scales.unsqueeze(2)).to(F8).float().view(rows, -1)[:, :k])


@pytest.mark.parametrize("dtype,bits,exponent", [(BF16, 7, -60), (BF16, 7, 0), (BF16, 7, 104), (BF16, 7, 127), (F16, 10, 0), (F16, 10, 13)])
def test_quantize_every_half_value(rq, dtype, bits, exponent):
    """Every pair of a largest value's fraction and another's, down to where codes are 0, to the last bit."""
    _say("every", dtype, exponent)
    low = max(exponent - 19, -14 if dtype == F16 else -126)
    step = 2.0 ** -bits
    fractions = 1 + torch.arange(1 << bits, dtype=torch.float64) * step
    others = torch.cat([fractions * 2.0 ** e for e in range(low, exponent + 1)])
    others = torch.nn.functional.pad(others, (0, -len(others) % 127)).view(-1, 127)
    for part in fractions.split(128):
        top = (part * 2.0 ** exponent).view(-1, 1, 1).expand(-1, others.shape[0], 1)
        x = torch.cat([top, torch.minimum(others.expand(len(part), -1, -1), top)], 2).reshape(-1, 128).to(dtype).to(DEV)
        x = torch.where(torch.arange(128, device=DEV) % 3 == 0, -x, x)
        got = rq.quantize_f8(x)
        scales = x.float().abs().amax(1, keepdim=True).clamp(min=448.0 * LEAST) / 448.0
        assert torch.equal(got.scales, scales)
        assert torch.equal(got.codes.view(torch.uint8), (x.float() / scales).to(F8).view(torch.uint8))


@pytest.mark.parametrize("exponent", [-120, -119, -70, 0, 60, 95, 96, 97, 110])
def test_quantize_next_to_ties(rq, exponent):
    """Values within some steps of a midpoint of two codes, scales within some steps of eighths of a power of two and
    anywhere: the codes of f32 quotients, which are rounded twice."""
    _say("ties", exponent)
    r = np.random.default_rng(exponent + 200)
    groups = 12000
    near = 0x100000 * r.integers(0, 8, groups) + r.integers(-130, 131, groups)
    s = np.where(r.random(groups) < 0.8, near % (1 << 23), r.integers(0, 1 << 23, groups)).astype(np.uint32)
    s = (s + np.uint32((127 + exponent) << 23)).view(np.float32)
    x = np.empty((groups, 128), np.float32)
    x[:, 0] = (s.astype(np.float64) * 448).astype(np.float32)
    s = x[:, 0] * (np.float32(1) / np.float32(448))
    tie = r.integers(16, 32, (groups, 127)) * np.exp2(r.integers(-10, 5, (groups, 127)))  # 1/64 .. 496
    tie = np.where(r.random(tie.shape) < 0.1, r.integers(0, 17, tie.shape) * 2.0 ** -10, np.minimum(tie, 432))
    v = (tie * s[:, None].astype(np.float64)).astype(np.float32)
    v = (v.view(np.int32) + np.where(v > 0, r.integers(-3, 4, v.shape), 0).astype(np.int32)).view(np.float32)
    x[:, 1:] = np.where(r.random(v.shape) < 0.5, v, -v)
    x = torch.from_numpy(x)
    codes, scales = _quantized(x)
    got = rq.quantize_f8(x.to(DEV))
    assert torch.equal(got.scales.cpu(), scales)
    wrong = got.codes.view(torch.uint8).cpu() != codes
    assert not wrong.any(), (int(wrong.sum()), wrong.nonzero()[:5].tolist())


@pytest.mark.parametrize("k", [128, 1000, 9000, 33001])
def test_norm_is_quantized_like_rows(rq, k):
    """The norm's codes and scales are those of its f32 result."""
    x = _values(20, k, F32, k, 1.0)
    out, _, y = rq.add_rmsnorm_f8(x.to(DEV), None, torch.rand(k, generator=_gen(1)).to(DEV), 1e-6, want_y=True)
    codes, scales = _quantized(y.cpu())
    assert torch.equal(out.scales.cpu(), scales) and torch.equal(out.codes.view(torch.uint8).cpu(), codes)


def test_silu_at_the_ends(rq):
    """Gates from -inf to inf; below -87 the result is 0."""
    gate = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20.0, -20.0, 80.0, -80.0, -86.0, 1e4, 3e38, 1.0, -1.0, 0.5, -40.0, 60.0])
    up = torch.tensor([1.0, -2.0, 3.0, 0.5, -1.0, 7.0, 1e-3, 1e30, 1e20, 1.0, 1.0, 0.0, 1e-30, -4.0, 1.0, 1.0])
    for g, u in zip(gate, up):  # each in a group of its own
        got = rq.silu_and_mul_f8(g.view(1, 1).to(DEV), u.view(1, 1).to(DEV))
        v = g.double() * torch.sigmoid(g.double()) * u.double()
        _check_codes(got.codes, got.scales, v.view(1, 1), 2.0 ** -20)
    for g, u in ((-100.0, 1.0), (-3e38, 5.0)):
        got = rq.silu_and_mul_f8(torch.full((1, 3), g, device=DEV), torch.full((1, 3), u, device=DEV))
        assert (got.codes.float() == 0).all() and torch.isfinite(got.scales).all()
    for g, u in ((float("inf"), 1.0), (float("nan"), 1.0), (1.0, float("nan")), (3e38, 3e38), (-float("inf"), 1.0)):
        got = rq.silu_and_mul_f8(torch.full((1, 3), g, device=DEV), torch.full((1, 3), u, device=DEV))
        assert torch.isnan(got.scales).all()


def test_silu_of_far_gates(rq):
    """Gates whose exp(gate) is below f32's normal range, beside large ups: gate exp(gate) up is an ordinary value down
    to gates of -197 and is kept, each in a group of its own and all in one row."""
    gate = torch.cat([torch.linspace(-86.5, -88.9, 97), torch.linspace(-89, -200, 223), torch.tensor([-256.0, -257.0, -3e4, -3e38])])
    for top in (1.0, 1e20, -3e38, 2.0 ** -140):
        up = torch.full_like(gate, top)
        v = gate.double() * torch.exp(gate.double()) / (1 + torch.exp(gate.double())) * up.double()
        v = torch.where(gate < -300, torch.zeros_like(v), v)
        got = rq.silu_and_mul_f8(gate.view(-1, 1).to(DEV), up.view(-1, 1).to(DEV))
        codes, scales = got.codes.cpu().float().double()[:, 0], got.scales.cpu().double()[:, 0]
        # a group of one value: the scale is its size / 448 (2^-22 and SiLU's 2^-20; below 2^-126 a step of 2^-149 more, as
        # the product and its last factor each round there)
        size = v.abs().clamp(min=448 * LEAST) / 448
        assert ((scales - size).abs() <= size * (2.0 ** -22 + 2.0 ** -20)).all()
        sure = v.abs() >= 448 * LEAST
        assert (codes[sure] == torch.sign(v[sure]) * 448).all()
        half = torch.clamp(v.abs() / scales * 2.0 ** -4, min=2.0 ** -10)
        assert ((codes - v / scales).abs() <= half * (1 + 2.0 ** -10) + v.abs() / scales * 2.0 ** -19).all()
        _check_codes(*(lambda o: (o.codes, o.scales))(rq.silu_and_mul_f8(gate.view(1, -1).to(DEV), up.view(1, -1).to(DEV))),
                     v.view(1, -1), 2.0 ** -20)
    for dtype in (F16, BF16):
        g, u = gate[:300].to(dtype), torch.full((300,), 6e4).to(dtype)
        v = g.double() * torch.exp(g.double()) / (1 + torch.exp(g.double())) * u.double()
        got = rq.silu_and_mul_f8(g.view(1, -1).to(DEV), u.view(1, -1).to(DEV))
        _check_codes(got.codes, got.scales, v.view(1, -1), 2.0 ** -20)
    mixed = torch.randn(40, 700, generator=_gen(8)) * 60  # near and far ones side by side
    ups = torch.randn(40, 700, generator=_gen(9)) * 1e30
    got = rq.silu_and_mul_f8(mixed.to(DEV), ups.to(DEV))
    m = mixed.double()
    _check_codes(got.codes, got.scales, m * torch.sigmoid(m) * ups.double(), 2.0 ** -20)
    got = rq.silu_and_mul_f8(torch.tensor([[-200.0, -math.inf]], device=DEV), torch.ones(1, 2, device=DEV))
    assert torch.isnan(got.scales).all()


@pytest.mark.parametrize("k", [128, 4096, 40000])
def test_norm_of_odd_rows(rq, k):
    """Rows of zeros, of huge and of tiny values, a row that is not finite: the others keep their results."""
    x = _values(6, k, F32, k, 0.0)
    x[1] = 0.0
    x[2] *= 2.0 ** -70
    x[3] *= 2.0 ** 55
    x[4, k // 2] = float("nan")
    w = torch.ones(k)
    out, _, y = rq.add_rmsnorm_f8(x.to(DEV), None, w.to(DEV), 1e-6, want_y=True)
    assert torch.isnan(out.scales[4]).all() and torch.isnan(y[4]).all()
    keep = [0, 1, 2, 3, 5]
    _check_norm(x[keep], None, w, 1e-6, rq.F8Rows(out.codes[keep], out.scales[keep]), None, y[keep])
    assert (y[1] == 0).all()


def test_rows_past_4_gib(rq):
    """The last rows of a matrix whose offsets pass 32 bits."""
    k, stride, rows = 256, 1 << 20, 4100
    buf = torch.empty(rows * stride, dtype=torch.uint8, device=DEV)
    out = rq.F8Rows(buf.view(rows, stride)[:, :k], torch.empty(rows, 2, device=DEV))
    x = torch.randn(rows, k, generator=_gen(3))
    rq.quantize_f8(x.to(DEV), out=out)
    at = [0, 1, 2047, 2048, 4095, 4096, 4099]
    _check_codes(out.codes[at].contiguous().view(F8), out.scales[at], x[at].double(), 0.0)
    rq.add_rmsnorm_f8(x.to(DEV), None, torch.ones(k, device=DEV), 1e-6, out=out)
    _check_norm(x[at], None, torch.ones(k), 1e-6, rq.F8Rows(out.codes[at].contiguous().view(F8), out.scales[at]), None, None)
    w = torch.randn(100, k, generator=_gen(4)).to(F8)
    ws = torch.rand(1, 2, generator=_gen(5)) + 0.5
    y = rq.gemm_f8(out, rq.F8Weight(w.to(DEV), ws.to(DEV)))
    _check_product(out.codes[at].contiguous().view(F8).cpu(), out.scales[at].cpu(), w, ws, y[at])


# ------------------------------------------------------------------ products

def _wide(codes, scales):
    """[rows, k] e4m3 codes with a scale for each 128 of a row, in 64 bits."""
    return codes.float().double() * scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]


def _wide_weight(codes, scales):
    return _wide(codes, scales.repeat_interleave(128, 0)[:codes.shape[0]])


def _eights(codes, scales):
    """2^e of the largest exponent of each eight neighbouring codes of a row, times their scale."""
    rows, k = codes.shape
    e = torch.exp2(torch.floor(torch.log2(codes.float().double().abs().clamp(min=2.0 ** -6))))
    e = torch.nn.functional.pad(e, (0, _blocks(k) * 128 - k)).view(rows, -1, 8).amax(2)
    return e * scales.double().repeat_interleave(16, 1)


def _slack(x, xs, w, ws, y_type):
    """What the eights of the matrix instructions may lose."""
    if y_type == F32:
        return 0.0
    return 2.0 ** -10 * (_eights(x, xs) @ _eights(w, ws.repeat_interleave(128, 0)[:w.shape[0]]).t())


def _check_product(x, xs, w, ws, y):
    """y [rows, n] on the GPU against x @ w.T of both with their scales (where x is)."""
    xd, wd = _wide(x, xs), _wide_weight(w, ws)
    want, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    bound = size * (_blocks(x.shape[1]) + 32) * 2.0 ** -23 + want.abs() * torch.finfo(y.dtype).eps / 2 + TINY[y.dtype]
    bound = bound + _slack(x, xs, w, ws, y.dtype) * (1 + torch.finfo(y.dtype).eps)
    got = y.to(x.device).double()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist(), float((got - want).abs().max()))


def _case(rows, k, n, seed, count=None):
    g = _gen(seed)
    x = torch.randn(rows, k, generator=g).mul_(60).clamp_(-448, 448).to(F8)
    xs = torch.exp(torch.randn(rows, _blocks(k), generator=g)) / 60
    shape = (n, k) if count is None else (count, n, k)
    w = torch.randn(*shape, generator=g).mul_(60).clamp_(-448, 448).to(F8)
    ws = torch.exp(torch.randn(*(shape[:-2] + (_blocks(n), _blocks(k))), generator=g)) / 6000
    return x, xs, w, ws


PRODUCTS = [(1, 1, 1), (1, 128, 16), (1, 4096, 1024), (2, 127, 3), (3, 129, 17), (4, 256, 128), (5, 1000, 130), (8, 768, 2048),
            (16, 2048, 768), (17, 384, 257), (31, 1235, 1531), (32, 4096, 512), (33, 640, 640), (48, 2048, 320),
            (64, 1024, 4096), (65, 1152, 129), (100, 512, 512), (127, 300, 200), (128, 2048, 1024), (130, 4096, 256),
            (200, 896, 1000), (256, 1024, 2048), (257, 768, 768), (333, 1235, 1531), (512, 512, 4096), (1000, 400, 1100),
            (1025, 256, 2304), (2100, 384, 1300), (4200, 640, 2200)]


@pytest.mark.parametrize("y_type", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k,n", PRODUCTS)
def test_gemm(rq, rows, k, n, y_type):
    x, xs, w, ws = _case(rows, k, n, rows + k + n)
    _say("gemm", rows, k, n, y_type)
    y = rq.gemm_f8(rq.F8Rows(x.to(DEV), xs.to(DEV)), rq.F8Weight(w.to(DEV), ws.to(DEV)), dtype=y_type)
    assert y.dtype == y_type and y.shape == (rows, n)
    _check_product(x, xs, w, ws, y)


@pytest.mark.parametrize("y_type", [F32, F16, BF16])
@pytest.mark.parametrize("xshift,xpad,wshift,yshift,ypad", [(0, 0, 1, 0, 0), (1, 0, 0, 1, 1), (5, 3, 7, 2, 3), (16, 16, 16, 8, 8),
                                                            (4, 12, 8, 4, 4), (0, 128, 0, 0, 128)])
@pytest.mark.parametrize("rows,k,n", [(1, 512, 64), (9, 300, 130), (40, 1024, 200), (150, 640, 333), (600, 512, 400)])
def test_gemm_strides(rq, rows, k, n, xshift, xpad, wshift, yshift, ypad, y_type):
    """Strides and alignment of all operands; NaN codes and scales between the rows, and y's gaps left as they were."""
    _say("gemm strides", rows, k, n, xshift, xpad, wshift, yshift, ypad, y_type)
    x, xs, w, ws = _case(rows, k, n, rows + k)
    xd, _ = _strided(x.view(torch.uint8), k + xpad, xshift, 0x7F)
    xsd, _ = _strided(xs, _blocks(k) + xpad, xshift, 0xFF)
    wd, _ = _strided(w.view(torch.uint8).reshape(1, -1), n * k, wshift, 0x7F)
    y, buf = _strided(torch.zeros(rows, n, dtype=y_type), n + ypad, yshift, 0xA5)
    before = buf.clone()
    rq.gemm_f8(rq.F8Rows(xd, xsd), rq.F8Weight(wd.view(n, k), ws.to(DEV)), out=y)
    _check_product(x, xs, w, ws, y)
    y.copy_(before[yshift:yshift + rows * (n + ypad)].view(rows, n + ypad)[:, :n])
    assert torch.equal(buf.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.parametrize("y_type", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [1, 5, 20, 40, 70, 130, 300, 600, 1100])
def test_gemm_every_code(rq, rows, y_type):
    """Rows of one 1.0 among zeros pick single weights: every code comes through as it is, NaN in its place."""
    k, n = 256, 256
    w = torch.arange(256, dtype=torch.uint8).view(1, 256).repeat(n, 1)
    w = torch.stack([torch.roll(w[i], i) for i in range(n)])  # w[n][k] = code (k - n) mod 256
    x = torch.zeros(rows, k)
    pick = (torch.arange(rows) * 7) % k
    x[torch.arange(rows), pick] = 1.0
    scales = torch.ones(rows, 2)
    y = rq.gemm_f8(rq.F8Rows(x.to(F8).to(DEV), scales.to(DEV)), rq.F8Weight(w.to(DEV), torch.ones(2, 2, device=DEV)),
                   dtype=y_type)
    # a NaN weight anywhere in column n's row makes every product with that row NaN: 0 * NaN
    assert torch.isnan(y).all()
    clean = torch.where((w & 0x7F) == 0x7F, torch.zeros_like(w), w)
    y = rq.gemm_f8(rq.F8Rows(x.to(F8).to(DEV), scales.to(DEV)), rq.F8Weight(clean.to(DEV), torch.ones(2, 2, device=DEV)),
                   dtype=y_type)
    want = clean.view(F8).float()[:, pick].t()
    assert torch.equal(y.cpu().float(), want)


@pytest.mark.parametrize("y_type", [F32, BF16])
@pytest.mark.parametrize("rows,k,n", [(1, 300, 40), (12, 512, 300), (40, 1024, 256), (140, 640, 300), (700, 384, 520)])
def test_gemm_not_finite(rq, rows, k, n, y_type):
    """NaN codes, NaN and infinite scales: the results that they belong to, and no others."""
    x, xs, w, ws = _case(rows, k, n, 5)
    x.view(torch.uint8)[rows // 2, k - 1] = 0x7F
    w.view(torch.uint8)[n // 3, 0] = 0xFF
    xs[rows - 1, 0] = float("nan")
    ws[-1, -1] = float("inf")
    y = rq.gemm_f8(rq.F8Rows(x.to(DEV), xs.to(DEV)), rq.F8Weight(w.to(DEV), ws.to(DEV)), dtype=y_type).cpu()
    bad = torch.zeros(rows, n, dtype=torch.bool)
    bad[rows // 2] = bad[rows - 1] = True
    bad[:, n // 3] = True
    bad[:, 128 * (_blocks(n) - 1):] = True  # infinite or NaN
    assert not torch.isfinite(y[bad]).any()
    assert torch.isfinite(y[~bad]).all()
    if not bad.all():  # the good columns lie in whole blocks, but for one whose products are left out
        row, full = (~bad).any(1), 128 * (_blocks(n) - 1)
        w[n // 3] = 0.0
        y[:, n // 3] = 0.0
        _check_product(x[row], xs[row], w[:full], ws[:-1], y[row][:, :full])


@pytest.mark.parametrize("y_type", [F32, BF16])
@pytest.mark.parametrize("rows,n", [(1, 40), (40, 300), (300, 2050), (900, 2100), (2040, 4090), (4090, 4090)])
@pytest.mark.parametrize("k", [128, 300, 336, 640, 645])
def test_gemm_infinite_scale(rq, rows, n, k, y_type):
    """Positive values and a scale that is infinite in the last block of K: infinity there, not NaN of blocks behind it."""
    x, w = (torch.full((r, k), 1.0).to(F8).to(DEV) for r in (rows, n))
    xs, ws = torch.ones(rows, _blocks(k), device=DEV), torch.ones(_blocks(n), _blocks(k), device=DEV)
    xs[rows // 2, -1] = math.inf
    _say("infinite scale", rows, n, k, y_type)
    y = rq.gemm_f8(rq.F8Rows(x, xs), rq.F8Weight(w, ws), dtype=y_type)
    assert (y[rows // 2] == math.inf).all()
    y[rows // 2] = float(k)  # exact in f32; bf16 rounds it
    assert (y == torch.tensor(float(k)).to(y_type)).all()


def test_gemm_matrix_past_4_gib(rq):
    """Weights of more than 4 GiB: rows at both ends, for few and for many rows."""
    k, n = 16384, (1 << 18) + 136
    w = torch.zeros(n, k, dtype=torch.uint8, device=DEV)
    ws = torch.ones(_blocks(n), _blocks(k), device=DEV)
    at = torch.tensor([0, 1, 200, 131071, 131072, n - 130, n - 2, n - 1])
    part = torch.randn(len(at), k, generator=_gen(1)).to(F8)
    w[at.to(DEV)] = part.view(torch.uint8).to(DEV)
    for rows in (1, 20, 300):
        x, xs, _, _ = _case(rows, k, 1, rows)
        y = rq.gemm_f8(rq.F8Rows(x.to(DEV), xs.to(DEV)), rq.F8Weight(w, ws), dtype=BF16)
        got = y[:, at.to(DEV)]
        xd = _wide(x, xs)
        want, size = xd @ part.float().double().t(), xd.abs() @ part.float().double().abs().t()
        slack = 2.0 ** -10 * (_eights(x, xs) @ _eights(part, torch.ones(len(at), _blocks(k))).t())
        assert ((got.cpu().double() - want).abs() <= size * (_blocks(k) + 32) * 2.0 ** -23 + want.abs() * 2.0 ** -8
                + 1.01 * slack).all()
        rest = torch.ones(n, dtype=torch.bool)
        rest[at] = False
        assert not y[:, rest.to(DEV)].any()


@pytest.mark.parametrize("rows,gap", [(3, 1 << 31), (200, 1 << 25)])
@pytest.mark.parametrize("what", ["codes", "scales"])
def test_gemm_rows_past_4_gib(rq, rows, gap, what):
    """Rows, or their scales, that lie further apart than 32 bits of bytes reach."""
    x, xs, w, ws = (t.to(DEV) for t in _case(rows, 400, 300, rows))
    far = x.view(torch.uint8) if what == "codes" else xs
    step = gap // far.element_size()
    buf = torch.empty((rows - 1) * step + far.shape[1], dtype=far.dtype, device=DEV)
    view = buf.as_strided(far.shape, (step, 1))
    view.copy_(far)
    _say("past 4 GiB", rows, what)
    rows_ = rq.F8Rows(view.view(F8), xs) if what == "codes" else rq.F8Rows(x, view)
    weight = rq.F8Weight(w, ws)
    for y_type in (F32, BF16):
        _check_product(x, xs, w, ws, rq.gemm_f8(rows_, weight, dtype=y_type))
    back = torch.arange(rows - 1, -1, -1, dtype=torch.int32, device=DEV)
    y = rq.grouped_gemm_f8(rows_, weight, torch.tensor([0, rows], dtype=torch.int32, device=DEV), rows, x_index=back)
    _check_product(x.view(torch.uint8).flip(0).view(F8), xs.flip(0), w, ws, y)


@pytest.mark.parametrize("k,n", [(16, 5), (17, 5), (128, 130)])
def test_gemm_many_rows(rq, k, n):
    rows = 2_000_003
    g = torch.Generator(DEV).manual_seed(k)
    x = torch.randint(-1, 2, (rows, k), generator=g, device=DEV).float().to(F8)
    w = torch.randint(-1, 2, (n, k), generator=g, device=DEV).float().to(F8)
    xs = torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g, device=DEV).float())
    _say("many rows", k, n)
    y = rq.gemm_f8(rq.F8Rows(x, xs), rq.F8Weight(w, torch.ones(_blocks(n), 1, device=DEV)))
    assert torch.equal(y, (x.float() @ w.float().t()) * xs)  # whole numbers times powers of two


def _whole(rows, k, seed):
    """Codes of -1, 0 and 1."""
    return torch.randint(-1, 2, (rows, k), generator=torch.Generator(DEV).manual_seed(seed), device=DEV).float().to(F8)


def _launches(rq, x, w, rows, grouped, y_type):
    import ctypes

    how = rq.RfxqF8Launch()
    ty = {F32: 0, F16: 1, BF16: 30}[y_type]
    assert rq.lib().rfxq_gemm_f8_launch(x._c, w._c, rows, grouped, ty, ctypes.byref(how)) == 0
    return how.launches


PERIOD = (1 << 20) + 77


def test_gemm_more_rows_than_a_launch(rq):
    """A narrow product of more workgroups than a launch takes: every row, the gaps between rows left as they were."""
    rows, k, n = (1 << 27) + 12345, 17, 5
    few, w = _whole(PERIOD, k, 1), _whole(n, k, 2)
    few_scales = torch.exp2(torch.randint(-3, 4, (PERIOD, 1), generator=torch.Generator(DEV).manual_seed(3), device=DEV).float())
    times = -(-rows // PERIOD)
    x = rq.F8Rows(few.view(torch.uint8).repeat(times, 1)[:rows].view(F8), few_scales.repeat(times, 1)[:rows])
    weight = rq.F8Weight(w, torch.ones(1, 1, device=DEV))
    _say("rows", rows, _launches(rq, x, weight, rows, 0, F16))
    assert _launches(rq, x, weight, rows, 0, F16) > 1
    buf = torch.full((rows + 1, n + 1), 7.0, dtype=F16, device=DEV)
    rq.gemm_f8(x, weight, out=buf[:rows, :n])
    want = ((few.float() @ w.float().t()) * few_scales).to(F16)  # whole numbers times powers of two
    for at in range(0, rows, PERIOD):
        part = buf[at:min(at + PERIOD, rows)]
        assert torch.equal(part[:, :n], want[:part.shape[0]]), at
    assert (buf[:, n] == 7.0).all() and (buf[rows] == 7.0).all()


def test_gemm_more_columns_than_a_launch(rq):
    rows, k, n = 1, 17, (1 << 27) + 77
    x, few = _whole(rows, k, 1), _whole(PERIOD, k, 2)
    times = -(-n // PERIOD)
    scales = torch.exp2((torch.arange(_blocks(n), device=DEV) % 7 - 3).float())
    weight = rq.F8Weight(few.view(torch.uint8).repeat(times, 1)[:n].view(F8), scales.view(-1, 1))
    xr = rq.F8Rows(x, torch.ones(rows, 1, device=DEV))
    _say("columns", n, _launches(rq, xr, weight, rows, 0, F32))
    assert _launches(rq, xr, weight, rows, 0, F32) > 1
    y = rq.gemm_f8(xr, weight)[0]
    want = (few.float() @ x[0].float()).repeat(times)[:n] * scales.repeat_interleave(128)[:n]
    assert torch.equal(y, want)


def test_grouped_more_places_than_a_launch(rq):
    """Places of three groups that name few rows of x, some none."""
    rows, k, n = (1 << 27) + 999, 17, 5
    x, w = _whole(PERIOD, k, 1), torch.stack([_whole(n, k, 2 + e) for e in range(3)])
    offsets = [3, 1000, (1 << 26) + 5, rows - 2]
    index = torch.arange(rows, dtype=torch.int32, device=DEV) % (PERIOD + 1) - 1  # -1: no row
    xr, weight = rq.F8Rows(x, torch.ones(PERIOD, 1, device=DEV)), rq.F8Weight(w, torch.ones(3, 1, 1, device=DEV))
    _say("places", rows, _launches(rq, xr, weight, rows, 1, F16))
    assert _launches(rq, xr, weight, rows, 1, F16) > 1
    y = torch.full((rows, n), 7.0, dtype=F16, device=DEV)
    rq.grouped_gemm_f8(xr, weight, torch.tensor(offsets, dtype=torch.int32, device=DEV), rows, x_index=index, out=y)
    each = [torch.cat([torch.full((1, n), 7.0, device=DEV), x.float() @ w[e].float().t()]).to(F16) for e in range(3)]
    step = 1 << 22
    for at in range(0, rows, step):
        end = min(at + step, rows)
        want = torch.full((end - at, n), 7.0, dtype=F16, device=DEV)
        for e in range(3):
            lo, hi = max(offsets[e], at), min(offsets[e + 1], end)
            if lo < hi:
                want[lo - at:hi - at] = each[e][index[lo:hi].long() + 1]
        assert torch.equal(y[at:end], want), at


def test_more_groups_than_a_launch(rq):
    """More rows than the largest launches have places for."""
    rows = (1 << 24) + 77
    x = torch.randn(rows, 1, generator=torch.Generator(DEV).manual_seed(1), device=DEV)
    one = torch.ones_like(x)
    for out, v in ((rq.quantize_f8(x), x), (rq.silu_and_mul_f8(x, one), torch.nn.functional.silu(x))):
        _say("groups", rows)
        # a group of one value: the largest code, but for 0, whose quotient by the least scale is 0
        assert torch.equal(out.codes.float().abs(), torch.where(v == 0, 0.0, 448.0))
        assert ((out.codes.float() * out.scales - v).abs() <= v.abs() * 2.0 ** -18).all()
    rows = (1 << 20) + 37
    x = torch.randn(rows, 8, generator=torch.Generator(DEV).manual_seed(2), device=DEV)
    out, _, y = rq.add_rmsnorm_f8(x, None, torch.ones(8, device=DEV), 1e-6, want_y=True)
    want = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -20).all()
    assert ((out.codes.double() * out.scales.double() - y.double()).abs()
            <= torch.maximum(y.abs().double() * 2.0 ** -4, out.scales.double() * 2.0 ** -10) * (1 + 2.0 ** -18)).all()


ANY, FEW, STREAM, COPIED, LARGE = range(5)


def _kernel(rq, x, w, rows, grouped, y_type):
    import ctypes

    p = rq.RfxqF8Policy()
    ty = {F32: 0, F16: 1, BF16: 30}[y_type]
    assert rq.lib().rfxq_gemm_f8_policy(x._c, w._c, rows, grouped, ty, ctypes.byref(p)) == 0
    return p.kernel, p.tile_m, p.tile_n


# each kernel over short and long K: whole and odd numbers of blocks, a last block of one piece, more blocks than
# a kernel's buffers, places or staged scales hold; tiles that end inside one
EACH = [
    (3, 9360, 48, F32, (STREAM, 16, 16)), (16, 16, 1000, BF16, (STREAM, 16, 32)), (7, 3856, 1040, F16, (STREAM, 16, 16)),
    (5, 8448, 4992, BF16, (STREAM, 16, 32)), (30, 8208, 4100, F32, (STREAM, 16, 32)), (60, 8304, 4090, BF16, (STREAM, 32, 32)),
    (130, 8304, 3600, F32, (STREAM, 32, 32)), (300, 4368, 3600, F16, (COPIED, 64, 128)), (512, 784, 3100, BF16, (COPIED, 64, 128)),
    (128, 8304, 4090, BF16, (STREAM, 32, 64)), (120, 9360, 3800, F32, (STREAM, 32, 64)), (250, 784, 2040, F16, (STREAM, 32, 64)),
    (200, 8304, 4090, F32, (STREAM, 64, 64)), (250, 9360, 3900, BF16, (STREAM, 64, 64)), (250, 1040, 4050, F32, (STREAM, 64, 64)),
    (400, 4368, 3100, F32, (COPIED, 64, 128)), (390, 784, 2600, F32, (COPIED, 64, 128)), (600, 4368, 4090, BF16, (COPIED, 128, 128)),
    (1000, 2176, 4000, F16, (COPIED, 128, 128)), (700, 1040, 3600, F32, (COPIED, 128, 128)), (1000, 4368, 4000, F32, (COPIED, 128, 128)),
    (1024, 1664, 7000, BF16, (LARGE, 128, 256)), (2040, 128, 4090, F16, (LARGE, 128, 256)), (2048, 1168, 4000, BF16, (LARGE, 128, 256)),
    (4095, 656, 4090, BF16, (LARGE, 256, 256)), (4090, 128, 4096, F16, (LARGE, 256, 256)), (4096, 16, 4096, BF16, (LARGE, 256, 256)),
    (4090, 1040, 4088, F16, (LARGE, 256, 256)),
    (1, 4099, 4099, F32, (FEW, 16, 16)), (16, 1237, 300, BF16, (FEW, 16, 16)), (333, 1235, 1531, F32, (ANY, 32, 64)),
    (100, 4101, 1531, F16, (ANY, 32, 64)), (333, 4099, 4099, F32, (ANY, 64, 128)), (900, 13, 4099, F32, (ANY, 32, 64)),
    (700, 1301, 2100, F32, (ANY, 64, 128)),
    (1000, 4099, 4099, BF16, (ANY, 64, 128)), (333, 2099, 4099, F16, (ANY, 64, 128)), (900, 7, 3100, BF16, (ANY, 64, 128)),
    (300, 3, 1700, F32, (ANY, 32, 64)), (5, 11, 100, BF16, (FEW, 16, 16)),
]


@pytest.mark.parametrize("rows,k,n,y_type,kernel", EACH)
def test_gemm_each_kernel(rq, rows, k, n, y_type, kernel):
    x, xs, w, ws = (t.to(DEV) for t in _case(rows, k, n, rows + k))
    xr, weight = rq.F8Rows(x, xs), rq.F8Weight(w, ws)
    _say("each", rows, k, n, y_type, kernel)
    assert _kernel(rq, xr, weight, rows, 0, y_type) == kernel
    y = torch.full((rows + 2, n + 3), 7.0, dtype=y_type, device=DEV)
    rq.gemm_f8(xr, weight, out=y[1:rows + 1, :n])
    _check_product(x, xs, w, ws, y[1:rows + 1, :n])
    y[1:rows + 1, :n] = 7.0
    assert (y == 7.0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,k,n,kernel", [(r, k, n, p) for r, k, n, t, p in EACH if t == F32] + [
    (30, 700, 900, None), (300, 333, 500, None), (60, 8304, 4090, (STREAM, 32, 32)), (2048, 4096, 4096, (COPIED, 128, 128))])
def test_gemm_exact(rq, rows, k, n, kernel, dtype):
    """exact: half results are f32 results rounded once, to the last bit, in every kernel that has them."""
    x, xs, w, ws = (t.to(DEV) for t in _case(rows, k, n, rows + k))
    xr, weight = rq.F8Rows(x, xs), rq.F8Weight(w, ws)
    _say("exact", rows, k, n, kernel, dtype)
    assert kernel is None or _kernel(rq, xr, weight, rows, 0, F32) == kernel
    want = rq.gemm_f8(xr, weight)
    assert torch.equal(rq.gemm_f8(xr, weight, dtype=dtype, exact=True), want.to(dtype))
    assert torch.equal(rq.gemm_f8(xr, weight, exact=True), want)
    y = torch.full((rows + 2, n + 3), 7.0, dtype=dtype, device=DEV)
    assert rq.gemm_f8(xr, weight, out=y[1:rows + 1, :n], exact=True).data_ptr() == y[1:].data_ptr()
    assert torch.equal(y[1:rows + 1, :n], want.to(dtype))
    y[1:rows + 1, :n] = 7.0
    assert (y == 7.0).all()


def test_gemm_exact_keeps_small_products(rq):
    """Products below 2^-13 of their neighbours add up: 7 of them in each eight, in each kernel of many rows."""
    for rows, n in ((100, 1024), (200, 4090), (400, 3100), (1000, 4000), (2048, 4000)):
        k = 1024
        x = torch.full((rows, k), 0.5)
        x[:, ::8] = 256.0
        w = torch.full((n, k), 2.0 ** -6)
        w[:, ::8] = 1.0
        w[:, 8::16] = -1.0  # the large ones cancel
        one, two = torch.ones(rows, _blocks(k), device=DEV), torch.ones(_blocks(n), _blocks(k), device=DEV)
        y = rq.gemm_f8(rq.F8Rows(x.to(F8).to(DEV), one), rq.F8Weight(w.to(F8).to(DEV), two), dtype=F16, exact=True)
        assert (y == 7 * 128 * 2.0 ** -7).all()


# a size of each kernel that cuts products, over short and long K, and of kernels that do not
RMS = [(120, 1280, 3800, (STREAM, 32, 64)), (128, 8304, 4090, (STREAM, 32, 64)), (200, 2048, 4050, (STREAM, 64, 64)),
       (250, 9360, 3900, (STREAM, 64, 64)), (512, 784, 3100, (COPIED, 64, 128)), (300, 4368, 3600, (COPIED, 64, 128)),
       (1000, 512, 4000, (COPIED, 128, 128)), (600, 4368, 4090, (COPIED, 128, 128)), (2040, 256, 4090, (LARGE, 128, 256)),
       (1024, 8192, 7000, (LARGE, 128, 256)), (4090, 256, 4096, (LARGE, 256, 256)), (4096, 4096, 4096, (LARGE, 256, 256)),
       (100, 1101, 1531, (ANY, 32, 64)), (100, 4101, 1531, (ANY, 32, 64)), (333, 2099, 4099, (ANY, 64, 128)),
       (1000, 4099, 4099, (ANY, 64, 128)), (64, 4096, 4096, (STREAM, 32, 32)), (16, 1237, 1100, (FEW, 16, 16))]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k,n,kernel", RMS)
def test_gemm_error_of_normal_values(rq, rows, k, n, kernel, dtype):
    """What results are off by as a whole, where the bound of each by itself has to allow for the worst.

    A product of codes has 8 bits: cut to multiples of 2^-13 2^e (e the largest sum of two codes' exponents among eight) it
    loses something only if its own exponents sum to e - 8 or less, so that it is below 2^-6 2^e. For normal values these are 5%
    of the products and 2^e is 1.1 of a product's deviation; each losing anything up to 2^-13 2^e, evenly spread, they
    are sqrt(0.05 / 3) 1.1 2^-13 = 1.7e-5 of a result (the cut itself, carried out on such codes: 1.5e-5): 2e-5. Sums: 2^-23 an
    addition, K / 128 + 32 of them in a row, by chance: sqrt(105) 2^-23 = 1.2e-6 at K = 9360. Beyond that a result is
    rounded once: as much as the 64-bit value's rounding, give or take 2% for the few of 16000 and more that round to the
    other side."""
    cut = 0.0 if dtype == F32 or kernel in ((STREAM, 32, 32), (FEW, 16, 16)) else 2e-5
    x, xs, w, ws = (t.to(DEV) for t in _case(rows, k, n, rows + k + n))
    xr, weight = rq.F8Rows(x, xs), rq.F8Weight(w, ws)
    _say("rms", rows, k, n, dtype, _kernel(rq, xr, weight, rows, 0, dtype))
    assert dtype == F32 or _kernel(rq, xr, weight, rows, 0, dtype) == kernel
    want = _wide(x, xs) @ _wide_weight(w, ws).t()
    for exact in (False, True):
        y = rq.gemm_f8(xr, weight, dtype=dtype, exact=exact).double()
        # rows have scales of their own: each by its own size
        size = want.square().mean(1, keepdim=True).sqrt()
        off = ((y - want) / size).square().mean().sqrt()
        rounded = ((want.to(dtype).double() - want) / size).square().mean().sqrt()
        _say("off by", float(off), "rounding", float(rounded))
        assert off <= 1.02 * rounded + (0.0 if exact else cut) + 1.5e-6


@pytest.mark.parametrize("extra", [0, 16, 112, 128, 129, 240])
@pytest.mark.parametrize("blocks", range(1, 15))
@pytest.mark.parametrize("rows,n,y_type", [(2, 40, F32), (40, 300, BF16), (200, 2100, F32), (300, 2050, BF16), (2048, 2050, BF16),
                                           (1100, 2050, F32)])
def test_gemm_every_number_of_blocks(rq, rows, n, y_type, blocks, extra):
    """Few rows of ones and a last row that counts blocks: what each block gives is a power of two of its own."""
    k = 128 * (blocks - 1) + (extra or 128)
    g = _gen(blocks + extra)
    x = torch.where(torch.rand(rows, k, generator=g) < 0.5, 1.0, -1.0).to(F8).to(DEV)
    xs = torch.exp2(torch.arange(_blocks(k)).float()).repeat(rows, 1).to(DEV)
    w = torch.where(torch.rand(n, k, generator=g) < 0.5, 1.0, 0.5).to(F8).to(DEV)
    ws = torch.ones(_blocks(n), _blocks(k), device=DEV)
    y = rq.gemm_f8(rq.F8Rows(x, xs), rq.F8Weight(w, ws), dtype=y_type)
    want = _wide(x, xs) @ _wide_weight(w, ws).t()
    # sums of halves below 2^24 are exact in f32
    half = 0.0 if y_type == F32 else torch.finfo(y_type).eps / 2
    assert ((y.double() - want).abs() <= want.abs() * half).all()


def test_gemm_rows_that_repeat(rq):
    """A matrix of one row repeated (stride 0 is refused; equal rows are not): equal rows give equal bits in every kernel."""
    for rows, n in ((13, 64), (100, 1024), (400, 3100), (2048, 4000)):
        x, xs, w, ws = (t.to(DEV) for t in _case(1, 1168, n, rows))
        y = rq.gemm_f8(rq.F8Rows(x.repeat(rows, 1), xs.repeat(rows, 1)), rq.F8Weight(w, ws), dtype=BF16)
        assert (y == y[:1]).all()


# ------------------------------------------------------------------ grouped products

def _run_grouped(rq, x, xs, w, ws, ids, top_k, side, y_type, spare=3):
    """Pairs grouped by `ids`; gate: x a row per token; down: a row per pair. Returns (y, what it held before, order)."""
    count = w.shape[0]
    g = rq.group_rows(ids.to(DEV), count)
    rows = ids.numel()
    y = torch.full((rows + spare, w.shape[1]), 7.0, dtype=y_type, device=DEV)
    weight, xr = rq.F8Weight(w.to(DEV), ws.to(DEV)), rq.F8Rows(x.to(DEV), xs.to(DEV))
    if side == "gate":
        rq.grouped_gemm_f8(xr, weight, g.offsets, rows, x_index=g.order, x_div=top_k, out=y)
    else:
        rq.grouped_gemm_f8(xr, weight, g.offsets, rows, y_index=g.order, out=y)
    return y, g


def _check_grouped(x, xs, w, ws, ids, top_k, side, y, g):
    offsets, order = g.offsets.cpu().long(), g.order.cpu().long()
    rows = ids.numel()
    for e in range(w.shape[0]):
        at = torch.arange(int(offsets[e]), int(offsets[e + 1]))
        if at.numel():
            src, dst = (order[at] // top_k, at) if side == "gate" else (at, order[at])
            _check_product(x[src], xs[src], w[e], ws[e], y[dst.to(DEV)])
    none = torch.arange(int(offsets[-1]), rows)
    left = torch.cat([none if side == "gate" else order[none], torch.arange(rows, y.shape[0])])
    assert (y[left.to(DEV)] == 7.0).all()


GROUPED = [(1, 8, 8, 256, 128), (1, 1, 1, 130, 30), (4, 16, 2, 768, 320), (32, 128, 8, 256, 200), (60, 5, 1, 300, 257),
           (100, 3, 2, 1024, 384), (300, 4, 2, 512, 512), (500, 11, 3, 1235, 531), (700, 2, 1, 640, 640),
           (40, 160, 8, 128, 64), (2000, 3, 2, 256, 500)]


@pytest.mark.parametrize("y_type", [F32, F16, BF16])
@pytest.mark.parametrize("side", ["gate", "down"])
@pytest.mark.parametrize("tokens,count,top_k,k,n", GROUPED)
def test_grouped(rq, tokens, count, top_k, k, n, side, y_type):
    _say("grouped", tokens, count, top_k, k, n, side, y_type)
    pairs = tokens * top_k
    x, xs, w, ws = _case(tokens if side == "gate" else pairs, k, n, tokens + k, count)
    r = np.random.default_rng(tokens + n)
    ids = torch.from_numpy(r.integers(-1, count + 1, pairs).astype(np.int32))  # some in no group
    y, g = _run_grouped(rq, x, xs, w, ws, ids, top_k, side, y_type)
    _check_grouped(x, xs, w, ws, ids, top_k, side, y, g)


GROUPED_EACH = [
    (100, 3, 8320, 48, F32, (STREAM, 16, 16)), (260, 60, 8320, 1040, BF16, (STREAM, 16, 32)), (300, 7, 768, 520, BF16, (STREAM, 32, 32)),
    (260, 120, 1040, 1040, F32, (STREAM, 16, 64)), (260, 120, 784, 2050, F16, (STREAM, 16, 64)), (3000, 6, 4240, 520, F32, (COPIED, 64, 128)),
    (1800, 7, 400, 1100, BF16, (COPIED, 128, 128)), (3000, 6, 656, 1030, F32, (COPIED, 128, 128)),
    (6000, 6, 400, 1030, F16, (LARGE, 128, 256)), (8000, 5, 1040, 1100, BF16, (LARGE, 256, 256)),
]


@pytest.mark.parametrize("side", ["gate", "down"])
@pytest.mark.parametrize("pairs,count,k,n,y_type,kernel", GROUPED_EACH)
def test_grouped_each_kernel(rq, pairs, count, k, n, y_type, kernel, side):
    top_k = 2
    x, xs, w, ws = _case(pairs // top_k if side == "gate" else pairs, k, n, pairs + k, count)
    _say("grouped each", pairs, count, k, n, y_type, kernel, side)
    r = np.random.default_rng(pairs + n)
    ids = torch.from_numpy(r.integers(-1, count + 1, pairs).astype(np.int32))
    x, xs, w, ws = (t.to(DEV) for t in (x, xs, w, ws))
    assert _kernel(rq, rq.F8Rows(x, xs), rq.F8Weight(w, ws), pairs, 1, y_type) == kernel
    y, g = _run_grouped(rq, x, xs, w, ws, ids, top_k, side, y_type)
    offsets, order = g.offsets.cpu().long(), g.order.long()
    for e in range(count):
        at = torch.arange(int(offsets[e]), int(offsets[e + 1]), device=DEV)
        if at.numel():
            src, dst = (order[at] // top_k, at) if side == "gate" else (at, order[at])
            _check_product(x[src], xs[src], w[e], ws[e], y[dst])
    none = torch.arange(int(offsets[-1]), pairs, device=DEV)
    left = torch.cat([none if side == "gate" else order[none], torch.arange(pairs, y.shape[0], device=DEV)])
    assert (y[left] == 7.0).all()


def _threads(rq, x, w, rows, grouped, y_type):
    """The kernel, its tile and threads: two kernels of rows at any byte have one tile."""
    import ctypes

    how = rq.RfxqF8Launch()
    ty = {F32: 0, F16: 1, BF16: 30}[y_type]
    assert rq.lib().rfxq_gemm_f8_launch(x._c, w._c, rows, grouped, ty, ctypes.byref(how)) == 0
    return _kernel(rq, x, w, rows, grouped, y_type) + (how.threads,)


# each kernel of rows at any byte: K below 16, of less than a block, of whole blocks and a short one, of many
GROUPED_ANY = [
    (40, 8, 11, 531, F32, (FEW, 16, 16, 512)), (16, 30, 1235, 531, F16, (FEW, 16, 16, 512)), (100, 30, 645, 100, BF16, (FEW, 16, 16, 512)),
    (500, 120, 129, 20, F32, (FEW, 16, 16, 512)),
    (2500, 8, 3, 100, F32, (ANY, 32, 64, 512)), (600, 3, 2099, 531, F32, (ANY, 32, 64, 512)), (4000, 3, 129, 1100, F32, (ANY, 32, 64, 512)),
    (4000, 1, 13, 100, F16, (ANY, 32, 64, 512)), (600, 30, 300, 531, BF16, (ANY, 32, 64, 512)), (260, 1, 1235, 2100, F16, (ANY, 32, 64, 512)),
    (1200, 120, 3, 531, BF16, (ANY, 64, 128, 256)), (2500, 8, 645, 2100, F16, (ANY, 64, 128, 256)), (4000, 3, 11, 531, BF16, (ANY, 64, 128, 256)),
    (2500, 3, 3, 531, F32, (ANY, 64, 128, 512)), (1200, 8, 1235, 2100, F32, (ANY, 64, 128, 512)), (2500, 8, 2099, 531, F32, (ANY, 64, 128, 512)),
    (600, 1, 645, 2100, F16, (ANY, 64, 128, 512)), (2500, 8, 645, 531, BF16, (ANY, 64, 128, 512)), (1200, 8, 1235, 1100, F16, (ANY, 64, 128, 512)),
]


@pytest.mark.parametrize("side", ["gate", "down"])
@pytest.mark.parametrize("pairs,count,k,n,y_type,kernel", GROUPED_ANY)
def test_grouped_each_kernel_of_any_byte(rq, pairs, count, k, n, y_type, kernel, side):
    """Rows and matrices at odd bytes, NaN between the rows and in front of the stack; some places in no group."""
    top_k = 2 if pairs % 2 == 0 else 1
    x, xs, w, ws = _case(pairs // top_k if side == "gate" else pairs, k, n, pairs + k, count)
    _say("grouped any", pairs, count, k, n, y_type, kernel, side)
    ids = torch.from_numpy(np.random.default_rng(pairs + n).integers(-1, count + 1, pairs).astype(np.int32))
    xd, _ = _strided(x.view(torch.uint8), k + 3, 1, 0x7F)
    xsd, _ = _strided(xs, _blocks(k) + 1, 1, 0xFF)
    wd, _ = _strided(w.view(torch.uint8).reshape(1, -1), w.numel(), 3, 0x7F)
    xr, weight = rq.F8Rows(xd, xsd), rq.F8Weight(wd.view(count, n, k), ws.to(DEV))
    assert _threads(rq, xr, weight, pairs, 1, y_type) == kernel
    g = rq.group_rows(ids.to(DEV), count)
    y, buf = _strided(torch.full((pairs, n), 7.0, dtype=y_type), n + 5, 3, 0xA5)
    before = buf.clone()
    more = {"x_index": g.order, "x_div": top_k} if side == "gate" else {"y_index": g.order}
    rq.grouped_gemm_f8(xr, weight, g.offsets, pairs, out=y, **more)
    offsets, order = g.offsets.cpu().long(), g.order.long()
    x, xs, w, ws = (t.to(DEV) for t in (x, xs, w, ws))
    for e in range(count):
        at = torch.arange(int(offsets[e]), int(offsets[e + 1]), device=DEV)
        if at.numel():
            src, dst = (order[at] // top_k, at) if side == "gate" else (at, order[at])
            _check_product(x[src], xs[src], w[e], ws[e], y[dst])
            y[dst] = 7.0
    assert torch.equal(buf.view(torch.uint8), before.view(torch.uint8))  # and nothing else was written


@pytest.mark.parametrize("pairs,k,n,y_type,kernel", [
    (30, 13, 211, F32, (FEW, 16, 16, 512)), (30, 301, 211, BF16, (FEW, 16, 16, 512)), (600, 1235, 531, F32, (ANY, 32, 64, 512)),
    (600, 301, 1100, F16, (ANY, 32, 64, 512)), (2500, 333, 1100, BF16, (ANY, 64, 128, 256)), (2500, 1235, 1100, F32, (ANY, 64, 128, 512)),
    (2500, 1235, 531, F16, (ANY, 64, 128, 512)), (2500, 7, 531, F32, (ANY, 64, 128, 512)),
    (30, 256, 211, BF16, (STREAM, 16, 32, 512)), (2000, 656, 1030, F32, (COPIED, 128, 128, 512)), (2500, 400, 1030, BF16, (COPIED, 128, 128, 512)),
    (4000, 400, 1030, F16, (LARGE, 128, 256, 512)), (8000, 1040, 1100, BF16, (LARGE, 256, 256, 512))])
def test_grouped_indexes_out_of_range_in_each_kernel(rq, pairs, k, n, y_type, kernel):
    """Places whose index names no row, in three groups of which one is short and one ends inside a tile."""
    x, xs, w, ws = (t.to(DEV) for t in _case(pairs, k, n, pairs + k, 3))
    weight, xr = rq.F8Weight(w, ws), rq.F8Rows(x, xs)
    _say("out of range", pairs, k, n, y_type, kernel)
    assert _threads(rq, xr, weight, pairs, 1, y_type) == kernel
    offsets = [0, 5, 5 + (pairs - 5) * 2 // 3, pairs]
    index = torch.arange(pairs - 1, -1, -1, dtype=torch.int32, device=DEV)
    for bad, at in ((-1, 0), (pairs, 1), (-(1 << 31), 3), ((1 << 31) - 1, 8)):
        index[at::11] = bad
    index[offsets[2]:offsets[2] + 40] = -1  # whole operands of a tile
    good = (index >= 0) & (index < pairs)
    for kind in ("x_index", "y_index"):
        y = torch.full((pairs + 2, n), 7.0, dtype=y_type, device=DEV)
        rq.grouped_gemm_f8(xr, weight, torch.tensor(offsets, dtype=torch.int32, device=DEV), pairs, out=y[:pairs], **{kind: index})
        for e in range(3):
            at = torch.arange(offsets[e], offsets[e + 1], device=DEV)
            at = at[good[at]]
            src, dst = (index[at].long(), at) if kind == "x_index" else (at, index[at].long())
            if at.numel():
                _check_product(x[src], xs[src], w[e], ws[e], y[dst])
                y[dst] = 7.0
        assert (y == 7.0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("pairs,count,k,n", [(100, 3, 384, 520), (300, 7, 768, 520), (3000, 6, 656, 1030), (500, 11, 1235, 531)])
def test_grouped_exact(rq, pairs, count, k, n, dtype):
    x, xs, w, ws = (t.to(DEV) for t in _case(pairs, k, n, pairs + k, count))
    ids = torch.from_numpy(np.random.default_rng(pairs).integers(-1, count + 1, pairs).astype(np.int32))
    g = rq.group_rows(ids.to(DEV), count)
    _say("grouped exact", pairs, count, k, n, dtype)
    args = rq.F8Rows(x, xs), rq.F8Weight(w, ws), g.offsets, pairs
    want = rq.grouped_gemm_f8(*args, y_index=g.order)
    got = rq.grouped_gemm_f8(*args, y_index=g.order, dtype=dtype, exact=True)
    assert got.dtype == dtype and torch.equal(got, want.to(dtype))


@pytest.mark.parametrize("rows", [20, 300, 3000])
def test_grouped_a_row_twice(rq, rows):
    """A source that many places name; a destination that two places name holds one of their results."""
    x, xs, w, ws = (t.to(DEV) for t in _case(rows, 256, 140, rows, 2))
    offsets = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=DEV)
    xr, weight = rq.F8Rows(x, xs), rq.F8Weight(w, ws)
    same = torch.full((rows,), 3, dtype=torch.int32, device=DEV)
    y = rq.grouped_gemm_f8(xr, weight, offsets, rows, x_index=same)
    for e in range(2):
        at = torch.arange(int(offsets[e]), int(offsets[e + 1]), device=DEV)
        _check_product(x[3:4].repeat(at.numel(), 1), xs[3:4].repeat(at.numel(), 1), w[e], ws[e], y[at])
    twice = torch.arange(rows, dtype=torch.int32, device=DEV) // 2
    z = torch.full((rows, 140), 7.0, device=DEV)
    rq.grouped_gemm_f8(xr, weight, offsets, rows, y_index=twice, out=z)
    each = rq.grouped_gemm_f8(xr, weight, offsets, rows)
    for d in range((rows + 1) // 2):
        named = each[2 * d:2 * d + 2]
        assert any(torch.equal(z[d], r) for r in named) or all(((z[d] == r) | (z[d] == named[0])).all() for r in named)
    assert (z[(rows + 1) // 2:] == 7.0).all()


@pytest.mark.parametrize("how", ["one", "first", "none"])
@pytest.mark.parametrize("rows", [3, 90, 700])
def test_grouped_uneven(rq, rows, how):
    """All rows in one group, in the first, in none."""
    x, xs, w, ws = _case(rows, 384, 260, rows, 5)
    ids = torch.full((rows,), {"one": 4, "first": 0, "none": -1}[how], dtype=torch.int32)
    for side in ("gate", "down"):
        y, g = _run_grouped(rq, x, xs, w, ws, ids, 1, side, F32)
        _check_grouped(x, xs, w, ws, ids, 1, side, y, g)


@pytest.mark.parametrize("rows", [10, 200, 900])
def test_grouped_indexes_out_of_range(rq, rows):
    """Places with an index that names no row leave y as it was; offsets that do not rise, or lead past the rows, read
    and write nothing else."""
    x, xs, w, ws = _case(rows, 256, 200, rows, 3)
    weight, xr = rq.F8Weight(w.to(DEV), ws.to(DEV)), rq.F8Rows(x.to(DEV), xs.to(DEV))
    third = rows // 3
    offsets = torch.tensor([0, third, 2 * third, rows], dtype=torch.int32)
    idx = torch.arange(rows, dtype=torch.int32)
    idx[::3] = -1
    idx[1::3] = rows
    idx[4] = -(1 << 31)
    for kind in ("x", "y"):
        y = torch.full((rows, 200), 7.0, device=DEV)
        more = {"x_index": idx.to(DEV)} if kind == "x" else {"y_index": idx.to(DEV)}
        rq.grouped_gemm_f8(xr, weight, offsets.to(DEV), rows, out=y, **more)
        good = (idx >= 0) & (idx < rows)
        for e in range(3):
            at = torch.arange(int(offsets[e]), int(offsets[e + 1]))
            at = at[good[at]]
            _check_product(x[at], xs[at], w[e], ws[e], y[at.to(DEV)])
        assert (y[(~good).to(DEV)] == 7.0).all()
    for bad in ([0, rows, third, rows], [5, 2, 1, 0], [-7, third, rows + 50, 1 << 30], [rows, rows, rows, rows]):
        y = torch.full((rows + 4, 200), 7.0, device=DEV)
        rq.grouped_gemm_f8(xr, weight, torch.tensor(bad, dtype=torch.int32, device=DEV), rows, out=y)
        assert (y[rows:] == 7.0).all()


@pytest.mark.parametrize("rows", [6, 250])
def test_grouped_2d_weight_and_new_output(rq, rows):
    x, xs, w, ws = _case(rows, 512, 130, 1)
    offsets = torch.tensor([0, rows - 2], dtype=torch.int32, device=DEV)
    y = rq.grouped_gemm_f8(rq.F8Rows(x.to(DEV), xs.to(DEV)), rq.F8Weight(w.to(DEV), ws.to(DEV)), offsets, rows, dtype=F16)
    assert y.dtype == F16
    _check_product(x[:-2], xs[:-2], w, ws, y[:-2])
    assert not y[-2:].any()


def test_nothing_to_do(rq):
    """No rows: nothing is read or written."""
    none = rq.F8Rows(torch.empty(0, 256, dtype=F8, device=DEV), torch.empty(0, 2, device=DEV))
    x, xs, w, ws = _case(4, 256, 64, 1, 2)
    weight = rq.F8Weight(w.to(DEV), ws.to(DEV))
    assert rq.quantize_f8(torch.empty(0, 256, device=DEV)).codes.shape == (0, 256)
    assert rq.silu_and_mul_f8(torch.empty(0, 256, device=DEV), torch.empty(0, 256, device=DEV)).scales.shape == (0, 2)
    assert rq.add_rmsnorm_f8(torch.empty(0, 256, device=DEV), None, torch.ones(256, device=DEV), 1e-6)[0].codes.numel() == 0
    assert rq.gemm_f8(none, rq.F8Weight(w[0].to(DEV), ws[0].to(DEV))).shape == (0, 64)
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert rq.grouped_gemm_f8(none, weight, zero, 0).shape == (0, 64)
    y = torch.full((4, 64), 7.0, device=DEV)
    rq.grouped_gemm_f8(rq.F8Rows(x.to(DEV), xs.to(DEV)), weight, zero, 4, out=y)
    assert (y == 7.0).all()


# ------------------------------------------------------------------ as they are used

def _layer_weights(hidden, ffn, seed, count=None):
    g = _gen(seed)
    made = []
    for n, k in ((2 * ffn, hidden), (hidden, ffn)):
        shape = (n, k) if count is None else (count, n, k)
        w = torch.randn(*shape, generator=g)
        made.append((w.mul_(100).clamp_(-448, 448).to(F8),
                     (torch.rand(*(shape[:-2] + (_blocks(n), _blocks(k))), generator=g) + 0.5) / (100 * k ** 0.5)))
    return made


def _layer(rq, x, residual, norm, weights, eps=1e-5):
    """norm with the residual's addition -> gate and up in one product -> SiLU -> down, all in 8 bits."""
    act, total, _ = rq.add_rmsnorm_f8(x, residual, norm, eps)
    both = rq.gemm_f8(act, weights[0], dtype=x.dtype)
    ffn = both.shape[1] // 2
    inner = rq.silu_and_mul_f8(both[:, :ffn], both[:, ffn:])
    return rq.gemm_f8(inner, weights[1], dtype=x.dtype), total, act, both, inner


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,hidden,ffn", [(1, 512, 640), (19, 384, 300), (160, 1024, 1000)])
def test_layer(rq, rows, hidden, ffn, dtype):
    """An FFN: each step against its definition on what the step before it gave."""
    x, r = _values(rows, hidden, dtype, rows, 0.3), _values(rows, hidden, dtype, rows + 1, 0.3)
    norm = torch.rand(hidden, generator=_gen(2)) + 0.5
    (gu, gus), (dn, dns) = _layer_weights(hidden, ffn, 3)
    weights = [rq.F8Weight(gu.to(DEV), gus.to(DEV)), rq.F8Weight(dn.to(DEV), dns.to(DEV))]
    y, total, act, both, inner = _layer(rq, x.to(DEV), r.to(DEV), norm.to(DEV), weights)
    _check_norm(x, r, norm, 1e-5, act, total, None)
    _check_product(act.codes.cpu(), act.scales.cpu(), gu, gus, both)
    b = both.cpu().double()
    g, u = b[:, :ffn], b[:, ffn:]
    _check_codes(inner.codes, inner.scales, g * torch.sigmoid(g) * u, 2.0 ** -20)
    _check_product(inner.codes.cpu(), inner.scales.cpu(), dn, dns, y)


@pytest.mark.parametrize("tokens,count,top_k,hidden,ffn", [(1, 16, 4, 512, 256), (21, 6, 2, 384, 200), (260, 4, 2, 512, 384)])
def test_expert_layer(rq, tokens, count, top_k, hidden, ffn):
    """Experts: routed on the device, grouped, gate and up, SiLU, down back into the pairs' order."""
    logits = torch.randn(tokens, count, generator=_gen(1))
    x = _values(tokens, hidden, BF16, 2, 0.3)
    (gu, gus), (dn, dns) = _layer_weights(hidden, ffn, 3, count)
    wg, wd = rq.F8Weight(gu.to(DEV), gus.to(DEV)), rq.F8Weight(dn.to(DEV), dns.to(DEV))
    ids, _ = rq.moe_route_device(logits.to(DEV), tokens, count, top_k, True, 1.0)
    pairs = tokens * top_k
    groups = rq.group_rows(ids.reshape(-1), count)
    act = rq.quantize_f8(x.to(DEV))
    both = rq.grouped_gemm_f8(act, wg, groups.offsets, pairs, x_index=groups.order, x_div=top_k, dtype=BF16)
    inner = rq.silu_and_mul_f8(both[:, :ffn], both[:, ffn:])
    y = rq.grouped_gemm_f8(inner, wd, groups.offsets, pairs, y_index=groups.order)
    _check_codes(act.codes, act.scales, x.double(), 0.0)
    which = ids.reshape(-1).cpu().long()
    order = groups.order.cpu().long()
    for p in range(pairs):
        pair = int(order[p])
        e, t = int(which[pair]), pair // top_k
        _check_product(act.codes[t:t + 1].cpu(), act.scales[t:t + 1].cpu(), gu[e], gus[e], both[p:p + 1])
        _check_product(inner.codes[p:p + 1].cpu(), inner.scales[p:p + 1].cpu(), dn[e], dns[e], y[pair:pair + 1])


@pytest.mark.parametrize("rows", [1, 24, 200, 800])
def test_captured_and_replayed(rq, rows):
    """A layer and an expert layer in a graph: replays follow new inputs, with eager work between them."""
    hidden, ffn, count = 512, 384, 4
    (gu, gus), (dn, dns) = _layer_weights(hidden, ffn, 3)
    weights = [rq.F8Weight(gu.to(DEV), gus.to(DEV)), rq.F8Weight(dn.to(DEV), dns.to(DEV))]
    (eg, egs), _ = _layer_weights(hidden, ffn, 4, count)
    stack = rq.F8Weight(eg.to(DEV), egs.to(DEV))
    norm = torch.ones(hidden, device=DEV)
    x, r = torch.empty(rows, hidden, device=DEV), torch.empty(rows, hidden, device=DEV)
    ids = torch.empty(rows, dtype=torch.int32, device=DEV)

    def step():
        y, total, act, _, _ = _layer(rq, x, r, norm, weights)
        g = rq.group_rows(ids, count)
        z = rq.grouped_gemm_f8(act, stack, g.offsets, rows, x_index=g.order)
        return y, total, z

    def inputs(seed):
        x.copy_(_values(rows, hidden, F32, seed, 0.3))
        r.copy_(_values(rows, hidden, F32, seed + 1, 0.3))
        ids.copy_(torch.from_numpy(np.random.default_rng(seed).integers(-1, count, rows).astype(np.int32)))

    inputs(1)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 5, 9, 5):
        inputs(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("rows,k,n,dtype", [(1, 4099, 500, BF16), (300, 645, 531, F16), (333, 2099, 4099, BF16), (130, 4096, 700, F16),
                                            (250, 1040, 3900, BF16), (500, 784, 3100, F16), (2048, 640, 4000, BF16)])
def test_products_captured(rq, rows, k, n, dtype, exact):
    """Products in a graph, dense and grouped, aligned and not: replays follow new inputs, with eager work between them."""
    x, xs, w, ws = (t.to(DEV) for t in _case(rows, k, n, rows + k, 2))
    xr, weight, stack = rq.F8Rows(x, xs), rq.F8Weight(w[0], ws[0]), rq.F8Weight(w, ws)
    offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=DEV)

    def step():
        return (rq.gemm_f8(xr, weight, dtype=dtype, exact=exact),
                rq.grouped_gemm_f8(xr, stack, offsets, rows, dtype=dtype, exact=exact))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3, 1):
        other = _case(rows, k, 1, seed)
        x.copy_(other[0].to(DEV))
        xs.copy_(other[1].to(DEV))
        offsets[1] = seed * rows // 7
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_other_stream(rq):
    """Work goes on the caller's current stream."""
    x, xs, w, ws = _case(300, 1024, 512, 1)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        weight = rq.F8Weight(w.to(DEV), ws.to(DEV))
        v = _values(300, 1024, F32, 2, 0.3).to(DEV)
        torch.cuda._sleep(20_000_000)
        v += 1.0
        rows = rq.quantize_f8(v)
        y = rq.gemm_f8(rows, weight)
    s.synchronize()
    _check_codes(rows.codes, rows.scales, v.cpu().double(), 0.0)
    _check_product(rows.codes.cpu(), rows.scales.cpu(), w, ws, y)


def test_two_streams_at_once(rq):
    """Calls on two streams share nothing."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    work = []
    for i, (rows, n) in enumerate(((40, 2048), (500, 1024))):
        x, xs, w, ws = _case(rows, 2048, n, i)
        work.append((rq.F8Rows(x.to(DEV), xs.to(DEV)), rq.F8Weight(w.to(DEV), ws.to(DEV))))
    want = [rq.gemm_f8(*p) for p in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(rq.gemm_f8(*work[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i]) for t in got[i])


def test_threads(rq):
    """Calls of four host threads at once, a stream each."""
    import threading

    sizes = [(1, 1024, 640), (40, 2048, 512), (130, 1536, 1024), (300, 645, 333)]
    cases = [tuple(t.to(DEV) for t in _case(rows, k, n, rows)) for rows, k, n in sizes]
    values = [torch.randn(rows, k, generator=_gen(rows)).to(DEV) for rows, k, _ in sizes]
    want = [(rq.gemm_f8(rq.F8Rows(x, xs), rq.F8Weight(w, ws)), rq.quantize_f8(v)) for (x, xs, w, ws), v in zip(cases, values)]
    torch.cuda.synchronize()
    right = []

    def work(i):
        (x, xs, w, ws), (y, q) = cases[i], want[i]
        rows, weight = rq.F8Rows(x, xs), rq.F8Weight(w, ws)
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got, codes = rq.gemm_f8(rows, weight), rq.quantize_f8(values[i])
                torch.cuda.current_stream().synchronize()
                if (torch.equal(got, y) and torch.equal(codes.codes.view(torch.uint8), q.codes.view(torch.uint8))
                        and torch.equal(codes.scales, q.scales)):
                    right.append(i)

    _say("threads")
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(right) == 20 * len(sizes)


@pytest.mark.parametrize("rows,k,n", [(1, 4096, 4096), (30, 2048, 1024), (100, 4096, 512), (700, 1024, 1024), (1500, 2048, 2048)])
def test_same_results_every_time(rq, rows, k, n):
    x, xs, w, ws = _case(rows, k, n, 2)
    xr, weight = rq.F8Rows(x.to(DEV), xs.to(DEV)), rq.F8Weight(w.to(DEV), ws.to(DEV))
    first = rq.gemm_f8(xr, weight)
    for _ in range(10):
        assert torch.equal(rq.gemm_f8(xr, weight), first)

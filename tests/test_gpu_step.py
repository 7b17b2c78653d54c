"""The operators of a token's step against 64 bits: norms with their residual,
rows in 8 bits and their product, rotary positions, and a run of all of them around
the cache."""
import numpy as np
import pytest

import omnivoice_amd as ov

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150}  # half the smallest step


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def spread(t, extra):
    """The same values in rows `extra` elements further apart."""
    wide = torch.full((t.shape[0], t.shape[1] + extra), 7.0).to(t.dtype).cuda()
    wide[:, :t.shape[1]] = t.cuda()
    return wide[:, :t.shape[1]], wide


def values(codes, scales):
    return codes.view(torch.float8_e4m3fn).float().cpu().double() * \
        scales.cpu().double()[:, None]


def scales_of(y):
    """The smallest power of two, 2^-100 or more, that takes amax into 448: exact."""
    m, e = np.frexp(np.abs(y).max(-1))
    return np.where(m > 0, np.ldexp(1.0, np.maximum(e - 9 + (m > 0.875), -100)), 2.0 ** -100)


def check_codes(codes, scales, y, slack):
    """Codes are off by half a step: 2^-4 of the value, or 2^-10 of the scale where
    it is below e4m3's normal numbers; `slack` is the relative error of what they
    stand for."""
    y = y.double().numpy()
    want = scales_of(y)
    np.testing.assert_array_equal(scales.cpu().double().numpy(), want)
    got = values(codes, scales).numpy()
    bound = np.maximum(np.abs(y) * 2.0 ** -4, want[:, None] * 2.0 ** -10) + slack * np.abs(y)
    assert (np.abs(got - y) <= bound).all(), np.abs(got - y).max()


# ------------------------------------------------------------------ norm

# The squares' sum: eight in a row, eight such, six levels of lanes and sixteen waves,
# each 2^-24 of a sum of positive terms: 38; halved by the root; the root, the mean and
# two products another 6.
NORM = 26 * 2.0 ** -24


def norm_of(x, residual, weight, eps):
    """(total as stored, y in 64 bits)."""
    s, total = x.float(), None
    if residual is not None:
        total = (s + residual.float()).to(residual.dtype)
        s = total
    s = s.double()
    return total, weight.double() * s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)


def run_norm(x, weight, residual, out, eps, extra=0):
    rows, width = x.shape
    xs, _ = spread(x, extra)
    rs = ts = scales = None
    if residual is not None:
        rs, _ = spread(residual, 2 * extra)
        ts, t_wide = spread(torch.zeros_like(residual), extra)
    if out == "e4m3":
        to, o_wide = spread(torch.zeros(rows, width, dtype=torch.uint8), extra)
        scales = torch.zeros(rows, device="cuda")
    else:
        to, o_wide = spread(torch.zeros(rows, width, dtype=TYPES[out]), extra)
    ov.op_add_rmsnorm(xs, weight.cuda(), to, eps, residual=rs, total=ts, scales=scales)
    assert (o_wide[:, width:].float() == 7).all()
    if residual is not None:
        assert (t_wide[:, width:].float() == 7).all()
        assert torch.equal(rs.cpu(), residual)
    return None if ts is None else ts.cpu(), to, scales


def check_norm(x, weight, residual, out, eps, extra=0):
    total, to, scales = run_norm(x, weight, residual, out, eps, extra)
    want_total, y = norm_of(x, residual, weight, eps)
    if residual is not None:
        assert torch.equal(total, want_total)
    if out == "e4m3":
        check_codes(to, scales, y, NORM)
    else:
        off = (to.cpu().double() - y).abs()
        assert (off <= y.abs() * (NORM + HALF_STEP[out]) + TINY[out]).all(), (off / y.abs()).max()


@pytest.mark.parametrize("x,residual,out", [
    ("bf16", "f32", "e4m3"), ("bf16", "bf16", "bf16"), ("f16", "f16", "e4m3"),
    ("f16", "", "f16"), ("f32", "f32", "f16"), ("f32", "", "e4m3"), ("f16", "f32", "f32"),
    ("bf16", "", "f32"), ("f32", "f32", "bf16")])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 8), (5, 9), (70, 64), (3, 100),
                                        (9, 1000), (6, 1024), (5, 1025), (3, 2049), (2, 5003),
                                        (3, 8192), (2, 8200), (1, 40001), (2, 65536)])
def test_norm(x, residual, out, rows, width):
    a = normal(width, rows, width).to(TYPES[x])
    r = (normal(width + 1, rows, width) * 3).to(TYPES[residual]) if residual else None
    check_norm(a, 1 + 0.3 * normal(width + 2, width), r, out, 1e-6, extra=width % 5)


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1e18, 1e25, 3e37])
def test_norm_of_any_loudness(scale):
    """Squares that pass float32's range, or vanish beside epsilon."""
    x = normal(1, 6, 700) * scale
    check_norm(x, 1 + 0.1 * normal(2, 700), None, "f32", 1e-6)
    check_norm(x, 1 + 0.1 * normal(2, 700), torch.zeros(6, 700), "e4m3", 1e-6)


def test_norm_beside_a_scale_border():
    """Rows whose largest value is 448 times a power of two to a few parts in 2^24: the
    scale is the formula's, not that of its rounding."""
    width, rows = 1024, 4000
    x = normal(3, rows, width)
    x[:, 17] = 30.0
    y = norm_of(x, None, torch.ones(width), 1e-6)[1]
    aim = 1.75 * 2.0 ** 4 * (1 + torch.randint(-6, 7, (rows,), generator=torch.Generator()
                                               .manual_seed(4)).double() * 2.0 ** -25)
    weight = torch.ones(width)
    for r in range(0, rows, 400):  # one weight is one row's aim; the others come as they are
        weight[17] = float(aim[r] / y[r, 17])
        check_norm(x[r:r + 400], weight, None, "e4m3", 1e-6)


def test_norm_of_zeros_infinities_and_nan():
    x = normal(5, 5, 200)
    x[1] = 0.0
    x[2, 3] = np.inf
    x[3, 199] = np.nan
    scales = torch.zeros(5, device="cuda")
    codes = torch.full((5, 200), 9, dtype=torch.uint8, device="cuda")
    w = torch.ones(200, device="cuda")
    ov.op_add_rmsnorm(x.cuda(), w, codes, 1e-6, scales=scales)
    s = scales.cpu()
    assert s[1] == 2.0 ** -100 and (codes[1] == 0).all()
    assert torch.isnan(s[2:4]).all() and (codes[2:4] == 0).all()
    keep = [0, 4]
    check_codes(codes[keep], scales[keep], norm_of(x[keep], None, torch.ones(200), 1e-6)[1], NORM)


def test_norm_in_place():
    x = normal(6, 40, 520).half()
    r = normal(7, 40, 520)
    w = 1 + 0.2 * normal(8, 520)
    total, y = norm_of(x, r, w, 1e-5)
    xd, rd = x.cuda(), r.cuda()
    ov.op_add_rmsnorm(xd, w.cuda(), xd, 1e-5, residual=rd)  # total into the residual, out into x
    assert torch.equal(rd.cpu(), total)
    off = (xd.cpu().double() - y).abs()
    assert (off <= y.abs() * (NORM + 2.0 ** -11) + 2.0 ** -25).all()
    x2, r2 = x.cuda(), x.flip(0).cuda()
    total, y = norm_of(x, x.flip(0), w, 1e-5)
    ov.op_add_rmsnorm(x2, w.cuda(), r2, 1e-5, residual=r2, total=x2)  # into each other
    assert torch.equal(x2.cpu(), total)
    assert ((r2.cpu().double() - y).abs() <= y.abs() * (NORM + 2.0 ** -11) + 2.0 ** -25).all()


def test_rows_past_32_bit_offsets():
    rows, width = (1 << 22) - 3, 600
    x = torch.empty(rows, width, dtype=torch.float16, device="cuda")
    x[:8] = normal(9, 8, width).half().cuda()
    x[-8:] = normal(10, 8, width).half().cuda()
    x[8:-8] = 1.0
    w = 1 + 0.1 * normal(11, width)
    out = torch.zeros(rows, width, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows, device="cuda")
    ov.op_add_rmsnorm(x, w.cuda(), out, 1e-6, scales=scales)
    for part in (slice(0, 8), slice(rows - 8, rows)):
        check_codes(out[part], scales[part], norm_of(x[part].cpu(), None, w, 1e-6)[1], NORM)
    ov.op_quantize8(x, out, scales)
    for part in (slice(0, 8), slice(rows - 8, rows)):
        check_codes(out[part], scales[part], x[part].cpu(), 0.0)


# ------------------------------------------------------------------ quantize

# e^-g = 2^(-g log2 e): the product's rounding and the constant's are 1.5 |g| 2^-24 of it,
# with |g| under 21 here, the power itself 2; the sum, the quotient and the product 2 more
# each.
GATE = 40 * 2.0 ** -24


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 1), (2, 5), (33, 16), (5, 1023), (7, 1024), (2, 2050),
                                        (580, 4096), (3, 9001), (1, 65536)])
def test_quantize(kind, gated, rows, width):
    x = (normal(width, rows, width) * torch.exp(2 * normal(1, rows, 1))).to(TYPES[kind])
    gate = (normal(width + 1, rows, width) * 4).to(TYPES[kind]) if gated else None
    xs, _ = spread(x, 3)
    codes, wide = spread(torch.zeros(rows, width, dtype=torch.uint8), 5)
    scales = torch.zeros(rows, device="cuda")
    ov.op_quantize8(xs, codes, scales, gate=spread(gate, 1)[0] if gated else None)
    y = x.double()
    if gated:
        y = y * gate.double() * torch.sigmoid(gate.double())
    check_codes(codes, scales, y, GATE if gated else 0.0)
    assert (wide[:, width:] == 7).all()


def test_quantize_borders_and_lost_rows():
    """448 exactly, the next number above, the largest float32, denormal numbers, zero;
    rows with an infinity or a NaN."""
    rows = [448.0, np.nextafter(np.float32(448), np.float32(500)), 1.75, 1.7500001, 3.4028234e38,
            1e-40, 0.0, 2.0 ** -92 * 1.75, 2.0 ** -93, -448.0]
    x = torch.zeros(len(rows) + 3, 40)
    for i, v in enumerate(rows):
        x[i, i * 3] = float(v)
    x[-3, 0], x[-2, 39], x[-1, 7] = np.inf, np.nan, -np.inf
    codes = torch.full(x.shape, 1, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(len(x), device="cuda")
    ov.op_quantize8(x.cuda(), codes, scales)
    n = len(rows)
    check_codes(codes[:n], scales[:n], x[:n], 0.0)
    assert torch.isnan(scales[n:]).all() and (codes[n:] == 0).all()


def test_gate_of_any_size():
    g = torch.tensor([[-np.inf, -1e30, -200.0, -89.0, -1.0, 0.0, 1.0, 89.0, 1e30]])
    x = torch.ones(1, 9)
    codes = torch.zeros(1, 8, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(1, device="cuda")
    ov.op_quantize8(x[:, 1:].contiguous().cuda(), codes, scales, gate=g[:, 1:].contiguous().cuda())
    y = (g * torch.sigmoid(g.double()))[:, 1:]
    check_codes(codes, scales, y, 0.01)
    ov.op_quantize8(x[:, :8].contiguous().cuda(), codes, scales, gate=g[:, :8].contiguous().cuda())
    assert torch.isnan(scales).all()  # -inf * 0


# Gates down to -88 and so the error of their power, which is the product's: (1.5 |g| + 8) 2^-24.
DEEP_GATE = (1.5 * 88 + 8) * 2.0 ** -24


@pytest.mark.parametrize("low,high", [(-24.0, -8.0), (-64.0, -24.0), (-87.0, -64.0)])
def test_gates_beside_a_scale_border(low, high):
    """Rows whose largest product is 448 times a power of two to a hundred parts in 2^24, by
    gates that make its rounding that large: the scale is the formula's."""
    rows, width = 20000, 24
    gen = torch.Generator().manual_seed(50)
    g = torch.zeros(rows, width)
    g[:, 5] = low + (high - low) * torch.rand(rows, generator=gen)
    x = torch.zeros(rows, width)
    s = g[:, 5].double() * torch.sigmoid(g[:, 5].double())
    aim = -1.75 * (1 + torch.randint(-100, 101, (rows,), generator=gen).double() * 2.0 ** -24)
    x[:, 5] = (aim / s).float()
    codes = torch.zeros(rows, width, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows, device="cuda")
    ov.op_quantize8(x.cuda(), codes, scales, gate=g.cuda())
    check_codes(codes, scales, x.double() * g.double() * torch.sigmoid(g.double()), DEEP_GATE)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_deep_gates_of_loud_rows(kind):
    """Gates whose power leaves float32's range beside values that bring the product back."""
    g = torch.tensor([-64.0, -70.0, -80.0, -87.0, -88.5, -89.0, -95.0, -103.0, -104.0, -120.0,
                      -150.0, -155.0, -160.0])
    x = torch.tensor([1.0, 1e10, -1e20, 3e35, 1e38, 3.3e38, -3.3e38])
    gate = g[:, None, None].expand(-1, len(x), 11).reshape(-1, 11).clone()
    value = x[None, :, None].expand(len(g), -1, 11).reshape(-1, 11).clone()
    gate[:, 3:] += normal(51, *gate[:, 3:].shape)
    value[:, ::2] *= 0.9
    value = value.clamp(-65504, 65504) if kind == "f16" else value
    gate, value = gate.to(TYPES[kind]), value.to(TYPES[kind])
    codes = torch.zeros(gate.shape, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(len(gate), device="cuda")
    ov.op_quantize8(value.cuda(), codes, scales, gate=gate.cuda())
    d = gate.double()
    check_codes(codes, scales, value.double() * d * torch.exp(d) / (1 + torch.exp(d)), DEEP_GATE)


def test_gates_past_every_power():
    """Nothing is left of what is finite; an infinite value or gate is the row's."""
    g = torch.tensor([[-200.0], [-299.0], [-301.0], [-3e38], [-100.0], [-np.inf], [-100.0]])
    x = torch.tensor([[3e38], [-3e38], [3e38], [3e38], [np.inf], [1.0], [np.nan]])
    codes = torch.full((7, 1), 9, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(7, device="cuda")
    ov.op_quantize8(x.cuda(), codes, scales, gate=g.cuda())
    assert (codes[:, 0].cpu() & 0x7F == 0).all()
    assert (scales[:4].cpu() == 2.0 ** -100).all() and torch.isnan(scales[4:]).all()


# ------------------------------------------------------------------ product

def whole_codes(seed, rows, width, most=8):
    """Whole numbers as e4m3: their products' sums are exact in float32."""
    x = torch.randint(-most, most + 1, (rows, width), generator=torch.Generator()
                      .manual_seed(seed)).float()
    return x, x.to(torch.float8_e4m3fn)


def powers(seed, n):
    e = torch.randint(-6, 7, (n,), generator=torch.Generator().manual_seed(seed))
    return torch.exp2(e.float())


SHAPES = [(1, 16, 1), (1, 1024, 4096), (2, 48, 17), (16, 1024, 100), (17, 160, 64),
          (31, 2064, 33), (64, 4096, 1000), (65, 128, 256), (100, 400, 300), (128, 1024, 1024),
          (129, 144, 129), (255, 640, 511), (256, 512, 256), (300, 1024, 2049),
          (580, 2048, 1024), (700, 8208, 520), (1024, 272, 1024), (2050, 1040, 600), (5, 65536, 40)]


@pytest.mark.parametrize("rows,width,out", SHAPES)
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_product_of_whole_numbers(rows, width, out, kind):
    """Every sum is a whole number under 2^24 (64 * 65536 = 2^22): whatever the order, the
    result is the exact one, rounded once."""
    a, x = whole_codes(rows, rows, width)
    b, w = whole_codes(out + 1, out, width)
    xs, ws = powers(3, rows), powers(4, out) * 2.0 ** -6
    wide = torch.full((rows, width + 32), 0x7F, dtype=torch.uint8)  # NaN beside the rows
    wide[:, :width] = x.view(torch.uint8)
    y, y_wide = spread(torch.zeros(rows, out, dtype=TYPES[kind]), 3)
    ov.op_linear8(wide.cuda()[:, :width], xs.cuda(), w.cuda(), ws.cuda(), y)
    want = (a.double() @ b.double().t()) * xs.double()[:, None] * ws.double()
    assert torch.equal(y.cpu(), want.to(TYPES[kind]))
    assert (y_wide[:, out:].float() == 7).all()


@pytest.mark.parametrize("rows,width,out", [(3, 1024, 200), (40, 4096, 64), (200, 1024, 300),
                                            (600, 2048, 520)])
def test_product_of_any_codes(rows, width, out):
    """Sums of `width` terms, each addition off by 2^-23 of the terms' sizes at most."""
    x, w = (normal(s, n, width).to(torch.float8_e4m3fn) for s, n in ((1, rows), (2, out)))
    xs, ws = torch.rand(rows) + 0.5, torch.rand(out) + 0.5
    y = torch.zeros(rows, out, device="cuda")
    ov.op_linear8(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), y)
    a = x.double() * xs.double()[:, None]
    b = w.double() * ws.double()[:, None]
    bound = (width * 2.0 ** -23 + 2.0 ** -22) * (a.abs() @ b.abs().t())
    assert ((y.cpu().double() - a @ b.t()).abs() <= bound).all()
    # The sums are float32's: the error of a case as a whole is far below that of 16 bits.
    rel = (y.cpu().double() - a @ b.t()).norm() / (a @ b.t()).norm()
    assert rel < 2.0 ** -16


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,width,out", [(1, 1024, 48), (16, 1024, 4096), (17, 1040, 33),
                                            (32, 1040, 900), (64, 1024, 300)])
def test_product_of_few_rows_keeps_small_products(rows, width, out, kind):
    """Ones beside products of 448 * 448 that cancel one another, eight codes in a row: whole
    numbers, whose sums stay under 2^24 (65 * 200704), so that nothing may be lost. 64 rows
    of 300 columns are too few tiles for those, and go the same way."""
    a, b = torch.ones(rows, width), torch.ones(out, width)
    for r in range(rows):
        a[r, r % 8::16], a[r, r % 8 + 8::16] = 448.0, -448.0
    for k in range(8):
        b[k::8, k::8] = 448.0
    x, w = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
    y = torch.zeros(rows, out, dtype=TYPES[kind], device="cuda")
    one = torch.ones(max(rows, out), device="cuda")
    ov.op_linear8(x.cuda(), one[:rows].contiguous(), w.cuda(), one[:out].contiguous(), y)
    assert torch.equal(y.cpu(), (a.double() @ b.double().t()).to(TYPES[kind]))


@pytest.mark.parametrize("rows", [4, 40, 300])
def test_product_of_lost_rows_and_far_scales(rows):
    """A NaN scale or code is its own row's, a far scale no overflow."""
    a, x = whole_codes(1, rows, 256)
    b, w = whole_codes(2, 90, 256)
    xs, ws = torch.ones(rows), torch.ones(90)
    xs[1], ws[5] = np.nan, np.nan
    xs[2], ws[7] = 2.0 ** -100, 2.0 ** 100
    x.view(torch.uint8)[3, 100] = 0x7F
    y = torch.zeros(rows, 90, device="cuda")
    ov.op_linear8(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), y)
    want = (a.double() @ b.double().t()) * xs.double()[:, None] * ws.double()
    want[3] = np.nan
    assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(y.cpu()), torch.nan_to_num(want.float()))


def test_product_past_32_bit_offsets():
    rows, out, width = 70001, 32768, 16
    a, x = whole_codes(1, rows, width)
    b, w = whole_codes(2, out, width)
    y = torch.zeros(rows, out, dtype=torch.float16, device="cuda")
    one = torch.ones(rows, device="cuda")
    ov.op_linear8(x.cuda(), one, w.cuda(), one[:out], y)
    for part in (slice(0, 5), slice(65530, 65540), slice(rows - 5, rows)):
        assert torch.equal(y[part].cpu(), (a[part].double() @ b.double().t()).half())


# ------------------------------------------------------------------ rotary

def rotated(x, positions, frequencies, interleaved, magnitude, weight, eps):
    """In 64 bits, and the size that an element's error goes by."""
    y = x.double()
    if weight is not None:
        y = weight.double() * y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
    n = 2 * len(frequencies)
    angle = positions.double()[:, None, None] * frequencies.double()
    c, s = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    z = y.clone()
    if interleaved:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        z[..., 0:n:2], z[..., 1:n:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :n // 2], y[..., n // 2:n]
        z[..., :n // 2], z[..., n // 2:n] = a * c - b * s, b * c + a * s
    size = y.abs()
    both = (a.abs() + b.abs()) * max(1.0, abs(magnitude))
    if interleaved:
        size[..., 0:n:2] = size[..., 1:n:2] = both
    else:
        size[..., :n // 2] = size[..., n // 2:n] = both
    return z, size


# cos and sin to 2^-23 (a Taylor sum in float32, the angle's rounding), the magnitude's
# product, two products and a sum: 2^-21 of |a| + |b|. A norm's 26 * 2^-24 before it.
TURN = 2.0 ** -21


def check_rotary(got, x, positions, frequencies, interleaved, magnitude, weight, eps, kind):
    z, size = rotated(x, positions, frequencies, interleaved, magnitude, weight, eps)
    slack = TURN + (0 if weight is None else NORM)
    off = (got.cpu().double() - z).abs()
    bound = size * slack + z.abs() * HALF_STEP[kind] + TINY[kind]
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (64, 64), (80, 80), (80, 32),
                                        (96, 20), (256, 256), (2, 2), (6, 4), (512, 510),
                                        (128, 16), (48, 32)])
def test_rotary(kind, interleaved, dim, rotary):
    rows, heads, kv_heads = 13, 5, 2
    fused = normal(dim, rows, heads + 2 * kv_heads, dim).to(TYPES[kind])
    positions = torch.tensor([0, 1, 2, 77, 4095, 90000, 1 << 20, -5, 12345678, 3, (1 << 30) - 1,
                              -(1 << 30), 131071], dtype=torch.int32)
    f, _ = ov.rotary_frequencies(rotary, 1e4)
    f = torch.tensor(f)
    dev = fused.cuda()
    q, k = dev[:, :heads], dev[:, heads:heads + kv_heads]
    for normed in (False, True):
        wq, wk = (1 + 0.3 * normal(s, dim) if normed else None for s in (1, 2))
        magnitude = 1.25 if normed else 1.0
        q_out = torch.zeros(rows, heads, dim, dtype=TYPES[kind], device="cuda")
        k_out = torch.zeros(rows, kv_heads, dim, dtype=TYPES[kind], device="cuda")
        ov.op_rotary(q, q_out, k, k_out, f.cuda(), positions=positions.cuda(),
                     interleaved=interleaved, magnitude=magnitude,
                     q_norm=wq if wq is None else wq.cuda(),
                     k_norm=wk if wk is None else wk.cuda(), eps=1e-5)
        check_rotary(q_out, fused[:, :heads], positions, f, interleaved, magnitude, wq, 1e-5, kind)
        check_rotary(k_out, fused[:, heads:heads + kv_heads], positions, f, interleaved, magnitude,
                     wk, 1e-5, kind)
    assert torch.equal(dev.cpu(), fused)


@pytest.mark.parametrize("rows,heads", [(1, 1), (1, 24), (3, 7), (257, 3), (1000, 24)])
def test_rotary_in_place_of_one_tensor(rows, heads):
    """A fused row's heads, one norm for some of them, the values behind untouched."""
    fused = normal(rows, rows, heads + 2, 128).half()
    positions = torch.arange(rows, dtype=torch.int32) * 37
    f = torch.tensor(ov.rotary_frequencies(128)[0])
    dev = fused.cuda()
    ov.op_rotary(dev[:, :heads], dev[:, :heads], None, None, f.cuda(), positions=positions.cuda())
    check_rotary(dev[:, :heads], fused[:, :heads], positions, f, False, 1.0, None, 0, "f16")
    assert torch.equal(dev[:, heads:].cpu(), fused[:, heads:])


def test_rotary_one_norm_of_two():
    x = normal(1, 9, 6, 64)
    positions = torch.arange(9, dtype=torch.int32)
    f = torch.tensor(ov.rotary_frequencies(64)[0])
    w = 1 + 0.2 * normal(2, 64)
    for which in (0, 1):
        q, k = x[:, :4].cuda().contiguous(), x[:, 4:].cuda().contiguous()
        ov.op_rotary(q, q, k, k, f.cuda(), positions=positions.cuda(),
                     q_norm=w.cuda() if which == 0 else None,
                     k_norm=w.cuda() if which == 1 else None)
        check_rotary(q, x[:, :4], positions, f, False, 1.0, w if which == 0 else None, 1e-6, "f32")
        check_rotary(k, x[:, 4:], positions, f, False, 1.0, w if which == 1 else None, 1e-6, "f32")


def test_rotary_keeps_infinities_of_dims_that_stay():
    x = normal(1, 3, 2, 128)
    x[:, :, 100] = np.inf
    x[:, :, 101] = np.nan
    f = torch.tensor(ov.rotary_frequencies(64)[0])
    for interleaved in (False, True):
        out = torch.zeros(3, 2, 128, device="cuda")
        ov.op_rotary(x.cuda(), out, None, None, f.cuda(), interleaved=interleaved,
                     positions=torch.tensor([5, 0, 9], dtype=torch.int32).cuda())
        assert torch.equal(torch.nan_to_num(out.cpu()[:, :, 64:]), torch.nan_to_num(x[:, :, 64:]))
        assert torch.isfinite(out[:, :, :64]).all()


@pytest.mark.parametrize("count", [1, 3, 70, 300])
def test_rotary_by_sequences(count):
    """Positions of the sequences' tokens, as the cache places them; rows of nobody, in
    front, behind and of empty sequences' places, stay."""
    g = torch.Generator().manual_seed(count)
    new = torch.randint(0, 5, (count,), generator=g)
    new[0] = 3
    front, behind = 2, 3
    begins = torch.cat([torch.zeros(1), new.cumsum(0)]).int() + front
    lengths = (new + torch.randint(0, 5000, (count,), generator=g)).int()
    rows = int(begins[-1]) + behind
    positions = torch.zeros(rows, dtype=torch.int32)
    for i in range(count):
        a, b = int(begins[i]), int(begins[i + 1])
        positions[a:b] = torch.arange(int(lengths[i]) - (b - a), int(lengths[i])).int()
    x = normal(1, rows, 3, 64).half()
    f = torch.tensor(ov.rotary_frequencies(64)[0])
    seq = ov.KVSequences(torch.zeros(count, 1, dtype=torch.int32).cuda(), lengths.cuda(),
                         begins.cuda())
    out = torch.full((rows, 3, 64), 7.0, dtype=torch.float16, device="cuda")
    ov.op_rotary(x.cuda(), out, None, None, f.cuda(), sequences=seq)
    inside = slice(front, rows - behind)
    check_rotary(out[inside], x[inside], positions[inside], f, False, 1.0, None, 0, "f16")
    assert (out[:front] == 7).all() and (out[rows - behind:] == 7).all()
    other = torch.zeros(rows, 3, 64, dtype=torch.float16, device="cuda")
    ov.op_rotary(x.cuda(), other, None, None, f.cuda(), positions=positions.cuda())
    assert torch.equal(other[inside], out[inside])


def test_rotary_past_32_bit_offsets():
    rows = 600011
    x = torch.empty(rows, 32, 128, dtype=torch.float16, device="cuda")
    x.fill_(1.0)
    x[-4:] = normal(1, 4, 32, 128).half().cuda()
    positions = torch.arange(rows, dtype=torch.int32)
    f = torch.tensor(ov.rotary_frequencies(128)[0])
    held = x[-4:].cpu()
    ov.op_rotary(x, x, None, None, f.cuda(), positions=positions.cuda())
    check_rotary(x[-4:], held, positions[-4:], f, False, 1.0, None, 0, "f16")


# ------------------------------------------------------------------ together

class Layer:
    """A layer over the cache, and the same in 64 bits step by step: every operator's
    result is checked for the inputs that it had."""

    def __init__(self, seed, hidden=256, heads=4, kv_heads=2, inter=512, vocab=700):
        self.hidden, self.heads, self.kv_heads, self.inter = hidden, heads, kv_heads, inter
        self.w = {}
        for i, (name, out, width) in enumerate((
                ("qkv", (heads + 2 * kv_heads) * 128, hidden), ("o", hidden, heads * 128),
                ("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter),
                ("head", vocab, hidden))):
            raw = normal(seed + i, out, width) * width ** -0.5 * 2
            codes = torch.zeros(out, width, dtype=torch.float8_e4m3fn, device="cuda")
            scales = torch.zeros(out, device="cuda")
            ov.op_quantize8(raw.cuda(), codes, scales)
            self.w[name] = (codes, scales)
        self.norms = [(1 + 0.2 * normal(seed + 10 + i, hidden)).cuda() for i in range(3)]
        self.q_norm, self.k_norm = ((1 + 0.2 * normal(seed + 20 + i, 128)).cuda()
                                    for i in range(2))
        self.f = torch.tensor(ov.rotary_frequencies(128, 1e4, "parts", 4.0, 2048)[0]).cuda()
        self.magnitude = ov.rotary_frequencies(128, 1e4, "parts", 4.0, 2048)[1]

    def buffers(self, rows):
        def z(*shape, dtype=torch.bfloat16):
            return torch.zeros(*shape, dtype=dtype, device="cuda")
        b = dict(stream=z(rows, self.hidden, dtype=torch.float32), x=z(rows, self.hidden),
                 qkv=z(rows, self.heads + 2 * self.kv_heads, 128), att=z(rows, self.heads, 128),
                 gate=z(rows, self.inter), up=z(rows, self.inter),
                 logits=z(rows, self.w["head"][0].shape[0], dtype=torch.float32),
                 random=z(rows, dtype=torch.float32), tokens=z(rows, dtype=torch.int32),
                 logprob=z(rows, dtype=torch.float32), entropy=z(rows, dtype=torch.float32))
        for name, width in (("n", self.hidden), ("a", self.heads * 128), ("g", self.inter)):
            b[name] = z(rows, width, dtype=torch.uint8)
            b[name + "s"] = z(rows, dtype=torch.float32)
        return b

    def step(self, b, cache, seq, check=None):
        def product(name, x, y):
            ov.op_linear8(b[x], b[x + "s"], *self.w[name], y)
            if check is not None:
                a = values(b[x], b[x + "s"])
                w = values(*self.w[name])
                want = a @ w.t()
                room = (a.shape[1] + 2) * 2.0 ** -23 * (a.abs() @ w.abs().t())
                half = 2.0 ** -8 if y.dtype is torch.bfloat16 else 2.0 ** -24
                assert ((y.cpu().double() - want).abs() <= room + half * want.abs()).all(), name

        def norm(i, x):
            held = b["stream"].cpu().clone() if check is not None else None
            ov.op_add_rmsnorm(x, self.norms[i], b["n"], 1e-6, residual=b["stream"],
                              scales=b["ns"])
            if check is not None:
                total, y = norm_of(x.cpu(), held, self.norms[i].cpu(), 1e-6)
                assert torch.equal(b["stream"].cpu(), total)
                check_codes(b["n"], b["ns"], y, NORM)

        rows, h, kv = b["x"].shape[0], self.heads, self.kv_heads
        norm(0, b["x"])
        product("qkv", "n", b["qkv"].view(rows, -1))
        q, k, v = b["qkv"][:, :h], b["qkv"][:, h:h + kv], b["qkv"][:, h + kv:]
        held = b["qkv"].cpu().clone() if check is not None else None
        ov.op_rotary(q, q, k, k, self.f, sequences=seq, magnitude=self.magnitude,
                     q_norm=self.q_norm, k_norm=self.k_norm)
        if check is not None:
            for t, x, w in ((q, held[:, :h], self.q_norm), (k, held[:, h:h + kv], self.k_norm)):
                check_rotary(t, x, check, self.f.cpu(), False, self.magnitude, w.cpu(), 1e-6,
                             "bf16")
            assert torch.equal(v.cpu(), held[:, h + kv:])
        ov.op_cache_write(cache, seq, k, v)
        ov.op_cache_attention(cache, seq, q, b["att"], causal=True)
        ov.op_quantize8(b["att"].view(rows, -1), b["a"], b["as"])
        product("o", "a", b["x"])
        norm(1, b["x"])
        product("gate", "n", b["gate"])
        product("up", "n", b["up"])
        ov.op_quantize8(b["up"], b["g"], b["gs"], gate=b["gate"])
        if check is not None:
            g = b["gate"].cpu().double()
            check_codes(b["g"], b["gs"], b["up"].cpu().double() * g * torch.sigmoid(g), GATE)
        product("down", "g", b["x"])
        norm(2, b["x"])
        product("head", "n", b["logits"])
        ov.op_sample(b["logits"], b["random"], b["tokens"], temperature=0.8, top_k=40, top_p=0.95)
        ov.op_token_logprobs(b["logits"], b["tokens"], b["logprob"], b["entropy"])


def plan(lengths, new, width=16, block=32):
    tables = torch.arange(len(lengths) * width, dtype=torch.int32).view(len(lengths), width)
    begins = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32)
    return ov.KVSequences(tables.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(),
                          begins.cuda())


def positions_of(lengths, new):
    return torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, new)]).int()


def test_a_step_around_the_cache():
    """Prompts, then single tokens, each operator against 64 bits on the inputs it had."""
    layer = Layer(100)
    cache = ov.KVCache.empty(64, 2, 128, 32)
    for lengths, new in (([37, 5, 200], [37, 5, 200]), ([38, 6, 201], [1, 1, 1])):
        b = layer.buffers(sum(new))
        b["stream"].copy_(normal(1, *b["stream"].shape))
        b["random"].copy_(torch.rand(sum(new), generator=torch.Generator().manual_seed(2)))
        layer.step(b, cache, plan(lengths, new), check=positions_of(lengths, new))
        tokens = b["tokens"].cpu().long()
        assert ((tokens >= 0) & (tokens < 700)).all()
        # What was drawn is among the 40 best and rated as the logits say.
        z = b["logits"].cpu().double()
        assert ((z > z.gather(1, tokens[:, None])).sum(1) < 40).all()
        want = torch.log_softmax(z, -1).gather(1, tokens[:, None])[:, 0]
        assert ((b["logprob"].cpu().double() - want).abs() < 1e-4).all()


def test_a_captured_step_follows_its_arrays():
    """One graph of the whole step, replayed over growing sequences with eager work
    between, beside the same steps called one by one; on a stream of its own."""
    layer = Layer(200)
    lengths, new = [9, 30, 64, 1], [1, 1, 1, 1]
    caches = [ov.KVCache.empty(64, 2, 128, 32) for _ in range(2)]
    seqs = [plan(lengths, new) for _ in range(2)]
    sides = [layer.buffers(4) for _ in range(2)]
    for b, cache, seq in zip(sides, caches, seqs):  # warm up
        layer.step(b, cache, seq)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        layer.step(sides[0], caches[0], seqs[0])
    for t in range(5):
        for b, seq in zip(sides, seqs):
            b["stream"].copy_(normal(300 + t, 4, 256))
            b["x"].copy_(normal(400 + t, 4, 256))
            b["random"].copy_(torch.rand(4, generator=torch.Generator().manual_seed(t)))
            seq.lengths.add_(1)
        graph.replay()
        layer.step(sides[1], caches[1], seqs[1])
        torch.cuda.synchronize()
        for name in sides[0]:
            assert torch.equal(sides[0][name].view(torch.uint8), sides[1][name].view(torch.uint8)), \
                (t, name)
        assert torch.equal(caches[0].data, caches[1].data)


def test_streams():
    """Calls on two streams at once, in neither's way, and by a raw handle."""
    x = normal(1, 2000, 1024).half().cuda()
    w = torch.ones(1024, device="cuda")
    want = [torch.zeros(2000, 1024, dtype=torch.uint8, device="cuda"),
            torch.zeros(2000, device="cuda")]
    ov.op_add_rmsnorm(x, w, want[0], 1e-6, scales=want[1])
    logits, u = normal(2, 300, 5000).cuda(), torch.rand(300).cuda()
    tokens = torch.zeros(300, dtype=torch.int32, device="cuda")
    ov.op_sample(logits, u, tokens, top_p=0.9)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        o = [torch.zeros_like(want[0]), torch.zeros_like(want[1]), torch.zeros_like(tokens)]
        torch.cuda.synchronize()
        for _ in range(5):
            ov.op_add_rmsnorm(x, w, o[0], 1e-6, scales=o[1], stream=s.cuda_stream)
            ov.op_sample(logits, u, o[2], top_p=0.9, stream=s.cuda_stream)
        got.append(o)
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
        assert torch.equal(o[2], tokens)


# ------------------------------------------------------------------ far sizes and values

@pytest.mark.parametrize("eps", [1e-45, 1e-38, 1e-20])
@pytest.mark.parametrize("scale", [1e-22, 1e-12, 1.0])
def test_norm_of_a_tiny_epsilon(eps, scale):
    """Means under float32's smallest numbers."""
    x = normal(31, 5, 300) * scale
    w = 1 + 0.1 * normal(32, 300)
    eps = float(np.float32(eps))
    check_norm(x, w, None, "f32", eps)
    check_norm(x, w, None, "e4m3", eps)


@pytest.mark.parametrize("scale", [1e-22, 1.0, 1e25])
def test_rotary_norms_of_any_loudness(scale):
    x = normal(33, 6, 5, 96) * scale
    positions = torch.arange(6, dtype=torch.int32) * 1000
    f = torch.tensor(ov.rotary_frequencies(96)[0])
    w = 1 + 0.2 * normal(34, 96)
    eps = float(np.float32(1e-45)) if scale < 1 else 1e-6
    for interleaved in (False, True):
        out = torch.zeros(6, 5, 96, device="cuda")
        ov.op_rotary(x.cuda(), out, None, None, f.cuda(), positions=positions.cuda(),
                     q_norm=w.cuda(), eps=eps, interleaved=interleaved)
        check_rotary(out, x, positions, f, interleaved, 1.0, w, eps, "f32")


def test_rotary_of_the_most_rows():
    rows = (1 << 24) - 1
    q = torch.ones(rows, 1, 2, dtype=torch.float16, device="cuda")
    positions = torch.zeros(rows, dtype=torch.int32, device="cuda")
    positions[-3:] = torch.tensor([1, 2, 3], dtype=torch.int32)
    ov.op_rotary(q, q, None, None, torch.ones(1, device="cuda"), positions=positions)
    assert (q[:-3] == 1).all()
    check_rotary(q[-3:], torch.ones(3, 1, 2, dtype=torch.float16),
                 torch.tensor([1, 2, 3]), torch.ones(1), False, 1.0, None, 0, "f16")


@pytest.mark.parametrize("rows,width,out", [(2100, 2064, 2100), (4100, 128, 2300),
                                            (3900, 384, 2500), (2300, 1152, 4100),
                                            (4096, 256, 4096), (33000, 128, 250),
                                            (4300, 384, 4200), (9000, 128, 2100),
                                            (100, 128, 70000), (64, 256, 9000), (50, 2064, 2500),
                                            (1000, 528, 130), (32, 400, 9000), (1300, 528, 2000),
                                            (4000, 128, 1030), (1025, 272, 2100)])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_product_of_whole_numbers_in_large_tiles(rows, width, out, kind):
    test_product_of_whole_numbers(rows, width, out, kind)


@pytest.mark.parametrize("rows", [3, 70])
def test_product_of_rows_far_apart(rows):
    stride = (1 << 23) + 16
    a, x = whole_codes(41, rows, 272)
    b, w = whole_codes(42, 130, 272)
    wide = torch.zeros(rows, stride, dtype=torch.uint8, device="cuda")
    wide[:, :272] = x.view(torch.uint8).cuda()
    y = torch.zeros(rows, 130, device="cuda")
    one = torch.ones(130, device="cuda")
    ov.op_linear8(wide[:, :272], one[:rows], w.cuda(), one, y)
    assert torch.equal(y.cpu().double(), a.double() @ b.double().t())


@pytest.mark.parametrize("rows,out", [(16, 64), (64, 9000), (300, 200), (4100, 2300)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_product_of_loud_codes_in_16_bits(rows, out, kind):
    """One loud code in eight, quiet ones of one sign around it: what the sums of eight
    products cut off is under 7 * 2^-13 of the products' magnitudes; the additions of the
    256 / 8 sums and the scales' products are 2^-18 more."""
    width = 256
    g = torch.Generator().manual_seed(43)
    x = torch.rand(rows, width, generator=g) * 0.02 + 0.01
    x[:, ::8] = 448.0 * torch.sign(normal(44, rows, width // 8))
    x = x.to(torch.float8_e4m3fn)
    w = (torch.rand(out, width, generator=g) * 2 + 0.5).to(torch.float8_e4m3fn)
    one = torch.ones(max(rows, out), device="cuda")
    y = torch.zeros(rows, out, dtype=TYPES[kind], device="cuda")
    scale = one[:rows] * 2.0 ** -6
    ov.op_linear8(x.cuda(), scale, w.cuda(), one[:out], y)
    a = x.float().double() * 2.0 ** -6
    want, size = a @ w.float().double().t(), a.abs() @ w.float().double().t()
    bound = size * (7 * 2.0 ** -13 + 2.0 ** -18) * (1 + HALF_STEP[kind]) + \
        want.abs() * HALF_STEP[kind] + TINY[kind]
    assert ((y.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("rows,width", [(2, 4096), (3, 4100), (2, 16384), (2, 16390), (3, 20001),
                                        (1, 32768), (2, 33000), (2, 65530)])
def test_wide_rows(rows, width):
    """Every width's number of lanes and runs, loud rows and gates among them."""
    x = normal(51, rows, width)
    r = normal(52, rows, width)
    w = 1 + 0.2 * normal(53, width)
    for out in ("e4m3", "bf16"):
        check_norm(x.half(), w, r.half(), out, 1e-6, extra=3)
        check_norm(x * 1e25, w, None, out, 1e-6)
    gate = (normal(54, rows, width) * 4).half()
    codes = torch.zeros(rows, width, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows, device="cuda")
    ov.op_quantize8(x.half().cuda(), codes, scales, gate=gate.cuda())
    g = gate.double()
    check_codes(codes, scales, x.half().double() * g * torch.sigmoid(g), GATE)
    ov.op_quantize8(x.cuda(), codes, scales)
    check_codes(codes, scales, x, 0.0)
    lost = x.clone()
    lost[0, width - 1], w2 = np.nan, w.clone()
    ov.op_quantize8(lost.cuda(), codes, scales)
    assert torch.isnan(scales[0]) and (codes[0] == 0).all() and torch.isfinite(scales[1:]).all()
    w2[width // 2] = np.inf
    ov.op_add_rmsnorm(x.cuda(), w2.cuda(), codes, 1e-6, scales=scales)
    assert torch.isnan(scales).all() and (codes == 0).all()


def test_wide_rows_beside_a_scale_border():
    """As test_norm_beside_a_scale_border, in rows whose weights are read twice."""
    for width in (20000, 40000):
        x = normal(55, 12, width)
        x[:, 17] = 30.0
        y = norm_of(x, None, torch.ones(width), 1e-6)[1]
        weight = torch.ones(width)
        for r in range(12):
            weight[17] = float(1.75 * 2.0 ** 4 * (1 + (r - 6) * 2.0 ** -25) / y[r, 17])
            check_norm(x[r:r + 1], weight, None, "e4m3", 1e-6)

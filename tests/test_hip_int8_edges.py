"""GPU: the 8-bit integer operators at the places where their definition is sharp: quotients on the border between two
integers, results next to the end of fp32's range, and the tiled forms of the product at shapes that divide nothing."""
import pytest
import torch

from test_hip_int8 import check_product, exact_swiglu, product_case, swiglu_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
TINY = 2.0 ** -126


@pytest.fixture(scope="module")
def hip():
    from nano_qwen3tts_vllm import hip as h
    assert torch.cuda.is_available()
    return h


def fp32(x):
    """An operation's result in fp32.  A quotient and a root of fp32 numbers, computed in float64 and rounded again, are the
    correctly rounded ones (53 >= 2 * 24 + 2 bits); the CPU's own fp32 root is not, on every machine."""
    return x.float().double()


def rows_in_fp32(y):
    """q and scales of fp32 rows (CPU) by the definition, every operation rounded to fp32, ties to even."""
    y = y.double()
    s = fp32(y.abs().amax(-1) / 127).clamp_min(TINY)
    return fp32(y / s[:, None]).round().float(), s.float()


# ---------------------------------------------------------------- borders between two integers
def mantissa_rows(exponent):
    """A row for every mantissa a maximum can have; in it every mantissa at its own size and at each half of that, down to
    2^-9 of it.  x / scale is 63.5 or its neighbour at half the maximum."""
    m = torch.arange(128, 256, dtype=torch.float64)
    x = m[None, :, None] * 2.0 ** -torch.arange(10, dtype=torch.float64)
    x = torch.where(x <= m[:, None, None], x, 0.0).reshape(128, -1)
    x = torch.cat([m[:, None], x, -x], 1) * 2.0 ** exponent
    return x.bfloat16()                                          # small exponents: denormal numbers among them, rounded here


@pytest.mark.parametrize("exponent", [0, 60, 118, -60, -93, -100, -107, -113, -120, -126, -128, -133])
def test_quantised_values_are_the_rounded_fp32_quotients(hip, exponent):
    """Equal, as the definition is exact arithmetic up to its roundings: the scale is one fp32 division, q another and the
    rounding to the nearest integer, ties to even."""
    x = mantissa_rows(exponent)
    want_q, want_s = rows_in_fp32(x.float())
    for rows in (x, x[:3], x.repeat(1, 8), x.repeat(20, 1)):     # the same through other numbers of threads a row, and long rows
        q, s = hip.quantize_int8(rows.to(DEV))
        n, k = rows.shape[0], rows.shape[1] // x.shape[1]
        take = torch.arange(n) % 128
        assert torch.equal(s.cpu(), want_s[take])
        assert torch.equal(q.cpu().float(), want_q[take].repeat(1, k))


@pytest.mark.parametrize("M,H", [(64, 256), (64, 1024), (4100, 2048), (300, 8192), (6, 32768)])
def test_normed_rows_are_quantised_by_fp32_quotients(hip, M, H):
    """Whole numbers whose squares add up without rounding (below 2^24), lengths a power of two, eps 0: what is left are the
    root, h / root * w and the quotient by the scale, each rounded to fp32.  Rows have numbers at half of their maximum."""
    g = torch.Generator().manual_seed(M + H)
    h = torch.randint(-16, 17, (M, H), generator=g).float() * (2.0 if H <= 8192 else 1.0)
    w = 2.0 ** torch.randint(-1, 2, (H,), generator=g).float()
    root = fp32(fp32(h.double().pow(2).sum(-1) / H).sqrt())
    want_q, want_s = rows_in_fp32(fp32(fp32(h.double() / root[:, None]) * w))
    q, s = hip.rmsnorm_int8(h.bfloat16().to(DEV), w.bfloat16().to(DEV), 0.0)
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().float(), want_q)


def test_normed_rows_whose_mean_overflows(hip):
    """fp32 holds the mean: rows of finite numbers whose squares pass its range become zeros with the smallest scale, an infinity
    among them NaN."""
    x = torch.full((3, 600), 3e38).bfloat16()
    x[1, ::2] = -1e30
    x[2, 5] = float("inf")
    q, s = hip.rmsnorm_int8(x.to(DEV), torch.ones(600, dtype=torch.bfloat16, device=DEV), 1e-6)
    assert not q.any() and s[:2].tolist() == [TINY, TINY] and bool(torch.isnan(s[2]))


@pytest.mark.parametrize("K", [992, 990])
def test_a_single_row_of_a_wider_buffer(hip, K):
    """Its stride means nothing and may be anything: also one that rows of int8 values could not have."""
    g = torch.Generator(device=DEV).manual_seed(K)
    x = torch.randn(3, 1000, generator=g, device=DEV).bfloat16()[:1, :K]
    qbuf = torch.full((3, 1000), 99, dtype=torch.int8, device=DEV)
    q, s = hip.quantize_int8(x, out=qbuf[:1, :K])
    want, want_s = hip.quantize_int8(x.contiguous())
    assert torch.equal(q, want) and torch.equal(s, want_s) and torch.all(qbuf[:1, K:] == 99) and torch.all(qbuf[1:] == 99)
    w, ws = torch.randint(-128, 128, (40, K), generator=g, device=DEV, dtype=torch.int8), torch.ones(40, device=DEV)
    p = hip.pack_weight_int8(w)
    assert torch.equal(hip.linear_int8(q, s, p, ws, 40), hip.linear_int8(want, s, p, ws, 40))


# ---------------------------------------------------------------- the product in every form
# (form, M, N, K): forms 0-5 split K over waves, 6-10 are the tiles.  For each tile: at most a tile a workgroup and several, two
# k-steps (fewer than the stages that are requested ahead) and many; nothing is a multiple of anything.  Form 8 takes
# shapes with at most 256 tiles only, which is a tile a workgroup.  A row or column more or less may change the form, so the
# form is asserted (also on the host, in the tests that need no device).
LINEAR_FORMS = [
    (0, 108, 356, 1180), (0, 360, 69, 1093), (1, 11, 1319, 2308), (1, 185, 85, 2390), (2, 230, 46, 172), (2, 9, 4535, 179),
    (3, 353, 453, 355), (4, 693, 439, 129), (5, 12, 82, 2651), (5, 25, 358, 365),
    (6, 1111, 872, 980), (6, 2898, 944, 4), (6, 8446, 203, 144), (6, 323, 5781, 657),
    (7, 2600, 2558, 156), (7, 1351, 5867, 3), (7, 2615, 3179, 134), (7, 1924, 4447, 656),
    (8, 1549, 1507, 660), (8, 2916, 1353, 176), (8, 1301, 2713, 3),
    (9, 3151, 1330, 660), (9, 4880, 1495, 130), (9, 4964, 3222, 742),
    (10, 2070, 5994, 663), (10, 5946, 2321, 258), (10, 6514, 4830, 587), (10, 5625, 5573, 642),
]
SWIGLU_FORMS = [
    (0, 148, 135, 1562), (1, 11, 1091, 1501), (2, 593, 26, 243), (3, 100, 667, 222), (4, 196, 830, 310), (5, 23, 79, 230),
    (6, 303, 929, 1660), (6, 664, 1585, 267), (6, 6510, 421, 2),
    (7, 4916, 779, 648), (7, 2647, 3729, 155), (7, 3500, 4635, 2),
    (8, 2692, 419, 654), (8, 579, 2509, 134), (8, 2570, 611, 3),
    (9, 2900, 721, 643), (9, 1477, 2649, 129), (9, 2595, 2995, 724),
    (10, 4465, 1391, 654), (10, 1344, 5046, 265), (10, 8846, 1749, 558),
]


def inside(M, N, wider, offset):
    """A view [M, N] with a row stride of N + wider, `offset` elements into a buffer of sevens, and a check that the rest of
    the buffer still holds them."""
    buf = torch.full((offset + M * (N + wider) + 9,), 7.0, dtype=torch.bfloat16, device=DEV)
    view = buf.as_strided((M, N), (N + wider, 1), offset)

    def rest_is_untouched():
        inside = torch.zeros_like(buf, dtype=torch.bool)
        inside.as_strided((M, N), (N + wider, 1), offset).fill_(True)
        return bool(((buf == 7.0) | inside).all())

    return view, rest_is_untouched


@pytest.mark.parametrize("form,M,N,K", LINEAR_FORMS)
def test_linear_in_every_form(hip, form, M, N, K):
    """Dense, and with bias and residual into the residual's own place inside a wider buffer at odd alignments: float64, and the
    same bits as into a buffer of its own."""
    assert hip.lib.qtts_linear_int8_form(M, N, K, 0) == form
    x, xs, w, ws, b, r = product_case(hip, M, N, K, True, True, seed=1)
    p = hip.pack_weight_int8(w)
    check_product(hip.linear_int8(x, xs, p, ws, N), x, xs, w, ws)
    got = hip.linear_int8(x, xs, p, ws, N, bias=b, residual=r)
    check_product(got, x, xs, w, ws, b, r)
    wide = torch.full((M, (K + 15) // 16 * 16 + 48), -1, dtype=torch.int8, device=DEV)[:, 16:16 + K]
    wide.copy_(x)
    assert torch.equal(hip.linear_int8(wide, xs, p, ws, N, bias=b, residual=r), got)
    for wider, offset in ((5, 3), (8, 8)):
        view, rest_is_untouched = inside(M, N, wider, offset)
        view.copy_(r)
        assert hip.linear_int8(x, xs, p, ws, N, bias=b, residual=view, out=view) is view
        assert torch.equal(view, got) and rest_is_untouched()
        other, rest_is_untouched = inside(M, N, wider + 4, offset + 1)
        view.copy_(r)
        hip.linear_int8(x, xs, p, ws, N, bias=b, residual=view, out=other)
        assert torch.equal(other, got) and rest_is_untouched() and torch.equal(view, r)


@pytest.mark.parametrize("form,M,I,K", SWIGLU_FORMS)
def test_swiglu_in_every_form(hip, form, M, I, K):
    assert hip.lib.qtts_linear_int8_form(M, I, K, 1) == form
    x, xs, gate, gs, up, us = swiglu_case(hip, M, I, K)
    p = hip.pack_gate_up_int8(gate, up)
    got = hip.linear_swiglu_int8(x, xs, p, gs, us, I)
    g, u, want = exact_swiglu(x, xs, gate, gs, up, us)
    off = (got.double() - want).abs() - ((2.0 ** -8 + (g.abs() + 2) * 2.0 ** -20) * want.abs() + 2.0 ** -118 * (g * u).abs())
    assert float(off.max()) <= 0, float(off.max())
    for wider, offset in ((5, 3), (8, 8)):
        view, rest_is_untouched = inside(M, I, wider, offset)
        hip.linear_swiglu_int8(x, xs, p, gs, us, I, out=view)
        assert torch.equal(view, got) and rest_is_untouched()


# ---------------------------------------------------------------- results next to the end of fp32's range
def one_of_each_form(cases):
    return [next(c for c in cases if c[0] == form) for form in range(11)]


def huge_rows(x, xs):
    """Every fifth row with the scale of a row at bf16's maximum or near it, a row of NaN, and a row of infinity as the row
    operators leave it."""
    xs[::5] = 2.6e36 * (0.5 + 0.5 * torch.rand_like(xs[::5]))
    xs[1], xs[2] = float("nan"), float("inf")
    x[1], x[2] = 0, 0
    fine = torch.ones_like(xs, dtype=torch.bool)
    fine[1:3] = False
    return fine


@pytest.mark.parametrize("form,M,N,K", one_of_each_form(LINEAR_FORMS))
def test_linear_of_huge_rows(hip, form, M, N, K):
    """Sum times row scale passes fp32's range, the result does not (|sum| <= 2^14 K < 2^26, channel scales of at most 2^-24)."""
    x, xs, w, ws, b, r = product_case(hip, M, N, K, True, True, seed=2)
    fine = huge_rows(x, xs)
    ws = (0.1 + 0.9 * torch.rand_like(ws)) * 2.0 ** -24
    got = hip.linear_int8(x, xs, hip.pack_weight_int8(w), ws, N, bias=b, residual=r)
    assert torch.isnan(got[~fine]).all()
    check_product(got[fine], x[fine], xs[fine], w, ws, b, r[fine])
    assert float(got[fine].abs().max()) > 2.0 ** 100


@pytest.mark.parametrize("form,M,I,K", one_of_each_form(SWIGLU_FORMS))
def test_swiglu_of_huge_rows(hip, form, M, I, K):
    """The bound of the other sizes; for positive gates silu's relative slope stays below 1.3, so that |g| does not enter it.  The
    rows that are not huge have gates and products of 1e-25 each here, whose product is below the smallest normal number: half a
    step of a denormal bf16 number is 2^-134, of an fp32 one 2^-150, together below 2^-133."""
    x, xs, gate, gs, up, us = swiglu_case(hip, M, I, K)
    fine = huge_rows(x, xs)
    gs, us = (t / t.max() * 2.0 ** -100 for t in (gs, us))
    got = hip.linear_swiglu_int8(x, xs, hip.pack_gate_up_int8(gate, up), gs, us, I).double()
    assert torch.isnan(got[~fine]).all()
    g, u, want = (t[fine] for t in exact_swiglu(x, xs, gate, gs, up, us))
    off = (got[fine] - want).abs() - ((2.0 ** -8 + (3 + (-g).clamp_min(0)) * 2.0 ** -20) * want.abs() + 2.0 ** -118 * (g * u).abs() + 2.0 ** -133)
    assert float(off.max()) <= 0, float(off.max())
    assert float(got[fine].abs().max()) > 2.0 ** 40

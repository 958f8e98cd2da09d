"""GPU: the 8-bit integer operators at the places where their definition is sharp: quotients on the border between two
integers, results next to the end of fp32's range, and the tiled forms of the product at shapes that divide nothing."""
import pytest
import torch

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

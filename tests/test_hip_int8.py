"""GPU: the 8-bit integer operators (qtts_quantize_int8, qtts_rmsnorm_int8, qtts_linear_int8, qtts_linear_swiglu_int8 and the
packing calls) against their definitions in float64.

Tolerances, with u = 2^-24 (half a step of fp32) and 2^-8 (half a step of bf16):
* the scale of quantize_int8 is one fp32 division of a bf16 number: equal.  q is x * (1 / s) rounded, three fp32 roundings
  before the last one: |q - x / s| <= 1/2 + 127 * 3 u < 1/2 + 3e-5.
* rmsnorm_int8 adds at most 16 * 8 squares in a row per thread, then 6 + 32 partial sums: the mean is off by at most 168 u,
  its root by half of that, with the root, the quotient, eps and the two products y is off by at most 92 u < 6e-6, and so is
  the scale; q by 127 times twice that: |q - y / s| <= 1/2 + 2e-3.  h is one bf16 rounding of an fp32 sum of two bf16
  numbers: equal to the float32 sum's rounding.
* the integer sum is exact; its conversion, the two products and the two additions are one u each of the terms' magnitudes,
  the store is half a step of bf16: |got - want| <= 2^-8 |want| + 2^-21 (|p| + |bias| + |res|)   (room for the product of both).
* SwiGLU: g and u are off by 3 u; exp2(g log2 e) by (|g| + 2) 2 u in relative terms and its reciprocal by 2 u, a relative
  error of g grows by 1 + |g| in silu: (8 |g| + 16) u in all, below (|g| + 2) 2^-20; then the store.  Where exp overflows, silu
  is -0 instead of less than 2^-118 |g|.
"""
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


def gen(*seed):
    return torch.Generator(device=DEV).manual_seed(hash(seed) % (1 << 31))


def rand_bf16(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).bfloat16()


def rand_int8(g, M, K, low=-128):
    return torch.randint(low, 128, (M, K), generator=g, device=DEV, dtype=torch.int8)


def padded(hip, q):
    """q as the operators take it, with the worst values behind the last column."""
    out = hip.int8_rows(*q.shape, q.device)
    full = out.as_strided((out.shape[0], (out.shape[1] + 15) // 16 * 16), (out.stride(0), 1))
    full.fill_(-128)
    out.copy_(q)
    return out


def check_rows(q, s, y, s_tol, q_tol):
    """q, s of rows y [M, K] (float64, finite)."""
    want = (y.abs().amax(-1) / 127).clamp_min(TINY)
    assert torch.all((s.double() - want).abs() <= s_tol * want)
    off = (q.double() - y / want[:, None]).abs()
    assert float(off.max()) <= 0.5 + q_tol, float(off.max())
    assert int(q.abs().max()) <= 127


# ---------------------------------------------------------------- rows
SHAPES = [(1, 1), (3, 7), (2, 64), (5, 1000), (1, 2048), (9, 2049), (4, 4095), (3, 6144), (2, 8200), (2, 16385), (1, 40000), (1, 131071),
          (1030, 256), (300, 2048), (17, 512), (2100, 40)]


@pytest.mark.parametrize("M,K", SHAPES)
def test_quantize(hip, M, K):
    x = rand_bf16(gen(1, M, K), M, K, scale=3.0)
    q, s = hip.quantize_int8(x)
    want = (x.float().abs().amax(-1) / torch.full((), 127.0, device=DEV)).clamp_min(TINY)
    assert torch.equal(s, want)
    check_rows(q, s, x.double(), 2.0 ** -24, 3e-5)


@pytest.mark.parametrize("M,H", SHAPES)
@pytest.mark.parametrize("with_delta", [False, True])
def test_rmsnorm(hip, M, H, with_delta):
    g = gen(2, M, H)
    x, d = rand_bf16(g, M, H, scale=2.0), rand_bf16(g, M, H)
    w = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).bfloat16()
    r = hip.rmsnorm_int8(x, w, 1e-6, delta=d if with_delta else None)
    h = x
    if with_delta:
        h = (x.float() + d.float()).bfloat16()
        assert torch.equal(r[2], h)
    y = h.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.double()
    check_rows(r[0], r[1], y, 6e-6, 2e-3)


@pytest.mark.parametrize("K", [300, 1000, 1111, 2048, 2500, 4096, 5001, 6144])
def test_a_row_is_quantised_the_same_among_many(hip, K):
    """More rows are given fewer threads each: the same bits."""
    M = 4200
    g = gen(30, K)
    x, d, w = rand_bf16(g, M, K), rand_bf16(g, M, K), rand_bf16(g, K)
    many = hip.rmsnorm_int8(x, w, 1e-6, delta=d)
    plain = hip.quantize_int8(x)
    for m in (1, 7, 600, 2100):
        for a, b in zip(hip.rmsnorm_int8(x[:m], w, 1e-6, delta=d[:m]), many):
            assert torch.equal(a, b[:m]), m
        for a, b in zip(hip.quantize_int8(x[:m]), plain):
            assert torch.equal(a, b[:m]), m


@pytest.mark.parametrize("off,ld", [(0, 1000), (1, 1001), (3, 1008), (8, 1016)])
def test_rows_with_other_strides_and_alignments(hip, off, ld):
    """Rows inside a wider buffer: the same result as dense rows, and nothing written beside them."""
    M, K = 6, 992
    g = gen(3, off, ld)
    x, d = (rand_bf16(g, M * ld + 16).as_strided((M, K), (ld, 1), off) for _ in range(2))
    w = rand_bf16(g, K + 8)[off % 8:off % 8 + K]
    dense = hip.rmsnorm_int8(x.contiguous(), w.clone(), 1e-6, delta=d.contiguous())
    buf = torch.full((M * ld + 16,), 7.0, dtype=torch.bfloat16, device=DEV)
    qbuf = torch.full((M * 1024,), 99, dtype=torch.int8, device=DEV)
    q, s, h = hip.rmsnorm_int8(x, w, 1e-6, delta=d, sum_out=buf.as_strided((M, K), (ld, 1), off), out=qbuf.as_strided((M, K), (1024, 1)))
    for a, b in zip((q, s, h), dense):
        assert torch.equal(a, b)
    assert torch.all(qbuf.view(M, 1024)[:, K:] == 99)
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep.as_strided((M, K), (ld, 1), off).fill_(False)
    assert torch.all(buf[keep] == 7.0)
    qd, sd = hip.quantize_int8(x)
    qc, sc = hip.quantize_int8(x.contiguous())
    assert torch.equal(qd, qc) and torch.equal(sd, sc)


@pytest.mark.parametrize("into", ["x", "delta"])
@pytest.mark.parametrize("H", [512, 2047, 5000, 20001])
def test_rmsnorm_sum_in_place(hip, into, H):
    g = gen(4, H)
    x, d, w = rand_bf16(g, 5, H), rand_bf16(g, 5, H), rand_bf16(g, H)
    want = hip.rmsnorm_int8(x, w, 1e-5, delta=d)
    x2, d2 = x.clone(), d.clone()
    got = hip.rmsnorm_int8(x2, w, 1e-5, delta=d2, sum_out=x2 if into == "x" else d2)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(x2 if into == "x" else d2, want[2]) and torch.equal(d2 if into == "x" else x2, d if into == "x" else x)


def test_rows_at_the_borders_of_the_type(hip):
    """Zeros, denormals, the largest values, NaN and infinities: only the rows that hold them show it."""
    K = 300
    x = rand_bf16(gen(5), 9, K)
    x[0] = 0.0
    x[1] = 0.0
    x[1, 7] = 9.2e-41                                # the smallest bf16 denormal
    x[2] = torch.finfo(torch.bfloat16).max * torch.sign(x[2].float()).bfloat16()
    x[3, 299] = float("inf")
    x[4, 0] = float("nan")
    x[5, 17] = -float("inf")
    x[6] = 1e-38
    q, s = hip.quantize_int8(x)
    assert torch.all(q[0] == 0) and float(s[0]) == TINY and torch.all(q[1] == 0) and float(s[1]) == TINY
    assert torch.all(q[2].abs()[x[2] != 0] == 127) and bool(torch.isfinite(s[2]))
    for i in (3, 4, 5):
        assert torch.all(q[i] == 0) and not bool(torch.isfinite(s[i]))
    assert bool(torch.isnan(s[4])) and float(s[3]) == float("inf") and float(s[5]) == float("inf")
    fine = [2, 7, 8]
    check_rows(q[fine], s[fine], x[fine].double(), 2.0 ** -24, 3e-5)
    w = torch.ones(K, dtype=torch.bfloat16, device=DEV)
    qn, sn = hip.rmsnorm_int8(x, w, 1e-6)
    for i in (3, 4, 5):
        assert torch.all(qn[i] == 0) and not bool(torch.isfinite(sn[i]))
    assert torch.all(qn[0] == 0) and float(sn[0]) == TINY
    y = x[[7, 8]].double()
    check_rows(qn[[7, 8]], sn[[7, 8]], y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6), 6e-6, 2e-3)
    # eps = 0 and a row of zeros: 0 / 0
    q0, s0 = hip.rmsnorm_int8(torch.zeros(2, 40, dtype=torch.bfloat16, device=DEV), w[:40].clone(), 0.0)
    assert torch.all(q0 == 0) and bool(torch.isnan(s0).all())
    # a row that is not finite makes exactly its own products NaN
    wq = rand_int8(gen(6), 48, K)
    out = hip.linear_int8(q, s, hip.pack_weight_int8(wq), torch.ones(48, device=DEV), 48)
    assert torch.isnan(out[3:6]).all() and torch.isfinite(out[[0, 1, 6, 7, 8]]).all()


def test_quantize_ties_go_to_even(hip):
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 125.5, -126.5]], device=DEV).bfloat16()
    q, s = hip.quantize_int8(x)
    assert float(s[0]) == 1.0
    assert q[0].tolist() == [127] + [int(v) for v in torch.round(x[0, 1:].double()).tolist()]


def test_no_rows(hip):
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    q, s = hip.quantize_int8(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    p = hip.pack_weight_int8(rand_int8(gen(7), 16, 64))
    assert hip.linear_int8(q, s, p, torch.ones(16, device=DEV), 16).shape == (0, 16)


# ---------------------------------------------------------------- the product
def unpack(packed, N, K):
    """The packed order's definition: [tile][step][lane][16]."""
    steps = 2 * ((K + 127) // 128)
    p = packed.view(torch.int8).view(-1, steps, 4, 16, 16)            # tile, step, lane / 16, lane % 16, byte
    return p.permute(0, 3, 1, 2, 4).reshape(p.shape[0] * 16, steps * 64)


@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (17, 65), (100, 200), (33, 1111)])
def test_packing(hip, N, K):
    w, up = rand_int8(gen(8, N), N, K), rand_int8(gen(9, N), N, K)
    full = unpack(hip.pack_weight_int8(w), N, K)
    assert torch.equal(full[:N, :K], w) and not full[N:].any() and not full[:, K:].any()
    wide = torch.full((N, K + 3), 5, dtype=torch.int8, device=DEV)[:, 1:K + 1]
    wide.copy_(w)
    assert torch.equal(hip.pack_weight_int8(wide), hip.pack_weight_int8(w))
    full = unpack(hip.pack_gate_up_int8(w, up), N, K).view(-1, 4, 4, full.shape[1])     # tile, p, j
    rows = full[:, :, :2].reshape(-1, full.shape[-1]), full[:, :, 2:].reshape(-1, full.shape[-1])
    for got, want in zip(rows, (w, up)):
        assert torch.equal(got[:N, :K], want) and not got[N:].any() and not got[:, K:].any()


def product_case(hip, M, N, K, bias, residual, seed=0):
    g = gen(10, M, N, K, seed)
    x, w = rand_int8(g, M, K), rand_int8(g, N, K)
    xs = torch.rand(M, generator=g, device=DEV) * 0.02 + 1e-4
    ws = torch.rand(N, generator=g, device=DEV) * 0.01 + 1e-4
    b = rand_bf16(g, N) if bias else None
    r = rand_bf16(g, M, N, scale=4.0) if residual else None
    return padded(hip, x), xs, w, ws, b, r


def exact_product(x, xs, w, ws):
    return (x.double() @ w.double().t().contiguous()) * xs.double()[:, None] * ws.double()


def check_product(got, x, xs, w, ws, b=None, r=None):
    p = exact_product(x, xs, w, ws)
    b = torch.zeros((), device=DEV) if b is None else b.double()
    r = torch.zeros((), device=DEV) if r is None else r.double()
    want = p + b + r
    off = (got.double() - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -21 * (p.abs() + b.abs() + r.abs()))
    assert float(off.max()) <= 0, (float(off.max()), (off > 0).nonzero()[:4].tolist())


PRODUCTS = [(1, 1, 1), (1, 16, 64), (1, 4096, 2048), (2, 100, 33), (8, 4, 300), (9, 13, 8000), (20, 9, 1025), (300, 7, 2000), (6, 2043, 2049), (7, 1000, 200), (8, 2048, 6144), (15, 48, 4097), (16, 2048, 2048),
            (17, 250, 129), (33, 512, 512), (48, 1000, 1111), (64, 4096, 1024), (65, 77, 6000), (100, 2050, 300), (128, 128, 128),
            (129, 257, 640), (200, 4096, 2048), (255, 511, 96), (257, 300, 1025), (500, 1000, 1000), (777, 1000, 1111), (1000, 64, 5000),
            (1025, 2047, 257), (2048, 2048, 512), (3000, 24, 24), (4100, 1030, 130)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, True)])
def test_linear(hip, M, N, K, bias, residual):
    x, xs, w, ws, b, r = product_case(hip, M, N, K, bias, residual)
    got = hip.linear_int8(x, xs, hip.pack_weight_int8(w), ws, N, bias=b, residual=r)
    check_product(got, x, xs, w, ws, b, r)


@pytest.mark.parametrize("M", [1, 200, 600])
def test_linear_extreme_sums(hip, M):
    """The largest sum int32 holds: every product 2^14, K = 131071."""
    K, N = 131071, 20
    x = padded(hip, torch.full((M, K), -128, dtype=torch.int8, device=DEV))
    w = torch.full((N, K), -128, dtype=torch.int8, device=DEV)
    ones = torch.ones(M, device=DEV), torch.full((N,), 2.0 ** -20, device=DEV)
    got = hip.linear_int8(x, ones[0], hip.pack_weight_int8(w), ones[1], N)
    assert torch.all(got.double() == torch.tensor(16384.0 * K / 2 ** 20).bfloat16().double())
    x[:, 1::2] = 127
    got = hip.linear_int8(x, ones[0], hip.pack_weight_int8(w), ones[1], N)
    check_product(got, x, ones[0], w, ones[1])


def exact_swiglu(x, xs, gate, gs, up, us):
    g, u = exact_product(x, xs, gate, gs), exact_product(x, xs, up, us)
    return g, u, g * torch.sigmoid(g) * u


def swiglu_case(hip, M, I, K):
    g = gen(11, M, I, K)
    x, gate, up = padded(hip, rand_int8(g, M, K)), rand_int8(g, I, K), rand_int8(g, I, K)
    size = 3.0 / (74.0 * 74.0 * K ** 0.5)                       # gates of a few units, a few rows with very large ones
    xs = torch.where(torch.rand(M, generator=g, device=DEV) < 0.1, 60.0, 1.0) * (torch.rand(M, generator=g, device=DEV) + 0.1)
    gs = size * (torch.rand(I, generator=g, device=DEV) + 0.5)
    us = size * (torch.rand(I, generator=g, device=DEV) + 0.5)
    return x, xs, gate, gs, up, us


@pytest.mark.parametrize("M,I,K", [(1, 1, 1), (1, 6144, 2048), (3, 100, 33), (8, 3, 500), (5, 1021, 2100), (8, 6144, 2048), (16, 1023, 512), (17, 8, 64), (40, 250, 129),
                                   (64, 2048, 1024), (100, 1001, 300), (130, 70, 2000), (200, 6144, 2048), (300, 129, 640),
                                   (513, 1000, 1111), (1030, 2047, 96), (2048, 1024, 512), (4100, 515, 130)])
def test_linear_swiglu(hip, M, I, K):
    x, xs, gate, gs, up, us = swiglu_case(hip, M, I, K)
    got = hip.linear_swiglu_int8(x, xs, hip.pack_gate_up_int8(gate, up), gs, us, I).double()
    g, u, want = exact_swiglu(x, xs, gate, gs, up, us)
    off = (got - want).abs() - ((2.0 ** -8 + (g.abs() + 2) * 2.0 ** -20) * want.abs() + 2.0 ** -118 * (g * u).abs())
    assert float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("N,K", [(500, 1111), (2048, 2048)])
def test_a_row_does_not_depend_on_the_rows_beside_it(hip, N, K):
    """The sums are exact and the epilogue is the same in every form: equal bits whatever the number of rows."""
    M = 1100
    x, xs, w, ws, b, r = product_case(hip, M, N, K, True, True)
    p = hip.pack_weight_int8(w)
    full = hip.linear_int8(x, xs, p, ws, N, bias=b, residual=r)
    for m in (1, 3, 16, 17, 40, 64, 100, 130, 256, 300, 520):
        assert torch.equal(hip.linear_int8(x[:m], xs[:m].clone(), p, ws, N, bias=b, residual=r[:m]), full[:m]), m
    I = N // 2
    pg = hip.pack_gate_up_int8(w[:I], w[I:2 * I])
    full = hip.linear_swiglu_int8(x, xs, pg, ws[:I].clone(), ws[I:2 * I].clone(), I)
    for m in (1, 3, 16, 17, 40, 64, 100, 130, 256, 300, 520):
        assert torch.equal(hip.linear_swiglu_int8(x[:m], xs[:m].clone(), pg, ws[:I].clone(), ws[I:2 * I].clone(), I), full[:m]), m


@pytest.mark.parametrize("M", [5, 70, 400])
@pytest.mark.parametrize("off,ld", [(0, 304), (1, 301), (2, 302), (4, 312)])
def test_products_inside_wider_buffers(hip, M, off, ld):
    """Output and residual rows with other strides and alignments, in place too; nothing beside them is written."""
    N, K = 300, 200
    x, xs, w, ws, b, r = product_case(hip, M, N, K, True, True)
    wide = torch.full((M, 272), -1, dtype=torch.int8, device=DEV)[:, 16:16 + K]
    wide.copy_(x)
    p = hip.pack_weight_int8(w)
    want = hip.linear_int8(x, xs, p, ws, N, bias=b, residual=r)
    buf = torch.full((M * ld + 8,), 7.0, dtype=torch.bfloat16, device=DEV)
    view = buf.as_strided((M, N), (ld, 1), off)
    view.copy_(r)
    assert torch.equal(hip.linear_int8(wide, xs, p, ws, N, bias=b, residual=view, out=view), want)
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep.as_strided((M, N), (ld, 1), off).fill_(False)
    assert torch.all(buf[keep] == 7.0)
    pg = hip.pack_gate_up_int8(w, w.flip(0))
    want = hip.linear_swiglu_int8(x, xs, pg, ws, ws, N)
    buf.fill_(7.0)
    assert torch.equal(hip.linear_swiglu_int8(wide, xs, pg, ws, ws, N, out=view), want)
    assert torch.all(buf[keep] == 7.0)


def test_offsets_beyond_32_bits(hip):
    """2.5 GB of int8 rows, 4.9 GB of bf16 rows: the last rows equal the same rows computed alone."""
    K, M = 8192, 300_032
    x = torch.empty(M, K, dtype=torch.bfloat16, device=DEV)
    x[:-64] = 1.0
    x[-64:] = rand_bf16(gen(12), 64, K)
    tail = x[-64:].clone()
    q, s = hip.quantize_int8(x)
    qt, st = hip.quantize_int8(tail)
    assert torch.equal(q[-64:], qt) and torch.equal(s[-64:], st) and torch.all(q[:-64] == 127)
    w = torch.ones(K, dtype=torch.bfloat16, device=DEV)
    d = torch.zeros_like(x)
    d[-64:] = rand_bf16(gen(13), 64, K)
    dt = d[-64:].clone()
    want = hip.rmsnorm_int8(tail, w, 1e-6, delta=dt)
    got = hip.rmsnorm_int8(x, w, 1e-6, delta=d, sum_out=d)
    for a, b in zip(got, want):
        assert torch.equal(a[-64:], b)
    del x, d, got
    wq = rand_int8(gen(14), 24, K)
    p, ws = hip.pack_weight_int8(wq), torch.full((24,), 1e-3, device=DEV)
    assert torch.equal(hip.linear_int8(q, s, p, ws, 24)[-64:], hip.linear_int8(qt, st, p, ws, 24))
    del q, s
    # an output of 2.4 G elements
    N = 4096
    q, s, wn = rand_int8(gen(15), 600_000, 16), torch.ones(600_000, device=DEV), rand_int8(gen(16), N, 16)
    p, ws = hip.pack_weight_int8(wn), torch.full((N,), 1e-3, device=DEV)
    out = hip.linear_int8(q, s, p, ws, N)
    assert torch.equal(out[-70:], hip.linear_int8(q[-70:].clone(), s[-70:].clone(), p, ws, N))
    check_product(out[-70:], q[-70:], s[-70:], wn, ws)


@pytest.mark.parametrize("M,K", [((1 << 22) + 9, 8), ((1 << 20) + 5, 520)])
def test_more_rows_than_workgroups_of_a_launch(hip, M, K):
    """Workgroups take several rows each: the last rows equal the same rows computed alone."""
    g = gen(31, K)
    x, w = rand_bf16(g, M, K), rand_bf16(g, K)
    d = x.flip(0)
    for got, alone in ((hip.quantize_int8(x), hip.quantize_int8(x[-40:])),
                       (hip.rmsnorm_int8(x, w, 1e-6, delta=d), hip.rmsnorm_int8(x[-40:], w, 1e-6, delta=d[-40:]))):
        for a, b in zip(got, alone):
            assert torch.equal(a[-40:], b)
    q, s = hip.quantize_int8(x)
    check = torch.arange(0, M, 4099, device=DEV)
    for a, b in zip((q, s), hip.quantize_int8(x[check])):
        assert torch.equal(a[check], b)


@pytest.mark.parametrize("M", [600_001, 1_100_000, 2_200_000])
def test_more_rows_than_a_grid_is_high(hip, M):
    """Row blocks of the forms for few columns pass 65535: forms with larger blocks are taken."""
    N, K = 3, 16
    x, xs, w, ws, b, r = product_case(hip, M, N, K, True, True)
    check_product(hip.linear_int8(x, xs, hip.pack_weight_int8(w), ws, N, bias=b, residual=r), x, xs, w, ws, b, r)
    up, us = w.flip(0).contiguous(), ws.flip(0).contiguous()
    pg = hip.pack_gate_up_int8(w, up)
    got = hip.linear_swiglu_int8(x, xs, pg, ws, us, N)
    for at in (0, M // 2, M - 50):
        assert torch.equal(got[at:at + 50], hip.linear_swiglu_int8(x[at:at + 50], xs[at:at + 50].clone(), pg, ws, us, N))


# ---------------------------------------------------------------- a run of them, as an MLP makes it
def mlp_weights(hip, H, I, seed):
    g = gen(17, seed)
    names = {}
    for name, (n, k) in {"gate": (I, H), "up": (I, H), "down": (H, I)}.items():
        names[name] = hip.quantize_int8(rand_bf16(g, n, k, scale=k ** -0.5))
    names["norm"] = (1 + 0.1 * torch.randn(H, generator=g, device=DEV)).bfloat16()
    names["gate_up_packed"] = hip.pack_gate_up_int8(names["gate"][0], names["up"][0])
    names["down_packed"] = hip.pack_weight_int8(names["down"][0])
    return names


def mlp(hip, W, x, delta, H, I):
    q, s, h = hip.rmsnorm_int8(x, W["norm"], 1e-6, delta=delta)
    a = hip.linear_swiglu_int8(q, s, W["gate_up_packed"], W["gate"][1], W["up"][1], I)
    qa, sa = hip.quantize_int8(a)
    return hip.linear_int8(qa, sa, W["down_packed"], W["down"][1], H, residual=h)


def mlp_64(W, x, delta):
    """The same block in float64 from the operators' definitions, on the 8-bit weights."""
    def rows(y):
        s = (y.abs().amax(-1, keepdim=True) / 127).clamp_min(TINY)
        return torch.round(y / s) * s

    def weight(name):
        return (W[name][0].double() * W[name][1].double()[:, None]).t().contiguous()

    h = (x.float() + delta.float()).bfloat16().double()
    y = rows(h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * W["norm"].double())
    g, u = y @ weight("gate"), y @ weight("up")
    a = rows((g * torch.sigmoid(g) * u).bfloat16().double())
    return h, a @ weight("down")


@pytest.mark.parametrize("M", [1, 8, 37, 300, 1500])
def test_mlp_block(hip, M):
    """In norm: the store of the block's output and that of the SwiGLU output are at most half a bf16 step, 2^-8, and on
    average less than half of that, of random sign; a value of q that lies within 2e-3 steps of a border may come out a step
    apart (a step is 1/127 of its row's largest value, four values in a thousand at the bound's worst), which the norm sees as
    sqrt(4e-3) / 127 * 4 = 2e-3.  Together below 2^-8."""
    H, I = 512, 1280
    W = mlp_weights(hip, H, I, 1)
    g = gen(18, M)
    x, delta = rand_bf16(g, M, H, scale=2.0), rand_bf16(g, M, H, scale=0.5)
    got = mlp(hip, W, x, delta, H, I)
    h, down = mlp_64(W, x, delta)
    want = h + down
    err = (got.double() - want).norm() / want.norm()
    assert float(err) <= 2.0 ** -8, float(err)
    assert bool(torch.isfinite(got).all())


def test_another_stream_and_a_captured_graph(hip):
    """The block on a stream of its own, then captured once and replayed on other inputs, eager work in between."""
    H, I, M = 512, 1280, 24
    W = mlp_weights(hip, H, I, 2)
    g = gen(19)
    inputs = [(rand_bf16(g, M, H), rand_bf16(g, M, H)) for _ in range(4)]
    want = [mlp(hip, W, *i, H, I) for i in inputs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [mlp(hip, W, *i, H, I) for i in inputs]
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    x, d = torch.empty_like(inputs[0][0]), torch.empty_like(inputs[0][1])
    q, s, h = hip.int8_rows(M, H, DEV), torch.empty(M, device=DEV), torch.empty_like(x)
    a, qa, sa = torch.empty(M, I, dtype=torch.bfloat16, device=DEV), hip.int8_rows(M, I, DEV), torch.empty(M, device=DEV)
    out = torch.empty_like(x)

    def block():
        hip.rmsnorm_int8(x, W["norm"], 1e-6, delta=d, sum_out=h, out=q, scales=s)
        hip.linear_swiglu_int8(q, s, W["gate_up_packed"], W["gate"][1], W["up"][1], I, out=a)
        hip.quantize_int8(a, out=qa, scales=sa)
        hip.linear_int8(qa, sa, W["down_packed"], W["down"][1], H, residual=h, out=out)

    with torch.cuda.stream(side):
        x.copy_(inputs[0][0]), d.copy_(inputs[0][1])
        block()
        side.synchronize()
        graph = hip.Graph.capture(block)
        for k in (1, 2, 3, 0, 2):
            x.copy_(inputs[k][0]), d.copy_(inputs[k][1])
            graph.launch()
            side.synchronize()
            assert torch.equal(out, want[k]), k
            assert torch.equal(mlp(hip, W, *inputs[(k + 1) % 4], H, I), want[(k + 1) % 4])


def test_a_tensor_of_another_device_is_refused(hip, monkeypatch):
    x = rand_bf16(gen(22), 4, 64)
    monkeypatch.setattr(hip, "current_device", lambda: x.device.index + 1)
    with pytest.raises(hip.QttsError, match="current device"):
        hip.quantize_int8(x)
    with pytest.raises(hip.QttsError, match="current device"):
        hip.rmsnorm_int8(x, x[0].clone())


def test_refusals_on_the_device(hip):
    x = rand_bf16(gen(20), 4, 64)
    q, s = hip.quantize_int8(x)
    p, ws = hip.pack_weight_int8(rand_int8(gen(21), 16, 64)), torch.ones(16, device=DEV)
    with pytest.raises(hip.QttsError, match="bytes that packing made"):
        hip.linear_int8(q, s, p, torch.ones(32, device=DEV), 32)
    with pytest.raises(hip.QttsError, match="x_scales"):
        hip.linear_int8(q, s[:3], p, ws, 16)
    with pytest.raises(hip.QttsError, match="residual"):
        hip.linear_int8(q, s, p, ws, 16, residual=x)
    with pytest.raises(hip.QttsError, match="x: need"):
        hip.linear_int8(q.t(), s, p, ws, 16)
    with pytest.raises(hip.QttsError, match="x: need"):
        hip.linear_int8(x, s, p, ws, 16)
    with pytest.raises(hip.QttsError, match="multiple of 16"):
        hip.linear_int8(torch.zeros(4, 72, dtype=torch.int8, device=DEV)[:, :64], s, p, ws, 16)
    with pytest.raises(hip.QttsError, match="misaligned"):
        hip.linear_int8(torch.zeros(4, 96, dtype=torch.int8, device=DEV)[:, 8:72], s, p, ws, 16)
    with pytest.raises(hip.QttsError, match="readable bytes"):
        hip.linear_int8(torch.zeros(1, 60, dtype=torch.int8, device=DEV), s[:1], p, ws, 16)
    with pytest.raises(hip.QttsError, match="on cpu"):
        hip.quantize_int8(x.cpu())
    with pytest.raises(hip.QttsError, match="row strides"):
        hip.quantize_int8(x[:1].expand(4, 64))
    with pytest.raises(hip.QttsError, match="sum_out without delta"):
        hip.rmsnorm_int8(x, x[0].clone(), sum_out=x)

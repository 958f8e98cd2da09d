"""What the 8-bit integer entry points refuse, on the host (no device: made-up pointers that are never dereferenced; on a
box that has a GPU a check that went missing would launch a kernel on them, so this file does not run there)."""
import pytest
import torch

from nano_qwen3tts_vllm import hip

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up device pointers: host-side validation only")

P = 0x7F0000001000
L = hip.lib


def refuses(rc, *words):
    message = L.qtts_last_error().decode()
    assert rc == -1
    for w in words:
        assert w in message, message


def quantize(x=P, ldx=64, q=P, ldq=64, s=P, M=4, K=64):
    return L.qtts_quantize_int8(x, ldx, q, ldq, s, M, K, None)


@pytest.mark.parametrize("kwargs,word", [
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(s=None), "null"), (dict(M=0), "shape"), (dict(M=-3), "shape"),
    (dict(K=0), "shape"), (dict(K=131072, ldx=131072, ldq=131072), "shape"), (dict(M=0x7f800001), "shape"), (dict(ldx=63), "strides"), (dict(ldq=48), "strides"),
    (dict(ldq=72), "strides"), (dict(x=P + 1), "misaligned"), (dict(q=P + 8), "misaligned"), (dict(s=P + 2), "misaligned"),
])
def test_quantize_refuses(kwargs, word):
    refuses(quantize(**kwargs), "quantize_int8:", word)


def rmsnorm(x=P, ldx=64, d=P, ldd=64, w=P, sm=P, lds=64, q=P, ldq=64, s=P, M=4, H=64):
    return L.qtts_rmsnorm_int8(x, ldx, d, ldd, w, 1e-6, sm, lds, q, ldq, s, M, H, None)


@pytest.mark.parametrize("kwargs,word", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(q=None), "null"), (dict(s=None), "null"), (dict(d=None), "come together"),
    (dict(sm=None), "come together"), (dict(M=0), "shape"), (dict(M=0x7fffffff), "shape"), (dict(ldx=72, d=P + 4096, lds=64), "in the place of x"),
    (dict(x=P + 4096, ldd=72), "in the place of x or delta"), (dict(H=0), "shape"), (dict(H=131072, ldx=1 << 18, ldd=1 << 18, lds=1 << 18,
    ldq=1 << 18), "shape"), (dict(ldx=60), "strides"), (dict(ldd=60), "strides"), (dict(lds=60), "strides"), (dict(ldq=60), "strides"),
    (dict(ldq=72), "strides"), (dict(x=P + 1), "misaligned"), (dict(d=P + 1), "misaligned"), (dict(w=P + 1), "misaligned"),
    (dict(sm=P + 1), "misaligned"), (dict(q=P + 4), "misaligned"), (dict(s=P + 1), "misaligned"),
])
def test_rmsnorm_refuses(kwargs, word):
    refuses(rmsnorm(**kwargs), "rmsnorm_int8:", word)


def linear(x=P, ldx=64, xs=P, w=P, ws=P, b=None, r=None, ldr=0, out=P, ldo=32, M=4, N=32, K=64):
    return L.qtts_linear_int8(x, ldx, xs, w, ws, b, r, ldr, out, ldo, M, N, K, None)


@pytest.mark.parametrize("kwargs,word", [
    (dict(x=None), "null"), (dict(xs=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"), (dict(out=None), "null"),
    (dict(M=0), "shape"), (dict(N=0), "shape"), (dict(K=0), "shape"), (dict(K=131072, ldx=131072), "shape"), (dict(N=-1), "shape"),
    (dict(M=0x7f800001), "shape"), (dict(N=0x4000000, ldo=0x4000000), "shape"), (dict(r=P, ldr=40), "in the place of the residual"),
    (dict(ldx=48), "row stride"), (dict(ldx=72), "row stride"), (dict(ldo=31), "strides"), (dict(r=P, ldr=31), "strides"),
    (dict(x=P + 8), "misaligned"), (dict(w=P + 8), "misaligned"), (dict(xs=P + 2), "misaligned"), (dict(ws=P + 2), "misaligned"),
    (dict(out=P + 1), "misaligned"), (dict(b=P + 1), "misaligned"), (dict(r=P + 1, ldr=32), "misaligned"),
])
def test_linear_refuses(kwargs, word):
    refuses(linear(**kwargs), "linear_int8:", word)


def swiglu(x=P, ldx=64, xs=P, w=P, gs=P, us=P, out=P, ldo=32, M=4, I=32, K=64):
    return L.qtts_linear_swiglu_int8(x, ldx, xs, w, gs, us, out, ldo, M, I, K, None)


@pytest.mark.parametrize("kwargs,word", [
    (dict(x=None), "null"), (dict(xs=None), "null"), (dict(w=None), "null"), (dict(gs=None), "null"), (dict(us=None), "null"),
    (dict(out=None), "null"), (dict(M=0), "shape"), (dict(I=0), "shape"), (dict(K=0), "shape"), (dict(K=131072, ldx=131072), "shape"),
    (dict(ldx=72), "row stride"), (dict(ldo=31), "strides"), (dict(us=P + 2), "misaligned"), (dict(out=P + 1), "misaligned"),
])
def test_swiglu_refuses(kwargs, word):
    refuses(swiglu(**kwargs), "linear_swiglu_int8:", word)


def test_packing_refuses_and_sizes():
    refuses(L.qtts_pack_weight_int8(None, 64, P, 16, 64, None), "pack_weight_int8:", "null")
    refuses(L.qtts_pack_weight_int8(P, 63, P, 16, 64, None), "pack_weight_int8:", "shape")
    refuses(L.qtts_pack_weight_int8(P, 1 << 18, P, 16, 131072, None), "pack_weight_int8:", "shape")
    refuses(L.qtts_pack_weight_int8(P, 64, P + 8, 16, 64, None), "pack_weight_int8:", "misaligned")
    refuses(L.qtts_pack_weight_int8(P, 64, P, 0x4000000, 64, None), "pack_weight_int8:", "shape")
    refuses(L.qtts_pack_gate_up_int8(P, None, 64, P, 16, 64, None), "pack_gate_up_int8:", "null")
    refuses(L.qtts_pack_gate_up_int8(P, P, 64, P, 0, 64, None), "pack_gate_up_int8:", "shape")
    assert L.qtts_packed_weight_int8_bytes(16, 128) == 2048 and L.qtts_packed_weight_int8_bytes(17, 129) == 2 * 2 * 2048
    assert L.qtts_packed_gate_up_int8_bytes(8, 128) == 2048 and L.qtts_packed_gate_up_int8_bytes(9, 1) == 2 * 2048
    assert L.qtts_packed_weight_int8_bytes(0, 64) == 0 and L.qtts_packed_weight_int8_bytes(16, 131072) == 0
    assert L.qtts_packed_weight_int8_bytes(1 << 20, 131071) == (1 << 16) * 1024 * 2048      # beyond 32 bits


def test_wrappers_refuse_what_is_not_on_the_device():
    x, q = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.int8)
    v, p = torch.ones(4), torch.zeros(2048, dtype=torch.uint8)
    for call in (lambda: hip.quantize_int8(x), lambda: hip.rmsnorm_int8(x, x[0]), lambda: hip.pack_weight_int8(q),
                 lambda: hip.pack_gate_up_int8(q, q), lambda: hip.linear_int8(q, v, p, torch.ones(16), 16),
                 lambda: hip.linear_swiglu_int8(q, v, p, torch.ones(8), torch.ones(8), 8)):
        with pytest.raises(hip.QttsError, match="on cpu"):
            call()


def test_wrappers_refuse_numbers_beyond_an_int():
    """ctypes hands on the low 32 bits: 2^32 + 64 would arrive as 64.  (meta tensors: shapes and strides without memory)"""
    def rows(M, K, ld, dtype=torch.bfloat16):
        return torch.empty_strided((M, K), (ld, 1), dtype=dtype, device="meta")

    for M, K, ld in ((2, 64, 2 ** 32 + 64), (2, 64, 2 ** 31), (2 ** 32 + 4, 64, 64), (2 ** 31, 1, 1), (3, 2 ** 32 + 64, 2 ** 32 + 64)):
        for call, dtype in ((hip._rows_of, torch.bfloat16), (hip._rows_of, torch.int8)):
            with pytest.raises(hip.QttsError, match="below 2"):
                call(rows(M, K, ld, dtype), dtype, "x", -1)
        with pytest.raises(hip.QttsError, match="below 2"):
            hip._int8_rows_of(rows(M, K, ld, torch.int8), "x", -1)
    assert hip._rows_of(rows(2, 64, 2 ** 31 - 1), torch.bfloat16, "x", -1) == (2, 64, 2 ** 31 - 1)


def test_a_single_row_has_no_stride_of_its_own():
    wide = torch.zeros(3, 1000, dtype=torch.int8)
    assert hip._int8_rows_of(wide[:1, :992], "x", -1) == (1, 992, 992)
    assert hip._int8_rows_of(wide[:1, :990], "x", -1) == (1, 990, 992)
    assert hip._rows_of(torch.empty_strided((1, 64), (2 ** 40, 1), dtype=torch.bfloat16, device="meta"), torch.bfloat16, "x", -1) == (1, 64, 64)
    with pytest.raises(hip.QttsError, match="readable bytes"):
        hip._int8_rows_of(torch.zeros(1, 60, dtype=torch.int8), "x", -1)


def test_the_form_of_a_product():
    """A host-only query.  The device tests cover every form: a change of the choice must not take one out of them."""
    import test_hip_int8_edges as edges
    for swiglu, cases in enumerate((edges.LINEAR_FORMS, edges.SWIGLU_FORMS)):
        for form, M, N, K in cases:
            assert L.qtts_linear_int8_form(M, N, K, swiglu) == form, (M, N, K, swiglu)
        assert {case[0] for case in cases} == set(range(11))
    for M, N, K in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), (1, 0x4000000, 1), (0x7f800001, 1, 1)):
        assert L.qtts_linear_int8_form(M, N, K, 0) == -1 and L.qtts_linear_int8_form(M, N, K, 1) == -1

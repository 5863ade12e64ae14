"""More refusals of the 8-bit operators, none of which needs a GPU."""
import pytest

from test_q8_cpu import P, bwd, dequantize, gemm, norm, quantize, wgrad

F32 = 4

# every operand of more than a byte an element, at an address below its type's alignment
MISALIGNED = [
    (quantize, dict(X=P + 1)), (quantize, dict(X=P + 2, dtype=F32)), (quantize, dict(s=P + 2)),
    (dequantize, dict(X=P + 1)), (dequantize, dict(X=P + 2, dtype=F32)), (dequantize, dict(s=P + 1)),
    (norm, dict(X=P + 1)), (norm, dict(R=P + 1)), (norm, dict(W=P + 1)), (norm, dict(W=P + 2, w=F32)), (norm, dict(H=2 * P + 1)),
    (norm, dict(s=P + 2)), (norm, dict(rstd=P + 2)),
    (gemm, dict(C=P + 2)), (gemm, dict(C=P + 1, c=1)), (gemm, dict(sa=P + 2)), (gemm, dict(sb=P + 1)), (gemm, dict(bias=P + 3)),
    (wgrad, dict(dY=P + 1)), (wgrad, dict(s=P + 2)), (wgrad, dict(dW=P + 2)), (wgrad, dict(dW=P + 1, c=1)),
    (bwd, dict(dY=P + 1)), (bwd, dict(X=P + 1, x=1, xs=None)), (bwd, dict(X=P + 2, x=F32, xs=None)), (bwd, dict(xs=P + 2)),
    (bwd, dict(W=P + 1)), (bwd, dict(rstd=P + 2)), (bwd, dict(dR=P + 1)), (bwd, dict(dX=2 * P + 1)), (bwd, dict(dw=P + 2)),
]


@pytest.mark.parametrize("call,bad", MISALIGNED, ids=["%s-%s" % (c.__name__, "-".join(map(str, k))) for c, k in MISALIGNED])
def test_pointers_below_their_types_alignment(b2g, call, bad):
    """A kernel's access to such an address would be an error of the GPU: the call is refused on the host."""
    assert call(b2g, **bad) == b2g.ERR_INVALID_ARG
    assert b"aligned to its element type" in b2g.load().b2g_last_error_string()


@pytest.fixture
def host_tensors(b2g, monkeypatch):
    """The binding with host memory taken for the current device's, and the library calls that it makes."""
    torch = pytest.importorskip("torch")
    calls = []
    class Lib:
        def b2g_call_q8(self, call, words):
            calls.append(call)
            return b2g.OK
    b2g._device()
    monkeypatch.setattr(b2g, "load", lambda: Lib())
    monkeypatch.setattr(b2g, "_device", lambda: -1)  # what get_device() says of a host tensor
    return torch, calls


def test_binding_checks_a_given_leading_dimension(b2g, host_tensors):
    """A leading dimension that the caller names has to stay inside the tensor's storage, in every operand."""
    torch, calls = host_tensors
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t)
    bf, i8 = torch.bfloat16, torch.int8
    x, q, s, w = z(4, 8, t=bf), z(4, 8, t=i8), z(4), z(8, t=bf)
    k = dict(stream=1)
    ok = [
        lambda: b2g.quantize_q8(x, q, s, 4, 8, dtype=1, ldx=8, ldq=8, **k),
        lambda: b2g.quantize_q8(z(4, 16, t=bf)[:, 8:], q, s, 4, 8, dtype=1, ldx=16, **k),   # ends with its storage
        lambda: b2g.quantize_q8(z(1, 8, t=bf), z(1, 8, t=i8), s, 1, 8, dtype=1, ldx=1000, ldq=1000, **k),  # one row: no pitch
        lambda: b2g.quantize_q8(x, q, s, 2, 8, dtype=1, ldx=24, ldq=24, **k),
        lambda: b2g.quantize_q8(x, q, s, 0, 8, dtype=1, ldx=1000, ldq=1000, **k),
    ]
    for call in ok:
        call()
    assert len(calls) == len(ok)
    bad = [
        lambda: b2g.quantize_q8(x, q, s, 4, 8, dtype=1, ldx=9, **k),
        lambda: b2g.quantize_q8(z(4, 16, t=bf)[:, 9:], q, s, 4, 8, dtype=1, ldx=16, **k),
        lambda: b2g.quantize_q8(x, q, s, 4, 8, dtype=1, ldq=9, **k),
        lambda: b2g.quantize_q8(x, q, s, 3, 8, dtype=1, ldx=1 << 60, **k),
        lambda: b2g.dequantize_q8(q, s, x, 4, 8, dtype=1, ldq=9, **k),
        lambda: b2g.dequantize_q8(q, s, x, 4, 8, dtype=1, ldx=9, **k),
        lambda: b2g.rmsnorm_q8(x, w, q, s, 4, 8, dtype=1, ldx=9, **k),
        lambda: b2g.rmsnorm_q8(x, w, q, s, 4, 8, dtype=1, R=x, ldr=9, **k),
        lambda: b2g.rmsnorm_q8(x, w, q, s, 4, 8, dtype=1, H=x, ldh=9, **k),
        lambda: b2g.rmsnorm_q8(x, w, q, s, 4, 8, dtype=1, ldq=9, **k),
        lambda: b2g.gemm_q8(q, q, z(4, 4), 4, 4, 8, lda=9, **k),
        lambda: b2g.gemm_q8(q, q, z(4, 4), 4, 4, 8, ldb=9, **k),
        lambda: b2g.gemm_q8(q, q, z(4, 4), 4, 4, 8, ldc=5, **k),
        lambda: b2g.wgrad_q8(x, q, s, z(8, 8), 4, 8, 8, ldy=9, **k),
        lambda: b2g.wgrad_q8(x, q, s, z(8, 8), 4, 8, 8, ldq=9, **k),
        lambda: b2g.wgrad_q8(x, q, s, z(8, 8), 4, 8, 8, ldw=9, **k),
        lambda: b2g.rmsnorm_bwd_q8(x, q, s, w, s, x, z(8), 4, 8, ldy=9, **k),
        lambda: b2g.rmsnorm_bwd_q8(x, q, s, w, s, x, z(8), 4, 8, ldx=9, **k),
        lambda: b2g.rmsnorm_bwd_q8(x, q, s, w, s, x, z(8), 4, 8, dres=x, ldr=9, **k),
        lambda: b2g.rmsnorm_bwd_q8(x, q, s, w, s, x, z(8), 4, 8, lddx=9, **k),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(b2g.B2GError, match="leading dimension"):
            call()
        assert len(calls) == len(ok), i


def test_binding_names_an_unknown_type_code(b2g, host_tensors):
    torch, calls = host_tensors
    x, q, s = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for kw in (dict(dtype=b2g.DTYPE_E5M2), dict(dtype=77), dict(dtype=b2g.DTYPE_BF16, q_dtype=b2g.DTYPE_E5M2)):
        with pytest.raises(b2g.B2GError, match="unsupported type code"):
            b2g.quantize_q8(x, q, s, 4, 8, stream=1, **kw)
    assert not calls

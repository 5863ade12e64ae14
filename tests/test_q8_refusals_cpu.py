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

"""Refusals and empty calls of the 8-bit operators (b2g_*_q8): argument checks run before any CUDA
call, so they need no GPU.  Pointers are never dereferenced on the host."""
import pytest

P = 4096  # a non-null pointer that no refused call may touch


def quantize(b, X=P, Q=P, s=P, M=4, N=8, ldx=8, ldq=8, dtype=1, q=5, pow2=0):
    return b.load().b2g_quantize_q8(X, Q, s, M, N, ldx, ldq, dtype, q, pow2, None)


def dequantize(b, Q=P, s=P, X=P, M=4, N=8, ldq=8, ldx=8, q=5, dtype=1):
    return b.load().b2g_dequantize_q8(Q, s, X, M, N, ldq, ldx, q, dtype, None)


def norm(b, X=P, R=P, W=P, H=2 * P, Q=P, s=P, rstd=P, M=4, N=8, ldx=8, ldr=8, ldh=8, ldq=8, dtype=1,
         w=1, q=5, eps=1e-6, pow2=0):
    return b.load().b2g_rmsnorm_q8(X, R, W, H, Q, s, rstd, M, N, ldx, ldr, ldh, ldq, dtype, w, q, eps,
                                   pow2, None)


def gemm(b, A=P, B=P, C=P, M=4, N=8, K=16, lda=16, ldb=16, ldc=8, dtype=5, sa=P, sb=P, bias=P, c=4):
    return b.load().b2g_gemm_q8(A, B, C, M, N, K, lda, ldb, ldc, dtype, sa, sb, bias, c, None)


def wgrad(b, dY=P, Q=P, s=P, dW=P, M=4, N=8, K=16, ldy=8, ldq=16, ldw=16, dtype=1, q=5, acc=0, c=4):
    return b.load().b2g_wgrad_q8(dY, Q, s, dW, M, N, K, ldy, ldq, ldw, dtype, q, acc, c, None)


def bwd(b, dY=P, X=P, xs=P, W=P, rstd=P, dR=P, dX=2 * P, dw=P, M=4, N=8, ldy=8, ldx=8, ldr=8, lddx=8,
        dtype=1, x=5, w=1):
    return b.load().b2g_rmsnorm_bwd_q8(dY, X, xs, W, rstd, dR, dX, dw, M, N, ldy, ldx, ldr, lddx, dtype,
                                       x, w, None)


REFUSED = [
    (quantize, dict(dtype=2)), (quantize, dict(dtype=5)), (quantize, dict(q=3)), (quantize, dict(q=1)),
    (quantize, dict(M=-1)), (quantize, dict(N=-1)), (quantize, dict(N=0)), (quantize, dict(ldx=7)),
    (quantize, dict(ldq=7)), (quantize, dict(X=None)), (quantize, dict(Q=None)), (quantize, dict(s=None)),
    (dequantize, dict(dtype=5)), (dequantize, dict(q=4)), (dequantize, dict(ldx=7)),
    (dequantize, dict(s=None)), (dequantize, dict(Q=None)), (dequantize, dict(X=None)),
    (norm, dict(dtype=3)), (norm, dict(w=5)), (norm, dict(q=0)), (norm, dict(eps=-1.0)),
    (norm, dict(eps=float("nan"))), (norm, dict(N=0)), (norm, dict(ldr=7)), (norm, dict(ldh=7)),
    (norm, dict(W=None)), (norm, dict(X=None)), (norm, dict(Q=None)), (norm, dict(s=None)),
    (norm, dict(H=P, ldh=9)),
    (gemm, dict(dtype=0)), (gemm, dict(dtype=3)), (gemm, dict(c=5)), (gemm, dict(M=-1)),
    (gemm, dict(lda=15)), (gemm, dict(ldb=15)), (gemm, dict(ldc=7)), (gemm, dict(A=None)),
    (gemm, dict(B=None)), (gemm, dict(C=None)), (gemm, dict(K=131072, lda=131072, ldb=131072)),
    (wgrad, dict(dtype=4)), (wgrad, dict(q=0)), (wgrad, dict(c=2)), (wgrad, dict(acc=1, c=1)),
    (wgrad, dict(ldy=7)), (wgrad, dict(ldq=15)), (wgrad, dict(ldw=15)), (wgrad, dict(dY=None)),
    (wgrad, dict(Q=None)), (wgrad, dict(s=None)), (wgrad, dict(dW=None)), (wgrad, dict(K=-1)),
    (bwd, dict(dtype=2)), (bwd, dict(x=3)), (bwd, dict(w=5)), (bwd, dict(xs=None)), (bwd, dict(x=1)),
    (bwd, dict(dY=None)), (bwd, dict(X=None)), (bwd, dict(W=None)), (bwd, dict(rstd=None)),
    (bwd, dict(dX=None)), (bwd, dict(ldr=7)), (bwd, dict(dX=P, lddx=9)), (bwd, dict(M=-1)),
]


@pytest.mark.parametrize("call,bad", REFUSED, ids=["%s-%s" % (c.__name__, "-".join(map(str, k))) for c, k in REFUSED])
def test_refused(b2g, call, bad):
    assert call(b2g, **bad) == b2g.ERR_INVALID_ARG
    assert b2g.load().b2g_last_error_string()


class Packed:
    """The library with the six operators called through b2g_call_q8, and the words of the last call."""
    CALLS = ["b2g_quantize_q8", "b2g_dequantize_q8", "b2g_rmsnorm_q8", "b2g_gemm_q8", "b2g_wgrad_q8",
             "b2g_rmsnorm_bwd_q8"]

    def __init__(self, b2g):
        self.lib = b2g.load()

    def load(self):
        return self

    def __getattr__(self, name):
        import struct
        def call(*args):
            form = "".join("d" if isinstance(a, float) else "q" for a in args)
            self.words = struct.pack(form, *(a or 0 for a in args))
            return self.lib.b2g_call_q8(self.CALLS.index(name), self.words)
        return call


@pytest.mark.parametrize("call,bad", REFUSED, ids=["%s-%s" % (c.__name__, "-".join(map(str, k))) for c, k in REFUSED])
def test_refused_packed(b2g, call, bad):
    """The packed form refuses what the call itself refuses, with its message."""
    assert call(b2g, **bad) == b2g.ERR_INVALID_ARG
    want = b2g.load().b2g_last_error_string()
    assert call(Packed(b2g), **bad) == b2g.ERR_INVALID_ARG
    assert b2g.load().b2g_last_error_string() == want


def test_packed_calls(b2g):
    p = Packed(b2g)
    assert quantize(p, M=0) == b2g.OK and len(p.words) == 8 * 11
    assert dequantize(p, M=0) == b2g.OK and len(p.words) == 8 * 10
    assert norm(p, M=0) == b2g.OK and len(p.words) == 8 * 19
    assert gemm(p, M=0) == b2g.OK and len(p.words) == 8 * 15
    assert wgrad(p, N=0) == b2g.OK and len(p.words) == 8 * 15
    assert bwd(p, N=0) == b2g.OK and len(p.words) == 8 * 18
    assert p.lib.b2g_call_q8(6, p.words) == b2g.ERR_INVALID_ARG
    assert p.lib.b2g_call_q8(-1, p.words) == b2g.ERR_INVALID_ARG
    assert p.lib.b2g_call_q8(0, None) == b2g.ERR_INVALID_ARG


def test_binding_packs_every_argument_in_its_place(b2g, monkeypatch):
    """What the binding packs is what the calls take: distinct values, compared word by word."""
    import struct
    seen = []
    class Lib:
        def b2g_call_q8(self, call, words):
            seen.append((call, words))
            return b2g.OK
    monkeypatch.setattr(b2g, "load", lambda: Lib())
    monkeypatch.setattr(b2g, "_device", lambda: None)
    q = lambda *a: struct.pack("%dq" % len(a), *a)
    b2g.quantize_q8(11, 12, 13, 4, 5, dtype=1, q_dtype=2, pow2=True, ldx=6, ldq=7, stream=99)
    b2g.dequantize_q8(11, 12, 13, 4, 5, dtype=1, q_dtype=2, ldq=6, ldx=7, stream=99)
    b2g.rmsnorm_q8(11, 12, 13, 14, 4, 5, dtype=1, q_dtype=2, R=15, H=16, rstd=17, w_dtype=4, eps=0.5, pow2=False,
                   ldx=21, ldr=22, ldh=23, ldq=24, stream=99)
    b2g.gemm_q8(11, 12, 13, 4, 5, 6, dtype=2, a_scale=14, b_scale=15, bias=16, c_dtype=1, lda=21, ldb=22, ldc=23, stream=99)
    b2g.wgrad_q8(11, 12, 13, 14, 4, 5, 6, dtype=0, q_dtype=2, accumulate=True, c_dtype=4, ldy=21, ldq=22, ldw=23, stream=99)
    b2g.rmsnorm_bwd_q8(11, 12, 13, 14, 15, 16, 17, 4, 5, dtype=0, x_dtype=2, w_dtype=1, dres=18, ldy=21, ldx=22, ldr=23,
                       lddx=24, stream=99)
    b2g.gemm_q8(11, 12, 13, 4, 5, 6, stream=99)
    assert seen == [
        (0, q(11, 12, 13, 4, 5, 6, 7, 1, 2, 1, 99)),
        (1, q(11, 12, 13, 4, 5, 6, 7, 2, 1, 99)),
        (2, q(11, 15, 12, 16, 13, 14, 17, 4, 5, 21, 22, 23, 24, 1, 4, 2) + struct.pack("d", 0.5) + q(0, 99)),
        (3, q(11, 12, 13, 4, 5, 6, 21, 22, 23, 2, 14, 15, 16, 1, 99)),
        (4, q(11, 12, 13, 14, 4, 5, 6, 21, 22, 23, 0, 2, 1, 4, 99)),
        (5, q(11, 12, 13, 14, 15, 18, 16, 17, 4, 5, 21, 22, 23, 24, 0, 2, 1, 99)),
        (3, q(11, 12, 13, 4, 5, 6, 6, 6, 5, 5, 0, 0, 0, 4, 99)),
    ]


def test_empty_calls_need_no_device(b2g):
    assert quantize(b2g, M=0, X=None, Q=None, s=None) == b2g.OK
    assert dequantize(b2g, M=0, Q=None) == b2g.OK
    assert dequantize(b2g, N=0, Q=None) == b2g.OK
    assert norm(b2g, M=0, X=None) == b2g.OK
    assert gemm(b2g, M=0, A=None) == b2g.OK
    assert gemm(b2g, N=0, B=None) == b2g.OK
    assert b2g.last_path() == b2g.PATH_EMPTY
    assert wgrad(b2g, N=0, dY=None) == b2g.OK
    assert wgrad(b2g, K=0, Q=None) == b2g.OK
    assert bwd(b2g, M=0, dY=None, dw=None) == b2g.OK
    assert bwd(b2g, N=0, dY=None) == b2g.OK


def test_binding_refuses_wrong_tensors(b2g):
    """The Python binding checks the type and the place of torch tensors before any library call."""
    torch = pytest.importorskip("torch")
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    q = torch.zeros(4, 8, dtype=torch.int8)
    s = torch.zeros(4)
    with pytest.raises(b2g.B2GError, match="type code"):
        b2g.quantize_q8(x, q, s, 4, 8, dtype=b2g.DTYPE_F16)
    with pytest.raises(b2g.B2GError, match="not on a GPU"):
        b2g.quantize_q8(x, q, s, 4, 8, dtype=b2g.DTYPE_BF16)
    with pytest.raises(TypeError):
        b2g.quantize_q8("x", q, s, 4, 8)

"""GPU tests of the 8-bit layer's products: sums of many tokens, scales, and launches that fail."""
import pytest

from test_q8_gpu import BF16, E4M3, F16, F32, I8, NAMES, half_step, q8_matrix, scales, tt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("M,N,K", [(8192, 128, 3840), (4096, 1024, 1024), (8192, 3840, 128), (3000, 2048, 256), (20001, 264, 520)])
def test_weight_gradient_split_over_ctas_keeps_fp32(b2g, cuda, M, N, K, dt):
    """Sums split over CTAs, whose launches each take a part of the tokens: at most 1e-6 off 64 bits (2-norm), or
    1.5 times what the fp32 product is.  An accumulator's error grows by about 1.15e-9 a token and
    may sum 768 of them (8.8e-7); the fp32 additions of the parts are below 1e-7 on top."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(M)
    dY = torch.randn(M, N, generator=g, device="cuda").to(tt(torch, dt))
    Q = torch.randn(M, K, generator=g, device="cuda").mul_(30).clamp_(-127, 127).round_().to(torch.int8)
    s = scales(torch, M, 5, pow2=True)
    dW = torch.zeros(N, K, device="cuda")
    b2g.wgrad_q8(dY, Q, s, dW, M, N, K, dtype=dt)
    x = Q.float() * s[:, None]
    ref = dY.double().t() @ x.double()
    rel = lambda v: float((v.double() - ref).norm() / ref.norm())
    assert rel(dW) <= max(1e-6, 1.5 * rel(dY.float().t() @ x)), rel(dW)
    assert b2g.device_status() == 0


def test_failed_launch_leaves_no_error_behind(b2g, cuda):
    """A product whose launch the driver refuses (the legacy stream while a blocking stream records a graph)
    reports it; the next operator of the thread, a row kernel, does not report it again."""
    torch = cuda
    runtime = pytest.importorskip("cuda.bindings.runtime")
    A, B = (torch.ones(n, 2048, dtype=torch.int8, device="cuda") for n in (1, 512))
    C = torch.zeros(1, 512, device="cuda")
    x = torch.full((4, 64), 127.0, device="cuda")
    Q, s = torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    err, stream = runtime.cudaStreamCreate()
    assert int(err) == 0
    err, = runtime.cudaStreamBeginCapture(stream, runtime.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal)
    assert int(err) == 0
    try:
        with pytest.raises(b2g.B2GError, match="gemm_q8_few_kernel"):
            b2g.gemm_q8(A, B, C, 1, 512, 2048, stream=0)
    finally:
        runtime.cudaStreamEndCapture(stream)
        runtime.cudaStreamDestroy(stream)
    b2g.quantize_q8(x, Q, s, 4, 64, dtype=b2g.DTYPE_F32, stream=0)
    b2g.gemm_q8(A, B, C, 1, 512, 2048, stream=0)
    torch.cuda.synchronize()
    assert bool((Q == 127).all()) and bool((s == 1).all()) and bool((C == 2048).all())


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("K", [1, 2, 3])
@pytest.mark.parametrize("M", [9, 200])
def test_products_of_narrow_operands_at_odd_bases(b2g, cuda, M, K, q):
    """Contiguous operands of one to three columns, one byte past a word's start: sums of up to three products of
    small integers, exact in every type."""
    torch = cuda
    def narrow(rows, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        buf = torch.zeros(rows * K + 16, dtype=torch.int8, device="cuda").view(tt(torch, q))
        v = buf[1:1 + rows * K].view(rows, K)
        v.copy_(torch.randint(-8, 9, (rows, K), generator=g, device="cuda").float())
        return v
    N = 130
    A, B = narrow(M, 1), narrow(N, 2)
    C = torch.zeros(M, N, device="cuda")
    b2g.gemm_q8(A, B, C, M, N, K, dtype=q)
    assert torch.equal(C, A.float() @ B.float().t())
    # the same in the weight gradient: dY of one to three columns, two bytes past a word's start
    y = torch.zeros(M * K + 8, dtype=torch.bfloat16, device="cuda")[1:1 + M * K].view(M, K)
    y.copy_(torch.randint(-3, 4, (M, K), device="cuda"))
    X = torch.randint(-8, 9, (M, 24), device="cuda").float().to(tt(torch, q))
    dW = torch.zeros(K, 24, device="cuda")
    b2g.wgrad_q8(y, X, torch.ones(M, device="cuda"), dW, M, K, 24, q_dtype=q)
    assert torch.equal(dW, y.float().t() @ X.float())
    assert b2g.device_status() == 0


@pytest.mark.parametrize("ld", [1 << 41, (1 << 41) + 3])
def test_the_pitch_of_a_single_row_does_not_matter(b2g, cuda, ld):
    """One token, one output channel, one row of dY or dW: any leading dimension, past what TMA can address."""
    torch = cuda
    ones = lambda *s, t=torch.int8: torch.ones(*s, dtype=t, device="cuda")
    C = torch.zeros(1, 4096, device="cuda")
    b2g.gemm_q8(ones(1, 4096), ones(4096, 4096), C, 1, 4096, 4096, lda=ld, ldc=ld)
    assert bool((C == 4096).all())
    C = torch.zeros(300, 1, device="cuda")
    b2g.gemm_q8(ones(300, 520), ones(1, 520), C, 300, 1, 520, ldb=ld)
    assert bool((C == 520).all())
    dW = torch.zeros(264, 520, device="cuda")
    b2g.wgrad_q8(ones(1, 264, t=torch.bfloat16), ones(1, 520), torch.ones(1, device="cuda"), dW, 1, 264, 520, ldy=ld, ldq=ld)
    assert bool((dW == 1).all())
    dW = torch.zeros(1, 520, device="cuda")
    b2g.wgrad_q8(ones(300, 1, t=torch.bfloat16), ones(300, 520), torch.ones(300, device="cuda"), dW, 300, 1, 520, ldw=ld)
    assert bool((dW == 300).all())
    x, q, s = ones(1, 520, t=torch.bfloat16), ones(1, 520), torch.ones(1, device="cuda")
    b2g.quantize_q8(x, q, s, 1, 520, dtype=BF16, ldx=ld, ldq=ld)
    assert bool((q == 127).all()) and b2g.device_status() == 0


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("dt,c", [(BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)], ids=["bf16-f32", "f16-f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(70, 130, 264), (1500, 520, 392), (5000, 264, 1040)])
def test_weight_gradient_with_ordinary_scales(b2g, cuda, M, N, K, dt, c, q):
    """Scales that are no powers of two: q * scale is rounded to dY's type before the product, half a step of it
    (2^-8 relative in bf16, 2^-11 in fp16, whose subnormals add 2^-25) in every term, and no more."""
    torch = cuda
    u = 2.0 ** -24
    dY = (torch.randn(M, N, device="cuda") * 0.1).to(tt(torch, dt))
    _, Q = q8_matrix(torch, M, K, q, 7)
    s = scales(torch, M, 3)
    dW = torch.zeros(N, K, dtype=tt(torch, c), device="cuda")
    b2g.wgrad_q8(dY, Q, s, dW, M, N, K, dtype=dt, q_dtype=q, c_dtype=c)
    x, y = Q.double() * s.double()[:, None], dY.double()
    ref, size = y.t() @ x, y.abs().t() @ x.abs()
    tol = (half_step(torch, dt) + u) * size + (2.0 ** -25 * y.abs().sum(0)[:, None] if dt == F16 else 0)  # the rounding of q * scale
    tol = tol + 2 * (M + 1) * u * size * 1.01 + half_step(torch, c) * ref.abs() + (2.0 ** -25 if c == F16 else 0)
    err = (dW.double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    assert b2g.device_status() == 0

"""GPU tests of the 8-bit layer's products: sums of many tokens, scales, and launches that fail."""
import pytest

from test_q8_gpu import BF16, F16, NAMES, scales, tt

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

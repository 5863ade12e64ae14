"""GPU tests of the 8-bit layer's row kernels where rows pass through a ring of buffers in shared memory."""
import pytest

from gpu_util import options
from test_q8_gpu import BF16, E4M3, F16, F32, I8, NAMES, check_bwd, check_norm, grid, pad_untouched, padded, row_quant64, rows, tt

pytestmark = pytest.mark.gpu


def check_quantize(torch, b2g, M, N, dt, q, pad=0):
    _, x = padded(torch, M, N, dt, pad, rows(torch, M, N, N))
    (buf, Q), s = padded(torch, M, N, q, pad), torch.zeros(M, device="cuda")
    b2g.quantize_q8(x, Q, s, M, N, dtype=dt, q_dtype=q)
    t, want = row_quant64(torch, x.double(), q, False)
    assert torch.equal(s.double(), want)
    r, half = grid(torch, t, q)
    if dt != F32:
        assert torch.equal(Q.double(), r)
    else:  # the product with qmax and the quotient round once each
        assert bool(((Q.double() - t).abs() <= half * (1 + 2 ** -20) + 4 * 2.0 ** -24 * t.abs()).all())
    assert pad_untouched(torch, buf, N)


# Stages of 56832, 75776 and 113664 bytes: four, three and two of them fill the shared memory to its
# last byte, so that there is no room left for their barriers.
@pytest.mark.parametrize("dt,N", [(BF16, 14208), (BF16, 18944), (F16, 28416), (F32, 7104), (F32, 9472), (F32, 14208)])
def test_norm_rings_that_fill_shared_memory(b2g, cuda, dt, N):
    check_norm(cuda, b2g, 300, N, dt, I8, True, False, 0)


@pytest.mark.parametrize("N", [14193, 14196, 14200])
def test_norm_odd_rings_that_fill_shared_memory(b2g, cuda, N):
    check_norm(cuda, b2g, 5, N, BF16, E4M3, True, False, 5)


@pytest.mark.parametrize("dt,N", [(BF16, 28416), (F32, 14208), (F32, 14203)])
def test_quantize_rings_that_fill_shared_memory(b2g, cuda, dt, N):
    check_quantize(cuda, b2g, 300, N, dt, I8)


@pytest.mark.parametrize("dt,xt,res,N", [(F32, F32, True, 4736), (F32, F32, True, 9472), (BF16, BF16, False, 14208),
                                         (BF16, BF16, True, 9472), (F32, I8, True, 6307)])
def test_backward_rings_that_fill_shared_memory(b2g, cuda, dt, xt, res, N):
    check_bwd(cuda, b2g, 7, N, dt, xt, res)


def lost_copies(torch, b2g, call):
    """Runs `call` with the rings' copies left out (test option): its waits run out after 2 ms, it ends and
    says so, and the next call is sound."""
    with options(b2g, fault_flags=1, timeout_ns=2000000):
        call()
        assert b2g.device_status() == 8
    assert b2g.device_status() == 0


# (M, N, pitch): aligned rows and rows of any alignment, over a hundred of them a block
RINGS = [(60000, 1024, 1024), (60000, 1027, 1029)]


@pytest.mark.parametrize("M,N,pitch", RINGS)
def test_rows_behind_a_lost_copy_are_marked(b2g, cuda, M, N, pitch):
    """Every row whose copy did not arrive, or that came after one in its block, has the scale NaN and zeros,
    or a NaN gradient: also those whose buffer would have been filled several times by then."""
    torch = cuda
    x = torch.ones(M, pitch, dtype=torch.bfloat16, device="cuda")[:, :N]
    w = torch.ones(N, dtype=torch.bfloat16, device="cuda")
    Q, s = torch.ones(M, pitch, dtype=torch.int8, device="cuda")[:, :N], torch.ones(M, device="cuda")
    h, rstd = torch.ones(M, pitch, dtype=torch.bfloat16, device="cuda")[:, :N], torch.ones(M, device="cuda")
    for res in (None, x):
        Q.fill_(1)
        lost_copies(torch, b2g, lambda: b2g.rmsnorm_q8(x, w, Q, s, M, N, dtype=BF16, R=res, H=h, rstd=rstd))
        assert bool(torch.isnan(s).all()) and bool(torch.isnan(rstd).all()) and not Q.any()
        assert bool(torch.isnan(h).all())
        h.fill_(1)
    Q.fill_(1)
    lost_copies(torch, b2g, lambda: b2g.quantize_q8(x, Q, s, M, N, dtype=BF16))
    assert bool(torch.isnan(s).all()) and not Q.any()
    d, ones = torch.ones(M, pitch, dtype=torch.bfloat16, device="cuda")[:, :N], torch.ones(M, device="cuda")
    lost_copies(torch, b2g, lambda: b2g.rmsnorm_bwd_q8(x, Q, ones, w, ones, d, None, M, N, dtype=BF16))
    assert bool(torch.isnan(d).all())
    b2g.quantize_q8(x, Q, s, M, N, dtype=BF16)
    assert bool((Q == 127).all()) and b2g.device_status() == 0


# the kernels that hold a row in registers, that unpack it twice, and that take any alignment
@pytest.mark.parametrize("N,pitch", [(1024, 1024), (16384, 16384), (1027, 1029)])
def test_weight_gradient_of_the_norm_tells_of_a_lost_copy(b2g, cuda, N, pitch):
    """dw is a sum over all rows: NaN where one of them did not arrive."""
    torch = cuda
    M = 3000
    y = torch.ones(M, pitch, dtype=torch.bfloat16, device="cuda")[:, :N]
    x = torch.ones(M, pitch, dtype=torch.int8, device="cuda")[:, :N]
    w, ones, dw = torch.ones(N, dtype=torch.bfloat16, device="cuda"), torch.ones(M, device="cuda"), torch.zeros(N, device="cuda")
    d = torch.ones(M, pitch, dtype=torch.bfloat16, device="cuda")[:, :N]
    lost_copies(torch, b2g, lambda: b2g.rmsnorm_bwd_q8(y, x, ones, w, ones, d, dw, M, N, dtype=BF16))
    assert bool(torch.isnan(dw).all()) and bool(torch.isnan(d).all())
    b2g.rmsnorm_bwd_q8(y, x, ones, w, ones, d, dw, M, N, dtype=BF16)
    assert bool((dw == M).all()) and not d.any() and b2g.device_status() == 0


def test_least_time_limit(b2g, cuda):
    """With a limit of 1 ns a wait may give up at any time, with copies in flight: calls then end with code 8
    (or a product's) or with the right rows, and no later call is disturbed."""
    torch = cuda
    from test_q8_gpu import check_gemm
    M, N = 4000, 2048
    x, w = rows(torch, M, N, 1).to(torch.bfloat16), torch.ones(N, dtype=torch.bfloat16, device="cuda")
    Q, s, rstd = torch.zeros(M, N, dtype=torch.int8, device="cuda"), torch.zeros(M, device="cuda"), torch.ones(M, device="cuda")
    d, dw = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda"), torch.zeros(N, device="cuda")
    A, C = torch.ones(100, N, dtype=torch.int8, device="cuda"), torch.zeros(100, M, device="cuda")
    def step():
        b2g.rmsnorm_q8(x, w, Q, s, M, N, dtype=BF16, R=x, rstd=rstd)
        b2g.rmsnorm_bwd_q8(x, Q, s, w, rstd, d, dw, M, N, dtype=BF16)
        b2g.gemm_q8(A, Q, C, 100, M, N)
        return [t.clone() for t in (Q, s, rstd, d, dw, C)]
    want = step()
    assert b2g.device_status() == 0
    with options(b2g, timeout_ns=1):
        for _ in range(20):
            got = step()
            assert b2g.device_status() != 0 or all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    check_gemm(torch, b2g, 100, 520, 1184, I8, F32)
    assert b2g.device_status() == 0


# (most blocks an SM, N, pad): nine rows and more a block, so that each of up to four buffers is refilled twice; rows of
# whole 16-byte vectors of every kernel width, and rows of any alignment
MANY = [(14, 1024, 0), (9, 1544, 0), (7, 4096, 8), (4, 8192, 0), (2, 16384, 0), (8, 1001, 5), (8, 2047, 0), (4, 4001, 2), (2, 8191, 0),
        (1, 16001, 0)]


def rows_of_many(torch, blocks):
    return 9 * blocks * torch.cuda.get_device_properties(0).multi_processor_count + 7


@pytest.mark.parametrize("dt", [F16, BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("blocks,N,pad", MANY)
def test_many_rows_into_8_bits(b2g, cuda, blocks, N, pad, dt):
    M = rows_of_many(cuda, blocks)
    q = I8 if dt != F16 else E4M3
    check_norm(cuda, b2g, M, N, dt, q, True, False, pad)
    check_norm(cuda, b2g, M, N, dt, q, True, False, pad, inplace=True, seed=3)
    check_norm(cuda, b2g, M, N, dt, q, False, True, pad, seed=6)
    check_quantize(cuda, b2g, M, N, dt, q, pad)
    assert b2g.device_status() == 0


@pytest.mark.parametrize("xt", [I8, E4M3, None], ids=["i8", "e4m3", "same"])
@pytest.mark.parametrize("dt", [BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("blocks,N,pad", MANY)
def test_many_rows_backward(b2g, cuda, blocks, N, pad, dt, xt):
    M, xt = rows_of_many(cuda, blocks), dt if xt is None else xt
    check_bwd(cuda, b2g, M, N, dt, xt, True, pad)
    check_bwd(cuda, b2g, M, N, dt, xt, False, pad, inplace=True)
    assert b2g.device_status() == 0


@pytest.mark.parametrize("blocks,N,pad", [(14, 1024, 0), (4, 8192, 0), (8, 1001, 5), (2, 8191, 0)])
def test_many_rows_in_place_and_again(b2g, cuda, blocks, N, pad):
    """H in X, dX in dY (with dR) and dX in dR give what separate outputs do, bit for bit, time after time."""
    torch = cuda
    M = rows_of_many(torch, blocks)
    bf = torch.bfloat16
    new = lambda t=bf: torch.zeros(M, N + pad, dtype=t, device="cuda")[:, :N]
    x, y, r = (new() for _ in range(3))
    for i, t in enumerate((x, y, r)):
        t.copy_(rows(torch, M, N, i))
    w = (1 + 0.2 * torch.randn(N, device="cuda")).to(bf)
    def norm(src, dst):
        q, s, rstd = new(torch.int8), torch.zeros(M, device="cuda"), torch.zeros(M, device="cuda")
        b2g.rmsnorm_q8(src, w, q, s, M, N, dtype=BF16, H=dst, rstd=rstd)
        return q, s, rstd
    h = new()
    q, s, rstd = norm(x, h)
    assert torch.equal(h, x)
    def bwd(dy, dr, dst):
        dw = torch.zeros(N, device="cuda")
        b2g.rmsnorm_bwd_q8(dy, q, s, w, rstd, dst, dw, M, N, dtype=BF16, dres=dr)
        return dst.clone(), dw
    want = bwd(y, r, new())
    for _ in range(3):
        again = new()
        again.copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(norm(again, again), (q, s, rstd))) and torch.equal(again, x)
        for at in (0, 1):
            a, b = new(), new()
            a.copy_(y)
            b.copy_(r)
            assert all(torch.equal(g, v) for g, v in zip(bwd(a, b, (a, b)[at]), want))
    assert b2g.device_status() == 0

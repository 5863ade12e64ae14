"""GPU tests of the 8-bit operators against their formulas in 64 bits.

u = 2^-24 is half a step of fp32.  A sum of n fp32 terms in any order is off by at most
n * u * sum|terms| to first order (2 u a step where the tensor core truncates instead of rounding); a
rounding to a 16-bit type by half a step of it, eps(t) / 2 relative.
"""
import numpy as np
import pytest

from gpu_util import options

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F16, BF16, E4M3, F32, I8 = 0, 1, 2, 4, 5
NAMES = {F16: "f16", BF16: "bf16", E4M3: "e4m3", F32: "f32", I8: "i8"}
QMAX = {I8: 127.0, E4M3: 448.0}


def tt(torch, code):
    return {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32, I8: torch.int8,
            E4M3: torch.float8_e4m3fn}[code]


def half_step(torch, code):
    return 0.0 if code == F32 else torch.finfo(tt(torch, code)).eps / 2


def padded(torch, M, N, code, pad, fill=None):
    """An M x N view of a buffer of row pitch N + pad whose pad columns hold NaN (or 77)."""
    if code in (I8, E4M3):
        buf = torch.full((M, N + pad), 77, dtype=torch.int8, device="cuda").view(tt(torch, code))
    else:
        buf = torch.full((M, N + pad), float("nan"), dtype=tt(torch, code), device="cuda")
    if fill is not None:
        buf[:, :N] = fill.to(buf.dtype)
    return buf, buf[:, :N]


def pad_untouched(torch, buf, N):
    p = buf[:, N:]
    if p.numel() == 0:
        return True
    if p.dtype.itemsize == 1:
        return bool((p.contiguous().view(torch.int8) == 77).all())
    return bool(torch.isnan(p).all())


def rows(torch, M, N, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ch = torch.exp(torch.randn(N, generator=g, device="cuda"))
    return torch.randn((M, N), generator=g, device="cuda") * ch


def q8_matrix(torch, M, K, code, seed, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if code == I8:
        v = torch.randint(-128, 128, (M, K), generator=g, device="cuda").to(torch.int8)
    else:
        v = torch.randn((M, K), generator=g, device="cuda").to(torch.float8_e4m3fn)
    buf, view = padded(torch, M, K, code, pad)
    view.copy_(v)
    return buf, view


def scales(torch, n, seed, pow2=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    e = torch.randint(-9, 3, (n,), generator=g, device="cuda").float()
    s = torch.exp2(e)
    return s if pow2 else s * (1 + torch.rand(n, generator=g, device="cuda"))


def grid(torch, t, q):
    """t (fp64) rounded to the 8-bit type, ties to even; also half a step of the type at t."""
    if q == I8:
        return torch.round(t), torch.full_like(t, 0.5)
    a = t.abs().clamp(min=2.0 ** -6)
    e = (a.view(torch.int64) >> 52) - 1023
    step = ((e - 3 + 1023) << 52).view(torch.float64)
    return (torch.round(t / step) * step).clamp(-448, 448), step / 2


def row_quant64(torch, y, q, pow2):
    """(t, scale): the unrounded 8-bit values and the fp32 scale of fp64 rows y (fp32 values)."""
    top = y.abs().amax(1)
    s = (top / torch.full_like(top, QMAX[q])).float().clamp(min=2.0 ** -126).double()
    if pow2:
        m, e = torch.frexp(s.cpu())
        s = torch.ldexp(torch.ones_like(m), e - (m == 0.5).int()).to(y.device)
        return y / s[:, None], s
    low = top < QMAX[q] * 2.0 ** -126
    t = torch.where(low[:, None], y / s[:, None], y * QMAX[q] / torch.where(low, 1.0, top)[:, None])
    return t, s


# ---------------------------------------------------------------- rows into 8 bits
SHAPES = [(1, 1), (1, 8192), (3, 7), (5, 33), (2, 1000), (7, 1024), (130, 2056), (3, 4097), (2, 8200),
          (2, 16384), (1, 40000), (700, 128), (2000, 264)]


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("dt", [F16, BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("pad", [0, 5])
def test_quantize(b2g, cuda, M, N, dt, q, pad):
    """16-bit rows: every 8-bit value and scale is the formula's.  fp32 rows: the product with
    qmax and the quotient round once each, so t may be 3 u off before it is rounded."""
    torch = cuda
    xb, x = padded(torch, M, N, dt, pad, rows(torch, M, N, M * N + dt))
    for pow2 in (False, True):
        qb, qv = padded(torch, M, N, q, pad)
        s = torch.full((M,), float("nan"), device="cuda")
        b2g.quantize_q8(x, qv, s, M, N, dtype=dt, q_dtype=q, pow2=pow2)
        t, want = row_quant64(torch, x.double(), q, pow2)
        assert torch.equal(s.double(), want)
        r, half = grid(torch, t, q)
        if dt != F32:
            assert torch.equal(qv.double(), r)
        assert bool(((qv.double() - t).abs() <= half * (1 + 2 ** -20) + 4 * U * t.abs()).all())
        assert pad_untouched(torch, qb, N)
        vb, v = padded(torch, M, N, BF16, pad)
        b2g.dequantize_q8(qv, s, v, M, N, dtype=BF16, q_dtype=q)
        assert torch.equal(v, (qv.float() * s[:, None]).to(torch.bfloat16))
        assert pad_untouched(torch, vb, N)


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("N", [64, 1001])
def test_quantize_special_rows(b2g, cuda, N, q):
    """Zero rows, ties, the type's largest and least values, NaN and infinities."""
    torch = cuda
    big, tiny = 3.3895e38, 9.2e-41
    base = torch.linspace(-1, 1, N, device="cuda")
    X = torch.stack([base * 0, base * big, base * tiny, torch.full_like(base, 127.0), base * 2.0 ** -120,
                     torch.arange(N, device="cuda") % 128 / 2.0, base, base, base]).to(torch.bfloat16)
    X[6, N // 2] = float("nan")
    X[7, N - 1] = float("inf")
    X[8, 0] = -float("inf")
    M = X.shape[0]
    for pow2 in (False, True):
        Q = torch.full((M, N), 77, dtype=torch.int8, device="cuda").view(tt(torch, q))
        s = torch.zeros(M, device="cuda")
        b2g.quantize_q8(X, Q, s, M, N, dtype=BF16, q_dtype=q, pow2=pow2)
        t, want = row_quant64(torch, X[:6].double(), q, pow2)
        assert torch.equal(s[:6].double(), want)
        assert torch.equal(Q[:6].double(), grid(torch, t, q)[0])
        assert bool(torch.isnan(s[6:]).all()) and not Q[6:].float().any()
    V = torch.zeros(M, N, device="cuda")
    b2g.dequantize_q8(Q, s, V, M, N, dtype=F32, q_dtype=q)
    assert bool(torch.isnan(V[6:]).all()) and bool(torch.isfinite(V[:6]).all())


# ---------------------------------------------------------------- norm
def check_norm(torch, b2g, M, N, dt, q, res, pow2, pad, w_dt=None, inplace=False, eps=1e-6, seed=0):
    w_dt = dt if w_dt is None else w_dt
    _, x = padded(torch, M, N, dt, pad, rows(torch, M, N, seed + 1))
    rb, r = padded(torch, M, N, dt, pad, rows(torch, M, N, seed + 2)) if res else (None, None)
    w = (1 + 0.2 * torch.randn(N, device="cuda")).to(tt(torch, w_dt))
    h32 = x.float() + r.float() if res else x.float()
    hb, h = (rb, r) if inplace else padded(torch, M, N, dt, pad) if res else (None, None)
    qb, qv = padded(torch, M, N, q, pad)
    s, rstd = torch.zeros(M, device="cuda"), torch.zeros(M, device="cuda")
    b2g.rmsnorm_q8(x, w, qv, s, M, N, dtype=dt, q_dtype=q, R=r, H=h, rstd=rstd, w_dtype=w_dt, eps=eps, pow2=pow2)
    if res:
        assert torch.equal(h, h32.to(h.dtype))
        assert pad_untouched(torch, hb, N)
    assert pad_untouched(torch, qb, N)
    h64 = h32.double()
    want = 1 / torch.sqrt((h64 * h64).mean(1) + eps)
    # sum of N positive terms (relative N u), mean, eps, root and reciprocal: half of the sum's error reaches rstd
    rel = (N / 2 + 4) * U
    assert bool(((rstd.double() - want).abs() <= rel * want).all())
    y = h64 * want[:, None] * w.double()
    rel += 4 * U  # h * w, times rstd, over qmax
    t, ws = row_quant64(torch, y, q, pow2)
    if pow2:  # a scale within rel of a power of two may go to either side of it
        near = (torch.log2(row_quant64(torch, y, q, False)[1]) % 1)
        ok = (near > 4 * rel) & (near < 1 - 4 * rel)
        assert torch.equal(s.double()[ok], ws[ok])
        t = y / s.double()[:, None]
    else:
        assert bool(((s.double() - ws).abs() <= rel * ws).all())
    half = grid(torch, t, q)[1]
    assert bool(((qv.double() - t).abs() <= half * (1 + 2 ** -20) + rel * t.abs()).all())


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("dt", [F16, BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("pad", [0, 3])
def test_norm(b2g, cuda, M, N, dt, q, pad):
    for res, pow2 in ((True, False), (False, True)):
        check_norm(cuda, b2g, M, N, dt, q, res, pow2, pad)


@pytest.mark.parametrize("w_dt", [F16, BF16, F32], ids=NAMES.get)
def test_norm_weight_types_in_place_and_eps(b2g, cuda, w_dt):
    check_norm(cuda, b2g, 9, 1032, BF16, I8, True, False, 8, w_dt=w_dt, inplace=True)
    check_norm(cuda, b2g, 9, 1031, F16, E4M3, True, False, 0, w_dt=w_dt, inplace=True, eps=0.0)


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("dt", [F16, BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("M,N,pad", [(5, 40960, 0), (400, 33024, 8), (5, 33003, 5), (310, 20001, 1)])
def test_norm_long_rows(b2g, cuda, M, N, pad, dt, q):
    """Rows too long for registers, with and without a residual, more rows than blocks among them."""
    check_norm(cuda, b2g, M, N, dt, q, res=True, pow2=False, pad=pad, inplace=pad == 8)
    check_norm(cuda, b2g, M, N, dt, q, res=False, pow2=True, pad=pad)


def test_norm_zero_and_bad_rows(b2g, cuda):
    """A row of zeros gives rstd = 1/sqrt(eps), the least scale and zeros; a NaN or infinity stays
    in its row."""
    torch = cuda
    M, N = 5, 520
    x = torch.randn(M, N, device="cuda").half()
    x[1] = 0
    x[2, 17] = float("nan")
    x[3, 519] = float("inf")
    w = torch.ones(N, device="cuda").half()
    q = torch.full((M, N), 77, dtype=torch.int8, device="cuda")
    s, rstd = torch.zeros(M, device="cuda"), torch.zeros(M, device="cuda")
    b2g.rmsnorm_q8(x, w, q, s, M, N, dtype=F16, rstd=rstd)
    assert float(s[1]) == 2.0 ** -126 and not q[1].any() and abs(float(rstd[1]) - 1000) < 0.01
    assert bool(torch.isnan(s[2:4]).all()) and not q[2:4].any()
    assert bool(torch.isfinite(s[[0, 4]]).all()) and int(q[0].abs().max()) == 127


# ---------------------------------------------------------------- scaled product
def check_gemm(torch, b2g, M, N, K, q, c, pad=0, bias=True, scaled=True, offset=0):
    _, A = q8_matrix(torch, M, K, q, M + 3 * K, pad)
    _, B = q8_matrix(torch, N, K, q, N + 5 * K, pad)
    sa = scales(torch, M + offset, 1)[offset:] if scaled else None
    sb = scales(torch, N + offset, 2)[offset:] if scaled else None
    bi = torch.randn(N + offset, device="cuda")[offset:] if bias else None
    cb, C = padded(torch, M, N, c, pad)
    b2g.gemm_q8(A, B, C, M, N, K, dtype=q, a_scale=sa, b_scale=sb, bias=bi, c_dtype=c)
    a, b = A.double(), B.double()
    s = (sa.double()[:, None] * sb.double()) if scaled else torch.ones((), dtype=torch.float64, device="cuda")
    prod = (a @ b.t()) * s
    ref = prod + (bi.double() if bias else 0)
    # conversion to fp32, two scales, bias: one rounding each; e4m3 sums 2 u a step on top
    tol = 4 * U * (prod.abs() + ref.abs()) + half_step(torch, c) * ref.abs() + (2.0 ** -25 if c == F16 else 0)
    if q == E4M3:
        tol = tol + 2 * K * U * (a.abs() @ b.abs().t()) * s
    got = C.double()
    if c == F16:  # a result of 65520 or more in size rounds to fp16's infinity: it is checked for its sign and size only
        over = ref.abs() + tol >= 65520
        assert bool((got[over] * torch.sign(ref[over]) >= ref[over].abs().clamp(max=65504.0) - tol[over]).all())
        got, ref, tol = got[~over], ref[~over], tol[~over]
    err = (got - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    assert pad_untouched(torch, cb, N)
    assert b2g.device_status() == 0


GEMMS = [(1, 1, 1), (1, 256, 512), (1, 257, 4096), (2, 300, 1000), (3, 1024, 64), (8, 512, 2048), (9, 515, 1040),
         (16, 640, 768), (17, 129, 144), (31, 512, 4112), (48, 1000, 512), (64, 4096, 1024), (65, 200, 96), (128, 520, 2064),
         (200, 1000, 272), (257, 384, 1104), (300, 2000, 4096), (1030, 513, 160), (2048, 2304, 528)]


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("M,N,K", GEMMS)
def test_gemm(b2g, cuda, M, N, K, q):
    for c, pad in ((F32, 0), (BF16, 16), (F16, 5)):
        check_gemm(cuda, b2g, M, N, K, q, c, pad)


# (CTAs per tile, tile width) of the tiles for larger batches
TILES = [(1, 128), (1, 256), (2, 256), (2, 512)]
SPLITS = [dict(split_k=1), dict(split_k=3), dict(split_k=4, cluster_fixup=0), dict(split_k=3, serial_fixup=1)]


@pytest.mark.parametrize("split", SPLITS, ids=["whole", "cluster", "parallel", "serial"])
@pytest.mark.parametrize("cg,tn", TILES)
@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
def test_gemm_tiles_and_splits(b2g, cuda, q, cg, tn, split):
    """Every tile, whole and with K split each way, with whole and ragged edges and an unaligned C."""
    with options(b2g, cta_group=cg, tile_n=tn, tail_split=0, **split):
        for M, N, K, c, pad in ((300, 1040, 1600, F32, 0), (385, 777, 2064, BF16, 16), (200, 600, 520, F16, 5)):
            check_gemm(cuda, b2g, M, N, K, q, c, pad)
            assert b2g.last_path() == (b2g.PATH_TC_1CTA if cg == 1 else b2g.PATH_TC_2CTA)


@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("M", [17, 32, 33, 64, 65, 128])
@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
def test_gemm_decoding_batches(b2g, cuda, q, M, splits):
    with options(b2g, split_k=splits):
        check_gemm(cuda, b2g, M, 520, 1184, q, F32, 0)
        check_gemm(cuda, b2g, M, 129, 1040, q, BF16, 3)
        assert b2g.last_path() == b2g.PATH_TC_1CTA


def test_gemm_few_tokens_path(b2g, cuda):
    for M, N, K in ((1, 512, 2048), (8, 100, 64), (9, 33, 16), (16, 515, 4112)):
        check_gemm(cuda, b2g, M, N, K, I8, F32)
        assert b2g.last_path() == b2g.PATH_FEW
        check_gemm(cuda, b2g, M, N, K, E4M3, F16, 16)
        assert b2g.last_path() == b2g.PATH_FEW


@pytest.mark.parametrize("M", [40, 300])
def test_gemm_wait_that_runs_out_is_reported(b2g, cuda, M):
    """With its loads left out (test option), the product's bounded wait gives up: an error word, no
    hang, and the next call is sound."""
    torch = cuda
    _, A = q8_matrix(torch, M, 1024, I8, 1)
    _, B = q8_matrix(torch, 512, 1024, I8, 2)
    C = torch.zeros(M, 512, device="cuda")
    with options(b2g, fault_flags=1, timeout_ns=2000000):
        b2g.gemm_q8(A, B, C, M, 512, 1024)
        assert b2g.device_status() != 0
    check_gemm(torch, b2g, M, 512, 1024, I8, F32)


def test_gemm_optional_vectors_and_offsets(b2g, cuda):
    """No scales, no bias, and scale vectors that are not 16-byte aligned."""
    for M in (1, 20, 150):
        check_gemm(cuda, b2g, M, 260, 256, I8, F32, bias=False, scaled=False)
        check_gemm(cuda, b2g, M, 260, 256, E4M3, BF16, offset=1)
        check_gemm(cuda, b2g, M, 260, 256, I8, BF16, bias=False, offset=3)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_gemm_int8_extremes_are_exact(b2g, cuda, M):
    """-128 * -128 over the longest K: the int32 sum does not wrap.  K = 0: C is the bias."""
    torch = cuda
    K, N = 131071, 32
    A = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    B = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    C = torch.zeros(M, N, device="cuda")
    b2g.gemm_q8(A, B, C, M, N, K)
    assert bool((C == float(np.float32(K * 16384))).all())
    bias = torch.randn(N, device="cuda")
    b2g.gemm_q8(A, B, C, M, N, 0, bias=bias, lda=K, ldb=K)
    assert torch.equal(C, bias.expand(M, N))


def test_gemm_bad_scale_stays_in_its_row(b2g, cuda):
    torch = cuda
    for M in (3, 200):
        _, A = q8_matrix(torch, M, 512, I8, 1)
        _, B = q8_matrix(torch, 256, 512, I8, 2)
        sa = torch.ones(M, device="cuda")
        sa[1] = float("nan")
        C = torch.zeros(M, 256, device="cuda")
        b2g.gemm_q8(A, B, C, M, 256, 512, a_scale=sa)
        assert bool(torch.isnan(C[1]).all()) and bool(torch.isfinite(C[[0, 2]]).all())


# ---------------------------------------------------------------- weight gradient
def check_wgrad(torch, b2g, M, N, K, dt, q, c, pad=0, acc=False):
    yb, dY = padded(torch, M, N, dt, pad, torch.randn(M, N, device="cuda") * 0.1)
    _, Q = q8_matrix(torch, M, K, q, 7, pad)
    s = scales(torch, M, 3, pow2=True)
    wb, dW = padded(torch, N, K, c, pad)
    if acc:
        dW.copy_(torch.randn(N, K, device="cuda"))
    w0 = dW.double() if acc else torch.zeros((), dtype=torch.float64, device="cuda")
    b2g.wgrad_q8(dY, Q, s, dW, M, N, K, dtype=dt, q_dtype=q, accumulate=acc, c_dtype=c)
    x = Q.double() * s.double()[:, None]
    y = dY.double()
    ref = y.t() @ x + w0
    tol = 2 * (M + 1) * U * (y.abs().t() @ x.abs()) + 2 * U * ref.abs() + half_step(torch, c) * ref.abs() + (2.0 ** -25 if c == F16 else 0)
    err = (dW.double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    assert pad_untouched(torch, wb, K)
    assert b2g.device_status() == 0


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("dt", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 256), (5, 70, 33), (63, 264, 128), (64, 128, 512), (200, 129, 1000),
                                   (1000, 256, 264), (1025, 520, 2048), (4100, 384, 136)])
def test_wgrad(b2g, cuda, M, N, K, dt, q):
    for c, pad, acc in ((F32, 0, False), (F32, 8, True), (dt, 3, False), (F32, 5, True), (dt, 16, False)):
        check_wgrad(cuda, b2g, M, N, K, dt, q, c, pad, acc)


@pytest.mark.parametrize("split", SPLITS, ids=["whole", "cluster", "parallel", "serial"])
@pytest.mark.parametrize("cg,tn", TILES)
def test_wgrad_tiles_and_splits(b2g, cuda, cg, tn, split):
    """Every tile, whole (long sums in parts) and with the tokens split each way."""
    with options(b2g, cta_group=cg, tile_n=tn, tail_split=0, **split):
        check_wgrad(cuda, b2g, 1700, 300, 1040, BF16, I8, F32, 0)
        check_wgrad(cuda, b2g, 1601, 520, 777, F16, E4M3, F32, 3, True)
        check_wgrad(cuda, b2g, 900, 264, 600, BF16, E4M3, BF16, 8)


def test_wgrad_long_sums_keep_fp32(b2g, cuda):
    """Relative error (2-norm) against 64 bits at most 1e-6, or 1.5 times that of the fp32 product where
    that is more, however many tokens are summed: the tensor core's accumulator alone is 2.4e-6 off
    at 2048."""
    torch = cuda
    for M, N, K, dt in ((2048, 1024, 1024, F16), (5000, 768, 1032, BF16), (16384, 512, 512, F16), (16384, 2048, 2048, BF16)):
        g = torch.Generator(device="cuda").manual_seed(M)
        dY = torch.randn(M, N, generator=g, device="cuda").to(tt(torch, dt))
        Q = torch.randn(M, K, generator=g, device="cuda").mul_(30).clamp_(-127, 127).round_().to(torch.int8)
        s = scales(torch, M, 5, pow2=True)
        dW = torch.zeros(N, K, device="cuda")
        b2g.wgrad_q8(dY, Q, s, dW, M, N, K, dtype=dt)
        x = Q.float() * s[:, None]
        ref = dY.double().t() @ x.double()
        rel = lambda v: float((v.double() - ref).norm() / ref.norm())
        assert rel(dW) <= max(1e-6, 1.5 * rel(dY.float().t() @ x))


@pytest.mark.parametrize("M", [96, 4096, 9000])
def test_wgrad_is_exact_on_small_integers(b2g, cuda, M):
    """Operands whose sums are integers below 2^24: every order of summation gives the same dW."""
    torch = cuda
    N, K = 392, 520
    dY = torch.randint(-1, 2, (M, N), device="cuda").to(torch.bfloat16)
    Q = torch.randint(-3, 4, (M, K), device="cuda").to(torch.int8)
    s = torch.exp2(torch.randint(0, 4, (M,), device="cuda").float())
    dW = torch.zeros(N, K, device="cuda")
    b2g.wgrad_q8(dY, Q, s, dW, M, N, K)
    ref = dY.double().t() @ (Q.double() * s.double()[:, None])
    assert torch.equal(dW.double(), ref)
    b2g.wgrad_q8(dY, Q, s, dW, M, N, K, accumulate=True)
    assert torch.equal(dW.double(), 2 * ref)


def test_wgrad_no_tokens(b2g, cuda):
    torch = cuda
    e = torch.zeros(0, 64, device="cuda")
    dW = torch.full((64, 64), 3.0, device="cuda")
    b2g.wgrad_q8(e.bfloat16(), e.to(torch.int8), e[:, 0], dW, 0, 64, 64, accumulate=True)
    assert bool((dW == 3).all())
    b2g.wgrad_q8(e.bfloat16(), e.to(torch.int8), e[:, 0], dW, 0, 64, 64)
    assert not dW.any()


# ---------------------------------------------------------------- norm backward
def check_bwd(torch, b2g, M, N, dt, xt, res, pad=0, w_dt=None, inplace=False, want_dw=True):
    w_dt = dt if w_dt is None else w_dt
    if xt in (I8, E4M3):
        _, X = q8_matrix(torch, M, N, xt, 11, pad)
        xs = scales(torch, M, 12)
        x = X.double() * xs.double()[:, None]
    else:
        _, X = padded(torch, M, N, xt, pad, rows(torch, M, N, 13))
        xs, x = None, X.double()
    rstd = (1 / torch.sqrt((x * x).mean(1) + 1e-6)).float()
    _, dY = padded(torch, M, N, dt, pad, rows(torch, M, N, 14) * 0.1)
    _, dR = padded(torch, M, N, dt, pad, rows(torch, M, N, 15) * 0.1) if res else (None, None)
    y, r = dY.double(), dR.double() if res else 0.0  # before an update in place
    w = (1 + 0.2 * torch.randn(N, device="cuda")).to(tt(torch, w_dt))
    xb, dX = (None, dR if res else dY) if inplace else padded(torch, M, N, dt, pad)
    dw = torch.full((N,), float("nan"), device="cuda") if want_dw else None
    b2g.rmsnorm_bwd_q8(dY, X, xs, w, rstd, dX, dw, M, N, dtype=dt, x_dtype=xt, w_dtype=w_dt, dres=dR)
    rs = rstd.double()[:, None]
    xh, g = x * rs, y * w.double()
    c = (g * xh).mean(1, keepdim=True)
    dx = rs * (g - xh * c)
    # g, xh, their product and the sum of N of them; then the difference, times rstd, plus dr
    tol = rs * (4 * U * (g.abs() + (xh * c).abs()) + xh.abs() * (N + 8) * U * (g * xh).abs().mean(1, keepdim=True))
    ref = dx + r
    tol = tol + 2 * U * (dx.abs() + ref.abs()) + half_step(torch, dt) * ref.abs() + (2.0 ** -25 if dt == F16 else 0)
    err = (dX.double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    if want_dw:
        assert bool(((dw.double() - (y * xh).sum(0)).abs() <= (M + 8) * U * (y * xh).abs().sum(0)).all())
    if xb is not None:
        assert pad_untouched(torch, xb, N)


@pytest.mark.parametrize("xt", [I8, E4M3, BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("dt", [F16, BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("M,N", SHAPES)
def test_norm_backward(b2g, cuda, M, N, dt, xt):
    for res, pad in ((True, 0), (False, 3)):
        check_bwd(cuda, b2g, M, N, dt, xt, res, pad)


@pytest.mark.parametrize("w_dt", [F16, BF16, F32], ids=NAMES.get)
def test_norm_backward_variants(b2g, cuda, w_dt):
    check_bwd(cuda, b2g, 40, 1032, BF16, I8, True, 8, w_dt=w_dt, inplace=True)
    check_bwd(cuda, b2g, 40, 1031, F16, E4M3, False, 0, w_dt=w_dt, inplace=True)
    check_bwd(cuda, b2g, 40, 2048, BF16, F16, True, 0, w_dt=w_dt, want_dw=False)


@pytest.mark.parametrize("xt", [I8, E4M3, BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("M,N,pad", [(3, 40960, 0), (330, 16640, 8), (5, 33003, 5), (310, 9001, 1), (320, 7, 0)])
def test_norm_backward_long_and_short_rows(b2g, cuda, M, N, pad, xt):
    """Rows too long, too short or of other types than the ring kernels take, more rows than blocks among them."""
    check_bwd(cuda, b2g, M, N, BF16, xt, True, pad)
    check_bwd(cuda, b2g, M, N, F32, xt, False, pad)


def test_norm_backward_no_tokens(b2g, cuda):
    torch = cuda
    e = torch.zeros(0, 64, device="cuda")
    dw = torch.full((64,), 3.0, device="cuda")
    b2g.rmsnorm_bwd_q8(e.bfloat16(), e.to(torch.int8), e[:, 0], torch.ones(64, device="cuda").bfloat16(), e[:, 0],
                       e.bfloat16(), dw, 0, 64)
    assert not dw.any()


def test_norm_gradient_against_differences(b2g, cuda):
    """The formula itself: central differences, in fp64, of sum(dy * norm(h)) along random
    directions.  The step's error is its square (1e-8) times third derivatives of order one; the
    kernel's fp32 output adds (N + 20) u of the terms' sizes."""
    torch = cuda
    M, N, eps = 6, 96, 1e-6
    h = torch.randn(M, N, device="cuda")
    w, dy = 1 + 0.2 * torch.randn(N, device="cuda"), torch.randn(M, N, device="cuda")

    def loss(h64, w64):
        return (dy.double() * h64 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + eps) * w64).sum()

    rstd = (1 / torch.sqrt(h.double().square().mean(1) + eps)).float()
    dx, dw = torch.zeros(M, N, device="cuda"), torch.zeros(N, device="cuda")
    b2g.rmsnorm_bwd_q8(dy, h, None, w, rstd, dx, dw, M, N, dtype=F32, x_dtype=F32)
    for seed in range(4):
        torch.manual_seed(seed)
        vh, vw = torch.randn(M, N, device="cuda").double(), torch.randn(N, device="cuda").double()
        d = 1e-4
        num = (loss(h.double() + d * vh, w.double()) - loss(h.double() - d * vh, w.double())) / (2 * d)
        got = (dx.double() * vh).sum()
        assert abs(float(num - got)) <= 1e-5 * float((dx.double() * vh).abs().sum())
        num = (loss(h.double(), w.double() + d * vw) - loss(h.double(), w.double() - d * vw)) / (2 * d)
        assert abs(float(num - (dw.double() * vw).sum())) <= 1e-5 * float((dw.double() * vw).abs().sum())


# ---------------------------------------------------------------- together
class Layer:
    """One training step of y = linear(norm(x + r)): forward, weight gradient and norm backward."""

    def __init__(self, torch, M, D, F, q, seed):
        torch.manual_seed(seed)
        bf = torch.bfloat16
        self.M, self.D, self.F, self.q = M, D, F, q
        self.x, self.r = (torch.randn(M, D, device="cuda").to(bf) for _ in range(2))
        self.w = (1 + 0.1 * torch.randn(D, device="cuda")).to(bf)
        self.W = (torch.randn(F, D, device="cuda") / D ** 0.5).to(bf)
        self.dy = (0.1 * torch.randn(M, F, device="cuda")).to(bf)
        e = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")
        self.Wq, self.Ws = e(F, D, t=tt(torch, q)), e(F)
        self.h, self.aq, self.asc, self.rstd = e(M, D, t=bf), e(M, D, t=tt(torch, q)), e(M), e(M)
        self.hq, self.hs = e(M, D, t=tt(torch, q)), e(M)
        self.y, self.dW = e(M, F, t=bf), e(F, D)
        self.da = (0.1 * torch.randn(M, D, device="cuda")).to(bf)
        self.dx, self.dw = e(M, D, t=bf), e(D)

    def step(self, b, stream=None):
        M, D, F, q = self.M, self.D, self.F, self.q
        k = dict(stream=stream)
        b.quantize_q8(self.W, self.Wq, self.Ws, F, D, dtype=BF16, q_dtype=q, **k)
        b.rmsnorm_q8(self.x, self.w, self.aq, self.asc, M, D, dtype=BF16, q_dtype=q, R=self.r, H=self.h, rstd=self.rstd,
                     pow2=True, **k)
        b.quantize_q8(self.h, self.hq, self.hs, M, D, dtype=BF16, q_dtype=q, **k)
        b.gemm_q8(self.aq, self.Wq, self.y, M, F, D, dtype=q, a_scale=self.asc, b_scale=self.Ws, c_dtype=BF16, **k)
        b.wgrad_q8(self.dy, self.aq, self.asc, self.dW, M, F, D, dtype=BF16, q_dtype=q, **k)
        b.rmsnorm_bwd_q8(self.da, self.hq, self.hs, self.w, self.rstd, self.dx, self.dw, M, D, dtype=BF16, x_dtype=q, **k)
        return [self.y, self.dW, self.dx, self.dw, self.h]

    def check(self, torch):
        """Against the same step in 64 bits without any 8-bit rounding: int8 rows are at most half a
        step, amax / 254 (pow2: amax / 127), off per element, e4m3 values 2^-4 relative."""
        h = self.x.double() + self.r.double()
        a = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * self.w.double()
        W = self.W.double()
        if self.q == I8:
            ea = (a.abs().amax(1, keepdim=True) / 127).expand_as(a)
            ew = (W.abs().amax(1, keepdim=True) / 254).expand_as(W)
        else:
            ea, ew = a.abs() / 16 + a.abs().amax(1, keepdim=True) * 2 ** -17, W.abs() / 16 + W.abs().amax(1, keepdim=True) * 2 ** -17
        y = a @ W.t()
        tol = (a.abs() + ea) @ ew.t() + ea @ W.abs().t()
        assert bool(((self.y.double() - y).abs() <= tol * 1.01 + 2 ** -8 * y.abs()).all())
        dy = self.dy.double()
        assert bool(((self.dW.double() - dy.t() @ a).abs() <= 1.01 * (dy.abs().t() @ ea)).all())


@pytest.mark.parametrize("q", [I8, E4M3], ids=NAMES.get)
@pytest.mark.parametrize("M,D,F", [(1, 512, 768), (24, 1024, 640), (300, 520, 1048), (77, 513, 771)])
def test_layer_step_eager_captured_and_on_two_streams(b2g, cuda, M, D, F, q):
    torch = cuda
    a, b = Layer(torch, M, D, F, q, 1), Layer(torch, M, D, F, q, 2)
    want = [[o.clone() for o in l.step(b2g)] for l in (a, b)]
    a.check(torch)
    b.check(torch)
    # two graphs, replayed at once on two streams, twice
    s = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for l, st in zip((a, b), s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            l.step(b2g)
        graphs.append(g)
    for _ in range(2):
        for l in (a, b):
            for o in (l.y, l.dW, l.dx, l.dw, l.h, l.aq, l.hq):
                o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, s):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for l, w in zip((a, b), want):
            assert all(torch.equal(x, y) for x, y in zip([l.y, l.dW, l.dx, l.dw, l.h], w))
    # eager on two streams at once
    for _ in range(3):
        for l, st in zip((a, b), s):
            l.step(b2g, stream=st)
    torch.cuda.synchronize()
    for l, w in zip((a, b), want):
        assert all(torch.equal(x, y) for x, y in zip([l.y, l.dW, l.dx, l.dw, l.h], w))
    assert b2g.device_status() == 0
    del graphs


def test_split_products_of_several_streams_at_once(b2g, cuda):
    """Products whose CTAs wait for one another (K split over them), of different tiles and sizes, queued on four
    streams at once and replayed from four graphs at once: no wait runs out and no value changes."""
    torch = cuda
    shapes = [(300, 5000, 4096), (1000, 1304, 2064), (520, 2048, 4096), (2000, 5120, 4096)]
    prods = []
    for i, (M, N, K) in enumerate(shapes):
        A, B = (q8_matrix(torch, r, K, I8, seed)[0] for r, seed in ((M, 10 + i), (N, 20 + i)))
        prods.append((A, B, torch.empty(M, N, device="cuda"), M, N, K))
    def run(p, st=None):
        b2g.gemm_q8(p[0], p[1], p[2], *p[3:], stream=st)
    for fix in ({}, {"cluster_fixup": 0}):
        with options(b2g, **fix):
            want = []
            for p in prods:
                run(p)
                want.append(p[2].clone())
            streams = [torch.cuda.Stream() for _ in prods]
            graphs = []
            for p, st in zip(prods, streams):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=st):
                    for _ in range(5):
                        run(p)
                graphs.append(g)
            for p in prods:
                p[2].zero_()
            torch.cuda.synchronize()
            for _ in range(8):
                for p, st in zip(prods, streams):
                    run(p, st)
            torch.cuda.synchronize()
            assert all(torch.equal(p[2], w) for p, w in zip(prods, want))
            for p in prods:
                p[2].zero_()
            torch.cuda.synchronize()
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p[2], w) for p, w in zip(prods, want))
            assert b2g.device_status() == 0
            del graphs


@pytest.mark.parametrize("more", [16, 3], ids=["aligned", "odd"])
def test_offsets_past_32_bits(b2g, cuda, more):
    """Rows 2^27 elements apart: every operator gives what it gives for rows close together, bit for bit."""
    torch = cuda
    D, M, N, K = dict(device="cuda"), 20, 300, 320
    def placed(pitch):
        """x's values at that pitch (one buffer per name and element size, never filled as a whole)."""
        bufs = {}
        def place(x, name):
            key = (name, x.dtype.itemsize)
            if key not in bufs:
                bufs[key] = torch.empty((M - 1) * pitch * x.dtype.itemsize + 4096, dtype=torch.uint8, **D)
            v = bufs[key][:bufs[key].numel() // 16 * 16].view(x.dtype).as_strided(x.shape, (pitch, 1))
            v.copy_(x)
            return v
        return place
    x = rows(torch, M, K, 1).to(torch.bfloat16)
    w = torch.randn(K, **D)
    _, wq = q8_matrix(torch, M, K, I8, 5)  # (20 output channels: weights at the wide pitch too)
    dy = torch.randn(M, N, **D).to(torch.bfloat16)
    def step(place):
        h, q = place(torch.zeros_like(x), "h"), place(torch.zeros(M, K, dtype=torch.int8, **D), "q")
        s, rstd, dw = torch.empty(M, **D), torch.empty(M, **D), torch.empty(K, **D)
        b2g.rmsnorm_q8(place(x, "x"), w, q, s, M, K, dtype=BF16, w_dtype=F32, H=h, rstd=rstd, pow2=True)
        q2 = place(torch.zeros(M, K, dtype=torch.int8, **D), "q2")
        b2g.quantize_q8(h, q2, s.clone(), M, K, dtype=BF16, pow2=True)
        v = place(torch.zeros_like(x), "x")
        b2g.dequantize_q8(q, s, v, M, K, dtype=BF16)
        c = []
        for m in (4, M):
            out = place(torch.zeros(M, M, dtype=torch.bfloat16, **D), "c")
            b2g.gemm_q8(q, place(wq, "w"), out, m, M, K, a_scale=s, c_dtype=BF16)
            c.append(out.clone())
        many = torch.zeros(300, K, dtype=torch.int8, **D).random_(-128, 128, generator=torch.Generator(device="cuda").manual_seed(9))
        ct = torch.empty(300, M, **D)
        b2g.gemm_q8(many, place(wq, "w"), ct, 300, M, K)
        g = place(torch.zeros(M, K, **D), "g")
        y = place(dy, "c")
        b2g.wgrad_q8(y, q, s, g, M, M, K)
        d = place(torch.zeros_like(x), "x")
        b2g.rmsnorm_bwd_q8(place(rows(torch, M, K, 3).to(torch.bfloat16), "d"), q, s, w, rstd, d, dw, M, K, w_dtype=F32)
        return [t.clone() for t in (h, q, s, rstd, q2, v, *c, ct, g, d, dw)]
    near = step(placed(K + more))
    wide = step(placed((1 << 27) + more))
    assert b2g.device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(near, wide))
    torch.cuda.empty_cache()  # about 40 GB, for the tests that follow


def test_generic_products_agree(b2g, cuda):
    """option force_generic: the products' generic kernels meet the same bounds."""
    with options(b2g, force_generic=1):
        check_gemm(cuda, b2g, 70, 100, 130, I8, F32, 3)
        check_gemm(cuda, b2g, 70, 100, 130, E4M3, BF16, 0)
        check_wgrad(cuda, b2g, 100, 70, 130, BF16, I8, F32, 3, True)
        check_wgrad(cuda, b2g, 100, 70, 130, F16, E4M3, F16, 0)
        assert b2g.last_path() == b2g.PATH_GENERIC


def test_bench_runs_the_layer():
    """bench.py --workload linear_q8 (the operators one after the other) runs and its output is sound."""
    import json
    import os
    import subprocess
    import sys
    from conftest import ROOT
    for dt in ("i8", "e4m3"):
        run = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--workload", "linear_q8", "--dtype", dt,
                              "--shape", "256,512,640", "--steps", "3", "--warmup", "3", "--kernel-only"],
                             capture_output=True, text=True, timeout=300)
        assert run.returncode == 0, run.stderr[-2000:]
        line = json.loads(run.stdout.strip().splitlines()[-1])
        assert line["token0_out_of_tolerance"] == 0 and line["device_status"] == 0 and line["gpu_launches"] >= 15

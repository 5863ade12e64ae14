"""ctypes binding of libb2g_gemm.so, the C ABI declared in include/b2g_gemm.h.

This is the Python mirror of the reference's drop-in surface: GEMM(A, B, C, M, N, K) for
the kernel launch of mmm.cpp:1496 and contract5d(...) for the G pack + contraction launch
of mmmTensor.cpp:329-369.  Operands are device pointers (ints) or objects exposing
``data_ptr()`` (e.g. torch CUDA tensors, used only as device-memory plumbing).

The binding never computes anything itself: if the shared library is missing it raises,
and every call goes to the CUDA kernels.
"""
import ctypes
import os
import re
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "libb2g_gemm.so")
HEADER = os.path.join(ROOT, "include", "b2g_gemm.h")

OK = 0
ERR_INVALID_ARG = 1
ERR_UNSUPPORTED = 2
ERR_CUDA = 3
ERR_TIMEOUT = 4
ERR_NCCL = 5

DTYPE_F16, DTYPE_BF16, DTYPE_E4M3, DTYPE_E5M2, DTYPE_F32, DTYPE_I8 = 0, 1, 2, 3, 4, 5

PATH_NONE, PATH_TC_1CTA, PATH_TC_2CTA, PATH_GENERIC, PATH_ZERO, PATH_EMPTY, PATH_FEW = range(7)
PATH_NAMES = {0: "none", 1: "tc_1cta", 2: "tc_2cta", 3: "generic", 4: "zero", 5: "empty", 6: "few"}


class B2GError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__("b2g error %d: %s" % (code, msg))
        self.code = code


_lib = None


def load(path=None):
    """Load libb2g_gemm.so (built by build.py).  Raises if it is missing."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = path or LIB_PATH
    if not os.path.exists(p):
        raise FileNotFoundError(
            "libb2g_gemm.so not found at %s; build it with python rdna4-gemm-wmma_b200/build.py" % p)
    L = ctypes.CDLL(p)
    i64, vp = ctypes.c_int64, ctypes.c_void_p
    i64p = ctypes.POINTER(ctypes.c_int64)
    L.b2g_gemm_f16_f32.restype = ctypes.c_int
    L.b2g_gemm_f16_f32.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, vp]
    L.b2g_gemm_ex.restype = ctypes.c_int
    L.b2g_gemm_ex.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, ctypes.c_float,
                              ctypes.c_float, vp]
    L.b2g_contract5d_ex.restype = ctypes.c_int
    L.b2g_contract5d_ex.argtypes = [vp, i64p, i64p, vp, i64p, i64p, vp, i64p, i64p,
                                    ctypes.c_float, ctypes.c_float, vp]
    L.b2g_gemm.restype = ctypes.c_int
    L.b2g_gemm.argtypes = [vp, vp, vp, i64, i64, i64]
    L.b2g_gemm_typed.restype = ctypes.c_int
    L.b2g_gemm_typed.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, ctypes.c_int,
                                 ctypes.c_float, ctypes.c_float, vp]
    L.b2g_contract5d_typed.restype = ctypes.c_int
    L.b2g_contract5d_typed.argtypes = [vp, i64p, i64p, vp, i64p, i64p, vp, i64p, i64p,
                                       ctypes.c_int, ctypes.c_float, ctypes.c_float, vp]
    L.b2g_fill_uniform.restype = ctypes.c_int
    L.b2g_fill_uniform.argtypes = [vp, i64, ctypes.c_int, ctypes.c_uint64, ctypes.c_uint64, vp]
    L.b2g_gemm_f16_f32_noalloc.restype = ctypes.c_int
    L.b2g_gemm_f16_f32_noalloc.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, vp]
    L.b2g_contract5d_f16_f32.restype = ctypes.c_int
    L.b2g_contract5d_f16_f32.argtypes = [vp, i64p, i64p, vp, i64p, i64p, vp, i64p, i64p, vp]
    L.b2g_fill_uniform_f16.restype = ctypes.c_int
    L.b2g_fill_uniform_f16.argtypes = [vp, i64, ctypes.c_uint64, ctypes.c_uint64, vp]
    L.b2g_last_error_string.restype = ctypes.c_char_p
    L.b2g_last_error_string.argtypes = []
    L.b2g_last_path.restype = ctypes.c_int
    L.b2g_device_status.restype = ctypes.c_int
    L.b2g_device_status.argtypes = [ctypes.c_int]
    L.b2g_set_option.restype = ctypes.c_int
    L.b2g_set_option.argtypes = [ctypes.c_char_p, i64]
    L.b2g_get_option.restype = i64
    L.b2g_get_option.argtypes = [ctypes.c_char_p]
    L.b2g_tile_coord.restype = None
    L.b2g_tile_coord.argtypes = [ctypes.c_int] * 4 + [ctypes.POINTER(ctypes.c_int)] * 2
    L.b2g_version.restype = ctypes.c_char_p
    L.b2g_gemm_sharded.restype = ctypes.c_int
    L.b2g_gemm_sharded.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, vp, ctypes.c_int,
                                   ctypes.c_int, vp]
    L.b2g_gemm_sharded_k.restype = ctypes.c_int
    L.b2g_gemm_sharded_k.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, vp, vp]
    L.b2g_gemm_sharded_n.restype = ctypes.c_int
    L.b2g_gemm_sharded_n.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, vp, ctypes.c_int,
                                     ctypes.c_int, vp, vp]
    L.b2g_rs_plan_create.restype = ctypes.c_int
    L.b2g_rs_plan_create.argtypes = [vp, i64, i64, ctypes.POINTER(ctypes.c_void_p)]
    L.b2g_rs_plan_destroy.restype = ctypes.c_int
    L.b2g_rs_plan_destroy.argtypes = [vp]
    L.b2g_gemm_sharded_k_p2p.restype = ctypes.c_int
    L.b2g_gemm_sharded_k_p2p.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, vp]
    L.b2g_gemm_sum_slots.restype = ctypes.c_int
    L.b2g_gemm_sum_slots.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, vp, i64,
                                     ctypes.c_int, ctypes.c_int, vp, ctypes.c_uint32, vp]
    L.b2g_chain_plan_create.restype = ctypes.c_int
    L.b2g_chain_plan_create.argtypes = [vp, vp, i64, ctypes.c_int, ctypes.POINTER(ctypes.c_void_p)]
    L.b2g_chain_plan_destroy.restype = ctypes.c_int
    L.b2g_chain_plan_destroy.argtypes = [vp]
    L.b2g_gemm_sharded_chain.restype = ctypes.c_int
    L.b2g_gemm_sharded_chain.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, ctypes.c_int, vp]
    L.b2g_chain_broadcast.restype = ctypes.c_int
    L.b2g_chain_broadcast.argtypes = [vp, i64, ctypes.c_int, vp]
    L.b2g_plan_preview.restype = ctypes.c_int
    L.b2g_plan_preview.argtypes = [i64, i64, i64, ctypes.c_int, ctypes.c_int] + \
        [ctypes.POINTER(ctypes.c_int)] * 5
    L.b2g_gemm_sharded_n_chain.restype = ctypes.c_int
    L.b2g_gemm_sharded_n_chain.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, ctypes.c_int, vp]
    L.b2g_gemm_epilogue.restype = ctypes.c_int
    L.b2g_gemm_epilogue.argtypes = [vp, vp, vp, i64, i64, i64, i64, i64, i64, ctypes.c_int,
                                    ctypes.c_float, ctypes.c_float, vp, ctypes.c_int, vp]
    L.b2g_contract5d_epilogue.restype = ctypes.c_int
    L.b2g_contract5d_epilogue.argtypes = [vp, i64p, i64p, vp, i64p, i64p, vp, i64p, i64p,
                                          ctypes.c_int, ctypes.c_float, ctypes.c_float, vp,
                                          ctypes.c_int, vp]
    L.b2g_contract5d_batched.restype = ctypes.c_int
    L.b2g_contract5d_batched.argtypes = [vp, i64p, i64p, vp, i64p, i64p, i64, vp, i64p, i64p,
                                         ctypes.c_int, ctypes.c_float, ctypes.c_float, vp]
    L.b2g_gemm_batched.restype = ctypes.c_int
    L.b2g_gemm_batched.argtypes = [vp, vp, vp] + [i64] * 10 + [vp]
    L.b2g_slab_rows.restype = ctypes.c_int
    L.b2g_slab_rows.argtypes = [i64, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_int64),
                                ctypes.POINTER(ctypes.c_int64)]
    L.b2g_comm_unique_id.restype = ctypes.c_int
    L.b2g_comm_unique_id.argtypes = [vp]
    L.b2g_comm_init.restype = ctypes.c_int
    L.b2g_comm_init.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_int, ctypes.c_int, vp]
    L.b2g_comm_destroy.restype = ctypes.c_int
    L.b2g_comm_destroy.argtypes = [vp]
    L.b2g_comm_check.restype = ctypes.c_int
    L.b2g_comm_check.argtypes = [vp, i64, vp]
    c_int = ctypes.c_int
    L.b2g_quantize_q8.restype = c_int
    L.b2g_quantize_q8.argtypes = [vp] * 3 + [i64] * 4 + [c_int] * 3 + [vp]
    L.b2g_dequantize_q8.restype = c_int
    L.b2g_dequantize_q8.argtypes = [vp] * 3 + [i64] * 4 + [c_int] * 2 + [vp]
    L.b2g_rmsnorm_q8.restype = c_int
    L.b2g_rmsnorm_q8.argtypes = [vp] * 7 + [i64] * 6 + [c_int] * 3 + [ctypes.c_float, c_int, vp]
    L.b2g_gemm_q8.restype = c_int
    L.b2g_gemm_q8.argtypes = [vp] * 3 + [i64] * 6 + [c_int, vp, vp, vp, c_int, vp]
    L.b2g_wgrad_q8.restype = c_int
    L.b2g_wgrad_q8.argtypes = [vp] * 4 + [i64] * 6 + [c_int] * 4 + [vp]
    L.b2g_rmsnorm_bwd_q8.restype = c_int
    L.b2g_rmsnorm_bwd_q8.argtypes = [vp] * 8 + [i64] * 6 + [c_int] * 3 + [vp]
    L.b2g_call_q8.restype = c_int
    L.b2g_call_q8.argtypes = [c_int, ctypes.c_char_p]
    if path is None:
        _lib = L
    return L


def declared_symbols(header=HEADER):
    """Names of the functions include/b2g_gemm.h declares."""
    txt = open(header).read()
    txt = re.sub(r"/\*.*?\*/", "", txt, flags=re.S)
    return sorted(set(re.findall(r"\b(b2g_[a-z0-9_]+)\s*\(", txt)))


def _ptr(x):
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    raise TypeError("expected a device pointer (int) or an object with data_ptr()")


def _stream(s):
    if s is None:
        try:
            import torch  # plumbing only: the caller's current stream
            if torch.cuda.is_available():
                return torch.cuda.current_stream().cuda_stream
        except ImportError:
            pass
        return None
    if isinstance(s, int):
        return s
    return s.cuda_stream


def _check(rc):
    if rc != OK:
        raise B2GError(rc, load().b2g_last_error_string().decode())


def gemm(A, B, C, M, N, K, lda=None, ldb=None, ldc=None, stream=None):
    """C[M,N] = A[M,K] . B[K,N] (fp16 in, fp32 out, row-major)."""
    L = load()
    _check(L.b2g_gemm_f16_f32(_ptr(A), _ptr(B), _ptr(C), M, N, K,
                              K if lda is None else lda, N if ldb is None else ldb,
                              N if ldc is None else ldc, _stream(stream)))


def gemm_ex(A, B, C, M, N, K, alpha=1.0, beta=0.0, lda=None, ldb=None, ldc=None, stream=None):
    """C = alpha * A[M,K].B[K,N] + beta * C."""
    L = load()
    _check(L.b2g_gemm_ex(_ptr(A), _ptr(B), _ptr(C), M, N, K, K if lda is None else lda,
                         N if ldb is None else ldb, N if ldc is None else ldc, float(alpha),
                         float(beta), _stream(stream)))


def GEMM(A, B, C, M, N, K):
    """The reference's drop-in form (contiguous, default stream)."""
    _check(load().b2g_gemm(_ptr(A), _ptr(B), _ptr(C), M, N, K))


def _arr(vals, n):
    vals = [int(v) for v in vals]
    assert len(vals) == n
    return (ctypes.c_int64 * n)(*vals)


def contract5d(A, a_shape, a_stride, B, b_shape, b_stride, C, c_shape, c_stride, stream=None):
    """C[a,b,i,n] = sum_{j,k} A[a,b,i,j,k] B[j,k,n]; shapes/strides in elements."""
    L = load()
    _check(L.b2g_contract5d_f16_f32(_ptr(A), _arr(a_shape, 5), _arr(a_stride, 5), _ptr(B),
                                    _arr(b_shape, 3), _arr(b_stride, 3), _ptr(C), _arr(c_shape, 4),
                                    _arr(c_stride, 4), _stream(stream)))


def contract5d_ex(A, a_shape, a_stride, B, b_shape, b_stride, C, c_shape, c_stride, alpha=1.0,
                  beta=0.0, stream=None):
    L = load()
    _check(L.b2g_contract5d_ex(_ptr(A), _arr(a_shape, 5), _arr(a_stride, 5), _ptr(B),
                               _arr(b_shape, 3), _arr(b_stride, 3), _ptr(C), _arr(c_shape, 4),
                               _arr(c_stride, 4), float(alpha), float(beta), _stream(stream)))


def fill_uniform(dst, n, seed, offset=0, stream=None, dtype=DTYPE_F16):
    """n elements of the seeded U[-1,1] sequence (element offset `offset`) in `dtype`."""
    _check(load().b2g_fill_uniform(_ptr(dst), n, dtype, seed, offset, _stream(stream)))


def gemm_typed(A, B, C, M, N, K, dtype, alpha=1.0, beta=0.0, lda=None, ldb=None, ldc=None,
               stream=None):
    """C = alpha * A.B + beta * C with A, B of operand type `dtype` (DTYPE_*)."""
    _check(load().b2g_gemm_typed(_ptr(A), _ptr(B), _ptr(C), M, N, K, K if lda is None else lda,
                                 N if ldb is None else ldb, N if ldc is None else ldc, dtype,
                                 float(alpha), float(beta), _stream(stream)))


def last_path():
    return load().b2g_last_path()


def device_status(clear=True):
    return load().b2g_device_status(1 if clear else 0)


def set_option(key, value):
    rc = load().b2g_set_option(key.encode(), int(value))
    if rc != OK:
        raise B2GError(rc, "bad option %s=%r" % (key, value))


def get_option(key):
    return load().b2g_get_option(key.encode())


def tile_coord(t, num_m, num_n, group):
    tm, tn = ctypes.c_int(), ctypes.c_int()
    load().b2g_tile_coord(t, num_m, num_n, group, ctypes.byref(tm), ctypes.byref(tn))
    return tm.value, tn.value


def slab_rows(M, world, rank):
    """(row0, rows) of rank's M-row slab (balanced contiguous partition)."""
    r0, n = ctypes.c_int64(), ctypes.c_int64()
    _check(load().b2g_slab_rows(M, world, rank, ctypes.byref(r0), ctypes.byref(n)))
    return r0.value, n.value


def comm_unique_id():
    """128-byte NCCL unique id (bytes) for b2g_comm_init."""
    buf = ctypes.create_string_buffer(128)
    _check(load().b2g_comm_unique_id(buf))
    return buf.raw


def comm_init(world, rank, uid):
    comm = ctypes.c_void_p()
    buf = ctypes.create_string_buffer(bytes(uid), 128)
    _check(load().b2g_comm_init(ctypes.byref(comm), world, rank, buf))
    return comm.value


def comm_destroy(comm):
    _check(load().b2g_comm_destroy(comm))


def comm_check(comm, timeout_ms=5000, stream=None):
    """Liveness check between steps: B2G_OK if every rank answered within timeout_ms, else the
    communicator is aborted and B2GError (ERR_TIMEOUT) is raised."""
    _check(load().b2g_comm_check(comm, int(timeout_ms), None if stream is None else _stream(stream)))


def gemm_sharded(A_slab, B, C_slab, M, N, K, comm, root=0, k_panels=4, lda=None, ldb=None,
                 ldc=None, stream=None):
    """This rank's part of the M-row-slab sharded GEMM; B is broadcast from root in K panels."""
    _check(load().b2g_gemm_sharded(_ptr(A_slab), _ptr(B), _ptr(C_slab), M, N, K,
                                   K if lda is None else lda, N if ldb is None else ldb,
                                   N if ldc is None else ldc, comm, root, k_panels,
                                   _stream(stream)))


def _ld(x, given, what):
    if given is not None:
        return given
    if hasattr(x, "stride"):
        return max(1, x.stride(0))
    raise ValueError(what + " is required for a raw pointer")


def gemm_sharded_k(A_kslab, B_kslab, C_slab, M, N, K, comm, lda=None, ldb=None, ldc=None,
                   stream=None):
    """K-split GEMM + reduce-scatter: this rank holds K slab slab_rows(K, world, rank) of A and
    B and receives rows [rank*M/world, (rank+1)*M/world) of C.  Leading dimensions default to
    the tensors' row strides."""
    _check(load().b2g_gemm_sharded_k(_ptr(A_kslab), _ptr(B_kslab), _ptr(C_slab), M, N, K,
                                     _ld(A_kslab, lda, "lda"), _ld(B_kslab, ldb, "ldb"),
                                     _ld(C_slab, ldc, "ldc"), comm, _stream(stream)))


def gemm_sharded_n(A, B_nslab, C_nslab, M, N, K, comm, root=0, m_panels=4, C_full=None,
                   lda=None, ldb=None, ldc=None, stream=None):
    """N-slab GEMM: A broadcast from root in row panels, this rank's column slab of C
    computed locally; with C_full, every rank also receives the whole C (all-gather)."""
    _check(load().b2g_gemm_sharded_n(_ptr(A), _ptr(B_nslab), _ptr(C_nslab), M, N, K,
                                     _ld(A, lda, "lda"), _ld(B_nslab, ldb, "ldb"),
                                     _ld(C_nslab, ldc, "ldc"), comm, root, m_panels,
                                     _ptr(C_full), _stream(stream)))


def rs_plan_create(comm, M, N):
    """Collective: receive slots for the peer-memory reduce-scatter of an M x N product."""
    plan = ctypes.c_void_p()
    _check(load().b2g_rs_plan_create(comm, M, N, ctypes.byref(plan)))
    return plan.value


def rs_plan_destroy(plan):
    _check(load().b2g_rs_plan_destroy(plan))


def gemm_sharded_k_p2p(plan, A_kslab, B_kslab, C_slab, M, N, K, lda=None, ldb=None, ldc=None,
                       stream=None):
    """gemm_sharded_k with the reduce-scatter fused into the GEMMs over peer memory."""
    _check(load().b2g_gemm_sharded_k_p2p(plan, _ptr(A_kslab), _ptr(B_kslab), _ptr(C_slab), M, N, K,
                                         _ld(A_kslab, lda, "lda"), _ld(B_kslab, ldb, "ldb"),
                                         _ld(C_slab, ldc, "ldc"), _stream(stream)))


def gemm_sum_slots(A, B, C, M, N, K, slots, slot_stride, count, self_index, status=None,
                   epoch=0, lda=None, ldb=None, ldc=None, stream=None):
    """C = sum over s < count, in order, of term s: A.B for s == self_index, else the fp32
    M x N block at slots + s * slot_stride (the peer-memory K-split's epilogue on its own)."""
    _check(load().b2g_gemm_sum_slots(_ptr(A), _ptr(B), _ptr(C), M, N, K,
                                     K if lda is None else lda, N if ldb is None else ldb,
                                     N if ldc is None else ldc,
                                     None if slots is None else _ptr(slots), slot_stride, count,
                                     self_index, None if status is None else _ptr(status),
                                     epoch, _stream(stream)))


def chain_plan_create(comm, B, nbytes, root=0):
    """Collective: copy-engine broadcast chain over `comm` for this rank's B buffer."""
    plan = ctypes.c_void_p()
    _check(load().b2g_chain_plan_create(comm, _ptr(B), nbytes, root, ctypes.byref(plan)))
    return plan.value


def chain_plan_destroy(plan):
    _check(load().b2g_chain_plan_destroy(plan))


def gemm_sharded_chain(plan, A_slab, C_slab, M, N, K, k_panels=8, lda=None, ldb=None, ldc=None,
                       stream=None):
    """This rank's part of the M-row-slab GEMM with B arriving through the chain plan."""
    _check(load().b2g_gemm_sharded_chain(plan, _ptr(A_slab), _ptr(C_slab), M, N, K,
                                         K if lda is None else lda, N if ldb is None else ldb,
                                         N if ldc is None else ldc, k_panels, _stream(stream)))


def chain_broadcast(plan, nbytes, panels=8, stream=None):
    """The plan's buffer (first nbytes) from the root to every rank along the chain."""
    _check(load().b2g_chain_broadcast(plan, nbytes, panels, _stream(stream)))


def plan_preview(M, N, K, dtype=0, sm_count=148, rows=False):
    """(cta_group, tile_n, k_splits, num_full) the library would choose (no GPU needed); with
    rows=True also the A rows per CTA (128, or 64 for half-height pair tiles)."""
    out = [ctypes.c_int() for _ in range(5)]
    _check(load().b2g_plan_preview(M, N, K, dtype, sm_count, *[ctypes.byref(x) for x in out]))
    vals = tuple(x.value for x in out)
    return vals if rows else vals[:4]


def gemm_sharded_n_chain(plan, B_nslab, C_nslab, M, N, K, m_panels=4, lda=None, ldb=None,
                         ldc=None, stream=None):
    """N-slab GEMM with A (the plan's buffer) arriving in row panels through the chain."""
    _check(load().b2g_gemm_sharded_n_chain(plan, _ptr(B_nslab), _ptr(C_nslab), M, N, K,
                                           K if lda is None else lda, _ld(B_nslab, ldb, "ldb"),
                                           _ld(C_nslab, ldc, "ldc"), m_panels, _stream(stream)))


def gemm_epilogue(A, B, C, M, N, K, dtype=0, alpha=1.0, beta=0.0, bias=None, c_dtype=4,
                  lda=None, ldb=None, ldc=None, stream=None):
    """C = alpha*A.B + beta*C + bias with C of type c_dtype (DTYPE_F32 / DTYPE_F16 / DTYPE_BF16)."""
    _check(load().b2g_gemm_epilogue(_ptr(A), _ptr(B), _ptr(C), M, N, K, K if lda is None else lda,
                                    N if ldb is None else ldb, N if ldc is None else ldc, dtype,
                                    float(alpha), float(beta), _ptr(bias), c_dtype,
                                    _stream(stream)))


def contract5d_epilogue(A, a_shape, a_stride, B, b_shape, b_stride, C, c_shape, c_stride, dtype=0,
                        alpha=1.0, beta=0.0, bias=None, c_dtype=4, stream=None):
    _check(load().b2g_contract5d_epilogue(_ptr(A), _arr(a_shape, 5), _arr(a_stride, 5), _ptr(B),
                                          _arr(b_shape, 3), _arr(b_stride, 3), _ptr(C),
                                          _arr(c_shape, 4), _arr(c_stride, 4), dtype, float(alpha),
                                          float(beta), _ptr(bias), c_dtype, _stream(stream)))


def gemm_batched(A, B, C, L, M, N, K, stride_a, stride_b, stride_c, lda=None, ldb=None,
                 ldc=None, stream=None):
    """C[l] = A[l].B[l] for l < L (batch strides in elements)."""
    _check(load().b2g_gemm_batched(_ptr(A), _ptr(B), _ptr(C), L, M, N, K,
                                   K if lda is None else lda, N if ldb is None else ldb,
                                   N if ldc is None else ldc, stride_a, stride_b, stride_c,
                                   _stream(stream)))


def contract5d_batched(A, a_shape, a_stride, B, b_shape, b_stride, b_batch_stride, C, c_shape,
                       c_stride, dtype=0, alpha=1.0, beta=0.0, stream=None):
    """C[a,b,i,n] = alpha*sum_{j,k} A[a,b,i,j,k] B[a,j,k,n] + beta*C (mode a is a batch mode)."""
    _check(load().b2g_contract5d_batched(_ptr(A), _arr(a_shape, 5), _arr(a_stride, 5), _ptr(B),
                                         _arr(b_shape, 3), _arr(b_stride, 3), b_batch_stride,
                                         _ptr(C), _arr(c_shape, 4), _arr(c_stride, 4), dtype,
                                         float(alpha), float(beta), _stream(stream)))


_torch = None
_raw_stream = None  # device -> its current stream as an integer, where this torch has it
_torch_types = {}  # type code -> the torch dtypes that hold it


def _device():
    """The current device, which every tensor of a call has to be on (None without torch)."""
    global _torch, _raw_stream
    if _torch is None:
        try:
            import torch
        except ImportError:
            return None
        _torch = torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        for code, names in ((DTYPE_F16, ["float16"]), (DTYPE_BF16, ["bfloat16"]), (DTYPE_F32, ["float32"]),
                            (DTYPE_I8, ["int8"]), (DTYPE_E4M3, ["float8_e4m3fn", "uint8"])):
            _torch_types[code] = tuple(getattr(torch, n) for n in names if hasattr(torch, n))
    return _torch.cuda.current_device() if _torch.cuda.is_initialized() else None


def _refuse(msg, *args):
    raise B2GError(ERR_INVALID_ARG, msg % args)


def _wrong_tensor(x, dtype, what):
    if dtype not in _torch_types:
        _refuse("%s: unsupported type code %r", what, dtype)
    if x.dtype not in _torch_types[dtype]:
        _refuse("%s is %s, not of type code %r", what, x.dtype, dtype)
    _refuse("%s is not on %s", what, "the current device" if x.is_cuda else "a GPU")


def _matrix(x, dtype, what, rows, cols, ld, dev):
    """(pointer, leading dimension) of a rows x cols operand of the 8-bit operators.  A raw pointer is
    taken as it is (leading dimension `cols` unless given).  A torch tensor has to be of the type
    that the call names and on the current device, and a row-major matrix of that size at least,
    whose row stride is the default leading dimension; with another one, its storage has to hold the rows."""
    if x is None or isinstance(x, int) or _torch is None or not isinstance(x, _torch.Tensor):
        return _ptr(x) or 0, (cols or 1) if ld is None else ld
    if x.get_device() != dev or x.dtype not in _torch_types.get(dtype, ()):
        _wrong_tensor(x, dtype, what)
    if ld is None:
        ld = cols or 1
        if rows and cols:
            st, sh = x.stride(), x.shape
            if len(st) != 2:
                if not x.is_contiguous() or x.numel() < rows * cols:
                    _refuse("%s is no row-major matrix of %d x %d", what, rows, cols)
            elif sh[0] < rows or sh[1] < cols or (st[1] != 1 and cols > 1):
                _refuse("%s is no row-major matrix of %d x %d", what, rows, cols)
            elif rows > 1:
                ld = st[0]
    elif rows and cols and (rows - 1) * ld + cols > x.untyped_storage().nbytes() // x.element_size() - x.storage_offset():
        _refuse("%s ends before %d rows of %d at leading dimension %d", what, rows, cols, ld)
    return x.data_ptr(), ld


def _vector(x, dtype, what, n, dev):
    """Pointer of a vector of n contiguous values (None: an optional one that is not given)."""
    if x is None or isinstance(x, int) or _torch is None or not isinstance(x, _torch.Tensor):
        return _ptr(x) or 0
    if x.get_device() != dev or x.dtype not in _torch_types.get(dtype, ()):
        _wrong_tensor(x, dtype, what)
    if x.numel() < n or not x.is_contiguous():
        _refuse("%s has fewer than %d contiguous values", what, n)
    return x.data_ptr()


def _stream_of(stream, dev):
    """_stream(), by the shorter way where the tensors' device is known (building a Stream object
    costs as much as the launch)."""
    if stream is None and dev is not None and _raw_stream is not None:
        return _raw_stream(dev)
    return _stream(stream) or 0


def _call(call, words, *args):
    """One of the six operators, its arguments packed into 64-bit words: ctypes converts each argument
    of a call on its own, which costs more than the launch."""
    _check(load().b2g_call_q8(call, words(*args)))


_WORDS = {n: struct.Struct("%dq" % n).pack for n in (10, 11, 15, 18)}
_NORM_WORDS = struct.Struct("16qd2q").pack


def quantize_q8(X, Q, scale, M, N, dtype=DTYPE_F16, q_dtype=DTYPE_I8, pow2=False, ldx=None,
                ldq=None, stream=None):
    """Q, scale = rows of X (M x N, type dtype) in 8 bits: scale = max|x| / qmax, with pow2
    rounded up to a power of two.  Leading dimensions default to the tensors' row strides."""
    dev = _device()
    x, ldx = _matrix(X, dtype, "X", M, N, ldx, dev)
    q, ldq = _matrix(Q, q_dtype, "Q", M, N, ldq, dev)
    s = _vector(scale, DTYPE_F32, "scale", M, dev)
    _call(0, _WORDS[11], x, q, s, M, N, ldx, ldq, dtype, q_dtype, 1 if pow2 else 0, _stream_of(stream, dev))


def dequantize_q8(Q, scale, X, M, N, dtype=DTYPE_F16, q_dtype=DTYPE_I8, ldq=None, ldx=None,
                  stream=None):
    """X (M x N, type dtype) = Q * scale (one scale per row)."""
    dev = _device()
    q, ldq = _matrix(Q, q_dtype, "Q", M, N, ldq, dev)
    s = _vector(scale, DTYPE_F32, "scale", M, dev)
    x, ldx = _matrix(X, dtype, "X", M, N, ldx, dev)
    _call(1, _WORDS[10], q, s, x, M, N, ldq, ldx, q_dtype, dtype, _stream_of(stream, dev))


def rmsnorm_q8(X, W, Q, scale, M, N, dtype=DTYPE_F16, q_dtype=DTYPE_I8, R=None, H=None, rstd=None,
               w_dtype=None, eps=1e-6, pow2=False, ldx=None, ldr=None, ldh=None, ldq=None,
               stream=None):
    """h = X + R, Q, scale = (h / sqrt(mean(h^2) + eps) * W) in 8 bits.  Optional outputs: H = h
    in type dtype (may be X or R itself), rstd (M fp32 values, for rmsnorm_bwd_q8)."""
    dev = _device()
    w_dtype = dtype if w_dtype is None else w_dtype
    x, ldx = _matrix(X, dtype, "X", M, N, ldx, dev)
    r, ldr = _matrix(R, dtype, "R", M, N, ldr, dev)
    w = _vector(W, w_dtype, "W", N, dev)
    h, ldh = _matrix(H, dtype, "H", M, N, ldh, dev)
    q, ldq = _matrix(Q, q_dtype, "Q", M, N, ldq, dev)
    s = _vector(scale, DTYPE_F32, "scale", M, dev)
    rs = _vector(rstd, DTYPE_F32, "rstd", M, dev)
    _call(2, _NORM_WORDS, x, r, w, h, q, s, rs, M, N, ldx, ldr, ldh, ldq, dtype, w_dtype, q_dtype, eps,
          1 if pow2 else 0, _stream_of(stream, dev))


def gemm_q8(A, B, C, M, N, K, dtype=DTYPE_I8, a_scale=None, b_scale=None, bias=None,
            c_dtype=DTYPE_F32, lda=None, ldb=None, ldc=None, stream=None):
    """C = (A . B^T) * a_scale[:, None] * b_scale + bias with A M x K and B N x K of 8-bit type
    dtype (int32 sums for DTYPE_I8) and C of type c_dtype."""
    dev = _device()
    a, lda = _matrix(A, dtype, "A", M, K, lda, dev)
    b, ldb = _matrix(B, dtype, "B", N, K, ldb, dev)
    c, ldc = _matrix(C, c_dtype, "C", M, N, ldc, dev)
    sa = _vector(a_scale, DTYPE_F32, "a_scale", M, dev)
    sb = _vector(b_scale, DTYPE_F32, "b_scale", N, dev)
    bi = _vector(bias, DTYPE_F32, "bias", N, dev)
    _call(3, _WORDS[15], a, b, c, M, N, K, lda, ldb, ldc, dtype, sa, sb, bi, c_dtype, _stream_of(stream, dev))


def wgrad_q8(dY, Q, scale, dW, M, N, K, dtype=DTYPE_BF16, q_dtype=DTYPE_I8, accumulate=False,
             c_dtype=DTYPE_F32, ldy=None, ldq=None, ldw=None, stream=None):
    """dW (N x K) = dY^T . (Q * scale) from the 8-bit checkpoint Q (M x K) of a linear layer's
    input and the gradient dY (M x N) of its output; accumulate adds into an fp32 dW."""
    dev = _device()
    y, ldy = _matrix(dY, dtype, "dY", M, N, ldy, dev)
    q, ldq = _matrix(Q, q_dtype, "Q", M, K, ldq, dev)
    s = _vector(scale, DTYPE_F32, "scale", M, dev)
    w, ldw = _matrix(dW, c_dtype, "dW", N, K, ldw, dev)
    _call(4, _WORDS[15], y, q, s, w, M, N, K, ldy, ldq, ldw, dtype, q_dtype, 1 if accumulate else 0, c_dtype,
          _stream_of(stream, dev))


def rmsnorm_bwd_q8(dY, X, x_scale, W, rstd, dX, dw, M, N, dtype=DTYPE_BF16, x_dtype=DTYPE_I8,
                   w_dtype=None, dres=None, ldy=None, ldx=None, ldr=None, lddx=None, stream=None):
    """Backward pass of rmsnorm_q8: dX = rstd * (dY*W - xh * mean(dY*W*xh)) (+ dres) and
    dw = sum over rows of dY * xh, xh = (the checkpoint X * x_scale of h) * rstd.  dw may be None."""
    dev = _device()
    w_dtype = dtype if w_dtype is None else w_dtype
    y, ldy = _matrix(dY, dtype, "dY", M, N, ldy, dev)
    x, ldx = _matrix(X, x_dtype, "X", M, N, ldx, dev)
    xs = _vector(x_scale, DTYPE_F32, "x_scale", M, dev)
    w = _vector(W, w_dtype, "W", N, dev)
    rs = _vector(rstd, DTYPE_F32, "rstd", M, dev)
    r, ldr = _matrix(dres, dtype, "dres", M, N, ldr, dev)
    d, lddx = _matrix(dX, dtype, "dX", M, N, lddx, dev)
    g = _vector(dw, DTYPE_F32, "dw", N, dev)
    _call(5, _WORDS[18], y, x, xs, w, rs, r, d, g, M, N, ldy, ldx, ldr, lddx, dtype, x_dtype, w_dtype,
          _stream_of(stream, dev))


def version():
    return load().b2g_version().decode()

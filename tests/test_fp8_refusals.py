"""What the 8-bit operators and the router balance refuse, on the CPU: every
check comes before the first CUDA call, so made-up pointers are never used."""
import pytest

from fp8_util import BF16, F16, F32

ARG, UNSUPPORTED = -1, -4
A = 1 << 20  # an aligned address that nothing reads


def refused(lib, name, args, code):
    from textsift_b200 import abi
    assert getattr(lib, name)(*args) == code
    assert abi.last_error()


def changed(base, **kw):
    return [kw.get(k, v) for k, v in base.items()]


QUANT = dict(x=A, dt=F16, ldx=640, rows=4, cols=640, transpose=0, codes=A, ldc=640, scales=A, lds=4, stream=None)
TRANSPOSE = dict(codes=A, ldw=640, scales=A, E=2, N=64, K=640, codes_t=A, ldt=64, scales_t=A, stream=None)
MATMUL = dict(a=A, lda=640, asc=A, ldas=64, w=A, ldw=640, ws=A, ldws=64, block=128, bias=None, seg=None, E=1, out=A, dt=F16,
              ldo=64, acc=0, M=64, N=64, K=640, stream=None)
MATVEC = dict(x=A, dt=F16, ldx=640, w=A, ldw=640, ws=A, bias=None, out=A, odt=F16, ldo=64, M=2, N=64, K=640, stream=None)
BALANCE = dict(z=A, dt=F32, ldl=128, idx=A, mask=None, seq=None, S=1, T=10, E=128, k=4, alpha=0.01, scale=1.0, counts=A,
               prob=A, loss=A, grad=A, ldg=128, work=A, nbytes=1 << 20, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=3), ARG), (dict(x=None), ARG), (dict(codes=None), ARG), (dict(scales=None), ARG), (dict(ldx=639), ARG),
    (dict(ldc=624), ARG), (dict(ldc=648), UNSUPPORTED), (dict(codes=A + 8), UNSUPPORTED), (dict(lds=3), ARG),
    (dict(x=A + 1), ARG), (dict(scales=A + 2), ARG), (dict(transpose=1), ARG), (dict(dt=F32, x=A + 2), ARG),
    (dict(transpose=1, ldc=16, lds=600), ARG)])
def test_quant(cuda_lib, kw, code):
    refused(cuda_lib, "ts_cuda_op_quant_fp8", changed(QUANT, **kw), code)


@pytest.mark.parametrize("kw,code", [
    (dict(codes=None), ARG), (dict(scales=None), ARG), (dict(codes_t=None), ARG), (dict(scales_t=None), ARG),
    (dict(ldw=632), ARG), (dict(ldt=48), ARG), (dict(ldt=72), UNSUPPORTED), (dict(codes=A + 4), UNSUPPORTED),
    (dict(scales=A + 1), ARG), (dict(E=70000), UNSUPPORTED)])
def test_transpose(cuda_lib, kw, code):
    refused(cuda_lib, "ts_cuda_op_transpose_fp8", changed(TRANSPOSE, **kw), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=0), ARG), (dict(acc=1), ARG), (dict(acc=1, dt=BF16), ARG), (dict(block=64), ARG), (dict(E=0), ARG),
    (dict(E=2), ARG), (dict(block=1, seg=A), ARG), (dict(block=1, seg=A, E=2), ARG), (dict(seg=A, E=1025), UNSUPPORTED),
    (dict(M=1 << 31, ldas=1 << 31), UNSUPPORTED), (dict(a=None), ARG), (dict(asc=None), ARG), (dict(w=None), ARG),
    (dict(ws=None), ARG), (dict(out=None), ARG), (dict(ldo=63), ARG), (dict(out=A + 1), ARG), (dict(asc=A + 2), ARG),
    (dict(ws=A + 2), ARG), (dict(bias=A + 1), ARG), (dict(seg=A + 2), ARG), (dict(lda=624), ARG), (dict(lda=648), UNSUPPORTED),
    (dict(a=A + 8), UNSUPPORTED), (dict(ldw=632), ARG), (dict(w=A + 8), UNSUPPORTED), (dict(ldas=63), ARG),
    (dict(block=1, ldws=63), ARG)])
def test_matmul(cuda_lib, kw, code):
    refused(cuda_lib, "ts_cuda_op_matmul_fp8", changed(MATMUL, **kw), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=3), ARG), (dict(odt=0), ARG), (dict(M=17), UNSUPPORTED), (dict(x=None), ARG), (dict(w=None), ARG),
    (dict(ws=None), ARG), (dict(out=None), ARG), (dict(ldx=639), ARG), (dict(ldo=63), ARG), (dict(x=A + 1), ARG),
    (dict(out=A + 1), ARG), (dict(ws=A + 2), ARG), (dict(bias=A + 1), ARG), (dict(ldw=624), ARG),
    (dict(ldw=648), UNSUPPORTED), (dict(w=A + 8), UNSUPPORTED)])
def test_matvec(cuda_lib, kw, code):
    refused(cuda_lib, "ts_cuda_op_matvec_fp8", changed(MATVEC, **kw), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=0), ARG), (dict(E=0, ldl=0), ARG), (dict(k=0), ARG), (dict(S=0), ARG), (dict(S=2), ARG),
    (dict(E=1025, ldl=1025, ldg=1025), UNSUPPORTED), (dict(k=65), UNSUPPORTED), (dict(T=(1 << 23) + 1), UNSUPPORTED),
    (dict(z=None), ARG), (dict(idx=None), ARG), (dict(counts=None), ARG), (dict(prob=None), ARG), (dict(loss=None), ARG),
    (dict(work=None), ARG), (dict(nbytes=64), ARG), (dict(work=A + 4), ARG), (dict(z=A + 2), ARG), (dict(grad=A + 2), ARG),
    (dict(idx=A + 2), ARG), (dict(seq=A + 1), ARG), (dict(counts=A + 2), ARG), (dict(prob=A + 2), ARG),
    (dict(loss=A + 2), ARG), (dict(ldl=127), ARG), (dict(ldg=127), ARG)])
def test_balance(cuda_lib, kw, code):
    refused(cuda_lib, "ts_cuda_op_router_balance", changed(BALANCE, **kw), code)


def test_nothing_to_do(cuda_lib):
    """Empty calls succeed without a look at any pointer."""
    none = dict.fromkeys(("x", "codes", "scales", "codes_t", "scales_t", "a", "asc", "w", "ws", "out"))
    for name, base, kw in (("ts_cuda_op_quant_fp8", QUANT, dict(rows=0)), ("ts_cuda_op_quant_fp8", QUANT, dict(cols=0)),
                           ("ts_cuda_op_transpose_fp8", TRANSPOSE, dict(E=0)), ("ts_cuda_op_matmul_fp8", MATMUL, dict(M=0)),
                           ("ts_cuda_op_matmul_fp8", MATMUL, dict(N=0)), ("ts_cuda_op_matvec_fp8", MATVEC, dict(M=0))):
        assert getattr(cuda_lib, name)(*changed(base, **{k: v for k, v in none.items() if k in base}, **kw)) == 0


def test_balance_work_fits(cuda_lib):
    for S, E in ((1, 1), (1, 128), (44, 128), (300, 1024)):
        assert cuda_lib.ts_cuda_router_balance_work(S, E) <= 16 * S * (E + 2) + 256

"""Every kernel of gemm_fp8 in every tail, named by the query that the library launches from, and the choices under
`policy_rows`. Oracle and tolerances as in test_gpu_fp8.py."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

import echo_tts_amd  # noqa: E402,F401
import fp8_ref as R  # noqa: E402
import test_gpu_fp8 as T  # noqa: E402
from echo_tts_amd import _lib as L  # noqa: E402
from echo_tts_amd import ops  # noqa: E402

DEV, BF = "cuda", torch.bfloat16


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


def planned(M, N, K, epilogue=L.EPI_STORE, quantize=False):
    P = 1 << 20
    a = L.GemmFp8Args(M=M, N=N, K=K, epilogue=epilogue, A=P, lda=K, a_scale=P, ld_as=M, W=P, ldw=K, w_scale=P, ld_ws=N, C=P, ldc=N)
    if epilogue == L.EPI_RESID:
        a.aux, a.ld_aux = P, N
    if quantize:
        a.c_scale, a.ld_cs = P, M
    return L.load().echo_gemm_fp8_planned_kernel(C.byref(a))


# kernel (echo_gemm_fp8_planned_kernel's numbers), M, N, K. A ring holds the scales of 8192 of K at a time: K of one, two and
# three such segments, the last of one K-tile that is cut short, of two, and of two; the persistent kernel ends at K = 7680
PLAIN = [(0, 33, 32, 400), (0, 65, 32, 8336), (1, 65, 1040, 1552), (1, 65, 1040, 8208), (2, 65, 2064, 400), (2, 300, 528, 8336),
         (3, 300, 1040, 1552), (3, 157, 2064, 8208), (4, 300, 2064, 400), (4, 300, 2064, 8336), (5, 2100, 528, 1552), (5, 2100, 528, 8208),
         (5, 2100, 528, 8336), (5, 2100, 528, 16640), (6, 2100, 1040, 1552), (6, 2100, 1040, 8208), (6, 1300, 2064, 8336),
         (6, 2100, 1040, 16640), (9, 2100, 2064, 512), (9, 2100, 2064, 7552), (9, 2100, 2064, 7680)]
GLU = [(1, 7, 33, 32, 400), (2, 7, 65, 2080, 1552), (2, 7, 300, 544, 8336), (3, 7, 300, 1056, 8208), (4, 7, 300, 2080, 400), (5, 7, 2100, 544, 8336),
       (5, 7, 2100, 544, 16640), (6, 8, 2100, 1056, 8208), (6, 8, 1300, 2080, 8336), (6, 8, 2100, 1056, 1552), (9, 9, 2100, 2080, 7552),
       (9, 9, 2100, 2080, 7680)]


@pytest.mark.parametrize("kernel,M,N,K", PLAIN)
def test_store_and_residual(kernel, M, N, K):
    assert planned(M, N, K) == planned(M, N, K, L.EPI_RESID) == kernel
    T.test_gemm_store(M, N, K)
    T.test_gemm_residual(M, N, K)


@pytest.mark.parametrize("kernel,quantised,M,N,K", GLU)
def test_swiglu(kernel, quantised, M, N, K):
    assert planned(M, N, K, L.EPI_SWIGLU) == kernel and planned(M, N, K, L.EPI_SWIGLU, True) == quantised
    T.test_gemm_swiglu(M, N, K)


def test_every_kernel_is_named():
    assert {k for k, *_ in PLAIN} == set(range(7)) | {9}
    assert {k for k, *_ in GLU} == set(range(1, 7)) | {9} and {k for _, k, *_ in GLU} == {7, 8, 9}


@pytest.mark.parametrize("kernel,M,N,K", [c for c in PLAIN if c[3] < 8192])
def test_scales_far_from_one(kernel, M, N, K):
    """Powers of two in the scales come out as such, to the bit: 2^100 against 2^-100, and 2^30 twice."""
    a, a_s, _, w, w_s, _ = T.gemm_inputs(M, N, K)

    def moved(s, by):
        b = s.view(torch.uint8).to(torch.int32)
        return torch.where(b > 0, b + by, b).to(torch.uint8).view(R.E8M0)
    assert planned(M, N, K) == kernel
    out = ops.gemm_fp8(a, a_s, w, w_s)
    assert torch.equal(ops.gemm_fp8(a, moved(a_s, 100), w, moved(w_s, -100)), out)
    assert torch.equal(ops.gemm_fp8(a, moved(a_s, 30), w, moved(w_s, 30)), out * 2.0 ** 60)


@pytest.mark.parametrize("M,N,K,parts", [(160, 2048, 5888, 8), (40, 2048, 2048, 16), (640, 1056, 640, 4), (33, 544, 8336, 3)])
def test_policy_rows(M, N, K, parts):
    """A share of a batch's rows under `policy_rows` gives the whole batch's bits, in every tail."""
    a, a_s, av, w, w_s, wv = T.gemm_inputs(M * parts, N, K)
    h, gate, bias = (torch.randn(*n, device=DEV).to(BF) for n in ((M * parts, N), (N,), (N,)))
    calls = [lambda r: (ops.gemm_fp8(a[r], a_s[:, r], w, w_s),),
             lambda r: (ops.gemm_fp8(a[r], a_s[:, r], w, w_s, bias=bias, epilogue=L.EPI_RESID, aux=h[r], gate=gate),),
             lambda r: (ops.gemm_fp8(a[r], a_s[:, r], w, w_s, epilogue=L.EPI_SWIGLU),),
             lambda r: ops.gemm_fp8(a[r], a_s[:, r], w, w_s, epilogue=L.EPI_SWIGLU, quantize=True)]
    ref, err = T.products(av[:M], wv)
    for i, f in enumerate(calls):
        whole = f(slice(None))
        for p in range(parts):
            r = slice(p * M, (p + 1) * M)
            with ops.policy_rows(parts, 1):
                part = f(r)
            if i == 0 and p == 0:
                T.within(part[0], ref, ref.abs() * T.U16 + err * (1 + T.U16) + 1e-30)
            assert T.same_bytes(part[0], whole[0][r]), (i, p)
            assert len(part) == 1 or T.same_bytes(part[1], whole[1][:, r]), (i, p)


@pytest.mark.parametrize("n,cap", [(1, 4096), (1, 700), (33, 2100), (200, 1000)])
def test_policy_rows_attention(n, cap):
    rows, H, parts = 8, 4, 4
    q = torch.randn(rows, n, H, 128, device=DEV).to(BF)
    cache, scale, kv = T.coded(rows, cap, H)
    lens = torch.randint(1, cap + 1, (rows,), dtype=torch.int32, device=DEV)
    whole = ops.attention(q, [T.segment(cache, scale, lens=lens)])
    T.within(whole, *T.attention_ref(q, [(kv[:, :, 0], kv[:, :, 1], T.prefix(lens, n, cap))], None))
    for p in range(parts):
        r = slice(p * rows // parts, (p + 1) * rows // parts)
        with ops.policy_rows(parts, 1):
            part = ops.attention(q[r], [T.segment(cache[r], scale[r], lens=lens[r])])
        assert torch.equal(part, whole[r]), p

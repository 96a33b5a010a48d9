"""Sizes that no launch can hold are refused before one is made (no device)."""
import ctypes as C

import pytest

import echo_tts_amd  # noqa: F401
from echo_tts_amd import _lib as L

P, ESHAPE, IMAX = 1 << 20, -3, (1 << 31) - 1


@pytest.fixture(scope="module")
def lib():
    return L.load()


@pytest.mark.parametrize("M,N,K", [(1 << 30, 64, 16), (IMAX, 16, 16), (16, IMAX // 16 * 16, 16)])
def test_gemm(lib, M, N, K):
    a = L.GemmFp8Args(M=M, N=N, K=K, epilogue=0, A=P, lda=K, a_scale=P, ld_as=M, W=P, ldw=K, w_scale=P, ld_ws=N, C=P, ldc=min(N, 1 << 21))
    assert lib.echo_gemm_fp8(C.byref(a), None) == ESHAPE


@pytest.mark.parametrize("rows,heads,n_q,nsplit", [(1 << 20, 16, 1, 1), (1 << 17, 16, 1, 4), (IMAX, IMAX, IMAX, 1), (1 << 12, 16, 1 << 17, 1), (1 << 16, 1 << 14, IMAX - 128, 1),
                                                   (1, 1, IMAX, 1)])
def test_attention(lib, rows, heads, n_q, nsplit):
    a = L.AttnFp8Args(rows=rows, n_q=n_q, heads=heads, nseg=1, q=P, q_ld_tok=128, q_ld_batch=128, out=P, o_ld_tok=128, o_ld_batch=128, scale=0.1)
    a.seg[0] = L.KVSegmentFp8(k=P, v=P, ld_tok=128, ld_batch=128, ld_head=128, k_scale=P, v_scale=P, s_tok=1, s_batch=1, s_head=1,
                              batch_mod=1, capacity=4096)
    assert lib.echo_attention_fp8(C.byref(a), nsplit, P, 1 << 62, None) == ESHAPE
    assert lib.echo_attention_fp8_pick_split(C.byref(a)) >= 1

"""The 8-bit operators at the ends of fp32's range; oracle and tolerances as in test_gpu_fp8.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import echo_tts_amd  # noqa: E402,F401
import fp8_ref as R  # noqa: E402
import test_gpu_fp8 as T  # noqa: E402
from echo_tts_amd import _lib as L  # noqa: E402
from echo_tts_amd import ops  # noqa: E402

DEV, BF, D = "cuda", torch.bfloat16, torch.float64


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


@pytest.mark.parametrize("hot,size", [((270,), 100), ((130, 270), 81)])
@pytest.mark.parametrize("coded", [True, False])
@pytest.mark.parametrize("nsplit", [1, 3])
@pytest.mark.parametrize("n", [3, 40, 200])
def test_attention_large_values(n, nsplit, coded, hot, size):
    """Large values at keys whose scores lie up to 2^46 above the first tile's: the output is finite, the sum stays small,
    and only P times V passes fp32's range where the first tile's maximum is the reference; at 2^100 in one part, at 2^81
    (2^127.2 a part) in the sum of two parts."""
    lens = 300
    q = torch.zeros(1, n, 1, 128, device=DEV)
    q[0, :, 0, 0] = torch.linspace(0, 4, n, device=DEV)
    q = q.to(BF)
    kv = torch.randn(1, lens, 2, 1, 128, device=DEV)
    kv[:, :, 0] *= 0.01
    for key in hot:  # in the second tiles of the last two of 3 parts
        kv[0, key, 0, 0, 0], kv[0, key, 1] = 8.0, 1.0
    kv[:, :, 1] *= 2.0 ** size
    if coded:
        c, b = R.quantize(kv)
        cache, scale = T.new_cache(1, lens, 1, 1, "plain")
        cache.view(torch.uint8)[:, :, 0] = c.view(torch.uint8)
        scale.view(torch.uint8)[:, 0] = b[..., 0].permute(0, 2, 3, 1)
        kv, seg = R.values(c, b), T.segment(cache, scale)
    else:
        kv = kv.to(BF)
        seg = ops.Segment(kv[:, :, 0], kv[:, :, 1])
        kv = kv.to(D)
    ref, tol = T.attention_ref(q, [(kv[:, :, 0], kv[:, :, 1], torch.ones(1, n, lens, dtype=torch.bool, device=DEV))], None, 1.0)
    with ops.attention_split(nsplit):  # beside the long unseen segment more than 32 queries go to the kernel for many
        T.within(ops.attention(q, [seg, T.unseen(1, 1)], scale=1.0), ref, tol)


FAR = [-64.0, -64.5, -72.0, -88.0, -89.0, -92.0, -96.0, -100.0, -104.0, -112.0, -130.0, 0.0, 30.0]


SHAPES = [(13, 32), (13, 512), (160, 1056), (640, 1024), (4100, 1408)]


@pytest.mark.parametrize("M,N", SHAPES)
def test_swiglu_far(M, N):
    """silu(a) b with e^a below fp32's range and b = 2^100: a normal number, in bf16 and in 8 bits."""
    swiglu_of(FAR, M, N)


@pytest.mark.parametrize("M,N", SHAPES)
def test_swiglu_border(M, N):
    """Around a = -87, below which the reciprocal of 1 + e^-a is no normal number."""
    swiglu_of([-86.0, -86.5, -87.0, -87.5, -88.0], M, N)


def swiglu_of(values, M, N):
    K = 384
    a = torch.tensor(values, dtype=D, device=DEV).repeat(-(-M // len(values)))[:M]
    x = torch.zeros(M, K, dtype=D, device=DEV)
    x[:, 0] = torch.trunc(a / 8) * 8  # two codes that add up to a, exactly
    x[:, 1] = a - x[:, 0]
    x[:, 128] = 2.0 ** 100
    w = torch.zeros(N, K, dtype=D, device=DEV)
    w.view(N // 32, 2, 16, K)[:, 0, :, :2] = 1.0
    w.view(N // 32, 2, 16, K)[:, 1, :, 128] = 1.0
    (aq, a_s, av), (wq, w_s, wv) = R.matrix(x), R.matrix(w)
    assert torch.equal(av, x) and torch.equal(wv, w)
    ref = (a / (1 + torch.exp(-a)) * 2.0 ** 100)[:, None].expand(M, N // 2)
    err = ref.abs() * ((1.5 * a.abs() + 12) * T.U32)[:, None]  # test_gpu_fp8.swiglu's
    T.within(ops.gemm_fp8(aq, a_s, wq, w_s, epilogue=L.EPI_SWIGLU), ref, ref.abs() * T.U16 + err * 1.01)
    q, s = ops.gemm_fp8(aq, a_s, wq, w_s, epilogue=L.EPI_SWIGLU, quantize=True)
    R.quantized_well(q, R.bytes_of(s, N // 2), ref, 0.0, err * 1.01)


@pytest.mark.parametrize("n", [1, 40, 200])
def test_attention_small_values(n):
    """Blocks below 2^-118 keep the smallest scale, 2^-127 (byte 0): values of 2^-120 come back, and keys alike."""
    lens = 200
    kv = torch.randn(1, lens, 2, 1, 128, device=DEV) * 2.0 ** -120
    c, b = R.quantize(kv)
    assert int(b.max()) <= 2 and int(b.min()) == 0
    cache, scale = T.new_cache(1, lens, 1, 1, "plain")
    cache.view(torch.uint8)[:, :, 0] = c.view(torch.uint8)
    scale.view(torch.uint8)[:, 0] = b[..., 0].permute(0, 2, 3, 1)
    kv = R.values(c, b)
    q = torch.randn(1, n, 1, 128, device=DEV).to(BF) * 2.0 ** 118  # scores of a few units
    ref, tol = T.attention_ref(q, [(kv[:, :, 0], kv[:, :, 1], torch.ones(1, n, lens, dtype=torch.bool, device=DEV))], None)
    # attention_ref's tolerance has 1e-30 beside the relative part: here in units of 2^120
    e = (tol - 1e-30) * 2.0 ** 120
    for segs in ([T.segment(cache, scale)], [T.segment(cache, scale), T.unseen(1, 1)]):
        out = ops.attention(q, segs)
        T.within(out.to(D) * 2.0 ** 120, ref * 2.0 ** 120, e + 2.0 ** -13)  # 2^-133: bf16's last subnormal bit

"""The 8-bit operators at the ends of fp32's range; oracle and tolerances as in test_gpu_fp8.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import echo_tts_amd  # noqa: E402,F401
import fp8_ref as R  # noqa: E402
import test_gpu_fp8 as T  # noqa: E402
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

"""The 8-bit operators beyond 2^32 threads of a launch (a grid dimension's limit) and beyond 32-bit offsets."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import echo_tts_amd  # noqa: E402,F401
import fp8_ref as R  # noqa: E402
import test_gpu_fp8 as T  # noqa: E402
from echo_tts_amd import ops  # noqa: E402

DEV, BF, D = "cuda", torch.bfloat16, torch.float64
ROWS = (1 << 26) + 5  # a wave a row: 2^32 threads and 320


@pytest.fixture(scope="module")
def tall():
    """[ROWS, 16] bf16, and the rows that are compared: the first, the last, and those around the 2^32nd thread."""
    torch.manual_seed(0)
    x = torch.empty(ROWS, 16, device=DEV, dtype=BF).normal_()
    at = torch.cat([torch.arange(300), torch.arange((1 << 26) - 300, ROWS), torch.randint(0, ROWS, (5000,))]).to(DEV)
    return x, at


def test_quantize_tall(tall):
    x, at = tall
    q, s = ops.quantize_fp8(x)
    want, b = R.quantize(x[at])
    assert T.same_bytes(q[at], want) and torch.equal(s.view(torch.uint8)[:, at], R.words(b))


def test_adaln_tall(tall):
    x, at = tall
    one = torch.ones(16, device=DEV, dtype=BF)
    q, s = ops.adaln_modulate_fp8(x, one * 0, one, 1e-5)
    xd = x[at].to(D)
    y = xd / (xd.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    R.quantized_well(q[at], R.bytes_of(s[:, at], 16), y, 0.0, (16 / 2 + 6) * y.abs() * T.U32)  # test_gpu_fp8.test_adaln's


def test_kv_write_tall():
    """One call of 2^25 + 7 tokens (two waves each), of which the last 40 meet a slot."""
    tokens, cap = (1 << 25) + 7, 40
    torch.manual_seed(0)
    kv = torch.empty(tokens, 256, device=DEV, dtype=BF)
    kv[-cap:] = torch.randn(cap, 256, device=DEV)
    cache, scale = T.new_cache(1, cap, 1, 1, "plain")
    ops.kv_write_fp8(kv, cache, scale, start=torch.tensor([cap - tokens], dtype=torch.int32, device=DEV))
    want, b = R.quantize(kv[-cap:].view(1, cap, 1, 2, 1, 128))
    assert T.same_bytes(cache, want) and torch.equal(scale.view(torch.uint8), b[..., 0].permute(0, 2, 3, 4, 1))


@pytest.mark.parametrize("n", [1, 40, 150])
def test_attention_past_32_bits(n):
    """One layer of a cache of 65000 tokens and 24 layers: its last tokens lie 6 GB behind its first. They are written by
    kv_write_fp8 and read by attention, whole and by the last tokens alone."""
    cap, layers, H, new, layer = 65000, 24, 16, 300, 23
    torch.manual_seed(0)
    cache = torch.empty(1, cap, layers, 2, H, 128, dtype=torch.uint8, device=DEV).view(R.E4M3)
    scale = torch.full((1, layers, 2, H, cap), 120, dtype=torch.uint8, device=DEV).view(R.E8M0)
    cache.view(torch.uint8)[:, :, layer] = torch.randint(0, 112, (1, cap, 2, H, 128), dtype=torch.uint8, device=DEV)
    cache.view(torch.uint8)[:, -new:] = 0x33
    kv = torch.randn(new, layers * 2 * H * 128, device=DEV)
    ops.kv_write_fp8(kv, cache, scale, start=torch.tensor([cap - new], dtype=torch.int32, device=DEV))
    want, b = R.quantize(kv.view(1, new, layers, 2, H, 128))
    assert T.same_bytes(cache[:, -new:], want) and torch.equal(scale.view(torch.uint8)[..., -new:], b[..., 0].permute(0, 2, 3, 4, 1))
    q = torch.randn(1, n, H, 128, device=DEV).to(BF)
    k, v = (cache[:, :, layer, i].to(D) * scale[:, layer, i].to(D).transpose(1, 2)[..., None] for i in (0, 1))
    for first in (cap - new, 0):
        s = slice(first, cap)
        seg = ops.Segment(cache[:, s, layer, 0], cache[:, s, layer, 1], k_scale=scale[:, layer, 0, :, s], v_scale=scale[:, layer, 1, :, s])
        out = ops.attention(q, [seg])
        for h in range(0, H, 5):
            ref, tol = T.attention_ref(q[:, :, h:h + 1], [(k[:, s, h:h + 1], v[:, s, h:h + 1],
                                                          torch.ones(1, n, cap - first, dtype=torch.bool, device=DEV))], None)
            T.within(out[:, :, h:h + 1], ref, tol)

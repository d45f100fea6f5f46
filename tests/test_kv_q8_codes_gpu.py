"""The quantiser of qkv_rope_append_q8 next to a code's border: bf16 values whose quotient by the row's maximum lies
half-way between two codes."""
import pytest
import torch
from test_kv_q8_gpu import DEV, TOP, TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("t", ["int8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("M", [3, 700, 2500])  # each form of the kernel
def test_value_codes_are_the_nearest_and_halves_go_to_the_even_one(t, hd, M):
    """Value rows are quantised as they are. In 64 bits x * TOP is exact and its quotient by the row's maximum correctly
    rounded, so halves, which 64 bits hold, are met exactly. A quotient that is no half differs from one by more than
    2^-18 of itself (an integer over an 8-bit significand times TOP), where fp32 has steps of 2^-24: the codes are the
    definition's."""
    from dflash_b200 import ops
    g = torch.Generator().manual_seed(hd + M)
    Hkv = 2
    v = torch.randn(M, Hkv, hd, generator=g).bfloat16()
    top = v.abs().amax(-1, keepdim=True)
    for i, f in enumerate((0.5, -0.5, 0.75, -0.375, 0.1875, 0.25)):  # of the maximum: bf16 where its last bits allow it
        v[..., 7 * i + 1] = (top[..., 0].float() * f).bfloat16()
    v[:, 1] = (v[:, 1].float() * 2.0 ** torch.randint(-90, 90, (M, 1), generator=g)).bfloat16()  # exact
    kv_rows = torch.cat([torch.randn(M, Hkv * hd, generator=g).bfloat16(), v.reshape(M, Hkv * hd)], 1).to(DEV)
    codes = torch.zeros((2, 1, Hkv, M, hd), dtype=torch.uint8, device=DEV).view(TYPES[t])
    scale = torch.zeros((2, 1, Hkv, M), device=DEV)
    kv = ops.QuantKV(codes[0], codes[1], scale[0], scale[1])
    w = torch.ones(hd).bfloat16().to(DEV)
    ops.qkv_rope_append_q8(kv_rows, torch.arange(M, dtype=torch.int32, device=DEV), None, w, torch.ones(hd // 2, device=DEV),
                           kv, 0, hd, 1e-6, do_q=False)
    assert ops.device_error() == 0
    z = v.double() * TOP[t] / v.double().abs().amax(-1, keepdim=True)
    want = z.round() if t == "int8" else z.float().to(TYPES[t]).double()  # fp32 holds e4m3's halves, and keeps off them
    got = codes[1, 0].double().cpu().transpose(0, 1)
    assert torch.equal(got, want), f"{int((got != want).sum())} of {got.numel()} codes"
    frac = (z.abs() - z.abs().floor() - 0.5).abs()
    assert t != "int8" or int((frac == 0).sum()) > M  # the halves are there
    assert torch.equal(scale[1, 0].cpu().T, (v.float().abs().amax(-1) / TOP[t]))

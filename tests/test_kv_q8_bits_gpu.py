"""What the bits of an 8-bit cache's attention do not depend on: the sizes of the call around a row; and its scratch."""
import pytest
import torch
from test_kv_q8_gpu import DEV, Cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("form", ["warp", "tc", "wide"])
@pytest.mark.parametrize("t,Hkv,G,hd,gated", [("int8", 2, 4, 128, False), ("e4m3", 2, 3, 128, True), ("int8", 4, 8, 64, True),
                                              ("e4m3", 1, 6, 256, False)])
def test_max_kv_changes_no_bit(form, t, Hkv, G, hd, gated):
    """One chunk or several: rows whose keys lie in the first give the same bits, signs of zeros among them."""
    from dflash_b200 import ops
    B, rows = 24, 16
    g = torch.Generator().manual_seed(hd + G)
    lens = [int(n) for n in torch.randint(rows, 513, (B,), generator=g)]
    lens[0] = 512
    c = Cache(t, lens, Hkv, hd, 64, seed=G)
    c.codes[1].view(torch.uint8)[..., 5] = 0x80 if t == "e4m3" else 0  # a dim of negative zeros
    q = (1.5 * torch.randn(B * rows, Hkv * G, hd, generator=g)).bfloat16().to(DEV)
    seq = torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(rows)
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32, device=DEV)
    gate = torch.randn(B * rows, Hkv * G * hd, generator=g).bfloat16().to(DEV) if gated else None
    one, *more = [ops.attention_q8(q, c.kv, pos, True, max_kv, row_seq=seq, seq_rows=rows, form=form, key_chunk=512,
                                   gate=gate).view(torch.int16) for max_kv in (512, 513, 1024, 5000)]
    assert ops.device_error() == 0
    for x in more:
        assert torch.equal(one, x), int((one != x).sum())


@pytest.mark.parametrize("form", ["warp", "tc", "wide"])
@pytest.mark.parametrize("t,G,hd", [("int8", 4, 128), ("e4m3", 6, 256), ("int8", 2, 64)])
def test_rows_alone_and_together_over_scales_far_apart(form, t, G, hd):
    """Blocks of keys whose V scales are near one another beside blocks where they are not, cut by rows' limits: the
    base of a row's weights is its own."""
    from dflash_b200 import ops
    lens, rows, Hkv = [700, 90, 333], 40, 2
    c = Cache(t, lens, Hkv, hd, 64, seed=8)
    g = torch.Generator().manual_seed(8)
    shape = c.scale.shape[1:]
    far = 2.0 ** torch.randint(-40, 40, shape, generator=g) * (torch.rand(shape, generator=g) < 0.01)
    c.scale[1] *= torch.where(far > 0, far, torch.ones(shape)).to(DEV)
    q = (1.5 * torch.randn(len(lens) * rows, Hkv * G, hd, generator=g)).bfloat16().to(DEV)
    seq = torch.arange(len(lens), dtype=torch.int32, device=DEV).repeat_interleave(rows)
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32, device=DEV)
    kw = dict(causal=True, max_kv=700, form=form, key_chunk=256)
    whole = ops.attention_q8(q, c.kv, pos, row_seq=seq, seq_rows=rows, **kw)
    alone = ops.attention_q8(q, c.kv, pos, row_seq=seq, seq_rows=1, **kw)
    assert ops.device_error() == 0 and whole.isfinite().all()
    assert torch.equal(whole, alone), int((whole != alone).sum())


@pytest.mark.parametrize("form", ["warp", "tc", "wide"])
def test_lengths_that_a_graph_changes_between_its_replays(form):
    """kv_len, rewritten on the device each step as a draft's is: the merge kernel looks up a row's chunks before it
    waits for the chunk kernel, and must find the new ones."""
    from dflash_b200 import ops
    B, rows, Hkv, G, hd = 8, 4, 2, 4, 128
    c = Cache("int8", [1200] * B, Hkv, hd, 64, seed=14)
    g = torch.Generator().manual_seed(14)
    q = torch.randn(B * rows, Hkv * G, hd, generator=g).bfloat16().to(DEV)
    seq = torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(rows)
    pos = torch.zeros(B * rows, dtype=torch.int32, device=DEV)
    kv_len, step = torch.full((B,), 20, dtype=torch.int32, device=DEV), torch.arange(100, 100 + B, dtype=torch.int32, device=DEV)
    out = torch.zeros(B * rows, Hkv * G * hd, dtype=torch.bfloat16, device=DEV)

    def call(lens, o):
        return ops.attention_q8(q, c.kv, pos, False, 1200, kv_len=lens, row_seq=seq, seq_rows=rows, form=form, key_chunk=128,
                                out=o)

    call(kv_len, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_len.add_(step)
        call(kv_len, out)
    for i in range(1, 11):
        graph.replay()
        assert torch.equal(out, call(20 + i * step, torch.zeros_like(out))), i
    assert ops.device_error() == 0


def test_a_workspace_of_another_device_is_refused():
    """Before any launch, whether the call has partial results to put there or not."""
    from types import SimpleNamespace

    from dflash_b200 import ops
    c = Cache("int8", [300], 2, 128)
    q, pos = torch.randn(1, 4, 128).bfloat16().to(DEV), torch.full((1,), 299, dtype=torch.int32, device=DEV)
    elsewhere = SimpleNamespace(attn=torch.empty(1 << 20, dtype=torch.uint8), ensure_attn=lambda n: None)
    for chunk in (128, 512):
        with pytest.raises(ValueError, match="workspace"):
            ops.attention_q8(q, c.kv, pos, True, 300, ws=elsewhere, form="warp", key_chunk=chunk)
        mine = ops.Workspace(torch.device(DEV), gemm_bytes=256, attn_bytes=256)
        a = ops.attention_q8(q, c.kv, pos, True, 300, ws=mine, form="warp", key_chunk=chunk)
        assert torch.equal(a, ops.attention_q8(q, c.kv, pos, True, 300, form="warp", key_chunk=chunk))
    assert ops.device_error() == 0


@pytest.mark.parametrize("form", ["warp", "tc", "wide"])
@pytest.mark.parametrize("t,G,hd", [("int8", 4, 128), ("e4m3", 12, 256), ("int8", 16, 64)])
def test_zeros_have_one_sign(form, t, G, hd):
    """A softmax of one key whose values are zero in half of the dims, beside keys of negative values whose weights vanish:
    the zeros of a call of one chunk are those of a call of several."""
    from dflash_b200 import ops
    lens, rows, Hkv = [700, 350, 90], 24, 2
    c = Cache(t, lens, Hkv, hd, 64, seed=31)
    g = torch.Generator().manual_seed(31)
    raw = c.codes[1].view(torch.uint8)
    neg = 0xF6 if t == "int8" else 0xB4  # -10, -0.75
    raw.copy_(torch.where(torch.rand(raw.shape, generator=g) < 0.5, 0, neg).to(torch.uint8))
    q = (30 * torch.randn(len(lens) * rows, Hkv * G, hd, generator=g)).bfloat16().to(DEV)
    seq = torch.arange(len(lens), dtype=torch.int32, device=DEV).repeat_interleave(rows)
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32, device=DEV)
    one, several = [ops.attention_q8(q, c.kv, pos, True, max_kv, row_seq=seq, seq_rows=rows, form=form, key_chunk=1024)
                    for max_kv in (1024, 1025)]
    assert ops.device_error() == 0 and (one == 0).any()
    one, several = one.view(torch.int16), several.view(torch.int16)
    assert torch.equal(one, several), int((one != several).sum())

"""Sessions over 8-bit K/V caches: speculative decode equals plain decode token for token (one
stream, batches, the hybrid), paged equals contiguous, the caches read back what a bf16 session
holds to within the quantiser's step, and the public entry points take kv_dtype."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.fixture(scope="module")
def tiny():
    from dflash_b200.config import tiny_pair
    from dflash_b200.model import DraftModel, TargetModel
    from dflash_b200.weights import random_draft_weights, random_target_weights
    tcfg, dcfg = tiny_pair()
    target = TargetModel(tcfg, random_target_weights(tcfg, 0), DEV)
    return tcfg, dcfg, target, DraftModel(dcfg, random_draft_weights(dcfg, 0), target)


def _prompts(vocab, lens, seed=8):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lens]


def _decode(target, draft, prompts, n, bs, kv_dtype, **kw):
    from dflash_b200 import ops
    from dflash_b200.runtime import S_FINISHED, SpecSession
    sess = SpecSession(target, draft, len(prompts), max(map(len, prompts)) + n, bs, set(), kv_dtype=kv_dtype, **kw)
    sess.prefill(prompts, n)
    for _ in range(n + 1):
        if bool(sess.state[:, S_FINISHED].all().item()):
            break
        sess.step()
    assert ops.device_error() == 0
    return sess, sess.outputs()[0]


@pytest.mark.parametrize("kv_dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("lens", [[300], [200, 9], [300, 20, 41, 9, 150]])
def test_speculative_decode_equals_plain_decode(tiny, kv_dtype, lens):
    tcfg, dcfg, target, draft = tiny
    prompts = _prompts(tcfg.vocab_size, lens)
    sess, spec = _decode(target, draft, prompts, 40, dcfg.block_size, kv_dtype)
    assert sess.tcache.quantized and sess.dcache.quantized
    assert spec == _decode(target, None, prompts, 40, 1, kv_dtype)[1]
    assert spec == _decode(target, draft, prompts, 40, dcfg.block_size, kv_dtype, paged=False, use_graph=False)[1]


@pytest.mark.parametrize("kv_dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("lens", [[70], [40, 5, 64, 33]])
def test_hybrid_speculative_decode_equals_plain_decode(kv_dtype, lens):
    from dflash_b200.config import tiny_hybrid_pair
    from dflash_b200.hybrid import HybridTargetModel
    from dflash_b200.model import DraftModel
    from dflash_b200.weights import random_draft_weights, random_target_weights
    tcfg, dcfg = tiny_hybrid_pair()
    target = HybridTargetModel(tcfg, random_target_weights(tcfg, 0, std=0.05), DEV)
    draft = DraftModel(dcfg, random_draft_weights(dcfg, 0), target, mask_mode="causal")
    prompts = _prompts(tcfg.vocab_size, lens)
    spec = _decode(target, draft, prompts, 24, dcfg.block_size, kv_dtype)[1]
    assert spec == _decode(target, None, prompts, 24, 1, kv_dtype)[1]


@pytest.mark.parametrize("kv_dtype,step", [("int8", 1 / 254), ("e4m3", 2.0 ** -4)])
def test_first_layer_cache_holds_the_bf16_rows_to_a_step(tiny, kv_dtype, step):
    """Layer 0 sees the same projection rows in both sessions: the 8-bit cache is the bf16 one to
    within half a quantiser step of the row's largest magnitude (int8: max / 254; e4m3: 2^-4 of the
    value, at most 2^-4 max) and the bf16 path's own roundings of K (norm and store, 2^-8 each,
    through a rotation that adds two of them: 4 x 2^-8 of the row's largest)."""
    tcfg, dcfg, target, draft = tiny
    prompts = _prompts(tcfg.vocab_size, [200, 130])
    ref = _decode(target, draft, prompts, 1, dcfg.block_size, "bf16")[0]
    got = _decode(target, draft, prompts, 1, dcfg.block_size, kv_dtype)[0]
    for b, p in enumerate(prompts):
        n = len(p)
        for x, y in zip(ref.tcache.gather(0, b, n), got.tcache.gather(0, b, n)):
            assert x.shape == y.shape and y.dtype == torch.bfloat16
            top = x.float().abs().amax(-1, keepdim=True)
            assert ((x.float() - y.float()).abs() <= (step * 1.02 + 5 * 2.0 ** -8) * top).all()
    bytes_of = lambda c: sum(t.numel() * t.element_size() for t in (c.k, c.v, c.k_scale, c.v_scale) if t is not None)  # noqa: E731
    assert bytes_of(got.tcache) < 0.54 * bytes_of(ref.tcache)  # (64 + 4) / 128


def test_public_entry_points_take_kv_dtype(tiny):
    from dflash_b200.adapters import Qwen3TargetAdapter
    from dflash_b200.runtime import SpecSession, dflash_generate, dflash_generate_batch_stream
    tcfg, dcfg, target, draft = tiny
    prompt = _prompts(tcfg.vocab_size, [50])[0]
    want = _decode(target, None, [prompt], 12, 1, "int8")[1][0]
    toks, metrics = dflash_generate(target, draft, prompt, 12, 0.0, set(), None, None, kv_dtype="int8")
    assert toks == want and metrics["num_output_tokens"] == 12
    got = [t for evs in dflash_generate_batch_stream(target, draft, [prompt], [12], 0.0, set(), kv_dtype="int8")
           for e in evs for t in e.token_ids]
    assert prompt + got == want
    with pytest.raises(ValueError, match="kv_dtype"):
        SpecSession(target, draft, 1, 64, 8, kv_dtype="fp8")
    # the adapter contract over an 8-bit cache: a block in two halves gives the rows of one call
    ad = Qwen3TargetAdapter()
    rows = torch.tensor(prompt, dtype=torch.int32)
    one, two = ad.make_cache(target, 64, kv_dtype="e4m3"), ad.make_cache(target, 64, kv_dtype="e4m3")
    whole = ad.forward_with_hidden_states(target, rows[:16], one, [1, 3])[0]
    halves = [ad.forward_with_hidden_states(target, rows[i:i + 8], two, [1, 3])[0] for i in (0, 8)]
    assert torch.equal(whole, torch.cat(halves, 1))

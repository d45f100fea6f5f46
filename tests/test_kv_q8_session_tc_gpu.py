"""Sessions over 8-bit K/V caches whose sizes select the tcgen05 attention: speculative decode equals plain decode, in
its tokens and in every committed row of the caches."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.fixture(scope="module")
def dense():
    from dflash_b200.config import tiny_pair
    from dflash_b200.model import DraftModel, TargetModel
    from dflash_b200.weights import random_draft_weights, random_target_weights
    tcfg, dcfg = tiny_pair()
    target = TargetModel(tcfg, random_target_weights(tcfg, 0), DEV)
    return tcfg, dcfg, target, DraftModel(dcfg, random_draft_weights(dcfg, 0), target)


@pytest.fixture(scope="module")
def hybrid():
    from dflash_b200.config import tiny_hybrid_pair
    from dflash_b200.hybrid import HybridTargetModel
    from dflash_b200.model import DraftModel
    from dflash_b200.weights import random_draft_weights, random_target_weights
    tcfg, dcfg = tiny_hybrid_pair()
    target = HybridTargetModel(tcfg, random_target_weights(tcfg, 0, std=0.05), DEV)
    return tcfg, dcfg, target, DraftModel(dcfg, random_draft_weights(dcfg, 0), target, mask_mode="causal")


def _decode(target, draft, prompts, n, bs, kv_dtype, max_total):
    from dflash_b200 import ops
    from dflash_b200.runtime import S_FINISHED, SpecSession
    sess = SpecSession(target, draft, len(prompts), max_total, bs, set(), kv_dtype=kv_dtype)
    sess.prefill(prompts, n)
    for _ in range(n + 1):
        if bool(sess.state[:, S_FINISHED].all().item()):
            break
        sess.step()
    assert ops.device_error() == 0
    return sess, sess.outputs()[0]


def _rows(sess, b, n):
    """Codes and scales of positions [0, n) of sequence b, every layer."""
    kv = getattr(sess.tcache, "kv", sess.tcache)
    out = []
    for t in (kv.k.view(torch.uint8), kv.v.view(torch.uint8), kv.k_scale, kv.v_scale):
        if kv.page_table is None:
            out.append(t[:, b, :, :n])
        else:
            pages = kv.page_table[b, :(n + kv.page_size - 1) // kv.page_size].long()
            out.append(t[:, pages].transpose(1, 2).flatten(2, 3)[:, :, :n])
    return out


def _check(models, lens, n, kv_dtype, max_total, split):
    tcfg, dcfg, target, draft = models
    g = torch.Generator().manual_seed(sum(lens))
    prompts = [torch.randint(0, tcfg.vocab_size, (p,), generator=g).tolist() for p in lens]
    spec, toks = _decode(target, draft, prompts, n, dcfg.block_size, kv_dtype, max_total)
    plain, want = _decode(target, None, prompts, n, 1, kv_dtype, max_total)
    for s in (spec, plain):
        assert s.step_split == {"form": split[0], "key_chunk": split[1]}
    assert toks == want
    for b, p in enumerate(lens):
        for x, y in zip(_rows(spec, b, p + n - 1), _rows(plain, b, p + n - 1)):
            assert torch.equal(x, y), (b, int((x != y).sum()))
    return spec, plain


@pytest.mark.parametrize("kv_dtype", ["int8", "e4m3"])
def test_one_chunk_and_several(dense, kv_dtype):
    """max_kv holds a session's block size: plain decode has one chunk of keys, speculative decode two."""
    lens = [int(n) for n in torch.randint(2, 150, (64,), generator=torch.Generator().manual_seed(1))]
    spec, plain = _check(dense, lens, 24, kv_dtype, 500, ("tc", 512))
    assert plain.cap <= 512 < spec.cap


@pytest.mark.parametrize("kv_dtype", ["int8", "e4m3"])
def test_prompts_of_several_prefill_splits(dense, kv_dtype):
    """Prompts beyond 2048 tokens beside short ones; the steps' rows have up to five chunks."""
    _check(dense, [2300, 9, 600, 2049, 1, 77, 31, 513, 128, 1100], 20, kv_dtype, 2400, ("tc", 512))


@pytest.mark.parametrize("kv_dtype", ["int8", "e4m3"])
def test_hybrid(hybrid, kv_dtype):
    """Gated attention at head_dim 256; one chunk and two again."""
    _check(hybrid, [70, 300, 5, 64, 129, 33, 200, 18, 256, 90, 3, 41, 150, 60, 20, 10], 16, kv_dtype, 500, ("tc", 512))

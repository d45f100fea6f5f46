"""Models whose heads the 8-bit cache kernels do not take: refused where a cache, session or generator is made (no GPU)."""
from types import SimpleNamespace

import pytest

from dflash_b200.config import DraftConfig, TargetConfig, qwen3_4b_pair

BAD = [dict(num_attention_heads=34, num_key_value_heads=2), dict(num_attention_heads=10, num_key_value_heads=4),
       dict(head_dim=96), dict(head_dim=32)]


def _model(cfg):
    return SimpleNamespace(cfg=cfg, device="meta", attn_index={})


@pytest.mark.parametrize("kw", BAD + [dict(partial_rotary_factor=0.0625)])
@pytest.mark.parametrize("name", ["int8", "e4m3"])
def test_targets(kw, name):
    from dflash_b200.hybrid import HybridTargetModel
    from dflash_b200.model import TargetModel
    from dflash_b200.runtime import SpecSession
    model = _model(TargetConfig(**kw))
    for make in (lambda: TargetModel.make_cache(model, 1, 64, dtype=name),
                 lambda: TargetModel.make_cache(model, 1, 64, lengths=[10], dtype=name),
                 lambda: HybridTargetModel.make_cache(model, 1, 64, dtype=name),
                 lambda: SpecSession(model, None, 1, 64, 1, kv_dtype=name)):
        with pytest.raises(ValueError, match="kv_dtype"):
            make()


@pytest.mark.parametrize("kw", BAD)
def test_drafts(kw):
    from dflash_b200.model import DraftModel
    from dflash_b200.runtime import SpecSession
    model = _model(DraftConfig(**kw))
    for make in (lambda: DraftModel.make_cache(model, 1, 64, dtype="int8"),
                 lambda: SpecSession(_model(TargetConfig()), model, 1, 64, 16, kv_dtype="int8")):
        with pytest.raises(ValueError, match="kv_dtype"):
            make()


def test_the_limits_are_the_kernels(lib):
    """What model_kv_dtype takes the scratch query and the append take too, and the other way round."""
    import ctypes

    import torch
    from dflash_b200 import _lib, ops
    from dflash_b200.model import model_kv_dtype
    for cfg in qwen3_4b_pair():
        assert model_kv_dtype(cfg, "int8") is torch.int8 and model_kv_dtype(cfg, "bf16") is torch.bfloat16
    for kw in BAD:
        model_kv_dtype(TargetConfig(**kw), "bf16")  # as it was
    for G in (1, 16, 17):
        desc = ops.KvQ8(n_kv_heads=2, n_seqs=1, cap=4096, head_dim=128)
        need = _lib.query("dfl_attention_q8_workspace_bytes", ctypes.byref(desc), 1, 2 * G, 1, 1, 4096, 1, 128)
        assert (need > 0) == (G <= ops.Q8_MAX_GROUP)


def test_generators(monkeypatch):
    from dflash_b200 import api
    from dflash_b200.adapters import LoadedTargetModel
    target = LoadedTargetModel.__new__(LoadedTargetModel)
    object.__setattr__(target, "__dict__", {"model": _model(TargetConfig(num_attention_heads=34, num_key_value_heads=2)),
                                            "adapter": SimpleNamespace(family="qwen3")})
    draft = api.DraftModel.__new__(api.DraftModel)
    draft.cfg = DraftConfig()
    with pytest.raises(ValueError, match="kv_dtype"):
        api.DFlashGenerator(target, draft, kv_dtype="int8")
    assert api.DFlashGenerator(target, draft).kv_dtype == "bf16"


@pytest.mark.parametrize("rows,max_kv", [(1024, 131072), (4096, 32768), (4096, 131072), (16384, 65536), (16384, 131072),
                                         (65536, 131072), (16384, 2 ** 31 - 1)])
def test_scratch_of_long_prompts_stays_bounded(lib, rows, max_kv):
    """The partials of a call that fills the SMs many times over: at most 8 KB a key of the longest row, whatever the rows
    (a chunk of 8192 keys for each wave of 148 CTAs, of 256 (row, head) pairs of 128 floats and two: 19.7 MB / 8192)."""
    import ctypes

    from dflash_b200 import _lib, ops
    desc = ops.KvQ8(n_kv_heads=8, n_seqs=1, cap=max_kv, head_dim=128)
    need = _lib.query("dfl_attention_q8_workspace_bytes", ctypes.byref(desc), rows, 32, rows, 1, max_kv, 0, 0)
    assert need <= 8192 * max_kv

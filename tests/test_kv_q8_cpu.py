"""8-bit K/V cache: host-side refusals of the C entry points and the Python wrappers (no GPU)."""
import ctypes

import pytest
import torch


def _desc(**kw):
    from dflash_b200.ops import KvQ8
    d = dict(k=64, v=64, k_scale=64, v_scale=64, seq_stride=1024 * 128, head_stride=512 * 128,
             scale_seq_stride=1024, scale_head_stride=512, page_table=None, pt_stride=0, page_size=0, n_seqs=2,
             n_pages=0, cap=512, n_kv_heads=2, head_dim=128, type=0)
    d.update(kw)
    return ctypes.byref(KvQ8(**d))


def _append(desc, **kw):
    a = dict(qkv=64, ld=1024, qs=128, pos=64, row_seq=None, qn=64, kn=64, inv=64, q_out=64, M=2, Hq=4, rot=128, eps=1e-6,
             do_q=1)
    a.update(kw)
    return ("dfl_qkv_rope_append_q8", a["qkv"], a["ld"], a["qs"], a["pos"], a["row_seq"], a["qn"], a["kn"], a["inv"],
            a["q_out"], desc, a["M"], a["Hq"], a["rot"], a["eps"], a["do_q"], None)


def _attn(desc, **kw):
    a = dict(q=64, pos=64, row_seq=None, kv_len=None, seq_rows=0, M=2, Hq=4, causal=1, scale=0.1, max_kv=512, form=0, chunk=0,
             out=64, ldo=512, ws=None, ws_bytes=0)
    a.update(kw)
    return ("dfl_attention_q8", a["q"], desc, a["pos"], a["row_seq"], a["kv_len"], a["seq_rows"], a["M"], a["Hq"],
            a["causal"], a["scale"], a["max_kv"], a["form"], a["chunk"], a["out"], a["ldo"], None, 0, 0, a["ws"], a["ws_bytes"],
            None)


def _read(desc, **kw):
    a = dict(pos=64, row_seq=None, M=2, k=64, v=64)
    a.update(kw)
    return ("dfl_kv_read_q8", desc, a["pos"], a["row_seq"], a["M"], a["k"], a["v"], None)


@pytest.mark.parametrize("bad,status", [
    (dict(k=None), 1), (dict(v_scale=None), 1), (dict(type=2), 1), (dict(head_dim=96), 2), (dict(n_kv_heads=0), 1),
    (dict(cap=0), 1), (dict(n_seqs=0), 1), (dict(seq_stride=-16), 1), (dict(k=72), 2), (dict(head_stride=8), 2),
    (dict(page_table=64, page_size=32, pt_stride=4, n_pages=3), 1),
    (dict(page_table=64, page_size=96, pt_stride=4, n_pages=3), 1),
    (dict(page_table=64, page_size=64, pt_stride=0, n_pages=3), 1),
    (dict(page_table=64, page_size=64, pt_stride=4, n_pages=0), 1),
])
def test_bad_caches_are_refused_by_every_entry_point(lib, bad, status):
    from dflash_b200 import _lib
    for make in (_append, _attn, _read):
        with pytest.raises(_lib.DFlashKernelError) as e:
            _lib.call(*make(_desc(**bad)))
        assert e.value.status == status and make(_desc())[0] in str(e.value)


@pytest.mark.parametrize("call,status", [
    (_append(_desc(), pos=None), 1), (_append(_desc(), q_out=None), 1), (_append(_desc(), rot=24), 2),
    (_append(_desc(), rot=144), 2), (_append(_desc(), ld=1020), 2), (_append(_desc(), ld=1016), 2),
    (_append(_desc(), qs=64), 2), (_append(_desc(), qkv=66), 2), (_append(_desc(), M=-1), 1),
    (_append(None), 1), (_attn(None), 1), (_read(None), 1),
    (_read(_desc(), pos=None), 1), (_read(_desc(), k=72), 2), (_read(_desc(), M=-3), 1),
    (_attn(_desc(), q=None), 1), (_attn(_desc(), causal=0), 1), (_attn(_desc(), Hq=5), 1), (_attn(_desc(), Hq=34), 2),
    (_attn(_desc(), max_kv=0), 1), (_attn(_desc(), chunk=64), 1), (_attn(_desc(), chunk=-128), 1),
    (_attn(_desc(), scale=float("nan")), 1), (_attn(_desc(), scale=float("inf")), 1), (_attn(_desc(), ldo=510), 2),
    (_attn(_desc(), ldo=256), 2), (_attn(_desc(), out=68), 2), (_attn(_desc(), q=72), 2),
    (_attn(_desc(), chunk=128), 4), (_attn(_desc(), chunk=128, ws=64, ws_bytes=100), 4),
    (_attn(_desc(), seq_rows=-1), 1), (_attn(_desc(), form=4), 1), (_attn(_desc(), form=-1), 1), (_attn(_desc(cap=1 << 30), max_kv=1 << 30, chunk=128, ws=64, ws_bytes=1 << 62), 2),
])
def test_bad_arguments_are_refused_before_any_launch(lib, call, status):
    from dflash_b200 import _lib
    with pytest.raises(_lib.DFlashKernelError) as e:
        _lib.call(*call)
    assert e.value.status == status and call[0] in str(e.value)


def test_empty_calls_succeed_and_scratch_follows_the_chunks(lib):
    from dflash_b200 import _lib
    for make in (_append, _attn, _read):
        _lib.call(*make(_desc(), M=0))
    size = lambda *a: _lib.query("dfl_attention_q8_workspace_bytes", _desc(), *a)  # noqa: E731
    for form in (1, 2, 3):
        assert size(2, 4, 1, 0, 512, form, 512) == 0  # one chunk
        assert size(2, 4, 1, 0, 512, form, 128) == 4 * 2 * 4 * 128 * 4 + 4 * 2 * 4 * 8
        assert size(2, 4, 1, 0, 513, form, 128) > size(2, 4, 1, 0, 512, form, 128)
        assert size(0, 4, 1, 0, 512, form, 128) == 0 and size(2, 4, 1, 0, 512, form, 100) == 0
    assert size(2, 4, 1, 0, 512, 4, 128) == 0


def test_wrappers_take_cuda_tensors_only():
    from dflash_b200 import ops
    z = torch.zeros((1, 2, 64, 128), dtype=torch.int8)
    s = torch.zeros((1, 2, 64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.QuantKV(z, z, s, s)


def test_scratch_query_answers_0_where_the_call_would_refuse(lib):
    """Head counts that the attention refuses (no whole group, more than 16 heads a group, none at
    all) give 0 bytes, not an arithmetic fault."""
    from dflash_b200 import _lib, ops
    c = ops.KvQ8(n_kv_heads=8, n_seqs=1, cap=4096, head_dim=128)
    ref = ctypes.byref(c)
    for Hq in (4, 12, 136, 264):
        assert _lib.query("dfl_attention_q8_workspace_bytes", ref, 16, Hq, 16, 1, 4096, 0, 0) == 0
    assert _lib.query("dfl_attention_q8_workspace_bytes", ref, 16, 32, 16, 1, 4096, 0, 0) > 0
    assert _lib.query("dfl_attention_q8_workspace_bytes", ref, 16, 128, 16, 1, 4096, 1, 128) > 0


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_session_split_follows_the_shared_sizes(hd):
    """Forms the entry point knows, chunks it takes; short streams in the warp form, long or many in tcgen05."""
    from dflash_b200.model import q8_split
    from dflash_b200.ops import Q8_CHUNK, Q8_FORMS
    seen = set()
    for batch in (1, 2, 4, 64):
        for total in (64, 1000, 5000, 40000, 131072):
            form, chunk = q8_split(batch, 8, total, hd)
            assert form in Q8_FORMS and chunk % Q8_CHUNK == 0 and Q8_CHUNK <= chunk <= 8192
            assert (form == "warp") == (total * batch * 8 <= (14336 if hd == 256 else 36864))
            seen.add(form)
    assert seen == {"warp", "tc"}

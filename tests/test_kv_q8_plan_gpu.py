"""attention_q8 with the form and split that it chooses itself, on both sides of its thresholds, and the wide form's second
softmax group, against 64 bits."""
import pytest
import torch
from test_kv_q8_gpu import DEV, Cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _attention64(val, q, lens, pos, causal, gate):
    """(o, tolerance) of runs of q.shape[0] / len(lens) rows, in 64 bits; the tolerance is that of test_kv_q8_gpu.py: the
    output's bf16, the weights' fp16 and its lower end, scores and sums in fp32."""
    B, (M, Hq, hd) = len(lens), q.shape
    T, Hkv = M // B, val.shape[2]
    o, tol = torch.zeros(M, Hq * hd, dtype=torch.float64), torch.zeros(M, Hq * hd, dtype=torch.float64)
    smax, A, low = 0.0, torch.zeros_like(o), torch.zeros_like(o)
    for b, n in enumerate(lens):
        k, v = val[0, b, :, :n].to(DEV), val[1, b, :, :n].to(DEV)
        s = slice(b * T, (b + 1) * T)
        qb = q[s].to(DEV).double().view(T, Hkv, -1, hd)
        x = torch.einsum("thgd,hnd->thgn", qb, k) * hd ** -0.5
        if causal:
            x = x.masked_fill((torch.arange(n, device=DEV) > pos[s, None].to(DEV))[:, None, None], -torch.inf)
        p = torch.softmax(x, -1)
        smax = max(smax, float(torch.einsum("thgd,hnd->thgn", qb.abs(), k.abs()).max()) * hd ** -0.5)
        o[s] = torch.einsum("thgn,hnd->thgd", p, v).reshape(T, -1).cpu()
        A[s] = torch.einsum("thgn,hnd->thgd", p, v.abs()).reshape(T, -1).cpu()
        top = (n * 2.0 ** -28 * v.abs().amax((1, 2))).cpu()
        low[s] = top[:, None, None].expand(Hkv, Hq // Hkv, hd).reshape(1, -1).expand(T, -1)
    if gate is not None:
        g = torch.sigmoid(gate.double())
        o, A, low = o * g, A * g, low * g
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2.0 ** -18 + 2 * hd * 2.0 ** -23 * smax) * A + low
    return o, tol


def _check(t, lens, rows, Hkv, G, hd, page, causal, gated, **kw):
    from dflash_b200 import ops
    c = Cache(t, lens, Hkv, hd, page, seed=hd + rows, wide=rows % 2 == 1)
    g = torch.Generator().manual_seed(7)
    B, Hq = len(lens), Hkv * G
    q = (1.5 * torch.randn(B * rows, Hq, hd, generator=g)).bfloat16()
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32)
    assert int(pos.min()) >= 0
    gate = torch.randn(B * rows, Hq * hd, generator=g).bfloat16() if gated else None
    seq = torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(rows) if B > 1 else None
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    run = lambda **k: ops.attention_q8(q.to(DEV), c.kv, pos.to(DEV), causal, max(lens), kv_len=kv_len, row_seq=seq,  # noqa: E731
                                       seq_rows=rows, gate=gate.to(DEV) if gated else None, **k)
    out = run(**kw)
    assert ops.device_error() == 0
    ref, tol = _attention64(c.val, q, lens, pos, causal, gate)
    err = (out.double().cpu() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())
    return out, run


@pytest.mark.parametrize("t,lens,rows,Hkv,G,hd,page,causal,gated,chunk", [
    # 129 to 256 (token, head) rows a tile: a second group of 1 to 128 rows, one tile or several, one chunk or several
    ("int8", [513], 43, 2, 3, 64, 64, True, True, 128),
    ("e4m3", [700], 33, 2, 4, 128, 64, True, True, 1024),
    ("int8", [700], 64, 2, 4, 128, 64, True, True, 256),
    ("e4m3", [1300], 64, 2, 4, 64, 0, True, False, 512),
    ("int8", [650, 300], 50, 2, 4, 128, 64, False, True, 1024),
    ("e4m3", [900], 130, 1, 8, 128, 64, True, True, 384),
    ("e4m3", [257, 512, 129], 16, 1, 16, 128, 128, True, False, 256),
    ("int8", [1, 2000], 1, 1, 16, 128, 0, True, False, 512),
    ("int8", [333], 300, 1, 1, 128, 0, True, True, 512),
    ("e4m3", [150], 149, 1, 1, 128, 64, False, False, 512),
])
def test_wide_tiles_of_two_groups(t, lens, rows, Hkv, G, hd, page, causal, gated, chunk):
    _check(t, lens, rows, Hkv, G, hd, page, causal, gated, form="wide", key_chunk=chunk)


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


@pytest.mark.parametrize("t,lens,rows,Hkv,G,hd,page,causal,gated,form,chunk", [
    # small calls: the warp form in tiles of 16 rows (head_dim 256: 32), and what is just too large for that
    ("int8", [700], 16, 8, 4, 128, 64, True, False, "warp", 128),
    ("e4m3", [1100], 16, 4, 6, 256, 0, True, True, "warp", 256),
    ("int8", [2200] + _spread(600, 1900, 3), 16, 8, 4, 128, 64, True, False, "tc", 512),
    # single tokens: all of a wave's SMs by chunks; runs of one chunk cut in halves and at three quarters; uncut
    ("e4m3", _spread(100, 2300, 9), 1, 8, 4, 128, 64, True, False, "warp", 384),
    ("e4m3", _spread(200, 2100, 36), 1, 8, 4, 128, 64, True, False, "warp", 1152),
    ("int8", _spread(200, 2100, 64), 1, 8, 4, 128, 64, False, False, "warp", 1664),
    ("int8", _spread(200, 1900, 64), 1, 8, 4, 128, 64, True, True, "warp", 1920),
    ("int8", _spread(1, 500, 30), 1, 8, 4, 64, 0, True, False, "warp", 512),
    # many chunks of one kv head
    ("int8", [40000], 2, 1, 16, 128, 64, True, False, "warp", 640),
    ("e4m3", [60000], 10, 1, 4, 64, 64, True, False, "tc", 1024),
    # verify blocks of many sequences, gated blocks at head_dim 256, prompt rows
    ("int8", _spread(16, 1500, 64), 16, 8, 4, 128, 64, True, False, "tc", 1536),
    ("e4m3", _spread(300, 2000, 8), 16, 4, 6, 256, 0, True, True, "wide", 512),
    ("int8", [4000], 128, 8, 4, 128, 64, True, False, "wide", 512),
    ("e4m3", [3000], 512, 4, 4, 64, 0, True, True, "wide", 768),
    # a second wave of tc tiles; long rows of many sequences
    ("int8", _spread(82, 99, 48), 82, 2, 4, 64, 64, True, False, "wide", 512),
    ("int8", _spread(100, 9000, 80), 16, 1, 16, 64, 64, True, False, "wide", 4608),
])
def test_the_choice_of_a_call(t, lens, rows, Hkv, G, hd, page, causal, gated, form, chunk):
    """Right against 64 bits, and the bits of the call that names the form and split expected here."""
    out, run = _check(t, lens, rows, Hkv, G, hd, page, causal, gated)
    assert torch.equal(out, run(form=form, key_chunk=chunk))
    others = [run(form=f, key_chunk=k) for f, k in ((form, chunk + 128), (form, max(128, chunk - 128)))]
    if min(lens) > chunk:  # rows of several chunks: another split rounds otherwise, so the one above is the one
        assert not all(torch.equal(out, x) for x in others)

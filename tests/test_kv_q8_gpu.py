"""8-bit K/V cache: the quantising append, the attention over the codes and the read-back, each
against a plain implementation in 64 bits; rows that do not depend on their neighbours, masked
garbage, untouched rows, strides, streams and graphs.

Tolerances count the roundings: half a step is eps / 2 relative to the value (bf16 2^-8, fp16 2^-11,
e4m3 2^-4); fp32 work in between is given 2^-18 of the largest term (a few ulps of 2^-24 per step
over sums of at most 256)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}


@pytest.fixture(scope="module", autouse=True)
def _need(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _quantise(x, t):
    a = x.abs().amax(-1)
    y = x * torch.where(a > 0, TOP[t] / a, torch.zeros_like(a))[..., None]
    return (y.round() if t == "int8" else y).to(TYPES[t]), a / TOP[t]


class Cache:
    """Random codes for B sequences of the given lengths; everything behind a length is garbage
    (NaN and huge scales, random codes without e4m3 NaNs)."""

    def __init__(self, t, lens, Hkv, hd, page=0, seed=0, slack=5, wide=False):
        from dflash_b200 import ops
        g = torch.Generator().manual_seed(seed)
        B, cap = len(lens), max(lens) + slack
        x = torch.randn((2, B, Hkv, cap, hd), generator=g)
        x[0, ..., ::16] *= 5
        x *= torch.exp(2 * torch.randn((2, B, Hkv, cap, 1), generator=g)) if wide else 1 + torch.rand((2, B, Hkv, cap, 1), generator=g)
        codes, scale = _quantise(x, t)
        self.val = codes.double() * scale.double()[..., None]  # [2, B, Hkv, cap, hd]
        for b, n in enumerate(lens):
            scale[:, b, :, n:] = torch.tensor([math.nan, 3e30, math.inf, 1.0, -2.0])[torch.arange(cap - n) % 5]
        table = None
        if page:
            need = [(n + page - 1) // page for n in lens]
            order = torch.randperm(sum(need) + 1, generator=g)
            table = torch.full((B, max(need) + 1), -7, dtype=torch.int32)
            pc = torch.full((2, sum(need) + 1, Hkv, page, hd), 3, dtype=torch.uint8)
            ps = torch.full((2, sum(need) + 1, Hkv, page), math.nan)
            at = 0
            for b, n in enumerate(need):
                for i in range(n):
                    pg = int(order[at])
                    table[b, i] = pg
                    m = min(page, cap - i * page)
                    pc[:, pg, :, :m] = codes.view(torch.uint8)[:, b, :, i * page:i * page + m]
                    ps[:, pg, :, :m] = scale[:, b, :, i * page:i * page + m]
                    at += 1
            codes, scale = pc.view(TYPES[t]), ps
            table = table.to(DEV)
        self.codes, self.scale = codes.to(DEV), scale.to(DEV)
        self.kv = ops.QuantKV(self.codes[0], self.codes[1], self.scale[0], self.scale[1], page_table=table,
                              page_size=page)


def _attention64(val, q, lim, seq, scale, gate=None):
    """(o, tolerance): attention in 64 bits; rows with lim 0 are zero."""
    M, Hq, hd = q.shape
    Hkv = val.shape[2]
    G = Hq // Hkv
    o, A, smax = torch.zeros(M, Hq, hd, dtype=torch.float64), torch.zeros(M, Hq, hd, dtype=torch.float64), 0.0
    low = torch.zeros(M, Hq, hd, dtype=torch.float64)
    for m in range(M):
        n = int(lim[m])
        if n <= 0:
            continue
        k, v = val[0, int(seq[m]), :, :n], val[1, int(seq[m]), :, :n]
        qm = q[m].double().view(Hkv, G, hd)
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", qm, k) * scale, -1)
        smax = max(smax, float((torch.einsum("hgd,hnd->hgn", qm.abs(), k.abs()) * abs(scale)).max()))
        o[m] = torch.einsum("hgn,hnd->hgd", p, v).reshape(Hq, hd)
        A[m] = torch.einsum("hgn,hnd->hgd", p, v.abs()).reshape(Hq, hd)
        # fp16's lower end: a weight p_j vs_j is held in units in which the row's largest e_j times
        # the largest vs is at least 2^3, rounded there to a multiple of 2^-24 at worst: off by at
        # most 2^-25 / 2^3 = 2^-28 of max p * max vs <= max vs. Summed over n codes of at most TOP,
        # and max vs * TOP being the largest |v|: n 2^-28 max |v|
        low[m] = (n * 2.0 ** -28 * v.abs().amax((1, 2)))[:, None, None].expand(Hkv, G, hd).reshape(Hq, hd)
    o, A, low = o.reshape(M, Hq * hd), A.reshape(M, Hq * hd), low.reshape(M, Hq * hd)
    if gate is not None:
        s = torch.sigmoid(gate.double())
        o, A, low = o * s, A * s, low * s
    # weights: fp16 (2^-11) and their exponent's error: scores summed in fp32 over hd terms of at
    # most smax in all, 2^-23 each step, in numerator and denominator
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2.0 ** -18 + 2 * hd * 2.0 ** -23 * smax) * A + low
    return o, tol


CASES = [
    # type, lens, rows, Hkv, G, hd, page, causal, gate, form, key_chunk
    ("int8", [1], 1, 1, 1, 64, 0, True, False, "auto", 0),
    ("e4m3", [1], 1, 2, 4, 128, 64, True, False, "auto", 0),
    ("int8", [33, 32, 31], 1, 2, 3, 128, 64, True, True, "auto", 0),
    ("e4m3", [129, 640, 7], 1, 1, 8, 256, 128, True, False, "warp", 128),
    ("int8", [1000, 517], 5, 2, 4, 128, 0, True, False, "warp", 256),
    ("e4m3", [200, 130, 384], 16, 2, 4, 128, 64, True, False, "warp", 128),
    ("int8", [700, 90], 16, 1, 6, 256, 0, True, True, "warp", 512),
    ("e4m3", [150], 150, 2, 5, 64, 64, True, False, "warp", 128),
    ("int8", [261], 37, 1, 16, 128, 128, True, True, "auto", 0),
    ("int8", [300, 1, 64], 16, 2, 2, 64, 0, False, False, "warp", 128),
    ("e4m3", [77, 513], 8, 2, 4, 128, 64, False, True, "auto", 0),
    ("int8", [2100], 1, 2, 7, 128, 64, False, False, "warp", 128),
    # the tcgen05 form
    ("int8", [1], 1, 1, 1, 128, 64, True, False, "tc", 512),
    ("e4m3", [1025, 33, 511], 1, 2, 4, 128, 64, True, True, "tc", 512),
    ("int8", [1100, 97, 640], 16, 2, 4, 128, 0, True, False, "tc", 512),
    ("e4m3", [640, 130], 16, 1, 6, 256, 128, True, True, "tc", 512),
    ("int8", [700, 5], 5, 2, 3, 256, 0, False, False, "tc", 1024),
    ("e4m3", [900, 64], 16, 2, 2, 64, 64, False, True, "tc", 512),
    ("int8", [2500], 100, 1, 8, 64, 64, True, False, "tc", 1024),
    ("int8", [1300, 514], 5, 2, 4, 128, 64, True, False, "tc", 1024),
    # its 128-row tiles
    ("int8", [1], 1, 1, 1, 128, 64, True, False, "wide", 512),
    ("e4m3", [700, 33, 511], 32, 2, 4, 128, 64, True, True, "wide", 512),
    ("int8", [300], 300, 1, 1, 64, 0, True, False, "wide", 512),
    ("e4m3", [640, 130], 16, 1, 6, 256, 128, True, True, "wide", 512),
    ("int8", [700, 45], 40, 2, 3, 256, 0, False, False, "wide", 1024),
    ("e4m3", [900, 64, 65], 21, 2, 2, 64, 64, False, True, "wide", 384),
    ("int8", [1300, 514], 5, 2, 4, 128, 64, True, False, "wide", 1024),
]


@pytest.mark.parametrize("t,lens,rows,Hkv,G,hd,page,causal,gated,form,chunk", CASES)
def test_attention_matches_64_bits(t, lens, rows, Hkv, G, hd, page, causal, gated, form, chunk):
    from dflash_b200 import ops
    c = Cache(t, lens, Hkv, hd, page, seed=hd + rows, wide=rows == 5)
    g = torch.Generator().manual_seed(7)
    B, Hq = len(lens), Hkv * G
    q = (1.5 * torch.randn(B * rows, Hq, hd, generator=g)).bfloat16()
    seq = torch.arange(B, dtype=torch.int32).repeat_interleave(rows)
    # the run's last row sits at its sequence's last position (positions below 0: rows skipped)
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32).clamp_min(-1)
    kv_len = torch.tensor(lens, dtype=torch.int32)
    gate = torch.randn(B * rows, Hq * hd, generator=g).bfloat16() if gated else None
    out = torch.full((B * rows, Hq * hd), 9.0, dtype=torch.bfloat16, device=DEV)
    ops.attention_q8(q.to(DEV), c.kv, pos.to(DEV), causal, max(lens), kv_len=kv_len.to(DEV),
                     row_seq=seq.to(DEV) if B > 1 else None, seq_rows=rows, form=form, key_chunk=chunk, out=out,
                     gate=gate.to(DEV) if gated else None)
    lim = pos + 1 if causal else kv_len[seq.long()]
    ref, tol = _attention64(c.val, q, lim, seq, hd ** -0.5, gate)
    live = pos >= 0
    err = (out.double().cpu() - ref).abs()[live]
    assert ops.device_error() == 0
    assert (err <= tol[live]).all(), float((err / tol[live]).max())
    assert (out[~live.to(DEV)] == 9.0).all()  # rows with pos < 0 are left as they were


@pytest.mark.parametrize("t", ["int8", "e4m3"])
@pytest.mark.parametrize("form,chunk", [("warp", 128), ("warp", 512), ("tc", 128), ("tc", 512), ("wide", 128), ("wide", 512)])
@pytest.mark.parametrize("G,hd", [(1, 128), (4, 128), (2, 64), (3, 256), (6, 128)])
def test_rows_do_not_depend_on_the_rows_beside_them(t, G, hd, form, chunk):
    """A verify block's rows equal single-token calls bit for bit, with later rows' keys (masked for
    the earlier ones) NaN, infinite or huge; paged equals contiguous."""
    from dflash_b200 import ops
    lens, rows, Hkv = [700, 77], 16, 2
    flat, paged = Cache(t, lens, Hkv, hd, 0, seed=3), Cache(t, lens, Hkv, hd, 64, seed=3)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2 * rows, Hkv * G, hd, generator=g).bfloat16().to(DEV)
    seq = torch.arange(2, dtype=torch.int32, device=DEV).repeat_interleave(rows)
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32, device=DEV)
    kw = dict(causal=True, max_kv=700, form=form, key_chunk=chunk)
    full = ops.attention_q8(q, flat.kv, pos, row_seq=seq, seq_rows=rows, **kw)
    assert torch.equal(full, ops.attention_q8(q, paged.kv, pos, row_seq=seq, seq_rows=rows, **kw))
    assert torch.equal(full, ops.attention_q8(q, flat.kv, pos, row_seq=seq, **kw))  # any layout
    for b in range(2):
        one = ops.attention_q8(q[b * rows:b * rows + 5].contiguous(), flat.kv, pos[b * rows:b * rows + 5],
                               row_seq=seq[b * rows:b * rows + 5], seq_rows=1, **kw)
        assert torch.equal(one, full[b * rows:b * rows + 5])
    # later rows' keys and values poisoned: earlier rows keep their bits
    for bad in (math.nan, math.inf, 1e30):
        for b, n in enumerate(lens):
            flat.scale[:, b, :, n - 6:n] = bad
        got = ops.attention_q8(q, flat.kv, pos, row_seq=seq, seq_rows=rows, **kw)
        for b in range(2):
            assert torch.equal(got[b * rows:b * rows + 10], full[b * rows:b * rows + 10])
        if bad != 1e30:  # and the rows that see them say so
            assert got[10:16].isnan().all()
    assert ops.device_error() == 0


@pytest.mark.parametrize("form,chunk", [("warp", 128), ("warp", 512), ("tc", 128), ("tc", 512), ("wide", 128), ("wide", 512)])
def test_rows_without_keys_are_zero_and_empty_calls_do_nothing(form, chunk):
    from dflash_b200 import ops
    c = Cache("int8", [40, 40, 40], 2, 128)
    q = torch.randn(3, 4, 128).bfloat16().to(DEV)
    seq = torch.arange(3, dtype=torch.int32, device=DEV)
    pos = torch.tensor([0, 5, -1], dtype=torch.int32, device=DEV)
    kv_len = torch.tensor([40, 0, 40], dtype=torch.int32, device=DEV)
    for max_kv in (40, 1000):  # one chunk, several
        c2 = c if max_kv == 40 else Cache("int8", [40, 40, 1000], 2, 128)
        out = torch.full((3, 512), 5.0, dtype=torch.bfloat16, device=DEV)
        ops.attention_q8(q, c2.kv, pos, False, max_kv, kv_len=kv_len, row_seq=seq, seq_rows=1, out=out, form=form, key_chunk=chunk)
        assert (out[1] == 0).all() and (out[2] == 5).all() and out[0].isfinite().all() and (out[0] != 5).any()
    assert ops.attention_q8(q[:0], c.kv, pos[:0], True, 40).shape == (0, 512)
    assert ops.kv_read_q8(c.kv, pos[:0])[0].shape == (0, 2, 128)
    assert ops.device_error() == 0


@pytest.mark.parametrize("form,chunk", [("warp", 128), ("warp", 512), ("tc", 128), ("tc", 512), ("wide", 128), ("wide", 512)])
def test_scales_and_queries_of_extreme_size(form, chunk):
    """Values far from 1 keep their relative precision; a softmax scale of 0 averages the values."""
    from dflash_b200 import ops
    for ks, vs, qs in ((1e-20, 1e-20, 1e15), (1e12, 1e25, 1e-12), (1.0, 1e-30, 1.0)):
        c = Cache("int8", [200], 2, 128, seed=9)
        c.scale[0] *= ks
        c.scale[1] *= vs
        val = torch.stack([c.val[0] * ks, c.val[1] * vs])
        q = (torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(2)) * qs).bfloat16()
        pos = torch.tensor([196, 197, 198, 199], dtype=torch.int32)
        sc = 128 ** -0.5 / (ks * qs)
        out = ops.attention_q8(q.to(DEV), c.kv, pos.to(DEV), True, 200, form=form, key_chunk=chunk, scale=sc)
        ref, tol = _attention64(val, q, pos + 1, torch.zeros(4), sc)
        assert ((out.double().cpu() - ref).abs() <= tol).all()
        out = ops.attention_q8(q.to(DEV), c.kv, pos.to(DEV), True, 200, form=form, key_chunk=chunk, scale=0.0)
        ref, tol = _attention64(val, q, pos + 1, torch.zeros(4), 0.0)
        assert ((out.double().cpu() - ref).abs() <= tol).all()
        neg = ops.attention_q8((-q).to(DEV), c.kv, pos.to(DEV), True, 200, form=form, key_chunk=chunk, scale=-sc)
        assert torch.equal(neg, ops.attention_q8(q.to(DEV), c.kv, pos.to(DEV), True, 200, form=form, key_chunk=chunk, scale=sc))


def _append64(qkv, pos, qn, kn, inv, Hq, Hkv, hd, rot, qs, eps):
    x = qkv.double()
    M = x.shape[0]
    q = x[:, :Hq * qs].reshape(M, Hq, qs)[..., :hd] if Hq else x.new_zeros(M, 0, hd)
    k = x[:, Hq * qs:Hq * qs + Hkv * hd].reshape(M, Hkv, hd)
    v = x[:, Hq * qs + Hkv * hd:Hq * qs + 2 * Hkv * hd].reshape(M, Hkv, hd)
    out = []
    for y, w in ((q, qn), (k, kn)):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
        ang = pos.double()[:, None] * inv.double()
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        out.append(torch.cat([a * c - b * s, b * c + a * s, y[..., rot:]], -1))
    return out[0], out[1], v


@pytest.mark.parametrize("t", ["int8", "e4m3"])
@pytest.mark.parametrize("M,Hq,Hkv,hd,rot,gated,page,do_q", [
    (1, 1, 1, 64, 64, False, 0, True), (16, 32, 8, 128, 128, False, 64, True), (7, 24, 4, 256, 64, True, 0, True),
    (33, 0, 3, 128, 128, False, 128, False), (5, 3, 2, 64, 16, False, 64, True), (130, 5, 1, 256, 256, False, 64, True),
    (400, 32, 8, 128, 128, False, 64, True), (3, 4, 2, 128, 0, False, 0, True), (600, 6, 2, 64, 32, True, 0, True),
])
def test_append_matches_64_bits_and_reads_back(t, M, Hq, Hkv, hd, rot, gated, page, do_q):
    from dflash_b200 import ops
    g = torch.Generator().manual_seed(M)
    qs = 2 * hd if gated else hd
    qkv = torch.randn(M, Hq * qs + 2 * Hkv * hd + 8, generator=g).bfloat16()
    qkv[0, -8 - hd:-8] = 0  # a value row of zeros
    qn, kn = [(1 + 0.2 * torch.randn(hd, generator=g)).bfloat16() for _ in range(2)]
    inv = (1e6 ** (-torch.arange(0, max(rot, 2), 2, dtype=torch.float64) / max(rot, 2))).float()
    cap = 131072 if page == 64 and M == 16 else 1024
    pos = torch.randperm(cap - 100, generator=g)[:M].to(torch.int32)
    seq = torch.randint(0, 3, (M,), generator=g).to(torch.int32)
    if M > 4:
        pos[2] = -1
    n_pages = 3 * cap // page if page else 3
    shape = (n_pages, Hkv, page) if page else (3, Hkv, cap)
    table = torch.randperm(n_pages, generator=g).to(torch.int32).view(3, -1).to(DEV) if page else None
    codes = torch.full((2, *shape, hd), 0x55, dtype=torch.uint8, device=DEV).view(TYPES[t])
    scale = torch.full((2, *shape), 77.0, device=DEV)
    kv = ops.QuantKV(codes[0], codes[1], scale[0], scale[1], page_table=table, page_size=page)
    q = torch.full((M, Hq, hd), 9.0, dtype=torch.bfloat16, device=DEV) if do_q else None
    d = lambda x: x.to(DEV)  # noqa: E731
    ops.qkv_rope_append_q8(d(qkv), d(pos), d(qn), d(kn), d(inv), kv, Hq, rot, 1e-6, q_out=q, row_seq=d(seq),
                           q_stride=qs, do_q=do_q)
    k, v = ops.kv_read_q8(kv, d(pos), row_seq=d(seq))
    assert ops.device_error() == 0
    live = pos >= 0
    rq, rk, rv = _append64(qkv[:, :Hq * qs + 2 * Hkv * hd], pos, qn, kn, inv[:rot // 2], Hq, Hkv, hd, rot, qs, 1e-6)
    if do_q:
        err = (q.double().cpu() - rq).abs()[live]
        assert (err <= 2.0 ** -8 * rq.abs()[live] + 2.0 ** -18 * rq.abs().amax(-1, keepdim=True)[live]).all()
        assert (q.cpu()[~live] == 9).all()
    if page:
        at = table.cpu()[seq.long(), (pos // page).clamp_min(0).long()].long(), (pos % page).long()
    else:
        at = seq.long(), pos.long().clamp_min(0)
    for i, (ref, back) in enumerate(((rk, k), (rv, v))):
        s = scale[i].cpu()[at[0], :, at[1]].double()
        amax = ref.abs().amax(-1)
        assert ((s - amax / TOP[t]).abs()[live] <= 2.0 ** -18 * (amax / TOP[t])[live]).all()
        held = codes[i].cpu().view(torch.uint8)[at[0], :, at[1]].view(TYPES[t]).double() * s[..., None]
        half = 0.5 * s[..., None] if t == "int8" else 2.0 ** -4 * ref.abs() + 2.0 ** -10 * s[..., None]
        assert ((held - ref).abs() <= half + 2.0 ** -18 * amax[..., None])[live].all()
        # read-back: the held value rounded once
        f32 = codes[i].cpu().view(torch.uint8)[at[0], :, at[1]].view(TYPES[t]).float() * s.float()[..., None]
        assert torch.equal(back.cpu()[live], f32.bfloat16()[live])
    # nothing but the rows named was written
    touched = torch.zeros(shape, dtype=torch.bool)
    touched[at[0][live], :, at[1][live]] = True
    assert (scale.cpu()[:, ~touched] == 77).all()
    assert (codes.cpu().view(torch.uint8)[:, ~touched] == 0x55).all()


def test_rows_that_hold_infinities_or_nans_are_held_as_nan():
    from dflash_b200 import ops
    for t in TYPES:
        codes = torch.zeros((2, 1, 2, 64, 128), dtype=torch.uint8, device=DEV).view(TYPES[t])
        scale = torch.zeros((2, 1, 2, 64), device=DEV)
        kv = ops.QuantKV(codes[0], codes[1], scale[0], scale[1])
        qkv = torch.randn(3, 6 * 128).bfloat16()
        qkv[0, 4 * 128 + 5] = math.inf   # value head 0 of row 0
        qkv[1, 5 * 128 + 7] = math.nan   # value head 1 of row 1
        qkv[2, 4 * 128 + 5] = -math.inf
        w = torch.ones(128).bfloat16().to(DEV)
        ops.qkv_rope_append_q8(qkv.to(DEV), torch.arange(3, dtype=torch.int32, device=DEV), w, w,
                               torch.ones(64, device=DEV), kv, 2, 128, 1e-6)
        bad = scale[1, 0, :, :3].isnan().cpu()
        assert bad.tolist() == [[True, False, True], [False, True, False]]
        assert (codes[1, 0].view(torch.uint8).cpu()[:, :3][bad] == 0).all()
        k, v = ops.kv_read_q8(kv, torch.arange(3, dtype=torch.int32, device=DEV))
        assert v[0, 0].isnan().all() and v[0, 1].isfinite().all() and k.isfinite().all()


@pytest.mark.parametrize("form,chunk", [("warp", 128), ("warp", 512), ("tc", 128), ("tc", 512), ("wide", 128), ("wide", 512)])
@pytest.mark.parametrize("page", [0, 64])
def test_out_of_range_rows_are_refused_on_the_device(page, form, chunk):
    """Positions, sequences and pages out of range are not accessed and set the error word; the other
    rows of the call are served."""
    from dflash_b200 import ops
    c = Cache("int8", [100, 100], 2, 128, page, slack=28)
    cap = c.kv.cap
    q = torch.randn(2, 4, 128).bfloat16().to(DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    assert ops.device_error() == 0
    good = ops.attention_q8(q, c.kv, i32(50, 60), True, 100, form=form, key_chunk=chunk, row_seq=i32(0, 1), seq_rows=1)
    out = torch.zeros_like(good)
    ops.attention_q8(q, c.kv, i32(50, 60), True, 100, form=form, key_chunk=chunk, row_seq=i32(0, 2), seq_rows=1, out=out)  # no sequence 2
    assert ops.device_error() == 340 and torch.equal(out[0], good[0]) and (out[1] == 0).all()
    ops.attention_q8(q, c.kv, i32(50, 60), True, 100, form=form, key_chunk=chunk, row_seq=i32(0, 1), seq_rows=2, out=out)  # two in one run
    assert ops.device_error() == 340 and torch.equal(out[0], good[0]) and (out[1] == 0).all()
    ops.attention_q8(q, c.kv, i32(50, 1 << 30), True, 100, form=form, key_chunk=chunk, row_seq=i32(0, 1), seq_rows=1, out=out)
    assert ops.device_error() == 341 and torch.equal(out[0], good[0])
    before = c.codes.view(torch.uint8).clone()
    qkv = torch.randn(2, 8 * 128).bfloat16().to(DEV)
    w = torch.ones(128).bfloat16().to(DEV)
    for pos, seq, code in ((i32(cap, cap + 5), i32(0, 1), 341), (i32(3, 4), i32(-1, 2), 340)):
        ops.qkv_rope_append_q8(qkv, pos, w, w, torch.ones(64, device=DEV), c.kv, 4, 128, 1e-6, row_seq=seq)
        assert ops.device_error() == code
        ops.kv_read_q8(c.kv, pos, row_seq=seq)
        assert ops.device_error() == code
    if page:  # a table entry that is no page (the tables' last column holds -7)
        pos = i32(cap - 1, cap - 2)
        ops.qkv_rope_append_q8(qkv, pos, w, w, torch.ones(64, device=DEV), c.kv, 4, 128, 1e-6, row_seq=i32(0, 1))
        assert ops.device_error() == 342
        ops.attention_q8(q, c.kv, pos, True, cap, row_seq=i32(0, 1), seq_rows=1, form=form, key_chunk=chunk)
        assert ops.device_error() == 342
    assert torch.equal(before, c.codes.view(torch.uint8))


@pytest.mark.parametrize("form,chunk", [("warp", 128), ("warp", 512), ("tc", 128), ("tc", 512), ("wide", 128), ("wide", 512)])
def test_views_streams_and_graphs(form, chunk):
    """Strided caches (one layer of a [seq, layer, ...] pool), strided outputs and gates, another
    stream, and two captured graphs replayed out of order."""
    from dflash_b200 import ops
    g = torch.Generator().manual_seed(4)
    B, L, Hkv, cap, hd, G = 3, 2, 2, 700, 128, 4
    x = torch.randn((2, B, L, Hkv, cap, hd), generator=g)
    codes, scale = _quantise(x, "int8")
    val = codes.double() * scale.double()[..., None]
    codes, scale = codes.to(DEV), scale.to(DEV)
    kvs = [ops.QuantKV(codes[0][:, l], codes[1][:, l], scale[0][:, l], scale[1][:, l]) for l in range(L)]
    M, Hq = B * 2, Hkv * G
    q = torch.randn(M, Hq, hd, generator=g).bfloat16()
    qkvg = torch.randn(M, 2 * Hq * hd, generator=g).bfloat16()
    pos = torch.tensor([699, 698, 10, 11, 300, 301], dtype=torch.int32)
    seq = torch.arange(B, dtype=torch.int32).repeat_interleave(2)
    gate = qkvg.view(M, Hq, 2, hd)[:, :, 1].reshape(M, Hq * hd)
    dq, dg, dp, ds = q.to(DEV), qkvg.to(DEV), pos.to(DEV), seq.to(DEV)
    refs = [_attention64(val[:, :, l], q, pos + 1, seq, hd ** -0.5, gate) for l in range(L)]
    outs = [torch.zeros(M, Hq * hd + 4, dtype=torch.bfloat16, device=DEV) for _ in range(L)]

    def call(l):
        ops.attention_q8(dq, kvs[l], dp, True, cap, row_seq=ds, seq_rows=2, form=form, key_chunk=chunk, out=outs[l][:, :Hq * hd],
                         gate=dg[:, hd:], gate_head_stride=2 * hd)

    def check():
        for l, (ref, tol) in enumerate(refs):
            assert ((outs[l][:, :Hq * hd].double().cpu() - ref).abs() <= tol).all()
            assert (outs[l][:, Hq * hd:] == 0).all()
            outs[l].zero_()

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        call(0)
        call(1)
    s.synchronize()
    check()
    graphs = []
    for l in range(L):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(l)
        graphs.append(gr)
    for _ in range(3):  # side by side on two streams: no scratch is shared
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        check()


@pytest.mark.parametrize("form,chunk", [("warp", 128), ("warp", 512), ("tc", 512), ("wide", 512)])
@pytest.mark.parametrize("B,rows,Hkv,G,hd,causal", [
    (60, 3, 4, 4, 128, True), (60, 1, 4, 2, 64, False), (45, 16, 4, 3, 256, True), (255, 1, 1, 8, 128, True),
    (256, 2, 1, 8, 128, False), (300, 2, 1, 4, 64, True)])
def test_order_of_runs_changes_nothing(B, rows, Hkv, G, hd, causal, form, chunk):
    """Calls of many runs start the longest first; the answer is that of one call a run, bit for bit."""
    from dflash_b200 import ops
    g = torch.Generator().manual_seed(B)
    lens = [int(x) for x in torch.randint(rows, 600, (B,), generator=g)]
    lens[3] = lens[4] = lens[5]  # ties
    c = Cache("int8", lens, Hkv, hd, 64, seed=B)
    q = torch.randn(B * rows, Hkv * G, hd, generator=g).bfloat16().to(DEV)
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32)
    pos[7 * rows:8 * rows] = -1
    pos[9 * rows + rows - 1] = -1
    pos, kv_len = pos.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    seq = torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(rows)

    def call(a, b):
        out = torch.full((b - a, Hkv * G * hd), 9.0, dtype=torch.bfloat16, device=DEV)
        return ops.attention_q8(q[a:b], c.kv, pos[a:b], causal, 640, kv_len=kv_len, row_seq=seq[a:b], seq_rows=rows,
                                form=form, key_chunk=chunk, out=out)

    whole = call(0, B * rows)
    parts = torch.cat([call(b * rows, (b + 1) * rows) for b in range(B)])
    assert ops.device_error() == 0
    assert torch.equal(whole, parts)
    assert (whole[7 * rows:8 * rows] == 9).all() and whole.isfinite().all()


@pytest.mark.parametrize("t", ["int8", "e4m3"])
@pytest.mark.parametrize("M,Hq,Hkv,hd,rot,do_q", [
    (700, 6, 3, 128, 128, True), (2501, 3, 2, 64, 32, True), (701, 3, 2, 64, 16, False), (2402, 5, 1, 256, 64, True)])
def test_append_of_many_rows_is_that_of_few(t, M, Hq, Hkv, hd, rot, do_q):
    from dflash_b200 import ops
    g = torch.Generator().manual_seed(M)
    qkv = torch.randn(M, (Hq + 2 * Hkv) * hd, generator=g).bfloat16().to(DEV)
    qn, kn = [(1 + 0.2 * torch.randn(hd, generator=g)).bfloat16().to(DEV) for _ in range(2)]
    inv = torch.rand(rot // 2, generator=g).to(DEV)
    pos = torch.randperm(M + 40, generator=g)[:M].to(torch.int32)
    pos[5] = pos[M - 1] = -1
    pos = pos.to(DEV)
    got = []
    for step in (M, 11):
        codes = torch.full((2, 1, Hkv, M + 40, hd), 0x55, dtype=torch.uint8, device=DEV).view(TYPES[t])
        scale = torch.full((2, 1, Hkv, M + 40), 77.0, device=DEV)
        kv = ops.QuantKV(codes[0], codes[1], scale[0], scale[1])
        q = torch.full((M, Hq, hd), 9.0, dtype=torch.bfloat16, device=DEV)
        for i in range(0, M, step):
            j = min(i + step, M)
            ops.qkv_rope_append_q8(qkv[i:j], pos[i:j], qn, kn, inv, kv, Hq, rot, 1e-6,
                                   q_out=q[i:j] if do_q else None, do_q=do_q)
        got.append((codes.view(torch.uint8), scale, q))
    assert ops.device_error() == 0
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("t", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,rows,Hkv,G,hd,causal,gated", [
    ([700, 33, 400], 8, 4, 4, 128, True, False), ([130, 517], 20, 4, 4, 128, True, True),
    ([300, 257], 9, 8, 3, 64, False, False), ([391, 64], 7, 4, 6, 256, True, True)])
def test_larger_tiles_of_the_warp_form(t, lens, rows, Hkv, G, hd, causal, gated):
    """The warp form's tiles hold 16 rows when the call is small and 32 or 64 when max_kv (here far
    above the lengths) makes it large: the same bits, and within the tolerance of 64 bits."""
    from dflash_b200 import ops
    c = Cache(t, lens, Hkv, hd, 64, seed=hd)
    g = torch.Generator().manual_seed(9)
    B, Hq = len(lens), Hkv * G
    q = (1.5 * torch.randn(B * rows, Hq, hd, generator=g)).bfloat16()
    seq = torch.arange(B, dtype=torch.int32).repeat_interleave(rows)
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32)
    kv_len = torch.tensor(lens, dtype=torch.int32)
    gate = torch.randn(B * rows, Hq * hd, generator=g).bfloat16() if gated else None
    d = [x if x is None else x.to(DEV) for x in (q, pos, kv_len, seq, gate)]
    got = [ops.attention_q8(d[0], c.kv, d[1], causal, max_kv, kv_len=d[2], row_seq=d[3], seq_rows=rows, form="warp",
                            key_chunk=256, gate=d[4]) for max_kv in (max(lens), 60000)]
    assert ops.device_error() == 0
    assert torch.equal(*got)
    ref, tol = _attention64(c.val, q, pos + 1 if causal else kv_len[seq.long()], seq, hd ** -0.5, gate)
    assert ((got[0].double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("form", ["warp", "tc", "wide", "auto"])
def test_last_run_may_be_short_and_outputs_may_be_views(form):
    """M no multiple of seq_rows, seq_rows above M, an output and a gate that are column slices."""
    from dflash_b200 import ops
    Hkv, G, hd = 2, 4, 128
    c = Cache("e4m3", [300, 41, 500], Hkv, hd, 64, seed=6)
    g = torch.Generator().manual_seed(6)
    M = 37  # runs of 16, 16 and 5 rows
    q = torch.randn(M, Hkv * G, hd, generator=g).bfloat16().to(DEV)
    seq = (torch.arange(M, dtype=torch.int32) // 16).to(DEV)
    pos = torch.tensor([n - 16 + i for n in (300, 41, 500) for i in range(16)][:M], dtype=torch.int32, device=DEV)
    gate = torch.randn(M, 3, Hkv * G * hd, generator=g).bfloat16().to(DEV)
    buf = torch.full((M, 2, Hkv * G * hd), 9.0, dtype=torch.bfloat16, device=DEV)
    kw = dict(causal=True, max_kv=500, form=form, key_chunk=256)
    ops.attention_q8(q, c.kv, pos, row_seq=seq, seq_rows=16, out=buf[:, 1], gate=gate[:, 2], **kw)
    assert (buf[:, 0] == 9).all()
    for a in (0, 16, 32):
        b = min(a + 16, M)
        one = ops.attention_q8(q[a:b], c.kv, pos[a:b], row_seq=seq[a:b], seq_rows=64, gate=gate[a:b, 2].contiguous(), **kw)
        if form != "auto":  # whose form may differ with the call's size
            assert torch.equal(one, buf[a:b, 1])
    ref, tol = _attention64(c.val, q.cpu(), pos.cpu() + 1, seq.cpu(), hd ** -0.5, gate[:, 2].cpu())
    assert ((buf[:, 1].double().cpu() - ref).abs() <= tol).all()
    assert ops.device_error() == 0


def test_wrappers_refuse_what_does_not_fit():
    from dflash_b200 import ops
    c = Cache("int8", [64], 2, 128)
    q, pos = torch.randn(3, 4, 128).bfloat16().to(DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    w, inv, qkv = torch.ones(128).bfloat16().to(DEV), torch.ones(64, device=DEV), torch.randn(3, 8 * 128).bfloat16().to(DEV)
    att = lambda **kw: ops.attention_q8(**{**dict(q=q, kv=c.kv, pos=pos, causal=True, max_kv=64), **kw})  # noqa: E731
    app = lambda **kw: ops.qkv_rope_append_q8(**{**dict(qkv=qkv, pos=pos, q_norm=w, k_norm=w, inv_freq=inv, kv=c.kv, Hq=4,  # noqa: E731
                                                        rot_dim=128, eps=1e-6), **kw})
    for call, kw in ((att, dict(q=q.float())), (att, dict(q=q[:, :, :64])), (att, dict(q=q.transpose(0, 1))),
                     (att, dict(pos=pos[:2])), (att, dict(pos=pos.long())), (att, dict(pos=pos.cpu())),
                     (att, dict(row_seq=pos[::2])), (att, dict(kv_len=pos[:0])), (att, dict(form="mma")),
                     (att, dict(out=torch.empty(3, 512, device=DEV))), (att, dict(gate=qkv[:2])),
                     (app, dict(qkv=qkv[:, :900])), (app, dict(qkv=qkv.float())), (app, dict(q_norm=None)),
                     (app, dict(k_norm=w[:64])), (app, dict(inv_freq=inv[:10])), (app, dict(pos=pos[:1])),
                     (app, dict(q_out=q[:2]))):
        with pytest.raises(ValueError):
            call(**kw)
    for call, kw in ((att, dict(key_chunk=100)), (att, dict(max_kv=0)), (att, dict(causal=False)),
                     (att, dict(scale=math.inf)), (app, dict(rot_dim=24)), (app, dict(q_stride=64))):
        with pytest.raises(Exception, match="dfl_"):
            call(**kw)
    assert ops.device_error() == 0


@pytest.mark.parametrize("paged", [False, True])
def test_offsets_beyond_32_bits(paged):
    """Sequences (or pages) more than 2^31 bytes apart: append, read-back and every form of the attention
    give the bits of a small cache."""
    from dflash_b200 import ops
    Hkv, G, hd, n = 2, 4, 128, 128
    far = 2 ** 31 + 4096
    buf = torch.zeros(far + 2 ** 20, dtype=torch.int8, device=DEV)
    sbuf = torch.zeros(2 ** 14, device=DEV)
    cut = lambda b, o, st, shape: torch.as_strided(b, shape, st, o)  # noqa: E731
    rows = 64 if paged else n
    shape = (2, Hkv, rows, hd)
    k, v = [cut(buf, o, (far, rows * hd, hd, 1), shape) for o in (0, 2 ** 19)]
    ks, vs = [cut(sbuf, o, (2 ** 12, rows, 1), shape[:3]) for o in (0, 2 ** 13)]
    small = [torch.zeros(shape, dtype=torch.int8, device=DEV) for _ in range(2)] + [torch.zeros(shape[:3], device=DEV) for _ in range(2)]
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV) if paged else None
    got = []
    for kv in (ops.QuantKV(k, v, ks, vs, table, 64 if paged else 0), ops.QuantKV(*small, table, 64 if paged else 0)):
        g = torch.Generator().manual_seed(8)
        seq = torch.full((n,), 0 if paged else 1, dtype=torch.int32, device=DEV)
        pos = torch.arange(n, dtype=torch.int32, device=DEV)
        qkv = torch.randn(n, (Hkv * G + 2 * Hkv) * hd, generator=g).bfloat16().to(DEV)
        w, inv = torch.ones(hd).bfloat16().to(DEV), torch.ones(hd // 2, device=DEV)
        q = ops.qkv_rope_append_q8(qkv, pos, w, w, inv, kv, Hkv * G, hd, 1e-6, row_seq=seq)
        out = [q, *ops.kv_read_q8(kv, pos, row_seq=seq)]
        for form in ("warp", "tc", "wide"):
            out.append(ops.attention_q8(q, kv, pos, True, n, row_seq=seq, seq_rows=n, form=form, key_chunk=128))
        got.append(out)
    assert ops.device_error() == 0
    assert got[0][1].abs().sum() > 0
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("form", ["warp", "tc", "wide"])
@pytest.mark.parametrize("page,causal", [(0, True), (64, False)])
def test_nan_codes_behind_the_last_key_are_not_read(form, page, causal):
    """Memory that no position of the call has reached may hold anything, e4m3's NaN codes included."""
    from dflash_b200 import ops
    lens, rows = [133, 64, 290], 7
    c = Cache("e4m3", lens, 2, 128, page, seed=12)
    g = torch.Generator().manual_seed(12)
    q = torch.randn(3 * rows, 8, 128, generator=g).bfloat16().to(DEV)
    seq = torch.arange(3, dtype=torch.int32, device=DEV).repeat_interleave(rows)
    pos = torch.tensor([n - rows + i for n in lens for i in range(rows)], dtype=torch.int32, device=DEV)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    call = lambda: ops.attention_q8(q, c.kv, pos, causal, 290, kv_len=kv_len, row_seq=seq, seq_rows=rows, form=form,  # noqa: E731
                                    key_chunk=128)
    before = call()
    raw = c.codes.view(torch.uint8)
    for b, n in enumerate(lens):
        if page:
            table = c.kv.tensors[4]
            raw[:, int(table[b, (n - 1) // page]), :, (n - 1) % page + 1:] = 0xff
        else:
            raw[:, b, :, n:] = 0x7f
    assert torch.equal(call(), before) and before.isfinite().all()
    assert ops.device_error() == 0


def test_large_calls_side_by_side_on_two_streams():
    """A prefill (all of an SM's TMEM) beside a batch of verify blocks (half of it) and single tokens."""
    from dflash_b200 import ops
    g = torch.Generator().manual_seed(13)
    calls = []
    for B, rows, n, form in ((1, 512, 1500, "wide"), (40, 16, 900, "tc"), (40, 1, 900, "warp")):
        kv = ops.QuantKV(*[torch.randint(-127, 128, (B, 4, n, 128), dtype=torch.int8, generator=g).to(DEV) for _ in range(2)],
                         *[torch.rand(B, 4, n, generator=g).div(60).to(DEV) for _ in range(2)])
        q = torch.randn(B * rows, 16, 128, generator=g).bfloat16().to(DEV)
        seq = torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(rows)
        pos = torch.arange(n - rows, n, dtype=torch.int32, device=DEV).repeat(B)
        calls.append(lambda kv=kv, q=q, seq=seq, pos=pos, rows=rows, n=n, form=form: ops.attention_q8(
            q, kv, pos, True, n, row_seq=seq, seq_rows=rows, form=form, key_chunk=512))
    alone = [f() for f in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, f in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append([f() for _ in range(3)])
        torch.cuda.synchronize()
        for a, outs in zip(alone, got):
            assert all(torch.equal(a, x) for x in outs)
    assert ops.device_error() == 0

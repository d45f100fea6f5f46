"""Measured cases of the 8-bit K/V cache operators: the append that quantises as it writes, the
attention that reads the codes, and the read-back of cache rows.

``run`` computes a case in plain torch operations (fp32, one rounding at the end) or, where
``own`` is true, through ``dflash_b200.ops``. A cache holds one byte per element and one fp32
scale per (token, kv head) for K and for V: the value held is code * scale.
"""
import math
import os
import sys

import torch

own = False
sys.path.insert(0, os.path.join(os.getcwd(), "dflash-mlx_b200"))  # the package is run in-tree

DEV = "cuda"
TYPES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def _attn(name, t, B, rows, lo, hi, Hkv=8, G=4, hd=128, page=64, causal=True, gate=False):
    return {"name": name, "op": "attention", "type": t, "B": B, "rows": rows, "lo": lo, "hi": hi, "Hkv": Hkv, "G": G,
            "hd": hd, "page": page, "causal": causal, "gate": gate}


def _append(name, t, B, rows, lo, hi, Hkv=8, G=4, hd=128, rot=128, page=64, gate=False):
    return {"name": name, "op": "append", "type": t, "B": B, "rows": rows, "lo": lo, "hi": hi, "Hkv": Hkv, "G": G,
            "hd": hd, "rot": rot, "page": page, "gate": gate}


def _read(name, t, B, lo, hi, Hkv=8, hd=128, page=64):
    return {"name": name, "op": "read", "type": t, "B": B, "lo": lo, "hi": hi, "Hkv": Hkv, "hd": hd, "page": page}


def listed():
    return [
        # one stream's plain decode step, a Qwen3-4B layer in the middle of an answer
        _attn("decode 1x1 int8", "int8", 1, 1, 1535, 1535),
        # the draft's block of 16 against its own cache (no mask inside the block), contiguous slots
        _attn("draft block 1x16 e4m3", "e4m3", 1, 16, 1037, 1037, page=0, causal=False),
        # plain decode of a batch of 64 ragged streams
        _attn("decode 64x1 e4m3", "e4m3", 64, 1, 512, 4096),
        # speculative verify of the same batch: 16 rows a stream
        _attn("verify 64x16 int8", "int8", 64, 16, 512, 4096),
        # few streams over very long contexts
        _attn("decode 4x1 long int8", "int8", 4, 1, 65501, 131055, page=128),
        # Qwen3.5 gated attention, head_dim 256, a verify block of a small batch
        _attn("verify 8x16 gated e4m3", "e4m3", 8, 16, 300, 6000, Hkv=4, G=6, hd=256, page=0, gate=True),
        # a prefill chunk of 128 rows deep in a prompt
        _attn("prefill 1x128 int8", "int8", 1, 128, 3968, 3968),
        # the append of one verify block, then its rows read back
        _append("append 1x16 int8", "int8", 1, 16, 1536, 1536),
        # the append of a batched verify block of the hybrid (partial rotation, gate between the q heads)
        _append("append 64x16 e4m3", "e4m3", 64, 16, 512, 4096, Hkv=4, G=6, hd=256, rot=64, page=0, gate=True),
        # a whole prompt's rows in one call, far positions among them
        _append("append 1x16384 int8", "int8", 1, 16384, 100001, 100001, page=128),
        # one sequence's cache read back (to hand a context on)
        _read("read 1 int8", "int8", 1, 513, 513),
        # a batch's caches read back
        _read("read 32 e4m3", "e4m3", 32, 512, 8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "read"])
    t = rng.choice(["int8", "e4m3"])
    hd = rng.choice([64, 128, 128, 256])
    Hkv, G = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 6, 8])
    B = _log(rng, 1, 64)
    page = rng.choice([0, 64, 128])
    if op == "attention":
        rows = rng.choice([1, 1, rng.randint(2, 16), 16, rng.randint(17, 128)])
        most = min(131072, int(1.2e8 / (B * Hkv * hd)), int(3e10 / (B * rows * Hkv * G * hd * 4)))
        hi = _log(rng, 1, max(2, most))
        return {k: v for k, v in _attn("", t, B, rows, rng.randint(0, hi), hi, Hkv, G, hd, page, rng.random() < 0.7,
                                       rng.random() < 0.3).items() if k != "name"}
    if op == "append":
        rows = _log(rng, 1, max(2, int(2.0e7 / (B * Hkv * (G + 2) * hd))))
        hi = _log(rng, 1, max(2, min(100000, int(2.0e8 / (B * Hkv * hd)))))
        return {k: v for k, v in _append("", t, B, rows, rng.randint(0, hi), hi, Hkv, G, hd,
                                         rng.choice([hd, hd // 2, hd // 4]), page, rng.random() < 0.3).items()
                if k != "name"}
    hi = _log(rng, 1, max(2, min(131072, int(1.2e8 / (B * Hkv * hd)))))
    return {k: v for k, v in _read("", t, B, rng.randint(0, hi), hi, Hkv, hd, page).items() if k != "name"}


def _contexts(case):
    """The streams' cached lengths before the call: spread over [lo, hi] by the golden ratio."""
    lo, hi = case["lo"], case["hi"]
    c = [lo + int((hi - lo) * ((b + 1) * 0.6180339887498949 % 1.0)) for b in range(case["B"])]
    c[-1] = hi
    return c


def _lengths(case):
    """Positions that each stream's cache holds once the call is done (one at least)."""
    return [max(1, c + case.get("rows", 0)) for c in _contexts(case)]


def _quantise(x, t):
    """fp32 [..., hd] -> codes and scale [...]: the absolute maximum of a row meets the type's largest code."""
    dtype, top = TYPES[t]
    a = x.abs().amax(-1)
    y = x * torch.where(a > 0, top / a, torch.zeros_like(a)).unsqueeze(-1)
    return (torch.round(y).to(dtype) if t == "int8" else y.to(dtype)), a / top


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    B, Hkv, hd, page = case["B"], case["Hkv"], case["hd"], case["page"]
    lens = _lengths(case)
    dtype = TYPES[case["type"]][0]
    s = {"case": case, "max_kv": max(lens)}
    if page:  # pools of pages, handed out in a scrambled order
        need = [(n + page - 1) // page for n in lens]
        order = torch.randperm(sum(need), device=DEV, generator=g).to(torch.int32)
        table = torch.zeros((B, max(need)), dtype=torch.int32, device=DEV)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        shape = (sum(need), Hkv, page)
    else:
        table = None
        shape = (B, Hkv, max(lens))
    s["table"] = table
    for name in ("k", "v"):
        if case["op"] == "append":  # an empty cache
            s[name] = torch.zeros((*shape, hd), dtype=torch.uint8, device=DEV).view(dtype)
            s[name + "_scale"] = torch.zeros(shape, dtype=torch.float32, device=DEV)
        else:
            x = torch.randn((*shape, hd), device=DEV, generator=g)
            if name == "k":  # a few channels carry most of a key's magnitude
                x[..., :: max(1, hd // 4)] *= 4
            x *= 1 + torch.rand((*shape, 1), device=DEV, generator=g)
            s[name], s[name + "_scale"] = _quantise(x, case["type"])
            del x
    rows = case.get("rows", 0)
    ctx = _contexts(case)
    if case["op"] == "read":
        pos = [torch.arange(n, dtype=torch.int32) for n in lens]
        seq = torch.cat([torch.full_like(p, b) for b, p in enumerate(pos)])
        pos = torch.cat(pos)
    else:
        pos = (torch.tensor(ctx)[:, None] + torch.arange(rows)[None]).reshape(-1).to(torch.int32)
        seq = torch.arange(B, dtype=torch.int32).repeat_interleave(rows)
    s["pos"], s["seq"] = pos.to(DEV), seq.to(DEV)
    s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if case["op"] != "read":
        M, Hq = B * rows, Hkv * case["G"]
        if case["op"] == "attention":
            s["q"] = (1.5 * torch.randn((M, Hq, hd), device=DEV, generator=g)).bfloat16()
            s["gate"] = torch.randn((M, Hq * hd), device=DEV, generator=g).bfloat16() if case["gate"] else None
        else:
            qs = 2 * hd if case["gate"] else hd
            s["qkv"] = torch.randn((M, Hq * qs + 2 * Hkv * hd), device=DEV, generator=g).bfloat16()
            s["q_norm"] = (1 + 0.2 * torch.randn(hd, device=DEV, generator=g)).bfloat16()
            s["k_norm"] = (1 + 0.2 * torch.randn(hd, device=DEV, generator=g)).bfloat16()
            rot = case["rot"]
            s["inv_freq"] = (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)).float()
    if own:  # the cache handle that a session keeps
        from dflash_b200 import ops
        s["kv"] = ops.QuantKV(s["k"], s["v"], s["k_scale"], s["v_scale"], page_table=table, page_size=page)
    return s


def _place(s, seq, pos):
    """(page or sequence, row in it) of cache positions."""
    page = s["case"]["page"]
    if not page:
        return seq.long(), pos.long()
    return s["table"][seq.long(), (pos // page).long()].long(), (pos % page).long()


def _values(s, name, n):
    """fp32 values of positions [0, n) of every stream: [B, Hkv, n, hd]."""
    B = s["case"]["B"]
    seq = torch.arange(B, device=DEV)[:, None].expand(B, n)
    page = s["case"]["page"]
    if not page:
        return s[name][:, :, :n].float() * s[name + "_scale"][:, :, :n, None]
    pages = s["table"].long()
    x = s[name][pages].float() * s[name + "_scale"][pages][..., None]  # [B, P, Hkv, page, hd]
    return x.transpose(1, 2).flatten(2, 3)[:, :, :n]


def _attention(s):
    c = s["case"]
    B, T, Hkv, G, hd, n = c["B"], c["rows"], c["Hkv"], c["G"], c["hd"], s["max_kv"]
    q = s["q"].float().view(B, T, Hkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, hd)
    x = q @ _values(s, "k", n).transpose(2, 3) * hd ** -0.5
    lim = (s["pos"] + 1).view(B, T) if c["causal"] else s["kv_len"][:, None].expand(B, T)
    hidden = torch.arange(n, device=DEV) >= lim.repeat_interleave(G, 1)[:, None, :, None]
    x = x.masked_fill_(hidden, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = (p @ _values(s, "v", n)) / p.sum(-1, keepdim=True)
    o = o.view(B, Hkv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(B * T, Hkv * G * hd)
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return o.bfloat16()


def _head_norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()


def _rotate(x, pos, inv_freq):
    r = 2 * inv_freq.numel()
    ang = pos.double()[:, None] * inv_freq.double()
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    a, b = x[..., :r // 2], x[..., r // 2:r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)


def _rows_back(s):
    page, row = _place(s, s["seq"], s["pos"])
    return [(s[n][page, :, row].float() * s[n + "_scale"][page, :, row][..., None]).bfloat16() for n in ("k", "v")]


def _append_rows(s):
    c = s["case"]
    M, Hq, Hkv, hd = s["pos"].numel(), c["Hkv"] * c["G"], c["Hkv"], c["hd"]
    qs = 2 * hd if c["gate"] else hd
    x = s["qkv"].float()
    q = _rotate(_head_norm(x[:, :Hq * qs].view(M, Hq, qs)[..., :hd], s["q_norm"]), s["pos"], s["inv_freq"])
    k = _rotate(_head_norm(x[:, Hq * qs:Hq * qs + Hkv * hd].view(M, Hkv, hd), s["k_norm"]), s["pos"], s["inv_freq"])
    v = x[:, Hq * qs + Hkv * hd:].view(M, Hkv, hd)
    page, row = _place(s, s["seq"], s["pos"])
    for name, y in (("k", k), ("v", v)):
        codes, scale = _quantise(y, c["type"])
        s[name].view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
        s[name + "_scale"][page, :, row] = scale
    return q.bfloat16()


def run(s):
    c = s["case"]
    if own:
        from dflash_b200 import ops
        kv, seq = s["kv"], s["seq"] if c["B"] > 1 else None
        if c["op"] == "attention":
            return ops.attention_q8(s["q"], kv, s["pos"], c["causal"], s["max_kv"], kv_len=s["kv_len"], row_seq=seq,
                                    seq_rows=c["rows"], gate=s["gate"])
        if c["op"] == "read":
            return ops.kv_read_q8(kv, s["pos"], row_seq=seq)
        q = ops.qkv_rope_append_q8(s["qkv"], s["pos"], s["q_norm"], s["k_norm"], s["inv_freq"], kv,
                                   c["Hkv"] * c["G"], c["rot"], 1e-6, row_seq=seq,
                                   q_stride=2 * c["hd"] if c["gate"] else c["hd"])
        return [q, *ops.kv_read_q8(kv, s["pos"], row_seq=seq), s["k_scale"], s["v_scale"]]
    if c["op"] == "attention":
        return _attention(s)
    if c["op"] == "read":
        return _rows_back(s)
    return [_append_rows(s), *_rows_back(s), s["k_scale"], s["v_scale"]]


def work(case):
    hd, Hkv = case["hd"], case["Hkv"]
    token = Hkv * 2 * (hd + 4)  # codes and scales of one position, K and V
    ctx, lens = _contexts(case), _lengths(case)
    if case["op"] == "read":
        return {"bytes": sum(lens) * (token + Hkv * 2 * hd * 2), "flops": sum(lens) * Hkv * 2 * hd}
    M, Hq, rows = case["B"] * case["rows"], Hkv * case["G"], case["rows"]
    if case["op"] == "append":  # projection rows in; q, codes and scales out; the codes back as bf16
        values = M * (Hq + 2 * Hkv) * hd
        return {"bytes": values * 2 + M * Hq * hd * 2 + 2 * M * token + M * Hkv * 2 * hd * 2, "flops": values * 12}
    pairs = sum(rows * c + rows * (rows + 1) // 2 for c in ctx) if case["causal"] else sum(n * rows for n in lens)
    io = M * Hq * hd * 2 * (3 if case["gate"] else 2)
    return {"bytes": sum(lens) * token + io, "flops": pairs * Hq * hd * 4}


def exact(case, seed):
    s = prepare(case, seed)
    B, Hkv, hd, page, lens = case["B"], case["Hkv"], case["hd"], case["page"], _lengths(case)
    top = {"int8": 127.0, "e4m3": 448.0}[case["type"]]

    def held(name, b, n):  # the values that the first n positions of stream b hold, [n, Hkv, hd]
        if page:
            ids = [int(i) for i in s["table"][b, :(n + page - 1) // page]]
            codes = torch.cat([s[name][i].transpose(0, 1) for i in ids])[:n]
            scale = torch.cat([s[name + "_scale"][i].transpose(0, 1) for i in ids])[:n]
        else:
            codes, scale = s[name][b, :, :n].transpose(0, 1), s[name + "_scale"][b, :, :n].transpose(0, 1)
        return codes.double() * scale.double().unsqueeze(-1)

    if case["op"] == "read":
        return [torch.cat([held(n, b, lens[b]) for b in range(B)]) for n in ("k", "v")]
    T, G = case["rows"], case["G"]
    M, Hq = B * T, Hkv * G
    if case["op"] == "attention":
        out = torch.empty((M, Hkv, G, hd), dtype=torch.float64, device=DEV)
        for b in range(B):
            k, v = held("k", b, lens[b]), held("v", b, lens[b])
            q = s["q"][b * T:(b + 1) * T].double().view(T, Hkv, G, hd)
            x = torch.einsum("thgd,nhd->thgn", q, k) / math.sqrt(hd)
            if case["causal"]:
                seen = torch.arange(lens[b], device=DEV) <= s["pos"][b * T:(b + 1) * T, None]
                x = torch.where(seen[:, None, None], x, -math.inf)
            out[b * T:(b + 1) * T] = torch.einsum("thgn,nhd->thgd", torch.softmax(x, -1), v)
        out = out.view(M, Hq * hd)
        return out * torch.sigmoid(s["gate"].double()) if case["gate"] else out
    rows, qs = s["qkv"].double(), 2 * hd if case["gate"] else hd
    heads = [rows[:, h * qs:h * qs + hd] for h in range(Hq)]
    heads += [rows[:, Hq * qs + h * hd:Hq * qs + (h + 1) * hd] for h in range(2 * Hkv)]
    x = torch.stack(heads, 1)
    qk = x[:, :Hq + Hkv]
    w = torch.cat([s["q_norm"].double().expand(Hq, hd), s["k_norm"].double().expand(Hkv, hd)])
    qk = qk / torch.sqrt(qk.pow(2).mean(-1, keepdim=True) + 1e-6) * w
    half = case["rot"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.outer(s["pos"].double(), s["inv_freq"].double()))
    z = torch.complex(qk[..., :half], qk[..., half:2 * half]) * turn[:, None]
    qk = torch.cat([z.real, z.imag, qk[..., 2 * half:]], -1)
    back, scales = [], []
    at = s["seq"].long(), s["pos"].long()
    if page:
        at = s["table"][at[0], at[1] // page].long(), at[1] % page
    for name, y in (("k", qk[:, Hq:]), ("v", x[:, Hq + Hkv:])):
        scale = y.abs().amax(-1) / top
        z = y / scale.clamp_min(1e-300).unsqueeze(-1)
        z = torch.round(z) if case["type"] == "int8" else z.float().to(torch.float8_e4m3fn).double()
        back.append(z * scale.unsqueeze(-1))
        grid = s[name + "_scale"].double()
        grid[at[0], :, at[1]] = scale
        scales.append(grid)
    return [qk[:, :Hq], *back, *scales]

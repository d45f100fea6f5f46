"""attention_q8 over V scales far apart."""
import pytest
import torch
from test_kv_q8_gpu import DEV, TOP, Cache

pytestmark = pytest.mark.gpu
FORMS = [("warp", 128), ("tc", 128), ("wide", 128)]


@pytest.fixture(scope="module", autouse=True)
def _need(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _reference(q, k, v, scale):
    """(o, tolerance) of rows that see all keys: q [M, H, hd], k, v [n, hd] in 64 bits."""
    n, hd = v.shape
    x = q.double() @ k.T * scale
    p = torch.softmax(x, -1)
    o, A = p @ v, p @ v.abs()
    smax = (q.double().abs() @ k.abs().T * abs(scale)).amax()
    # fp16's lower end: the largest weight p_j vs_j is held as 1 at least, the others as multiples of 2^-24 there:
    # off by at most 2^-25 of the largest each, times codes of at most TOP, whose product with vs_j is max |v_j|
    low = n * 2.0 ** -25 * (p * v.abs().amax(-1)).amax(-1, keepdim=True)
    # the other terms as in test_kv_q8_gpu.py: the output's bf16, the weights' fp16, scores and sums in fp32
    return o, 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2.0 ** -18 + 2 * hd * 2.0 ** -23 * smax) * A + low


def _case(t, n, hd, seed):
    c = Cache(t, [n], 1, hd, seed=seed, slack=0)
    g = torch.Generator().manual_seed(seed)
    q = (1.5 * torch.randn(4, 4, hd, generator=g)).bfloat16()
    return c, q


def _run(c, q, n, form, chunk):
    from dflash_b200 import ops
    out = ops.attention_q8(q.to(DEV), c.kv, torch.full((q.shape[0],), n - 1, dtype=torch.int32, device=DEV), True, n,
                           form=form, key_chunk=chunk)
    assert ops.device_error() == 0
    return out.double().cpu().view(*q.shape)


@pytest.mark.parametrize("form,chunk", FORMS + [("warp", 1024), ("tc", 1024), ("wide", 1024)])
@pytest.mark.parametrize("t,hd", [("int8", 128), ("e4m3", 64), ("int8", 256)])
@pytest.mark.parametrize("at", [0, 37, 600])
@pytest.mark.parametrize("shift", [24, 30, 60])
def test_a_key_of_no_weight_and_a_large_value_costs_no_bits(form, chunk, t, hd, at, shift):
    """A key that the softmax all but leaves out (below 2^-75) but whose V scale is 2^shift times the others':
    the weights are held relative to the largest product of weight and scale, not of the two maxima."""
    n = 700
    c, q = _case(t, n, hd, 21)
    q = q.abs().clamp_min(0.5)  # every query points one way, the key the other
    c.codes[0, 0, 0, at] = torch.full((hd,), -TOP[t]).to(c.codes.dtype).to(DEV)
    c.scale[0, 0, 0, at] = 5 / TOP[t]
    c.val[0, 0, 0, at] = -TOP[t] * float(c.scale[0, 0, 0, at])
    c.scale[1, 0, 0, at] *= 2.0 ** shift
    c.val[1, 0, 0, at] *= 2.0 ** shift
    k, v = c.val[0, 0, 0, :n], c.val[1, 0, 0, :n]
    scale = hd ** -0.5
    p = torch.softmax(q.double() @ k.T * scale, -1)
    assert float(p[..., at].max()) * 2.0 ** shift < 2.0 ** -10 * float(p.max())  # what it adds is small
    o, tol = _reference(q, k, v, scale)
    err = (_run(c, q, n, form, chunk) - o).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("form,chunk", FORMS + [("warp", 1024), ("tc", 1024), ("wide", 1024)])
@pytest.mark.parametrize("t,hd", [("int8", 128), ("e4m3", 64), ("e4m3", 256)])
@pytest.mark.parametrize("exps", [(-90, 0), (0, -90), (0, 80), (-60, 70), (70, -60), (-90, 80), (80, -90)])
def test_v_scales_far_apart_leave_the_softmax_sum_whole(form, chunk, t, hd, exps):
    """Halves of the keys whose V scales lie 2^80 to 2^170 apart: the small half adds nothing to the output but its
    softmax weights still divide it."""
    n = 512
    c, q = _case(t, n, hd, 22)
    for half, e in enumerate(exps):
        s = slice(half * n // 2, (half + 1) * n // 2)
        c.scale[1, 0, 0, s] *= 2.0 ** e
        c.val[1, 0, 0, s] *= 2.0 ** e
    o, tol = _reference(q, c.val[0, 0, 0, :n], c.val[1, 0, 0, :n], hd ** -0.5)
    err = (_run(c, q, n, form, chunk) - o).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("form,chunk", FORMS)
@pytest.mark.parametrize("qs,scale", [(1e-38, 1e-10), (2.0 ** -126, 2.0 ** -60), (1.0, 1e-44)])
def test_scores_that_vanish_average_the_keys_that_a_row_sees(form, chunk, qs, scale):
    """Queries and softmax scales so small that their product is below fp32's range: the weights are alike, and keys
    behind a row's position stay out (0 times their -inf would be NaN)."""
    from dflash_b200 import ops
    n, hd = 200, 128
    c, q = _case("int8", n, hd, 23)
    q = q.sign() * qs
    pos = torch.tensor([3, 150, 190, 199], dtype=torch.int32)
    out = ops.attention_q8(q.bfloat16().to(DEV), c.kv, pos.to(DEV), True, n, form=form, key_chunk=chunk, scale=scale)
    assert ops.device_error() == 0
    out = out.double().cpu().view(4, 4, hd)
    for m, p in enumerate(pos.tolist()):
        v = c.val[1, 0, 0, :p + 1]
        o, A = v.mean(0), v.abs().mean(0)
        # as above, with scores of 0
        tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2.0 ** -18) * A + n * 2.0 ** -25 * v.abs().amax() / (p + 1)
        assert ((out[m] - o).abs() <= tol).all(), m


@pytest.mark.parametrize("form,chunk", FORMS + [("warp", 1024), ("tc", 1024), ("wide", 1024)])
@pytest.mark.parametrize("t,hd", [("int8", 128), ("e4m3", 64), ("e4m3", 256)])
@pytest.mark.parametrize("k_to,v_to", [(2.0 ** 95, 2.0 ** 90), (2.0 ** 95, 2.0 ** -104), (2.0 ** -100, 2.0 ** 90)])
def test_scales_at_the_ends_of_the_stated_range(form, chunk, t, hd, k_to, v_to):
    from dflash_b200 import ops
    n = 700
    c, q = _case(t, n, hd, 24)
    fk = 2.0 ** torch.floor(torch.log2(torch.tensor(k_to) / c.scale[0].max())).item()
    lim = c.scale[1].max() if v_to > 1 else c.scale[1].min()
    fv = 2.0 ** (torch.floor if v_to > 1 else torch.ceil)(torch.log2(torch.tensor(v_to) / lim)).item()
    for i, f in enumerate((fk, fv)):
        c.scale[i] *= f
        c.val[i] *= f
    q = (q.double() * (1 / fk)).bfloat16()  # a power of two
    o, tol = _reference(q, c.val[0, 0, 0, :n], c.val[1, 0, 0, :n], hd ** -0.5)
    err = (_run(c, q, n, form, chunk) - o).abs()
    assert (err <= tol + 2.0 ** -134).all(), float((err / tol).max())  # half of bf16's smallest step

"""GPU tests of the sequence operators (attention over packed sequences, norm and rotation of
queries and keys, the 8-bit linear layer) against plain implementations in 64 bits.

Tolerances count roundings: u = eps / 2 of the stored type, fp32 work at 2^-24 a step.
"""

from __future__ import annotations

import ctypes
import math
from decimal import Decimal, localcontext

import pytest
import torch
from torch.autograd import forward_ad

from esmfold2_mlx_b200 import attention as att
from esmfold2_mlx_b200 import fp8, ops

pytestmark = pytest.mark.gpu

FP16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def assert_within(got, ref, tol, what=""):
    bad = ~((got.double() - ref).abs() <= tol)  # NaN counts as bad
    if bad.any():
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: "
                             f"{got[i].item()} against {ref[i].item()}, allowed {tol[i].item()}")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- attention -------------------------------------------------------------------------------

def attention_ref(q, k, v, lens, causal, scale, bias=None):
    """Output and tolerance in 64 bits.

    A row is sum p v / sum p.  Its weights are rounded to q's type (relative u, and 2^-25 absolute where
    fp16 turns subnormal, with the largest weight at 1 or above); a score is off by at most D 2^-24 of
    its absolute terms, the exponential by 2^-16, the sums by n 2^-24; the output is rounded once."""
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    u = half_step(q.dtype)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    beg = 0
    for s, n in enumerate(lens):
        if n == 0:
            continue
        r = slice(beg, beg + n)
        beg += n
        rep = hq // hkv
        qq = q[r].double().transpose(0, 1)
        kk = k[r].double().transpose(0, 1).repeat_interleave(rep, 0)
        vv = v[r].double().transpose(0, 1).repeat_interleave(rep, 0)
        x = qq @ kk.transpose(1, 2) * scale
        size = qq.abs() @ kk.abs().transpose(1, 2) * abs(scale)
        if bias is not None:
            m = min(n, bias.shape[2])
            b = bias[s if bias.shape[0] > 1 else 0][:, :m, :m].double()
            x[:, :m, :m] += b
            size[:, :m, :m] += b.nan_to_num(neginf=0.0).abs()
        if causal:
            x = x.masked_fill(torch.ones(n, n, device=q.device, dtype=torch.bool).triu(1), -math.inf)
        size = size.masked_fill(x == -math.inf, 0.0)
        mx = x.amax(-1, keepdim=True)
        mx = torch.where(mx == -math.inf, torch.zeros_like(mx), mx)
        p = (x - mx).exp()
        l = p.sum(-1, keepdim=True)
        some = l > 0
        l = torch.where(some, l, torch.ones_like(l))
        o = (p @ vv) / l
        a = (p @ vv.abs()) / l
        sub = 2.0 ** -25 * vv.abs().sum(1, keepdim=True) / l if q.dtype == FP16 else 0.0
        e = size.amax(-1, keepdim=True)
        rel = u + 2 * d * 2.0 ** -24 * e + 2.0 ** -15 + (2 * n + 8) * 2.0 ** -24
        t = u * o.abs() + a * rel + sub + least(q.dtype)
        out[r] = torch.where(some, o, torch.zeros_like(o)).transpose(0, 1)
        tol[r] = t.transpose(0, 1)
    return out, tol


def make_qkv(lens, hq, hkv, d, dtype, seed, extra=0, amp=1.5):
    t = sum(lens) + extra
    x = torch.randn(t, hq + 2 * hkv, d, generator=gen(seed), device="cuda")
    x[:, :hq] *= amp
    x = x.to(dtype)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)) if lens else [0], dtype=torch.int32, device="cuda")
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], cu


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,hq,hkv,d", [
    ([1], 1, 1, 64), ([2], 3, 1, 8), ([127], 2, 2, 64), ([128], 2, 1, 64), ([129], 2, 2, 128), ([255], 4, 2, 128),
    ([256], 1, 1, 48), ([257], 2, 2, 32), ([383], 4, 1, 120), ([640, 1, 0, 77, 130], 4, 2, 64),
    ([5, 1, 1, 300, 0, 0, 64, 2], 6, 2, 128), ([1025], 2, 1, 72), ([0, 33, 0], 2, 2, 16), ([2100], 2, 1, 64),
    ([1500, 700], 2, 2, 128), ([1] * 50, 3, 3, 40)])
def test_attention(lens, hq, hkv, d, causal, dtype):
    q, k, v, cu = make_qkv(lens, hq, hkv, d, dtype, 1)
    got = att.attention(q, k, v, cu, causal=causal)
    ref, tol = attention_ref(q, k, v, lens, causal, 1 / math.sqrt(d))
    assert_within(got, ref, tol)


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,h,d,shared", [
    ([76], 16, 48, True), ([146, 146], 4, 48, True), ([238, 100, 7], 4, 64, False), ([129], 3, 128, True),
    ([384, 384], 2, 32, False), ([513], 2, 64, True)])
def test_attention_bias(lens, h, d, shared, causal, dtype):
    q, k, v, cu = make_qkv(lens, h, h, d, dtype, 2)
    n = max(lens)
    b = 3 * torch.randn(1 if shared else len(lens), h, n, n, generator=gen(3), device="cuda")
    b[:, :, :, 3:6] = -math.inf           # hidden keys
    b[:, 0, 5, :] = -math.inf             # a row that sees nothing
    b[:, -1, 6, :] = torch.finfo(dtype).min  # a row of the type's lowest value sees all keys evenly
    b = b.to(dtype)
    got = att.attention(q, k, v, cu, causal=causal, bias=b)
    ref, tol = attention_ref(q, k, v, lens, causal, 1 / math.sqrt(d), b)
    assert_within(got, ref, tol)
    if lens[0] > 6:
        assert (got[5, 0] == 0).all()


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n,d", [(40, 64), (300, 48), (300, 128)])
def test_attention_masks_of_the_lowest_value(n, d, causal, dtype):
    """Keys masked by the type's lowest value.  The queries are 0, so a row is the mean of the keys it
    sees best: those at 0, or, where there are none, those at the lowest value (-inf hides for good).

    The weights are equal before they are rounded to q's type (u) and their exponentials off by 2^-16
    at most; the sums of v and of the weights add 2 n 2^-24, and the output is rounded once."""
    _, k, v, cu = make_qkv([n], 1, 1, d, dtype, 60)
    q = torch.zeros_like(k)
    low = torch.finfo(dtype).min
    b = torch.zeros(1, 1, n, n, device="cuda", dtype=dtype)
    b[0, 0, :, n // 2:] = low          # padding behind
    b[0, 0, 5:30, :n // 2] = low       # with that, rows of nothing but the lowest value
    b[0, 0, 20:25, ::3] = -math.inf    # with hidden keys among it
    b[0, 0, n // 2:, :] = low
    b[0, 0, n - 9:, n - 20:n - 3] = 0  # a later step's keys beat the first's
    got = att.attention(q, k, v, cu, causal=causal, bias=b)
    x = b[0, 0].double()
    if causal:
        x = x.masked_fill(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), -math.inf)
    top = x.amax(-1, keepdim=True)
    p = ((x == top) & (top > -math.inf)).double()
    p = p / p.sum(-1, keepdim=True).clamp(min=1)
    vv = v[:, 0].double()
    ref, a = p @ vv, p @ vv.abs()
    assert_within(got[:, 0], ref, half_step(dtype) * ref.abs()
                  + a * (half_step(dtype) + 2.0 ** -15 + (2 * n + 16) * 2.0 ** -24) + least(dtype))


def test_attention_bias_views():
    """A bias with odd row pitch, a shorter one than the sequence, and one broadcast over heads."""
    lens, h, d = [150, 90], 4, 64
    q, k, v, cu = make_qkv(lens, h, h, d, FP16, 4)
    big = torch.randn(3, 2, h, 157, 157, generator=gen(5), device="cuda").half()
    for b in (big[1][:, :, :151, :151], big[0][:1, :, 2:103, 1:102], big[2][:, :1, :150, :150].expand(2, h, 150, 150)):
        got = att.attention(q, k, v, cu, bias=b)
        ref, tol = attention_ref(q, k, v, lens, False, 1 / math.sqrt(d), b)
        assert_within(got, ref, tol)


def test_attention_bias_is_what_pair_cond_makes():
    """Blocks of a [nb, B, H, L, L] tensor go in as they are."""
    L, h, d, B = 77, 16, 48, 2
    q, k, v, cu = make_qkv([L] * B, h, h, d, FP16, 6)
    biases = torch.randn(3, B, h, L, L, generator=gen(7), device="cuda").half()
    for blk in biases:
        got = att.attention(q, k, v, cu, bias=blk)
        ref, tol = attention_ref(q, k, v, [L] * B, False, 1 / math.sqrt(d), blk)
        assert_within(got, ref, tol)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_ignores_other_tokens(causal, d):
    """NaN and infinities in other sequences and behind the last one reach nothing; rows of no
    sequence stay as they were."""
    for dtype in (FP16, BF16):
        lens = [130, 70, 200, 19]
        q, k, v, cu = make_qkv(lens, 4, 2, d, dtype, 8, extra=141)
        ref, tol = attention_ref(q, k, v, lens, causal, 1 / math.sqrt(d))
        for t in (q, k, v):
            t[419:] = float("nan")
            t[450:500] = float("inf")
        out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
        att.attention(q, k, v, cu, causal=causal, out=out)
        assert_within(out[:419], ref[:419], tol[:419])
        assert (out[419:] == 7.0).all()
        k[130:200] = float("inf")
        v[130:200] = float("nan")
        att.attention(q, k, v, cu, causal=causal, out=out)
        assert_within(out[:130], ref[:130], tol[:130])
        assert_within(out[200:419], ref[200:419], tol[200:419])


@pytest.mark.parametrize("d", [64, 128])
def test_attention_causal_future_scores_do_not_count(d):
    """Infinite and NaN keys and biases behind a causal row do not reach it."""
    lens = [300]
    q, k, v, cu = make_qkv(lens, 2, 2, d, FP16, 9)
    b = torch.randn(1, 2, 300, 300, generator=gen(10), device="cuda").half()
    ref, tol = attention_ref(q, k, v, lens, True, 1 / math.sqrt(d), b)
    b[:, :, :200, 200:] = float("nan")
    b[:, :, 100:150, 150:200] = float("inf")
    k[200:] = float("nan")
    got = att.attention(q, k, v, cu, causal=True, bias=b)
    assert_within(got[:150], ref[:150], tol[:150])
    assert got[200:].isnan().all()


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("d", [8, 40, 64, 128])
def test_attention_hidden_keys_do_not_count_whatever_they_hold(d, dtype):
    """NaN and infinities in k and v of keys that -inf hides (a padded batch), or that lie behind a
    causal row, reach no row that does not see them: also in a step of their own, in a row without
    keys, with shared heads, and beside another sequence."""
    lens, hq, hkv = [300, 33, 150], 4, 2
    q, k, v, cu = make_qkv(lens, hq, hkv, d, dtype, 63)
    b = torch.randn(3, hq, 300, 300, generator=gen(64), device="cuda").to(dtype)
    pads = [130, 20, 150]  # keys of each sequence that are there
    for s, n in enumerate(pads):
        b[s, :, :, n:] = -math.inf
    b[0, :, 3, :] = -math.inf
    scale = 1 / math.sqrt(d)
    for causal in (False, True):
        ref, tol = attention_ref(q, k, v, lens, causal, scale, b)
        k2, v2 = k.clone(), v.clone()
        k2[130:300:2], v2[131:300:2] = float("nan"), float("nan")
        k2[133:300:5], v2[135:300:7] = float("inf"), -float("inf")
        v2[320:333, :, ::3] = float("nan")
        got = att.attention(q, k2, v2, cu, causal=causal, bias=b)
        assert_within(got, ref, tol)
        assert (got[3] == 0).all()
    ref, tol = attention_ref(q, k, v, lens, True, scale)
    k2, v2 = k.clone(), v.clone()
    k2[200], v2[200:204] = float("nan"), float("inf")
    v2[310, 1, d - 1] = float("nan")
    got = att.attention(q, k2, v2, cu, causal=True)
    keep = torch.ones(got.shape, dtype=torch.bool, device="cuda")
    keep[200:300] = False           # these see keys 200 on
    keep[310:333, 2:, d - 1] = False  # key head 1 is query heads 2 and 3's
    assert_within(got[keep], ref[keep], tol[keep])
    assert got[200:300].isnan().all() and got[310:333, 2:, d - 1].isnan().all()


@pytest.mark.parametrize("d", [48, 64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_one_bad_score_spoils_its_row_only(bad, d):
    """A single NaN or +inf score, at every place of a step and in its first and a later one, makes its
    row NaN, as a softmax is, and no other."""
    n = 280
    q, k, v, cu = make_qkv([n], 1, 1, d, FP16, 51)
    b = torch.zeros(1, 1, n, n, device="cuda", dtype=FP16)
    rows = torch.arange(n, device="cuda")
    hit = rows[::3]
    b[0, 0, hit, (hit * 7 + 5) % n] = bad
    got = att.attention(q, k, v, cu, bias=b)
    assert got[hit].isnan().all()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[hit] = False
    ref, tol = attention_ref(q, k, v, [n], False, 1 / math.sqrt(d))
    assert_within(got[keep], ref[keep], tol[keep])
    q2 = q.clone()
    q2[hit] = bad  # the same without a bias: a row whose scores are NaN or infinite
    got = att.attention(q2, k, v, cu)
    assert got[hit].isnan().all()
    assert_within(got[keep], ref[keep], tol[keep])


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_bias_with_a_bad_value_that_rows_see(causal, d, dtype):
    """One NaN, or one infinity, in one column of one v that most rows see, under a bias that hides it from
    others: that column is what a softmax makes of it, the other columns and the rows that do not see it are
    untouched."""
    n, h, at = 1200, 4, 517
    q, k, v, cu = make_qkv([n], h, 2, d, dtype, 68)
    b = torch.randn(1, h, n, n, generator=gen(69), device="cuda").to(dtype)
    b[..., n - 50:] = -math.inf  # padding
    b[0, :, 800:900, at] = -math.inf
    ref, tol = attention_ref(q, k, v, [n], causal, 1 / math.sqrt(d), b)
    sees = torch.ones(n, dtype=torch.bool, device="cuda")
    sees[800:900] = False
    if causal:
        sees[:at] = False
    hit = torch.zeros(n, h, d, dtype=torch.bool, device="cuda")
    hit[sees, 2:, 5] = True  # key head 1 is query heads 2 and 3's
    for bad in (math.nan, math.inf, -math.inf):
        v[at, 1, 5] = bad
        got = att.attention(q, k, v, cu, causal=causal, bias=b)
        assert_within(got[~hit], ref[~hit], tol[~hit])
        seen = got[hit]
        assert (seen.isnan() | (seen == bad)).all() and (bad == bad or seen.isnan().all())


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_bias_a_bad_value_that_rows_see_costs_no_row(causal, padded):
    """A NaN in v that every row sees (key 0), beside a bias that hides other, finite keys or none, sends no
    row through its keys one by one, which takes hundreds of times as long as the call (9.4 ms for 0.04).
    What is allowed is the search for keys that could: a pass of each warp over k and v, 38 steps of 32 keys
    and two rows of loads each, under 4 us a step with everything waited for, beside the call."""
    n, h, d = 1200, 4, 64
    q, k, v, cu = make_qkv([n], h, 2, d, FP16, 70)
    b = torch.randn(1, h, n, n, generator=gen(71), device="cuda").to(FP16)
    if padded:
        b[..., n - 50:] = -math.inf
    out = att.attention(q, k, v, cu, causal=causal, bias=b)

    def timed():
        times = []
        for _ in range(5):
            a, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            att.attention(q, k, v, cu, causal=causal, bias=b, out=out)
            e.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(e))
        return min(times)

    base = timed()
    v[0, :, 5] = math.nan
    took = timed()
    assert out[:, :, 5].isnan().all()
    assert took < 2 * base + 38 * 0.004, (took, base)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-20, 3.0])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_scales(scale, d):
    lens = [200, 131]
    q, k, v, cu = make_qkv(lens, 2, 2, d, BF16, 52)
    b = torch.randn(2, 2, 200, 200, generator=gen(53), device="cuda").to(BF16)
    b[:, :, :, 7] = -math.inf
    for bias in (None, b):
        for causal in (False, True):
            got = att.attention(q, k, v, cu, scale=scale, bias=bias, causal=causal)
            assert_within(got, *attention_ref(q, k, v, lens, causal, scale, bias))


def test_attention_many_short_and_empty_sequences():
    """More sequences than one search step holds, empty ones among them."""
    g = torch.Generator().manual_seed(54)
    lens = [int(x) for x in torch.randint(0, 40, (1500,), generator=g)]
    q, k, v, cu = make_qkv(lens, 2, 1, 64, FP16, 55)
    for causal in (False, True):
        assert_within(att.attention(q, k, v, cu, causal=causal), *attention_ref(q, k, v, lens, causal, 0.125))


@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_attention_large_scores(dtype):
    """Scores whose maximum climbs from key to key by hundreds: the running maximum has to follow."""
    n, d = 700, 64
    q, k, v, cu = make_qkv([n], 2, 2, d, dtype, 11)
    k *= 0.01
    k[:, :, 0] = (torch.arange(n, device="cuda").float()[:, None] * 0.5).to(dtype)
    q[:, :, 0] = 8.0
    for sign in (1.0, -1.0):
        got = att.attention(q, k, v, cu, causal=False, scale=sign)
        ref, tol = attention_ref(q, k, v, [n], False, sign)
        assert_within(got, ref, tol)
        got = att.attention(q, k, v, cu, causal=True, scale=sign)
        ref, tol = attention_ref(q, k, v, [n], True, sign)
        assert_within(got, ref, tol)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("bits", [20, 26, 28])
@pytest.mark.parametrize("heavy", [0, 1000, 2047])
def test_attention_small_weights_add_up(heavy, bits, with_bias, d):
    """One key far above 2047 others whose values alone are not 0: the row is the sum of many weights of
    about 2^-bits.  In fp16 a weight is off by u of itself, or by 2^-25 where it is subnormal, with the row's
    largest weight at 2^7 or above; the rest as in attention_ref (a bias of its own size has one product)."""
    n, low = 2048, -bits * math.log(2)
    q, k, v, cu = make_qkv([n], 1, 1, d, FP16, 67)
    q.zero_(), k.zero_()
    v.abs_()
    v[heavy] = 0.0
    if with_bias:
        bias = torch.full((1, 1, n, n), low, dtype=FP16, device="cuda")
        bias[..., heavy] = 0.0
        x = bias[0, 0, 0].double()
    else:
        bias = None
        q[:, :, 0] = 8.0
        k[:, :, 0] = low / 8
        k[heavy] = 0.0
        x = 8.0 * k[:, 0, 0].double()
    got = att.attention(q, k, v, cu, scale=1.0, bias=bias)
    p = x.exp()
    ref = (p @ v[:, 0].double() / p.sum())[None, None].expand(n, 1, d)
    u = half_step(FP16)
    rel = u + 2 * d * 2.0 ** -24 * x.abs().max() + 2.0 ** -15 + (2 * n + 8) * 2.0 ** -24
    tol = u * ref + rel * ref + 2.0 ** -32 * v[:, 0].double().sum(0) / p.sum() + least(FP16)
    assert_within(got, ref, tol)


def test_attention_bad_cu_seqlens_stay_in_bounds():
    """Offsets outside the tokens are clamped; the good sequences are right."""
    q, k, v, _ = make_qkv([200], 2, 2, 64, FP16, 12)
    cu = torch.tensor([-5, 90, 90, 60, 1000], dtype=torch.int32, device="cuda")
    got = att.attention(q, k, v, cu)
    ref, tol = attention_ref(q[:90], k[:90], v[:90], [90], False, 0.125)
    torch.cuda.synchronize()
    assert_within(got[:60], ref[:60], tol[:60])


def test_attention_strides_out_and_empty():
    lens, hq, hkv, d = [140, 60], 4, 2, 48
    g = gen(13)
    qkv = torch.randn(hq + 2 * hkv, 200, 56, generator=g, device="cuda").half()  # heads outermost, padded rows
    q, k, v = (t.transpose(0, 1)[..., :d] for t in (qkv[:hq], qkv[hq:hq + hkv], qkv[hq + hkv:]))
    cu = torch.tensor([0, 140, 200], dtype=torch.int32, device="cuda")
    buf = torch.zeros(200, 2, hq, 64, device="cuda", dtype=FP16)
    out = buf[:, 1, :, :d]
    got = att.attention(q, k, v, cu, out=out)
    assert got.data_ptr() == out.data_ptr()
    ref, tol = attention_ref(q, k, v, lens, False, 1 / math.sqrt(d))
    assert_within(out, ref, tol)
    assert (buf[:, 0] == 0).all() and (buf[:, 1, :, d:] == 0).all()
    e = torch.empty(0, 2, 64, device="cuda", dtype=FP16)
    assert att.attention(e, e, e, cu[:1]).shape == (0, 2, 64)
    assert att.attention(e, e, e, torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 2, 64)


def test_attention_far_offsets():
    """Element offsets past 2^31."""
    d, n = 64, 300
    stride = 2 ** 23 + 8
    big = torch.empty(n * stride, device="cuda", dtype=FP16)
    small = torch.randn(3, n, 1, d, generator=gen(14), device="cuda").half()
    views = []
    for i in range(3):
        t = torch.as_strided(big, (n, 1, d), (stride, d, 1), i * 128)
        t.copy_(small[i])
        views.append(t)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out = torch.as_strided(big, (n, 1, d), (stride, d, 1), 512)
    att.attention(*views, cu, out=out)
    ref, tol = attention_ref(*small, [n], False, 0.125)
    assert_within(out, ref, tol)


# ---- norm and rotation -----------------------------------------------------------------------

def rope_ref(x, pos, rotary, norm, w, b, eps):
    """Output and tolerance in 64 bits: fp32 work of a few roundings (16 of 2^-24, plus the angle's
    2^-32 of a turn) on the values that meet, and one rounding to the stored type."""
    y = x.double()
    size = y.abs()
    if norm == "layer":
        size = size + y.mean(-1, keepdim=True).abs() + size.mean(-1, keepdim=True)
        y = y - y.mean(-1, keepdim=True)
    if norm is not None:
        r = 1.0 / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        y, size = y * r, size * r
        if w is not None:
            y, size = y * w.double(), size * w.double().abs()
        if b is not None:
            y, size = y + b.double(), size + b.double().abs()
    out = y.clone()
    if rotary is not None:
        f = torch.tensor(rotary.frequencies, dtype=torch.float64, device=x.device)
        ang = pos.double()[:, None] * f
        cos, sin = (ang.cos() * rotary.gain)[:, None], (ang.sin() * rotary.gain)[:, None]
        r = rotary.rot
        i1 = torch.arange(r // 2, device=x.device)
        i1, i2 = (i1, i1 + r // 2) if rotary.layout == "half" else (2 * i1, 2 * i1 + 1)
        out[..., i1] = y[..., i1] * cos - y[..., i2] * sin
        out[..., i2] = y[..., i2] * cos + y[..., i1] * sin
        both = (size[..., i1] + size[..., i2]) * rotary.gain
        size = size.clone()
        size[..., i1] = both
        size[..., i2] = both
    return out, half_step(x.dtype) * out.abs() + 16 * 2.0 ** -24 * size + least(x.dtype)


SCALINGS = [None, {"type": "linear", "factor": 8.0}, {"type": "ntk", "factor": 4.0},
            {"type": "yarn", "factor": 16.0, "original_length": 4096}]


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [None, "rms", "layer"])
@pytest.mark.parametrize("t,hq,hkv,d,rot", [(1, 1, 1, 16, 16), (3, 5, 2, 48, 32), (129, 4, 4, 64, 64), (2, 40, 40, 64, 64),
                                            (77, 3, 1, 128, 64), (31, 2, 2, 96, 96), (9, 7, 1, 256, 256),
                                            (700, 1, 1, 80, 16), (1, 33, 8, 112, 48)])
def test_qk_norm_rope(t, hq, hkv, d, rot, norm, layout, dtype):
    g = gen(20)
    x = (3 * torch.randn(t, hq + hkv + 1, d, generator=g, device="cuda")).to(dtype)
    q, k = x[:, :hq], x[:, hq:hq + hkv]
    pos = torch.randint(0, 5000, (t,), generator=g, device="cuda", dtype=torch.int32)
    par = {}
    if norm is not None:
        par = {"q_weight": torch.randn(d, generator=g, device="cuda"), "k_weight": torch.randn(d, generator=g, device="cuda")}
    if norm == "layer":
        par |= {"q_bias": torch.randn(d, generator=g, device="cuda"), "k_bias": torch.randn(d, generator=g, device="cuda")}
    rotary = att.Rotary(rot, layout=layout, scaling=SCALINGS[(t + d) % 4])
    qo, ko = att.qk_norm_rope(q, k, pos, rotary, norm=norm, **par)
    for got, src, s in ((qo, q, "q"), (ko, k, "k")):
        ref, tol = rope_ref(src, pos, rotary, norm, par.get(s + "_weight"), par.get(s + "_bias"), 1e-5)
        assert_within(got, ref, tol, s)
    # in place, the same bits; the neighbouring head stays
    before = x[:, -1].clone()
    att.qk_norm_rope(q, k, pos, rotary, norm=norm, q_out=q, k_out=k, **par)
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(x[:, -1], before)


def test_rotary_far_positions_and_types():
    """64-bit, far and negative positions; the int32 form gives the same bits."""
    g = gen(21)
    pos = torch.tensor([0, 1, -1, 12345, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31], device="cuda")
    q = torch.randn(7, 2, 64, generator=g, device="cuda").half()
    rotary = att.Rotary(64)
    q64, k64 = att.qk_norm_rope(q, q.clone(), pos, rotary)
    q32, _ = att.qk_norm_rope(q, q.clone(), pos.int(), rotary)
    assert torch.equal(q64, q32) and torch.equal(q64, k64)
    # the fixed point's frequency is off by half of 2^-64 of a turn: 2^-33 of a turn at 2^31 positions,
    # and the 64-bit angle of the reference by 2^-53 of 2^31 radians
    ref, tol = rope_ref(q, pos, rotary, None, None, None, 0.0)
    assert_within(q64, ref, tol + 2.0 ** -20 * q.double().abs().amax())
    assert torch.equal(q64[0], q[0])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_positions_past_32_bits(layout):
    """Angles against 70 digits.  The allowance is the frequency's rounding, 2^-65 of a turn a position,
    beside the fp32 work of the other tests (whose 2^-20 holds the angle's own rounding, 2^-26 of a turn)."""
    places = [2 ** 31 + 5, 2 ** 32 + 12345, 2 ** 33 - 1, -(2 ** 36) - 7, 2 ** 40 + 1, 2 ** 45 - 3, -(2 ** 48) + 11]
    rot, d = 64, 80
    q = torch.randn(len(places), 3, d, generator=gen(22), device="cuda").half()
    got, _ = att.qk_norm_rope(q, q.clone(), torch.tensor(places, device="cuda"), att.Rotary(rot, layout=layout))
    with localcontext() as ctx:
        ctx.prec = 70
        # pi by Machin's formula
        def arctan_inverse(x):
            total, term, k = Decimal(0), Decimal(1) / x, 1
            while abs(term) > Decimal(10) ** -75:
                total, term, k = total + term / k, -term / (x * x), k + 2
            return total
        pi = 4 * (4 * arctan_inverse(5) - arctan_inverse(239))
        turns = [[float(p * Decimal(10000) ** (Decimal(-2 * i) / rot) / (2 * pi) % 1) for i in range(rot // 2)]
                 for p in places]
    ang = 2 * math.pi * torch.tensor(turns, dtype=torch.float64, device="cuda")[:, None]
    i1 = torch.arange(rot // 2, device="cuda")
    i1, i2 = (i1, i1 + rot // 2) if layout == "half" else (2 * i1, 2 * i1 + 1)
    x = q.double()
    ref, size = x.clone(), x.abs()
    ref[..., i1] = x[..., i1] * ang.cos() - x[..., i2] * ang.sin()
    ref[..., i2] = x[..., i2] * ang.cos() + x[..., i1] * ang.sin()
    size[..., i1] = size[..., i2] = x[..., i1].abs() + x[..., i2].abs()
    far = torch.tensor([2 * math.pi * abs(p) * 2.0 ** -65 for p in places], dtype=torch.float64, device="cuda")
    tol = half_step(FP16) * ref.abs() + (16 * 2.0 ** -24 + far[:, None, None]) * size + least(FP16)
    assert_within(got, ref, tol)


def test_qk_norm_only_and_constant_rows():
    q = torch.full((4, 2, 64), 5.0, device="cuda", dtype=FP16)
    q[1] = 0.0
    a, b = att.qk_norm_rope(q, q.clone(), norm="layer")
    assert (a == 0).all() and (b == 0).all()
    a, _ = att.qk_norm_rope(q, q.clone(), norm="rms")
    assert (a[1] == 0).all() and (a[0] == 1).all()
    q[2, 1, 7] = float("nan")
    a, _ = att.qk_norm_rope(q, q.clone(), norm="rms")
    assert a[2, 1].isnan().all() and not a[2, 0].isnan().any()
    e = torch.empty(0, 2, 64, device="cuda", dtype=FP16)
    assert att.qk_norm_rope(e, e, norm="rms")[0].shape == (0, 2, 64)


# ---- the 8-bit linear layer ------------------------------------------------------------------

def quantize_ref(x):
    """e4m3 values and scales of fp32 quotients, in 64 bits."""
    m, k = x.shape
    kb = -(-k // 128)
    pad = torch.zeros(m, kb * 128, dtype=torch.float64, device=x.device)
    pad[:, :k] = x.double()
    blk = pad.view(m, kb, 128)
    s = (blk.abs().amax(-1) / 448.0).float().clamp(min=2.0 ** -126).double()
    v = (blk / s[..., None]).float().double()
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(v / step) * step, -448, 448).view(m, -1)[:, :k], s


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("m,k", [(1, 16), (3, 128), (17, 144), (5, 272), (129, 1024), (1000, 48), (2, 10240)])
def test_quantize_rows(m, k, dtype):
    x = (torch.randn(m, k + 8, generator=gen(30), device="cuda") * 10).to(dtype)[:, :k]
    x[0, :3] = torch.tensor([0.0, 1e-7, -65504.0], device="cuda").to(dtype)
    x[-1] = 0.0
    x8, s = fp8.quantize_rows(x)
    q, sr = quantize_ref(x)
    assert torch.equal(s.double(), sr) and torch.equal(x8.double(), q)


def test_quantize_rows_non_finite():
    x = torch.ones(4, 256, device="cuda", dtype=FP16)
    x[1, 3], x[2, 200] = float("inf"), float("nan")
    x8, s = fp8.quantize_rows(x)
    y = x8.float() * s.repeat_interleave(128, 1)
    assert y[1, 3].isnan() and y[2, 128:].isnan().all()
    assert (y[0] == 1).all() and (y[1, 128:] == 1).all() and (y[2, :128] == 1).all()


def linear_ref(x8, xs, w, bias, dtype):
    """Output and tolerance: fp32 sums of K products (each step 2^-24 of the absolute sum), the block
    scales (two roundings a block), one rounding of the output."""
    n, k = w.shape
    m = x8.shape[0]
    a = x8.double() * xs.double().repeat_interleave(128, 1)[:, :k]
    b = w.w8.double() * w.scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    out, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        out, size = out + bias.double(), size + bias.double().abs()
    steps = min(k, 128) + 3 * xs.shape[1] + 8
    return out, half_step(dtype) * out.abs() + steps * 2.0 ** -24 * size + least(dtype)


LINEAR_SIZES = [(1, 8, 16), (1, 128, 128), (1, 1000, 1360), (2, 77, 256), (3, 384, 2560), (7, 130, 400), (8, 256, 1024),
                (9, 100, 512), (16, 500, 640), (17, 129, 144), (33, 1, 256), (64, 512, 2048), (100, 1000, 1008),
                (127, 255, 384), (128, 256, 128), (129, 257, 1280), (238, 640, 5120), (300, 333, 208),
                (513, 1025, 896), (1000, 72, 80), (700, 2560, 640),
                (2500, 4100, 272), (257, 19000, 144), (38000, 130, 400), (3300, 3000, 4240)]


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("m,n,k", LINEAR_SIZES)
def test_linear(m, n, k, dtype):
    g = gen(31)
    x = torch.randn(m, k, generator=g, device="cuda")
    x[:, ::7] *= 15.0
    x = x.to(dtype)
    w = fp8.quantize_weight(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k))
    bias = torch.randn(n, generator=g, device="cuda")
    x8, xs = fp8.quantize_rows(x)
    ref, tol = linear_ref(x8, xs, w, bias, dtype)
    assert_within(fp8.linear(x, w, bias=bias), ref, tol)
    ref, tol = linear_ref(x8, xs, w, None, F32)
    got = fp8.linear(x8, w, x_scales=xs, out_dtype=F32)
    assert_within(got, ref, tol)
    assert torch.equal(got, fp8.linear(x, w, out_dtype=F32))  # the same bits by either way, and again


def test_linear_of_e4m3_rows_takes_no_second_copy():
    """The call's workspace for e4m3 x holds the scales (rounded up to 256 rows), not another x."""
    m, k = 5000, 2048
    x8, xs = fp8.quantize_rows(torch.randn(m, k, generator=gen(72), device="cuda").half())
    w = fp8.quantize_weight(torch.randn(64, k, generator=gen(73), device="cuda"))
    out = torch.empty(m, 64, dtype=FP16, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    fp8.linear(x8, w, x_scales=xs, out=out)
    assert torch.cuda.max_memory_allocated() - before <= 5120 * 16 * 4 + 512
    assert_within(out, *linear_ref(x8, xs, w, None, FP16))


def test_linear_views_and_shapes():
    g = gen(32)
    w = fp8.quantize_weight(torch.randn(200, 256, generator=g, device="cuda"))
    base = torch.randn(6, 5, 264, generator=g, device="cuda").half()
    x = base[..., :256]
    got = fp8.linear(x, w)
    assert got.shape == (6, 5, 200)
    assert torch.equal(got.view(30, 200), fp8.linear(x.reshape(30, 256).contiguous(), w))
    buf = torch.full((30, 203), 9.0, device="cuda", dtype=FP16)  # rows of odd pitch
    fp8.linear(x.reshape(30, 256), w, out=buf[:, 1:201])
    assert torch.equal(buf[:, 1:201], got.view(30, 200))
    assert (buf[:, 0] == 9).all() and (buf[:, 201:] == 9).all()
    assert fp8.linear(x[0, 0], w).shape == (200,)
    assert fp8.linear(x[:0], w).shape == (0, 5, 200)


@pytest.mark.parametrize("m", [5, 30])
def test_linear_beside_its_input(m):
    """x and out as columns of one buffer."""
    g = gen(34)
    w = fp8.quantize_weight(torch.randn(200, 256, generator=g, device="cuda"))
    buf = torch.randn(m, 456, generator=g, device="cuda").half()
    x = buf[:, :256].clone()
    want = fp8.linear(x, w)
    fp8.linear(buf[:, :256], w, out=buf[:, 256:])
    assert torch.equal(buf[:, 256:], want) and torch.equal(buf[:, :256], x)
    with pytest.raises(ValueError):
        fp8.linear(buf[:, :256], w, out=buf[:, 255:455])


def test_linear_non_finite_rows_stay_apart():
    g = gen(33)
    for m in (4, 200):
        x = torch.randn(m, 384, generator=g, device="cuda").half()
        w = fp8.quantize_weight(torch.randn(256, 384, generator=g, device="cuda"))
        clean = fp8.linear(x, w)
        x[1, 5] = float("inf")
        x[3, 380] = float("nan")
        got = fp8.linear(x, w)
        keep = torch.ones(m, dtype=torch.bool)
        keep[1] = keep[3] = False
        assert torch.equal(got[keep], clean[keep]) and got[1].isnan().all() and got[3].isnan().all()


@pytest.mark.parametrize("writer", ["copy", "linear"])
@pytest.mark.parametrize("m", [1, 16])
def test_linear_weight_of_the_kernel_in_front(m, writer):
    """Weights that the kernel directly in front writes, by a copy or by a linear layer that starts its
    successor early, eagerly and in a graph: each call multiplies by the new ones.

    The writing layer picks columns of a matrix of few-bit values, exactly: an fp16 value's two bytes are
    then an e4m3 value and a 0."""
    g = gen(35)
    n, k, deep = 256, 128, 10240
    values = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, -0.5, -1.0, -2.0], device="cuda")
    table = values[torch.randint(0, 8, (k // 2, deep), generator=g, device="cuda")]
    picker = fp8.BlockWeight(table.to(torch.float8_e4m3fn), torch.ones(1, deep // 128, device="cuda"))
    picks = [torch.nn.functional.one_hot(torch.randint(0, deep, (n,), generator=g, device="cuda"), deep).half()
             for _ in range(2)]
    new = [fp8.linear(p, picker) for p in picks]
    for p, y in zip(picks, new):
        assert torch.equal(y, table.t()[p.argmax(1)].half())
    buf = torch.zeros(n, k // 2, dtype=FP16, device="cuda")
    w = fp8.BlockWeight(buf.view(torch.float8_e4m3fn), torch.ones(n // 128, 1, device="cuda"))
    x = torch.randn(m, k, generator=g, device="cuda").half()
    want = []
    for y in new:
        buf.copy_(y)
        torch.cuda.synchronize()
        want.append(fp8.linear(x, w))
    torch.cuda.synchronize()
    assert not torch.equal(*want)

    def turns():
        outs = []
        for i in range(20):
            if writer == "copy":
                torch.add(new[i % 2], 0.0, out=buf)
            else:
                fp8.linear(picks[i % 2], picker, out=buf)
            outs.append(fp8.linear(x, w))
        return outs

    outs = turns()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(outs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = turns()
    for _ in range(5):
        graph.replay()
        assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(outs))


# ---- together --------------------------------------------------------------------------------

def layer(x, pos, cu, rotary, w_qkv, w_out, gq, gk, hq, hkv, d):
    qkv = fp8.linear(x, w_qkv).view(x.shape[0], hq + 2 * hkv, d)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    att.qk_norm_rope(q, k, pos, rotary, norm="layer", q_weight=gq, k_weight=gk, q_out=q, k_out=k)
    return fp8.linear(att.attention(q, k, v, cu).view(x.shape[0], -1), w_out)


def layer_state(seed=40):
    g = gen(seed)
    lens, hq, hkv, d, width = [76, 146, 1, 238], 8, 8, 64, 512
    t = sum(lens)
    x = torch.randn(t, width, generator=g, device="cuda").to(BF16)
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    cu = torch.tensor([0, 76, 222, 223, 461], dtype=torch.int32, device="cuda")
    w_qkv = fp8.quantize_weight(torch.randn((hq + 2 * hkv) * d, width, generator=g, device="cuda") / math.sqrt(width))
    w_out = fp8.quantize_weight(torch.randn(width, hq * d, generator=g, device="cuda") / math.sqrt(hq * d))
    gq, gk = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    return x, pos, cu, att.Rotary(64), w_qkv, w_out, gq, gk, hq, hkv, d


def test_layer_step_by_step():
    """Projection, norm with rotation, attention and projection, each step against its own reference on
    the step's own input."""
    x, pos, cu, rotary, w_qkv, w_out, gq, gk, hq, hkv, d = layer_state()
    x8, xs = fp8.quantize_rows(x)
    qkv = fp8.linear(x, w_qkv)
    assert_within(qkv, *linear_ref(x8, xs, w_qkv, None, BF16))
    qkv = qkv.view(-1, hq + 2 * hkv, d)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    qr, kr = att.qk_norm_rope(q, k, pos, rotary, norm="layer", q_weight=gq, k_weight=gk)
    assert_within(qr, *rope_ref(q, pos, rotary, "layer", gq, None, 1e-5))
    assert_within(kr, *rope_ref(k, pos, rotary, "layer", gk, None, 1e-5))
    o = att.attention(qr, kr, v, cu)
    assert_within(o, *attention_ref(qr, kr, v, [76, 146, 1, 238], False, 0.125))
    o = o.view(-1, hq * d)
    y = fp8.linear(o, w_out)
    assert_within(y, *linear_ref(*fp8.quantize_rows(o), w_out, None, BF16))
    assert torch.equal(y, layer(x, pos, cu, rotary, w_qkv, w_out, gq, gk, hq, hkv, d))


def test_layer_captured_and_on_other_streams():
    """A captured layer replays on new inputs; two graphs and an eager call on other streams agree."""
    st = layer_state()
    x = st[0]
    want = layer(*st)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            layer(*st)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(*st)
        graphs.append((g, y))
    for g, y in graphs:
        y.zero_()
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for _, y in graphs)
    x2 = layer_state(41)[0]
    want2 = layer(x2, *st[1:])
    x.copy_(x2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        graphs[0][0].replay()
    with torch.cuda.stream(s2):
        graphs[1][0].replay()
        eager = layer(*st)
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want2) and torch.equal(graphs[1][1], want2) and torch.equal(eager, want2)


def test_status_blocks():
    """A caller's status block stays clean over good calls, and a wrong one is refused."""
    q, k, v, cu = make_qkv([300, 20], 2, 2, 64, FP16, 61)
    status = ops.new_status(q.device)
    o = att.attention(q, k, v, cu, status=status)
    assert torch.equal(o, att.attention(q, k, v, cu))
    w = fp8.quantize_weight(torch.randn(4100, 256))
    for m in (3, 200, 2500):
        x = torch.randn(m, 256, generator=gen(62), device="cuda").half()
        assert torch.equal(fp8.linear(x, w, status=status), fp8.linear(x, w))
    ops.check_status(status, "sequence operators")
    for bad in (status.cpu(), status[:64], status.float()):
        with pytest.raises(ValueError):
            att.attention(q, k, v, cu, status=bad)
        with pytest.raises(ValueError):
            fp8.linear(x, w, status=bad)


def test_errors_of_calls_without_a_status_block_are_heard():
    """The device's own record: clean after good calls; an error in it (a bounded wait that runs out, put
    there by the library's self-test) is raised once, with its code, and cleared."""
    ops.check_sequence_status()
    q, k, v, cu = make_qkv([300, 20], 2, 2, 64, FP16, 65)
    want = att.attention(q, k, v, cu)
    x, w = torch.randn(200, 256, generator=gen(66), device="cuda").half(), fp8.quantize_weight(torch.randn(64, 256))
    fp8.linear(x, w)
    ops.check_sequence_status()
    lib = att._lib.load()
    block = ctypes.c_void_p(0)
    att._lib.check(lib.tmu_sequence_status(ctypes.byref(block)), "tmu_sequence_status")
    side = torch.cuda.Stream()
    for where in (torch.cuda.current_stream(), side):
        att._lib.check(lib.tmu_selftest_wait_timeout(block, 1000000, where.cuda_stream), "tmu_selftest_wait_timeout")
        with torch.cuda.stream(where), pytest.raises(att._lib.TmuError) as e:
            ops.check_sequence_status(q.device)
        assert e.value.name == "TMU_ERR_DEVICE_TIMEOUT"
        torch.cuda.synchronize()
        ops.check_sequence_status("cuda")
    assert torch.equal(att.attention(q, k, v, cu), want)


def test_every_input_that_asks_for_a_gradient_is_refused():
    """Scales and given outputs as much as the values, and tangents as much as gradients."""
    q, k, v, cu = make_qkv([20], 4, 2, 64, FP16, 74)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    o = torch.empty_like(q)
    w = fp8.quantize_weight(torch.randn(32, 64))
    x = torch.zeros(40, 64, device="cuda", dtype=FP16)
    x8, xs = fp8.quantize_rows(x)
    gs = torch.ones(64, device="cuda")
    y = torch.empty(40, 32, device="cuda", dtype=FP16)
    calls = [lambda **a: att.attention(**{"q": q, "k": k, "v": v, "out": o, **a}, cu_seqlens=cu),
             lambda **a: att.qk_norm_rope(**{"q": q, "k": k, "norm": "rms", "q_weight": gs, "q_out": o, **a}),
             lambda **a: fp8.linear(**{"x": x, "weight": w, "out": y, **a}),
             lambda **a: fp8.linear(**{"x": x8, "weight": w, "x_scales": xs, "out": y, **a}),
             lambda **a: fp8.quantize_rows(**{"x": x, **a})]
    given = [{"q": q, "k": k, "v": v, "out": o}, {"q": q, "k": k, "q_weight": gs, "q_out": o}, {"x": x, "out": y},
             {"x_scales": xs, "out": y}, {"x": x}]
    for call, names in zip(calls, given):
        call()
        for name, t in names.items():
            asks = t.detach().clone().requires_grad_()
            with pytest.raises(ValueError, match="backward"):
                call(**{name: asks})
            with torch.no_grad():
                call(**{name: asks})
            with forward_ad.dual_level(), pytest.raises(ValueError, match="forward"):
                call(**{name: forward_ad.make_dual(t, torch.ones_like(t))})
    with pytest.raises(ValueError, match="backward"):
        fp8.linear(x, fp8.BlockWeight(w.w8, w.scales.clone().requires_grad_()))


# ---- refusals that need CUDA tensors ----------------------------------------------------------

def test_refusals():
    q, k, v, cu = make_qkv([20], 4, 2, 64, FP16, 50)
    bias = torch.zeros(1, 4, 20, 20, device="cuda", dtype=FP16)
    for bad in (lambda: att.attention(q, k.to(BF16), v, cu), lambda: att.attention(q, k, v[:, :1], cu),
                lambda: att.attention(q, k[:10], v[:10], cu), lambda: att.attention(q, k, v, cu.long()),
                lambda: att.attention(q, k, v, cu.cpu()), lambda: att.attention(q, k, v, cu, out=q),
                lambda: att.attention(q, k, v, cu, bias=bias.float()), lambda: att.attention(q, k, v, cu, bias=bias[:, :2]),
                lambda: att.attention(q, k, v, cu, bias=bias[0]),
                lambda: att.attention(q, k, v, cu, bias=bias.transpose(2, 3)),
                lambda: att.attention(q.float().half().requires_grad_(), k, v, cu),
                lambda: att.attention(q, k, v, cu, out=q.new_zeros(1, 4, 64).expand(20, 4, 64)),
                lambda: att.qk_norm_rope(q, k, norm="batch"), lambda: att.qk_norm_rope(q, k, q_weight=torch.ones(64)),
                lambda: att.qk_norm_rope(q, k, rotary=att.Rotary(64)),
                lambda: att.qk_norm_rope(q, k, cu[:1].expand(20), att.Rotary(64)),
                lambda: att.qk_norm_rope(q, k, torch.zeros(20, device="cuda"), att.Rotary(64)),
                lambda: att.qk_norm_rope(q, k, torch.zeros(20, device="cuda").int(), att.Rotary(128)),
                lambda: att.qk_norm_rope(q, k, norm="rms", q_out=q, k_out=q[:, :2]),
                lambda: att.qk_norm_rope(q, k, norm="rms", k_out=q[:, 1:3])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: att.attention(q[:, :, :60], k[:, :, :60], v[:, :, :60], cu),
                lambda: att.attention(q[:, :, 4:60], k[:, :, 4:60], v[:, :, 4:60], cu),
                lambda: att.attention(q[:, :3], k, v, cu)):
        with pytest.raises(att._lib.TmuError):
            bad()
    w = fp8.quantize_weight(torch.randn(32, 64))
    x = torch.zeros(4, 64, device="cuda", dtype=FP16)
    x8, xs = fp8.quantize_rows(x)
    for bad in (lambda: fp8.linear(x[:, :48], w), lambda: fp8.linear(x8, w), lambda: fp8.linear(x, w, x_scales=xs),
                lambda: fp8.linear(x, w, bias=torch.zeros(32, device="cuda").half()),
                lambda: fp8.linear(x, w, out=x[:, :32]), lambda: fp8.linear(x.t(), w),
                lambda: fp8.linear(x.clone().requires_grad_(), w), lambda: fp8.linear(x, w, out=torch.zeros(4, 31, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        fp8.linear(x.float(), w)

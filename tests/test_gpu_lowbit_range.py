"""GPU tests of the low-precision serving ops at the ends of their ranges:
queries and scales of magnitudes near the type's limits, arguments and values
that are not numbers.

Tolerances are those of test_gpu_lowbit.py: probabilities and values enter the
products in float16 (2^-11 each), so |o - ref| <= 2^-9 max|v| + half an ulp of
o; a product is off by 2^-16 of sum |x| s (w + z) and half an ulp of y.
"""
import pytest
import torch

import b200k
from test_gpu_lowbit import HALF_ULP, attend64, fill, gen, make_tables, make_weight, randn, values64

pytestmark = pytest.mark.gpu


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("sq", [1, 5])
@pytest.mark.parametrize("magnitude", [1e-35, 1e-20, 1e20, 1e33, 1e34, 1e35, 3e37])
def test_attention_queries_over_the_whole_range_of_bfloat16(dim, group, sq, magnitude):
    # the scale brings the scores back to ordinary numbers
    g = gen(dim + sq)
    cache, k, v = fill(g, 8, 2, 16, dim, group, torch.bfloat16)
    table, lengths = make_tables(g, [100, 9], 16, 8)
    q = randn(g, 2, sq, 8, dim).clamp(-4, 4).mul(magnitude).bfloat16()
    kv = values64(cache, k, v)
    scale = dim ** -0.5 / magnitude
    for s in (scale, -scale):
        ro, rl = attend64(q, kv, table, [100, 9], 16, scale=s)
        o, lse = b200k.cache_attention(q, cache, table, lengths, scale=s, return_lse=True)
        assert ((o.double() - ro).abs() <= 2.0 ** -9 * kv[1].abs().max() + 2.0 ** -8 * ro.abs()).all()
        # fp32 sums of up to D products: 2^-18 of |q||k|, as the scale leaves it
        mag = q.double().norm(dim=-1).max() * kv[0].norm(dim=-1).max() * abs(s)
        assert ((lse.double() - rl).abs() <= 2.0 ** -18 * mag + 1e-5).all()


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128)])
def test_attention_scale_that_is_no_number(dim, group):
    g = gen(dim)
    cache, _, _ = fill(g, 4, 2, 16, dim, group, torch.bfloat16)
    table, lengths = make_tables(g, [40, 0], 16, 4)
    q = randn(g, 2, 1, 4, dim).bfloat16()
    o, lse = b200k.cache_attention(q, cache, table, lengths, scale=float("nan"), return_lse=True)
    assert o[0].isnan().all() and lse[0].isnan().all()
    assert (o[1] == 0).all() and (lse[1] == -float("inf")).all()      # a row that sees nothing
    # a scale of zero: every token counts alike
    o, lse = b200k.cache_attention(q, cache, table, lengths, scale=0.0, return_lse=True)
    assert o[0].isfinite().all() and (lse[0] - torch.log(torch.tensor(40.0))).abs().max() <= 1e-5


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128)])
@pytest.mark.parametrize("batch,tokens,hk", [(1, 40000, 1), (3, 9000, 1), (64, 1500, 2)])
def test_attention_a_nan_value_of_no_weight_reaches_its_dimensions(dim, group, batch, tokens, hk):
    # scores so far apart that nearly every token, and every part that a long
    # sequence is cut into, weighs 0 in fp32: 0 * NaN is NaN in each of them alike
    g = gen(dim + batch)
    page = 64
    wide = -(-tokens // page)
    cache, k, v = fill(g, batch * wide, hk, page, dim, group, torch.bfloat16)
    table = torch.arange(batch * wide, dtype=torch.int32, device="cuda").view(batch, wide)
    lengths = torch.full((batch,), tokens, dtype=torch.int32, device="cuda")
    for step in (0, 1, 2):
        at = torch.arange(batch, device="cuda") * wide * page + \
            (torch.arange(batch, device="cuda") * 397 + step * tokens // 3) % tokens
        part = v[at].clone()
        part[:, 0, group - 1] = float("nan")
        b200k.kv_cache_write(cache, k[at], part, at)
        q = randn(g, batch, 1, 2 * hk, dim).bfloat16()
        o, lse = b200k.cache_attention(q, cache, table, lengths, scale=20.0, return_lse=True)
        nan = torch.zeros(o.shape, dtype=torch.bool, device="cuda")
        nan[:, :, :2, :group] = True
        assert torch.equal(o.isnan(), nan) and lse.isfinite().all()
        b200k.kv_cache_write(cache, k[at], v[at], at)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group,page", [(64, 32, 16), (64, 64, 32), (128, 32, 64), (128, 64, 16),
                                            (128, 128, 64), (256, 32, 16), (256, 128, 32)])
def test_attention_a_partly_nan_value_reaches_its_own_dimensions_only(dtype, dim, group, page):
    # one group of one token's value is NaN: in every row that sees the token the
    # dimensions of that group are NaN, the others and the log-sum numbers,
    # whichever other rows and tokens it is computed with
    g = gen(dim + group + page)
    tokens, sq = 71, 9
    pages = -(-96 // page)
    cache, k, v = fill(g, pages, 2, page, dim, group, dtype)
    kv = values64(cache, k, v)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    q = randn(g, 1, sq, 8, dim).to(dtype)
    for at in (3, 62, 64, 66, 68, 70):             # the last four seen by some queries only
        for first in range(0, dim, group):
            part = v[at:at + 1].clone()
            part[:, 1, first] = float("nan")       # of the second head alone
            b200k.kv_cache_write(cache, k[at:at + 1], part, torch.tensor([at], device="cuda"))
            ro, rl = attend64(q, kv, table, [tokens], page)
            o, lse = b200k.cache_attention(q, cache, table, i32(tokens), return_lse=True)
            nan = torch.zeros(1, sq, 8, dim, dtype=torch.bool, device="cuda")
            nan[:, max(0, at - (tokens - sq)):, 4:, first:first + group] = True
            assert torch.equal(o.isnan(), nan)
            err = (o.double() - ro).abs()
            assert (err <= 2.0 ** -9 * kv[1].abs().max() + HALF_ULP[dtype] * ro.abs())[~nan].all()
            mag = q.double().norm(dim=-1).max() * kv[0].norm(dim=-1).max() * dim ** -0.5
            assert ((lse.double() - rl).abs() <= 2.0 ** -18 * mag + 1e-5).all()
            # each query by itself gives the same answer
            for i in (0, 4, 8):
                one = b200k.cache_attention(q[:, i:i + 1], cache, table, i32(tokens - sq + 1 + i))
                assert torch.equal(one.isnan(), nan[:, i:i + 1])
        b200k.kv_cache_write(cache, k[at:at + 1], v[at:at + 1], torch.tensor([at], device="cuda"))


@pytest.mark.parametrize("xt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("factor", [1e-37, 1e-30, 1e30, 1e34, 1e35, 1.5e36])
@pytest.mark.parametrize("m,per", [(1, None), (5, 64)])
def test_product_scales_of_8_bit_rows_over_the_whole_range(xt, factor, m, per):
    # up to what float32 rows are quantised with, 3.4e38 / 127; eight columns that
    # count, weights of about 1e-2: y is a number
    g = gen(m)
    n, k, group = 48, 320, 64
    w, q, s, zp = make_weight(g, n, k, group, True)
    x = randn(g, m, k) * 4
    x[:, 8:] = 0
    x = (x.round() if xt == torch.int8 else x).to(xt)
    xs = (torch.rand((m, k // per if per else 1), generator=g, device="cuda") + 0.5) * factor
    y = b200k.w4_matmul(x, w, x_scale=xs, out_dtype=torch.float32)
    xd = x.double() * (xs.double().repeat_interleave(per, 1) if per else xs.double())
    ref = xd @ (s.double() * (q.double() - zp)).T
    a = xd.abs() @ (s.double() * (q.double() + zp)).T
    assert ((y.double() - ref).abs() <= 2.0 ** -16 * a + 2.0 ** -24 * ref.abs() + 2.0 ** -146).all()


@pytest.mark.parametrize("m,n,k,group,zeros", [(1, 604, 1145, 128, True), (2, 604, 1145, 128, True),
                                               (3, 100, 1000, 32, True), (5, 333, 4096, 128, False),
                                               (8, 64, 640, 64, True), (19, 48, 2000, 64, False),
                                               (2, 96, 28672, 128, True)])
@pytest.mark.parametrize("loud", [1.0, 20.0, 100.0])
def test_product_of_float32_rows_keeps_float32(m, n, k, group, zeros, loud):
    # Some columns are `loud` times the others, as hidden states have them.  x in
    # parts of whole units makes a group's sums exact; what is left are three fp32
    # roundings a group and one for adding it up, each 2^-24 at most and 0.3 of
    # 2^-23 in the mean square, of partial sums that are at most the result's size
    # in the mean square: over G groups sqrt(G) 2^-24.7 of it, and the roundings
    # of a group's own share, which is sqrt(1/G) of it.
    g = gen(m + k)
    w, q, s, zp = make_weight(g, n, k, group, zeros)
    x = randn(g, m, k)
    x[:, torch.rand(k, generator=g, device="cuda") < 0.01] *= loud
    y = b200k.w4_matmul(x, w).double()
    ref = x.double() @ (s.double() * (q.double() - zp)).T
    groups = -(-k // group)
    bound = 1.2 * 2.0 ** -24.7 * (groups + 3) ** 0.5
    assert (y - ref).norm() <= bound * ref.norm(), float((y - ref).norm() / ref.norm())
    one = b200k.w4_matmul(x[m - 1:], w).double()     # the last row by itself
    assert (one - ref[m - 1:]).norm() <= 1.2 * bound * ref[m - 1:].norm()


@pytest.mark.parametrize("xt,m", [(torch.float32, 65535 * 8 + 5), (torch.float32, 65535 * 8),
                                  (torch.bfloat16, 65535 * 32 + 33), (torch.int8, 65535 * 32 + 1)])
def test_product_of_more_rows_than_one_launch_takes(xt, m):
    g = gen(9)
    w, q, s, zp = make_weight(g, 16, 40, 32, True)
    x = randn(g, m, 40)
    xs = torch.rand((m, 1), generator=g, device="cuda") + 0.5 if xt == torch.int8 else None
    x = (x * 30).round().clamp(-127, 127).to(xt) if xs is not None else x.to(xt)
    y = b200k.w4_matmul(x, w, x_scale=xs, out_dtype=torch.float32).double()
    xd = x.double() if xs is None else x.double() * xs.double()
    wd = s.double() * (q.double() - zp)
    a = xd.abs() @ (s.double() * (q.double() + zp)).T
    assert y.shape == (m, 16) and ((y - xd @ wd.T).abs() <= 2.0 ** -16 * a).all()

"""GPU tests of the low-precision serving ops' kernels for many rows, which
smaller calls do not reach: the row pipeline of the 8-bit norm, attention with
16 query rows a tile in every group size, and the merge of over 1024 parts.

Tolerances of the attention.  An entry o_d = sum_j p_j v_jd takes rounding
errors that are independent of one another: of the products' operands, each
2^-11 at most, and of the output.  At a mantissa of m the rounding to a unit u
of the leading one is uniform within u / (2 m), and over mantissas spread
evenly in their logarithm its mean square is (u/2)^2 / 3 * 0.541, that is
(0.4246 u/2)^2.  So over many outputs

    rms(error)^2 = 0.4246^2 (r (2^-11)^2 rms(noise)^2 + (u/2)^2 rms(o)^2),
    noise_d^2 = sum_j (p_j v_jd)^2,

with r operand roundings a term: one (the value lo + s n) for float16 queries,
whose probabilities are held in two parts; two (value, probability) for
bfloat16; with a single group per head, whose integers are exact, one (p s) for
bfloat16 and none for float16 (the last test; the others allow one).
fp32 scores add relative errors of about 1e-6.  Checked with 10 % above; one
more rounding of a float16 call's operands would be 22 % above.
"""
import pytest
import torch

import b200k
from test_gpu_lowbit import HALF_ULP, T16, fill, gen, make_tables, no_timeouts, norm_case, randn, values64

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------
# the norm's row pipeline: at least 256 vectors of 16 bytes a row, aligned, and
# more rows than resident blocks (at most 16 per SM, 2368 on 148 SMs)
@pytest.mark.parametrize("dtype,cols", [
    (torch.bfloat16, 2048), (torch.bfloat16, 2056), (torch.bfloat16, 8200), (torch.bfloat16, 16648),
    (torch.float16, 2056), (torch.float16, 4096), (torch.float16, 8192), (torch.float16, 16640),
    (torch.float32, 1024), (torch.float32, 2052), (torch.float32, 4100), (torch.float32, 8192)])
@pytest.mark.parametrize("out,group", [(torch.int8, None), (torch.int8, 64), (torch.float8_e4m3fn, None),
                                       (torch.float8_e4m3fn, 32), (torch.float8_e4m3fn, 128)])
def test_norm_quant_many_rows(dtype, cols, out, group):
    rows = 5003
    g = gen(cols)
    x, r = (randn(g, rows, cols) * 3).to(dtype), (randn(g, rows, cols) * 2).to(dtype)
    w = (1 + 0.3 * randn(g, cols)).to(dtype)
    # the ring's stages hold other rows' data: each row has a size of its own
    x *= torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g, device="cuda").float()).to(dtype)
    x0, r0 = x.clone(), r.clone()
    norm_case(x, r, w, out, group, b200k.add_rmsnorm_quant(x, r, w, dtype=out, group=group))
    q, scale = b200k.rmsnorm_quant(x, w, dtype=out, group=group)
    norm_case(x, None, w, out, group, (None, q, scale))
    assert torch.equal(x, x0) and torch.equal(r, r0)
    no_timeouts()


@pytest.mark.parametrize("out,group", [(torch.int8, None), (torch.float8_e4m3fn, 32)])
def test_norm_quant_many_rows_special(out, group):
    rows, cols = 5003, 2056
    g = gen(7)
    x, r = randn(g, rows, cols).bfloat16(), randn(g, rows, cols).bfloat16()
    w = torch.ones(cols, device="cuda").bfloat16()
    nan, inf, zero = [0, 400, 2500, rows - 1], [1, 3000], [2, 401, 4999]
    x[nan, [5, 2055, 100, 2048]] = float("nan")
    x[inf, 7] = float("inf")
    x[zero], r[zero] = 0, 0
    odd = torch.zeros(rows, dtype=torch.bool, device="cuda")
    odd[nan + inf + zero] = True
    h, q, s = b200k.add_rmsnorm_quant(x, r, w, dtype=out, group=group)
    assert s[nan].isnan().all()
    # an infinite row: 1 / rms is 0, so y is NaN in the infinity's own group, 0 in others
    assert s[inf, 0].isnan().all() and (s[inf, 1:] == 0).all()
    assert (s[zero] == 0).all() and (q[zero].float() == 0).all() and (h[zero] == 0).all()
    norm_case(x[~odd], r[~odd], w, out, group, (h[~odd], q[~odd], s[~odd]))
    # rows with a stride, and a residual with another
    big, wide = randn(g, rows, cols + 64).bfloat16(), randn(g, rows, cols + 8).bfloat16()
    x, r = big[:, 32:32 + cols], wide[:, :cols]
    norm_case(x, r, w, out, group, b200k.add_rmsnorm_quant(x, r, w, dtype=out, group=group))
    # the same rows few at a time, on the other kernel
    h, q, s = b200k.add_rmsnorm_quant(x, r, w, dtype=out, group=group)
    for at in (0, 147, 2367, 4990):
        few = b200k.add_rmsnorm_quant(x[at:at + 13], r[at:at + 13], w, dtype=out, group=group)
        assert torch.equal(few[0], h[at:at + 13])
        # their sums are added in another order: 2^-16, as the scale is
        torch.testing.assert_close(few[2], s[at:at + 13], rtol=2.0 ** -15, atol=0)
    no_timeouts()


# --------------------------------------------------------------------------
# attention
def attend64(q, kv, table, lens, page, scale):
    """(o, noise^2, lse) in 64 bits, causal; noise^2 = sum_j (p_j v_j)^2."""
    b, sq, h, d = q.shape
    hk = kv[0].shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    noise, lse = torch.zeros_like(o), torch.full((b, h, sq), -float("inf"), dtype=torch.float64, device=q.device)
    for i, n in enumerate(lens):
        if n == 0:
            continue
        j = torch.arange(n, device=q.device)
        slots = table[i, j // page].long() * page + j % page
        k, v = (x[slots] for x in kv)
        f = q[i].double().view(sq, hk, h // hk, d)
        z = torch.einsum("thgd,jhd->hgtj", f, k) * scale
        seen = j[None] <= n - sq + torch.arange(sq, device=q.device)[:, None]
        z = z.masked_fill(~seen, -float("inf"))
        lse[i] = torch.logsumexp(z, -1).reshape(h, sq)
        p = torch.softmax(z, -1).nan_to_num(0)
        o[i] = torch.einsum("hgtj,jhd->thgd", p, v).reshape(sq, h, d)
        noise[i] = torch.einsum("hgtj,jhd->thgd", p * p, v * v).reshape(sq, h, d)
    return o, noise, lse


def attend_case(seed, dtype, lens, sq, heads, hk, dim, group, page, offset=0.0, rounded=None):
    """Every element within 2^-9 of its own share sum_j p_j |v_j|, and all of
    them within the mean square above."""
    g = gen(seed)
    pages = sum(-(-n // page) for n in lens) + 1
    cache = b200k.KVCache4.zeros(pages, page, hk, dim, group)
    for at in range(0, pages * page, 1 << 16):
        n = min(1 << 16, pages * page - at)
        k = randn(g, n, hk, dim) + randn(gen(seed), hk, dim)
        v = randn(g, n, hk, dim) + offset
        b200k.kv_cache_write(cache, k.to(dtype), v.to(dtype), torch.arange(at, at + n, device="cuda"))
    table, lengths = make_tables(g, lens, page, pages)
    q = randn(g, len(lens), sq, heads, dim).to(dtype)
    kv = values64(cache, None, None)
    o, lse = b200k.cache_attention(q, cache, table, lengths, return_lse=True)
    ro, noise, rl = attend64(q, kv, table, lens, page, dim ** -0.5)
    empty = rl == -float("inf")
    assert torch.equal(lse == -float("inf"), empty)
    assert (o.permute(0, 2, 1, 3)[empty] == 0).all()
    mag = q.double().norm(dim=-1).max() * kv[0].norm(dim=-1).max() * dim ** -0.5
    assert ((lse.double() - rl)[~empty].abs() <= 2.0 ** -18 * mag + 1e-5).all()
    err = (o.double() - ro).permute(0, 2, 1, 3)[~empty]
    noise, ro = (t.permute(0, 2, 1, 3)[~empty] for t in (noise, ro))
    half = HALF_ULP[dtype]
    if rounded is None:
        rounded = 2 if dtype == torch.bfloat16 and group < dim else 1
    want = 0.4246 * (rounded * 2.0 ** -22 * noise.mean() + half ** 2 * (ro * ro).mean()).sqrt()
    got = (err * err).mean().sqrt()
    assert got <= 1.1 * want, (float(got), float(want))
    no_timeouts()


SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("sq,heads,hk,page", [
    (3, 8, 2, 16),      # 12 rows a head: one tile of 16
    (5, 14, 2, 64),     # 35: three
    (1, 24, 2, 48),     # 12 heads a head
    (1, 4, 1, 32),      # 4: a tile of 8
])
def test_attention_errors_are_those_of_its_roundings(dtype, dim, group, sq, heads, hk, page):
    # lengths that end inside a tile, cross tiles and warps, one short of the queries
    attend_case(dim + group + sq, dtype, [700, 33, 0, 1500, 2], sq, heads, hk, dim, group, page)


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 32), (128, 128), (256, 128)])
def test_attention_errors_with_an_offset_in_the_values(dim, group):
    # values around 3: the sums are large beside the rounded parts
    attend_case(dim, torch.float16, [900, 40], 4, 16, 4, dim, group, 32, offset=3.0)


@pytest.mark.parametrize("dtype,lens,sq,heads,hk", [
    (torch.bfloat16, [16384, 33], 1, 32, 4), (torch.float16, [16384, 33], 1, 8, 8),
    (torch.float16, [9000], 4, 16, 2), (torch.bfloat16, [20001], 3, 8, 1)])
@pytest.mark.parametrize("group", [32, 128])
def test_attention_errors_over_many_tokens(dtype, lens, sq, heads, hk, group):
    attend_case(len(lens) + sq, dtype, lens, sq, heads, hk, 128, group, 64)


@pytest.mark.parametrize("dtype,dim,group,sq,heads", [
    (torch.float16, 64, 64, 1, 4), (torch.bfloat16, 64, 32, 3, 4), (torch.float16, 128, 32, 1, 1)])
def test_attention_of_over_1024_parts(dtype, dim, group, sq, heads):
    # one segment, cut into a run of four tiles and less for every warp: more
    # parts than the merge holds at a time
    attend_case(5, dtype, [150001], sq, heads, 1, dim, group, 64)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,sq,heads,hk", [([700, 33, 0, 1500], 1, 8, 2), ([900, 40], 5, 14, 2),
                                              ([16384], 1, 8, 2), ([60000, 777], 1, 7, 1),
                                              ([20001], 3, 8, 1)])
def test_attention_of_float16_over_one_group_rounds_only_its_output(dim, lens, sq, heads, hk):
    # integers are exact and probabilities held in two parts: r = 0
    attend_case(dim + sq, torch.float16, lens, sq, heads, hk, dim, dim, 64, rounded=0)

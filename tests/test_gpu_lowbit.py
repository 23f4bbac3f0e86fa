"""GPU tests of the low-precision serving ops (b200k/lowbit.py) against their
definitions in 64 bits.

Tolerances, from the arithmetic of each op:
  norm    fp32 sums of squares: rows of at most 2^17 terms, summed in runs of
          at most 2^7 and then pairwise: relative error below 2^8 * 2^-24 =
          2^-16 in y and in the scale; the quantised value is then within half
          a step of y.
  cache   the stored integer is the nearest (or, within 2^-16 of a tie, either
          neighbour); reading back is one fp32 rounding and one to the type.
  attend  probabilities and values enter the products in float16 (2^-11 each),
          scores are fp32 sums: |o - ref| <= 2^-9 max|v| + half an ulp of o.
  product exact integer weights in float16 times float16 pieces of x with fp32
          sums: 2^-16 of A = sum |x| s (w + z), + half an ulp of y.
"""
import numpy as np
import pytest
import torch

import b200k

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
T16 = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def no_timeouts():
    torch.cuda.synchronize()
    assert b200k._lib.lib.b2k_pipeline_timeouts(0) == 0


# --------------------------------------------------------------------------
# norm
def norm_case(x, r, w, dtype, group, out):
    """Checks an (h, q, scale) against the definition in 64 bits."""
    h, q, scale = out
    n = x.shape[-1]
    hx = x if r is None else (x.double() + r.double()).to(x.dtype)
    if r is not None:
        assert torch.equal(h, hx)
    f = hx.double().reshape(-1, n)
    y = f * w.double() / torch.sqrt((f * f).mean(1, keepdim=True) + 1e-6)
    g = group or n
    ns = -(-n // g)
    assert q.shape == x.shape and q.dtype == dtype
    assert scale.shape == x.shape[:-1] + (ns,) and scale.dtype == torch.float32
    yp = torch.nn.functional.pad(y, (0, ns * g - n)).view(-1, ns, g)
    top = yp.abs().amax(-1)
    most = 127 if dtype == torch.int8 else 448
    want = torch.where(top < 1e-30, torch.zeros_like(top), top / most)
    s = scale.double().view(-1, ns)
    torch.testing.assert_close(s, want, rtol=2.0 ** -15, atol=0)
    per = s.repeat_interleave(g, 1)[:, :n]
    v = q.double().view(-1, n)
    unit = torch.where(per > 0, per, torch.ones_like(per))
    if dtype == torch.int8:
        half = torch.full_like(y, 0.5)
    else:  # half the distance of neighbouring e4m3 values
        a = (y / unit).abs().clamp(2.0 ** -6, 448)
        half = torch.exp2(torch.floor(torch.log2(a)) - 4)
    err = (v - torch.where(per > 0, y / unit, torch.zeros_like(y))).abs()
    assert (err <= half * (1 + 2.0 ** -10) + (y / unit).abs() * 2.0 ** -14).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("rows,cols,group", [
    (1, 1, None), (3, 7, 32), (5, 33, 32), (2, 64, 128), (9, 128, 64), (4, 200, 64), (7, 1000, 128),
    (300, 256, 128), (2, 4096, None), (3, 4097, 128), (2, 8192, 32), (2, 12288, None),
    (1, 16640, 64), (2, 40000, 128), (1, 70001, None)])
def test_norm_quant(dtype, out, rows, cols, group):
    g = gen(rows * 7 + cols)
    x, r = (randn(g, rows, cols) * 3).to(dtype), (randn(g, rows, cols) * 2).to(dtype)
    w = (1 + 0.3 * randn(g, cols)).to(dtype)
    x0 = x.clone()
    norm_case(x, r, w, out, group, b200k.add_rmsnorm_quant(x, r, w, dtype=out, group=group))
    q, scale = b200k.rmsnorm_quant(x, w, dtype=out, group=group)
    norm_case(x, None, w, out, group, (None, q, scale))
    assert torch.equal(x, x0)
    no_timeouts()


@pytest.mark.parametrize("cols,off", [(4096, 0), (4096, 3), (520, 8)])
def test_norm_quant_strides_and_dims(cols, off):
    g = gen(cols)
    x = randn(g, 2, 6, cols + 16).half()[..., off:off + cols]
    r = randn(g, 2, 6, cols).half()
    w = randn(g, 2 * cols)[::2].half()
    norm_case(x, r, w.contiguous(), torch.int8, None, b200k.add_rmsnorm_quant(x, r, w))
    one = b200k.rmsnorm_quant(x[0, 0], w)
    assert one[0].shape == (cols,) and one[1].shape == (1,)


def test_norm_quant_special_rows():
    g = gen(1)
    x = randn(g, 6, 512)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 9] = float("inf")
    x[3] = 1e-34                    # y = 1e-31: below the smallest maximum
    w = torch.ones(512, device="cuda")
    for dtype in (torch.int8, torch.float8_e4m3fn):
        q, s = b200k.rmsnorm_quant(x, w, dtype=dtype)
        assert s[0] == 0 and (q[0].float() == 0).all()
        assert s[1].isnan() and s[2].isnan()
        assert s[3] == 0 and (q[3].float() == 0).all()
        norm_case(x[4:], None, w, dtype, None, (None, q[4:], s[4:]))
        q, s = b200k.rmsnorm_quant(x, w, dtype=dtype, group=128)
        assert s[1].isnan().all()
        w2 = w.clone()
        w2[200] = float("nan")      # one group's weight: that group alone
        q, s = b200k.rmsnorm_quant(x[4:], w2, dtype=dtype, group=128)
        assert s[:, 1].isnan().all() and s[:, [0, 2, 3]].isfinite().all()


def test_norm_quant_empty_and_one_row_scales_feed_dequant():
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    h, q, s = b200k.add_rmsnorm_quant(*[torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)] * 2, w)
    assert h.shape == q.shape == (0, 64) and s.shape == (0, 1)
    g = gen(2)
    x = randn(g, 33, 4096).bfloat16()
    q, s = b200k.rmsnorm_quant(x, torch.ones(4096, device="cuda", dtype=torch.bfloat16))
    y = b200k.dequant_int8(q, s)
    torch.testing.assert_close(y.float(), (q.float() * s), rtol=2.0 ** -10, atol=0)


# --------------------------------------------------------------------------
# cache
def quantise64(x, group):
    x = x.double().clamp(-65408, 65408).unflatten(-1, (-1, group))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, lo = ((hi - lo) / 15).half().double(), lo.half().double()
    t = torch.where(s > 0, (x - lo) / torch.where(s > 0, s, 1.0), torch.zeros_like(x)).clamp(0, 15)
    return t, s, lo


def check_values(got, x, group):
    """got: what the cache stands for after x was written."""
    t, s, lo = quantise64(x, group)
    n = t.round()
    near = (t - t.floor() - 0.5).abs() < 2.0 ** -16
    got = got.unflatten(-1, (-1, group))
    ulp = 2 * HALF_ULP[got.dtype]

    def same(n):
        v = lo + n * s
        return (got.double() - v).abs() <= v.abs() * ulp / 2 + 2.0 ** -25

    ok = same(n) | (near & (same(t.floor()) | same(t.ceil())))
    assert ok.all(), (got.double() - (lo + n * s)).abs().max()


def fill(g, pages, heads, page, dim, group, dtype, loud=1.0):
    """A cache with every slot written: (cache, k, v) with k, v [slots, heads, dim]."""
    cache = b200k.KVCache4.zeros(pages, page, heads, dim, group)
    k = (randn(g, pages * page, heads, dim) * loud + randn(g, heads, dim)).to(dtype)
    v = randn(g, pages * page, heads, dim).to(dtype)
    b200k.kv_cache_write(cache, k, v, torch.arange(pages * page, device="cuda"))
    return cache, k, v


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128),
                                       (256, 32), (256, 64), (256, 128)])
@pytest.mark.parametrize("heads,page", [(1, 16), (3, 48), (8, 64)])
def test_cache_round_trip(dtype, dim, group, heads, page):
    g = gen(dim + group + page)
    cache, k, v = fill(g, 3, heads, page, dim, group, dtype)
    order = torch.randperm(3 * page, generator=g, device="cuda")
    rk, rv = b200k.kv_cache_read(cache, order, dtype=dtype)
    check_values(rk, k[order], group)
    check_values(rv, v[order], group)
    # the same bytes in the other type
    other = [t for t in T16 if t != dtype][0]
    ok, _ = b200k.kv_cache_read(cache, order, dtype=other)
    torch.testing.assert_close(ok.double(), rk.double(), rtol=2.0 ** -8, atol=2.0 ** -24)


def decode_bytes(cache, slot, head):
    """(k, v) of one token by the documented layout, with numpy."""
    page, off = divmod(slot, cache.page_size)
    d, g = cache.head_dim, cache.group
    m = cache.data[page, head, off // 16].cpu().numpy()
    t, out, at = off % 16, [], 0
    for is_key in (True, False):
        row = m[at + t * d // 2: at + (t + 1) * d // 2]
        at += 8 * d
        par = m[at + t * 4 * (d // g): at + (t + 1) * 4 * (d // g)].copy().view(np.float16)
        at += 64 * d // g
        y = np.empty(d)
        for i in range(d):
            j, c, e = i // 32, i % 32 // 8, i % 8
            p = (c * (d // 32) + j) * 8 + e if is_key else i
            n = row[p // 2] >> (4 * (p % 2)) & 15
            y[i] = np.float64(par[2 * (i // g) + 1]) + np.float64(par[2 * (i // g)]) * n
        out.append(y)
    return out


@pytest.mark.parametrize("dim,group,page", [(64, 64, 16), (128, 32, 64), (256, 128, 32)])
def test_cache_bytes_follow_the_layout(dim, group, page):
    g = gen(dim)
    cache, k, v = fill(g, 2, 2, page, dim, group, torch.float16)
    rk, rv = b200k.kv_cache_read(cache, torch.arange(2 * page, device="cuda"), dtype=torch.float16)
    for slot in (0, 1, 15, page - 1, page, 2 * page - 1):
        for head in range(2):
            dk, dv = decode_bytes(cache, slot, head)
            assert np.abs(rk[slot, head].double().cpu().numpy() - dk).max() <= 2.0 ** -11 * np.abs(dk).max()
            assert np.abs(rv[slot, head].double().cpu().numpy() - dv).max() <= 2.0 ** -11 * np.abs(dv).max()


def test_cache_special_values():
    cache = b200k.KVCache4.zeros(1, 16, 1, 64, 32)
    k = torch.zeros(4, 1, 64, device="cuda", dtype=torch.bfloat16)
    k[0] = 3.0                        # constant groups
    k[1, 0, 0] = float("nan")         # its group alone
    k[2, 0, 0], k[2, 0, 1] = 1e6, -float("inf")
    k[3, 0, :32] = 65408.0
    k[3, 0, 0] = -65408.0
    b200k.kv_cache_write(cache, k, k, torch.arange(4, device="cuda"))
    for r in b200k.kv_cache_read(cache, torch.arange(4, device="cuda"), dtype=torch.float16):
        assert (r[0] == 3).all()
        assert r[1, 0, :32].isnan().all() and (r[1, 0, 32:] == 0).all()
        assert r[2].isfinite().all() and r[2, 0, 1] <= -65000 and r[2, 0, 0] >= 64000
        assert r[3].isfinite().all() and r[3, 0, 1] >= 65000 and r[3, 0, 0] <= -65000


def test_cache_skips_and_slots_outside():
    g = gen(3)
    cache = b200k.KVCache4.zeros(2, 16, 2, 64, 32)
    before = cache.data.clone()
    k = randn(g, 5, 2, 64).half()
    slots = torch.tensor([-1, 32, 1 << 40, -(1 << 40), 7], device="cuda")
    b200k.kv_cache_write(cache, k, k, slots)
    changed = (cache.data != before).view(2, 2, 1, -1).any(-1)
    assert changed[0].all() and not changed[1].any()
    rk, rv = b200k.kv_cache_read(cache, slots, dtype=torch.float16)
    for r in (rk, rv):
        assert (r[0] == 0).all() and r[1].isnan().all() and r[2].isnan().all() and (r[3] == 0).all()
    check_values(rk[4:], k[4:], 32)
    # nothing to do
    b200k.kv_cache_write(cache, k[:0], k[:0], slots[:0])
    assert b200k.kv_cache_read(cache, slots[:0])[0].shape == (0, 2, 64)


def test_cache_write_from_strided_views():
    g = gen(4)
    qkv = randn(g, 2, 9, 12, 128).bfloat16()       # a fused projection: 8 q, 2 k, 2 v heads
    k, v = qkv[:, :, 8:10], qkv[:, :, 10:12]
    cache = b200k.KVCache4.zeros(2, 16, 2, 128, 64)
    slots = torch.randperm(32, generator=g, device="cuda")[:18].view(2, 9)
    b200k.kv_cache_write(cache, k, v, slots)
    rk, rv = b200k.kv_cache_read(cache, slots)
    assert rk.shape == (2, 9, 2, 128)
    check_values(rk, k, 64)
    check_values(rv, v, 64)
    odd = randn(g, 3, 2, 133).half()[..., 1:129]   # rows that are not 16-byte aligned
    b200k.kv_cache_write(cache, odd, odd, torch.tensor([4, 1, 30], device="cuda"))
    check_values(b200k.kv_cache_read(cache, torch.tensor([4, 1, 30], device="cuda"),
                                     dtype=torch.float16)[0], odd, 64)


# --------------------------------------------------------------------------
# attention
def attend64(q, kv, table, lens, page, causal=True, scale=None):
    """Definition in 64 bits: kv = (k, v) [slots, heads, D] of the whole pool."""
    b, sq, h, d = q.shape
    hk = kv[0].shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((b, h, sq), -float("inf"), dtype=torch.float64, device=q.device)
    for i, n in enumerate(lens):
        j = torch.arange(n, device=q.device)
        slots = table[i, j // page].long() * page + j % page
        for t in range(sq):
            m = max(0, n - sq + t + 1) if causal else n
            if m == 0:
                continue
            k, v = (x[slots[:m]].double().repeat_interleave(h // hk, 1) for x in kv)
            z = torch.einsum("hd,jhd->hj", q[i, t].double(), k) * (scale or d ** -0.5)
            o[i, t] = torch.einsum("hj,jhd->hd", torch.softmax(z, -1), v)
            lse[i, :, t] = torch.logsumexp(z, -1)
    return o, lse


def make_tables(g, lens, page, pages, extra=1, fill_value=-1):
    """Distinct random pages for every sequence; entries past its length are fill_value."""
    width = max(1, max(-(-n // page) for n in lens)) + extra
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), width), fill_value, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        c = -(-n // page)
        table[i, :c] = ids[at:at + c]
        at += c
    assert at <= pages
    return table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def attend_case(seed, dtype, lens, sq, heads, hk, dim, group, page, causal=True, scale=None,
                loud=1.0):
    g = gen(seed)
    pages = sum(-(-n // page) for n in lens) + 2
    cache, k, v = fill(g, pages, hk, page, dim, group, dtype, loud)
    # what lies in pages and rows that no length covers is garbage: NaN parameters
    table, lengths = make_tables(g, lens, page, pages)
    used = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    for i, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        used[table[i, j // page].long() * page + j % page] = True
    nan = torch.full((int((~used).sum()), hk, dim), float("nan"), dtype=dtype, device="cuda")
    b200k.kv_cache_write(cache, nan, nan, (~used).nonzero().flatten())
    q = randn(g, len(lens), sq, heads, dim).to(dtype)
    kv = values64(cache, k, v)
    o, lse = b200k.cache_attention(q, cache, table, lengths, causal=causal, scale=scale,
                                   return_lse=True)
    ro, rl = attend64(q, kv, table, lens, page, causal, scale)
    top = kv[1].nan_to_num(0).abs().max()
    err = (o.double() - ro).abs()
    assert (err <= 2.0 ** -9 * top + HALF_ULP[dtype] * ro.abs()).all(), (err.max(), top)
    empty = rl == -float("inf")
    assert torch.equal(lse == -float("inf"), empty)
    # scores are fp32 sums of up to D products of magnitude |q||k|
    mag = (q.double().norm(dim=-1).max() * kv[0].nan_to_num(0).norm(dim=-1).max()) * abs(scale or dim ** -0.5)
    assert ((lse.double() - rl)[~empty].abs() <= 2.0 ** -18 * mag + 1e-5).all()
    assert (o.permute(0, 2, 1, 3)[empty] == 0).all()
    no_timeouts()
    return cache, q, table, lengths, o


def values64(cache, k, v):
    """What every slot of the cache stands for, in 64 bits, by the documented layout."""
    d, g = cache.head_dim, cache.group
    data, out, at = cache.data, [], 0
    place = torch.arange(d, device="cuda")
    for is_key in (True, False):
        rows = data[..., at:at + 8 * d].unflatten(-1, (16, d // 2)).long()
        at += 8 * d
        par = data[..., at:at + 64 * d // g].contiguous().view(torch.float16)
        par = par.unflatten(-1, (16, d // g, 2)).double()
        at += 64 * d // g
        p = place % 32 // 8 * (d // 4) + place // 32 * 8 + place % 8 if is_key else place
        n = (rows[..., p // 2] >> (4 * (p % 2))) & 15
        y = par[..., place // g, 1] + par[..., place // g, 0] * n     # [pages, hk, P/16, 16, D]
        out.append(y.permute(0, 2, 3, 1, 4).reshape(-1, cache.kv_heads, d))
    return out


EDGE = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128),
                                       (256, 32), (256, 64), (256, 128)])
def test_attention_every_length(dtype, dim, group):
    attend_case(dim + group, dtype, EDGE, 1, 8, 2, dim, group, 16)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 256])
@pytest.mark.parametrize("sq", [1, 2, 5])
def test_attention_pages(page, sq):
    attend_case(page + sq, torch.bfloat16, EDGE + [300], sq, 4, 2, 64, 32, page)


@pytest.mark.parametrize("heads,hk", [(1, 1), (2, 2), (3, 1), (7, 1), (14, 2), (8, 1), (16, 1),
                                      (24, 2), (40, 1), (71, 1), (10, 10)])
@pytest.mark.parametrize("sq", [1, 3])
def test_attention_head_layouts(heads, hk, sq):
    attend_case(heads * 10 + sq, torch.float16, [5, 100, 0, 64], sq, heads, hk, 128, 32, 32)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sq,lens", [(17, [17, 5, 40, 0]), (33, [200, 33, 1]), (70, [70, 300, 69]),
                                     (128, [128, 129])])
def test_attention_many_queries(dim, sq, lens):
    attend_case(sq + dim, torch.bfloat16, lens, sq, 4, 2, dim, 32, 16)


@pytest.mark.parametrize("sq", [1, 4])
def test_attention_not_causal(sq):
    attend_case(sq, torch.float16, [3, 0, 90, 1], sq, 4, 2, 128, 64, 16, causal=False)


@pytest.mark.parametrize("lens", [[5000], [3000, 1, 0, 777], [16384, 33]])
@pytest.mark.parametrize("sq,heads,hk", [(1, 8, 8), (1, 32, 4), (4, 16, 2)])
def test_attention_long(lens, sq, heads, hk):
    attend_case(len(lens) + sq, torch.bfloat16, lens, sq, heads, hk, 128, 32, 64)


def test_attention_many_short_sequences():
    lens = [(i * 37) % 90 for i in range(333)]
    attend_case(9, torch.float16, lens, 1, 8, 4, 64, 64, 16)


def test_attention_sharp_scores_and_scale():
    # scores of several hundred: the softmax is nearly one-hot, the running
    # maximum moves often
    attend_case(11, torch.float16, [700, 64], 1, 8, 2, 128, 32, 16, scale=3.0, loud=4.0)
    attend_case(12, torch.float16, [700, 64], 1, 8, 2, 128, 32, 16, scale=-0.5)
    attend_case(13, torch.float16, [700, 64], 1, 8, 2, 128, 32, 16, scale=1e-4)


@pytest.mark.parametrize("factor", [1e-6, 1e-3, 300.0])
def test_attention_small_and_large_queries(factor):
    g = gen(14)
    cache, k, v = fill(g, 20, 2, 16, 128, 32, torch.bfloat16)
    table, lengths = make_tables(g, [300], 16, 20)
    q = (randn(g, 1, 1, 8, 128) * factor).bfloat16()
    kv = values64(cache, k, v)
    ro, _ = attend64(q, kv, table, [300], 16, scale=1.0 / (factor * 11.3))
    o = b200k.cache_attention(q, cache, table, lengths, scale=1.0 / (factor * 11.3))
    assert ((o.double() - ro).abs() <= 2.0 ** -9 * kv[1].abs().max() + 2.0 ** -8 * ro.abs()).all()


def test_attention_small_values():
    # values of 1e-4: their float16 parameters and products keep their precision
    g = gen(15)
    cache = b200k.KVCache4.zeros(10, 16, 1, 64, 32)
    k = randn(g, 160, 1, 64).half()
    v = (1e-4 * (1 + randn(g, 160, 1, 64))).half()
    b200k.kv_cache_write(cache, k, v, torch.arange(160, device="cuda"))
    table = torch.arange(10, dtype=torch.int32, device="cuda")[None]
    q = randn(g, 1, 1, 4, 64).half()
    kv = values64(cache, k, v)
    ro, _ = attend64(q, kv, table, [150], 16)
    o = b200k.cache_attention(q, cache, table, torch.tensor([150], dtype=torch.int32, device="cuda"))
    assert ((o.double() - ro).abs() <= 2.0 ** -9 * kv[1].abs().max() + 2.0 ** -11 * ro.abs()
            + 2.0 ** -25).all()


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 32), (128, 128), (256, 64)])
def test_attention_values_of_many_magnitudes(dim, group):
    # tokens whose values differ by 2^20 in size, constant groups (scale 0) and
    # zeros among them: what each contributes keeps its precision
    g = gen(dim + group + 1)
    n = 230
    cache = b200k.KVCache4.zeros(16, 16, 2, dim, group)
    k = randn(g, 256, 2, dim).half()
    v = randn(g, 256, 2, dim) * torch.exp2(torch.randint(-12, 9, (256, 1, 1), generator=g, device="cuda"))
    v[::5] = v[::5, :, :1]           # constant rows
    v[::7] = 0
    v = v.half()
    b200k.kv_cache_write(cache, k, v, torch.arange(256, device="cuda"))
    table = torch.arange(16, dtype=torch.int32, device="cuda")[None]
    q = randn(g, 1, 1, 8, dim).half()
    kv = values64(cache, k, v)
    ro, _ = attend64(q, kv, table, [n], 16)
    o = b200k.cache_attention(q, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    # each token's share is off by 2^-9 of itself
    z = torch.einsum("hd,jhd->hj", q[0, 0].double(), kv[0][:n].repeat_interleave(4, 1)) * dim ** -0.5
    share = torch.einsum("hj,jhd->hd", torch.softmax(z, -1), kv[1][:n].abs().amax(-1, keepdim=True)
                         .expand(-1, -1, dim).repeat_interleave(4, 1))
    assert ((o[0, 0].double() - ro[0, 0]).abs() <= 2.0 ** -9 * share + 2.0 ** -11 * ro[0, 0].abs()
            + 2.0 ** -25).all()


@pytest.mark.parametrize("group", [32, 128])
def test_attention_only_constant_values(group):
    g = gen(21)
    cache = b200k.KVCache4.zeros(8, 16, 1, 128, group)
    k = randn(g, 128, 1, 128).half()
    v = torch.full((128, 1, 128), 1.5, device="cuda").half()
    b200k.kv_cache_write(cache, k, v, torch.arange(128, device="cuda"))
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    o, lse = b200k.cache_attention(randn(g, 1, 1, 4, 128).half(), cache, table,
                                   torch.tensor([100], dtype=torch.int32, device="cuda"), return_lse=True)
    assert (o.float() - 1.5).abs().max() <= 2.0 ** -10 and lse.isfinite().all()


def test_attention_a_nan_token_is_not_seen_before_its_time():
    # several queries: a token of NaN, written last, must not reach the rows
    # before it (0 * NaN), nor what lies past the length any row
    g = gen(22)
    for dim, group in ((64, 32), (64, 64), (128, 32), (128, 128), (256, 128)):
        cache, k, v = fill(g, 3, 2, 32, dim, group, torch.float16)
        bad = torch.full((1, 2, dim), float("nan"), device="cuda", dtype=torch.float16)
        b200k.kv_cache_write(cache, bad, bad, torch.tensor([69], device="cuda"))
        table = torch.arange(3, dtype=torch.int32, device="cuda")[None]
        q = randn(g, 1, 4, 8, dim).half()
        o = b200k.cache_attention(q, cache, table, torch.tensor([71], dtype=torch.int32, device="cuda"))
        # rows see up to 67, 68, 69, 70
        assert o[0, :2].isfinite().all() and o[0, 2:].isnan().all()
        # a value of NaN alone (its key is a number)
        b200k.kv_cache_write(cache, k[69:70], bad, torch.tensor([69], device="cuda"))
        o = b200k.cache_attention(q, cache, table, torch.tensor([71], dtype=torch.int32, device="cuda"))
        assert o[0, :2].isfinite().all() and o[0, 2:].isnan().all()


def test_attention_under_a_graph():
    g = gen(23)
    cache, k, v = fill(g, 40, 2, 32, 128, 64, torch.bfloat16)
    table, lengths = make_tables(g, [900, 40], 32, 40)
    q = randn(g, 2, 1, 8, 128).bfloat16()
    want = b200k.cache_attention(q, cache, table, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b200k.cache_attention(q, cache, table, lengths)
    for n in ([900, 40], [17, 0], [1, 33]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, b200k.cache_attention(q, cache, table, lengths))
    lengths.copy_(torch.tensor([900, 40], dtype=torch.int32))
    graph.replay()
    assert torch.equal(got, want)


def test_attention_strided_queries_and_another_stream():
    g = gen(16)
    cache, k, v = fill(g, 12, 2, 16, 128, 32, torch.float16)
    table, lengths = make_tables(g, [100, 60], 16, 12)
    big = randn(g, 2, 3, 12, 128).half()
    q = big[:, :, 2:10]                                     # strided heads
    a = b200k.cache_attention(q, cache, table, lengths)
    b = b200k.cache_attention(q.contiguous(), cache, table, lengths)
    assert torch.equal(a, b)
    t = q.transpose(2, 3).contiguous().transpose(2, 3)      # inner stride is not one
    assert torch.equal(b200k.cache_attention(t, cache, table, lengths), b)
    odd = torch.empty(2 * 3 * 8 * 128 + 1, device="cuda", dtype=torch.float16)[1:]
    odd = odd.view(2, 3, 8, 128).copy_(q)                   # rows that are not 16-byte aligned
    assert torch.equal(b200k.cache_attention(odd, cache, table, lengths), b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [b200k.cache_attention(q, cache, table, lengths) for _ in range(5)]
    outs += [b200k.cache_attention(q, cache, table, lengths) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, b) for x in outs)


def test_attention_bad_pages_and_lengths_give_nan():
    g = gen(17)
    cache, k, v = fill(g, 8, 2, 16, 64, 32, torch.float16)
    q = randn(g, 4, 1, 4, 64).half()
    table = torch.tensor([[0, 1], [2, 99], [4, -1], [6, 7]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([20, 20, 20, 33], dtype=torch.int32, device="cuda")
    o, lse = b200k.cache_attention(q, cache, table, lengths, return_lse=True)
    assert o[0].isfinite().all() and lse[0].isfinite().all()
    for i in (1, 2, 3):
        assert o[i].isnan().all() and lse[i].isnan().all()
    # within their first page the second and third are fine, a negative length is empty
    lengths = torch.tensor([-5, 16, 16, 32], dtype=torch.int32, device="cuda")
    o = b200k.cache_attention(q, cache, table, lengths)
    assert (o[0] == 0).all() and o.isfinite().all()


def test_attention_nan_in_a_seen_token_goes_into_the_row():
    g = gen(18)
    cache, k, v = fill(g, 4, 2, 16, 64, 32, torch.float16)
    q = randn(g, 2, 1, 4, 64).half()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    bad = torch.full((1, 2, 64), float("nan"), device="cuda", dtype=torch.float16)
    b200k.kv_cache_write(cache, bad, bad, torch.tensor([20], device="cuda"))
    o = b200k.cache_attention(q, cache, table, torch.tensor([21, 32], dtype=torch.int32, device="cuda"))
    assert o[0].isnan().all() and o[1].isfinite().all()
    o = b200k.cache_attention(q, cache, table, torch.tensor([20, 32], dtype=torch.int32, device="cuda"))
    assert o.isfinite().all()


def test_attention_offsets_past_32_bits():
    # a pool of over 4 GiB, the pages used at its end
    g = gen(19)
    pages, page, hk, dim = 14000, 256, 8, 128
    cache = b200k.KVCache4(torch.empty((pages, hk, page // 16, 16 * (dim + 8 * dim // 32)),
                                       dtype=torch.uint8, device="cuda"), dim, 32)
    assert cache.data.numel() > 1 << 32
    k, v = (randn(g, 2 * page, hk, dim).half() for _ in range(2))
    slots = torch.arange((pages - 2) * page, pages * page, device="cuda")
    b200k.kv_cache_write(cache, k, v, slots)
    rk, rv = b200k.kv_cache_read(cache, slots, dtype=torch.float16)
    check_values(rk, k, 32)
    check_values(rv, v, 32)
    q = randn(g, 1, 1, 16, dim).half()
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    o = b200k.cache_attention(q, cache, table, torch.tensor([500], dtype=torch.int32, device="cuda"))
    order = torch.cat((slots[page:], slots[:page]))[:500]
    kk, vv = b200k.kv_cache_read(cache, order, dtype=torch.float16)
    ro, _ = attend64(q, (kk, vv), torch.zeros((1, 1), dtype=torch.int32, device="cuda"), [500], 512)
    # the reference's values are the float16 readings (2^-11 more in scores and values)
    mag = q.double().norm(dim=-1).max() * kk.double().norm(dim=-1).max() * dim ** -0.5
    assert ((o.double() - ro).abs() <= (2.0 ** -8 + 2.0 ** -11 * mag) * vv.abs().max()).all()


def test_attention_empty_shapes():
    cache = b200k.KVCache4.zeros(2, 16, 2, 64, 32)
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.empty(0, 1, 4, 64, device="cuda", dtype=torch.float16)
    assert b200k.cache_attention(q, cache, torch.empty(0, 3, **i32), torch.empty(0, **i32)).shape == q.shape
    q = torch.ones(3, 1, 4, 64, device="cuda", dtype=torch.float16)
    o = b200k.cache_attention(q, cache, torch.empty(3, 0, **i32), torch.zeros(3, **i32))
    assert (o == 0).all()


# --------------------------------------------------------------------------
# product
def product_case(xd, w, z, s, out_dtype, y):
    """y against sum x s (w - z) in 64 bits; w [n, k], s and z per column already."""
    x, s = xd, s.double()
    ref = x @ (s * (w.double() - z)).T
    a = x.abs() @ (s.abs() * (w.double() + z)).T
    assert y.dtype == out_dtype
    err = (y.double() - ref).abs()
    bound = 2.0 ** -16 * a + HALF_ULP[out_dtype] * ref.abs() + 2.0 ** -25
    assert (err <= bound).all(), (err / bound).max()


def make_weight(g, n, k, group, zeros, stype=torch.float16):
    q = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    groups = -(-k // group)
    s = ((0.5 + torch.rand((n, groups), generator=g, device="cuda")) * 0.02).to(stype)
    z = torch.randint(5, 12, (n, groups), generator=g, device="cuda").to(stype) if zeros else None
    w = b200k.w4_pack(q, s, z, group=group)
    per = s.repeat_interleave(group, 1)[:, :k]
    zp = z.repeat_interleave(group, 1)[:, :k].double() if zeros else torch.full((n, k), 8.0, device="cuda").double()
    return w, q, per, zp


@pytest.mark.parametrize("xt", [torch.float32, torch.float16, torch.bfloat16, torch.int8,
                                torch.float8_e4m3fn])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 128), (2, 17, 129), (3, 100, 31), (5, 250, 1000),
                                   (8, 33, 4096), (9, 64, 320), (1, 4096, 512), (17, 48, 640),
                                   (33, 40, 96), (70, 130, 300)])
def test_product(xt, group, zeros, m, n, k):
    g = gen(m * 31 + n + k)
    w, q, per, zp = make_weight(g, n, k, group, zeros)
    x = randn(g, m, k)
    xs, out = None, xt
    if xt in (torch.int8, torch.float8_e4m3fn):
        xs = torch.rand((m, 1), generator=g, device="cuda") + 0.5
        x = (x * 30).clamp(-127, 127)
        x = (x.round() if xt == torch.int8 else x).to(xt)
        xd = x.double() * xs.double()
        out = torch.bfloat16
    else:
        x = x.to(xt)
        xd = x.double()
    y = b200k.w4_matmul(x, w, x_scale=xs)
    assert y.shape == (m, n)
    product_case(xd, q, zp, per, out, y)
    no_timeouts()


@pytest.mark.parametrize("xgroup,group", [(32, 32), (64, 32), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("m,n,k", [(1, 64, 512), (6, 40, 700), (20, 33, 4100)])
def test_product_group_scales_of_x(xgroup, group, m, n, k):
    g = gen(xgroup + k)
    w, q, per, zp = make_weight(g, n, k, group, True, torch.bfloat16)
    x = (randn(g, m, k) * 40).clamp(-127, 127).round().to(torch.int8)
    xs = torch.rand((m, -(-k // xgroup)), generator=g, device="cuda") + 0.01
    xd = x.double() * xs.double().repeat_interleave(xgroup, 1)[:, :k]
    y = b200k.w4_matmul(x, w, x_scale=xs, out_dtype=torch.float32)
    product_case(xd, q, zp, per, torch.float32, y)


@pytest.mark.parametrize("m,n,k", [(1, 2048, 8192), (4, 20000, 256), (16, 1000, 11008), (2, 300, 28672),
                                   (8, 5003, 4099), (40, 4096, 1024)])
def test_product_large(m, n, k):
    g = gen(n)
    w, q, per, zp = make_weight(g, n, k, 128, False)
    x = randn(g, m, k).bfloat16()
    product_case(x.double(), q, zp, per, torch.bfloat16, b200k.w4_matmul(x, w))


@pytest.mark.parametrize("factor", [1e-30, 1e-7, 1e4, 1e30])
@pytest.mark.parametrize("xt", [torch.float32, torch.bfloat16])
def test_product_magnitudes(factor, xt):
    g = gen(5)
    w, q, per, zp = make_weight(g, 64, 500, 64, True)
    x = (randn(g, 4, 500) * factor).to(xt)
    y = b200k.w4_matmul(x, w, out_dtype=torch.float32)
    ref = x.double() @ (per.double() * (q.double() - zp)).T
    a = x.double().abs() @ (per.double() * (q.double() + zp)).T
    assert ((y.double() - ref).abs() <= 2.0 ** -16 * a).all()


def test_product_rows_with_a_loud_column():
    # one column 2^20 times the others: they keep their precision beside it
    g = gen(6)
    q = torch.randint(0, 16, (32, 256), generator=g, device="cuda", dtype=torch.uint8)
    q[:, 7] = 8                                   # the loud column's weights are zero
    s = torch.full((32, 8), 0.01, device="cuda").half()
    w = b200k.w4_pack(q, s, group=32)
    for xt in (torch.float32, torch.bfloat16, torch.float16):
        x = randn(g, 2, 256) * (2.0 ** -6 if xt == torch.float16 else 1.0)
        x[:, 7] = 2.0 ** 14 if xt == torch.float16 else 2.0 ** 20
        x = x.to(xt)
        y = b200k.w4_matmul(x, w, out_dtype=torch.float32)
        xd, wd = x.double(), s.double().repeat_interleave(32, 1) * (q.double() - 8)
        ref, a = xd @ wd.T, xd.abs() @ (s.double().repeat_interleave(32, 1) * (q.double() + 8)).T
        assert ((y.double() - ref).abs() <= 2.0 ** -20 * a + 1e-12).all()


def test_product_not_finite_rows():
    g = gen(7)
    w, q, per, zp = make_weight(g, 48, 300, 64, False)
    x = randn(g, 5, 300).half()
    x[1, 299], x[3, 0] = float("nan"), float("inf")
    y = b200k.w4_matmul(x, w)
    assert y[1].isnan().all() and y[3].isnan().all()
    rest = [0, 2, 4]
    product_case(x[rest].double(), q, zp, per, torch.float16, y[rest])
    # 8 bits: a NaN scale, or an e4m3 NaN
    x8 = x.nan_to_num(0, 0, 0).to(torch.float8_e4m3fn)
    xs = torch.ones(5, 1, device="cuda")
    xs[2] = float("nan")
    y = b200k.w4_matmul(x8, w, x_scale=xs)
    assert y[2].isnan().all() and y[[0, 1, 3, 4]].isfinite().all()


def test_product_views_dims_and_streams():
    g = gen(8)
    w, q, per, zp = make_weight(g, 96, 264, 32, True)
    x = randn(g, 2, 3, 300).half()[..., 5:269]
    y = b200k.w4_matmul(x, w)
    assert y.shape == (2, 3, 96)
    product_case(x.double().reshape(6, 264), q, zp, per, torch.float16, y.view(6, 96))
    one = b200k.w4_matmul(x[0, 0], w)
    assert one.shape == (96,) and torch.equal(one, b200k.w4_matmul(x[:1, 0], w)[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ys = [b200k.w4_matmul(x, w) for _ in range(4)]
    ys += [b200k.w4_matmul(x, w) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, y) for t in ys)


def test_product_empty():
    w = b200k.w4_pack(torch.zeros(16, 0, dtype=torch.uint8, device="cuda"),
                      torch.zeros(16, 0, dtype=torch.float16, device="cuda"))
    assert (b200k.w4_matmul(torch.ones(2, 0, device="cuda"), w) == 0).all()
    w = b200k.w4_pack(torch.zeros(16, 32, dtype=torch.uint8, device="cuda"),
                      torch.zeros(16, 1, dtype=torch.float16, device="cuda"))
    assert b200k.w4_matmul(torch.ones(0, 32, device="cuda"), w).shape == (0, 16)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k,group", [(40, 300, 32), (16, 128, 128), (5, 70, 64)])
def test_quantised_weights_are_near(zeros, dtype, n, k, group):
    g = gen(n + k)
    wt = (randn(g, n, k) * 0.1 + 0.02).to(dtype)
    w = b200k.w4_quantize(wt, group=group, zeros=zeros)
    x = torch.eye(k, device="cuda")
    got = b200k.w4_matmul(x, w).T.double()               # the weights themselves
    f = wt.double()
    gs = -(-k // group)
    fp = torch.nn.functional.pad(f, (0, gs * group - k)).view(n, gs, group)
    lo, hi = fp.amin(-1).clamp(max=0), fp.amax(-1).clamp(min=0)
    step = (hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7
    step = step.repeat_interleave(group, 1)[:, :k]
    # half a step, and half another where the zero was rounded; 2^-10 for the rounded scale
    assert ((got - f).abs() <= step * ((1.0 if zeros else 0.5) + 15 * 2.0 ** -10)).all()


# --------------------------------------------------------------------------
# refusals
def test_refusals():
    f16 = dict(dtype=torch.float16, device="cuda")
    x, w = torch.ones(4, 64, **f16), torch.ones(64, **f16)
    with pytest.raises(ValueError):
        b200k.add_rmsnorm_quant(x, x[:2], w)
    with pytest.raises(ValueError):
        b200k.rmsnorm_quant(x, w[:32])
    with pytest.raises(ValueError):
        b200k.rmsnorm_quant(x, w, group=48)
    with pytest.raises(TypeError):
        b200k.rmsnorm_quant(x, w.float())
    with pytest.raises(TypeError):
        b200k.rmsnorm_quant(x, w, dtype=torch.uint8)
    cache = b200k.KVCache4.zeros(2, 16, 2, 64)
    k, slots = torch.ones(3, 2, 64, **f16), torch.arange(3, device="cuda")
    for bad in (k[:, :1], k[..., :32], torch.ones(3, 2, 64, device="cuda")):
        with pytest.raises((ValueError, TypeError)):
            b200k.kv_cache_write(cache, bad, bad, slots)
    with pytest.raises(ValueError):
        b200k.kv_cache_write(cache, k, k, slots[:2])
    with pytest.raises(ValueError):
        b200k.kv_cache_write(cache, k, k[:2], slots)
    with pytest.raises(TypeError):
        b200k.kv_cache_write(cache, k, k, slots.int())
    with pytest.raises(TypeError):
        b200k.kv_cache_read(cache, slots, dtype=torch.float32)
    with pytest.raises(ValueError):
        b200k.KVCache4(cache.data, 128, 32)
    with pytest.raises(ValueError):
        b200k.KVCache4(cache.data.transpose(0, 1), 64, 32)
    with pytest.raises(ValueError):
        b200k.KVCache4.zeros(2, 24, 2, 64)
    with pytest.raises(ValueError):
        b200k.KVCache4.zeros(2, 16, 2, 96)
    with pytest.raises(ValueError):
        b200k.KVCache4.zeros(2, 16, 2, 64, 128)
    i32 = dict(dtype=torch.int32, device="cuda")
    q, t, n = torch.ones(1, 1, 4, 64, **f16), torch.zeros(1, 2, **i32), torch.ones(1, **i32)
    for args in ((q[..., :32], t, n), (q[:, :, :3], t, n), (q, t[:0], n), (q, t, n[:0]), (q[0], t, n)):
        with pytest.raises(ValueError):
            b200k.cache_attention(args[0], cache, *args[1:])
    for args in ((q.float(), t, n), (q, t.long(), n), (q, t, n.long())):
        with pytest.raises(TypeError):
            b200k.cache_attention(args[0], cache, *args[1:])
    wt = b200k.w4_quantize(torch.ones(32, 64, **f16), group=32)
    xs = torch.ones(4, 1, device="cuda")
    x8 = x.to(torch.int8)
    with pytest.raises(ValueError):
        b200k.w4_matmul(x[:, :32], wt)
    with pytest.raises(ValueError):
        b200k.w4_matmul(x8, wt)
    with pytest.raises(ValueError):
        b200k.w4_matmul(x, wt, x_scale=xs)
    with pytest.raises(TypeError):
        b200k.w4_matmul(x8, wt, x_scale=xs.half())
    with pytest.raises(ValueError):
        b200k.w4_matmul(x8, wt, x_scale=xs[:2])
    with pytest.raises(ValueError):
        b200k.w4_matmul(x8, wt, x_scale=torch.ones(4, 3, device="cuda"))
    with pytest.raises(TypeError):
        b200k.w4_matmul(x, wt, out_dtype=torch.int8)
    with pytest.raises(ValueError):
        b200k.w4_quantize(torch.ones(32, 64, **f16), group=16)
    with pytest.raises(ValueError):
        b200k.w4_pack(torch.zeros(4, 64, dtype=torch.uint8, device="cuda"), torch.ones(4, 3, **f16), group=32)
    with pytest.raises(ValueError):
        b200k.W4Weight(wt.tiles, wt.scales, wt.zeros, 33, 64)


# --------------------------------------------------------------------------
# the rounding of the cache, where it is hardest
@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("group", [32, 64])
def test_cache_rounding_at_ties_offsets_and_small_ranges(dtype, group):
    g = gen(31)
    rows = []
    for s in (1.0, 0.25, 2.0 ** -9, 8.0):             # exact ties: multiples of s / 2
        rows.append(torch.randint(0, 31, (64, 64), generator=g, device="cuda") * (s / 2))
    rows.append(1000 + 0.01 * randn(g, 64, 64))       # the minimum's rounding exceeds the step
    rows.append(-3000 + 4 * randn(g, 64, 64))
    rows.append(1e-5 * randn(g, 64, 64))              # subnormal steps
    rows.append(6e4 * randn(g, 64, 64).clamp(-1, 1))
    x = torch.cat(rows).to(dtype)[:, None].contiguous()     # [tokens, 1, 64]
    n = x.shape[0]
    cache = b200k.KVCache4.zeros(-(-n // 16), 16, 1, 64, group)
    slots = torch.arange(n, device="cuda")
    b200k.kv_cache_write(cache, x, x, slots)
    for got in values64(cache, x, x):
        t, s, lo = quantise64(x, group)
        want = lo + t.round() * s                     # ties to even, as stored
        got = got[:n].unflatten(-1, (-1, group))
        off = (got - want).abs() > s * 2.0 ** -20
        near = ((t - t.floor() - 0.5).abs() < 2.0 ** -22) & ((t - t.floor() - 0.5) != 0)
        assert not (off & ~near).any()


def test_handles_cannot_be_repointed():
    cache = b200k.KVCache4.zeros(2, 16, 1, 64)
    weight = b200k.w4_quantize(torch.ones((16, 32), device="cuda"), group=32)
    for handle in (cache, weight):
        for name in handle.__slots__:
            with pytest.raises(AttributeError):
                setattr(handle, name, None)
        with pytest.raises(AttributeError):
            handle.other = 1

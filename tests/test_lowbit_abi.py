"""Refusals of the low-precision serving ops that need no GPU: the C entry
points reject bad arguments with a status and a message before any launch,
the Python ones operands that are not on a GPU."""
import pytest
import torch

import b200k
from b200k import _lib as L

FAKE = 1 << 20   # an aligned address that is never read: every call below is refused


def refused(status, word):
    assert status == L.EINVAL, status
    assert word in L.last_error(), L.last_error()


def norm_quant(M=4, N=64, ldx=64, dtype=L.BF16, qt=L.I8, group=0, x=FAKE, r=None, h=None):
    return L.lib.b2k_norm_quant(x, ldx, r, 64, FAKE, h, 64, FAKE, 64, FAKE, 2, M, N, dtype, qt,
                                group, 1e-6, None)


def test_norm_quant_refusals():
    refused(norm_quant(M=-1), "negative")
    refused(norm_quant(qt=L.BF16), "qtype")
    refused(norm_quant(group=48), "group")
    refused(norm_quant(dtype=L.I8), "dtype")
    refused(norm_quant(x=None), "null")
    refused(norm_quant(h=FAKE), "residual")
    refused(norm_quant(ldx=32), "stride")
    assert norm_quant(M=0) == L.OK


def write(D=128, group=32, P=64, Hk=8, data=FAKE, dtype=L.F16, T=4, slots=FAKE):
    return L.lib.b2k_kv4_write(FAKE, 1024, 128, FAKE, 1024, 128, slots, T, data, 4, Hk, P, D, group,
                               dtype, None)


def test_cache_refusals():
    for call in (lambda **k: write(**k),
                 lambda D=128, group=32, P=64, Hk=8, data=FAKE, dtype=L.F16, T=4, slots=FAKE:
                 L.lib.b2k_kv4_read(data, 4, Hk, P, D, group, slots, T, FAKE, FAKE, dtype, None)):
        refused(call(D=96), "head dimension")
        refused(call(group=16), "group")
        refused(call(D=64, group=128), "group")
        refused(call(P=24), "page size")
        refused(call(Hk=0), "heads")
        refused(call(data=FAKE + 8), "aligned")
        refused(call(dtype=L.F32), "dtype")
        refused(call(T=-1), "tokens")
        refused(call(slots=None), "null")
        assert call(T=0) == L.OK


def attention(B=2, Sq=1, H=8, Hk=8, q=FAKE, dtype=L.BF16, table=FAKE):
    return L.lib.b2k_kv4_attention(q, 1024, 1024, 128, FAKE, None, FAKE, 4, Hk, 64, 128, 32, table,
                                   2, FAKE, B, Sq, H, 0.1, 1, dtype, None, 0, None)


def test_attention_refusals():
    refused(attention(B=-1), "negative")
    refused(attention(H=9), "multiple")
    refused(attention(dtype=L.F32), "dtype")
    refused(attention(q=None), "null")
    refused(attention(table=None), "null")
    refused(attention(), "workspace")
    refused(attention(B=1 << 20, Sq=1 << 20), "too many")
    assert attention(B=0) == L.OK
    assert L.lib.b2k_kv4_attention_workspace(-1, 1, 8, 8, 128) == -1


def product(N=64, K=128, M=2, xt=L.BF16, xs=None, xg=0, group=32, yt=L.BF16, y=FAKE, stype=L.F16,
            ldx=128):
    return L.lib.b2k_w4_matmul(FAKE, ldx, xt, xs, 4, xg, FAKE, FAKE, None, stype, group, M, N, K, y,
                               64, yt, None, 0, None)


def test_product_refusals():
    refused(product(N=-1), "negative")
    refused(product(group=16), "group")
    refused(product(stype=L.F32), "scales")
    refused(product(xt=L.I64), "x dtype")
    refused(product(yt=L.I8), "y dtype")
    refused(product(xs=FAKE), "scales")
    refused(product(xt=L.I8), "scales")
    refused(product(xt=L.I8, xs=FAKE, xg=32, group=64), "group")
    refused(product(xt=L.I8, xs=FAKE, xg=48), "group")
    refused(product(y=None), "null")
    refused(product(ldx=64), "stride")
    assert product(M=0) == L.OK
    pack = (FAKE, 128, FAKE, None, 4, 64, 128, 32, L.F16, FAKE, FAKE, None, None)
    for i, bad, word in ((0, None, "null"), (7, 48, "group"), (8, L.F32, "scales"), (5, -1, "negative"),
                         (11, FAKE, "null")):
        refused(L.lib.b2k_w4_pack(*pack[:i], bad, *pack[i + 1:]), word)
    quant = (FAKE, 128, 64, 128, L.F16, 32, L.F16, FAKE, FAKE, None, None)
    for i, bad, word in ((0, None, "null"), (4, L.I8, "dtype"), (5, 48, "group"), (6, L.F32, "scales")):
        refused(L.lib.b2k_w4_quantize(*quant[:i], bad, *quant[i + 1:]), word)


def test_operands_must_be_on_a_gpu():
    x, w = torch.ones(2, 64), torch.ones(64)
    for call in (lambda: b200k.rmsnorm_quant(x, w), lambda: b200k.add_rmsnorm_quant(x, x, w),
                 lambda: b200k.KVCache4(torch.zeros(1, 1, 1, 1280, dtype=torch.uint8), 64, 32),
                 lambda: b200k.w4_quantize(x), lambda: b200k.w4_pack(x.to(torch.uint8), x.half()),
                 lambda: b200k.W4Weight(x, x, None, 2, 64)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: b200k.kv_cache_write(x, x, x, x), lambda: b200k.kv_cache_read(x, x),
                 lambda: b200k.cache_attention(x, x, x, x), lambda: b200k.w4_matmul(x, x)):
        with pytest.raises(TypeError):
            call()



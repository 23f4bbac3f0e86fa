"""The decoder layer of examples/decode_layer.py: 8-bit activations, 4-bit
weights and cache through the package's ops, against the same layer in float32
from the same weights and cache.

Tolerances: int8 rows are off by at most half a step of 1/127 of the row's
maximum, uniformly, which for normal values (maximum about 4 sigma at these
widths) is 4 / 127 / sqrt(12) = 0.9 % of a row in the 2-norm and passes through
a product of independent weights unchanged; bfloat16 intermediates add 2^-9
each.  The stream adds an attention output (one such product, one of
bfloat16) to values of unit size: 2 %.  The block output goes through two int8
rows and SwiGLU, whose product doubles what enters: 5 %.
"""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    path = os.path.join(ROOT, "examples", "decode_layer.py")
    spec = importlib.util.spec_from_file_location("decode_layer", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("batch,heads,kv_heads,dim,group", [(1, 4, 4, 64, 32), (5, 8, 2, 128, 128),
                                                            (12, 16, 2, 64, 64)])
def test_decode_layer(batch, heads, kv_heads, dim, group):
    m = example()
    layer = m.DecoderLayer(batch, 200, hidden=512, ffn=1376, heads=heads, kv_heads=kv_heads, dim=dim,
                           page=16, group=group)
    lengths = torch.arange(batch, device="cuda") * 9 + 3
    layer.prompt(lengths)
    for i in range(3):
        g = torch.Generator(device="cuda").manual_seed(i)
        x = torch.randn((batch, 512), generator=g, device="cuda").bfloat16()
        residual = torch.randn((batch, 512), generator=g, device="cuda").bfloat16()
        h, y = layer.step(x, residual)
        assert torch.equal(layer.lengths.long(), lengths + i + 1)
        rh, ry = layer.reference(x, residual)
        assert m.relative(h, rh) <= 0.02
        assert m.relative(y, ry) <= 0.05


def test_decode_layer_under_a_graph_equals_eager_steps():
    m = example()
    outs = []
    for graphed in (False, True):
        layer = m.DecoderLayer(3, 64, hidden=256, ffn=512, heads=4, kv_heads=2, dim=64, page=16)
        layer.prompt(torch.tensor([1, 20, 40], device="cuda"))
        x = torch.ones((3, 256), device="cuda").bfloat16()
        out = []
        if graphed:
            layer.step(x, x)   # warm-up writes a token; taken back
            layer.lengths -= 1
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                h, y = layer.step(x, x)
            for _ in range(4):
                graph.replay()
                out.append((h.clone(), y.clone()))
        else:
            out = [layer.step(x, x) for _ in range(4)]
        torch.cuda.synchronize()
        outs.append(out)
    for (h0, y0), (h1, y1) in zip(*outs):
        assert torch.equal(h0, h1) and torch.equal(y0, y1)

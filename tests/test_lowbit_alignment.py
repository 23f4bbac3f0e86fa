"""What the kernels of the 4-bit weights copy in bulk has to start at 16 bytes:
the C entry points refuse other addresses before any launch (no GPU needed)."""
import pytest

from b200k import _lib as L

FAKE = 1 << 20   # an aligned address that is never read: every call below is refused


def refused(status, word):
    assert status == L.EINVAL, status
    assert word in L.last_error(), L.last_error()


@pytest.mark.parametrize("off", [1, 2, 4, 8])
@pytest.mark.parametrize("operand", [0, 1, 2])
def test_product_refuses_weights_off_16_bytes(operand, off):
    tiles, scales, zeros = (FAKE + (off if i == operand else 0) for i in range(3))
    refused(L.lib.b2k_w4_matmul(FAKE, 128, L.BF16, None, 1, 0, tiles, scales, zeros, L.F16, 32, 2, 64,
                                128, FAKE, 64, L.BF16, FAKE, 1 << 30, None), "16-byte aligned")


def test_product_refuses_a_workspace_off_16_bytes():
    need = L.lib.b2k_w4_matmul_workspace(1, 64, 14336, 32, L.BF16)
    assert need > 0
    refused(L.lib.b2k_w4_matmul(FAKE, 14336, L.BF16, None, 1, 0, FAKE, FAKE, None, L.F16, 32, 1, 64,
                                14336, FAKE, 64, L.BF16, FAKE + 8, need, None), "workspace")


@pytest.mark.parametrize("off", [1, 2, 4, 8])
@pytest.mark.parametrize("operand", [0, 1, 2])
def test_pack_and_quantize_refuse_outputs_off_16_bytes(operand, off):
    outs = [FAKE + (off if i == operand else 0) for i in range(3)]
    refused(L.lib.b2k_w4_pack(FAKE, 128, FAKE, FAKE, 4, 64, 128, 32, L.F16, *outs, None),
            "16-byte aligned")
    refused(L.lib.b2k_w4_quantize(FAKE, 128, 64, 128, L.F16, 32, L.F16, *outs, None),
            "16-byte aligned")

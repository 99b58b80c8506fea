"""Outputs that a caller gives and that lie over the input are refused."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_outputs_over_the_input():
    import cswap_b200 as cs
    space = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    x = space[1024:2048].view(torch.float32)
    need = cs.q8_bytes(256)
    assert need == 264
    for at in (1024 - 256, 1024, 1536, 2032):
        with pytest.raises(ValueError, match="overlaps"):
            cs.q8_compress(x, out=space[at:at + 272])
    for at in (1024 - 272, 2048):
        cs.q8_compress(x, out=space[at:at + 272])
    packed = space[:need]
    for at in (0, 256):
        with pytest.raises(ValueError, match="overlaps"):
            cs.q8_decompress(packed, 256, out=space[at:at + 512].view(torch.float16))
    cs.q8_decompress(packed, 256, out=space[272:272 + 512].view(torch.float16))
    cs.q8_compress(space[2560:3584].view(torch.float32), out=space[1024:])  # longer than it needs to be
    cs.q8_compress(x[:0], out=space[1024:1040])  # nothing is read
    torch.cuda.synchronize()

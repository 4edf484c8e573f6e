"""CPU: checkpoints of 8-bit moments over the whole range that their documentation names."""
import torch

from alphazero_amd.optim import _decode, _encode


def test_eight_bit_roots_survive_their_squares():
    """A checkpoint holds exp_avg_sq, the squares of the roots, in float32: exact while they are normal numbers (8 bits of
    mantissa), so every root from 2^-63 on comes back as the same code, beside any larger ones."""
    codes = torch.arange(1, 127, dtype=torch.uint8).view(torch.float8_e4m3fn)
    block = torch.zeros(256, dtype=torch.float8_e4m3fn)
    for exponent in (-80, -70, -60, -54, -40, 0, 50):
        for top in (1, 8, 56, 64, 126):
            held = block.clone()
            held[:top] = codes[:top]
            r = _decode(held, torch.tensor([2.0 ** exponent]))
            back = _decode(*_encode(r.square().sqrt(), True))
            kept = (r >= 2.0 ** -63) | (r == 0)
            assert torch.equal(back[kept], r[kept]), (exponent, top)

"""How far microscaled values may be off, as odie_amd.microscale states it: a quarter of themselves from a quarter of their
block's largest on (which is one scale at least), and below one scale a quarter of the scale."""
import torch

from microscale64 import quantize64, values64


def test_bound_of_a_value():
    worst = 0.0
    for largest in torch.arange(4.0, 8.0, 1 / 64):
        # every 64th of a scale up to the block's largest, both signs, 31 a block beside it
        values = torch.arange(0.0, float(largest) + 1e-9, 1 / 64)
        values = torch.cat((values, -values))
        values = torch.cat((values, values.new_zeros(-len(values) % 31))).view(-1, 31)
        rows = torch.cat((values, largest.expand(len(values), 1)), 1)
        codes, scales = quantize64(rows)
        assert (scales[:, 0] == 127).all()
        off = (values64(codes, scales, 32) - rows.double()).abs()
        size = rows.double().abs()
        from_quarter = size >= float(largest) / 4
        assert (off[from_quarter] <= size[from_quarter] / 4).all()
        assert (off[size < 1] <= 0.25).all()
        worst = max(worst, float((off / size.clamp(min=1e-9))[size >= float(largest) / 6].max()))
    # 0.75 scales, between a sixth and a quarter of a largest of 4, go to the even code, 1
    assert worst == 1 / 3

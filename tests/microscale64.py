"""The microscaled format restated on numpy's side of things: exact arithmetic in 64 bits, block by block."""
import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize64(x):
    """codes uint8 [N, 16 * blocks] and scales uint8 [N, blocks rounded up to 4] of x [N, width], on the CPU."""
    x = x.detach().cpu().double()
    n, width = x.shape
    blocks = (width + 31) // 32
    rows = torch.zeros(n, blocks * 32, dtype=torch.float64)
    rows[:, :width] = x
    rows = rows.view(n, blocks, 32)
    most = rows.abs().amax(2)
    broken = ~rows.isfinite().all(2)
    exponent = torch.floor(torch.log2(most.clamp(min=2.0 ** -149))) - 2
    # log2 rounds: the largest power of two that is not above the magnitude, exactly
    exponent += (torch.exp2(exponent + 3) <= most).double() - (torch.exp2(exponent + 2) > most).double()
    exponent = torch.where(most == 0, -127.0, exponent).clamp(-127, 127)
    size = rows.abs() / torch.exp2(exponent)[..., None]
    distance = (size[..., None] - torch.tensor(MAGNITUDES, dtype=torch.float64)).abs()
    # the nearest; of two as near the even code
    order = distance * 2 + (torch.arange(8) % 2) * 1e-9
    code = order.argmin(-1) + 8 * torch.signbit(rows)
    code = torch.where(broken[..., None], 0, code)
    scales = torch.zeros(n, (blocks + 3) // 4 * 4, dtype=torch.uint8)
    scales[:, :blocks] = torch.where(broken, 255, exponent + 127).to(torch.uint8)
    code = code.view(n, -1, 2)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scales


def values64(codes, scales, width):
    """The values [N, width] that codes and scales stand for, in 64 bits on their device."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=torch.float64, device=codes.device)
    scale = torch.exp2(scales.double() - 127)
    scale = torch.where(scales == 255, float('nan'), scale).repeat_interleave(32, -1)[..., :code.shape[-1]]
    return (table[code] * scale)[..., :width]

"""Plain statements in 64 bits of the dense layers whose rows are held in eight bits, for the tests."""
import numpy as np
import torch

GROUP = 16
LARGEST_SCALE = 576.0


def int8_rows(y):
    """(codes, scales) of float64 rows."""
    most = y.abs().amax(1, keepdim=True)
    codes = torch.where(most > 0, torch.round(127 * y / torch.where(most > 0, most, 1.0)), 0.0)
    return codes, most[:, 0] / 127


def kept_scales():
    """All scales by their bytes, as whole numbers of 2^-24."""
    return [(b & 7) if b < 8 else (8 + (b & 7)) << ((b >> 3) - 1) for b in range(255)]


def keep(x):
    """(codes int64 [N,C], bytes int64 [N,C/16]) of finite fp16 rows, in whole numbers of 2^-24: no rounding but the codes' own."""
    scales = np.array(kept_scales(), dtype=np.int64)
    units = (x.cpu().double() * 2.0 ** 24).long().numpy().reshape(x.shape[0], -1, GROUP)
    byte = np.searchsorted(127 * scales, np.abs(units).max(2), side="left")
    s = np.maximum(scales[byte], 1)[:, :, None]
    q, r = np.divmod(np.abs(units), s)
    q = q + ((2 * r > s) | ((2 * r == s) & (q % 2 == 1)))
    q = np.minimum(q, np.where(byte == 249, 113, 127)[:, :, None])
    return torch.from_numpy((np.sign(units) * q).reshape(x.shape)), torch.from_numpy(byte)


def kept(x):
    """float64: what the kept form of finite fp16 rows stands for."""
    codes, byte = keep(x)
    scales = torch.tensor(kept_scales(), dtype=torch.float64)[byte] * 2.0 ** -24
    return (codes.double().view(x.shape[0], -1, GROUP) * scales.unsqueeze(2)).view(x.shape).to(x.device)


def gelu(x):
    return x * torch.special.ndtr(x)


def gelu_slope(x):
    return torch.special.ndtr(x) + x * torch.exp(-x * x / 2) / np.sqrt(2 * np.pi)

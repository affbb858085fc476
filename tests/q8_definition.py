"""The 8-bit format from its definition, in 64 bits and without the package: what the tests of it compare with."""
import numpy as np
import torch

LOWEST = -117


def code_values():
    """The 256 numbers of e4m3: sign, 4 bits of exponent (bias 7), 3 of mantissa; no infinities, 0x7f and 0xff are NaN."""
    v = np.empty(256)
    for i in range(256):
        s, e, m = -1.0 if i & 128 else 1.0, (i >> 3) & 15, i & 7
        v[i] = np.nan if (i & 127) == 127 else s * (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return v


_POSITIVE = code_values()[:127]   # rising with the code


def nearest_code(z):
    """The code's number nearest to z (|z| <= 448), of two equally near ones that with the even code."""
    a = np.abs(z)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    down, up = a - _POSITIVE[lo], _POSITIVE[hi] - a
    pick = np.where(down < up, lo, np.where(up < down, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.copysign(_POSITIVE[pick], z)


def define(x):
    """float64 [R, C] -> numbers of the codes [R, C], scales [R, ceil(C / 128)]."""
    codes, scales = np.empty_like(x), []
    for b in range(0, x.shape[1], 128):
        y = x[:, b:b + 128]
        fine = np.isfinite(y)
        e = np.empty(len(y), dtype=np.int64)
        for r, amax in enumerate(np.abs(np.where(fine, y, 0)).max(1)):
            k = LOWEST
            while amax > 448 * 2.0 ** k:
                k += 1
            e[r] = k
        s = np.exp2(e.astype(np.float64))[:, None]
        codes[:, b:b + 128] = np.where(fine, nearest_code(np.where(fine, y, 0) / s), np.nan)
        scales.append(s)
    return codes, np.concatenate(scales, 1)


def decode(codes, scale):
    """Numbers (float64 numpy) of codes and scales given as tensors of the 8-bit types; from their bits."""
    v = code_values()[codes.cpu().view(torch.uint8).numpy()]
    b = scale.cpu().view(torch.uint8).numpy().astype(np.float64)
    s = np.where(b == 255, np.nan, np.exp2(b - 127))
    return v * np.repeat(s, 128, axis=-1)[..., :v.shape[-1]]


def hard_rows(rows, c, seed):
    """f32 rows of very different sizes; among them zeros, what is not finite, subnormals, ties and the borders of a scale."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, c, generator=g) * torch.exp2(torch.randint(-12, 13, (rows, 1), generator=g).float())
    x[0] = 0.0
    x[1, ::3] = 0.0
    x[2] = 2.0 ** -130 * torch.randn(c, generator=g)
    x[3] = torch.finfo(torch.float32).max * torch.rand(c, generator=g)
    x[4, c // 2] = float('nan')
    x[5, 0], x[5, c - 1] = float('inf'), -float('inf')
    x[6] = float('nan')
    x[7] = torch.linspace(-448, 448, c)
    x[7, 0] = 448.0                                        # the largest that scale 1 holds
    x[8] = x[7]
    x[8, 0] = 448.0 + 2.0 ** -15                           # and a step more
    x[9] = 17.0 + torch.arange(c) % 16                     # ties: between 16 and 18, 18 and 20, ...
    x[9, 0] = 448.0
    x[10] = 2.0 ** -10 * (torch.arange(c) % 64).float()    # ties of the smallest codes
    x[10, 0] = 448.0
    x[11] = -0.0
    x[12] = 2.0 ** -126
    return x

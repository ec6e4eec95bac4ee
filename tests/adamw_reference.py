"""The step of optim.AdamW written out in torch operations on the host, for the tests: fp32, one rounding for every operation, so
that a kernel that does the same operations gives the same bits."""
import math

import torch

BLOCK = 256


def mixed(x):
    x = ((x ^ (x >> 16)) * 0x6C8E9CF5) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x35297A4D) & 0xFFFFFFFF
    return x ^ (x >> 16)


def decode(codes, scale, n):
    """float64 values of e4m3 codes (uint8, whole blocks) with biased power-of-two scales (uint8)."""
    v = codes.view(torch.float8_e4m3fn).double().view(-1, BLOCK) * torch.ldexp(torch.ones(scale.numel(), dtype=torch.float64),
                                                                               scale.to(torch.int32) - 127)[:, None]
    return v.view(-1)[:n]


def encode(x, r16, keep_nonzero):
    """(codes, scales) of fp32 x: block maxima brought into [128, 256), then each value to one of its two neighbouring codes."""
    n = x.numel()
    blocks = -(-n // BLOCK)
    pad = lambda t: torch.nn.functional.pad(t, (0, blocks * BLOCK - n))  # noqa: E731
    codes, scales = torch.zeros(blocks * BLOCK, dtype=torch.uint8), torch.zeros(blocks, dtype=torch.uint8)
    fine = torch.isfinite(x)
    mag = pad(torch.where(fine, x.abs(), torch.zeros_like(x))).view(blocks, BLOCK)
    for b in range(blocks):
        top = mag[b].max().item()
        e = max(1, (math.frexp(top)[1] - 1 + 127 if top >= 2.0**-126 else 0) - 7)
        scales[b] = e
    inv = torch.ldexp(torch.ones(blocks), 127 - scales.to(torch.int32)).float()
    a = (mag * inv[:, None]).view(-1)[:n]
    # the 20 bits that are dropped, plus the random ones, carry into the code or do not; below 2^-6 codes are 2^-9 apart
    low = a < 2.0**-6
    c = torch.where(low, ((a.double() * 2.0**29).long() + (r16 << 4)) >> 20, ((a.view(torch.int32).long() + (r16 << 4)) >> 20) - 960)
    if keep_nonzero:
        c = torch.where((c == 0) & (x > 0), torch.ones_like(c), c)
    c = torch.where(fine, c | ((x < 0).long() << 7), torch.full_like(c, 127))
    codes[:n] = c.to(torch.uint8)
    return codes, scales


class Reference:
    """One parameter tensor on the host."""

    def __init__(self, p, index, bits, seed=0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, wd=1e-2):
        self.p, self.index, self.bits, self.seed = p.detach().cpu().clone(), index, bits, seed
        self.lr, self.betas, self.eps, self.wd, self.t = lr, betas, eps, wd, 0
        n = p.numel()
        self.m, self.v = torch.zeros(n), torch.zeros(n)
        if bits == 8:
            z = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.uint8), torch.ones(-(-n // BLOCK), dtype=torch.uint8)
            self.mc, self.ms, self.vc, self.vs = z[0], z[1], z[0].clone(), z[1].clone()

    def step(self, g, clip=1.0):
        self.t += 1
        (b1, b2), t, n = self.betas, self.t, self.p.numel()
        g = g.detach().cpu().reshape(-1).float() * torch.tensor(clip, dtype=torch.float32)
        p = self.p.reshape(-1).float()
        if self.bits == 8:  # (exact: a code times a power of two; subnormal products round once, as in fp32)
            self.m = decode(self.mc, self.ms, n).float()
            r = decode(self.vc, self.vs, n).float()
            self.v = r * r
        f = lambda x: torch.tensor(x, dtype=torch.float64).float()  # noqa: E731
        self.m = self.m * f(b1) + g * f(1 - b1)
        self.v = self.v * f(b2) + (g * g) * f(1 - b2)
        r = self.v.double().sqrt().float()  # (rounded once; torch's own fp32 root on the host is up to a step off)
        denom = r * f(1.0 / math.sqrt(1 - b2**t)) + f(self.eps)
        p = p * f(1 - self.lr * self.wd) - (self.m / denom) * f(self.lr / (1 - b1**t))
        self.p = p.to(self.p.dtype).view(self.p.shape)
        if self.bits == 8:
            key = int(mixed(torch.tensor((self.seed + 0x9E3779B9 * t + 0x632BE5AB * self.index) & 0xFFFFFFFF)))
            h = mixed(torch.arange(n) ^ key)
            self.mc, self.ms = encode(self.m, h & 0xFFFF, False)
            self.vc, self.vs = encode(r, h >> 16, True)

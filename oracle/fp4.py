"""The MXFP4 KV-cache format from its definition, in 64 bits on the CPU. TEST INFRASTRUCTURE ONLY.

The reference has no 4-bit cache; the format is OCP microscaling with E2M1 elements (two to a byte, element 2i in the
low nibble) and one E8M0 byte per 32 consecutive elements of a row. `quantize` works on float64
copies of the rows and compares every element with all eight magnitudes; `dequantize` decodes sign, exponent and
mantissa bits. `attention` is softmax attention over values so decoded, sequence by sequence, with the sum of |p v| that
rounding bounds are multiples of.
"""

from __future__ import annotations

import math

import torch

FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
BLOCK = 32


def e2m1_value(code: int) -> float:
    """The real number a 4-bit code stands for: sign, 2 exponent bits (bias 1, 0 subnormal), 1 mantissa bit."""
    e, m = (code >> 1) & 3, code & 1
    mag = m * 0.5 if e == 0 else (1 + 0.5 * m) * 2.0 ** (e - 1)
    return -mag if code & 8 else mag


def power_of_two(e: torch.Tensor) -> torch.Tensor:
    """2^e in float64 from its bits (torch.ldexp and exp2 may be off by an ulp on a GPU)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


MAGNITUDES = torch.tensor([e2m1_value(c) for c in range(8)], dtype=torch.float64)


def largest(dtype: torch.dtype) -> float:
    """The largest value that the format and a row's type both hold."""
    return 1.5 * 2.0 ** (15 if dtype == torch.float16 else 127)


def quantize(x: torch.Tensor, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [..., D] of `dtype` (x's own unless given) as (uint8 [..., D / 2], uint8 [..., D / 32])."""
    top = largest(dtype or x.dtype)
    x = x.detach().cpu().double().clamp(-top, top)
    b = x.unflatten(-1, (-1, BLOCK))
    nan = b.isnan().any(-1, keepdim=True)
    a = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(torch.where(nan, 1.0, a))  # a = m 2^e, m in [0.5, 1); mantissa 2 m, exponent e - 1
    e = torch.where(a == 0, torch.tensor(-200, dtype=e.dtype), e - 1 - 2 + (2 * m >= 1.75).to(e.dtype))
    s = (e + 127).clamp(min=2)
    y = b / power_of_two(s - 127)
    d = (y.abs().unsqueeze(-1) - MAGNITUDES).abs()
    near = d == d.amin(-1, keepdim=True)
    # of two magnitudes at the same distance, the one with the even code
    order = torch.tensor([0, 9, 2, 11, 4, 13, 6, 15])
    code = torch.where(near, order, 100).argmin(-1).to(torch.uint8)
    code = (code | (torch.signbit(x).unflatten(-1, (-1, BLOCK)).to(torch.uint8) << 3)).flatten(-2)
    s = torch.where(nan, torch.tensor(255, dtype=s.dtype), s).to(torch.uint8).squeeze(-1)
    return code[..., 0::2] | (code[..., 1::2] << 4), s


def dequantize(code: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """float64 values [..., D] of bytes [..., D / 2] and E8M0 bytes [..., D / 32] (uint8 views; on code's device)."""
    table = torch.tensor([e2m1_value(c) for c in range(16)], dtype=torch.float64, device=code.device)
    x = torch.stack((table[(code & 15).long()], table[(code >> 4).long()]), dim=-1).flatten(-2)
    f = power_of_two(s.int() - 127)
    return x * torch.where(s == 255, math.nan, f).repeat_interleave(BLOCK, dim=-1)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, block_tables: torch.Tensor, seq_lens: list[int],
              query_lens: list[int], scale: float) -> tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """(out, sum_j p_j |v_j|) [T, H, D] in 64 bits: q [T, H, D]; k, v caches [blocks, BS, Hkv, D] of float64 values.
    Table entries outside the pool are empty pages; rows that see no key give zeros."""
    T, H, D = q.shape
    nb, bs, Hkv, _ = k.shape
    out = torch.zeros((T, H, D), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    t0 = 0
    for i, (n, total) in enumerate(zip(query_lens, seq_lens)):
        if n == 0 or total <= 0:
            t0 += n
            continue
        ids = block_tables[i, : -(-total // bs)]
        there = ((ids >= 0) & (ids < nb)).repeat_interleave(bs)[:total]
        ids = ids.clamp(0, nb - 1)
        kk, vv = (x[ids].flatten(0, 1)[:total].masked_fill(~there[:, None, None], 0.0) for x in (k, v))
        pos = total - n + torch.arange(n, device=q.device)
        seen = (torch.arange(total, device=q.device) <= pos[:, None]) & there
        for h in range(H):
            g = h // (H // Hkv)
            w = (q[t0 : t0 + n, h].double() @ kk[:, g].t().contiguous()) * scale
            w = w.masked_fill(~seen, -math.inf)
            top = w.amax(-1, keepdim=True)
            p = torch.exp(w - top.masked_fill(top == -math.inf, 0.0))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            out[t0 : t0 + n, h] = p @ vv[:, g].contiguous()
            mag[t0 : t0 + n, h] = p @ vv[:, g].abs().contiguous()
        t0 += n
    return out, mag

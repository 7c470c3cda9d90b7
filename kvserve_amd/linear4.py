"""Products with weights held in 4 bits (kvh_linear4): a decode step streams its weights first of all, and these are
a quarter of the bytes."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from kvserve_amd import _lib
from kvserve_amd.attention import _calls, _current, _require, _stream_handle

GROUPS = (32, 64, 128)


@dataclass(frozen=True, eq=False)
class Weight4:
    """A weight [n, k] in 4 bits, laid out for `linear4` (kvh_linear4): W[r][c] = scale (code - zero), with a scale and
    a zero point for every row and `group` consecutive columns. Made by `pack` or `quantize_weight4`."""

    codes: torch.Tensor  # int32 [n / 16, k / 128, 256]
    scales: torch.Tensor  # int32 [n / 16, k / 128 * 128 / group, 16]
    shape: tuple[int, int]  # (n, k)
    group: int
    dtype: torch.dtype  # of the scales, and of x and y

    def __post_init__(self):
        n, k = self.shape
        _require(self.group in GROUPS and n >= 0 and k > 0 and k % self.group == 0, f"no groups of {self.group} in {self.shape}")
        tiles, blocks = -(-n // 16), -(-k // 128)
        for name, t, want in (("codes", self.codes, (tiles, blocks, 256)),
                              ("scales", self.scales, (tiles, blocks * (128 // self.group), 16))):  # fmt: skip
            _require(t.dtype == torch.int32 and t.shape == want and t.is_contiguous(), f"{name} must be contiguous int32 {want}")

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @classmethod
    def pack(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None) -> Weight4:
        """codes: uint8 [n, k / 2], element 2i in the low half of byte i; scales: fp16 or bf16 [n, k / group]; zeros: uint8
        [n, k / group] in 0 .. 15 (None: 8). Checks the zero points, so it waits for the device."""
        _require(codes.dtype == torch.uint8 and codes.dim() == 2, "codes must be uint8 [n, k / 2]")
        _require(scales.dtype in (torch.bfloat16, torch.float16), f"scales must be bf16 or fp16, not {scales.dtype}")
        n, k = codes.shape[0], 2 * codes.shape[1]
        _require(scales.dim() == 2 and scales.shape[0] == n and scales.shape[1] > 0 and k % scales.shape[1] == 0,
                 "scales must be [n, k / group]")  # fmt: skip
        group = k // scales.shape[1]
        _require(group in GROUPS, f"groups must be of {GROUPS} columns, not {group}")
        _require(scales.device == codes.device, "codes and scales are on different devices")
        if zeros is None:
            zeros = torch.full(scales.shape, 8, dtype=torch.uint8, device=codes.device)
        _require(zeros.dtype == torch.uint8 and zeros.shape == scales.shape and zeros.device == codes.device,
                 "zeros must be uint8 of the scales' shape and device")  # fmt: skip
        _require(not bool((zeros > 15).any()), "zeros must be 0 .. 15")
        tiles, blocks = -(-n // 16), -(-k // 128)
        packed = torch.zeros((tiles, blocks, 4, 16, 4), dtype=torch.int32, device=codes.device)
        for t in range(0, tiles, 64):  # a part of the rows at a time
            part = codes[16 * t : 16 * (t + 64)]
            full = torch.zeros((16 * (min(t + 64, tiles) - t), 64 * blocks), dtype=torch.uint8, device=codes.device)
            full[: len(part), : k // 2] = part
            # byte p of a lane's four: elements 2p (low half) and 2p + 1, for bits 4p and 16 + 4p of the dword
            b = full.view(-1, 16, blocks, 4, 4, 4).int()  # tile, row, block, u, j, p
            p = 4 * torch.arange(4, dtype=torch.int32, device=codes.device)
            d = ((b & 15) << p) | ((b >> 4) << (p + 16))
            packed[t : t + 64] = d.sum(-1, dtype=torch.int32).permute(0, 2, 4, 1, 3)  # disjoint bits
        # the scale in the low half of a dword, 16 + zero in the high one, both as scales' type
        pair = torch.stack((scales, (zeros.int() + 16).to(scales.dtype)), dim=-1).contiguous().view(torch.int32)[..., 0]
        full = torch.zeros((16 * tiles, blocks * (128 // group)), dtype=torch.int32, device=codes.device)
        full[:n, : k // group] = pair
        return cls(packed.view(tiles, blocks, 256), full.view(tiles, 16, full.shape[1]).transpose(1, 2).contiguous(), (n, k), group,
                   scales.dtype)  # fmt: skip

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weight [n, k], computed in fp32 and rounded to `dtype`."""
        (n, k), (tiles, blocks) = self.shape, self.codes.shape[:2]
        d = self.codes.view(tiles, blocks, 4, 16, 4).permute(0, 3, 1, 4, 2)[..., None]  # tile, row, block, u, j
        p = 4 * torch.arange(4, dtype=torch.int32, device=self.device)
        q = torch.stack(((d >> p) & 15, (d >> (p + 16)) & 15), dim=-1).reshape(16 * tiles, 128 * blocks)[:n, :k]
        pair = self.scales.transpose(1, 2).reshape(16 * tiles, self.scales.shape[1])[:n, : k // self.group]
        s, z = (half.to(torch.int16).view(self.dtype).float() for half in (pair, pair >> 16))
        return ((q.view(n, k // self.group, self.group) - (z - 16)[..., None]) * s[..., None]).view(n, k).to(dtype)

    def to(self, device: torch.device | str) -> Weight4:
        return Weight4(self.codes.to(device), self.scales.to(device), self.shape, self.group, self.dtype)


def quantize_weight4(weight: torch.Tensor, group: int = 128) -> Weight4:
    """A bf16 or fp16 weight [n, k] rounded to the nearest of 16 evenly spaced values over each group's range, zero among
    them. k a multiple of `group`; a group's range below 15 * 2^123, which is checked, so it waits for the device."""
    _require(weight.dim() == 2 and weight.dtype in (torch.bfloat16, torch.float16), "weight must be bf16 or fp16 [n, k]")
    _require(group in GROUPS and weight.shape[1] % group == 0 and weight.shape[1] > 0,
             f"groups must be of {GROUPS} columns that divide k (got {group}, k = {weight.shape[1]})")  # fmt: skip
    codes, scales, zeros = [], [], []
    for part in weight.split(1024):
        w = part.float().unflatten(1, (weight.shape[1] // group, group))
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).to(weight.dtype)
        # what kvh_linear4 takes; a NaN is in its group's range
        _require(bool((s < 2.0**123).all()), "weight must be finite, its groups' ranges below 15 * 2^123")
        step = s.float().masked_fill(s == 0, 1.0)
        z = (-lo / step).round().clamp(0, 15)
        q = ((w / step[..., None]).round() + z[..., None]).clamp(0, 15).to(torch.uint8).flatten(1)
        codes.append(q[:, 0::2] | (q[:, 1::2] << 4))
        scales.append(s)
        zeros.append(z.to(torch.uint8))
    return Weight4.pack(torch.cat(codes), torch.cat(scales), torch.cat(zeros))


def _product(x: torch.Tensor, weight: Weight4, silu_mul: bool, out: torch.Tensor | None) -> torch.Tensor:
    n, k = weight.shape
    calls = _calls()
    if calls is not None:
        r = calls.linear4(x, weight.codes, weight.scales, n, k, weight.group, _lib.KVH_DTYPE.get(weight.dtype), silu_mul, out)
        if type(r) is int:
            _lib.check(r, "kvh_linear4")
        if r is not None:
            return r
    _require(x.dim() == 2 and x.shape[1] == k and x.stride(-1) == 1, f"x must be [m, {k}] with a contiguous last dim")
    _require(x.dtype == weight.dtype, f"x is {x.dtype}, the weight's scales are {weight.dtype}")
    _require(x.is_cuda, "x must be on a HIP device")
    if weight.codes.get_device() != x.get_device() or weight.scales.get_device() != x.get_device():
        raise ValueError(f"the weight must be on x's device {x.device} (got {weight.device})")
    _require(not silu_mul or n % 32 == 0, f"the gated product needs whole 16s of gate and up rows, not {n} rows")
    m, cols = x.shape[0], n // 2 if silu_mul else n
    if out is None:
        out = torch.empty((m, cols), dtype=x.dtype, device=x.device)
    _require(out.shape == (m, cols) and out.dtype == x.dtype and out.stride(-1) == 1 and out.device == x.device,
             f"out must be [{m}, {cols}] of x's dtype and device with a contiguous last dim")  # fmt: skip
    lib = _lib.load()
    need = lib.kvh_linear4_workspace_size(m, n, k, int(silu_mul))
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    # the stride of a lone row may be anything
    x_stride, y_stride = (x.stride(0), out.stride(0)) if m > 1 else (k, -(-cols // 4) * 4)
    with _current(x.get_device()):
        st = lib.kvh_linear4(x.data_ptr(), x_stride, weight.codes.data_ptr(), weight.scales.data_ptr(), out.data_ptr(),
                             y_stride, m, n, k, weight.group, int(silu_mul), _lib.KVH_DTYPE[x.dtype],
                             ws.data_ptr() if ws is not None else None, need, _stream_handle(x.device))  # fmt: skip
    _lib.check(st, "kvh_linear4")
    return out


def linear4(x: torch.Tensor, weight: Weight4, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [m, k] @ weight.T as [m, n] (in `out` if given, which must not overlap x): bf16 or fp16, sums in fp32, rounded once. Up to
    1048560 rows; an infinity in a row makes its result NaN. Forward only: the output carries no gradient."""
    return _product(x, weight, False, out)


def linear4_silu_mul(x: torch.Tensor, weight: Weight4, out: torch.Tensor | None = None) -> torch.Tensor:
    """SiLU(x @ gate.T) * (x @ up.T) as [m, n / 2] of a weight whose first n / 2 rows are the gate's (n a multiple of 32);
    rounded once, behind the product. Otherwise as linear4."""
    return _product(x, weight, True, out)

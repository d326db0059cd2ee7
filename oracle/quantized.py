"""8-bit caches with power-of-two block scales, in 64 bits on the CPU: the
quantising append and the route commit as their definitions say, row by row."""

from __future__ import annotations

import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def grid(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """x (float64) rounded to the codes' values, to nearest, ties to even."""
    if dtype == torch.int8:
        return torch.nan_to_num(torch.round(x), nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127, 127)
    _, e = torch.frexp(x)
    step = torch.exp2(torch.clamp(e - 1, min=-6).double() - 3)
    y = (torch.round(x / step) * step).clamp(-448, 448)
    return torch.where(torch.isinf(x), torch.sign(x) * 448.0, y)


def least_scale(amax: float, dtype: torch.dtype) -> float:
    """The least power of two s >= 2^-126 with amax <= TOP * s."""
    s = 2.0 ** -126
    if amax > 0:
        s = max(s, 2.0 ** math.floor(math.log2(amax / TOP[dtype]) - 1))
    while amax > TOP[dtype] * s:
        s *= 2
    return s


class Block8Cache:
    """One layer's values: ``codes`` [pages, 2, Hkv, page_size, D] float64 and
    ``scales`` [pages, 2, Hkv] float64."""

    def __init__(self, layer: torch.Tensor, scales: torch.Tensor, kv_layout: str) -> None:
        self.dtype = layer.dtype
        self.layout = kv_layout
        c = layer.double()
        self.codes = (c.transpose(-2, -3) if kv_layout == "NHD" else c).clone()
        self.scales = scales.double().clone()
        self.page_size = self.codes.shape[3]

    def layer(self) -> torch.Tensor:
        """Codes in the layer's own shape, float64."""
        return self.codes.transpose(-2, -3) if self.layout == "NHD" else self.codes

    def append(self, k, v, append_indptr, kv_indptr, kv_indices, kv_lens) -> None:
        for b, n in enumerate(kv_lens):
            rows = append_indptr[b + 1] - append_indptr[b]
            lo = n - rows
            for lp in range(max(lo, 0) // self.page_size, -(-n // self.page_size)):
                page = int(kv_indices[kv_indptr[b] + lp])
                at = [p for p in range(lp * self.page_size, (lp + 1) * self.page_size) if max(lo, 0) <= p < n]
                if not at:
                    continue
                off = [p - lp * self.page_size for p in at]
                src = [append_indptr[b] + p - lo for p in at]
                for kv, x in ((0, k), (1, v)):
                    for h in range(self.codes.shape[2]):
                        new = x[src, h].double()
                        fin = new[torch.isfinite(new)].abs()
                        s = least_scale(float(fin.max()) if fin.numel() else 0.0, self.dtype)
                        if off[0] > 0:
                            was = float(self.scales[page, kv, h])
                            s = max(s, was)
                            if s != was:
                                old = self.codes[page, kv, h, :off[0]]
                                self.codes[page, kv, h, :off[0]] = grid(old * (was / s), self.dtype)
                        self.codes[page, kv, h, off] = grid(new / s, self.dtype)
                        self.scales[page, kv, h] = s

    def commit(self, src_pos, dst_pos, item_indptr, kv_indptr, kv_indices) -> None:
        ps = self.page_size
        for b in range(len(item_indptr) - 1):
            items = range(item_indptr[b], item_indptr[b + 1])
            held = kv_indptr[b + 1] - kv_indptr[b]
            items = [i for i in items if 0 <= src_pos[i] // ps < held and 0 <= dst_pos[i] // ps < held]

            def at(p):
                return int(kv_indices[kv_indptr[b] + p // ps]), p % ps

            moved, scale = [], {}
            for i in items:
                sp, so = at(src_pos[i])
                moved.append(self.codes[sp, :, :, so] * self.scales[sp][..., None])
                dp = at(dst_pos[i])[0]
                scale[dp] = torch.maximum(scale.get(dp, self.scales[dp]), self.scales[sp])
            for dp, s in scale.items():
                grown = (s != self.scales[dp])[..., None, None]
                self.codes[dp] = torch.where(
                    grown, grid(self.codes[dp] * (self.scales[dp] / s)[..., None, None], self.dtype), self.codes[dp])
            for dp, s in scale.items():
                self.scales[dp] = s
            for i, x in zip(items, moved):
                dp, do = at(dst_pos[i])
                self.codes[dp, :, :, do] = grid(x / self.scales[dp][..., None], self.dtype)

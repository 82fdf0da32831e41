"""4-bit page of the grouped-query K/V cache: 64 positions of one K/V head in 72 D bytes.

A row of D values (64, 128 or 256) is held in blocks of 16: scale byte
``s8 = e4m3(amax / 6 * 2^-exp)`` (round to nearest even, at most 448), element =
nearest e2m1 value to ``x / (s8 * 2^exp)``, ties to the even code, sign kept.  (The MLA
row of ``kv_nvfp4`` multiplies by a rounded reciprocal instead, to give the bytes of
another writer; here the quotient itself is rounded.)

The order of the bytes is the one in which the attention kernels' fragments read them
(``csrc/kernels/kv4.cuh``).  This module is the golden CPU encoder and decoder.
"""
from __future__ import annotations

from typing import Tuple

import torch

from .codebook import E2M1_VALUES

PAGE = 64


def quantise(x: torch.Tensor, exp: int = -6) -> Tuple[torch.Tensor, torch.Tensor]:
    """[..., D] -> codes u8 [..., D] (0..15), scale bytes u8 [..., D / 16]."""
    y = x.double().unflatten(-1, (-1, 16))
    amax = y.abs().amax(-1).float()
    s8 = (amax / 6 * 2.0 ** -exp).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = (s8.double() * 2.0 ** exp)[..., None]
    a = y.abs()
    code = ((a > 0.25 * s).int() + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s) + (a > 2.5 * s)
            + (a >= 3.5 * s) + (a > 5 * s))
    code = torch.where(s > 0, code, 0) + 8 * torch.signbit(y)
    return code.to(torch.uint8).flatten(-2), s8.view(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor, exp: int = -6) -> torch.Tensor:
    """codes [..., D], scale bytes [..., D / 16] -> f32 [..., D]."""
    v = E2M1_VALUES.float().to(codes.device)[codes.long()].unflatten(-1, (-1, 16))
    return (v * (scales.view(torch.float8_e4m3fn).float() * 2.0 ** exp)[..., None]).flatten(-2)


def _places(D: int):
    """Per (position, value): byte and nibble of its key code and of its value code in a page, and per
    (position, block): byte of its key scale and of its value scale."""
    SD = min(D, 128)
    j = torch.arange(PAGE)[:, None]
    d = torch.arange(D)[None, :]
    slab, r = d // SD, d % SD
    P = SD // 4                                    # values of a key piece
    kb = slab * (PAGE * SD // 2) + j * (SD // 2) + r // P * (SD // 8) + r % (P // 2)
    kn = (r % P // (P // 2)).expand(PAGE, D)
    E = SD // 8                                    # values of a value piece
    vb = 36 * D + slab * (PAGE * SD // 2) + j // 2 * SD + r // E * (SD // 8) + j % 2 * (SD // 16) + r % (E // 2)
    vn = (r % E // (E // 2)).expand(PAGE, D)
    b = torch.arange(D // 16)[None, :]
    return kb, kn, vb, vn, 32 * D + j * (D // 16) + b, 68 * D + j // 2 * (D // 8) + 2 * b + j % 2


def pack_page(k_codes, k_scales, v_codes, v_scales) -> torch.Tensor:
    """Codes [64, D] and scale bytes [64, D / 16] of keys and values -> the page's bytes u8 [72 D]."""
    D = k_codes.shape[-1]
    kb, kn, vb, vn, ks, vs = _places(D)
    page = torch.zeros(72 * D, dtype=torch.int32)
    page.index_add_(0, kb.flatten(), (k_codes.int() << (4 * kn)).flatten().int())
    page.index_add_(0, vb.flatten(), (v_codes.int() << (4 * vn)).flatten().int())
    page[ks.flatten()] = k_scales.int().flatten()
    page[vs.flatten()] = v_scales.int().flatten()
    return page.to(torch.uint8)


def unpack_page(page: torch.Tensor):
    """The page's bytes u8 [72 D] -> (k_codes, k_scales, v_codes, v_scales)."""
    D = page.shape[-1] // 72
    kb, kn, vb, vn, ks, vs = _places(D)
    p = page.int()
    return ((p[kb] >> (4 * kn) & 15).to(torch.uint8), page[ks], (p[vb] >> (4 * vn) & 15).to(torch.uint8), page[vs])


def bounds(k: torch.Tensor) -> Tuple[torch.Tensor, float]:
    """Key rows as held [64, D] -> (int8 [2, D]: ceil(max / unit), floor(min / unit); unit, the smallest
    power of two with max |k| <= 127 unit, 1 for a page of zeros)."""
    k = k.double()
    top = float(k.abs().max())
    unit = 1.0
    if top > 0:
        unit = 2.0 ** -100
        while top > 127 * unit:
            unit *= 2
    return torch.stack([torch.ceil(k.amax(0) / unit), torch.floor(k.amin(0) / unit)]).to(torch.int8), unit

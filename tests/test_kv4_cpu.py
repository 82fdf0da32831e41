"""The 4-bit grouped-query cache page on the CPU: rounding, byte layout, bounds; refusals that need no GPU."""
import math
import random

import pytest
import torch

from vllm_moet_b200.formats import kv4
from vllm_moet_b200.formats.codebook import E2M1_VALUES


@pytest.mark.parametrize("D", [64, 128, 256])
def test_page_layout_round_trip(D):
    g = torch.Generator().manual_seed(D)
    kc, vc = (torch.randint(0, 16, (64, D), generator=g, dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.randint(0, 127, (64, D // 16), generator=g, dtype=torch.uint8) for _ in range(2))
    page = kv4.pack_page(kc, ks, vc, vs)
    assert page.shape == (72 * D,)
    for got, want in zip(kv4.unpack_page(page), (kc, ks, vc, vs)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_every_byte_is_used_once(D):
    kb, kn, vb, vn, ks, vs = kv4._places(D)
    half = torch.cat([(kb * 2 + kn).flatten(), (vb * 2 + vn).flatten()])
    whole = torch.cat([ks.flatten(), vs.flatten()])
    used = torch.cat([half, whole * 2, whole * 2 + 1])
    assert torch.equal(used.sort().values, torch.arange(2 * 72 * D))
    # a position's value bytes are its own: rows can be written in any order
    owner = torch.arange(64)[:, None].expand(64, D)
    for b in vb.unique():
        assert len(owner[vb == b].unique()) == 1


def test_rounding_is_to_nearest_with_ties_to_even():
    """Against a search over every code, on values that lie on and beside the midpoints."""
    rng = random.Random(5)
    rows = []
    for _ in range(200):
        s = rng.choice([2.0 ** -5, 0.8125, 3.25, 2.0 ** -13])
        row = [rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0, 0.1, 5.9]) * s * rng.choice([-1, 1]) for _ in range(15)]
        rows.append(row + [6 * s])
    x = torch.tensor(rows, dtype=torch.float64)
    codes, s8 = kv4.quantise(x)
    scale = s8.view(torch.float8_e4m3fn).double() / 64
    mags = E2M1_VALUES.double()[:8]
    for r in range(x.shape[0]):
        for i in range(16):
            q = abs(float(x[r, i])) / float(scale[r, 0])
            best = min(range(8), key=lambda c: (abs(q - float(mags[c])), c % 2))
            assert int(codes[r, i]) & 7 == best, (q, best)


def test_zeros_and_saturation():
    codes, s8 = kv4.quantise(torch.zeros(2, 64))
    assert not s8.any() and not codes.any()
    codes, s8 = kv4.quantise(torch.full((1, 64), 1e6))
    assert (kv4.values(codes, s8) == 42).all()              # 6 * 448 / 64
    codes, s8 = kv4.quantise(torch.full((1, 64), 1e6), exp=4)
    assert (kv4.values(codes, s8, exp=4) == 6 * 448 * 16).all()


def test_bounds_hold_every_key():
    g = torch.Generator().manual_seed(3)
    k = torch.randn(64, 128, generator=g).double() * torch.rand(128, generator=g) * 8
    b, unit = kv4.bounds(k)
    assert math.log2(unit) == int(math.log2(unit)) and k.abs().max() <= 127 * unit and k.abs().max() > 63 * unit
    assert (b[0].double() * unit >= k.amax(0)).all() and (b[1].double() * unit <= k.amin(0)).all()
    b, unit = kv4.bounds(torch.zeros(64, 64))
    assert unit == 1 and not b.any()


def test_cache_refuses_what_it_cannot_hold():
    from vllm_moet_b200.ops.kv4 import KV4Cache
    for args, kw in (((4, 2, 96), {}), ((0, 2, 64), {}), ((4, 0, 64), {}), ((4, 2, 64), {"k_exp": 5}),
                     ((4, 2, 64), {"v_exp": -15}), ((4, 2, 64), {"device": "cpu"})):
        with pytest.raises(ValueError):
            KV4Cache(*args, **kw)


def test_the_sign_of_zero_is_kept():
    """As the format says, and as the kernel that writes the cache has it."""
    x = torch.zeros(3, 64)
    x[0] = -0.0
    x[1, ::2] = -0.0
    x[2, :4] = torch.tensor([-0.0, 6.0, -1e-9, 0.0])
    codes, s8 = kv4.quantise(x)
    assert (codes[0] == 8).all() and not s8[0].any()
    assert (codes[1, ::2] == 8).all() and (codes[1, 1::2] == 0).all()
    assert codes[2, :4].tolist() == [8, 7, 8, 0]
    assert torch.equal(kv4.values(codes, s8)[:2], torch.zeros(2, 64))


def test_a_page_s_score_bounds_the_rounded_query():
    """The score by which pages are chosen is an upper bound for the query rounded to 127 steps; a product of the query
    itself lies at most half a step times sum |k| above it, and some do (pages of equal keys, nothing else to hide it)."""
    g = torch.Generator().manual_seed(7)
    above = 0
    for _ in range(200):
        k = kv4.values(*kv4.quantise(torch.randn(1, 128, generator=g))).double().expand(64, 128)
        q = torch.randn(128, generator=g).double()
        (hi, lo), e = kv4.bounds(k)
        f = kv4.bounds(q[None])[1]
        r = torch.round(q / f)
        score = f * e * float(r.clamp(min=0) @ hi.double() + r.clamp(max=0) @ lo.double())
        assert float(f * r @ k[0]) <= score
        assert float(q @ k[0]) <= score + f / 2 * float(k[0].abs().sum())
        above += float(q @ k[0]) > score
    assert 0 < above < 60


def test_more_heads_than_a_grid_has_rows_are_refused():
    from vllm_moet_b200.ops.kv4 import KV4Cache
    with pytest.raises(ValueError, match="65535"):
        KV4Cache(1, 65536, 64)

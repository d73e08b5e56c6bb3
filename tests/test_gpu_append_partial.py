"""norm_rotate_append where only a part of a head turns: what is not a number stays where
the definition has it, angles of large positions, and parts that are no whole vectors."""
import math

import pytest
import torch

from emmy_b200 import paged
from test_gpu_quantised import BF16, E4M3, F16, F32, appended

pytestmark = pytest.mark.gpu


def append(rotation, norm, x, heads, kv_heads, positions, kind):
    """(queries, keys, values) as they are written, tokens in order."""
    tokens, _, dim = x.shape
    caches = [torch.zeros(1, tokens, kv_heads, dim, device="cuda").to(kind) for _ in range(2)]
    at = torch.arange(tokens, dtype=torch.int32, device="cuda")
    out = paged.norm_rotate_append(rotation, norm, *x.split([heads, kv_heads, kv_heads], 1), positions, at, *caches)
    return out.float(), *(c[0].float() for c in caches)


def same(got, want):
    return bool(((got == want) | (got.isnan() & want.isnan())).all())


@pytest.mark.parametrize("dim,rotary", [(64, 32), (128, 32), (128, 96), (96, 64), (96, 24), (80, 20), (256, 64), (7, 2), (64, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bits8", [True, False])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_components_that_are_not_finite(dim, rotary, interleaved, dtype, bits8, bad):
    """Each component of a head in turn, one a token.  One that does not turn concerns itself alone, one
    that turns its pair; a norm makes of a head with an infinity zeros and a NaN, of one with a NaN NaNs."""
    heads, kv_heads, kind = 3, 1, E4M3 if bits8 else dtype
    g = torch.Generator(device="cuda").manual_seed(dim)
    clean = torch.randn(dim, heads + 2 * kv_heads, dim, generator=g, device="cuda").to(dtype)
    x, each = clean.clone(), torch.arange(dim, device="cuda")
    x[each, :, each] = bad
    positions = torch.randint(1, 1000, (dim,), generator=g, device="cuda", dtype=torch.int32)
    rotation = paged.Rotation(torch.rand(rotary // 2, generator=g, device="cuda"), interleaved=interleaved)
    pairs = torch.arange(rotary, device="cuda")
    pairs = pairs ^ 1 if interleaved else (pairs + rotary // 2) % max(1, rotary)
    own = torch.eye(dim, dtype=torch.bool, device="cuda")             # [token, component]
    pair = own.clone()
    pair[torch.arange(rotary, device="cuda"), pairs] = True
    stored = math.copysign(448.0, bad) if bits8 and not math.isnan(bad) else bad
    want, got = append(rotation, None, clean, heads, kv_heads, positions, kind), append(rotation, None, x, heads, kv_heads, positions, kind)
    for i, (a, b) in enumerate(zip(got, want)):
        turned = i < 2
        there = b.clone()
        there[each, :, each] = stored if i else bad
        concerned = pair if turned else own
        if turned:
            there[:rotary] = torch.where(concerned[:rotary, None], a[:rotary], there[:rotary])     # (a pair of the two: the definition's below)
        assert same(a, there), i
        if turned and rotary:
            # an infinity times a cosine or sine, whose sign decides, or no number
            pair_of = a[:rotary].masked_select(pair[:rotary, None].expand_as(a[:rotary]))
            assert bool((~pair_of.isfinite() | (pair_of.abs() == 448)).all()), i
    w = torch.rand(dim, generator=g, device="cuda").to(dtype) + 0.5
    got = append(rotation, paged.Norm(w, w), x, heads, kv_heads, positions, kind)
    for a in got[:2]:
        assert bool(a[each, :, each].isnan().all())
        if math.isnan(bad):
            assert bool(a.isnan().all())
        else:
            assert bool((a[rotary:].masked_select(~own[rotary:, None].expand_as(a[rotary:])) == 0).all())
            assert bool((a[:rotary].masked_select(~pair[:rotary, None].expand_as(a[:rotary])) == 0).all())
    there = want[2].clone()
    there[each, :, each] = stored
    assert same(got[2], there)


@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 128), (96, 20), (80, 20), (96, 36), (7, 6), (33, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_angles_of_large_positions(dim, rotary, interleaved):
    """Pairs (1, 0) come out as cosine and sine, whichever kernel takes the head.  A cosine in 32 bits is
    off by 2 units in its last place at most and the step to the angle's rest by half a unit: 2.5 x 2^-23 of
    the value.  The angle in 64 bits: two roundings of up to 2^18.4 half turns, 2^-33.6 of one, 2^-31.9
    radians.  (An angle that ends at 32 bits is off by 2^-25 half turns, 9e-8 radians.)"""
    tokens, half = 4096, rotary // 2
    g = torch.Generator(device="cuda").manual_seed(rotary)
    x = torch.zeros(tokens, 3, dim, device="cuda")
    left = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    right = left + (1 if interleaved else half)
    x[..., left] = 1.0
    frequencies = torch.rand(half, generator=g, device="cuda")
    positions = torch.randint(-(1 << 20), 1 << 20, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    out, _, _ = append(paged.Rotation(frequencies, interleaved=interleaved), None, x, 1, 1, positions, E4M3)
    angle = positions.double()[:, None] * frequencies.double()           # (exact: 20 and 24 bits)
    for at, want in ((left, angle.cos()), (right, angle.sin())):
        off = (out[:, 0, at].double() - want).abs()
        assert bool((off <= 2.0 ** -21 * want.abs() + 2.0 ** -31).all()), float((off - 2.0 ** -21 * want.abs()).max())


@pytest.mark.parametrize("dim,rotary", [(96, 24), (96, 48), (80, 40), (80, 20), (192, 72), (128, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("bits8,norm", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_halves_that_are_no_vectors(dim, rotary, interleaved, bits8, norm, dtype):
    """Heads of whole vectors, of which a part turns whose halves are none."""
    appended(37, 6, 2, dim, rotary, 16, dtype, bits8, norm, interleaved=interleaved)
    appended(600, 12, 4, dim, rotary, 16, dtype, bits8, norm, interleaved=interleaved)

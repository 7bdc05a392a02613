"""Attention over 4-bit pages in bfloat16 against 64 bits, by the norm of the difference: a mean over many keys is many times smaller than the values are, and an error that a bound in terms of the values lets pass
may be as large as the result.

What the error is made of.  The result's rounding: half a step of 2^-7 / m relative to a value of mantissa m, uniform, is a root mean square of 2^-7 / sqrt(12 E[m^2]) of the results', 1.5e-3 for mantissas spread as those of
ordinary numbers are, 2.3e-3 at the very most (all at 1).  The soft-max's weights are float16 on their way into the second product: uniform in +- 2^-11 / m, 2e-4 at random, and they multiply codes of 0 to 15 (root mean square
8.8) where the values are codes less 7.5 (4.6): twice that, 4e-4, whatever the number of keys, as both sums grow with its root.  Together at most sqrt(2.3^2 + 0.4^2) = 2.4e-3."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NORM = 2.4e-3


def _attend(keys, tokens, heads, kv_heads, hd, rows, splits, form, seed, window=0, groups=512, used=None):
    """``tokens`` tokens at the end of ``keys`` keys (``rows``: each at its own end).  -> result and 64 bits, [tokens, heads, hd] on the GPU"""
    from nanospec_amd.kernels import ops

    page, gen = 16, torch.Generator(device=DEV).manual_seed(seed)
    pages = -(-keys // page)
    draw = lambda low, high, *shape: torch.randint(low, high, shape, generator=gen, device=DEV)
    # codes of all values alike; steps of 2^-4 to 2^-1, low = -7.5 steps, bfloat16 exactly: values of both signs
    sides, made = [], []
    for size in (1.5, 1.0):  # (scores of both signs, 1.7 at random)
        codes = draw(0, 16, pages, kv_heads, page, hd)
        step = (draw(4, 8, pages, kv_heads, page).float() * 2.0 ** -draw(5, 7, pages, kv_heads, page).float() * size).bfloat16()
        step = (step.view(torch.int16) & -32).view(torch.bfloat16)  # three bits: 7.5 times it is exact
        low = (-7.5 * step.float()).bfloat16()
        made += [codes.to(torch.uint8), step, low]
        sides.append((codes * step.double()[..., None] + low.double()[..., None]).transpose(0, 1).reshape(kv_heads, -1, hd)[:, :keys])
    pool = ops.Kv4Pages.from_codes(*made)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    q = (1.5 * torch.randn((tokens, heads * hd), generator=gen, device=DEV)).bfloat16()
    pos = torch.arange(keys - tokens, keys, device=DEV)
    if rows:
        tiles = [[0, 0, i, 1, keys - tokens + i + 1, 0, tokens * -(-keys // 32), 0] for i in range(tokens)]
    else:
        tiles = [[0, t0, 0, tokens, keys, 0, 0, -1] for t0 in range(0, tokens, 32)]
    tiles = torch.tensor(tiles, dtype=torch.int32, device=DEV)
    columns = tiles.shape[0] * (1 if rows else 32) * heads
    work = tuple(torch.full((columns * splits * w,), math.nan, device=DEV) for w in (hd, 1)) if splits > 1 else None
    out = torch.full((tokens, heads * hd), 7.0, dtype=torch.bfloat16, device=DEV)
    scale = hd**-0.5
    ops.attention_kv4(q, out, pool, tiles, table, heads, kv_heads, hd, scale, rows, window=window, splits=splits, workspace=work, groups=groups, form=form)
    if used is not None:
        used.append((work[1].view(columns, splits)[:heads] > -math.inf).sum(1))  # ranges of the first token's columns
    want = torch.empty((tokens, heads, hd), dtype=torch.float64, device=DEV)
    key = torch.arange(keys, device=DEV)
    hidden = key[None] > pos[:, None]
    if window:
        hidden |= key[None] <= pos[:, None] - window
    for h in range(heads):
        k, v = (side[h // (heads // kv_heads)] for side in sides)
        s = (q.double().view(tokens, heads, hd)[:, h] @ k.T.contiguous() * scale).masked_fill(hidden, -math.inf)
        want[:, h] = torch.softmax(s, 1) @ v
    return out.double().view(tokens, heads, hd), want


def _off(got, want):
    return float((got - want).norm() / want.norm())


# waves of a workgroup of single tokens, or tokens of a portion's tile that a wave takes; ranges
FORMS = [(True, 4, 1), (True, 8, 1), (True, 4, 7), (True, 4, 64), (False, 16, 1), (False, 32, 1), (False, 16, 5), (False, 32, 9), (False, 32, 64)]


@pytest.mark.parametrize("keys", [2000, 7001, 20000])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,form,splits", FORMS)
def test_every_form_over_many_keys(rows, form, splits, hd, keys):
    got, want = _attend(keys, 9 if rows else 45, 6, 2, hd, rows, splits, form, keys + hd)
    assert _off(got, want) <= NORM
    # and each token's by itself (fewer values: a third more)
    assert float(((got - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)).max()) <= 1.33 * NORM


@pytest.mark.parametrize("rows,form,splits", [(True, 4, 16), (False, 16, 2), (False, 32, 2), (False, 32, 40)])
@pytest.mark.parametrize("hd", [64, 128])
def test_nothing_grows_with_the_keys(hd, rows, form, splits):
    """300,000 keys: the norm's bound, and no part that is the same for all.  Roundings have both signs: a column's (token and head) mean over its channels is off by what its weights' roundings leave, 4e-4 of the root mean
    square at random (codes of a key have a mean), and that of 256 columns by 2.5e-5, the results' own roundings 1.6e-3 / sqrt(16,384) = 1.3e-5 beside it; five times the sum of their squares' root is 1.4e-4."""
    got, want = _attend(300_000, 32, 8, 2, hd, rows, splits, form, hd)
    assert _off(got, want) <= NORM
    assert abs(float((got - want).mean() / want.square().mean().sqrt())) <= 1.4e-4


@pytest.mark.parametrize("rows,form,splits", FORMS)
def test_windows_over_many_keys(rows, form, splits):
    got, want = _attend(9000, 9 if rows else 45, 6, 2, 64, rows, splits, form, 5, window=3001)
    assert _off(got, want) <= NORM


def test_the_same_bits_again():
    """The same call twice, other work between them."""
    for rows, form, splits in FORMS:
        first, _ = _attend(7001, 9 if rows else 45, 6, 2, 128, rows, splits, form, 3)
        _attend(2000, 5, 6, 2, 128, rows, splits, form, 4)
        again, _ = _attend(7001, 9 if rows else 45, 6, 2, 128, rows, splits, form, 3)
        assert torch.equal(first, again)


def _of_values(v, dtype, hd, heads=4, kv_heads=1, tokens=20, seed=1):
    """Every form's attention of the last ``tokens`` keys over values float64 [keys, hd], ordinary keys.  -> [(form, result)], 64 bits"""
    import kv4_oracle as oracle
    from nanospec_amd.kernels import ops

    held, page = v.shape[0], 16
    gen = torch.Generator().manual_seed(seed)
    k = 0.5 * torch.randn((held, hd), generator=gen, dtype=torch.float64)
    made, sides = [], []
    for x in (k, v):
        c, s, low = oracle.quantised(x.view(held // page, 1, page, hd))
        sides.append((s * c + low).view(held, hd))
        made += [c.to(torch.uint8).to(DEV), s[..., 0].bfloat16().to(DEV), low[..., 0].bfloat16().to(DEV)]
    pool = ops.Kv4Pages.from_codes(*made)
    table = torch.arange(held // page, dtype=torch.int32, device=DEV)[None]
    q = torch.randn((tokens, heads * hd), generator=gen).to(dtype)
    pos = torch.arange(held - tokens, held)
    s = (q.double().view(tokens, heads, hd) @ sides[0].T * hd**-0.5).masked_fill((torch.arange(held)[None] > pos[:, None])[:, None], -math.inf)
    want = torch.softmax(s, -1) @ sides[1]
    got = []
    kinds = [("plain", 0), ("rows", 4), ("rows", 8), ("tiles", 16)] + [("tiles", 32)] * (dtype == torch.bfloat16)
    for kind, form in kinds if hd in (64, 128) else kinds[:1]:
        for splits in (1, 3, 30):
            columns = (tokens if kind != "tiles" else 32) * heads
            work = tuple(torch.full((columns * splits * w,), math.nan, device=DEV) for w in (hd, 1)) if splits > 1 else None
            out = torch.full((tokens, heads * hd), 7.0, dtype=dtype, device=DEV)
            if kind == "plain":
                ops.attention_kv4_plain(q.to(DEV), out, pool, torch.zeros(tokens, dtype=torch.int32, device=DEV), pos.int().to(DEV), table, heads, kv_heads, hd, hd**-0.5, splits=splits, workspace=work)
            else:
                tiles = [[0, 0, i, 1, held - tokens + i + 1, 0, tokens * held // 32, 0] for i in range(tokens)] if kind == "rows" else [[0, 0, 0, tokens, held, 0, 0, -1]]
                ops.attention_kv4(q.to(DEV), out, pool, torch.tensor(tiles, dtype=torch.int32, device=DEV), table, heads, kv_heads, hd, hd**-0.5, kind == "rows", splits=splits, workspace=work,
                                  groups=1 << 20, form=form)
            got.append(((kind, form, splits), out.cpu().double().view(tokens, heads, hd)))
    return got, want


def _bound(dtype):
    """bfloat16 as above; one key may have all the weight, and its rounding, 2^-12 at most, multiplies codes (8.8) where values are 4.6: 4.7e-4 for 4e-4.  float32: 1e-5, as over many keys."""
    return 2.4e-3 if dtype == torch.bfloat16 else 1e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("size", [2.0**-99, 2.0**-70, 2.0**31, 2.0**50, 2.0**57, 2.0**90, -(2.0**100), 1.5 * 2.0**126])
def test_values_all_alike(size, hd, dtype):
    """Every key's value is a vector of one number (step 0), of any size that a page keeps: so is the mean."""
    got, want = _of_values(torch.full((1024, hd), size, dtype=torch.float64), dtype, hd)
    for form, out in got:
        assert bool(((out / want - 1).abs() <= _bound(dtype)).all()), form


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("low,high", [(-94, -94), (-80, -60), (95, 95), (-94, 94)])
def test_values_of_any_size(low, high, hd, dtype):
    """Values of steps from 2^-97 to 2^97, alike or mixed: the error in terms of the result is that of ordinary ones."""
    gen = torch.Generator().manual_seed(hd)
    v = torch.randn((1024, hd), generator=gen, dtype=torch.float64) * 2.0 ** torch.randint(low, high + 1, (1024, 1), generator=gen)
    got, want = _of_values(v, dtype, hd)
    for form, out in got:
        assert float((out - want).norm() / want.norm()) <= _bound(dtype), form


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_great_lowest_values_beside_small_steps(dtype):
    """Half of the keys' values lie about 2^40 with steps of 2^10, the others about 1."""
    gen = torch.Generator().manual_seed(1)
    v = torch.randn((1024, 64), generator=gen, dtype=torch.float64)
    v[::2] = 2.0**40 + 2.0**13 * v[::2]
    got, want = _of_values(v, dtype, 64)
    for form, out in got:
        assert float((out - want).norm() / want.norm()) <= _bound(dtype), form


@pytest.mark.parametrize("splits", [2, 8, 9, 33, 64])
@pytest.mark.parametrize("rows,tokens,heads,kv_heads,hd", [(True, 3, 4, 2, 64), (True, 140, 32, 8, 64), (True, 2, 8, 1, 128), (False, 40, 4, 2, 128), (False, 140, 32, 8, 64)])
def test_every_range_counts(rows, tokens, heads, kv_heads, hd, splits):
    """Few columns and many (a wave and four that join them), as many ranges as asked for: 64 of 256 keys are 16,384.  A range that is left out, or has another's weight, changes the result by the root of its share, 12% of 64."""
    used = []
    got, want = _attend(20_000, tokens, heads, kv_heads, hd, rows, splits, 4 if rows else 16, splits, groups=1 << 24, used=used)
    # (a range has share = blocks / splits + 1 of 625 blocks: of single tokens 64 make 10 each, 63 ranges)
    blocks = 20_000 // 32
    share = blocks // splits + 1 if rows else -(-blocks // splits)
    assert bool((used[0] == -(-blocks // share)).all()) and -(-blocks // share) >= splits - 1
    assert _off(got, want) <= NORM

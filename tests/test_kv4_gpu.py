"""Keys and values in 4 bits: the write into the pages, the read back, and attention over them, against their definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import kv4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROUND = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # a rounding is off by at most half a step, eps / 2 relative to the value


def _ops():
    from nanospec_amd.kernels import ops

    return ops


def _rand(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ------------------------------------------------------------------------------------------------ the write


def _written(lens, starts, heads, kv_heads, hd, rot, page, dtype, seed, interleaved=False, factor=1.0, q_out="in place", qkv=None, pad=0):
    ops = _ops()
    n = sum(lens)
    width = (heads + 2 * kv_heads) * hd
    qkv = _rand((n, width), seed, dtype) if qkv is None else qkv
    tables, pages = oracle.scattered_tables([-(-(a + b) // page) for a, b in zip(lens, starts)], 2, seed)
    positions = torch.cat([torch.arange(s, s + m) for m, s in zip(lens, starts)]).int()
    reqs = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).int()
    inv = (1.0 / 10000.0 ** (torch.arange(0, max(rot, 2), 2, dtype=torch.float32) / max(rot, 2)))[: max(1, rot // 2)]
    pool = ops.Kv4Pages.empty(pages, kv_heads, page, hd, DEV)
    room = torch.full((n + 1, width + pad), 5.0, dtype=dtype, device=DEV)
    dev = room[:n, pad:]  # rows further apart than they are long; with an odd ``pad`` they begin between 16 bytes
    dev.copy_(qkv)
    where = (positions.to(DEV), reqs.to(DEV), tables.to(DEV))
    q = None if q_out == "in place" else torch.empty((n, heads * hd), dtype=dtype, device=DEV)
    ops.rope_kv4_write(dev, *where, inv.to(DEV), pool, heads, kv_heads, hd, rot, interleaved=interleaved, factor=factor, q_out=q)
    torch.cuda.synchronize()
    x = qkv.double().view(n, heads + 2 * kv_heads, hd)
    turned = oracle.rotated(x[:, : heads + kv_heads], positions, inv[: rot // 2], rot, interleaved, factor)
    want = (turned[:, :heads], turned[:, heads:], x[:, heads + kv_heads :])
    if q is None:
        torch.testing.assert_close(dev[:, heads * hd :].cpu(), qkv[:, heads * hd :], rtol=0, atol=0, equal_nan=True)  # keys and values stay as the product left them
    else:
        torch.testing.assert_close(dev.cpu(), qkv, rtol=0, atol=0, equal_nan=True)
    assert bool((room[n] == 5).all()) and bool((room[:, :pad] == 5).all())
    got = (dev[:, : heads * hd] if q is None else q).cpu().double().view(n, heads, hd)
    return pool, where, want, got, tables, positions, reqs


CASES = [
    # lens, starts, heads, kv_heads, hd, rot, page
    ([1], [0], 1, 1, 32, 32, 8),
    ([1, 1, 1], [7, 8, 100], 4, 2, 64, 64, 16),
    ([5, 1, 19], [3, 15, 0], 6, 2, 96, 96, 8),
    ([33], [60000], 8, 8, 128, 128, 16),
    ([9, 2], [30, 31], 7, 1, 256, 128, 32),
    ([17], [1], 5, 5, 160, 20, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["in place", "out", "interleaved", "odd rows"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_write_keeps_what_the_definition_says(case, form, dtype):
    lens, starts, heads, kv_heads, hd, rot, page = CASES[case]
    pool, where, (wq, wk, wv), got, tables, positions, reqs = _written(lens, starts, heads, kv_heads, hd, rot, page, dtype, case, interleaved=form == "interleaved",
                                                                      factor=1.25 if form == "interleaved" else 1.0, q_out="out" if form == "out" else "in place",
                                                                      pad=3 if form == "odd rows" else 8)
    # cosine and sine to 4 units of 2^-24 each, two products, a sum and the factor: 8 roundings of 2^-24 of the pair's size; then the rounding to the type
    pair = 2 * 1.25 * float(max(wq.abs().max(), wk.abs().max()))
    slack = 8 * 2.0**-24 * pair
    assert bool(((got - wq).abs() <= slack + ROUND[dtype] * (wq.abs() + slack)).all())
    codes = pool.codes()
    page_of = tables[reqs.long(), positions.long() // page].long()
    at = (page_of, slice(None), positions.long() % page)
    kc, ks, kl, vc, vs, vl = (c.cpu()[at].double() for c in codes)
    # values are not computed with: equal to the definition, code for code
    c, s, low = oracle.quantised(wv)
    assert torch.equal(vs, s[..., 0]) and torch.equal(vl, low[..., 0]) and torch.equal(vc, c)
    # keys: the marks are those of rotated keys within ``slack``, and every channel lies within half a step of what its code stands for
    assert bool((kl <= wk.amin(-1) + slack).all()) and bool((kl >= oracle.outward(wk.amin(-1) - slack, up=False)).all())
    assert bool((kl + 15 * ks >= wk.amax(-1) - 2 * slack).all())
    assert bool((ks <= oracle.outward((wk.amax(-1) - kl + 2 * slack) / 15 * (1 + 2.0**-22), up=True)).all())
    stands = ks[..., None] * kc + kl[..., None]
    assert bool(((stands - wk).abs() <= ks[..., None] * (0.5 + 2.0**-20) + 2 * slack).all())
    # the other tokens' places are as they were: zeros
    touched = torch.zeros(pool.pages, page, dtype=torch.bool)
    touched[page_of, positions.long() % page] = True
    for t in codes:
        t = t.cpu().double().transpose(1, 2)
        assert bool((t[~touched] == 0).all())
    # read back: the value of the code in 32 bits, rounded once
    for out in (torch.bfloat16, torch.float32):
        k, v = _ops().kv4_read(pool, *where, dtype=out)
        for got_, c_, s_, l_ in ((k, kc, ks, kl), (v, vc, vs, vl)):
            assert torch.equal(got_.cpu(), (s_.float()[..., None] * c_.float() + l_.float()[..., None]).to(out))


def test_write_of_constant_tiny_huge_and_bad_rows():
    """Rows of one value, of steps below what is kept, of ranges beyond it, with infinities and with no numbers; beside ordinary ones."""
    heads, kv_heads, hd, page = 1, 1, 64, 8
    rows = torch.randn(9, 3 * hd, generator=torch.Generator().manual_seed(1))
    v = rows[:, 2 * hd :]
    v[0] = 1.5
    v[1] *= 2.0**-110
    v[2, 3] = 2.0**101
    v[3, 63] = math.inf
    v[4, 0] = -math.inf
    v[5, 17] = math.nan
    v[6] = 0.0
    v[7] = -v[7].abs() - 3
    rows[:, hd : 2 * hd] = v
    pool, where, (wq, wk, wv), *_ = _written([9], [0], heads, kv_heads, hd, 0, page, torch.float32, 3, qkv=rows)
    c, s, low = oracle.quantised(wv)
    kc, ks, kl, vc, vs, vl = (t.cpu().double() for t in pool.codes())
    page_of = where[2].cpu()[0, torch.arange(9) // page].long()
    at = (page_of, 0, torch.arange(9) % page)
    for codes, steps, lows in ((kc, ks, kl), (vc, vs, vl)):
        assert torch.equal(codes[at], c[:, 0])
        assert torch.equal(steps[at], s[:, 0, 0])
        torch.testing.assert_close(lows[at], low[:, 0, 0], rtol=0, atol=0, equal_nan=True)
    k, v = _ops().kv4_read(pool, *where, dtype=torch.float32)
    assert bool(torch.isnan(v[2:6]).all()) and bool(torch.isfinite(v[[0, 1, 6, 7, 8]]).all()) and bool((v[0] == 1.5).all())


def test_write_leaves_pages_alone_where_a_layer_only_reads():
    ops = _ops()
    qkv = _rand((3, 4 * 64), 0, torch.bfloat16).to(DEV)
    pool = ops.Kv4Pages.empty(2, 1, 8, 64, DEV)
    pos, req, table = torch.arange(3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    ops.rope_kv4_write(qkv, pos, req, table, torch.ones(32, device=DEV), pool, 2, 1, 64, 64, write_kv=False)
    assert not bool(pool.pool.any())
    ops.rope_kv4_write(qkv[:0], pos[:0], req[:0], table, torch.ones(32, device=DEV), pool, 2, 1, 64, 64)  # a step without tokens
    assert not bool(pool.pool.any()) and ops.kv4_read(pool, pos[:0], req[:0], table)[0].shape == (0, 1, 64)


# ------------------------------------------------------------------------------------------------ attention


def _pool(pages, kv_heads, page, hd, seed, spread=1.0, held=None):
    """Pages of quantised random keys and values, with a few large channels among the keys; places that ``held`` (bool [pages, page]) does not name
    hold no numbers and the largest steps.  -> Kv4Pages, keys, values in 64 bits, the largest step of a value"""
    gen = torch.Generator().manual_seed(seed)
    k = torch.randn((pages, kv_heads, page, hd), generator=gen, dtype=torch.float64) * (1 + 4 * (torch.arange(hd) % 23 == 3))
    v = torch.randn((pages, kv_heads, page, hd), generator=gen, dtype=torch.float64) * torch.exp(spread * torch.randn((pages, kv_heads, page, 1), generator=gen, dtype=torch.float64)) + 0.3
    made, sides = [], []
    for x in (k, v):
        c, s, low = oracle.quantised(x)
        sides.append(s * c + low)
        if held is not None:
            empty = ~held[:, None, :, None].expand_as(s)
            s, low = torch.where(empty, 2.0**99, s), torch.where(empty, math.nan, low)
        made += [c.to(torch.uint8).to(DEV), s[..., 0].bfloat16().to(DEV), low[..., 0].bfloat16().to(DEV)]
    return _ops().Kv4Pages.from_codes(*made), sides[0], sides[1], float(oracle.quantised(v)[1].max())


def tolerance(dtype, out, size, hd, keys, v_step, v_most):
    """How far attention may be off, for |out| and the sizes at hand (``size``: the largest sum of |q| |k| scale of a visible pair).
    A score is at most 2 hd + 4 roundings of 2^-24 of ``size`` off (products and sums in 32 bits).  bfloat16's queries are float16 on the matrix cores, scaled so that the
    largest channel lies at 256 (or 16, where codes count sixteen times): exact but for what is below 2^-29 of the largest; 70 roundings for every 8 channels are allowed for them.
    The soft-max's weights are off by exp(2 delta) - 1 and the roundings of 2^x (2 units); bfloat16 rounds them to float16 on their way into the second product: 2^-11, and 2^-25 of the
    largest for those below the normal range, times keys; sums over the keys add 2^-24 each, of all that is summed (values and codes times steps: at most v_most + 8 steps)."""
    exact = dtype == torch.float32
    delta = size * 2.0**-24 * ((2 * hd + 4) if exact else max(2 * hd + 4, 70 * (hd / 8 + 2)))
    weight = math.expm1(2 * delta) + 2.0**-21 + (2.0**-22 if exact else 2.0**-11)
    # (a weight in float16 below 2^-14 of the largest is off by 2^-25; in 32 bits by less than 2^-34)
    small = (2.0**-34 if exact else 2.0**-25) * min(keys, 2**14)
    sums = min(keys, 4096) * 2.0**-24
    return (v_most + 8 * v_step) * (weight + small + sums) + ROUND[dtype] * out.abs()


ATTENTION = {
    # name: lens, starts
    "one key": ([1], [0]),
    "singles": ([1, 1, 1, 1], [0, 30, 31, 257]),
    "a long single": ([1], [2999]),
    "portion": ([37], [0]),
    "portions": ([2, 64, 33], [0, 5, 300]),
    "mixed": ([1, 65, 1, 3], [63, 130, 500, 8]),
}
SHAPES = [(1, 1, 32, 8), (4, 2, 64, 8), (8, 2, 64, 16), (6, 1, 128, 16), (32, 8, 128, 32), (3, 3, 128, 64), (17, 1, 64, 16), (40, 2, 128, 16), (4, 2, 96, 16), (5, 5, 256, 8)]


def _attend(case, heads, kv_heads, hd, page, dtype, window=0, seed=0, q_scale=1.0, spread=1.0):
    from nanospec_amd.parts.attention import kv4_attention

    lens, starts = ATTENTION[case] if isinstance(case, str) else case
    tables, pages = oracle.scattered_tables([-(-(a + b) // page) for a, b in zip(lens, starts)], 2, seed)
    held = torch.zeros(pages, page, dtype=torch.bool)
    for r, (m, b) in enumerate(zip(lens, starts)):
        for key in range(0, m + b, page):
            held[int(tables[r, key // page]), : m + b - key] = True
    pool, keys, values, v_step = _pool(pages, kv_heads, page, hd, seed, spread, held)
    n = sum(lens)
    q = (q_scale * _rand((n, heads * hd), seed + 7)).to(dtype)
    wide = torch.full((n, heads * hd + 16), math.nan, dtype=dtype, device=DEV)  # q inside a wider row
    wide[:, : heads * hd] = q.to(DEV)
    if window:  # pages before every query's window have been given back: nobody may read them
        for r, s in enumerate(starts):
            tables[r, : max(0, s - window + 1) // page] = -1
    ctx = oracle.batch_context(lens, starts, tables, DEV)
    out = torch.full((n, heads * hd), 7.0, dtype=dtype, device=DEV)
    scale = hd**-0.5
    kv4_attention(ctx, wide, out, pool, ctx.block_tables[0], heads, kv_heads, hd, scale, window=window)
    torch.cuda.synchronize()
    want, size = oracle.attention(q.double().view(n, heads, hd), keys, values, lens, starts, tables, page, heads, kv_heads, scale, window)
    tol = tolerance(dtype, want, size, hd, max(a + b for a, b in zip(lens, starts)), v_step, float(values.abs().max()))
    return out.cpu().double().view(n, heads, hd), want, tol, (pool, ctx, wide, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", list(ATTENTION))
@pytest.mark.parametrize("heads,kv_heads,hd,page", SHAPES)
def test_attention(case, heads, kv_heads, hd, page, dtype):
    got, want, tol, _ = _attend(case, heads, kv_heads, hd, page, dtype, seed=heads + hd)
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, 7, 64, 129])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 64, 8), (4, 1, 128, 16), (2, 2, 96, 8)])
def test_attention_window(heads, kv_heads, hd, page, window, dtype):
    got, want, tol, _ = _attend("mixed", heads, kv_heads, hd, page, dtype, window=window, seed=window)
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 64, 16), (6, 1, 128, 16), (32, 8, 64, 8)])
def test_attention_where_the_kernel_takes_another_form(heads, kv_heads, hd, page, dtype):
    """Portions over more keys than go by 16 tokens a wave, in ranges; rows that are whole, more than there are compute units; rows of very different lengths, cut by them; values of very
    different steps."""
    rows = [(37 * i) % 700 for i in range(70)]
    for case, spread in ((([40, 33], [5000, 4097]), 1.0), (([1] * 70, rows), 1.0), (([1] * 5, [6000, 3, 900, 0, 2500]), 1.0), (([1, 50, 1], [2000, 100, 31]), 2.0)):
        if len(case[0]) == 2 and heads == 32:
            continue  # (the oracle's time)
        got, want, tol, _ = _attend(case, heads, kv_heads, hd, page, dtype, seed=len(rows) + hd, spread=spread)
        assert bool(((got - want).abs() <= tol).all()), (case, float(((got - want).abs() / tol).max()))


def _layer(hd, heads=4, kv_heads=2):
    return dict(heads=heads, kv_heads=kv_heads, hd=hd, inv=(1.0 / 10000.0 ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd)).to(DEV))


def _step(layer, qkv, lens, starts, tables, pool, dtype):
    """Write and attention of a step, as a layer calls them.  -> [tokens, heads * hd]"""
    from nanospec_amd.parts.attention import kv4_attention

    ops, heads, kv_heads, hd = _ops(), layer["heads"], layer["kv_heads"], layer["hd"]
    ctx = oracle.batch_context(lens, starts, tables, DEV)
    dev = qkv.to(device=DEV, dtype=dtype, copy=True)
    ops.rope_kv4_write(dev, ctx.positions, ctx.token_req, ctx.block_tables[0], layer["inv"], pool, heads, kv_heads, hd, hd)
    out = torch.empty((dev.shape[0], heads * hd), dtype=dtype, device=DEV)
    return kv4_attention(ctx, dev, out, pool, ctx.block_tables[0], heads, kv_heads, hd, hd**-0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_bad_key_or_value_is_seen_by_those_who_see_it(hd, bad, dtype):
    """A token whose key or value holds no number, or an infinity: whoever comes later in its request has no number in that head's group, everybody else the same bits as without it."""
    ops, layer = _ops(), _layer(hd)
    heads, kv_heads = layer["heads"], layer["kv_heads"]
    lens, starts = [70, 70], [0, 0]
    tables, pages = oracle.scattered_tables([6, 6], 1, 3)
    qkv = _rand((140, (heads + 2 * kv_heads) * hd), hd)
    run = lambda x: _step(layer, x, lens, starts, tables, ops.Kv4Pages.empty(pages, kv_heads, 16, hd, DEV), dtype).view(140, heads, hd).clone()
    clean = run(qkv)
    for column, group in ((heads * hd + 5, 0), ((heads + kv_heads) * hd + hd + 7, 1)):  # a key of head 0, a value of head 1
        worse = qkv.clone()
        worse[40, column] = bad
        got = run(worse)
        hit = torch.zeros(140, heads, dtype=torch.bool, device=DEV)
        hit[40:70, group * 2 : group * 2 + 2] = True
        assert bool(torch.isnan(got[hit]).all()) and torch.equal(got[~hit], clean[~hit])
        # single tokens behind it
        for pos, nan in ((40, True), (39, False)):
            pool = ops.Kv4Pages.empty(pages, kv_heads, 16, hd, DEV)
            _step(layer, worse[: pos + 1], [pos + 1], [0], tables[:1], pool, dtype)
            one = _step(layer, worse[pos : pos + 1], [1], [pos], tables[:1], pool, dtype).view(heads, hd)
            assert bool(torch.isnan(one[group * 2 : group * 2 + 2]).all()) == nan and bool(torch.isfinite(one[2 - group * 2 : 4 - group * 2]).all())


@pytest.mark.parametrize("hd", [96, 128])
def test_pages_beyond_4_gib(hd):
    """The same step in pages at a small pool's beginning and at the end of a pool of more than 2^32 bytes: the same bits."""
    ops, layer = _ops(), _layer(hd, heads=8, kv_heads=8)
    lens, starts = [40, 1, 1], [0, 0, 100]
    per_page = 8 * 2 * (8 * hd + 64)
    pages = 2**32 // per_page + 50
    small, _ = oracle.scattered_tables([3, 1, 7], 0, 1)
    far = torch.where(small >= 0, pages - 1 - small, small)
    results = []
    for tables, n in ((small, 11), (far, pages)):
        pool = ops.Kv4Pages.empty(n, 8, 16, hd, DEV)
        _step(layer, _rand((100, 24 * hd), 4), [100], [0], tables[2:], pool, torch.bfloat16)  # what the last request has
        out = _step(layer, _rand((42, 24 * hd), 5), lens, starts, tables, pool, torch.bfloat16)
        where = (torch.arange(101, dtype=torch.int32, device=DEV), torch.full((101,), 2, dtype=torch.int32, device=DEV), tables.to(DEV))
        results.append((out, *ops.kv4_read(pool, *where)))
        assert bool(pool.pool[int(tables.max())].any())
        del pool
    assert all(torch.equal(a, b) for a, b in zip(*results)) and bool(results[0][1].any())


def test_on_another_stream():
    ops, layer = _ops(), _layer(64)
    lens, starts = [50, 1], [0, 300]
    tables, pages = oracle.scattered_tables([4, 19], 1, 2)
    qkv, x = _rand((51, 8 * 64), 1), _rand((300, 8 * 64), 2)
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            pool = ops.Kv4Pages.empty(pages, 2, 16, 64, DEV)
            _step(layer, x, [300], [0], tables[1:], pool, torch.bfloat16)
            out = _step(layer, qkv, lens, starts, tables, pool, torch.bfloat16)
            rows = ops.int8_rows(out)
            results.append((out, ops.linear_int8(rows, ops.Int8Weight.from_float(_rand((300, 256), 3).to(DEV)))))
        stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("rows,splits", [(False, 1), (False, 3), (True, 1), (True, 4)])
def test_tokens_that_no_tile_describes_are_left_alone(rows, splits):
    """A step of a fixed shape: tiles without tokens among others, rows behind the last."""
    ops = _ops()
    pool, keys, values, _ = _pool(8, 2, 16, 64, 1)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
    q = _rand((60, 256), 2).bfloat16().to(DEV)
    n = 1 if rows else 40
    live = [[0, 0, 5, 1, 90, 0, 3, 0]] if rows else [[0, 0, 5, 40, 90, 0, 0, 0], [0, 32, 5, 40, 90, 0, 0, -1]]
    none = [[0, 0, 0, 0, 0, 0, 3, -1]]
    tiles = torch.tensor(none + live + none * 3, dtype=torch.int32, device=DEV)
    columns = tiles.shape[0] * (1 if rows else 32) * 4
    work = tuple(torch.full((columns * splits * w,), math.nan, device=DEV) for w in (64, 1)) if splits > 1 else None
    out = torch.full((60, 256), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.attention_kv4(q, out, pool, tiles, table, 4, 2, 64, 0.125, rows, splits=splits, workspace=work, groups=512)
    assert bool((out[:5] == 7).all()) and bool((out[5 + n :] == 7).all())
    want, _ = oracle.attention(q[5 : 5 + n].cpu().double().view(n, 4, 64), keys, values, [n], [90 - n], table.cpu(), 16, 4, 2, 0.125)
    # (weights in float16, 2^-11 of values of up to 20, and the result's rounding)
    assert float((out[5 : 5 + n].cpu().double().view(n, 4, 64) - want).abs().max()) <= 20 * (2.0**-11 + 2.0**-8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,starts", [([1], [90]), ([20], [71]), ([1], [3000])])
def test_values_of_a_key_without_weight_cost_the_others_nothing(lens, starts, dtype):
    """One key's values, and their step, are 2^40 times the others', and its score is so far below them that its weight is 2^-60 or less: the result is that of the others alone, to their own
    tolerance."""
    from nanospec_amd.parts.attention import kv4_attention

    ops, hd, page = _ops(), 64, 16
    held = lens[0] + starts[0]
    tables, pages = oracle.scattered_tables([-(-held // page)], 1, 1)
    gen = torch.Generator().manual_seed(5)
    k = 0.1 * torch.randn((pages, 1, page, hd), generator=gen, dtype=torch.float64)
    v = torch.randn((pages, 1, page, hd), generator=gen, dtype=torch.float64)
    at = (int(tables[0, 40 // page]), 0, 40 % page)
    k[at], v[at] = -8.0, v[at] * 2.0**40
    made, sides = [], []
    for x in (k, v):
        c, s, low = oracle.quantised(x)
        sides.append(s * c + low)
        made += [c.to(torch.uint8).to(DEV), s[..., 0].bfloat16().to(DEV), low[..., 0].bfloat16().to(DEV)]
    pool = ops.Kv4Pages.from_codes(*made)
    q = (1 + 0.1 * _rand((lens[0], 4 * hd), 3)).to(dtype)  # the key's score is about -8 * 64 / 8 = -64, or 92 octaves
    ctx = oracle.batch_context(lens, starts, tables, DEV)
    out = torch.empty((lens[0], 4 * hd), dtype=dtype, device=DEV)
    kv4_attention(ctx, q.to(DEV), out, pool, ctx.block_tables[0], 4, 1, hd, hd**-0.5)
    want, size = oracle.attention(q.double().view(-1, 4, hd), *sides, lens, starts, tables, page, 4, 1, hd**-0.5)
    alone = sides[1].clone()
    alone[at] = 0
    tol = tolerance(dtype, want, size, hd, held, float(alone.abs().max()) / 4, float(alone.abs().max())) + 2.0**-40
    assert bool(((out.cpu().double().view(-1, 4, hd) - want).abs() <= tol).all())


@pytest.mark.parametrize("rows,tokens,heads,kv_heads,hd", [(False, 150, 32, 8, 64), (False, 40, 4, 2, 128), (True, 3, 4, 2, 64), (True, 200, 32, 8, 128)])
def test_any_number_of_ranges(rows, tokens, heads, kv_heads, hd):
    """Few columns and many, joined from 2 to 64 ranges, some of them empty: the result of one range, but for weights rounded against another reference (2^-11 of values of up to 20) and the
    result's own rounding."""
    ops = _ops()
    pool, _, _, _ = _pool(80, kv_heads, 16, hd, 3)
    table = torch.arange(80, dtype=torch.int32, device=DEV).view(1, 80)
    q = _rand((tokens, heads * hd), 2).bfloat16().to(DEV)
    if rows:
        tiles = torch.tensor([[0, 0, i, 1, 1280 - 6 * i, 0, 8 * tokens, 0] for i in range(tokens)], dtype=torch.int32, device=DEV)
    else:
        tiles = torch.tensor([[0, t0, 0, tokens, 1270, 0, 0, -1] for t0 in range(0, tokens, 32)], dtype=torch.int32, device=DEV)
    results = []
    for splits in (1, 2, 8, 9, 33, 64):
        columns = tiles.shape[0] * (1 if rows else 32) * heads
        work = tuple(torch.full((columns * splits * w,), math.nan, device=DEV) for w in (hd, 1)) if splits > 1 else None
        out = torch.full((tokens, heads * hd), 7.0, dtype=torch.bfloat16, device=DEV)
        ops.attention_kv4(q, out, pool, tiles, table, heads, kv_heads, hd, hd**-0.5, rows, splits=splits, workspace=work, groups=1 << 20)
        results.append(out.float())
    assert all(float((r - results[0]).abs().max()) <= 20 * (2 * 2.0**-11 + 2 * 2.0**-8) for r in results[1:])


@pytest.mark.parametrize("lens,starts", [([1, 1], [4000, 18000]), ([20], [6000])])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_float32_over_many_keys(hd, lens, starts):
    """A mean of many values is many times smaller than they are, and than sums of codes apart from lowest values.  In 32 bits throughout, the error is a small part of it all the same: a score of size 4 is some
    2^-24 sqrt(2 hd) of that off, 4e-6, and weights that are off by so much at random change a sum of the values at random by as much of itself; the exponential adds 2^-22, the sums, of blocks that are added up
    by waves and ranges, 2^-24 for the root of their number.  Together under 1e-5 of the root mean square."""
    got, want, _, _ = _attend((lens, starts), 4, 2, hd, 16, torch.float32, seed=hd, spread=0.3)
    assert float((got - want).norm() / want.norm()) <= 1e-5


@pytest.mark.parametrize("window", [1, 5, 31, 33, 70])
@pytest.mark.parametrize("splits", [2, 5, 64])
def test_ranges_that_a_window_hides(window, splits):
    """Ranges of a portion's keys so short that some tokens' windows begin behind the first of them, and end in front of the last."""
    ops = _ops()
    pool, keys, values, v_step = _pool(20, 2, 16, 64, 3)
    table = torch.arange(20, dtype=torch.int32, device=DEV).view(1, 20)
    for dtype in (torch.bfloat16, torch.float32):
        q = _rand((45, 256), 2).to(dtype)
        tiles = torch.tensor([[0, 0, 0, 45, 300, 0, 0, -1], [0, 32, 0, 45, 300, 0, 0, -1]], dtype=torch.int32, device=DEV)
        work = tuple(torch.full((2 * 32 * 4 * splits * w,), math.nan, device=DEV) for w in (64, 1))
        out = torch.full((45, 256), 7.0, dtype=dtype, device=DEV)
        ops.attention_kv4(q.to(DEV), out, pool, tiles, table, 4, 2, 64, 0.125, False, window=window, splits=splits, workspace=work)
        want, size = oracle.attention(q.double().view(45, 4, 64), keys, values, [45], [255], table.cpu(), 16, 4, 2, 0.125, window)
        tol = tolerance(dtype, want, size, 64, 300, v_step, float(values.abs().max()))
        assert bool(((out.cpu().double().view(45, 4, 64) - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_scores_below_32_bits_are_written_whatever_the_ranges(hd, dtype):
    """A token whose scores all lie below float32's range (-8 hd 10^34 10^5) has zeros, whole and in any number of ranges, among tokens that have results."""
    ops, heads, kv_heads, page, pages = _ops(), 4, 2, 16, 60
    gen = torch.Generator().manual_seed(hd)
    v = torch.randn((pages, kv_heads, page, hd), generator=gen, dtype=torch.float64)
    c, s, low = oracle.quantised(v)
    keys = (torch.zeros(v.shape, dtype=torch.uint8), torch.zeros(v.shape[:3]).bfloat16(), torch.full(v.shape[:3], -8.0).bfloat16())
    pool = ops.Kv4Pages.from_codes(*(t.to(DEV) for t in (*keys, c.to(torch.uint8), s[..., 0].bfloat16(), low[..., 0].bfloat16())))
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    n, held = 3, 900
    q = torch.zeros((n, heads * hd), dtype=dtype, device=DEV)
    q[1] = 1e34
    live = (s * c + low).transpose(0, 1).reshape(kv_heads, -1, hd)
    # equal keys: the mean of the values that a token sees
    want = torch.stack([live[:, : held - n + i + 1].mean(1).repeat_interleave(heads // kv_heads, 0) for i in range(n)])
    pos = torch.arange(held - n, held, dtype=torch.int32, device=DEV)
    forms = [("plain", 0)] if hd == 96 else [("plain", 0), ("rows", 4), ("rows", 8), ("tiles", 16)] + [("tiles", 32)] * (dtype == torch.bfloat16)
    for kind, form in forms:
        for splits in (1, 2, 9, 40):
            tiles = [[0, 0, i, 1, held - n + i + 1, 0, 90, 0] for i in range(n)] if kind == "rows" else [[0, 0, 0, n, held, 0, 0, -1]]
            columns = (n if kind != "tiles" else 32) * heads
            work = tuple(torch.full((columns * splits * w,), 3.0, device=DEV) for w in (hd, 1)) if splits > 1 else None
            out = torch.full((n, heads * hd), 7.0, dtype=dtype, device=DEV)
            if kind == "plain":
                ops.attention_kv4_plain(q, out, pool, torch.zeros(n, dtype=torch.int32, device=DEV), pos, table, heads, kv_heads, hd, 1e5, splits=splits, workspace=work)
            else:
                ops.attention_kv4(q, out, pool, torch.tensor(tiles, dtype=torch.int32, device=DEV), table, heads, kv_heads, hd, 1e5, kind == "rows", splits=splits, workspace=work,
                                  groups=1 << 20, form=form)
            got = out.cpu().double().view(n, heads, hd)
            assert bool((got[1] == 0).all()), (kind, form, splits)
            # weights of 1 and sums of 900 in 32 bits (float16's 1 is exact, its products' cuts 2^-20 of codes up to 15 times steps), then the rounding
            assert float((got[[0, 2]] - want[[0, 2]]).abs().max()) <= 2.0**-12 + ROUND[dtype] * float(want.abs().max()), (kind, form, splits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 64, 8), (4, 1, 128, 32), (2, 2, 96, 16)])
@pytest.mark.parametrize("fill", [0xFF, 0x7F, 0x80])
def test_places_that_nobody_has_written_may_hold_anything(fill, heads, kv_heads, hd, page, dtype):
    """A pool that was not cleared: steps and lowest values that are no numbers, infinite or below zero in all places behind a request's last key and in front of a window.  The bits are those over a pool of zeros."""
    from nanospec_amd.parts.attention import kv4_attention

    ops, layer = _ops(), _layer(hd, heads, kv_heads)
    for lens, starts, window in (([1, 37, 1], [0, 0, 90], 0), ([1, 40], [3, 203], 50), ([1, 3], [700, 650], 0)):
        tables, pages = oracle.scattered_tables([-(-(a + b) // page) for a, b in zip(lens, starts)], 2, 3)
        results = []
        for clear in (True, False):
            pool = ops.Kv4Pages.empty(pages, kv_heads, page, hd, DEV)
            if not clear:
                pool.pool.fill_(fill)
                if fill == 0x7F:  # infinite steps, lowest values of both kinds
                    pool.pool[..., 8 * hd :] = torch.tensor([0x80, 0xFF, 0x80, 0x7F], dtype=torch.uint8, device=DEV).repeat(16)
            for r, (m, s) in enumerate(zip(lens, starts)):  # what each has before this step, from its window on
                first = max(0, s - window + 1) if window else 0
                if s > first:
                    before = (torch.arange(first, s, dtype=torch.int32, device=DEV), torch.full((s - first,), r, dtype=torch.int32, device=DEV), tables.to(DEV))
                    ops.rope_kv4_write(_rand((s - first, (heads + 2 * kv_heads) * hd), r).to(device=DEV, dtype=dtype), *before, layer["inv"], pool, heads, kv_heads, hd, hd)
            ctx = oracle.batch_context(lens, starts, tables, DEV)
            qkv = _rand((sum(lens), (heads + 2 * kv_heads) * hd), 9).to(device=DEV, dtype=dtype)
            ops.rope_kv4_write(qkv, ctx.positions, ctx.token_req, ctx.block_tables[0], layer["inv"], pool, heads, kv_heads, hd, hd)
            out = torch.full((sum(lens), heads * hd), 7.0, dtype=dtype, device=DEV)
            results.append(kv4_attention(ctx, qkv, out, pool, ctx.block_tables[0], heads, kv_heads, hd, hd**-0.5, window=window))
        assert bool(torch.isfinite(results[0]).all()) and torch.equal(*results)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("what", ["key", "value"])
def test_no_number_is_seen_however_small_its_weight(what, hd, dtype):
    """The scores of 32 keys, all that a wave has, lie 2,000 below the others', far below any weight that 32 bits hold.  The value of one of them is no number, or its key: so is the result of whoever sees it."""
    ops, heads, page, pages, held = _ops(), 4, 16, 8, 128
    k = torch.zeros((pages, 1, page, hd), dtype=torch.float64)
    v = _rand((pages, 1, page, hd), 1).double()
    q = torch.ones((1, heads * hd), dtype=dtype, device=DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    forms = [("plain", 0)] if hd == 96 else [("plain", 0), ("rows", 4), ("rows", 8), ("tiles", 16)] + [("tiles", 32)] * (dtype == torch.bfloat16)
    for at in (0, 37, 94, 127):
        bad = (at // page, 0, at % page)
        kk, vv = k.clone(), v.clone()
        kk[at // 32 * 2 : at // 32 * 2 + 2] = -2000.0 * hd**-0.5
        (kk if what == "key" else vv)[bad] = math.nan
        made = []
        for x in (kk, vv):
            c, s, low = oracle.quantised(x)
            made += [c.to(torch.uint8).to(DEV), s[..., 0].bfloat16().to(DEV), low[..., 0].bfloat16().to(DEV)]
        pool = ops.Kv4Pages.from_codes(*made)
        for kind, form in forms:
            for splits in (1, 2, 4):
                columns = (1 if kind != "tiles" else 32) * heads
                work = tuple(torch.full((columns * splits * w,), 3.0, device=DEV) for w in (hd, 1)) if splits > 1 else None
                out = torch.full((1, heads * hd), 7.0, dtype=dtype, device=DEV)
                if kind == "plain":
                    ops.attention_kv4_plain(q, out, pool, torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([held - 1], dtype=torch.int32, device=DEV), table, heads, 1, hd, hd**-0.5,
                                            splits=splits, workspace=work)
                else:
                    tiles = torch.tensor([[0, 0, 0, 1, held, 0, 4 if kind == "rows" else 0, 0 if kind == "rows" else -1]], dtype=torch.int32, device=DEV)
                    ops.attention_kv4(q, out, pool, tiles, table, heads, 1, hd, hd**-0.5, kind == "rows", splits=splits, workspace=work, groups=1 << 20, form=form)
                assert bool(torch.isnan(out).all()), (at, kind, form, splits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128])
def test_short_portions_in_a_captured_step_of_a_wide_table(hd, dtype):
    """A captured step knows of its portions' keys only what its block tables have room for.  Of a short portion the ranges are as many as its keys are worth: the others leave nothing (but that they are empty), what is whole is
    written at once, and the step, replayed with other lengths and work between, gives what 64 bits say."""
    from nanospec_amd.engine.arena import Arena
    from nanospec_amd.engine.context import BatchLayout, StepContext, fill_batch
    from nanospec_amd.parts.attention import TILES, kv4_attention
    import numpy as np

    ops, heads, kv_heads, page, width = _ops(), 8, 2, 16, 8192
    scale, n, reqs = hd**-0.5, 128, 3
    layout = BatchLayout(n, reqs, 1, 1, width, plans=[(TILES, TILES.shape_captured(0, n, 2))])
    tables = np.full((reqs, width), -1, dtype=np.int32)
    tables[0, :200], tables[1, :200], tables[2, 0] = np.arange(200), np.arange(200, 400), 400
    held = torch.ones(401, page, dtype=torch.bool)
    pool, keys, values, _ = _pool(401, kv_heads, page, hd, hd, spread=0.3, held=held)
    dev_buf = torch.zeros(layout.total, dtype=torch.int32, device=DEV)
    host = torch.zeros(layout.total, dtype=torch.int32)
    q, out = torch.zeros((n, heads * hd), dtype=dtype, device=DEV), torch.zeros((n, heads * hd), dtype=dtype, device=DEV)
    context = lambda arena: StepContext(layout, dev_buf, arena, max_position=0, max_kv_len=width * page, captured=True)

    def fill(lens, starts):
        tail = n - sum(lens)
        fill_batch(host.numpy(), layout, [0] * n, [*starts, 0], [*lens, tail], [0, 1, 2], [0], [tables], pad_tail=tail)
        dev_buf.copy_(host)

    run = lambda ctx: kv4_attention(ctx, q, out, pool, ctx.block_tables[0], heads, kv_heads, hd, scale)
    fill([2, 2], [0, 0])
    probe = Arena(torch.device(DEV))
    run(context(probe))
    torch.cuda.synchronize()
    arena, stream = Arena(torch.device(DEV), nbytes=probe.high_water, fixed=True), torch.cuda.Stream()
    graph = ops.Graph(stream)
    with graph:
        run(context(arena))
    for lens, starts in (([2, 2], [0, 5]), ([100, 20], [0, 0]), ([64, 33], [9, 3000]), ([128 - 2, 2], [3000, 127]), ([60, 31], [450, 600])):
        fill(lens, starts)
        q.copy_(_rand((n, heads * hd), sum(starts)))
        out.fill_(7.0)
        for chunk in arena._chunks:
            chunk.fill_(0xFF)  # no numbers
        torch.randn(1000, device=DEV).sum().item()
        stream.wait_stream(torch.cuda.current_stream())
        graph.launch()
        stream.synchronize()
        m = sum(lens)
        want, _ = oracle.attention(q[:m].cpu().double().view(m, heads, hd), keys, values, lens, starts, torch.from_numpy(tables), page, heads, kv_heads, scale)
        got = out[:m].cpu().double().view(m, heads, hd)
        # (by the norm: a bfloat16 result's rounding is 2.3e-3 at most, weights in float16 4.7e-4; 32 bits 1e-5)
        assert float((got - want).norm() / want.norm()) <= (2.4e-3 if dtype == torch.bfloat16 else 1e-5), (lens, starts)
        assert bool((out[m:] == 7).all())
        # float32 results were left for the ranges that are joined alone: of portions of up to 128 keys for none
        if max(a + b for a, b in zip(lens, starts)) <= 128:
            assert all(bool(torch.isnan(c.view(torch.float32)[: c.numel() // 8]).all()) for c in arena._chunks)

"""4-bit pages on the CPU: the layout's way there and back, and what is refused."""

from __future__ import annotations

import pytest
import torch

from nanospec_amd.kernels import ops


def _codes(pages, kv_heads, page, hd, seed=0):
    gen = torch.Generator().manual_seed(seed)
    codes = lambda: torch.randint(0, 16, (pages, kv_heads, page, hd), dtype=torch.uint8, generator=gen)
    marks = lambda: torch.randn((pages, kv_heads, page), generator=gen).bfloat16()
    return codes(), marks(), marks(), codes(), marks(), marks()


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("page", [8, 32])
def test_codes_there_and_back(hd, page):
    made = _codes(3, 2, page, hd)
    pages = ops.Kv4Pages.from_codes(*made)
    assert pages.page == page and pages.kv_heads == 2 and pages.pool.shape == (3, 2, page // 8, 8 * hd + 64)
    assert all(torch.equal(a, b) for a, b in zip(made, pages.codes()))


def test_places_of_codes_and_marks():
    """The bytes that csrc/kv4.h names."""
    hd, page = 96, 16
    k, ks, kl, v, vs, vl = _codes(2, 2, page, hd)
    pool = ops.Kv4Pages.from_codes(k, ks, kl, v, vs, vl).pool
    for at in ((0, 0, 0, 0), (1, 1, 11, 5), (1, 0, 15, 95), (0, 1, 8, 33), (1, 1, 3, 62)):
        p, h, tok, ch = at
        record, j = pool[p, h, tok // 8], tok % 8
        t, g, c = ch % 32 // 8, ch // 32, ch % 8
        words = record.view(torch.int32)
        word = int(words[j * (hd // 8) + t * (hd // 32) + g])
        assert word >> (4 * (c // 2) + 16 * (c % 2)) & 15 == int(k[at])
        assert int(record.view(torch.int16)[(4 * hd + 16 * (ch // 4)) // 2 + j]) >> 4 * (ch % 4) & 15 == int(v[at])
        marks = record[8 * hd :].view(torch.bfloat16)
        assert marks[2 * j] == kl[p, h, tok] and marks[2 * j + 1] == ks[p, h, tok]
        assert marks[16 + 2 * j] == vl[p, h, tok] and marks[16 + 2 * j + 1] == vs[p, h, tok]


@pytest.mark.parametrize("hd,page", [(16, 16), (80, 16), (288, 16), (64, 4), (64, 24), (0, 16)])
def test_sizes_that_are_refused(hd, page):
    assert not ops.kv4_takes(hd, page)
    with pytest.raises(ops.KernelRefused):
        ops.Kv4Pages.empty(2, 1, page, hd, "cpu")


def test_pools_and_codes_that_are_refused():
    good = torch.zeros((2, 1, 2, 8 * 64 + 64), dtype=torch.uint8)
    ops.Kv4Pages(good, 64)
    for pool, hd in ((good, 32), (good.int(), 64), (good[0], 64), (good.transpose(0, 2), 64), (torch.zeros((2, 1, 3, 576), dtype=torch.uint8), 64),
                     (torch.zeros(2 * 2 * 576 + 8, dtype=torch.uint8)[8:].view(2, 1, 2, 576), 64)):
        with pytest.raises(ops.KernelRefused):
            ops.Kv4Pages(pool, hd)
    made = list(_codes(2, 1, 8, 32))
    for i, bad in ((0, made[0].int()), (1, made[1].float()), (4, made[4][:, :, :4]), (3, made[3][..., :16])):
        with pytest.raises(ops.KernelRefused):
            ops.Kv4Pages.from_codes(*made[:i], bad, *made[i + 1 :])


def _call(monkeypatch, **change):
    """Arguments that ``rope_kv4_write`` takes but for where they live, with some changed."""
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: None)  # (the checks of shapes and types are the host's)
    n, heads, kv, hd = 3, 4, 2, 32
    args = dict(qkv=torch.zeros(n, (heads + 2 * kv) * hd), positions=torch.zeros(n, dtype=torch.int32), token_req=torch.zeros(n, dtype=torch.int32),
                block_table=torch.zeros((1, 2), dtype=torch.int32), inv_freq=torch.ones(hd // 2), pages=ops.Kv4Pages.empty(2, kv, 8, hd, "cpu"), heads=heads,
                kv_heads=kv, head_dim=hd, rotary_dim=hd)
    args.update(change)
    return args


@pytest.mark.parametrize("change", [
    dict(qkv=torch.zeros(3, 200)), dict(qkv=torch.zeros(2, 256)), dict(qkv=torch.zeros(256, 3).t()), dict(qkv=torch.zeros(3, 256, dtype=torch.float16)),
    dict(positions=torch.zeros(3, dtype=torch.int64)), dict(positions=torch.zeros(6, dtype=torch.int32)[::2]), dict(token_req=torch.zeros(2, dtype=torch.int32)),
    dict(block_table=torch.zeros((1, 2))), dict(block_table=torch.zeros(2, dtype=torch.int32)), dict(block_table=torch.zeros((2, 3), dtype=torch.int32).t()),
    dict(inv_freq=torch.ones(15)), dict(inv_freq=torch.ones(16).double()), dict(rotary_dim=31), dict(rotary_dim=34), dict(kv_heads=1), dict(head_dim=64),
    dict(pages=torch.zeros(2, 2, 1, 320, dtype=torch.uint8)), dict(q_out=torch.zeros(3, 64)), dict(q_out=torch.zeros(3, 128).bfloat16()),
    dict(qkv=torch.zeros(1, 256).expand(3, 256)), dict(q_out=torch.zeros(1, 128).expand(3, 128))])
def test_write_refuses(monkeypatch, change):
    with pytest.raises(ops.KernelRefused):
        ops.rope_kv4_write(**_call(monkeypatch, **change))


@pytest.mark.parametrize("change", [
    dict(heads=3), dict(kv_heads=4), dict(head_dim=64), dict(q=torch.zeros(3, 100)), dict(q=torch.zeros(128, 3).t()), dict(out=torch.zeros(3, 64)),
    dict(out=torch.zeros(3, 128).bfloat16()), dict(out=torch.zeros(3, 200)[:, :128]), dict(window=-1), dict(splits=0), dict(splits=65), dict(splits=2), dict(scale=0.0), dict(scale=float("inf")),
    dict(splits=2, workspace=(torch.zeros(8), torch.zeros(24))), dict(splits=2, workspace=(torch.zeros(768), torch.zeros(23))), dict(token_req=torch.zeros(4, dtype=torch.int32)),
    dict(positions=torch.zeros(2, dtype=torch.int32), token_req=torch.zeros(2, dtype=torch.int32)),
    dict(q=torch.zeros(3, 128, dtype=torch.float16), out=torch.zeros(3, 128, dtype=torch.float16))])
def test_attention_refuses(monkeypatch, change):
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: None)
    args = dict(q=torch.zeros(3, 128), out=torch.zeros(3, 128), pages=ops.Kv4Pages.empty(2, 2, 8, 32, "cpu"), token_req=torch.zeros(3, dtype=torch.int32),
                positions=torch.zeros(3, dtype=torch.int32), block_table=torch.zeros((1, 2), dtype=torch.int32), heads=4, kv_heads=2, head_dim=32, scale=1.0)
    args.update(change)
    with pytest.raises(ops.KernelRefused):
        ops.attention_kv4_plain(**args)


@pytest.mark.parametrize("change", [
    dict(heads=3), dict(kv_heads=4), dict(head_dim=128), dict(pages=ops.Kv4Pages.empty(2, 2, 8, 96, "cpu"), head_dim=96, q=torch.zeros(3, 384), out=torch.zeros(3, 384)),
    dict(pages=torch.zeros(2, 2, 1, 576, dtype=torch.uint8)), dict(q=torch.zeros(3, 200)), dict(out=torch.zeros(3, 200)), dict(out=torch.zeros(3, 256).bfloat16()), dict(q=torch.zeros(256)),
    dict(tiles=torch.zeros((2, 8), dtype=torch.int64)), dict(tiles=torch.zeros((2, 6), dtype=torch.int32)), dict(tiles=torch.zeros(8, dtype=torch.int32)),
    dict(block_table=torch.zeros((1, 2))), dict(window=-1), dict(splits=0), dict(splits=65), dict(splits=2), dict(groups=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(form=5), dict(form=16), dict(rows=False, form=8),
    dict(rows=False, form=32), dict(splits=2, workspace=(torch.zeros(2 * 4 * 2 * 64 - 1), torch.zeros(16))), dict(splits=2, rows=False, workspace=(torch.zeros(2 * 4 * 2 * 64), torch.zeros(16))),
    dict(splits=2, workspace=(torch.zeros(1024).bfloat16(), torch.zeros(16)))])
def test_attention_by_tiles_refuses(monkeypatch, change):
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: None)
    args = dict(q=torch.zeros(3, 256), out=torch.zeros(3, 256), pages=ops.Kv4Pages.empty(2, 2, 8, 64, "cpu"), tiles=torch.zeros((2, 8), dtype=torch.int32),
                block_table=torch.zeros((1, 2), dtype=torch.int32), heads=4, kv_heads=2, head_dim=64, scale=1.0, rows=True)
    args.update(change)
    with pytest.raises(ops.KernelRefused):
        ops.attention_kv4(**args)


def test_tensors_on_the_cpu_are_refused():
    with pytest.raises(ops.KernelRefused, match="GPU"):
        ops.kv4_read(ops.Kv4Pages.empty(1, 1, 8, 32, "cpu"), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32))


def test_tensors_of_another_device_are_refused(monkeypatch):
    from types import SimpleNamespace

    on = lambda index: SimpleNamespace(is_cuda=True, get_device=lambda: index, device=f"cuda:{index}")
    monkeypatch.setattr(ops, "_device_index", lambda: 1)
    ops._one_gpu(on(1), None, on(1))
    for tensors in ((on(0),), (on(0), on(0)), (on(1), None, on(0)), (on(0), on(1))):
        with pytest.raises(ops.KernelRefused, match="tensors on"):
            ops._one_gpu(*tensors)
    with pytest.raises(ops.KernelRefused, match="GPU"):
        ops._one_gpu(on(1), torch.zeros(1))


# ------------------------------------------------------------------------------------------------ which models and engines take them


def _model(needs, cache_from=None, mixers=None):
    from types import SimpleNamespace

    cache_from = cache_from or [None] * len(needs)
    order = [SimpleNamespace(cache_from=c, layer=i) for i, c in enumerate(cache_from)]
    layers = [SimpleNamespace(mixer=m) for m in (mixers or [None] * len(needs))]
    return SimpleNamespace(cache_needs=needs, spec=SimpleNamespace(run_order=order), layers=layers, serve_int4_cache=lambda: None)


def test_caches_in_4_bits_refuse_what_is_not_built():
    from types import SimpleNamespace

    from nanospec_amd.cache.storage import CacheStorage
    from nanospec_amd.parts.needs import PagedNeed

    fits, other = PagedNeed(2, 64, int4=True), PagedNeed(2, 64)
    assert fits == other and hash(fits) == hash(other)  # (groups of pages are what they were)
    make = lambda model, page=16, kv_format="int4": CacheStorage(model, [4] * len({n for n in model.cache_needs if n is not None}), page, 2, torch.float32, "cpu", kv_format)
    with pytest.raises(ValueError, match="kv_format"):
        make(_model([fits]), kv_format="int8")
    with pytest.raises(ValueError, match="does not keep its keys and values in 4 bits"):
        make(_model([fits, other]))
    with pytest.raises(ValueError, match="multiple of 32 channels"):
        make(_model([PagedNeed(2, 80, int4=True)]))
    for page in (4, 12):
        with pytest.raises(ValueError, match="power of two of tokens from 8"):
            make(_model([fits]), page)
    reads = SimpleNamespace(takes_int4_cache=True)
    with pytest.raises(ValueError, match="reads another entry"):
        make(_model([fits, None], [None, 0], [reads, SimpleNamespace()]))
    storage = make(_model([fits, None, None], [None, 0, None], [reads, reads, None]))
    assert storage.views[1] is storage.views[0] and storage.views[2] is None and storage.views[0].pages.pool.shape == (4, 2, 2, 8 * 64 + 64)
    with pytest.raises(ValueError, match="keeps no keys and values"):
        storage.kept(2, None, None, None)


def test_ranges_of_portions_keep_within_their_memory():
    """However long the keys are that a captured step's table has room for, the ranges' results come to a few rounds of the card: 4 rounds x 8 waves a unit x 32 tokens x the head's 32-bit sums."""
    from nanospec_amd.parts import attention as att

    units = 256
    for tiles in (1, 2, 3, 17, 19, 33, 64, 100):
        for heads in (4, 24, 32, 40, 64):
            for longest in (2, 127, 512, 2048, 4096, 20000, 100_000, 131_072, 1 << 20):
                for wave_tokens in (16, 32):
                    splits = att.kv4_portion_ranges(tiles, heads, longest, wave_tokens, units)
                    assert 1 <= splits <= 64 and (splits == 1 or longest // splits >= att.KV4_PORTION_KEYS[0])
                    waves = tiles * heads * (32 // wave_tokens)
                    assert splits == 1 or splits * waves <= att.KV4_PORTION_ROUNDS * 8 * units
    # (17 and 33 tiles of 32 heads of 128 channels over 131,072 keys took 442 and 858 MiB)
    assert all(tiles * 32 * 32 * 128 * 4 * att.kv4_portion_ranges(tiles, 32, 131_072, 32, units) <= 128 << 20 for tiles in (17, 33))
    # as measured
    assert [att.kv4_portion_ranges(t, 32, n, 32, units) for t, n in ((22, 20333), (16, 8512), (64, 2048))] == [8, 4, 1]


def test_rows_of_more_keys_than_their_ranges_are_cut_for_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: None)
    args = dict(q=torch.zeros(1, 256), out=torch.zeros(1, 256), pages=ops.Kv4Pages.empty(2, 2, 8, 64, "cpu"), tiles=torch.zeros((1, 8), dtype=torch.int32),
                block_table=torch.zeros((1, ops.KV4_ROW_KEYS // 8 + 1), dtype=torch.int32), heads=4, kv_heads=2, head_dim=64, scale=1.0)
    with pytest.raises(ops.KernelRefused, match="room for up to 134217728 keys"):
        ops.attention_kv4(**args, rows=True)


def test_ranges_by_reciprocals_hold_every_block():
    """The share of a row's blocks that the kernel for single tokens computes, in float32 with a reciprocal that is off by a unit of its last place either way: as many ranges of it hold all blocks, up to the most keys."""
    import numpy as np

    most = ops.KV4_ROW_KEYS // 32
    blocks = np.unique(np.concatenate([np.arange(1, 5000), most - np.arange(5000), np.random.RandomState(1).randint(1, most, 20000)]))
    for ranges in range(1, 65):
        blocks_r = np.unique(np.concatenate([blocks, blocks // ranges * ranges, np.minimum(blocks // ranges * ranges + 1, most)]))
        blocks_r = blocks_r[blocks_r > 0]
        exact = np.float32(1) / np.float32(ranges)
        for inverse in (np.nextafter(exact, np.float32(0)), exact, np.nextafter(exact, np.float32(2))):
            share = (blocks_r.astype(np.float32) * inverse).astype(np.int64) + 1
            assert (share * ranges >= blocks_r).all()

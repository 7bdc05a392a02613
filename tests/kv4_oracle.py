"""The 4-bit cache in 64 bits, from its definition: what a value is kept as, and attention over what is kept."""

from __future__ import annotations

import math

import numpy as np
import torch

TINY, HUGE = 2.0**-100, 2.0**100


def outward(x: torch.Tensor, up: bool) -> torch.Tensor:
    """float64 -> the next bfloat16 value that is no smaller (``up``) or no larger, as float64."""
    near = x.float().to(torch.bfloat16)
    toward = torch.full_like(near, math.inf if up else -math.inf)
    for _ in range(2):  # (rounding to 32 bits first may land one value off)
        wrong = (near.double() < x) if up else (near.double() > x)
        near = torch.where(wrong, torch.nextafter(near, toward), near)
    return near.double()


def quantised(x: torch.Tensor):
    """float64 [..., channels] -> codes, step, low (float64, the last two [..., 1])."""
    low = outward(x.amin(-1, keepdim=True), up=False)
    reach = x.amax(-1, keepdim=True) - low
    fine = (reach < HUGE) & torch.isfinite(x).all(-1, keepdim=True)
    reach = torch.where(fine, reach, 0.0)
    step = outward(reach / 15, up=True)
    step = torch.where(step < TINY, 0.0, step)
    codes = torch.where(step > 0, torch.round((x - low) / step), 0.0)
    return torch.where(fine, codes, 0.0).clamp(0, 15), step, torch.where(fine, low, math.nan)


def rotated(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, rot: int, interleaved: bool = False, factor: float = 1.0) -> torch.Tensor:
    """float64 [tokens, heads, dim]; the angle is formed in 32 bits, as everywhere in the engine."""
    angle = (positions.float()[:, None] * inv_freq[None, :]).double()[:, None]
    cos, sin = angle.cos() * factor, angle.sin() * factor
    out = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2 : rot])
    first, second = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = first, second
    else:
        out[..., : rot // 2], out[..., rot // 2 : rot] = first, second
    return out


def scattered_tables(counts, spare, seed):
    """Block tables [requests, widest] over a pool with every page somewhere of its own; the pages a request lacks are named -1.  -> tables, pages"""
    gen = torch.Generator().manual_seed(seed)
    total = sum(counts) + spare
    order = torch.randperm(total, generator=gen, dtype=torch.int32)
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at : at + c]
        at += c
    return table, total


def attention(q, keys, values, lens, starts, tables, page, heads, kv_heads, scale, window=0):
    """float64 CPU: q [tokens, heads, dim]; keys, values [pages, kv_heads, page, dim].  -> out [tokens, heads, dim], and the largest |score| bound terms
    that tolerances are derived from: (sum over channels of |q| |k|, times scale, the largest of any visible pair)."""
    out, at, size = torch.empty_like(q), 0, 0.0
    group = heads // kv_heads
    for r, (m, s) in enumerate(zip(lens, starts)):
        held = m + s
        lo = max(0, s - window + 1) if window else 0  # (pages before a window may have been released)
        pages = tables[r, lo // page : -(-held // page)].long()
        k0 = lo // page * page
        for h in range(kv_heads):
            k = keys[pages, h].reshape(-1, keys.shape[-1])[: held - k0]
            v = values[pages, h].reshape(-1, values.shape[-1])[: held - k0]
            pos, key = torch.arange(s, held), torch.arange(k0, held)
            hidden = key[None] > pos[:, None]
            if window:
                hidden = hidden | (key[None] <= pos[:, None] - window)
            for g in range(h * group, (h + 1) * group):
                qq = q[at : at + m, g]
                w = torch.softmax((qq @ k.T * scale).masked_fill(hidden, -math.inf), -1)
                # a weight of 0 takes nothing from a value that is no number
                seen = torch.where(hidden.all(0)[:, None], 0.0, v)
                nan = torch.isnan(seen).any(1)
                o = w @ torch.nan_to_num(seen)
                o[(~hidden & nan[None]).any(1)] = math.nan
                out[at : at + m, g] = o
                size = max(size, float((torch.nan_to_num(qq).abs() @ torch.nan_to_num(k).abs().T).max()) * scale)
        at += m
    return out, size


def batch_context(lens, starts, tables, device, captured=False):
    """The step's context that the attention part hands to its kernels."""
    from nanospec_amd.engine.arena import Arena
    from nanospec_amd.engine.context import BatchLayout, StepContext, fill_batch
    from nanospec_amd.parts.attention import TILES

    n = sum(lens)
    layout = BatchLayout(n, len(lens), 1, 1, tables.shape[1], plans=[(TILES, TILES.shape(lens))])
    host = torch.zeros(layout.total, dtype=torch.int32)
    fill_batch(host.numpy(), layout, [0] * n, starts, lens, list(range(len(lens))), [0], [np.asarray(tables)])
    held = [a + b for a, b in zip(lens, starts)]
    return StepContext(layout, host.to(device), Arena(torch.device(device)), max_position=max(held) - 1, max_kv_len=max(held),
                       max_chunk_kv=max((h for h, m in zip(held, lens) if m != 1), default=0), captured=captured)

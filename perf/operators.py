"""Operators of a model that is served in few bits: keys and values cached in 4 bits, matrix products in 8-bit integers.

* ``append``: the tokens of a step enter the cache: queries and keys rotated, keys and values of every head quantised to 4 bits
  and written into their pages.
* ``decode`` and ``portion``: attention over such pages, of single tokens and of portions of prompts.
* ``product``: a row's activations quantised to 8 bits (as they are, behind the RMS norm in front of a sublayer, or behind the
  gate of a feed-forward) and multiplied with a weight matrix in 8 bits.

What a value in few bits stands for.  Keys and values: the channels of a head's key, or value, of a token share a step and a lowest
value, both bfloat16, rounded outwards so that the range holds every channel: ``step * code + low``, codes 0 to 15.  Activations: a
row's values are ``scale * code`` with scale = largest magnitude / 127; weights likewise, a scale an output channel.

Shapes are those of the Llama 3 decoders that ``bench.py`` runs (1B: 32 heads of 64 over 8; 8B: 32 of 128 over 8; 70B: 64 of 128
over 8), lengths ragged as a server's requests are, pages of 16 tokens scattered over the pool.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TINY = 2.0**-100  # a step, or a row's largest magnitude, below this counts as 0
ROPE_BASE = 500000.0


def listed():
    b = dict(page=16, dtype="bf16")
    return [
        # decoding with the 1B shape: the tokens of 7 requests enter the cache
        dict(b, name="append-1b-7", kind="append", requests=7, tokens=1, context=900, heads=32, kv_heads=8, dim=64),
        # three long prompts of the 8B shape arrive in one step
        dict(b, name="append-8b-3x1365", kind="append", requests=3, tokens=1365, context=0, heads=32, kv_heads=8, dim=128),
        # one user's chat on the 1B shape: the latency of a token
        dict(b, name="decode-1b-1x1100", kind="decode", requests=1, context=1100, heads=32, kv_heads=8, dim=64, window=0),
        # eight requests of the 8B shape in the middle of a conversation
        dict(b, name="decode-8b-8x4000", kind="decode", requests=8, context=4000, heads=32, kv_heads=8, dim=128, window=0),
        # a loaded server: 61 requests of the 8B shape
        dict(b, name="decode-8b-61x6000", kind="decode", requests=61, context=6000, heads=32, kv_heads=8, dim=128, window=0),
        # two long documents on the 70B shape
        dict(b, name="decode-70b-2x100000", kind="decode", requests=2, context=100000, heads=64, kv_heads=8, dim=128, window=0),
        # a whole prompt of 2,048 tokens on the 8B shape
        dict(b, name="portion-8b-2048", kind="portion", requests=1, tokens=2048, context=0, heads=32, kv_heads=8, dim=128, window=0),
        # chunked prefill: portions of two long prompts of the 8B shape
        dict(b, name="portion-8b-2x333-at-20000", kind="portion", requests=2, tokens=333, context=20000, heads=32, kv_heads=8, dim=128, window=0),
        # output projection of the 1B shape for one token, in the 32-bit path: the smallest call
        dict(name="int8-f32-1x2048x2048", kind="product", rows=1, cols=2048, inner=2048, source="rows", dtype="f32"),
        # gate and up of the 8B shape behind the norm, eight requests decoding
        dict(name="int8-norm-8x28672x4096", kind="product", rows=8, cols=28672, inner=4096, source="norm", dtype="bf16"),
        # the down-projection of the 8B shape behind the gate, 61 requests decoding
        dict(name="int8-silu-61x4096x14336", kind="product", rows=61, cols=4096, inner=14336, source="silu", dtype="bf16"),
        # gate and up of the 8B shape for a prompt of 2,048 tokens
        dict(name="int8-2048x28672x4096", kind="product", rows=2048, cols=28672, inner=4096, source="rows", dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "portion", "product", "product"))
    if kind == "product":
        rows, inner = _log(rng, 1, 2048), _log(rng, 512, 14336)
        cols = _log(rng, 512, 28672)
        if rng.random() < 0.6:  # (most models' widths are round, some are not)
            inner, cols = -(-inner // 128) * 128, -(-cols // 64) * 64
        source = rng.choice(("rows", "norm", "silu"))
        dtype = "f32" if source == "rows" and rng.random() < 0.3 else "bf16"
        while rows * inner * cols > 2048 * 28672 * 4096:
            rows = max(1, rows // 2)
        return dict(kind=kind, rows=rows, cols=cols, inner=inner, source=source, dtype=dtype)
    heads, kv_heads, dim = rng.choice(((32, 8, 64), (32, 8, 128), (64, 8, 128), (16, 16, 64), (24, 8, 128), (40, 5, 128), (12, 2, 64), (28, 4, 128)))
    shape = dict(heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice((8, 16, 16, 16, 32, 64)), dtype="f32" if rng.random() < 0.15 else "bf16")
    if kind == "append":
        requests = _log(rng, 1, 64)
        return dict(shape, kind=kind, requests=requests, tokens=rng.choice((1, _log(rng, 1, 4095 // requests))), context=rng.choice((0, _log(rng, 1, 60000))))
    window = _log(rng, 64, 4096) if rng.random() < 0.15 else 0
    if kind == "decode":
        requests = _log(rng, 1, 64)
        return dict(shape, kind=kind, requests=requests, context=_log(rng, 1, min(100000, 366000 // requests)), window=window)
    requests = rng.choice((1, 1, 2, 3))
    tokens = _log(rng, 2, 2048 // requests)
    return dict(shape, kind=kind, requests=requests, tokens=tokens, context=rng.choice((0, _log(rng, 1, min(20000, 13000000 // (requests * tokens) + 1)))), window=window)


# ---------------------------------------------------------------------------------------------- what few bits stand for


def _floor_bf16(x):
    """The largest bfloat16 value that is no larger, as float32."""
    bits = x.contiguous().view(torch.int32)
    down = bits & -65536
    return torch.where((bits < 0) & ((bits & 65535) != 0), down + 65536, down).view(torch.float32)


def _quantise4(x):
    """float32 [..., channels] -> codes (uint8), step and low (float32 [..., 1], bfloat16 values)."""
    low = _floor_bf16(x.amin(-1, keepdim=True))
    reach = x.amax(-1, keepdim=True) - low
    step = -_floor_bf16(-(reach / torch.full_like(reach, 15.0)))
    fine = torch.isfinite(reach)
    step = torch.where(fine & (step >= TINY), step, 0.0)
    low = torch.where(fine, low, math.nan)
    # (divided, not times 1 / step: short numbers often lie half way between two codes exactly, which the quotient keeps)
    codes = torch.where(step > 0, torch.round((x - low) / step), 0.0).clamp(0, 15)
    return codes.to(torch.uint8), step, low


def _rotate(x, positions, inv_freq):
    """Channels j and j + dim / 2 of float32 [tokens, heads, dim] turn by position * inv_freq[j], an angle that is formed in 32 bits (as
    everywhere in the model: positions beyond what 32 bits tell apart would turn the queries and keys of other layers apart)."""
    angle = (positions.float()[:, None] * inv_freq[None, :])[:, None, :]
    cos, sin = torch.cos(angle), torch.sin(angle)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _types(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


# ---------------------------------------------------------------------------------------------- inputs


def _lengths(case, gen):
    """Ragged: (tokens of each request in this step, tokens that it has in the cache before)."""
    n = case["requests"]
    ragged = lambda mean, least: (mean * (0.5 + torch.rand(n, generator=gen))).long().clamp(least) if n > 1 else torch.full((1,), max(mean, least))
    most = case.get("tokens", 1)
    lens = torch.ones(n, dtype=torch.long)
    if most > 1:  # ragged, and as many tokens in all as the case says
        least = 2 if case["kind"] == "portion" else 1
        share = 0.5 + torch.rand(n, generator=gen, dtype=torch.float64)
        lens = (share * ((most - least) * n / float(share.sum()))).long() + least
        lens[0] += most * n - int(lens.sum())
    before = ragged(case["context"], 0) if case["context"] else torch.zeros(n, dtype=torch.long)
    if case["kind"] == "decode":
        before = (before.double() * (case["context"] * n / max(1.0, float(before.sum())))).long()
    return lens.tolist(), before.tolist()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    dtype = _types(case)
    if case["kind"] == "product":
        return _prepare_product(case, randn, dtype)
    lens, before = _lengths(case, torch.Generator().manual_seed(seed))
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    held = [a + b for a, b in zip(lens, before)]
    n, width = sum(lens), -(-max(held) // page)
    counts = [-(-h // page) for h in held]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 1), dtype=torch.int32)
    tables = torch.full((len(held), width), 0, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        tables[i, :c] = order[at : at + c]
        at += c
    state = dict(case=dict(case), lens=lens, before=before)
    inv_freq = (1.0 / ROPE_BASE ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim)).to(DEV)
    requests = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    positions = torch.cat([torch.arange(b, b + m) for m, b in zip(lens, before)])
    state.update(table=tables.to(DEV), positions=positions.to(DEV, torch.int32), token_req=requests.to(DEV, torch.int32), inv_freq=inv_freq, pages=pages)
    if case["kind"] == "append":
        # a product's output: a few channels of the keys are much larger than the others
        row = randn(n, (heads + 2 * kv_heads) * dim)
        row[:, heads * dim : (heads + kv_heads) * dim] *= 1 + 4 * (torch.arange(dim, device=DEV) % 29 == 3).float().repeat(kv_heads)
        state["qkv"] = row.to(dtype)
        if own:
            from nanospec_amd.kernels import ops

            state["pool"] = ops.Kv4Pages.empty(pages, kv_heads, page, dim, DEV)
        return state
    k = randn(pages, kv_heads, page, dim)
    k *= 1 + 3 * (torch.arange(dim, device=DEV) % 29 == 3).float()
    k_codes, k_step, k_low = _quantise4(k)
    del k
    v_codes, v_step, v_low = _quantise4(0.5 * randn(pages, kv_heads, page, dim))
    state["q"] = (1.3 * randn(n, heads * dim)).to(dtype)
    marks = [t[..., 0].to(torch.bfloat16) for t in (k_step, k_low, v_step, v_low)]
    if own:
        # what a server holds: the pages, and the step's batch as the engine lays it out for a layer's kernels
        from nanospec_amd.engine.arena import Arena
        from nanospec_amd.engine.context import BatchLayout, StepContext, fill_batch
        from nanospec_amd.kernels import ops
        from nanospec_amd.parts.attention import TILES

        state["pool"] = ops.Kv4Pages.from_codes(k_codes, marks[0], marks[1], v_codes, marks[2], marks[3])
        layout = BatchLayout(n, len(lens), 1, 1, width, plans=[(TILES, TILES.shape(lens))])
        host = torch.zeros(layout.total, dtype=torch.int32)
        fill_batch(host.numpy(), layout, [0] * n, before, lens, list(range(len(lens))), [0], [tables.numpy()])
        longest = max((h for h, m in zip(held, lens) if m != 1), default=0)
        state["ctx"] = StepContext(layout, host.to(DEV), Arena(torch.device(DEV, torch.cuda.current_device())), max_position=max(held) - 1, max_kv_len=max(held), max_chunk_kv=longest)
    else:
        state.update(k=(k_codes, marks[0], marks[1]), v=(v_codes, marks[2], marks[3]))
    return state


def _prepare_product(case, randn, dtype):
    rows, cols, inner, source = case["rows"], case["cols"], case["inner"], case["source"]
    w = 0.02 * randn(cols, inner)
    scale = w.abs().amax(1, keepdim=True) / torch.full_like(w[:, :1], 127.0)
    codes = torch.round(w / scale).to(torch.int8)
    state = dict(case=dict(case))
    # activations: a few channels are far larger than the others
    large = 1 + 15 * (torch.arange(inner, device=DEV) % 401 == 17).float()
    if source == "rows":
        state["x"] = (randn(rows, inner) * large).to(dtype)
    elif source == "norm":
        state.update(resid=(3 * randn(rows, inner)).to(dtype), delta=randn(rows, inner).to(dtype), weight=((1 + 0.1 * randn(inner)) * large).to(dtype), eps=1e-5)
    else:
        state["gate_up"] = randn(rows, 2 * inner).to(dtype)
    if own:
        from nanospec_amd.kernels import ops

        state["w"] = ops.Int8Weight(codes, scale[:, 0])
    else:
        state["w"] = (codes, scale[:, 0].contiguous())
    return state


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _run_own(state, case, kind)
    if kind == "product":
        return _plain_product(state, case)
    if kind == "append":
        return _plain_append(state, case)
    return _plain_attention(state, case)


def _run_own(state, case, kind):
    from nanospec_amd.kernels import ops

    if kind == "product":
        if case["source"] == "rows":
            return ops.linear_int8(ops.int8_rows(state["x"]), state["w"], dtype=state["x"].dtype)
        if case["source"] == "silu":
            return ops.linear_int8(ops.silu_mul_int8(state["gate_up"]), state["w"], dtype=state["gate_up"].dtype)
        resid = torch.empty_like(state["resid"])
        rows = ops.rmsnorm_int8(state["weight"], state["eps"], resid=state["resid"], x=state["delta"], resid_out=resid)
        return ops.linear_int8(rows, state["w"], dtype=resid.dtype), resid
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if kind == "append":
        qkv = state["qkv"]
        where = (state["positions"], state["token_req"], state["table"])
        q = torch.empty((qkv.shape[0], heads * dim), dtype=qkv.dtype, device=qkv.device)
        ops.rope_kv4_write(qkv, *where, state["inv_freq"], state["pool"], heads, kv_heads, dim, dim, q_out=q)
        keys, values = ops.kv4_read(state["pool"], *where, dtype=torch.bfloat16)
        return q, keys, values
    from nanospec_amd.parts.attention import kv4_attention

    ctx = state["ctx"]
    ctx.arena.reset()
    return kv4_attention(ctx, state["q"], torch.empty_like(state["q"]), state["pool"], ctx.block_tables[0], heads, kv_heads, dim, dim**-0.5, window=case["window"])


def _quantise8(x):
    """float32 [rows, k] -> codes (float32) and scales [rows, 1]."""
    most = x.abs().amax(1, keepdim=True)
    most = torch.where(most < TINY, 0.0, most)
    full = torch.full_like(most, 127.0)
    inverse = torch.where(most > 0, full / most, most)  # (0, or not a number where one is none)
    return torch.round(x * inverse).clamp(-127, 127), most / full


def _plain_product(state, case):
    codes, w_scale = state["w"]
    more = ()
    if case["source"] == "rows":
        dtype, x = state["x"].dtype, state["x"].float()
    elif case["source"] == "silu":
        dtype = state["gate_up"].dtype
        gate, up = state["gate_up"].float().chunk(2, 1)
        x = gate / (1 + torch.exp(-gate)) * up
    else:
        dtype = state["resid"].dtype
        resid = (state["resid"].float() + state["delta"].float()).to(dtype)
        r = resid.float()
        x = state["weight"].float() * (r * torch.rsqrt(r.square().mean(1, keepdim=True) + state["eps"]))
        more = (resid,)
    rows, scale = _quantise8(x)
    y = ((rows @ codes.float().t()) * scale * w_scale[None, :]).to(dtype)
    return (y, *more) if more else y


def _plain_append(state, case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    n = state["qkv"].shape[0]
    q, k, v = state["qkv"].float().view(n, heads + 2 * kv_heads, dim).split((heads, kv_heads, kv_heads), 1)
    q, k = _rotate(q, state["positions"], state["inv_freq"]), _rotate(k, state["positions"], state["inv_freq"])
    value = lambda t: t[0].float() * t[1] + t[2]
    return q.reshape(n, -1).to(state["qkv"].dtype), value(_quantise4(k)).to(torch.bfloat16), value(_quantise4(v)).to(torch.bfloat16)


def _plain_attention(state, case):
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = heads // kv_heads
    table, lens = state["table"].long(), state["lens"]
    count, most = len(lens), max(lens)
    keys = table.shape[1] * page

    def gathered(codes, step, low):  # [requests, kv_heads, keys, dim] in 32 bits
        of = lambda t: t[table].transpose(1, 2).reshape(count, kv_heads, keys, *t.shape[3:])
        return of(codes).float() * of(step).float()[..., None] + of(low).float()[..., None]

    # queries in a rectangle of requests and tokens; what a request does not bring reads row 0 and is left out at the end
    length = torch.tensor(lens, device=DEV)
    first = length.cumsum(0) - length
    token = torch.arange(most, device=DEV)
    brings = token[None, :] < length[:, None]
    rows = torch.where(brings, first[:, None] + token[None, :], 0)
    q = state["q"].float()[rows].view(count, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(count, kv_heads, group * most, dim)
    scores = torch.matmul(q, gathered(*state["k"]).transpose(2, 3)).view(count, kv_heads, group, most, keys) * dim**-0.5
    position = state["positions"].long()[rows]
    key = torch.arange(keys, device=DEV)
    seen = key[None, None, :] <= position[:, :, None]
    if case["window"]:
        seen = seen & (key[None, None, :] > position[:, :, None] - case["window"])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = scores.sum(-1, keepdim=True)
    o = torch.matmul(scores.view(count, kv_heads, group * most, keys), gathered(*state["v"])).view(count, kv_heads, group, most, dim) / total
    return o.permute(0, 3, 1, 2, 4)[brings].reshape(-1, heads * dim).to(state["q"].dtype)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "product":
        m, n, k = case["rows"], case["cols"], case["inner"]
        x = {"rows": 1, "norm": 3, "silu": 2}[case["source"]] * m * k * e  # (norm: two read, one written)
        return {"bytes": n * (k + 4) + x + m * n * e, "flops": 2 * m * n * k}
    heads, kv_heads, dim, requests, before = case["heads"], case["kv_heads"], case["dim"], case["requests"], case["context"]
    a_token = kv_heads * (dim + 8)  # codes of a key and a value, a step and a low each
    tokens = case.get("tokens", 1) if case["kind"] != "decode" else 1
    n = requests * tokens
    if case["kind"] == "append":
        return {"bytes": n * ((heads + 2 * kv_heads) * dim * e + heads * dim * e + a_token + 2 * kv_heads * dim * 2), "flops": n * dim * (6 * heads + 16 * kv_heads)}
    window = case["window"] or 1 << 40
    seen = min(before + 1, window) if tokens == 1 else sum(min(before + i + 1, window) for i in range(tokens)) / tokens
    held = min(before + tokens, window + tokens - 1)
    return {"bytes": requests * held * a_token + 2 * n * heads * dim * e, "flops": 4.0 * n * heads * dim * seen}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    global own
    before_own, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before_own
    if case["kind"] == "product":
        return _exact_product(state, case)
    if case["kind"] == "append":
        return _exact_append(state, case)
    return _exact_attention(state, case)


def _exact_product(state, case):
    codes, w_scale = state["w"]
    resid = None
    if case["source"] == "rows":
        x = state["x"].double()
    elif case["source"] == "silu":
        g = state["gate_up"][:, : case["inner"]].double()
        x = g * torch.sigmoid(g) * state["gate_up"][:, case["inner"] :].double()
    else:
        # (the stream is kept in the model's precision: the norm reads the rounded sum)
        resid = state["resid"].double() + state["delta"].double()
        r = resid.to(state["resid"].dtype).double()
        x = r / (r.pow(2).mean(1, keepdim=True) + state["eps"]).sqrt() * state["weight"].double()
    most = x.abs().max(1, keepdim=True).values
    # a code is the whole number next to x * (127 / most), formed in 32 bits
    inverse = torch.where(most >= TINY, torch.full_like(most, 127.0).float() / most.float(), 0.0)
    rows = torch.round(x.float() * inverse).double()
    y = torch.cat([rows @ part.double().t() for part in codes.split(4096)], 1) * (most / 127) * w_scale.double()
    return y if resid is None else (y, resid)


def _exact_append(state, case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    x = state["qkv"].double().view(-1, heads + 2 * kv_heads, dim)
    angle = (state["positions"].float()[:, None] * state["inv_freq"]).double()  # formed in 32 bits by definition
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]
    half = dim // 2
    turned = torch.complex(x[..., :half], x[..., half:])[:, : heads + kv_heads] * turn
    turned = torch.cat((turned.real, turned.imag), -1)
    out = []
    for t in (turned[:, heads:], x[:, heads + kv_heads :]):
        low = t.min(-1, keepdim=True).values
        near = low.to(torch.bfloat16)
        low = torch.where(near.double() > low, torch.nextafter(near, torch.full_like(near, -math.inf)), near).double()
        step = (t.max(-1, keepdim=True).values - low) / 15
        near = step.to(torch.bfloat16)
        step = torch.where(near.double() < step, torch.nextafter(near, torch.full_like(near, math.inf)), near).double()
        out.append(torch.round((t - low) / step).clamp(0, 15) * step + low)
    return turned[:, :heads].reshape(len(x), -1), out[0], out[1]


def _exact_attention(state, case):
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group, at, out = heads // kv_heads, 0, []
    for r, (m, b) in enumerate(zip(state["lens"], state["before"])):
        held = m + b
        at_pages = state["table"][r, : -(-held // page)].long()
        pos = torch.arange(b, held, device=DEV)
        key = torch.arange(held, device=DEV)
        hidden = key[None, :] > pos[:, None]
        if case["window"]:
            hidden |= key[None, :] <= pos[:, None] - case["window"]
        q = state["q"][at : at + m].double().view(m, heads, dim)
        o = torch.empty_like(q)
        for h in range(kv_heads):
            k, v = ((c[at_pages, h].double() * s[at_pages, h].double()[..., None] + z[at_pages, h].double()[..., None]).reshape(-1, dim)[:held]
                    for c, s, z in (state["k"], state["v"]))
            for g in range(h * group, (h + 1) * group):
                s = (q[:, g] @ k.t()) / math.sqrt(dim)
                o[:, g] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
        at += m
        out.append(o.reshape(m, -1))
    return torch.cat(out)
